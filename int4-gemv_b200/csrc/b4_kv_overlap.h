// b4_kv_overlap.h -- which outputs lie on what a call reads: rows of tokens and heads
// with strides of their own, by arithmetic on the host.
#pragma once

#include <algorithm>
#include <cstdint>
#include <cstdlib>

namespace b4 {

// n tokens of `heads` rows of `bytes`; strides in bytes
struct RowSet {
    __int128 at, tok, head;
    long long n, heads, bytes;
};

inline RowSet row_set(const void* at, long long item, long long tok, long long head, long long n, long long heads, long long columns)
{
    RowSet r = {(__int128)reinterpret_cast<uintptr_t>(at), (__int128)tok * item, (__int128)head * item, n, heads, columns * item};
    if (n <= 1) r.tok = 0;
    if (heads <= 1) r.head = 0;
    if (r.tok < 0) {                       // from the other end
        r.at += r.tok * (n - 1);
        r.tok = -r.tok;
    }
    if (r.head < 0) {
        r.at += r.head * (heads - 1);
        r.head = -r.head;
    }
    return r;
}

// `n` values in a row
inline RowSet row_set(const void* at, long long item, long long n) { return row_set(at, item, 0, 0, 1, 1, n); }

// Is there a k in [from, to] with -before < off + k * step < after?  step >= 0.
inline bool meets_step(__int128 off, __int128 before, __int128 after, __int128 step, long long from, long long to)
{
    if (from > to) return false;
    if (step == 0) return -before < off && off < after;
    const __int128 low = -before - off + 1, high = after - off - 1;        // low <= k * step <= high
    if (low > high) return false;
    const __int128 k0 = low >= 0 ? (low + step - 1) / step : -(-low / step), k1 = high >= 0 ? high / step : -((-high + step - 1) / step);
    return std::max<__int128>(k0, from) <= std::min<__int128>(k1, to);
}

// Do some bytes of a lie on some of b?  Exact where both have one token stride or one of them one token; sets whose
// token strides differ meet where the addresses between their ends do.
inline bool rows_meet(RowSet a, RowSet b)
{
    if (a.n < 1 || b.n < 1 || a.heads < 1 || b.heads < 1 || a.bytes < 1 || b.bytes < 1) return false;
    const __int128 wide_a = (a.heads - 1) * a.head + a.bytes, wide_b = (b.heads - 1) * b.head + b.bytes;      // of a token
    if (a.at + (a.n - 1) * a.tok + wide_a <= b.at || b.at + (b.n - 1) * b.tok + wide_b <= a.at) return false;
    if (a.n == 1) a.tok = b.tok;
    if (b.n == 1) b.tok = a.tok;
    if (a.tok != b.tok) return true;
    const long long from = 1 - b.n, to = a.n - 1;
    if (!meets_step(a.at - b.at, wide_a, wide_b, a.tok, from, to)) return false;
    if (a.heads == 1) a.head = b.head;
    if (b.heads == 1) b.head = a.head;
    if (a.head == b.head) {                // only how far apart two heads are
        for (long long h = 1 - b.heads; h < a.heads; ++h)
            if (meets_step(a.at - b.at + h * a.head, a.bytes, b.bytes, a.tok, from, to)) return true;
        return false;
    }
    for (long long h = 0; h < a.heads; ++h)
        for (long long i = 0; i < b.heads; ++i)
            if (meets_step(a.at + h * a.head - b.at - i * b.head, a.bytes, b.bytes, a.tok, from, to)) return true;
    return false;
}

// Do two rows of one set share bytes?
inline bool rows_overlap(const RowSet& a)
{
    if (a.n > 1 && a.tok < a.bytes) return true;
    if (a.head >= a.bytes && (a.n <= 1 || a.tok >= (a.heads - 1) * a.head + a.bytes)) return false;          // token after token
    if (a.heads > 1 && a.head >= (a.n - 1) * a.tok + a.bytes) return false;                                  // head after head
    for (long long h = 1; h < a.heads; ++h)
        if (meets_step(h * a.head, a.bytes, a.bytes, a.tok, 1 - a.n, a.n - 1)) return true;
    return false;
}

}  // namespace b4
