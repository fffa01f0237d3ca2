// b4_kv_rotary.cu -- the quantising append with the rotary embedding of queries and
// keys on the way.
//
// Mathematics.  A position's angle is position * turns mod 2^64, in whole steps of
// 2^-64 turn: exact relative to the table for any position (the table is off by 2^-52 of a
// frequency at most), so what is rounded is the angle itself (to 2^-53 of half a turn), its
// sine and cosine, and the rotated column, once.  Keys are rotated in fp64: their 4-bit
// codes are then those of the exact rotation by the table's angles but where it lies
// within 2^-50 of a border, whatever computes it, for 2 DFMA a column of a few heads;
// queries, whose rounding to 16 bits is next, in fp32.
//
// Split.  A warp takes a token, or a part of its vectors (heads of q, k and v), 32 * 8 / D
// of one kind at a time, and computes the token's angles itself, one or two a lane: no
// shared memory, no barrier.  A lane holds four pairs' columns, from both halves of a
// head (eight neighbours where neighbours pair), so a pair never leaves its lane.  (A CTA
// of eight warps for four tokens, angles in shared memory and pairs by shuffles, took
// 154 us where this takes 71.)
//
// What bounds it.  Many tokens: issue, 2.9 of 4 slots, beside memory: 20011 tokens x
// (28 + 2 x 4) x 128 from bf16 with three axes into NF4 take 71.4 us, 403 MB, 5.65 TB/s
// (NF4's codes are 32 instructions each, a token's angles some 300 for its warp); 6007 x
// (32 + 2 x 8) x 64 in fp16 into INT4, half of the columns turned, 21.6 us, 66 MB.  Few:
// latency, 64 x (64 + 2 x 8) x 128 from fp32 in 4.1 us (one token 2.5).
#include <climits>
#include <cmath>
#include <type_traits>

#include "b4_kv_overlap.h"
#include "b4_kv_quant.cuh"

namespace b4 {
namespace {

struct RotaryParams {
    KvLayout l;
    uint8_t* blocks;
    const void* src[3];                // k, v, q
    long long tok[3], head[3];         // their strides
    void* out;
    long long out_tok, out_head;
    const int32_t *positions, *slots;
    long long axis_stride;
    const uint64_t* turns;
    const uint8_t* axes;
    int n, heads, half, n_axes;
    int parts;                         // warps that share a token's vectors
    bool vec;                          // rows are 16-byte aligned
    float scale;
};

constexpr int kRotThreads = 256, kRotWarps = kRotThreads / 32;

// a lane's 8 columns of T as loaded, four at a and four at b (ADJ: right behind them), and as fp32
template <typename T, bool ADJ>
struct Pairs {
    uint32_t raw[2 * sizeof(T)];
    __device__ void load(const T* a, const T* b, bool vec)
    {
        if (!vec) {
            T* r = reinterpret_cast<T*>(raw);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                r[i] = a[i];
                r[4 + i] = b[i];
            }
        } else if (sizeof(T) == 4) {
            *reinterpret_cast<uint4*>(raw) = __ldg(reinterpret_cast<const uint4*>(a));
            *reinterpret_cast<uint4*>(raw + 4) = __ldg(reinterpret_cast<const uint4*>(b));
        } else if (ADJ) {
            *reinterpret_cast<uint4*>(raw) = __ldg(reinterpret_cast<const uint4*>(a));
        } else {
            *reinterpret_cast<uint2*>(raw) = __ldg(reinterpret_cast<const uint2*>(a));
            *reinterpret_cast<uint2*>(raw + 2) = __ldg(reinterpret_cast<const uint2*>(b));
        }
    }
    __device__ float get(int i) const { return kv_float(reinterpret_cast<const T*>(raw)[i]); }
};

template <typename T, typename O, int FMT, int D, bool ADJ>
__global__ void __launch_bounds__(kRotThreads, 4) kv_append_rotary_kernel(const RotaryParams p)
{
    constexpr int TPV = D / 8, VPW = 32 / TPV;         // threads a vector, vectors a warp
    constexpr int U = sizeof(T) == 2 ? 4 : 2;          // query items in flight
    constexpr int P = D / 64;                          // pairs whose angles a lane computes
    float boundary = 4.0f;
    int below = 0;
    if (FMT == B4_KV_NF4) nf4_bins(boundary, below);
    const int lane = threadIdx.x & 31, sub = lane % TPV;
    const int token = (int)blockIdx.x * kRotWarps + (threadIdx.x >> 5), part = blockIdx.y;
    kv_begin();
    if (token >= p.n) return;

    // this lane's columns: pairs i0 .. i0 + 3 where it turns, two groups of four of the others where not
    const bool turn = sub < p.half / 4;
    const int i0 = 4 * sub, rest = D - 2 * p.half;
    const int col_a = ADJ ? 8 * sub : turn ? i0 : p.half + i0;
    const int col_b = ADJ ? 8 * sub + 4 : turn ? p.half + i0 : p.half + rest / 2 + i0;
    const int kv_items = (p.l.kv_heads + VPW - 1) / VPW, q_items = (p.heads + VPW - 1) / VPW;
    auto head_of = [&](int item, int heads) { return min(item * VPW + lane / TPV, heads - 1); };   // whole warps take part in the shuffles
    auto load = [&](int kind, int head, Pairs<T, ADJ>& x) {
        const T* src = static_cast<const T*>(p.src[kind]) + token * p.tok[kind] + head * p.head[kind];
        x.load(src + col_a, src + col_b, p.vec);
    };

    // ---- keys and values: items 0 .. 2 kv_items - 1 of the token; the first is asked for before the angles are computed ----
    int at = part;
    Pairs<T, ADJ> x;
    if (at < 2 * kv_items) load(at >= kv_items, head_of(at < kv_items ? at : at - kv_items, p.l.kv_heads), x);
    const int slot = __ldg(p.slots + token), page = slot >> p.l.page_shift;

    double co[P], si[P];                               // pairs P * lane ..
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int pair = min(P * lane + i, p.half - 1);
        const int axis = p.axes ? min((int)__ldg(p.axes + pair), p.n_axes - 1) : 0;
        const long long pos = __ldg(p.positions + axis * p.axis_stride + token);
        const uint64_t phase = (uint64_t)pos * __ldg(reinterpret_cast<const unsigned long long*>(p.turns) + pair);
        sincospi((double)(int64_t)phase * 0x1p-63, &si[i], &co[i]);
        si[i] *= p.scale;
        co[i] *= p.scale;
    }
    // pair j of this lane's four
    auto cos_of = [&](int j) { return __shfl_sync(0xffffffffu, co[j % P], (4 * sub + j) / P & 31); };
    auto sin_of = [&](int j) { return __shfl_sync(0xffffffffu, si[j % P], (4 * sub + j) / P & 31); };

    const bool live = slot >= 0 && page < p.l.n_pages;
    for (; at < 2 * kv_items; at += p.parts) {
        const bool value = at >= kv_items;
        const int item = value ? at - kv_items : at;
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = x.get(j);
        if (const int next = at + p.parts; next < 2 * kv_items)
            load(next >= kv_items, head_of(next < kv_items ? next : next - kv_items, p.l.kv_heads), x);
        if (!value) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double c = cos_of(j), s = sin_of(j);
                float &a = ADJ ? v[2 * j] : v[j], &b = ADJ ? v[2 * j + 1] : v[4 + j];
                const double da = a, db = b;
                if (turn) {
                    a = (float)(da * c - db * s);
                    b = (float)(db * c + da * s);
                }
            }
        }
        float scale;
        __half sh;
        const uint32_t w = quantised_word<FMT, TPV>(v, boundary, below, scale, sh);
        const int head = item * VPW + lane / TPV;
        if (!live || head >= p.l.kv_heads) continue;
        uint8_t* block = p.blocks + ((long long)page * p.l.kv_heads + head) * p.l.block;
        const int row = (value ? p.l.page_size : 0) + (slot & (p.l.page_size - 1));
        if (ADJ) {
            reinterpret_cast<uint32_t*>(block + row * (D / 2))[sub] = w;
        } else {
            *reinterpret_cast<uint16_t*>(block + row * (D / 2) + col_a / 2) = (uint16_t)w;
            *reinterpret_cast<uint16_t*>(block + row * (D / 2) + col_b / 2) = (uint16_t)(w >> 16);
        }
        if (sub == 0) {
            if (FMT == B4_KV_INT4) reinterpret_cast<__half*>(block + p.l.page_size * D)[row] = sh;
            else reinterpret_cast<float*>(block + p.l.page_size * D)[row] = scale;
        }
    }

    // ---- queries ----
    at -= 2 * kv_items;
    if (at >= q_items) return;
    float c[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        c[j] = (float)cos_of(j);
        s[j] = (float)sin_of(j);
    }
    O* out = static_cast<O*>(p.out) + token * p.out_tok;
    for (; at < q_items; at += U * p.parts) {
        Pairs<T, ADJ> x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (at + u * p.parts < q_items) load(2, head_of(at + u * p.parts, p.heads), x[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int head = (at + u * p.parts) * VPW + lane / TPV;
            if (head >= p.heads) continue;
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = x[u].get(j);
            if (turn) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float &a = ADJ ? v[2 * j] : v[j], &b = ADJ ? v[2 * j + 1] : v[4 + j];
                    const float fa = a, fb = b;
                    a = fa * c[j] - fb * s[j];
                    b = fb * c[j] + fa * s[j];
                }
            }
            O* dst = out + head * p.out_head;
            const uint4 w = make_uint4(kv_round2<O>(v[0], v[1]), kv_round2<O>(v[2], v[3]), kv_round2<O>(v[4], v[5]), kv_round2<O>(v[6], v[7]));
            if (ADJ) {
                *reinterpret_cast<uint4*>(dst + col_a) = w;
            } else {
                *reinterpret_cast<uint2*>(dst + col_a) = make_uint2(w.x, w.y);
                *reinterpret_cast<uint2*>(dst + col_b) = make_uint2(w.z, w.w);
            }
        }
    }
}

template <typename T, typename O, int FMT, int D>
cudaError_t launch(RotaryParams p, bool adjacent, cudaStream_t st)
{
    constexpr int VPW = 256 / D;
    const int all = (p.heads + VPW - 1) / VPW + 2 * ((p.l.kv_heads + VPW - 1) / VPW);
    // few tokens: a token's vectors over as many warps as fill the GPU.  Each computes the token's angles, some 300
    // instructions, so no more: 8000 tokens x (28 + 2 x 4) x 128 take 34 us with one warp each, 36 with two, 47 with five
    p.parts = (int)std::max(1LL, std::min<long long>(all, (148LL * 4 * kRotWarps + p.n - 1) / p.n));
    const dim3 grid((unsigned)((p.n + kRotWarps - 1LL) / kRotWarps), (unsigned)p.parts);
    return adjacent ? kv_launch(kv_append_rotary_kernel<T, O, FMT, D, true>, grid, kRotThreads, 0, st, p)
                    : kv_launch(kv_append_rotary_kernel<T, O, FMT, D, false>, grid, kRotThreads, 0, st, p);
}

// q_out on what other warps read, or two of its rows on one another: q itself alone may be where it is
bool out_in_the_way(const b4_kv_cache* cache, const KvLayout& l, const b4_rotary* r, const b4_kv_rows* x)
{
    const long long n = x->n_tokens, item = x->dtype == B4_DTYPE_F32 ? 4 : 2, d = l.head_dim;
    const RowSet out = row_set(x->q_out, 2, x->out_stride_token, x->out_stride_head, n, x->heads, d);
    const bool in_place = x->q_out == x->q && item == 2 && (n == 1 || x->out_stride_token == x->q_stride_token) &&
                          (x->heads == 1 || x->out_stride_head == x->q_stride_head);
    return rows_overlap(out) || (!in_place && rows_meet(out, row_set(x->q, item, x->q_stride_token, x->q_stride_head, n, x->heads, d))) ||
           rows_meet(out, row_set(x->k, item, x->k_stride_token, x->k_stride_head, n, l.kv_heads, d)) ||
           rows_meet(out, row_set(x->v, item, x->v_stride_token, x->v_stride_head, n, l.kv_heads, d)) ||
           rows_meet(out, row_set(x->positions, 4, x->position_stride, 0, r->axes ? r->n_axes : 1, 1, n)) ||
           rows_meet(out, row_set(x->slots, 4, n)) || rows_meet(out, row_set(r->turns, 8, r->dim / 2)) ||
           (r->axes && rows_meet(out, row_set(r->axes, 1, r->dim / 2))) || rows_meet(out, row_set(cache->blocks, l.block, (long long)l.n_pages * l.kv_heads));
}

template <typename T, typename O>
cudaError_t launch(const RotaryParams& p, bool adjacent, cudaStream_t st)
{
    if (p.l.fmt == B4_KV_INT4) return p.l.head_dim == 64 ? launch<T, O, B4_KV_INT4, 64>(p, adjacent, st) : launch<T, O, B4_KV_INT4, 128>(p, adjacent, st);
    return p.l.head_dim == 64 ? launch<T, O, B4_KV_NF4, 64>(p, adjacent, st) : launch<T, O, B4_KV_NF4, 128>(p, adjacent, st);
}

}  // namespace
}  // namespace b4

using namespace b4;

extern "C" {

int b4_rotary_turns(const double* inv_freq, int n, uint64_t* turns)
{
    if (n < 0 || (n > 0 && (!inv_freq || !turns))) return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i)
        if (!std::isfinite(inv_freq[i])) return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i) {
        const double f = std::fabs(inv_freq[i] / 6.283185307179586476925287), part = f - std::floor(f);
        // 64 bits of the quotient's part: the upper 32, then what they leave, rounded; all but the quotient is exact
        const double hi = std::floor(part * 0x1p32), lo = std::nearbyint((part * 0x1p32 - hi) * 0x1p32);
        const uint64_t t = ((uint64_t)hi << 32) + (uint64_t)lo;
        turns[i] = inv_freq[i] < 0.0 ? 0 - t : t;
    }
    return cudaSuccess;
}

int b4_kv_append_rotary(const b4_kv_cache* cache, const b4_rotary* r, const b4_kv_rows* x, b4_stream_t stream)
{
    RotaryParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (!r || !x || x->n_tokens < 0 || x->heads < 0 || x->heads > 65536) return cudaErrorInvalidValue;
    if (r->dim < 16 || r->dim % 16 || r->dim > cache->head_dim || r->n_axes < 1 || r->n_axes > 256 || (r->flags & ~B4_ROTARY_ADJACENT) ||
        !std::isfinite(r->scale))
        return cudaErrorInvalidValue;
    if (x->dtype < B4_DTYPE_F16 || x->dtype > B4_DTYPE_F32) return cudaErrorInvalidValue;
    if (x->out_dtype != B4_DTYPE_F16 && x->out_dtype != B4_DTYPE_BF16) return cudaErrorInvalidValue;
    if (x->dtype != B4_DTYPE_F32 && x->dtype != x->out_dtype) return cudaErrorInvalidValue;
    if (x->n_tokens == 0) return cudaSuccess;
    const unsigned item = x->dtype == B4_DTYPE_F32 ? 4 : 2;
    if (!x->k || !x->v || !x->slots || !x->positions || !r->turns || (x->heads > 0 && (!x->q || !x->q_out))) return cudaErrorInvalidValue;
    if (!kv_aligned(x->k, item) || !kv_aligned(x->v, item) || !kv_aligned(x->slots, 4) || !kv_aligned(x->positions, 4) || !kv_aligned(r->turns, 8))
        return cudaErrorInvalidValue;
    if (x->heads > 0 && (!kv_aligned(x->q, item) || !kv_aligned(x->q_out, 16) || (x->out_stride_token | x->out_stride_head) % 8 != 0))
        return cudaErrorInvalidValue;
    if (r->n_axes > 1 && (!r->axes || x->position_stride < x->n_tokens)) return cudaErrorInvalidValue;
    if (x->heads > 0 && out_in_the_way(cache, p.l, r, x)) return cudaErrorInvalidValue;
    p.blocks = static_cast<uint8_t*>(cache->blocks);
    p.src[0] = x->k;
    p.src[1] = x->v;
    p.src[2] = x->q;
    p.tok[0] = x->k_stride_token;
    p.tok[1] = x->v_stride_token;
    p.tok[2] = x->q_stride_token;
    p.head[0] = x->k_stride_head;
    p.head[1] = x->v_stride_head;
    p.head[2] = x->q_stride_head;
    p.out = x->q_out;
    p.out_tok = x->out_stride_token;
    p.out_head = x->out_stride_head;
    p.positions = x->positions;
    p.slots = x->slots;
    p.axis_stride = x->position_stride;
    p.turns = r->turns;
    p.axes = r->axes;
    p.n = x->n_tokens;
    p.heads = x->heads;
    p.half = r->dim / 2;
    p.n_axes = r->n_axes;
    p.scale = r->scale;
    long long strides = p.tok[0] | p.head[0] | p.tok[1] | p.head[1];
    p.vec = kv_aligned(x->k, 16) && kv_aligned(x->v, 16);
    if (x->heads > 0) {
        strides |= p.tok[2] | p.head[2];
        p.vec = p.vec && kv_aligned(x->q, 16);
    }
    p.vec = p.vec && strides * (long long)item % 16 == 0;
    const bool adjacent = r->flags & B4_ROTARY_ADJACENT;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x->dtype == B4_DTYPE_F16) return launch<__half, __half>(p, adjacent, st);
    if (x->dtype == B4_DTYPE_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(p, adjacent, st);
    return x->out_dtype == B4_DTYPE_F16 ? launch<float, __half>(p, adjacent, st) : launch<float, __nv_bfloat16>(p, adjacent, st);
}

}  // extern "C"
