// b4_kv_attn_warp.cuh -- attention over the 4-bit cache for few queries a request
// (single tokens, drafted tokens): the cache is read once, at its 4 bits, and
// turned into matrix operands in registers.
//
// Mathematics.  The queries that share a kv head (query tokens x heads of the
// group) are the columns of a tile of 8 * NT.  Per 16 tokens:
//   S^T [16 tokens x 8 NT] = K [16 x D] Q^T,   O^T [D x 8 NT] += V^T [D x 16] P^T
// with the codes as the left operand of m16n8k16 in both products, so the tile's
// 8-wide side is the queries and none of it is padding for groups of 8.  A token's
// scale does not depend on the column, so the key's scale multiplies S and the
// value's scale P, in fp32; the operands hold the bare levels (INT4: exact
// integers; NF4: with bf16 queries rounded to fp16 (kNf4Even), which with bf16's own
// rounding, 1.7e-3 of an output's norm, makes 1.02 to 1.14 times as much; with fp16
// queries fp16 high and low parts in two products, since there keys rounded once put
// outputs 3.5e-4 to 6.1e-4 off, where their own rounding is 2.1e-4).
// Softmax's maximum and sum run along the tokens, in fp32, private to a warp;
// the maximum moves only when a score passes it by 2^8, which the weights'
// range allows.  P times the value scale goes to fp16 (its rounding is of the size of
// an fp16 output's own: outputs are 2.2e-4 to 3.1e-4 off, 2.1e-4 without it,
// a row that one token outweighs up to 5e-4), relative to that maximum and to a running
// power of two that bounds the value scales (kLift): a token whose value scale is 2^20 below the largest
// one keeps its 11 bits if its weight is the largest, so only what hardly counts loses bits.
//
// Split.  The (request, kv head, column tile, 32-token chunk) units of the whole
// call form one sequence; every CTA gets an equal run of it, every warp of a CTA
// an equal run of the CTA's, whatever the requests' lengths.  A segment (request,
// head, tile) inside one warp's run is written by the warp; others leave a piece
// (sum, maximum, unnormalised output) that the CTA joins in unit order, and
// segments that cross CTAs are joined by the last CTA to arrive, again in unit
// order: the same bits every time, one launch, no wait between CTAs.
//
// Feed.  Each warp brings its own chunks into its own ring of shared memory with
// 16-byte asynchronous copies, two or three chunks ahead, and reads page ids 32 at a
// time, so a warp waits for nothing but its own data.  (Bulk copies measured slower
// here: a warp that issues one spends some 35 instructions on it, and half a page
// of 64 takes four.)
//
// What bounds it.  INT4: the loop runs at 5.3 TB/s; around it a launch spends 5 us up to
// its first products (lengths, units, page ids, queries: four loads that wait for one
// another) and 6 to 9 on the joins.  NF4: the lookups, a shared load of 32 bits a byte of
// codes, of 64 with two parts (LSU 62 and 69 % busy).  Measured: 32 requests x 8192
// tokens, 64 heads over 8 x 128, INT4: 69 us, 4.03 TB/s over all; one request of 131071,
// NF4 in fp16: 64 us, 2.2 TB/s; 96 of 1 to 6000, 32 heads over 8 x 64, NF4 in bf16:
// 59 us, 2.8 TB/s; 24 x 5 drafts behind 2500 to 5500, 28 heads over 4 x 128, INT4: 68 us;
// one of 777, INT4: 11.8 us.
#pragma once

#include <type_traits>

#include "b4_kv_attn.cuh"

namespace b4 {

// What a segment (a request's head and column tile) costs a warp beside its chunks, in a chunk's time: 96 requests of 1 to
// 6000 tokens take 78 us without it, 69 with 1, 68 with 2 and with 4.
constexpr int kSegChunks = 2;

// PT: tokens of a page in shared memory, 16 or 32 (half a page of 64 lies there as a page of 32)
template <int FMT, int D, int NT, int PT>
struct WarpCfg {
    static constexpr int kWarps = NT == 1 ? 16 : 12;                   // 128 and 168 registers a thread
    static constexpr int kThreads = 32 * kWarps, kScan = 256;          // kScan threads add up the requests
    static constexpr int kRow = D / 2;                                 // bytes of a token's codes
    static constexpr int kScale = FMT == B4_KV_INT4 ? 2 : 4;
    static constexpr int kStage = 2 * kChunk * (kRow + kScale);
    static constexpr int kStages = FMT == B4_KV_NF4 ? (D == 128 ? 2 : 3) : D == 128 && NT == 1 ? 3 : 4;
    static constexpr int kPages = kChunk / PT, kBlock = 2 * PT * (kRow + kScale);
    static constexpr int kCols = 8 * NT;
    static constexpr int kPiece = kCols * (D + 2);                     // floats: output, maxima, sums
    static constexpr int kRing = kStages * kStage;                     // of one warp
    // NF4: 256 rows of 32 copies of 8 bytes at shared address 65536, so that one byte permutation makes a lookup's
    // address; the first warps' rings lie below it
    static constexpr int kTable = 65536, kBelow = FMT == B4_KV_NF4 ? (NT == 1 ? 6 : 5) : kWarps;
    static constexpr int kSmem = FMT == B4_KV_NF4 ? 2 * kTable + (kWarps - kBelow) * kRing : kWarps * kRing;
    static_assert(kRing >= kPiece * 4, "a warp's last piece goes into its ring");
    static_assert(FMT != B4_KV_NF4 || kBelow * kRing <= kTable - 8192 - 4096 * NT, "below the table: 1 KB of the system, the static part");
};

struct WarpPiece {
    long long s0, s1;          // the segment's units of chunks (kSegChunks more follow, with nothing to do)
    int q0, n, head, tile;
    int valid;
};

struct WarpWs {                // the workspace: counters, then pieces that other warps or CTAs read
    int* count;
    float* first;              // [grid][warps] a warp's first piece
    float* cross;              // [grid][2] a CTA's part of a segment that began before it / goes on after it
};

template <typename T, int FMT, int D, int NT, int PT>
__global__ void __launch_bounds__(WarpCfg<FMT, D, NT, PT>::kThreads, 1) kv_attn_warp_kernel(const AttnParams p, const WarpWs ws)
{
    using C = WarpCfg<FMT, D, NT, PT>;
    constexpr int kWarps = C::kWarps, kThreads = C::kThreads, kStages = C::kStages, kScan = C::kScan;
    constexpr bool kLow = std::is_same<T, __half>::value;          // NF4 levels in two parts
    constexpr float kUp = kLow ? kNf4Least : kNf4Even;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    __shared__ WarpPiece pieces[kWarps][2];
    __shared__ long long scan[kScan + 1], warp_sum[kWarps];
    __shared__ int4 cached[kScan];
    __shared__ float2 joined[C::kCols][32];
    __shared__ float factor[C::kCols][32];
    __shared__ int last_cta[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const b4_kv_attn& a = p.a;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(attn_smem);
    auto ring_of = [&](int w) { return attn_smem + (w < C::kBelow ? w * C::kRing : 2 * C::kTable - smem_at + (w - C::kBelow) * C::kRing); };
    if (tid < 2 * kWarps) pieces[tid >> 1][tid & 1].valid = 0;
    if (FMT == B4_KV_NF4) {
        // row b: 32 copies of (high, low) of byte b's two levels, the two swapped in the upper 16 copies: there the
        // high parts alone (keys) lie in the odd banks, and the two products of the values add up to the same
        for (int i = tid; i < 256 * 16; i += kThreads) {
            const uint32_t b = i >> 4, hi = nf4_pair(b, kUp), lo = nf4_pair_low(b, kUp);
            reinterpret_cast<uint4*>(attn_smem + C::kTable - smem_at)[i] = (i & 15) < 8 ? make_uint4(hi, lo, hi, lo) : make_uint4(lo, hi, lo, hi);
        }
    }
    kv_begin();

    // ---- the call's units, and each warp's run of them ----
    auto tiles_of = [&](const AttnReq& q) { return q.n * p.group <= p.rows_upto ? (q.n * p.group + C::kCols - 1) / C::kCols : 0; };
    auto units_of = [&](const AttnReq& q) { return (long long)p.l.kv_heads * tiles_of(q) * (q.chunks + kSegChunks); };
    const int per = (a.n_req + kScan - 1) / kScan;
    {
        long long sum = 0;
        if (tid < kScan) {
            for (int i = 0; i < per; ++i) {
                const int r = tid * per + i;
                if (r >= a.n_req) break;
                const AttnReq q = attn_request(p, r);
                if (per == 1) cached[r] = make_int4(q.q0, q.n, q.ctx, 0);
                sum += units_of(q);
            }
        }
        long long inc = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        long long base = 0;
#pragma unroll
        for (int w = 0; w < kScan / 32; ++w)
            if (w < warp) base += warp_sum[w];
        if (tid < kScan) scan[tid + 1] = base + inc;
        if (tid == 0) scan[0] = 0;
        __syncthreads();
    }
    auto request = [&](int r) {                // from shared memory where all fit there
        if (per > 1) return attn_request(p, r);
        const int4 x = cached[r];
        return attn_extent(p, x.x, x.y, x.z);
    };
    const long long total = scan[kScan];
    if (total == 0) return;
    // Equal runs; few units: one a warp, so that fewer pieces cross CTAs.  Where a CTA's run is short, a segment's end
    // nearby is worth more than equal runs (a join across CTAs costs some 2 us, a unit more a warp less): the run's ends
    // move to it.
    const int ctas = (int)min((long long)gridDim.x, (total + kWarps - 1) / kWarps);
    const int cta = blockIdx.x;
    if (cta >= ctas) return;
    const long long share = div64(total, ctas), rest = total - share * ctas;
    const int near = share <= 2 * kWarps ? kWarps : 0;
    auto owner = [&](long long u) {            // the CTA that the unit is in before any end moves
        return (int)(u < rest * (share + 1) ? div64(u, share + 1) : rest + div64(u - rest * (share + 1), share));
    };
    // the request that unit u is in, and that request's first unit
    auto find = [&](long long u, long long& at) {
        constexpr int kPer = kScan / 32;
        unsigned m = __ballot_sync(0xffffffffu, scan[lane * kPer] <= u);
        const int block = 31 - __clz(m);
        m = __ballot_sync(0xffffffffu, lane < kPer && scan[block * kPer + lane] <= u);
        const int i = block * kPer + 31 - __clz(m);
        int r = i * per;
        at = scan[i];
        for (; r < a.n_req - 1; ++r) {
            const long long n = units_of(request(r));
            if (u < at + n) break;
            at += n;
        }
        return r;
    };
    auto end_of = [&](int c) -> long long {    // where CTA c's run begins
        const long long u = c * share + min((long long)c, rest);
        if (near == 0 || u <= 0 || u >= total) return u;
        long long at;
        const int units = request(find(u, at)).chunks + kSegChunks;
        const long long s0 = at + div64(u - at, units) * units;
        return u - s0 <= near ? s0 : s0 + units - u <= near ? s0 + units : u;
    };
    const long long c0 = end_of(cta), c1 = end_of(cta + 1);
    auto run_start = [&](int w) {
        const int n = (int)(c1 - c0);
        return c0 + w * (n / kWarps) + min(w, n % kWarps);
    };

    if (const long long v0 = run_start(warp), v1 = run_start(warp + 1); v0 < v1) {
        // ---- a warp's run ----
        const int g = lane >> 2, t = lane & 3;
        uint8_t* ring = ring_of(warp);
        constexpr int W = D / 32;              // packed words of a token's codes that a lane of the key operand holds
        constexpr int VW = D / 64;             // ... of the value operand
        // this lane's places in a stage: its key and value rows of the chunk's two 16-token tiles, its token's scales.
        // Row g of a tile's eight is token gr: the pairs 2, 3 and 6, 7 are swapped, so that the four lanes t of a value
        // read (tokens gr(2t)) see rows of both parities and with them all banks
        const int gr = g ^ (g >> 1 & 1);
        const int k_at = gr * C::kRow + t * (W * 4), v_at = PT * C::kRow + (2 * t + (t & 1)) * C::kRow + g * (VW * 4);
        constexpr int tile1 = PT == 16 ? C::kBlock : 16 * C::kRow;
        const int v_other = t & 1 ? -C::kRow : C::kRow;
        const int s_at = lane / PT * C::kBlock + PT * D + lane % PT * C::kScale;
        const uint32_t t_key = C::kTable + lane * 8 + (lane >> 4) * 4, t_val = C::kTable + lane * 8;

        float o[NT][D / 16][4];                // m-tile mt: columns 2t, 2t + 1 of d = g * (D / 8) + 2 mt, and of d + 1
        float mx[NT][2], sum[NT][2], qf[NT][2];
        uint32_t qb[NT][D / 8];
        int lim[NT][2];                        // keys that a column sees: below lim, at or above lim - window
        int vexp;
        struct { int q0, n, ctx, head, tile, token; } u = {};   // the segment; a chunk's first token

        auto col_row = [&](int col, int& token, int& head) -> bool {
            const int c = u.tile * C::kCols + col;
            token = c / p.group;
            head = u.head * p.group + (c - token * p.group);
            return c < u.n * p.group;
        };
        // a segment's queries as the right operand, in the order of the decoded codes.  A negative factor of the scores
        // goes into the queries, so that a larger product is a larger score.
        auto load_queries = [&](int nt, uint4 (&v)[W]) {
            int token, head;
            const bool in = col_row(nt * 8 + g, token, head);
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (u.q0 + token) * a.q_stride_token +
                                                              head * a.q_stride_head + t * (D / 4));
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = in ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
        };
        auto begin_segment = [&](uint4 (&queries)[NT][W]) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                int token, head;
                uint4(&v)[W] = queries[nt];
                const float factor = query_operand<T, W>(v, a.scale < 0.0f);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const uint4 x = FMT == B4_KV_INT4 ? int4_pair_order(v[i]) : v[i];
                    qb[nt][4 * i] = x.x;
                    qb[nt][4 * i + 1] = x.y;
                    qb[nt][4 * i + 2] = x.z;
                    qb[nt][4 * i + 3] = x.w;
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    // not 0, so that a masked score's -infinity stays one
                    qf[nt][j] = fmaxf(__shfl_sync(0xffffffffu, factor, (2 * t + j) * 4) * (fabsf(a.scale) * kLog2e) *
                                          (FMT == B4_KV_NF4 ? 1.0f / kUp : 1.0f), 1e-30f);
                    col_row(nt * 8 + 2 * t + j, token, head);
                    lim[nt][j] = a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + token + 1);
                    mx[nt][j] = kNoMax;
                    sum[nt][j] = 0.0f;
                }
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][mt][j] = 0.0f;
            }
            vexp = kNoExp;
        };

        // 32 tokens; `masked` where some column does not see all of them
        auto compute = [&](const uint8_t* buf, int there, bool masked) {
            // the token of this lane: its scales
            const uint8_t* sp = buf + s_at;
            const float ks = FMT == B4_KV_INT4 ? __half2float(*reinterpret_cast<const __half*>(sp)) : *reinterpret_cast<const float*>(sp);
            float vs = FMT == B4_KV_INT4 ? __half2float(*reinterpret_cast<const __half*>(sp + PT * C::kScale))
                                         : *reinterpret_cast<const float*>(sp + PT * C::kScale);
            float s[2][NT][4];
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const uint8_t* kp = buf + k_at + st * tile1;
                uint32_t k0[W], k1[W];
                if (D == 128) {
                    const uint4 x = *reinterpret_cast<const uint4*>(kp), y = *reinterpret_cast<const uint4*>(kp + 8 * C::kRow);
                    k0[0] = x.x; k0[1] = x.y; k0[W - 2] = x.z; k0[W - 1] = x.w;
                    k1[0] = y.x; k1[1] = y.y; k1[W - 2] = y.z; k1[W - 1] = y.w;
                } else {
                    const uint2 x = *reinterpret_cast<const uint2*>(kp), y = *reinterpret_cast<const uint2*>(kp + 8 * C::kRow);
                    k0[0] = x.x; k0[1] = x.y;
                    k1[0] = y.x; k1[1] = y.y;
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[st][nt][j] = 0.0f;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    uint32_t x[4], y[4];
                    if (FMT == B4_KV_INT4) {
                        int4_word_to_half2(k0[i], x);
                        int4_word_to_half2(k1[i], y);
                    } else if (kLow) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            uint2 e[2], f[2];
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                e[b] = lds64(__byte_perm(k0[i], t_val, 0x7604 | (2 * c + b) << 4));
                                f[b] = lds64(__byte_perm(k1[i], t_val, 0x7604 | (2 * c + b) << 4));
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_f16(s[st][nt], e[0].x, f[0].x, e[1].x, f[1].x, qb[nt][4 * i + 2 * c], qb[nt][4 * i + 2 * c + 1]);
                                mma_f16(s[st][nt], e[0].y, f[0].y, e[1].y, f[1].y, qb[nt][4 * i + 2 * c], qb[nt][4 * i + 2 * c + 1]);
                            }
                        }
                        continue;
                    } else {
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            x[b] = lds32(__byte_perm(k0[i], t_key, 0x7604 | b << 4));
                            y[b] = lds32(__byte_perm(k1[i], t_key, 0x7604 | b << 4));
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_f16(s[st][nt], x[0], y[0], x[1], y[1], qb[nt][4 * i], qb[nt][4 * i + 1]);
                        mma_f16(s[st][nt], x[2], y[2], x[3], y[3], qb[nt][4 * i + 2], qb[nt][4 * i + 3]);
                    }
                }
            }
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float k = __shfl_sync(0xffffffffu, ks, 16 * st + 8 * h + gr);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 2 * h; j < 2 * h + 2; ++j) s[st][nt][j] *= k;
                }
            if (masked) {
                const int key = u.token + lane;
                const int end = a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + 1 + (u.tile * C::kCols + C::kCols - 1) / p.group);
                const int begin = a.window > 0 ? u.ctx - u.n + 1 + u.tile * C::kCols / p.group - a.window : 0;
                const bool in = (there >> lane / PT & 1) && key < end && key >= begin;     // some column sees it
                const unsigned some = __ballot_sync(0xffffffffu, in);
                if (!in) vs = 0.0f;
#pragma unroll
                for (int st = 0; st < 2; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int x = 16 * st + gr + 8 * (j >> 1), at = u.token + x;
                            if (!(some >> x & 1) || at >= lim[nt][j & 1] || (a.window > 0 && at < lim[nt][j & 1] - a.window))
                                s[st][nt][j] = -INFINITY;
                        }
            }
            float top[NT][2];
            bool moved = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    top[nt][j] = fmaxf(fmaxf(s[0][nt][j], s[0][nt][j + 2]), fmaxf(s[1][nt][j], s[1][nt][j + 2]));
                    moved |= top[nt][j] * qf[nt][j] > mx[nt][j] + 8.0f;
                }
            const unsigned vbits = __reduce_max_sync(0xffffffffu, vs < 3.4028235e38f ? __float_as_uint(fabsf(vs)) : 0u);
            const int ve = max(vexp, (int)(vbits >> 23) - 126);
            if (__any_sync(0xffffffffu, moved) || ve != vexp) {
                const float vkeep = pow2(max(vexp - ve, -126));
                vexp = ve;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float keep[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], off));
                        const float next = top[nt][j] == -INFINITY ? mx[nt][j] : fmaxf(mx[nt][j], top[nt][j] * qf[nt][j]);
                        keep[j] = fast_exp2(mx[nt][j] - next);
                        mx[nt][j] = next;
                        sum[nt][j] *= keep[j];
                        keep[j] *= vkeep;
                    }
#pragma unroll
                    for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[nt][mt][j] *= keep[j & 1];
                }
            }
            vs = fminf(vs * pow2(kLift - vexp), 3.4028235e38f);   // finite, so that a weight of 0 makes 0 of it
            // weights as the right operand: tokens along k, a query a lane's row
            uint32_t pb[2][NT][2];
#pragma unroll
            for (int st = 0; st < 2; ++st)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float v = __shfl_sync(0xffffffffu, vs, 16 * st + 8 * h + gr);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float w[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            w[j] = fast_exp2(fmaf(s[st][nt][2 * h + j], qf[nt][j], -mx[nt][j]));
                            sum[nt][j] += w[j];
                        }
                        pb[st][nt][h] = movmatrix(pack_half2(w[0] * v, w[1] * v));
                    }
                }
            // values: lane (g, t) holds d = g * (D / 8) .. of the tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                const uint8_t* vp = buf + v_at + st * tile1;
                uint32_t v[4][VW];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint8_t* x = vp + (j & 1 ? v_other : 0) + (j >> 1) * 8 * C::kRow;
                    if (VW == 2) {
                        const uint2 y = *reinterpret_cast<const uint2*>(x);
                        v[j][0] = y.x;
                        v[j][VW - 1] = y.y;
                    } else {
                        v[j][0] = *reinterpret_cast<const uint32_t*>(x);
                    }
                }
#pragma unroll
                for (int i = 0; i < VW; ++i) {
                    if (FMT == B4_KV_INT4) {
                        // halves: two bytes of the first token, the same two of the second: four columns' pairs
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            uint32_t e[4], f[4];
                            int4_word_to_half2(__byte_perm(v[0][i], v[1][i], b ? 0x7632 : 0x5410), e);
                            int4_word_to_half2(__byte_perm(v[2][i], v[3][i], b ? 0x7632 : 0x5410), f);
#pragma unroll
                            for (int c = 0; c < 2; ++c)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
                                    mma_f16(o[nt][4 * i + 2 * b + c], e[2 * c], e[2 * c + 1], f[2 * c], f[2 * c + 1], pb[st][nt][0], pb[st][nt][1]);
                        }
                    } else {
                        uint32_t e[2], f[2];                       // bytes of (first token, second token), even and odd columns
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t x = v[2 * j][i], y = v[2 * j + 1][i];
                            e[j] = (x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u);
                            f[j] = (x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u);
                        }
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            uint2 lo[2], hi[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                if (kLow) {
                                    lo[j] = lds64(__byte_perm(e[j], t_val, 0x7604 | b << 4));
                                    hi[j] = lds64(__byte_perm(f[j], t_val, 0x7604 | b << 4));
                                } else {
                                    lo[j].x = lds32(__byte_perm(e[j], t_key, 0x7604 | b << 4));
                                    hi[j].x = lds32(__byte_perm(f[j], t_key, 0x7604 | b << 4));
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                mma_f16(o[nt][4 * i + b], lo[0].x, hi[0].x, lo[1].x, hi[1].x, pb[st][nt][0], pb[st][nt][1]);
                                if (kLow) mma_f16(o[nt][4 * i + b], lo[0].y, hi[0].y, lo[1].y, hi[1].y, pb[st][nt][0], pb[st][nt][1]);
                            }
                        }
                    }
                }
            }
        };

        // ---- the run's segments ----
        int r, stage = 0, feed = 0;
        const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
        const int n16 = PT * C::kScale / 16, scale_at = lane < n16 ? lane * 16 : (p.l.page_size - PT) * C::kScale + lane * 16;
        long long v = v0, at;                  // the next unit; the request's first
        r = find(v0, at);
        while (v < v1 && r < a.n_req) {
            const AttnReq q = request(r);
            const long long units = units_of(q);
            if (v >= at + units) {
                at += units;
                ++r;
                continue;
            }
            const int tiles = tiles_of(q), seg = (int)div64(v - at, q.chunks + kSegChunks);
            const long long seg_unit = at + (long long)seg * (q.chunks + kSegChunks), seg_end = min(seg_unit + q.chunks + kSegChunks, v1);
            const int first = (int)(v - seg_unit);
            if (first >= q.chunks) {               // only of its end
                v = seg_end;
                continue;
            }
            const int last = (int)min((long long)q.chunks, first + (v1 - v));
            u.q0 = q.q0;
            u.n = q.n;
            u.ctx = q.ctx;
            u.head = seg / tiles;
            u.tile = seg - u.head * tiles;
            v = last == q.chunks ? seg_end : v1;

            // the feed: page ids by 32, `ids` from page `base` on and the 32 after those
            const int32_t* row = a.tables + (long long)r * a.table_stride;
            const uint8_t* blocks = p.blocks + u.head * p.l.block;
            const long long page_bytes = p.l.kv_heads * p.l.block;
            int base = (q.chunk0 + first) * kChunk >> p.l.page_shift, next = q.chunk0 + first, queue = 0;
            auto load_ids = [&](int page) { return page < a.table_width && (long long)page << p.l.page_shift < q.ctx ? __ldg(row + page) : -1; };
            int ids = load_ids(base + lane), more = load_ids(base + 32 + lane);
            auto issue = [&]() {               // the next chunk, if any, into stage `feed`
                int there = 0;
                if (next < q.chunk0 + last) {
                    const int page = next * kChunk >> p.l.page_shift;
                    if (page - base >= 32) {
                        ids = more;
                        base += 32;
                        more = load_ids(base + 32 + lane);
                    }
                    const int half = PT == 32 ? next * kChunk & (p.l.page_size - 1) : 0;       // of a page of 64
                    const uint32_t dst = ring_at + feed * C::kStage;
#pragma unroll
                    for (int i = 0; i < C::kPages; ++i) {
                        // a chunk of two pages begins at an even place of the 32: its second page is among them
                        const int id = __shfl_sync(0xffffffffu, ids, page - base + i);
                        if ((unsigned)id >= (unsigned)p.l.n_pages) continue;
                        there |= 1 << i;
                        const uint8_t* src = blocks + id * page_bytes;
                        const uint8_t *k = src + half * C::kRow + lane * 16, *v = k + p.l.page_size * C::kRow;
                        constexpr int kCodes = PT * C::kRow, n16 = PT * C::kScale / 16;
#pragma unroll
                        for (int x = 0; x < kCodes; x += 512) {
                            copy_async16(dst + i * C::kBlock + x, k + x);
                            copy_async16(dst + i * C::kBlock + kCodes + x, v + x);
                        }
                        if (lane < 2 * n16) copy_async16(dst + i * C::kBlock + 2 * kCodes, src + p.l.page_size * D + half * C::kScale + scale_at);
                    }
                    ++next;
                    if (++feed == kStages) feed = 0;
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
                queue = queue << 2 | there;
            };
            uint4 queries[NT][W];              // asked for before the feed waits for its page ids
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) load_queries(nt, queries[nt]);
#pragma unroll 1
            for (int i = 0; i < kStages; ++i) issue();
            begin_segment(queries);

            // every key of a chunk is seen by every column where the chunk lies in [clear, seen)
            const int seen = a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + 1 + u.tile * C::kCols / p.group);
            const int clear = a.window > 0 ? u.ctx - a.window : 0;
#pragma unroll 1
            for (int c = first; c < last; ++c) {
                u.token = (q.chunk0 + c) * kChunk;
                const int there = queue >> (2 * kStages - 2) & 3;
                asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
                __syncwarp();
                compute(ring + stage * C::kStage, there, u.token < clear || u.token + kChunk > seen || there != (1 << C::kPages) - 1);
                __syncwarp();
                issue();
                if (++stage == kStages) stage = 0;
            }

            // ---- the end of a segment, or of the run ----
            const float vup = pow2(vexp - kLift) * (FMT == B4_KV_NF4 ? 1.0f / kUp : 1.0f);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) sum[nt][j] += __shfl_xor_sync(0xffffffffu, sum[nt][j], off);
            if (first == 0 && last == q.chunks) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        int token, head;
                        if (!col_row(nt * 8 + 2 * t + j, token, head)) continue;
                        const float inv = sum[nt][j] > 0.0f ? vup / sum[nt][j] : 0.0f;
                        T* dst = static_cast<T*>(a.out) + (u.q0 + token) * a.out_stride_token + head * a.out_stride_head + g * (D / 8);
                        uint32_t w[D / 16];
#pragma unroll
                        for (int mt = 0; mt < D / 16; ++mt) {
                            const T lo = kv_round<T>(o[nt][mt][j] * inv), hi = kv_round<T>(o[nt][mt][j + 2] * inv);
                            w[mt] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
                        }
#pragma unroll
                        for (int k = 0; k < D / 64; ++k)
                            reinterpret_cast<uint4*>(dst)[k] = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                        if (a.lse && g == 0)
                            a.lse[(long long)(u.q0 + token) * a.heads + head] =
                                sum[nt][j] > 0.0f ? (mx[nt][j] + fast_log2(sum[nt][j])) * kLn2 : -INFINITY;
                    }
            } else {
                // a piece [column][D], maxima, sums: the run's last goes into the ring, which is free, its first to the workspace
                const bool is_last = v == v1;
                float* dst = is_last ? reinterpret_cast<float*>(ring) : ws.first + ((long long)cta * kWarps + warp) * C::kPiece;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int col = nt * 8 + 2 * t + j;
#pragma unroll
                        for (int mt = 0; mt < D / 16; mt += 2) {
                            float4 x = make_float4(o[nt][mt][j] * vup, o[nt][mt][j + 2] * vup, o[nt][mt + 1][j] * vup, o[nt][mt + 1][j + 2] * vup);
                            *reinterpret_cast<float4*>(dst + col * D + g * (D / 8) + 2 * mt) = x;
                        }
                        if (g == 0) {
                            dst[C::kCols * D + col] = mx[nt][j];
                            dst[C::kCols * (D + 1) + col] = sum[nt][j];
                        }
                    }
                if (lane == 0) {
                    WarpPiece pc;
                    pc.s0 = seg_unit;
                    pc.s1 = seg_unit + q.chunks;
                    pc.q0 = u.q0;
                    pc.n = u.n;
                    pc.head = u.head;
                    pc.tile = u.tile;
                    pc.valid = 1;
                    pieces[warp][is_last] = pc;
                }
            }
        }
    }
    __syncthreads();

    // ---- join the pieces of this CTA, in unit order: lane i looks at piece i (a warp's first at 2 warp, its last after it) ----
    auto piece_of = [&](int i) -> const float* {
        return i & 1 ? reinterpret_cast<const float*>(ring_of(i >> 1)) : ws.first + ((long long)cta * kWarps + (i >> 1)) * C::kPiece;
    };
    const bool mine = lane < 2 * kWarps && pieces[lane >> 1][lane & 1].valid;
    const long long my_s0 = mine ? pieces[lane >> 1][lane & 1].s0 : -1;
    const uint32_t have = __ballot_sync(0xffffffffu, mine);
    // the pieces of this lane's segment, which are neighbours in this order but for lanes without a piece: those count,
    // with nothing, to the segment before them
    const uint32_t my_list = __match_any_sync(0xffffffffu, my_s0);
    const uint32_t upto = have & (0xffffffffu >> (31 - lane));
    const uint32_t its_list = __shfl_sync(0xffffffffu, my_list, upto ? 31 - __clz(upto) : lane);
    const int lead = upto ? __ffs(its_list) - 1 : lane;
    const int tail = mine ? 31 - __clz(my_list) : lane;
    // maxima and sums of every segment (at its first piece) and the pieces' factors, a column a warp
    for (int col = warp; col < C::kCols; col += kWarps) {
        float m = kNoMax, l = 0.0f;
        if (mine) {
            const float* b = piece_of(lane) + C::kCols * D + col;
            m = b[0];
            l = b[C::kCols];
        }
        float top = m;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, top, off);
            if (lane - off >= lead) top = fmaxf(top, y);
        }
        top = __shfl_sync(0xffffffffu, top, tail);
        const float f = mine ? fast_exp2(m - top) : 0.0f;
        float all = f * l;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const float y = __shfl_up_sync(0xffffffffu, all, off);
            if (lane - off >= lead) all += y;
        }
        all = __shfl_sync(0xffffffffu, all, tail);
        if (mine && lane == lead) joined[col][lane] = make_float2(top, all);
        factor[col][lane] = f;
    }
    __syncthreads();
    auto emit = [&](const WarpPiece& pc, int e, float2 x, float m, float l) {      // two columns' outputs of one query
        const int c = pc.tile * C::kCols + e / D, token = c / p.group, head = pc.head * p.group + (c - token * p.group);
        if (c >= pc.n * p.group) return;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        const T w[2] = {kv_round<T>(x.x * inv), kv_round<T>(x.y * inv)};
        *reinterpret_cast<uint32_t*>(static_cast<T*>(a.out) + (pc.q0 + token) * a.out_stride_token + head * a.out_stride_head + e % D) =
            (uint32_t)*reinterpret_cast<const uint16_t*>(w) | (uint32_t)*reinterpret_cast<const uint16_t*>(w + 1) << 16;
        if (a.lse && e % D == 0)
            a.lse[(long long)(pc.q0 + token) * a.heads + head] = l > 0.0f ? (m + fast_log2(l)) * kLn2 : -INFINITY;
    };
    int cross[2] = {-1, -1};                   // the first pieces of the segments that began before this CTA, that go on after it
    // a warp takes 256 outputs of a segment, eight a lane, so that many short segments join side by side
    constexpr int kItems = C::kCols * D / 256;
    static_assert(kItems <= kWarps, "one of a segment's items a warp");
    int turn = warp;                           // of the kWarps items, the next that is this warp's
    for (uint32_t todo = have; todo;) {
        const int at = __ffs(todo) - 1;
        const uint32_t list = __shfl_sync(0xffffffffu, my_list, at), lasts = list & 0xaaaaaaaau, firsts = list & 0x55555555u;
        todo &= ~list;
        const WarpPiece& pc = pieces[at >> 1][at & 1];
        const bool inside = pc.s0 >= c0 && pc.s1 <= c1, begins = pc.s0 >= c0;
        if (!inside) {
            if (begins) cross[1] = at;
            else cross[0] = at;
        }
        const int item = turn;
        turn -= kItems;
        if (turn < 0) turn += kWarps;
        if (item >= kItems) continue;
        const int e0 = item * 256 + lane * 2;
        float2 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = make_float2(0.0f, 0.0f);
        auto add = [&](const float* b, int i, bool in) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int e = e0 + j * 64;
                const float k = in ? factor[e / D][i] : 0.0f;
                const float2 y = *reinterpret_cast<const float2*>(b + e);
                x[j].x += k * y.x;
                x[j].y += k * y.y;
            }
        };
        if (lasts) {
            const int w0 = (__ffs(lasts) - 1) >> 1, w1 = (31 - __clz(lasts)) >> 1;
#pragma unroll 4
            for (int w = w0; w <= w1; ++w) {
                const bool in = lasts >> (2 * w + 1) & 1;
                add(reinterpret_cast<const float*>(ring_of(in ? w : w0)), 2 * w + 1, in);
            }
        }
        if (firsts) add(piece_of(__ffs(firsts) - 1), __ffs(firsts) - 1, true);        // one at most: a run's first piece ends its segment
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = e0 + j * 64, col = e / D;
            const float2 ml = joined[col][at];
            if (inside) {
                emit(pc, e, x[j], ml.x, ml.y);
            } else {
                float* dst = ws.cross + ((long long)cta * 2 + begins) * C::kPiece;
                *reinterpret_cast<float2*>(dst + e) = x[j];
                if (e % D == 0) {
                    dst[C::kCols * D + col] = ml.x;
                    dst[C::kCols * (D + 1) + col] = ml.y;
                }
            }
        }
    }
    if (cross[0] < 0 && cross[1] < 0) return;

    // ---- segments that cross CTAs: the last to arrive joins them, in CTA order ----
    auto span = [&](const WarpPiece& pc, int& f) {         // the CTAs that hold pieces of the segment
        f = owner(min(pc.s0 + near, total - 1));
        return max(owner(max(min(pc.s1, pc.s1 + kSegChunks - near) - 1, 0LL)) - f, 0) + 1;
    };
    __syncthreads();
    if (tid < 2) {
        const int at = tid ? cross[1] : cross[0];
        int last = 0;
        if (at >= 0) {
            int f;
            const int n = span(pieces[at >> 1][at & 1], f);
            last = count_in(ws.count + f) == n - 1;
            if (last) ws.count[f] = 0;
        }
        last_cta[tid] = last;
    }
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < 2; ++k) {
        if (!last_cta[k]) continue;
        const int at = k ? cross[1] : cross[0];
        const WarpPiece& pc = pieces[at >> 1][at & 1];
        int f;
        const int n = span(pc, f);
        auto part = [&](int c) -> const float* { return ws.cross + ((long long)(f + c) * 2 + (c == 0)) * C::kPiece; };
        // every thread adds up its own columns' maxima and sums, so that all loads of eight parts are in flight at once
        for (int e = tid * 2; e < C::kCols * D; e += kThreads * 2) {
            const int col = e / D;
            float m = kNoMax, l = 0.0f;
            float2 x = make_float2(0.0f, 0.0f);
#pragma unroll 8
            for (int c = 0; c < n; ++c) {
                const float* b = part(c);
                const float mc = __ldcg(b + C::kCols * D + col), lc = __ldcg(b + C::kCols * (D + 1) + col);
                const float2 y = __ldcg(reinterpret_cast<const float2*>(b + e));
                const float top = fmaxf(m, mc), keep = fast_exp2(m - top), w = fast_exp2(mc - top);
                l = l * keep + lc * w;
                x = make_float2(x.x * keep + y.x * w, x.y * keep + y.y * w);
                m = top;
            }
            emit(pc, e, x, m, l);
        }
    }
}

}  // namespace b4
