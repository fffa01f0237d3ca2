// b4_kv_select.cu -- boxes around the keys of completed pages, and the choice of the
// pages that a query reads by a bound of its scores over the boxes.
//
// Mathematics.  Over a box [lo, hi] the largest q . k is the sum over columns of
// max(q, 0) hi + min(q, 0) lo; summed over the query heads that share a kv head that is
// linear in their sums of max(q, 0) and of min(q, 0), so a page costs one product of
// 2 * head_dim, whatever the group.  Both sides are 8-bit: the sum of products is a whole
// number below 2 * 128 * 127^2 < 2^24, exact in any order and in fp32, so scores, ties
// and the pages chosen are the same whatever adds them up.  A query's own scale is
// common to its pages and left out.
//
// Select.  16 boxes are the left operand of m16n8k32, up to 8 tokens of a request its
// columns: a box's bytes go from memory into the operand as they lie (the product's
// order of columns is free, so a lane's 16 bytes are its words of two steps).  Scores go
// to shared memory as ordered integers.  The least that is taken is found by histograms
// of their bits, then the lists are written in the context's order by ballots.
//
// Split.  A cluster of CTAs takes a tile of tokens and a kv head; its CTAs share the
// boxes, 16 at a time, and send the scores of token i to CTA i mod the cluster's size,
// which chooses for it.
//
// What bounds it.  A step of single tokens: a chain of waits.  One token behind 9000 in
// pages of 16 (4 kv heads) takes 8.0 us: 0.5 for the lengths, 0.8 for page ids, 1.1 for the
// queries, 1.5 for boxes and their products, 0.6 for the cluster's barriers, 2.6 for the
// choice, 0.5 of it the table again.  Code that runs once costs some 5 cycles an instruction
// here, whatever its kind, so the choice is short loops over shared memory, not unrolled
// registers (a bisection with 16 scores a lane in registers: 450 cycles a bit).  32 tokens
// behind 8 to 32 thousand in pages of 64 (8 kv heads): 13.3 us, of which the 21 MB of boxes
// take 6; one behind 131000 in pages of 16: 21.0 us, 17.8 MB; a chunk of 1024 behind 30000:
// 43.9 us for 8192 choices among 480 boxes, 13 of them the scores, the rest the choices.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "b4_kv.cuh"
#include "b4_kv_overlap.h"

namespace b4 {
namespace {

constexpr int kBoxTail = 16;               // scale and padding

__host__ __device__ inline long long box_bytes(int head_dim) { return 2 * head_dim + kBoxTail; }

// ---- boxes --------------------------------------------------------------------------
struct BoxParams {
    KvLayout l;
    const uint8_t* blocks;
    uint8_t* boxes;
    const int32_t* slots;
    int n, per;                            // tokens, and those that a CTA looks at
};

// int8 code of x in units of s, rounded to even
__device__ __forceinline__ int box_code(float x, float s) { return min(127, max(-127, __float2int_rn(__fdiv_rn(x, s)))); }

// A CTA makes the boxes of the completed pages among its tokens, of one kv head: its warps share a page's tokens, a
// lane holds the extremes of 8 columns over those of its rows (every second token, D = 128; fourth, D = 64).
// Bound by latency: 16 pages of 64 x 8 heads 4.1 us (a warp a page: 10.7); none completed, as in most steps of single tokens,
// 1.1 us.  A CTA looks at 1 to 16 tokens, 8 CTAs an SM before it takes more: 1024 tokens x 8 heads 4.4 us (9.9 with one each),
// 16384 14.9 (137).
constexpr int kBoxWarps = 8;

template <int FMT, int D>
__global__ void __launch_bounds__(32 * kBoxWarps) kv_boxes_kernel(const BoxParams p)
{
    constexpr int TPV = D / 8, ROWS = 32 / TPV, STEP = ROWS * kBoxWarps;
    __shared__ float extreme[kBoxWarps][2][D];
    __shared__ float tops[D / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, sub = lane % TPV, head = blockIdx.y;
    const long long first = (long long)blockIdx.x * p.per;
    const float level = c_nf4_table[lane & 15];
    kv_begin();
    const int slot = lane < p.per && first + lane < p.n ? __ldg(p.slots + first + lane) : -1;
    const int mask = p.l.page_size - 1;
    const bool ends = slot >= 0 && (slot & mask) == mask && slot >> p.l.page_shift < p.l.n_pages;
    for (unsigned todo = __ballot_sync(0xffffffffu, ends); todo; todo &= todo - 1) {       // the same in every warp
        const int page = __shfl_sync(0xffffffffu, slot, __ffs(todo) - 1) >> p.l.page_shift;
        const long long at = (long long)page * p.l.kv_heads + head;
        const uint8_t* block = p.blocks + at * p.l.block;
        const uint8_t* scales = block + p.l.page_size * D;
        float hi[8], lo[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hi[j] = -INFINITY;
            lo[j] = INFINITY;
        }
        uint32_t w[64 / STEP];
        float s[64 / STEP];
#pragma unroll
        for (int i = 0; i < 64 / STEP; ++i) {
            const int token = i * STEP + warp * ROWS + lane / TPV;
            w[i] = 0;
            s[i] = 0.0f;
            if (token > mask) continue;
            w[i] = reinterpret_cast<const uint32_t*>(block)[token * TPV + sub];
            s[i] = FMT == B4_KV_INT4 ? __half2float(reinterpret_cast<const __half*>(scales)[token]) : reinterpret_cast<const float*>(scales)[token];
        }
#pragma unroll
        for (int i = 0; i < 64 / STEP; ++i) {
            const bool in = i * STEP + warp * ROWS + lane / TPV <= mask;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t c = w[i] >> (4 * j) & 15;
                const float v = __fmul_rn(FMT == B4_KV_INT4 ? (float)((int)c - 8) : __shfl_sync(0xffffffffu, level, c), s[i]);
                if (in) {
                    hi[j] = fmaxf(hi[j], v);
                    lo[j] = fminf(lo[j], v);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
#pragma unroll
            for (int o = TPV; o < 32; o <<= 1) {
                hi[j] = fmaxf(hi[j], __shfl_xor_sync(0xffffffffu, hi[j], o));
                lo[j] = fminf(lo[j], __shfl_xor_sync(0xffffffffu, lo[j], o));
            }
            if (lane < TPV) {
                extreme[warp][0][8 * sub + j] = hi[j];
                extreme[warp][1][8 * sub + j] = lo[j];
            }
        }
        __syncthreads();
        float h = -INFINITY, l = INFINITY, top = 0.0f;             // of column tid
        if (tid < D) {
#pragma unroll
            for (int k = 0; k < kBoxWarps; ++k) {
                h = fmaxf(h, extreme[k][0][tid]);
                l = fminf(l, extreme[k][1][tid]);
            }
            if (h < l) h = l = 0.0f;                               // no number in the column
            top = fmaxf(fabsf(h), fabsf(l));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (lane == 0) tops[warp] = top;
        }
        __syncthreads();
        if (tid < D) {
#pragma unroll
            for (int k = 0; k < D / 32; ++k) top = fmaxf(top, tops[k]);
            const float unit = top > 0.0f ? __fmul_rn(top, 1.0f / 127.0f) : 1.0f;
            uint8_t* box = p.boxes + at * box_bytes(D);
            box[tid] = (uint8_t)box_code(h, unit);
            box[D + tid] = (uint8_t)box_code(l, unit);
            if (tid < 4) reinterpret_cast<uint32_t*>(box + 2 * D)[tid] = tid == 0 ? __float_as_uint(unit) : 0u;
        }
    }
}

// ---- select -------------------------------------------------------------------------
struct SelectParams {
    KvLayout l;
    b4_kv_choice c;
    int group, tile, cap;                  // heads of a kv head, tokens of a tile, words of a token's scores
    int lg;                                // a cluster has 2^lg CTAs
    int direct;                            // a tile index is a request's
};

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32, kSelBins = 256;
constexpr int kSelSmem = 200 * 1024;       // of scores

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// past L1, which keeps the table
__device__ __forceinline__ uint4 load_once(const uint4* p)
{
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// larger for larger x; 0 below all of them
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f);                  // -0 as 0
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void store_cluster(uint32_t at, uint32_t rank, uint32_t v)
{
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(v) : "memory");
}

// The codes of C columns of a query's sums above and below 0, from the definition; by whole warps.  Its first 8 heads as loaded.
// In 64 bits, one head after the other: exact for fp16 numbers, whose sums of 64 take 46 bits at most; bf16 numbers may lie
// further apart than any sum holds (two fp32 numbers in its place lost 2^-48 beside 2.5, and with it the side of a border).
template <typename T, int C, typename Raw>
__device__ void exact_codes(const Raw (&raw)[8], const T* src, int group, long long stride, uint32_t (&w)[2])
{
    double sum[2][C];
    float part[2][C], top = 0.0f;
#pragma unroll
    for (int j = 0; j < C; ++j) sum[0][j] = sum[1][j] = 0.0;
    auto add = [&](const Raw& r) {
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const float f = kv_float(reinterpret_cast<const T*>(&r)[j]);
            sum[0][j] += f > 0.0f ? f : 0.0f;
            sum[1][j] += f > 0.0f ? 0.0f : f;                      // NaN too
        }
    };
#pragma unroll
    for (int h = 0; h < 8; ++h)
        if (h < group) add(raw[h]);
    for (int h = 8; h < group; ++h) add(__ldg(reinterpret_cast<const Raw*>(src + h * stride)));
    bool finite = true;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < C; ++j) {
            part[k][j] = __double2float_rn(sum[k][j]);
            finite = finite && fabsf(part[k][j]) < INFINITY;
            top = fmaxf(top, fabsf(part[k][j]));
        }
    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
    finite = __all_sync(0xffffffffu, finite);
    const float unit = top > 0.0f ? __fmul_rn(top, 1.0f / 127.0f) : 1.0f;
    w[0] = w[1] = 0;
    if (!finite) return;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int j = 0; j < C; ++j) w[k] |= (uint32_t)(box_code(part[k][j], unit) & 255) << (8 * j);
}

// What a query sees: its pages, its own the last, and its list's entries and tokens.
struct Seen {
    int pages, entries, tokens;
};

__device__ __forceinline__ Seen seen_of(const SelectParams& p, int ctx, int n, int i)
{
    const int place = ctx - n + i;                                 // ctx >= 0: above -2^31
    const long long room = (long long)p.c.table_width * p.l.page_size;
    const int visible = place < 0 ? 0 : (int)min((long long)place + 1, room);
    Seen s = {0, 0, 0};
    if (visible > 0) {
        s.pages = ((visible - 1) >> p.l.page_shift) + 1;
        s.entries = min(s.pages, p.c.keep);
        s.tokens = (s.entries - 1) * p.l.page_size + visible - (s.pages - 1) * p.l.page_size;
    }
    return s;
}

// NT: eights of tokens in a tile; CTAS: of them on an SM
template <typename T, int D, int NT, int CTAS>
__global__ void __launch_bounds__(kSelThreads, CTAS) kv_select_kernel(const SelectParams p)
{
    constexpr int V = D / 32;                                      // 16-byte words of a box that a lane holds
    constexpr int C = D / 32;                                      // columns of a query that a lane holds
    constexpr int kRow = 2 * D + 64;
    constexpr int kAhead = NT == 1 ? 2 : 1;                        // steps of boxes in flight
    extern __shared__ __align__(16) uint32_t scores[];             // [tokens of this CTA][cap]
    __shared__ __align__(16) uint8_t query[8 * NT * kRow];         // above, below of a token
    __shared__ __align__(16) int bins[kSelWarps][kSelBins];        // of a team's warps together
    __shared__ uint2 range[16 * kSelWarps];                        // [CTAs][warps] least and largest score of the tile's tokens
    __shared__ int2 part[kSelWarps];
    __shared__ int4 found[kSelWarps];
    __shared__ uint32_t tied[kSelWarps][32];
    __shared__ int ties[kSelWarps];

    const b4_kv_choice& a = p.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int cluster = 1 << p.lg, rank = blockIdx.x & (cluster - 1), head = blockIdx.y;
    const int at_tile = blockIdx.x >> p.lg;
    const int stride = kSelWarps << p.lg, step0 = rank + (warp << p.lg);           // of 16 boxes
    kv_begin();

    // ---- the request and its tokens ----
    auto start = [&](int r) { return max(0, min(__ldg(a.q_starts + r), a.total_q)); };
    int r = at_tile, tile0 = 0;
    if (!p.direct) {
        // request r has the tiles from start / tile + r on, as many as it needs at least: the last that begins at or before this
        // one.  Tiles before the first request's, where it does not begin at row 0, have no tokens
        int lo = 0, n = a.n_req;
        while (n > 1) {
            const int step = (n + 31) / 32, probe = lo + lane * step;
            const bool in = lane * step < n && (lane == 0 || start(probe) / (8 * NT) + probe <= at_tile);
            const int last = 31 - __clz(__ballot_sync(0xffffffffu, in));
            n = min(step, n - last * step);
            lo += last * step;
        }
        r = lo;
        tile0 = at_tile - (start(r) / (8 * NT) + r);
    }
    const int32_t* table = a.tables + (long long)r * a.table_stride;
    auto ids_of = [&](int step, int (&id)[2]) {                    // page ids of rows g and g + 8
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int b = a.first + step * 16 + g + 8 * j;
            id[j] = b < a.table_width ? __ldg(table + b) : -1;
        }
    };
    int id[2], next[2];                    // asked for before the request's length is known
    ids_of(step0, id);
    ids_of(step0 + stride, next);
    const int q0 = start(r), n = max(0, start(r + 1) - q0), ctx = max(0, __ldg(a.ctx_len + r));

    for (int i0 = tile0 < 0 ? n : tile0 * p.tile, turn = 0; i0 < n; i0 = p.direct ? i0 + p.tile : n, ++turn) {
        const int nt = min(p.tile, n - i0);
        const Seen most = seen_of(p, ctx, n, i0 + nt - 1);
        const int m = most.pages > a.keep ? most.pages - a.first - a.last : 0;     // pages to score

        if (m > 0) {
            // ---- scores: this CTA's boxes, 16 a warp at a time, two steps of them in flight ----
            const int groups = (m + 15) / 16;
            struct Boxes {
                uint4 word[2][V];
                float unit[2];                                     // NaN: the page is missing
            };
            auto load = [&](const int (&id)[2], Boxes& x) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const bool there = (unsigned)id[j] < (unsigned)p.l.n_pages;
                    const uint8_t* src = static_cast<const uint8_t*>(a.boxes) + ((long long)(there ? id[j] : 0) * p.l.kv_heads + head) * box_bytes(D);
#pragma unroll
                    for (int i = 0; i < V; ++i) x.word[j][i] = load_once(reinterpret_cast<const uint4*>(src + 64 * i) + t);
                    const float unit = __ldg(reinterpret_cast<const float*>(src + 2 * D));
                    x.unit[j] = !there ? __uint_as_float(0x7fffffffu) : unit < INFINITY ? unit : INFINITY;
                }
            };
            // a token a warp (and every 8th): its first 8 heads, asked for before the boxes' page ids are waited for
            using Raw = typename std::conditional<C == 4, uint2, uint32_t>::type;
            auto row_of = [&](int i) {
                return static_cast<const T*>(a.q) + (q0 + i0 + i) * a.q_stride_token + (long long)head * p.group * a.q_stride_head + lane * C;
            };
            auto heads_of = [&](int i, Raw (&raw)[8]) {
                if (i < nt) {
                    const T* src = row_of(i);
#pragma unroll
                    for (int h = 0; h < 8; ++h)
                        if (h < p.group) raw[h] = __ldg(reinterpret_cast<const Raw*>(src + h * a.q_stride_head));
                }
            };
            Raw raw[8];
            heads_of(warp, raw);
            if (turn > 0) {
                ids_of(step0, id);
                ids_of(step0 + stride, next);
            }
            Boxes x[kAhead];
            int at = step0;
            if (at < groups) load(id, x[0]);

            // The sums of the heads' parts above and below 0, as int8: from sums in fp32 where every code is further from its
            // next than those can be off; from exact ones otherwise (5 % of the rows of 8 heads).  Off by 2^-24 of 127 units for
            // each rounding: a sum's, in it and in the largest (1.6e-5 for the two), the exact sums' own, the two units, the
            // reciprocal and the two quotients (7, 5.3e-5)
#pragma unroll 1
            for (int i = warp; i < 8 * NT; i += kSelWarps) {
                if (i > warp) heads_of(i, raw);
                uint32_t w[2] = {0, 0};
                if (i < nt) {
                    float part[2][C], top = 0.0f;
                    bool finite = true;
#pragma unroll
                    for (int j = 0; j < C; ++j) {
                        float v[8];
#pragma unroll
                        for (int h = 0; h < 8; ++h) v[h] = h < p.group ? kv_float(reinterpret_cast<const T*>(&raw[h])[j]) : 0.0f;
                        part[0][j] = ((fmaxf(v[0], 0.0f) + fmaxf(v[1], 0.0f)) + (fmaxf(v[2], 0.0f) + fmaxf(v[3], 0.0f))) +
                                     ((fmaxf(v[4], 0.0f) + fmaxf(v[5], 0.0f)) + (fmaxf(v[6], 0.0f) + fmaxf(v[7], 0.0f)));
                        part[1][j] = ((fminf(v[0], 0.0f) + fminf(v[1], 0.0f)) + (fminf(v[2], 0.0f) + fminf(v[3], 0.0f))) +
                                     ((fminf(v[4], 0.0f) + fminf(v[5], 0.0f)) + (fminf(v[6], 0.0f) + fminf(v[7], 0.0f)));
                        const float sum = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
                        finite = finite && fabsf(sum) < INFINITY;                          // NaN too
                    }
                    const T* src = row_of(i);
#pragma unroll 4
                    for (int h = 8; h < p.group; ++h) {
                        const Raw r = __ldg(reinterpret_cast<const Raw*>(src + h * a.q_stride_head));
#pragma unroll
                        for (int j = 0; j < C; ++j) {
                            const float v = kv_float(reinterpret_cast<const T*>(&r)[j]);
                            part[0][j] += fmaxf(v, 0.0f);
                            part[1][j] += fminf(v, 0.0f);
                            finite = finite && fabsf(v) < INFINITY;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < C; ++j) top = fmaxf(top, fmaxf(part[0][j], -part[1][j]));
                    top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
                    const float inv = __frcp_rn(__fmul_rn(top, 1.0f / 127.0f)), clear = 0.5f - 5.6e-5f - 1.6e-5f * (p.group <= 8 ? 3 : p.group);
                    bool sure = finite && top > 1e-30f && top < 1e30f;
#pragma unroll
                    for (int k = 0; k < 2; ++k)
#pragma unroll
                        for (int j = 0; j < C; ++j) {
                            const float y = part[k][j] * inv, r = y + 12582912.0f;         // 1.5 * 2^23: the integer nearest to y in the low bits
                            sure = sure && fabsf(y - (r - 12582912.0f)) < clear;
                            w[k] |= (__float_as_uint(r) & 255) << (8 * j);
                        }
                    if (!__all_sync(0xffffffffu, sure)) exact_codes<T, C>(raw, src, p.group, a.q_stride_head, w);
                }
                uint8_t* dst = query + i * kRow + lane * C;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (C == 4) *reinterpret_cast<uint32_t*>(dst + k * D) = w[k];
                    else *reinterpret_cast<uint16_t*>(dst + k * D) = (uint16_t)w[k];
                }
            }
            if (kAhead == 2) {
                if (at + stride < groups) load(next, x[kAhead - 1]);
                ids_of(at + 2 * stride, next);
            }
            if (cluster > 1) cluster_sync();                       // the others have begun, or are done with the last tile's scores
            else __syncthreads();

            auto query_of = [&](int nt8, int i) { return *reinterpret_cast<const uint4*>(query + (nt8 * 8 + g) * kRow + 64 * i + 16 * t); };
            const uint32_t scores_at = (uint32_t)__cvta_generic_to_shared(scores);
            uint32_t lo = 0xffffffffu, hi = 0;
            auto score = [&](int step, const Boxes& x) {
                const int b = step * 16 + g;
                // every row is a page with a finite box, but at the list's end and beside pages that are not
                const bool plain = __all_sync(0xffffffffu, step * 16 + 16 <= m && x.unit[0] < INFINITY && x.unit[1] < INFINITY);
#pragma unroll
                for (int nt8 = 0; nt8 < NT; ++nt8) {
                    if (nt8 * 8 >= nt) break;
                    int acc[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const uint4 q = query_of(nt8, i);
                        mma_s8(acc, x.word[0][i].x, x.word[1][i].x, x.word[0][i].y, x.word[1][i].y, q.x, q.y);
                        mma_s8(acc, x.word[0][i].z, x.word[1][i].z, x.word[0][i].w, x.word[1][i].w, q.z, q.w);
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int token = nt8 * 8 + 2 * t + c;
                        if (token >= nt) continue;
                        const uint32_t place = (uint32_t)(token >> p.lg) * p.cap + b;
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            uint32_t key;
                            if (plain) {
                                key = ordered(__fmul_rn((float)acc[2 * r + c], x.unit[r]));
                            } else {
                                if (b + 8 * r >= m) continue;
                                key = x.unit[r] < INFINITY ? ordered(__fmul_rn((float)acc[2 * r + c], x.unit[r])) : x.unit[r] == INFINITY ? ordered(INFINITY) : 0u;
                            }
                            lo = min(lo, key);
                            hi = max(hi, key);
                            if (cluster > 1) store_cluster(scores_at + 4 * (place + 8 * r), token & (cluster - 1), key);
                            else scores[place + 8 * r] = key;
                        }
                    }
                }
            };
            // `next` holds the ids of the step after those in flight
            for (; at < groups; at += kAhead * stride) {
#pragma unroll
                for (int j = 0; j < kAhead; ++j) {
                    if (at + j * stride >= groups) break;
                    score(at + j * stride, x[j]);
                    if (at + (kAhead + j) * stride < groups) load(next, x[j]);
                    ids_of(at + (kAhead + 1 + j) * stride, next);
                }
            }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            if (cluster > 1) {
                const uint32_t at = (uint32_t)__cvta_generic_to_shared(range + rank * kSelWarps + warp);
                if (lane < cluster) {
                    store_cluster(at, lane, lo);
                    store_cluster(at + 4, lane, hi);
                }
            } else if (lane == 0) {
                range[warp] = make_uint2(lo, hi);
            }
            if (cluster > 1) cluster_sync();
            else __syncthreads();
        }

        // ---- the choice: tokens rank, rank + cluster, .. of the tile, by teams of warps ----
        const int mine = nt > rank ? (nt - rank + cluster - 1) >> p.lg : 0;
        const int most_lg = mine <= 1 ? 3 : mine <= 2 ? 2 : mine <= 4 ? 1 : 0;
        int lg = 0;                                                // 2^lg warps in a team: more where scores are many
        while (lg < most_lg && m > 64 << lg) ++lg;
        const int tw = 1 << lg, team = warp >> lg, member = warp & (tw - 1), threads = 32 << lg, i = member * 32 + lane;
        auto team_sync = [&]() {
            if (tw == 1) __syncwarp();
            else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(threads) : "memory");
        };
        int* hist = bins[team << lg];
        for (int slot = team; slot < mine; slot += kSelWarps >> lg) {
            const int token = (slot << p.lg) + rank;
            const Seen s = seen_of(p, ctx, n, i0 + token);
            int32_t* list = a.lists + ((long long)(q0 + i0 + token) * p.l.kv_heads + head) * a.keep;
            if (head == 0 && i == 0) a.seen[q0 + i0 + token] = s.tokens;
            auto entry = [&](int b) {
                const int id = __ldg(table + b);
                return (unsigned)id < (unsigned)p.l.n_pages ? id : -1;
            };
            if (s.pages <= a.keep) {
#pragma unroll 4
                for (int b = i; b < a.keep; b += threads) list[b] = b < s.pages ? entry(b) : -1;
                continue;
            }
            const uint32_t* keys = scores + (size_t)slot * p.cap;
            const int mt = s.pages - a.first - a.last, need = a.keep - a.first - a.last;
            for (int j = i; j < a.first + a.last; j += threads)
                list[j < a.first ? j : j + need] = entry(j < a.first ? j : s.pages - a.first - a.last + j);
            if (need == 0) continue;

            // the range of all the tile's scores: queries are in units of their largest, so their scores are of one size
            uint32_t lo = 0xffffffffu, hi = 0;
            for (int e = lane; e < cluster * kSelWarps; e += 32) {
                const uint2 x = range[e];
                lo = min(lo, x.x);
                hi = max(hi, x.y);
            }
            lo = __reduce_min_sync(0xffffffffu, lo);
            hi = __reduce_max_sync(0xffffffffu, hi);
            // The least score that is taken, and how many of those equal to it: a histogram of the scores in [lo, hi] by their
            // upper bits; the bin that holds the `rest`-th largest of them; its scores, ranked by a warp where 32 hold
            // them, or that bin as the next range
            uint32_t least = lo;
            int rest = need, equal_taken;
            while (true) {
                const int shift = lo == hi ? 0 : max(0, 32 - __clz(hi - lo) - (8 + lg));
                reinterpret_cast<int4*>(hist)[2 * i] = reinterpret_cast<int4*>(hist)[2 * i + 1] = make_int4(0, 0, 0, 0);
                if (i == 0) ties[team] = 0;
                team_sync();
#pragma unroll 8
                for (int b = i; b < mt; b += threads) {
                    const uint32_t key = keys[b];
                    if (key >= lo && key <= hi) atomicAdd(hist + ((key - lo) >> shift), 1);
                }
                team_sync();
                // eight bins a thread, the highest first
                const int top = (kSelBins << lg) - 8 * (i + 1);
                int own[8], sum = 0;
                *reinterpret_cast<int4*>(own) = reinterpret_cast<const int4*>(hist + top)[0];
                *reinterpret_cast<int4*>(own + 4) = reinterpret_cast<const int4*>(hist + top)[1];
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += own[j];
                int upto = sum;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                if (tw > 1) {
                    if (lane == 31) part[warp].x = upto;
                    team_sync();
                    upto += __reduce_add_sync(0xffffffffu, lane < member ? part[(team << lg) + lane].x : 0);
                }
                if (upto - sum < rest && rest <= upto) {
                    int above = upto - sum;
#pragma unroll
                    for (int j = 7; j >= 0; --j) {
                        if (above < rest && rest <= above + own[j]) found[team] = make_int4(top + j, rest - above, own[j], 0);
                        above += own[j];
                    }
                }
                team_sync();
                const int4 f = found[team];
                least = lo + ((uint32_t)f.x << shift);
                rest = f.y;
                equal_taken = rest;
                if (rest == f.z) {                                 // the whole bin: those at its least too
                    equal_taken = INT_MAX;
                    break;
                }
                if (shift == 0) break;                             // it is one score
                hi = least + min(hi - least, (1u << shift) - 1);
                lo = least;
                if (f.z <= 32) {
                    if (tw == 1) {                                 // by ballots, which wait less than counts in memory
                        int at = 0;
#pragma unroll 4
                        for (int b0 = 0; b0 < mt; b0 += 32) {
                            const uint32_t key = b0 + lane < mt ? keys[b0 + lane] : 0;
                            const bool in = b0 + lane < mt && key >= lo && key <= hi;
                            const unsigned mask = __ballot_sync(0xffffffffu, in);
                            if (in) tied[team][at + __popc(mask & ((1u << lane) - 1))] = key;
                            at += __popc(mask);
                        }
                    } else {
#pragma unroll 8
                        for (int b = i; b < mt; b += threads) {
                            const uint32_t key = keys[b];
                            if (key >= lo && key <= hi) tied[team][atomicAdd(ties + team, 1)] = key;
                        }
                    }
                    team_sync();
                    const uint32_t key = lane < f.z ? tied[team][lane] : 0;
                    int larger = 0;
                    for (int j = 0; j < f.z; ++j) larger += __shfl_sync(0xffffffffu, key, j) > key;
                    least = __reduce_min_sync(0xffffffffu, lane < f.z && larger < rest ? key : 0xffffffffu);
                    equal_taken = rest - __popc(__ballot_sync(0xffffffffu, lane < f.z && key > least));
                    break;
                }
            }
            // In order: each thread's run of scores, of odd length, so that a warp's lie in different banks; their places go by
            // way of shared memory where they fit there, so that the table is read all at once
            const bool by_way = need <= kSelBins << lg;
            const int per = min(31, ((mt + threads - 1) >> (5 + lg)) | 1);
            team_sync();
            for (int from = 0, above0 = 0, equal0 = 0; from < mt; from += per * threads) {
                const int b0 = from + i * per, size = min(per, mt - b0);
                uint32_t above = 0, equal = 0;
#pragma unroll 8
                for (int j = 0; j < size; ++j) {
                    const uint32_t key = keys[b0 + j];
                    above |= (key > least ? 1u : 0u) << j;
                    equal |= (key == least ? 1u : 0u) << j;
                }
                const int mine = __popc(above) + (__popc(equal) << 16);            // below 2^13 each over the team
                int upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int x = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += x;
                }
                int all = __shfl_sync(0xffffffffu, upto, 31);
                if (tw > 1) {
                    if (lane == 0) part[warp].y = all;
                    team_sync();
                    const int x = lane < tw ? part[(team << lg) + lane].y : 0;
                    upto += __reduce_add_sync(0xffffffffu, lane < member ? x : 0);
                    all = __reduce_add_sync(0xffffffffu, x);
                }
                const int e = equal0 + ((upto - mine) >> 16);
                for (int drop = __popc(equal) - max(0, min(__popc(equal), equal_taken - e)); drop > 0; --drop) equal &= ~(0x80000000u >> __clz(equal));
                int place = above0 + ((upto - mine) & 0xffff) + min(e, equal_taken);
                for (uint32_t left = above | equal; left; left &= left - 1, ++place) {
                    const int b = b0 + __ffs(left) - 1;
                    if (by_way) hist[place] = b;
                    else list[a.first + place] = entry(a.first + b);
                }
                above0 += all & 0xffff;
                equal0 += all >> 16;
                if (tw > 1 && from + per * threads < mt) team_sync();
            }
            if (by_way) {
                team_sync();
#pragma unroll 4
                for (int j = i; j < need; j += threads) list[a.first + j] = entry(a.first + hist[j]);
            }
            team_sync();                                           // before the next token's
        }
    }

    // rows of no request
    if (head == 0) {
        const int end = start(a.n_req);
        for (long long t = end + (long long)blockIdx.x * kSelThreads + tid; t < a.total_q; t += (long long)gridDim.x * kSelThreads) a.seen[t] = -1;
        if (const int begin = start(0); begin > 0)
            for (long long t = (long long)blockIdx.x * kSelThreads + tid; t < begin; t += (long long)gridDim.x * kSelThreads) a.seen[t] = -1;
    }
}

// Two CTAs on an SM, with registers for the boxes ahead; with heads of 64 four, with half the registers, where there are so
// many that more at once pay, above 370: 64 tokens behind 8000 in pages of 32 (8 kv heads) 13.6 us (15.9 with two), 1024 behind
// 30000 34.7 (38.0); 320 CTAs of 40 requests with 1 to 9 drafts behind up to 6000 13.2 (11.4), though 40 single tokens behind
// 8000 13.2 (14.7).  With heads of 128 even three spill: 58.7 us for 44.4.
template <typename T, int D, int NT>
cudaError_t launch_tiles(SelectParams& p, long long tiles, cudaStream_t st)
{
    auto fn = kv_select_kernel<T, D, NT, 2>;
    if constexpr (D == 64) {
        const long long likely = p.direct ? tiles : tiles - p.c.n_req / 2;                 // a request's last tile half full
        if (likely * p.l.kv_heads << p.lg > 148 * 5 / 2) fn = kv_select_kernel<T, D, NT, 4>;
    }
    const size_t smem = (size_t)((p.tile + (1 << p.lg) - 1) >> p.lg) * p.cap * 4;
    if (smem > 24 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSelSmem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t lc = {};
    lc.blockDim = dim3(kSelThreads);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    auto grid = [&]() {
        attr[0].val.clusterDim.x = 1u << p.lg;
        lc.gridDim = dim3((unsigned)(tiles << p.lg), (unsigned)p.l.kv_heads);
    };
    if (p.lg > 3) {                                                // a size that a GPU need not take
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        int n = 0;
        lc.numAttrs = 1;
        grid();
        if (cudaOccupancyMaxActiveClusters(&n, fn, &lc) != cudaSuccess || n < 1) {
            cudaGetLastError();
            p.lg = 3;
        }
    }
    if (tiles < 1 || tiles << p.lg > INT_MAX) return cudaErrorInvalidValue;
    lc.numAttrs = 2;
    grid();
    return cudaLaunchKernelEx(&lc, fn, p);
}

// Tiles and clusters.  Tiles of 16 tokens read the boxes half as often as those of 8, which fill the GPU with fewer tokens:
// a chunk of 1024 behind 30000 (8 kv heads, pages of 64) takes 43.8 us with 16, 57.3 with 8; one of 100 behind 8000 14.1 and
// 10.4.  A cluster's CTAs share a tile's boxes, 16 a warp at a time, where there are fewer tiles than SMs: one token behind
// 32000 in pages of 16 (4 kv heads) takes 20.2 us with one CTA, 15.6 with 2, 12.7 with 4, 11.0 with 8, 10.6 with 16; one
// behind 131000 80.9 to 23.0 and 19.5; where tiles fill the GPU, more CTAs only add their own 7 us (32 tokens x 8 heads: 13.4
// us with one, 20.4 with 2).  They pay from 128 pages a CTA for one token (128 of them 7.3 us with one CTA, 7.8 with 2; 157
// 7.6 and 7.5), 120 for several (5 tokens, 94 pages 8.1 and 8.5; 251 with 2 and 4 9.1 and 8.6).
// Pages are counted by the table's width, for lengths are on the device: short contexts in wide tables get clusters and
// score rows that they do not need.  Single tokens behind 2000 lose 0 to 1.5 us to a table of 8192 pages; tiles of several
// tokens, whose score rows then fill an SM, much more: 32 requests x 4 tokens 34.5 us for 11.2, a chunk of 512 80.4 for 15.9.
// The counts of SMs and CTAs here are a whole B200's.
template <typename T, int D>
cudaError_t launch_select(SelectParams p, cudaStream_t st)
{
    p.cap = (p.c.table_width + 11) / 16 * 16 + 4;                  // the scores of a lane's neighbours in other banks
    p.direct = p.c.max_q <= 8;
    auto bytes = [&]() { return (size_t)((p.tile + (1 << p.lg) - 1) >> p.lg) * p.cap * 4; };
    const long long rows = (long long)p.c.total_q * p.l.kv_heads;
    p.lg = 0;
    if (!p.direct && p.c.total_q > 16LL * p.c.n_req && rows > 8 * 2 * 148) {
        p.tile = 16;
        while (p.lg < 3 && bytes() > 64 * 1024) ++p.lg;
        if (bytes() <= kSelSmem) return launch_tiles<T, D, 2>(p, p.c.total_q / 16 + (long long)p.c.n_req, st);
        p.lg = 0;
    }
    p.tile = p.c.max_q <= 1 ? 1 : 8;
    const int least = p.tile == 1 ? 128 : 120;
    const long long tiles = p.direct ? p.c.n_req : p.c.total_q / 8 + (long long)p.c.n_req;
    while (p.lg < 3 && tiles * p.l.kv_heads << p.lg < 148 && p.c.table_width > least << p.lg) ++p.lg;
    if (p.lg == 3 && tiles * p.l.kv_heads << 4 <= 148 && p.c.table_width > 1024) p.lg = 4;
    while (p.lg < 3 && bytes() > kSelSmem) ++p.lg;
    return launch_tiles<T, D, 1>(p, tiles, st);
}

template <int FMT>
cudaError_t launch_boxes(const BoxParams& p, cudaStream_t st)
{
    const dim3 grid((unsigned)((p.n + (long long)p.per - 1) / p.per), (unsigned)p.l.kv_heads);
    return p.l.head_dim == 64 ? kv_launch(kv_boxes_kernel<FMT, 64>, grid, 32 * kBoxWarps, 0, st, p)
                              : kv_launch(kv_boxes_kernel<FMT, 128>, grid, 32 * kBoxWarps, 0, st, p);
}

}  // namespace
}  // namespace b4

using namespace b4;

extern "C" {

int b4_kv_box_bytes(int head_dim, size_t* bytes)
{
    if (!bytes || (head_dim != 64 && head_dim != 128)) return cudaErrorInvalidValue;
    *bytes = (size_t)box_bytes(head_dim);
    return cudaSuccess;
}

int b4_kv_boxes(const b4_kv_cache* cache, const int32_t* slots, int n_tokens, void* boxes, b4_stream_t stream)
{
    BoxParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (n_tokens < 0) return cudaErrorInvalidValue;
    if (n_tokens == 0) return cudaSuccess;
    if (!slots || !boxes || !kv_aligned(slots, 4) || !kv_aligned(boxes, 16)) return cudaErrorInvalidValue;
    p.blocks = static_cast<const uint8_t*>(cache->blocks);
    p.boxes = static_cast<uint8_t*>(boxes);
    p.slots = slots;
    p.n = n_tokens;
    p.per = (int)std::max(1LL, std::min(16LL, (long long)n_tokens * p.l.kv_heads / (148 * 8)));
    return p.l.fmt == B4_KV_INT4 ? launch_boxes<B4_KV_INT4>(p, reinterpret_cast<cudaStream_t>(stream))
                                 : launch_boxes<B4_KV_NF4>(p, reinterpret_cast<cudaStream_t>(stream));
}

int b4_kv_select(const b4_kv_cache* cache, const b4_kv_choice* c, b4_stream_t stream)
{
    SelectParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (!c || c->n_req < 0 || c->total_q < 0 || c->max_q < 0 || c->table_width < 0 || c->table_width > B4_KV_SELECT_MAX_WIDTH ||
        c->table_stride < c->table_width)
        return cudaErrorInvalidValue;
    if (c->heads < 1 || c->heads % p.l.kv_heads || c->heads / p.l.kv_heads > 64) return cudaErrorInvalidValue;
    if (c->dtype != B4_DTYPE_F16 && c->dtype != B4_DTYPE_BF16) return cudaErrorInvalidValue;
    if (c->first < 0 || c->last < 1 || c->keep < 1 || c->keep > B4_KV_SELECT_MAX_WIDTH || (long long)c->first + c->last > c->keep ||
        (long long)c->keep * p.l.page_size > 0x80000000LL - 64)
        return cudaErrorInvalidValue;
    if (c->total_q == 0) return cudaSuccess;
    if (!c->q || !c->boxes || !c->lists || !c->seen || (c->n_req > 0 && (!c->ctx_len || !c->q_starts || (c->table_width > 0 && !c->tables))))
        return cudaErrorInvalidValue;
    // every CTA reads these while others write what they chose
    const RowSet lists = row_set(c->lists, 4, (long long)c->total_q * p.l.kv_heads * c->keep), seen = row_set(c->seen, 4, c->total_q);
    const RowSet reads[] = {row_set(c->tables, 4, c->n_req > 0 ? (c->n_req - 1) * c->table_stride + c->table_width : 0), row_set(c->ctx_len, 4, c->n_req),
                            row_set(c->q_starts, 4, c->n_req + 1LL), row_set(c->boxes, box_bytes(p.l.head_dim), (long long)p.l.n_pages * p.l.kv_heads),
                            row_set(c->q, 2, c->q_stride_token, c->q_stride_head, c->total_q, c->heads, p.l.head_dim)};
    if (rows_meet(lists, seen)) return cudaErrorInvalidValue;
    for (const RowSet& r : reads)
        if (rows_meet(r, lists) || rows_meet(r, seen)) return cudaErrorInvalidValue;
    if (!kv_aligned(c->q, 16) || !kv_aligned(c->boxes, 16) || (c->q_stride_token | c->q_stride_head) % 8 != 0) return cudaErrorInvalidValue;
    p.c = *c;
    p.group = c->heads / p.l.kv_heads;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (c->n_req == 0) return cudaMemsetAsync(c->seen, 0xff, 4 * (size_t)c->total_q, st);
    if (c->dtype == B4_DTYPE_F16) return p.l.head_dim == 64 ? launch_select<__half, 64>(p, st) : launch_select<__half, 128>(p, st);
    return p.l.head_dim == 64 ? launch_select<__nv_bfloat16, 64>(p, st) : launch_select<__nv_bfloat16, 128>(p, st);
}

}  // extern "C"
