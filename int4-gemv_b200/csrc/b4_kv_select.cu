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
#include <algorithm>
#include <climits>

#include "b4_kv.cuh"

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
    int group, tile, cluster, cap;         // heads of a kv head, tokens of a tile, CTAs of a cluster, scores of a token
    int direct;                            // a tile index is a request's
};

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32, kSelTile = 8, kSelBins = 256;

__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// larger for larger x; 0 below all of them
__device__ __forceinline__ uint32_t ordered(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f);                  // -0 as 0
    return u & 0x80000000u ? ~u : u | 0x80000000u;
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

template <typename T, int D>
__global__ void __launch_bounds__(kSelThreads) kv_select_kernel(const SelectParams p)
{
    constexpr int V = D / 32;                                      // 16-byte words of a box that a lane holds
    constexpr int kRow = 2 * D + 64;
    extern __shared__ __align__(16) uint32_t scores[];             // [tokens of this CTA][cap]
    __shared__ __align__(16) uint8_t query[kSelTile * kRow];       // above, below of a token
    __shared__ __align__(16) int bins[kSelWarps][kSelBins];        // of a team's warps together; then the places of its choice
    __shared__ int2 part[kSelWarps], found[kSelWarps];

    const b4_kv_choice& a = p.c;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int rank = blockIdx.x % p.cluster, head = blockIdx.y;
    const int at_tile = blockIdx.x / p.cluster;
    kv_begin();

    // ---- the request and its tokens ----
    auto start = [&](int r) { return max(0, min(__ldg(a.q_starts + r), a.total_q)); };
    int r = at_tile, tile0 = 0;
    if (!p.direct) {
        // request r has the tiles from start / 8 + r on, more than it needs at most: the last that begins at or before this one
        int lo = 0, n = a.n_req;
        while (n > 1) {
            const int step = (n + 31) / 32, probe = lo + lane * step;
            const bool in = lane * step < n && (lane == 0 || start(probe) / kSelTile + probe <= at_tile);
            const int last = 31 - __clz(__ballot_sync(0xffffffffu, in));
            n = min(step, n - last * step);
            lo += last * step;
        }
        r = lo;
        tile0 = at_tile - (start(r) / kSelTile + r);
    }
    const int q0 = start(r), n = max(0, start(r + 1) - q0), ctx = max(0, __ldg(a.ctx_len + r));
    // rows of no request
    if (head == 0) {
        const int end = start(a.n_req);
        for (long long t = end + (long long)blockIdx.x * kSelThreads + tid; t < a.total_q; t += (long long)gridDim.x * kSelThreads) a.seen[t] = -1;
        if (const int begin = start(0); begin > 0)
            for (long long t = (long long)blockIdx.x * kSelThreads + tid; t < begin; t += (long long)gridDim.x * kSelThreads) a.seen[t] = -1;
    }
    const int32_t* table = a.tables + (long long)r * a.table_stride;

    for (int i0 = tile0 * p.tile; i0 < n; i0 = p.direct ? i0 + p.tile : n) {
        const int nt = min(p.tile, n - i0);
        const Seen most = seen_of(p, ctx, n, i0 + nt - 1);
        const int m = most.pages > a.keep ? most.pages - a.first - a.last : 0;     // pages to score

        if (m > 0) {
            // ---- scores: this CTA's boxes, 16 a warp at a time ----
            const int g = lane >> 2, t = lane & 3;
            const int groups = (m + 15) / 16;
            struct Boxes {                                         // of a step: rows g and g + 8
                uint4 word[2][V];
                float unit[2];
                bool there[2];
            };
            const int stride = p.cluster * kSelWarps;
            int at = rank + p.cluster * warp;
            auto ids_of = [&](int at, int (&id)[2]) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int b = at * 16 + g + 8 * j;
                    id[j] = b < m ? __ldg(table + a.first + b) : -1;
                }
            };
            auto load = [&](const int (&id)[2], Boxes& x) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    x.there[j] = (unsigned)id[j] < (unsigned)p.l.n_pages;
                    const uint8_t* src = static_cast<const uint8_t*>(a.boxes) + ((long long)(x.there[j] ? id[j] : 0) * p.l.kv_heads + head) * box_bytes(D);
#pragma unroll
                    for (int i = 0; i < V; ++i) x.word[j][i] = __ldg(reinterpret_cast<const uint4*>(src + 64 * i) + t);
                    x.unit[j] = __ldg(reinterpret_cast<const float*>(src + 2 * D));
                }
            };
            Boxes x[2];                                            // two steps' boxes and the next one's page ids in flight
            int id[2], next[2];
            ids_of(at, id);
            ids_of(at + stride, next);
            if (at < groups) load(id, x[0]);
            if (at + stride < groups) load(next, x[1]);
            ids_of(at + 2 * stride, id);

            // a token a warp: the sums of its heads' parts above and below 0, as int8
            if (warp < p.tile) {
                constexpr int C = D / 32;                          // columns of a lane
                double above[C], below[C];
#pragma unroll
                for (int j = 0; j < C; ++j) above[j] = below[j] = 0.0;
                if (warp < nt) {
                    const T* src = static_cast<const T*>(a.q) + (q0 + i0 + warp) * a.q_stride_token + (long long)head * p.group * a.q_stride_head + lane * C;
#pragma unroll 8
                    for (int h = 0; h < p.group; ++h) {
                        T x[C];
                        if (C == 4) *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(src + h * a.q_stride_head));
                        else *reinterpret_cast<uint32_t*>(x) = __ldg(reinterpret_cast<const uint32_t*>(src + h * a.q_stride_head));
#pragma unroll
                        for (int j = 0; j < C; ++j) {
                            const float v = kv_float(x[j]);
                            above[j] += v > 0.0f ? v : 0.0f;
                            below[j] += v > 0.0f ? 0.0f : v;       // NaN too
                        }
                    }
                }
                float hi[C], lo[C], top = 0.0f;
                bool finite = true;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    hi[j] = (float)above[j];
                    lo[j] = (float)below[j];
                    const float x = fmaxf(hi[j], -lo[j]);
                    finite = finite && hi[j] < INFINITY && lo[j] > -INFINITY;
                    top = fmaxf(top, x);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                finite = __all_sync(0xffffffffu, finite);
                const float s = top > 0.0f ? __fmul_rn(top, 1.0f / 127.0f) : 1.0f;
                uint32_t wh = 0, wl = 0;
#pragma unroll
                for (int j = 0; j < C; ++j) {
                    wh |= (uint32_t)(finite ? box_code(hi[j], s) & 255 : 0) << (8 * j);
                    wl |= (uint32_t)(finite ? box_code(lo[j], s) & 255 : 0) << (8 * j);
                }
                uint8_t* dst = query + warp * kRow + lane * C;
                if (C == 4) {
                    *reinterpret_cast<uint32_t*>(dst) = wh;
                    *reinterpret_cast<uint32_t*>(dst + D) = wl;
                } else {
                    *reinterpret_cast<uint16_t*>(dst) = (uint16_t)wh;
                    *reinterpret_cast<uint16_t*>(dst + D) = (uint16_t)wl;
                }
            }
            if (p.cluster > 1) cluster_sync();                     // the others have begun, or are done with the last tile's scores
            else __syncthreads();

            uint4 qw[V];
#pragma unroll
            for (int i = 0; i < V; ++i)
                qw[i] = g < p.tile ? *reinterpret_cast<const uint4*>(query + g * kRow + 64 * i + 16 * t) : make_uint4(0, 0, 0, 0);
            const uint32_t scores_at = (uint32_t)__cvta_generic_to_shared(scores);
            auto score = [&](int at, const Boxes& x) {
                int acc[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    mma_s8(acc, x.word[0][i].x, x.word[1][i].x, x.word[0][i].y, x.word[1][i].y, qw[i].x, qw[i].y);
                    mma_s8(acc, x.word[0][i].z, x.word[1][i].z, x.word[0][i].w, x.word[1][i].w, qw[i].z, qw[i].w);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int token = 2 * t + (j & 1), b = at * 16 + g + 8 * (j >> 1);
                    if (token >= nt || b >= m) continue;
                    const float unit = x.unit[j >> 1];
                    const uint32_t key = !x.there[j >> 1] ? 0u : ordered(unit < INFINITY ? __fmul_rn((float)acc[j], unit) : INFINITY);
                    const uint32_t place = (uint32_t)(token / p.cluster) * p.cap + b;
                    if (p.cluster > 1) store_cluster(scores_at + 4 * place, token % p.cluster, key);
                    else scores[place] = key;
                }
            };
            for (; at < groups; at += 2 * stride) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (at + j * stride >= groups) break;
                    score(at + j * stride, x[j]);
                    if (at + (2 + j) * stride < groups) load(id, x[j]);
                    ids_of(at + (3 + j) * stride, id);
                }
            }
            if (p.cluster > 1) cluster_sync();
            else __syncthreads();
        }

        // ---- the choice: tokens rank, rank + cluster, .. of the tile, by teams of warps ----
        const int mine = nt > rank ? (nt - rank + p.cluster - 1) / p.cluster : 0;
        const int tw = mine <= 1 ? 8 : mine <= 2 ? 4 : mine <= 4 ? 2 : 1;          // warps of a team
        const int team = warp / tw, member = warp % tw;
        if (team < mine) {
            const int token = team * p.cluster + rank, threads = tw * 32, i = member * 32 + lane;
            const Seen s = seen_of(p, ctx, n, i0 + token);
            int32_t* list = a.lists + ((long long)(q0 + i0 + token) * p.l.kv_heads + head) * a.keep;
            if (head == 0 && i == 0) a.seen[q0 + i0 + token] = s.tokens;
            auto entry = [&](int b) {
                const int id = __ldg(table + b);
                return (unsigned)id < (unsigned)p.l.n_pages ? id : -1;
            };
            if (s.pages <= a.keep) {
                for (int b = i; b < a.keep; b += threads) list[b] = b < s.pages ? entry(b) : -1;
            } else {
                const uint32_t* keys = scores + (size_t)team * p.cap;
                const int mt = s.pages - a.first - a.last, need = a.keep - a.first - a.last;
                for (int b = i; b < a.first + a.last; b += threads)
                    list[b < a.first ? b : b + need] = entry(b < a.first ? b : s.pages - a.last + (b - a.first));
                auto team_sync = [&]() {
                    if (tw == 1) __syncwarp();
                    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(threads) : "memory");
                };
                if (need > 0) {
                    int* hist = bins[team * tw];
                    // the range of the scores
                    uint32_t lo = 0xffffffffu, hi = 0;
#pragma unroll 8
                    for (int b = i; b < mt; b += threads) {
                        lo = min(lo, keys[b]);
                        hi = max(hi, keys[b]);
                    }
                    lo = __reduce_min_sync(0xffffffffu, lo);
                    hi = __reduce_max_sync(0xffffffffu, hi);
                    if (tw > 1) {
                        if (lane == 0) part[warp] = make_int2((int)lo, (int)hi);
                        team_sync();
                        for (int w = 0; w < tw; ++w) {
                            lo = min(lo, (uint32_t)part[team * tw + w].x);
                            hi = max(hi, (uint32_t)part[team * tw + w].y);
                        }
                    }
                    // The least score that is taken, and how many of those equal to it: a histogram of the scores in [lo, hi]
                    // by their upper bits, the bin that holds the `rest`-th largest of them, that bin as the next range
                    uint32_t least = lo;
                    for (int rest = need; lo < hi;) {
                        const int shift = max(0, 32 - __clz(hi - lo) - (31 - __clz(kSelBins * tw)));
                        reinterpret_cast<int4*>(hist)[2 * i] = reinterpret_cast<int4*>(hist)[2 * i + 1] = make_int4(0, 0, 0, 0);
                        team_sync();
#pragma unroll 8
                        for (int b = i; b < mt; b += threads) {
                            const uint32_t key = keys[b];
                            if (key >= lo && key <= hi) atomicAdd(hist + ((key - lo) >> shift), 1);
                        }
                        team_sync();
                        // eight bins a thread, the highest first
                        const int top = kSelBins * tw - 8 * (i + 1);
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
                            for (int w = 0; w < member; ++w) upto += part[team * tw + w].x;
                        }
                        if (upto - sum < rest && rest <= upto) {
                            int above = upto - sum;
#pragma unroll
                            for (int j = 7; j >= 0; --j) {
                                if (above < rest && rest <= above + own[j]) found[team] = make_int2(top + j, rest - above == own[j] ? 0 : rest - above);
                                above += own[j];
                            }
                        }
                        team_sync();
                        const int2 f = found[team];
                        least = lo + ((uint32_t)f.x << shift);
                        rest = f.y;
                        if (rest == 0 || shift == 0) break;        // the whole bin is taken, or it is one score
                        hi = least + min(hi - least, (1u << shift) - 1);
                        lo = least;
                    }
                    // each member's run of scores: those above it, and those at it, the first of which are taken
                    const int run = ((mt + threads - 1) / threads) * 32, b0 = min(mt, member * run), b1 = min(mt, b0 + run);
                    int above0 = 0, equal0 = 0, ties;
                    {
                        int above = 0, equal = 0;
#pragma unroll 8
                        for (int b = b0 + lane; b < b1; b += 32) {
                            above += keys[b] > least;
                            equal += keys[b] == least;
                        }
                        above = __reduce_add_sync(0xffffffffu, above);
                        equal = __reduce_add_sync(0xffffffffu, equal);
                        int all = above;
                        if (tw > 1) {
                            team_sync();
                            if (lane == 0) part[warp] = make_int2(above, equal);
                            team_sync();
                            all = 0;
                            for (int w = 0; w < tw; ++w) {
                                const int2 c = part[team * tw + w];
                                all += c.x;
                                if (w < member) {
                                    above0 += c.x;
                                    equal0 += c.y;
                                }
                            }
                        }
                        ties = need - all;
                    }
                    // their places in order, by way of shared memory where they fit, so that the table is read all at once
                    const bool fits = need <= kSelBins * tw;
                    for (int b = b0; b < b1; b += 32) {
                        const uint32_t key = b + lane < b1 ? keys[b + lane] : 0;
                        const unsigned gt = __ballot_sync(0xffffffffu, b + lane < b1 && key > least), eq = __ballot_sync(0xffffffffu, b + lane < b1 && key == least);
                        const unsigned before = (1u << lane) - 1;
                        const int e = equal0 + __popc(eq & before);
                        if (gt >> lane & 1 || (eq >> lane & 1 && e < ties)) {
                            const int place = above0 + __popc(gt & before) + min(e, ties);
                            if (fits) hist[place] = b + lane;
                            else list[a.first + place] = entry(a.first + b + lane);
                        }
                        above0 += __popc(gt);
                        equal0 += __popc(eq);
                    }
                    if (fits) {
                        team_sync();
                        for (int j = i; j < need; j += threads) list[a.first + j] = entry(a.first + hist[j]);
                    }
                }
            }
        }
    }
}

template <typename T, int D>
cudaError_t launch_select(SelectParams p, cudaStream_t st)
{
    auto fn = kv_select_kernel<T, D>;
    p.tile = p.c.max_q <= 1 ? 1 : kSelTile;
    p.direct = p.c.max_q <= kSelTile;
    const long long tiles = p.direct ? p.c.n_req : p.c.total_q / kSelTile + p.c.n_req;
    if (tiles < 1 || tiles * 8 > INT_MAX) return cudaErrorInvalidValue;
    p.cap = (p.c.table_width + 15) / 16 * 16;
    // a CTA's boxes, 16 a warp, where few tiles would leave SMs without one; and shared memory for the scores
    p.cluster = 1;
    while (p.cluster < 8 && tiles * p.l.kv_heads * p.cluster < 148 && p.cap > 128 * p.cluster) p.cluster *= 2;
    auto bytes = [&]() { return (size_t)((p.tile + p.cluster - 1) / p.cluster) * p.cap * 4; };
    while (p.cluster < 8 && bytes() > 200 * 1024) p.cluster *= 2;
    const size_t smem = bytes();
    if (smem > 32 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)(tiles * p.cluster), (unsigned)p.l.kv_heads);
    lc.blockDim = dim3(kSelThreads);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)p.cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    lc.attrs = attr;
    lc.numAttrs = 2;
    return cudaLaunchKernelEx(&lc, fn, p);
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
    if (!kv_aligned(c->q, 16) || !kv_aligned(c->boxes, 16) || (c->q_stride_token | c->q_stride_head) % 8 != 0) return cudaErrorInvalidValue;
    p.c = *c;
    p.group = c->heads / p.l.kv_heads;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (c->n_req == 0) return cudaMemsetAsync(c->seen, 0xff, 4 * (size_t)c->total_q, st);
    if (c->dtype == B4_DTYPE_F16) return p.l.head_dim == 64 ? launch_select<__half, 64>(p, st) : launch_select<__half, 128>(p, st);
    return p.l.head_dim == 64 ? launch_select<__nv_bfloat16, 64>(p, st) : launch_select<__nv_bfloat16, 128>(p, st);
}

}  // extern "C"
