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
// integers; NF4: kNf4Up).  Softmax's maximum and sum run along the tokens, in
// fp32, private to a warp; P goes to fp16 (its rounding is of the size of the
// output's own), relative to the running maximum of the weights and a running
// power of two that bounds the value scales, so small scales lose nothing.
//
// Split.  The (request, kv head, column tile, 64-token chunk) units of the whole
// call form one sequence; every CTA gets an equal run of it, every warp of a CTA
// an equal run of the CTA's, whatever the requests' lengths.  A segment (request,
// head, tile) inside one warp's run is written by the warp; others leave a piece
// (sum, maximum, unnormalised output) that the CTA joins in unit order, and
// segments that cross CTAs are joined by the last CTA to arrive, again in unit
// order: the same bits every time, one launch, no wait between CTAs.
//
// Feed.  Each warp brings its own chunks into its own ring of shared memory with
// bulk copies (a copy a page: a head's part of a page is one block), and reads page
// ids one unit ahead of the copies, so a warp never waits for another.
#pragma once

#include <type_traits>

#include "b4_kv_attn.cuh"
#include "b4_tma.cuh"

namespace b4 {

constexpr int kAttnStages = 2;

template <int FMT, int D, int NT>
struct WarpCfg {
    static constexpr int kWarps = FMT == B4_KV_NF4 && NT > 1 ? 6 : 8;  // what shared memory holds
    static constexpr int kRow = D / 2;                                 // bytes of a token's codes
    static constexpr int kScale = FMT == B4_KV_INT4 ? 2 : 4;
    static constexpr int kStage = 2 * kChunk * (kRow + kScale);
    static constexpr int kCols = 8 * NT;
    static constexpr int kPiece = kCols * (D + 2);                     // floats: output, maxima, sums
    static constexpr int kTable = FMT == B4_KV_NF4 ? 65536 : 0;        // 256 rows of 32 copies, 256 bytes apart
    static constexpr int kQ = NT == 1 ? 0 : kCols * D * 2;             // the queries' operands, of one warp
    static constexpr int kRing = kWarps * kAttnStages * kStage;
    static constexpr int kSmem = kTable + kRing + kWarps * kQ;
    static_assert(kAttnStages * kStage >= kPiece * 4, "a warp's last piece goes into its ring");
};

// a unit as the warp that reads it sees it
struct __align__(16) AttnUnit {
    int q0, n, ctx, head;      // the request's queries and tokens, the kv head
    int tile, token, flags, pages;
};
constexpr int kUnitFirst = 1, kUnitLast = 2;   // of its segment

struct WarpPiece {
    long long s0, s1;          // the segment's units
    int q0, n, head, tile;
    int valid;
};

struct WarpWs {                // the workspace: counters, then pieces that other warps or CTAs read
    int* count;
    float* first;              // [grid][warps] a warp's first piece
    float* cross;              // [grid][2] a CTA's part of a segment that began before it / goes on after it
};

// Walks the units of a run in order.
struct UnitWalk {
    AttnReq q;
    int r, seg, chunk, tiles;
};

template <typename T, int FMT, int D, int NT>
__global__ void __launch_bounds__(WarpCfg<FMT, D, NT>::kWarps * 32, 1) kv_attn_warp_kernel(const AttnParams p, const WarpWs ws)
{
    using C = WarpCfg<FMT, D, NT>;
    constexpr int kAttnWarps = C::kWarps, kThreads = 32 * kAttnWarps;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    __shared__ uint64_t full[kAttnWarps][kAttnStages];
    __shared__ AttnUnit units[kAttnWarps][kAttnStages];
    __shared__ WarpPiece pieces[kAttnWarps][2];
    __shared__ long long scan[kAttnWarps * 32 + 1], warp_sum[kAttnWarps];
    __shared__ int last_cta[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t = lane & 3;
    const b4_kv_attn& a = p.a;
    uint8_t* ring = attn_smem + C::kTable + warp * kAttnStages * C::kStage;
    uint8_t* table = attn_smem;
    if (lane < kAttnStages) mbar_init(&full[warp][lane], 1);
    if (lane < 2) pieces[warp][lane].valid = 0;
    if (FMT == B4_KV_NF4) {
        for (int b = tid; b < 256; b += kThreads) {
            const uint32_t v = nf4_pair(b);
            uint4* row = reinterpret_cast<uint4*>(table + b * 256);
#pragma unroll
            for (int i = 0; i < 8; ++i) row[(i + b) & 7] = make_uint4(v, v, v, v);
        }
    }
    fence_mbar_init();
    kv_begin();

    // ---- the call's units, and this warp's run of them ----
    auto tiles_of = [&](const AttnReq& q) { return (q.n * p.group + C::kCols - 1) / C::kCols; };
    auto units_of = [&](const AttnReq& q) { return (long long)p.l.kv_heads * tiles_of(q) * q.chunks; };
    const int per = (a.n_req + kAttnWarps * 32 - 1) / (kAttnWarps * 32);
    {
        long long sum = 0;
        for (int i = 0; i < per; ++i) {
            const int r = tid * per + i;
            if (r < a.n_req) sum += units_of(attn_request(p, r));
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
        for (int w = 0; w < kAttnWarps; ++w)
            if (w < warp) base += warp_sum[w];
        scan[tid + 1] = base + inc;
        if (tid == 0) scan[0] = 0;
        __syncthreads();
    }
    const long long total = scan[kAttnWarps * 32];
    if (total == 0) return;
    // few units: four a CTA at least, so that fewer pieces cross CTAs
    const long long ctas = min((long long)gridDim.x, (total + 3) / 4);
    const int cta = blockIdx.x;
    if (cta >= ctas) return;
    const long long c0 = cta * total / ctas, c1 = (cta + 1) * total / ctas;
    const long long v0 = c0 + warp * (c1 - c0) / kAttnWarps, v1 = c0 + (warp + 1) * (c1 - c0) / kAttnWarps;

    if (v0 < v1) {
        // ---- walk: find the run's first unit, then step ----
        UnitWalk w;
        long long at;                          // the current request's first unit
        {
            int lo = 0, hi = kAttnWarps * 32;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (scan[mid] <= v0) lo = mid;
                else hi = mid;
            }
            w.r = lo * per;
            at = scan[lo];
            for (;;) {
                w.q = attn_request(p, w.r);
                const long long u = units_of(w.q);
                if (v0 < at + u) break;
                at += u;
                ++w.r;
            }
            w.tiles = tiles_of(w.q);
            const long long in = v0 - at;
            w.seg = (int)(in / w.q.chunks);
            w.chunk = (int)(in - (long long)w.seg * w.q.chunks);
        }
        const int pages_per = kChunk >> p.l.page_shift;
        const uint64_t policy = evict_first_policy();
        auto page_id = [&]() -> int {          // of this lane's page in the walk's unit, -1 where there is none
            const int token = (w.q.chunk0 + w.chunk) * kChunk + (lane << p.l.page_shift);
            if (lane >= pages_per || token >= w.q.ctx) return -1;
            return __ldg(a.tables + (long long)w.r * a.table_stride + (token >> p.l.page_shift));
        };
        auto step = [&]() {
            if (++w.chunk < w.q.chunks) return;
            w.chunk = 0;
            if (++w.seg < p.l.kv_heads * w.tiles) return;
            w.seg = 0;
            do {
                w.q = attn_request(p, ++w.r);
            } while (w.q.n == 0);
            w.tiles = tiles_of(w.q);
        };
        auto issue = [&](int stage, int id) {  // the walk's unit into a stage
            const bool there = (unsigned)id < (unsigned)p.l.n_pages;
            const unsigned mask = __ballot_sync(0xffffffffu, there);
            const int head = w.seg / w.tiles;
            if (lane == 0) {
                AttnUnit u;
                u.q0 = w.q.q0;
                u.n = w.q.n;
                u.ctx = w.q.ctx;
                u.head = head;
                u.tile = w.seg - head * w.tiles;
                u.token = (w.q.chunk0 + w.chunk) * kChunk;
                u.flags = (w.chunk == 0 ? kUnitFirst : 0) | (w.chunk == w.q.chunks - 1 ? kUnitLast : 0);
                u.pages = (int)mask;
                units[warp][stage] = u;
                fence_proxy_async();
                mbar_arrive_expect_tx(&full[warp][stage], (uint32_t)(__popc(mask) * p.l.block));
            }
            __syncwarp();
            if (there)
                bulk_g2s(ring + stage * C::kStage + lane * (int)p.l.block, p.blocks + ((long long)id * p.l.kv_heads + head) * p.l.block,
                         (uint32_t)p.l.block, &full[warp][stage], policy);
        };

        const int count = (int)(v1 - v0);
        long long seg_unit = v0 - w.chunk;     // the segment's first unit
        int seg_chunks = w.q.chunks;
        int ids[kAttnStages + 1], produced = 0;
        // the first stages' page ids together, one round trip
        UnitWalk start = w;
#pragma unroll
        for (int s = 0; s <= kAttnStages; ++s) {
            ids[s] = -1;
            if (s < count) {
                if (s > 0) step();
                ids[s] = page_id();
            }
        }
        w = start;
#pragma unroll
        for (int s = 0; s < kAttnStages; ++s) {
            if (s >= count) break;
            issue(s, ids[s]);
            ++produced;
            if (s + 1 < count) step();
        }
        int next_id = ids[kAttnStages];

        // ---- per segment: queries, running statistics, output ----
        float o[NT][D / 8 / 2][4];             // m-tile mt: columns 2t, 2t + 1 of d = g * (D / 8) + 2 mt, and of d + 1
        float mx[NT][2], sum[NT][2], qf[NT][2];
        int lim[NT][2];                        // keys that a column sees: below lim, at or above lim - window
        uint32_t qb[NT == 1 ? D / 8 : 1];
        uint4* qs = reinterpret_cast<uint4*>(attn_smem + C::kTable + C::kRing + warp * C::kQ);
        int vexp = -126;
        constexpr int W = D / 32;              // packed words of a token's codes that a lane of the key operand holds
        uint4 raw[NT == 1 ? W : 1];

        auto col_row = [&](const AttnUnit& u, int col, int& token, int& head) -> bool {
            const int c = u.tile * C::kCols + col;
            token = c / p.group;
            head = u.head * p.group + (c - token * p.group);
            return c < u.n * p.group;
        };
        auto q_words = [&](const AttnUnit& u, int nt, uint4 (&v)[W]) {
            int token, head;
            const bool in = col_row(u, nt * 8 + g, token, head);
            const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (u.q0 + token) * a.q_stride_token +
                                                              head * a.q_stride_head + t * (D / 4));
#pragma unroll
            for (int i = 0; i < W; ++i) v[i] = in ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
        };
        // the operand's pairs in the order of the decoded codes, fp16; bf16 rows times a power of two that
        // brings their largest to [2^10, 2^11), so that fp16's range holds them (its 11 bits hold bf16's 8)
        auto q_operand = [&](uint4 (&v)[W], float& factor) {
            factor = 1.0f;
            if (std::is_same<T, __nv_bfloat16>::value) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = max(top, max(x[j] << 16 & 0x7fffffffu, x[j] & 0x7fff0000u));
                }
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const int e = min(max((int)(top >> 23) - 127, -110), 126);
                const float up = pow2(10 - e);
                factor = pow2(e - 10 < -126 ? -126 : e - 10);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    uint32_t* x = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        x[j] = pack_half2(__uint_as_float(x[j] << 16) * up, __uint_as_float(x[j] & 0xffff0000u) * up);
                }
            }
            if (FMT == B4_KV_INT4) {
#pragma unroll
                for (int i = 0; i < W; ++i) v[i] = int4_pair_order(v[i]);
            }
        };
        auto begin_segment = [&](const AttnUnit& u) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float factor;
                if (NT == 1) {
                    q_operand(*reinterpret_cast<uint4(*)[W]>(raw), factor);
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        qb[4 * i] = raw[i].x;
                        qb[4 * i + 1] = raw[i].y;
                        qb[4 * i + 2] = raw[i].z;
                        qb[4 * i + 3] = raw[i].w;
                    }
                } else {
                    uint4 v[W];
                    q_words(u, nt, v);
                    q_operand(v, factor);
#pragma unroll
                    for (int i = 0; i < W; ++i) qs[(nt * W + i) * 32 + lane] = v[i];
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qf[nt][j] = __shfl_sync(0xffffffffu, factor, (2 * t + j) * 4) * (a.scale * kLog2e) *
                                (FMT == B4_KV_NF4 ? 1.0f / kNf4Up : 1.0f);
                    int token, head;
                    col_row(u, nt * 8 + 2 * t + j, token, head);
                    lim[nt][j] = a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + token + 1);
                    mx[nt][j] = -INFINITY;
                    sum[nt][j] = 0.0f;
                }
#pragma unroll
                for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][mt][j] = 0.0f;
            }
            if (NT > 1) __syncwarp();
            vexp = -126;
        };

        int stage = 0, phase = 0;
        bool whole = false;                    // the current segment's first unit is in this run
        AttnUnit u = units[warp][0];
        if (NT == 1) q_words(u, 0, *reinterpret_cast<uint4(*)[W]>(raw));

        for (int i = 0; i < count; ++i) {
            const bool fresh = i == 0 || (u.flags & kUnitFirst);
            if (fresh) {
                begin_segment(u);
                whole = u.flags & kUnitFirst;
            }
            AttnUnit nu;
            if (i + 1 < count) {               // the next unit's queries are asked for before this one is computed
                nu = units[warp][stage ^ 1];
                if (NT == 1 && (nu.flags & kUnitFirst)) q_words(nu, 0, *reinterpret_cast<uint4(*)[W]>(raw));
            }
            mbar_wait_bounded(&full[warp][stage], phase);
            const uint8_t* buf = ring + stage * C::kStage;
            // every key seen by every column: no masks
            const int seen = a.flags & B4_KV_FULL ? u.ctx : u.ctx - u.n + 1 + u.tile * C::kCols / p.group;
            // the keys that some column of the tile sees
            const int tile_end = a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + 1 + (u.tile * C::kCols + C::kCols - 1) / p.group);
            const int tile_begin = a.window > 0 ? u.ctx - u.n + 1 + u.tile * C::kCols / p.group - a.window : 0;
            const bool masked = u.token + kChunk > min(seen, u.ctx) || u.pages != (1 << pages_per) - 1 ||
                                (a.window > 0 && u.token < u.ctx - a.window);
            constexpr int G = NT == 1 ? 4 : NT == 2 ? 2 : 1;       // 16-token tiles between two softmax steps
#pragma unroll
            for (int s0 = 0; s0 < 4; s0 += G) {
                float s[G][NT][4], vs[G][2];
                float top[NT][2], vtop = 0.0f;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
                for (int st = 0; st < G; ++st) {
                    const int tok = (s0 + st) * 16, blk = tok >> p.l.page_shift, row = tok & (p.l.page_size - 1);
                    const uint8_t* bp = buf + blk * (int)p.l.block;
                    const uint8_t* kp = bp + row * C::kRow;
                    const uint8_t* sp = bp + p.l.page_size * D + (row + g) * C::kScale;
                    uint32_t k0[W], k1[W];
                    if (D == 128) {
                        const uint4 x = *reinterpret_cast<const uint4*>(kp + g * C::kRow + t * 16);
                        const uint4 y = *reinterpret_cast<const uint4*>(kp + (g + 8) * C::kRow + t * 16);
                        k0[0] = x.x; k0[1] = x.y; k0[W - 2] = x.z; k0[W - 1] = x.w;
                        k1[0] = y.x; k1[1] = y.y; k1[W - 2] = y.z; k1[W - 1] = y.w;
                    } else {
                        const uint2 x = *reinterpret_cast<const uint2*>(kp + g * C::kRow + t * 8);
                        const uint2 y = *reinterpret_cast<const uint2*>(kp + (g + 8) * C::kRow + t * 8);
                        k0[0] = x.x; k0[1] = x.y;
                        k1[0] = y.x; k1[1] = y.y;
                    }
                    float ks[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint8_t* q = sp + 8 * j * C::kScale;
                        ks[j] = FMT == B4_KV_INT4 ? __half2float(*reinterpret_cast<const __half*>(q)) : *reinterpret_cast<const float*>(q);
                        q += p.l.page_size * C::kScale;
                        vs[st][j] = FMT == B4_KV_INT4 ? __half2float(*reinterpret_cast<const __half*>(q)) : *reinterpret_cast<const float*>(q);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) s[st][nt][j] = 0.0f;
#pragma unroll
                    for (int i2 = 0; i2 < W; ++i2) {
                        uint32_t x[4], y[4];
                        if (FMT == B4_KV_INT4) {
                            int4_word_to_half2(k0[i2], x);
                            int4_word_to_half2(k1[i2], y);
                        } else {
#pragma unroll
                            for (int b = 0; b < 4; ++b) {
                                x[b] = *reinterpret_cast<const uint32_t*>(table + __byte_perm(k0[i2], lane * 4, 0x7604 | b << 4));
                                y[b] = *reinterpret_cast<const uint32_t*>(table + __byte_perm(k1[i2], lane * 4, 0x7604 | b << 4));
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            uint4 b;
                            if (NT == 1) b = make_uint4(qb[4 * i2], qb[4 * i2 + 1], qb[4 * i2 + 2], qb[4 * i2 + 3]);
                            else b = qs[(nt * W + i2) * 32 + lane];
                            mma_f16(s[st][nt], x[0], y[0], x[1], y[1], b.x, b.y);
                            mma_f16(s[st][nt], x[2], y[2], x[3], y[3], b.z, b.w);
                        }
                    }
                    bool in[2] = {true, true};
                    if (masked) {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int key = tok + g + 8 * j;
                            in[j] = (u.pages >> (key >> p.l.page_shift) & 1) && u.token + key < tile_end && u.token + key >= tile_begin;
                            if (!in[j]) vs[st][j] = 0.0f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) vtop = fmaxf(vtop, vs[st][j] < INFINITY ? vs[st][j] : 0.0f);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float& x = s[st][nt][j];
                            x *= ks[j >> 1] * qf[nt][j & 1];
                            if (masked) {
                                const int key = u.token + tok + g + 8 * (j >> 1);
                                const bool ok = in[j >> 1] && key < lim[nt][j & 1] &&
                                                (a.window == 0 || key >= lim[nt][j & 1] - a.window);
                                if (!ok) x = -INFINITY;
                            }
                            top[nt][j & 1] = fmaxf(top[nt][j & 1], x);
                        }
                }
                // running maxima, of the scores and of the values' scales
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) {
                    vtop = fmaxf(vtop, __shfl_xor_sync(0xffffffffu, vtop, off));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) top[nt][j] = fmaxf(top[nt][j], __shfl_xor_sync(0xffffffffu, top[nt][j], off));
                }
                const int ve = min(max((int)(__float_as_uint(vtop) >> 23) - 126, vexp), 126);
                const float vkeep = pow2(max(vexp - ve, -126)), vdown = pow2(-ve);
                bool moved = ve != vexp;
                vexp = ve;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j) moved |= top[nt][j] > mx[nt][j];
                if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float keep[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const float next = fmaxf(mx[nt][j], top[nt][j]);
                            keep[j] = next == -INFINITY ? 1.0f : fast_exp2(mx[nt][j] - next);
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
                // weights, as the right operand: tokens along k, a query a lane's row
                uint32_t pb[G][NT][2];
                const uint32_t swap = t & 1 ? 0x1032 : 0x3210;     // odd lanes read their pair's second token first
#pragma unroll
                for (int st = 0; st < G; ++st)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float w0 = mx[nt][0] == -INFINITY ? 0.0f : fast_exp2(s[st][nt][2 * j] - mx[nt][0]);
                            float w1 = mx[nt][1] == -INFINITY ? 0.0f : fast_exp2(s[st][nt][2 * j + 1] - mx[nt][1]);
                            sum[nt][0] += w0;
                            sum[nt][1] += w1;
                            const float v = vs[st][j] * vdown;
                            float x0 = w0 * v, x1 = w1 * v;
                            if (masked) {                      // 0 whatever an unseen token's scale is
                                x0 = w0 == 0.0f ? 0.0f : x0;
                                x1 = w1 == 0.0f ? 0.0f : x1;
                            }
                            pb[st][nt][j] = __byte_perm(movmatrix(pack_half2(x0, x1)), 0, swap);
                        }
                // values: lane (g, t) holds d = g * (D / 8) .. of the tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int st = 0; st < G; ++st) {
                    const int tok = (s0 + st) * 16, blk = tok >> p.l.page_shift, row = tok & (p.l.page_size - 1);
                    const uint8_t* vp = buf + blk * (int)p.l.block + (p.l.page_size + row) * C::kRow + g * (D / 16);
                    const int ta = 2 * t + (t & 1), tb = 2 * t + 1 - (t & 1);
                    constexpr int VW = D / 64;                     // packed words of a token that a lane holds
                    uint32_t v[4][VW];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint8_t* q = vp + ((j & 1 ? tb : ta) + 8 * (j >> 1)) * C::kRow;
                        if (VW == 2) {
                            const uint2 x = *reinterpret_cast<const uint2*>(q);
                            v[j][0] = x.x;
                            v[j][VW - 1] = x.y;
                        } else {
                            v[j][0] = *reinterpret_cast<const uint32_t*>(q);
                        }
                    }
#pragma unroll
                    for (int i2 = 0; i2 < VW; ++i2) {
                        uint32_t e[2], f[2];                       // NF4: bytes of (first token, second token), even and odd columns
                        if (FMT == B4_KV_NF4) {
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const uint32_t x = v[2 * j][i2], y = v[2 * j + 1][i2];
                                e[j] = (x & 0x0f0f0f0fu) | (y << 4 & 0xf0f0f0f0u);
                                f[j] = (x >> 4 & 0x0f0f0f0fu) | (y & 0xf0f0f0f0u);
                            }
                        }
#pragma unroll
                        for (int b = 0; b < 4; ++b) {
                            uint32_t lo[2], hi[2];
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                if (FMT == B4_KV_INT4) {
                                    const uint32_t x = __byte_perm(v[2 * j][i2], v[2 * j + 1][i2], b | b << 4 | (4 + b) << 8 | (4 + b) << 12);
                                    lo[j] = hsub2_bits(lop3_and_or<0x000f000fu, 0x64006400u>(x), 0x6408);
                                    hi[j] = hsub2_bits(lop3_and_or<0x00f000f0u, 0x54005400u>(x), 0x5480);
                                } else {
                                    lo[j] = *reinterpret_cast<const uint32_t*>(table + __byte_perm(e[j], lane * 4, 0x7604 | b << 4));
                                    hi[j] = *reinterpret_cast<const uint32_t*>(table + __byte_perm(f[j], lane * 4, 0x7604 | b << 4));
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma_f16(o[nt][4 * i2 + b], lo[0], hi[0], lo[1], hi[1], pb[st][nt][0], pb[st][nt][1]);
                        }
                    }
                }
            }
            __syncwarp();

            // the stage is free: the unit after next goes into it
            if (produced < count) {
                issue(stage, next_id);
                ++produced;
                if (produced < count) {
                    step();
                    next_id = page_id();
                }
            }

            // ---- the end of a segment, or of the run ----
            if ((u.flags & kUnitLast) || i + 1 == count) {
                const float vup = pow2(vexp) * (FMT == B4_KV_NF4 ? 1.0f / kNf4Up : 1.0f);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int off = 4; off < 32; off <<= 1) sum[nt][j] += __shfl_xor_sync(0xffffffffu, sum[nt][j], off);
                if (whole && (u.flags & kUnitLast)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            int token, head;
                            if (!col_row(u, nt * 8 + 2 * t + j, token, head)) continue;
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
                    // a piece [column][D], maxima, sums: the run's first goes to the workspace, its last into the ring
                    const bool is_last = i + 1 == count;
                    float* dst = is_last ? reinterpret_cast<float*>(ring) : ws.first + ((long long)cta * kAttnWarps + warp) * C::kPiece;
                    __syncwarp();
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
                        pc.s1 = seg_unit + seg_chunks;
                        pc.q0 = u.q0;
                        pc.n = u.n;
                        pc.head = u.head;
                        pc.tile = u.tile;
                        pc.valid = 1;
                        pieces[warp][is_last] = pc;
                    }
                }
            }
            if (i + 1 < count) {
                if (u.flags & kUnitLast) {
                    seg_unit = v0 + i + 1;
                    // a segment's chunks are counted when it ends in another run: from its request's extent
                    const int begin = a.window > 0 ? max(0, nu.ctx - nu.n + 1 - a.window) : 0;
                    seg_chunks = max(1, (nu.ctx + kChunk - 1) / kChunk - begin / kChunk);
                }
                u = nu;
                stage ^= 1;
                if (stage == 0) phase ^= 1;
            }
        }
    }
    __syncthreads();

    // ---- join the pieces of this CTA, in unit order ----
    auto emit = [&](const WarpPiece& pc, int e, const float4& x, float m, float l) {    // four columns' outputs of one query
        const int c = pc.tile * C::kCols + e / D, token = c / p.group, head = pc.head * p.group + (c - token * p.group);
        if (c >= pc.n * p.group) return;
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        T w[4] = {kv_round<T>(x.x * inv), kv_round<T>(x.y * inv), kv_round<T>(x.z * inv), kv_round<T>(x.w * inv)};
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + (pc.q0 + token) * a.out_stride_token + head * a.out_stride_head + e % D) =
            *reinterpret_cast<const uint2*>(w);
        if (a.lse && e % D == 0)
            a.lse[(long long)(pc.q0 + token) * a.heads + head] = l > 0.0f ? (m + fast_log2(l)) * kLn2 : -INFINITY;
    };
    // joins `n` pieces (piece i at base(i)) for the four values at e
    auto join = [&](int n, int e, auto base, float4& x, float& m, float& l) {
        const int col = e / D;
        m = -INFINITY;
        for (int i = 0; i < n; ++i) m = fmaxf(m, base(i)[C::kCols * D + col]);
        x = make_float4(0, 0, 0, 0);
        l = 0.0f;
        for (int i = 0; i < n; ++i) {
            const float* b = base(i);
            const float mi = b[C::kCols * D + col], k = mi == -INFINITY ? 0.0f : fast_exp2(mi - m);
            const float4 y = *reinterpret_cast<const float4*>(b + e);
            l += k * b[C::kCols * (D + 1) + col];
            x.x += k * y.x;
            x.y += k * y.y;
            x.z += k * y.z;
            x.w += k * y.w;
        }
    };
    auto piece_at = [&](int i) -> const float* {
        return i & 1 ? reinterpret_cast<const float*>(attn_smem + C::kTable + (i >> 1) * kAttnStages * C::kStage)
                     : ws.first + ((long long)cta * kAttnWarps + (i >> 1)) * C::kPiece;
    };
    WarpPiece cross[2];
    cross[0].valid = cross[1].valid = 0;
    for (int i = 0; i < 2 * kAttnWarps;) {
        const WarpPiece pc = pieces[i >> 1][i & 1];
        if (!pc.valid) {
            ++i;
            continue;
        }
        uint64_t list = i;                     // four bits a piece
        int n = 1, j = i + 1;
        for (; j < 2 * kAttnWarps; ++j) {
            const WarpPiece& x = pieces[j >> 1][j & 1];
            if (!x.valid) continue;
            if (x.s0 != pc.s0) break;
            list |= (uint64_t)j << (4 * n);
            ++n;
        }
        i = j;
        const bool inside = pc.s0 >= c0 && pc.s1 <= c1;
        const int which = pc.s0 >= c0;
        if (!inside) cross[which] = pc;
        for (int e = tid * 4; e < C::kCols * D; e += kThreads * 4) {
            float4 x;
            float m, l;
            join(n, e, [&](int k) { return piece_at((int)(list >> (4 * k)) & 15); }, x, m, l);
            if (inside) {
                emit(pc, e, x, m, l);
            } else {
                float* dst = ws.cross + ((long long)cta * 2 + which) * C::kPiece;
                *reinterpret_cast<float4*>(dst + e) = x;
                if (e % D == 0) {
                    dst[C::kCols * D + e / D] = m;
                    dst[C::kCols * (D + 1) + e / D] = l;
                }
            }
        }
    }
    if (!cross[0].valid && !cross[1].valid) return;

    // ---- segments that cross CTAs: the last to arrive joins them ----
    auto owner = [&](long long u) { return (int)(((u + 1) * ctas - 1) / total); };
    __threadfence();
    __syncthreads();
    if (tid < 2) {
        last_cta[tid] = 0;
        if (cross[tid].valid) {
            const int f = owner(cross[tid].s0), n = owner(cross[tid].s1 - 1) - f + 1;
            last_cta[tid] = atomicAdd(ws.count + f, 1) == n - 1;
            if (last_cta[tid]) ws.count[f] = 0;
        }
    }
    __syncthreads();
    __threadfence();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if (!last_cta[k]) continue;
        const WarpPiece pc = cross[k];
        const int f = owner(pc.s0), n = owner(pc.s1 - 1) - f + 1;
        for (int e = tid * 4; e < C::kCols * D; e += kThreads * 4) {
            float4 x;
            float m, l;
            join(n, e, [&](int c) -> const float* { return ws.cross + ((long long)(f + c) * 2 + (c == 0)) * C::kPiece; }, x, m, l);
            emit(pc, e, x, m, l);
        }
    }
}

}  // namespace b4
