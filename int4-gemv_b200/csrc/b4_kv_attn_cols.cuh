// b4_kv_attn_cols.cuh -- a warp's part of attention over the 4-bit cache for few
// queries: a tile of 8 * NT query columns against chunks of 32 tokens, its feed, and
// what it leaves; shared by the kernel over block tables and the one over lists.
#pragma once

#include "b4_kv_attn.cuh"

namespace b4 {

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

// NF4's lookup table, at shared address kTable: row b holds 32 copies of (high, low) of byte b's two levels, the two swapped
// in the upper 16 copies: there the high parts alone (keys) lie in the odd banks, and the two products of the values add up
// to the same.
template <typename C>
__device__ __forceinline__ void fill_levels(uint8_t* smem, uint32_t smem_at, int tid, float up)
{
    for (int i = tid; i < 256 * 16; i += C::kThreads) {
        const uint32_t b = i >> 4, hi = nf4_pair(b, up), lo = nf4_pair_low(b, up);
        reinterpret_cast<uint4*>(smem + C::kTable - smem_at)[i] = (i & 15) < 8 ? make_uint4(hi, lo, hi, lo) : make_uint4(lo, hi, lo, hi);
    }
}

// ONE: a segment is one query's, its columns the heads of the group alone
template <typename T, int FMT, int D, int NT, int PT, bool ONE>
struct WarpTile {
    using C = WarpCfg<FMT, D, NT, PT>;
    static constexpr int kStages = C::kStages;
    static constexpr bool kLow = std::is_same<T, __half>::value;          // NF4 levels in two parts
    static constexpr float kUp = kLow ? kNf4Least : kNf4Even;
    static constexpr int W = D / 32;       // packed words of a token's codes that a lane of the key operand holds
    static constexpr int VW = D / 64;      // ... of the value operand
    static constexpr int tile1 = PT == 16 ? C::kBlock : 16 * C::kRow;

    const AttnParams& p;
    const b4_kv_attn& a;
    const int lane, g, t;
    uint8_t* const ring;
    // this lane's places in a stage: its key and value rows of the chunk's two 16-token tiles, its token's scales.
    // Row g of a tile's eight is token gr: the pairs 2, 3 and 6, 7 are swapped, so that the four lanes t of a value
    // read (tokens gr(2t)) see rows of both parities and with them all banks
    const int gr, k_at, v_at, v_other, s_at;
    const uint32_t t_key, t_val, ring_at;
    const int n16, scale_at;
    int stage, feed;

    float o[NT][D / 16][4];                // m-tile mt: columns 2t, 2t + 1 of d = g * (D / 8) + 2 mt, and of d + 1
    float mx[NT][2], sum[NT][2], qf[NT][2];
    uint32_t qb[NT][D / 8];
    int lim[NT][2];                        // keys that a column sees: below lim, at or above lim - window
    int vexp;
    struct { int q0, n, ctx, head, tile, token; } u = {};   // the segment; a chunk's first token

    __device__ __forceinline__ WarpTile(const AttnParams& params, uint8_t* warps_ring, int its_lane)
        : p(params), a(params.a), lane(its_lane), g(its_lane >> 2), t(its_lane & 3), ring(warps_ring), gr(g ^ (g >> 1 & 1)),
          k_at(gr * C::kRow + t * (W * 4)), v_at(PT * C::kRow + (2 * t + (t & 1)) * C::kRow + g * (VW * 4)),
          v_other(t & 1 ? -C::kRow : C::kRow), s_at(its_lane / PT * C::kBlock + PT * D + its_lane % PT * C::kScale),
          t_key(C::kTable + its_lane * 8 + (its_lane >> 4) * 4), t_val(C::kTable + its_lane * 8),
          ring_at((uint32_t)__cvta_generic_to_shared(warps_ring) + its_lane * 16), n16(PT * C::kScale / 16),
          scale_at(its_lane < n16 ? its_lane * 16 : (params.l.page_size - PT) * C::kScale + its_lane * 16), stage(0), feed(0)
    {
    }

    __device__ __forceinline__ bool col_row(int col, int& token, int& head) const
    {
        const int c = u.tile * C::kCols + col;
        if (ONE) {
            token = 0;
            head = u.head * p.group + c;
            return c < p.group;
        }
        token = c / p.group;
        head = u.head * p.group + (c - token * p.group);
        return c < u.n * p.group;
    }

    // a segment's queries as the right operand, in the order of the decoded codes.  A negative factor of the scores
    // goes into the queries, so that a larger product is a larger score.
    __device__ __forceinline__ void load_queries(int nt, uint4 (&v)[W])
    {
        int token, head;
        const bool in = col_row(nt * 8 + g, token, head);
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (u.q0 + token) * a.q_stride_token +
                                                          head * a.q_stride_head + t * (D / 4));
#pragma unroll
        for (int i = 0; i < W; ++i) v[i] = in ? __ldg(src + i) : make_uint4(0, 0, 0, 0);
    }

    __device__ __forceinline__ void begin_segment(uint4 (&queries)[NT][W])
    {
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
                lim[nt][j] = ONE || a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + token + 1);
                mx[nt][j] = kNoMax;
                sum[nt][j] = 0.0f;
            }
#pragma unroll
            for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[nt][mt][j] = 0.0f;
        }
        vexp = kNoExp;
    }


    // 32 tokens; `masked` where some column does not see all of them
    __device__ __forceinline__ void compute(const uint8_t* buf, int there, bool masked)
    {
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
            const int end = ONE || a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + 1 + (u.tile * C::kCols + C::kCols - 1) / p.group);
            const int begin = !ONE && a.window > 0 ? u.ctx - u.n + 1 + u.tile * C::kCols / p.group - a.window : 0;
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
                        if (!(some >> x & 1) || at >= lim[nt][j & 1] || (!ONE && a.window > 0 && at < lim[nt][j & 1] - a.window))
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
    }

    // A run of a segment's chunks: its page ids by 32, `ids` from page `base` on and the 32 after those; the segment's queries.
    struct Run {
        const int32_t* row;
        int first, last, base, ids, more;
        uint4 queries[NT][W];
    };

    __device__ __forceinline__ int load_id(const Run& r, int page) const
    {
        return page < a.table_width && (long long)page << p.l.page_shift < u.ctx ? __ldg(r.row + page) : -1;
    }

    // chunks first .. last - 1 of the segment u, whose page ids are `row`: asks for what walk() needs first
    __device__ __forceinline__ void open(Run& r, const int32_t* row, int first, int last)
    {
        r.row = row;
        r.first = first;
        r.last = last;
        r.base = first * kChunk >> p.l.page_shift;
        r.ids = load_id(r, r.base + lane);
        r.more = load_id(r, r.base + 32 + lane);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) load_queries(nt, r.queries[nt]);
    }

    __device__ __forceinline__ void walk(Run& r)
    {
        const uint8_t* blocks = p.blocks + u.head * p.l.block;
        const long long page_bytes = p.l.kv_heads * p.l.block;
        int next = r.first, queue = 0;
        auto issue = [&]() {               // the next chunk, if any, into stage `feed`
            int there = 0;
            if (next < r.last) {
                const int page = next * kChunk >> p.l.page_shift;
                if (page - r.base >= 32) {
                    r.ids = r.more;
                    r.base += 32;
                    r.more = load_id(r, r.base + 32 + lane);
                }
                const int half = PT == 32 ? next * kChunk & (p.l.page_size - 1) : 0;       // of a page of 64
                const uint32_t dst = ring_at + feed * C::kStage;
#pragma unroll
                for (int i = 0; i < C::kPages; ++i) {
                    // a chunk of two pages begins at an even place of the 32: its second page is among them
                    const int id = __shfl_sync(0xffffffffu, r.ids, page - r.base + i);
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
#pragma unroll 1
        for (int i = 0; i < kStages; ++i) issue();
        begin_segment(r.queries);

        // every key of a chunk is seen by every column where the chunk lies in [clear, seen)
        const int seen = ONE || a.flags & B4_KV_FULL ? u.ctx : min(u.ctx, u.ctx - u.n + 1 + u.tile * C::kCols / p.group);
        const int clear = !ONE && a.window > 0 ? u.ctx - a.window : 0;
#pragma unroll 1
        for (int c = r.first; c < r.last; ++c) {
            u.token = c * kChunk;
            const int there = queue >> (2 * kStages - 2) & 3;
            asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
            __syncwarp();
            compute(ring + stage * C::kStage, there, u.token < clear || u.token + kChunk > seen || there != (1 << C::kPages) - 1);
            __syncwarp();
            issue();
            if (++stage == kStages) stage = 0;
        }
    }

    // The sums over the lanes; returns the factor of the outputs.
    __device__ __forceinline__ float finish()
    {
        const float vup = pow2(vexp - kLift) * (FMT == B4_KV_NF4 ? 1.0f / kUp : 1.0f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int off = 4; off < 32; off <<= 1) sum[nt][j] += __shfl_xor_sync(0xffffffffu, sum[nt][j], off);
        return vup;
    }

    // a whole segment's outputs
    __device__ __forceinline__ void store(float vup)
    {
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
    }

    // a piece: [column][D], maxima, sums
    __device__ __forceinline__ void store_piece(float* dst, float vup)
    {
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
    }
};

}  // namespace b4
