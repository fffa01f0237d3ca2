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

#include "b4_kv_attn_cols.cuh"

namespace b4 {

// What a segment (a request's head and column tile) costs a warp beside its chunks, in a chunk's time: 96 requests of 1 to
// 6000 tokens take 78 us without it, 69 with 1, 68 with 2 and with 4.
constexpr int kSegChunks = 2;

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
    constexpr int kWarps = C::kWarps, kThreads = C::kThreads, kScan = C::kScan;
    constexpr float kUp = WarpTile<T, FMT, D, NT, PT, false>::kUp;
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
    if (FMT == B4_KV_NF4) fill_levels<C>(attn_smem, smem_at, tid, kUp);
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
        // ---- a warp's run, by segments ----
        WarpTile<T, FMT, D, NT, PT, false> tile(p, ring_of(warp), lane);
        auto& u = tile.u;
        int r;
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

            typename WarpTile<T, FMT, D, NT, PT, false>::Run run;
            tile.open(run, a.tables + (long long)r * a.table_stride, q.chunk0 + first, q.chunk0 + last);
            tile.walk(run);

            // ---- the end of a segment, or of the run ----
            const float vup = tile.finish();
            if (first == 0 && last == q.chunks) {
                tile.store(vup);
            } else {
                // a piece: the run's last goes into the ring, which is free, its first to the workspace
                const bool is_last = v == v1;
                tile.store_piece(is_last ? reinterpret_cast<float*>(tile.ring) : ws.first + ((long long)cta * kWarps + warp) * C::kPiece, vup);
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
