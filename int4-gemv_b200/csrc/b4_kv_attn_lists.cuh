// b4_kv_attn_lists.cuh -- attention over lists of pages, one for each query and kv
// head: the products and the softmax of b4_kv_attn_cols.cuh, with a schedule for lists.
//
// Split.  A list is short (tens of pages) and there are many, of lengths that are alike
// (a choice keeps as many pages for every query), so a list goes to half a CTA's warps,
// which share its chunks in runs and join what they leave in shared memory: the two
// halves of an SM's CTA work on lists of their own, one through its beginning and end
// while the other multiplies.  The kernel over block tables gives every warp an equal
// run of all chunks instead: even for any lengths, for searches before and joins across
// CTAs after that cost lists of 32 pages of 64 as much as their products (64 heads over
// 8 x 128, 32 queries, INT4: 28.9 us).  Where there are fewer lists than halves of CTAs
// some share a list, whose pieces the last to arrive joins in the list's order: the
// same bits every time.
#pragma once

#include "b4_kv_attn_cols.cuh"

namespace b4 {

struct ListWs {                // the workspace
    int* count;                // [lists] parts that have arrived, where several share one
    float* pieces;             // [lists][parts]
};

// Four columns of a query, e of [column][D], of n pieces (at(w): the w-th, in global memory or not) relative to their
// largest maximum.
struct Joined {
    float4 x;
    float m, l;
};

template <typename C, int D, bool GLOBAL, typename At>
__device__ __forceinline__ Joined join_pieces(int e, int n, At at)
{
    const int col = e / D;
    auto one = [](const float* v) { return GLOBAL ? __ldcg(v) : *v; };
    Joined j = {make_float4(0.0f, 0.0f, 0.0f, 0.0f), kNoMax, 0.0f};
#pragma unroll 4
    for (int w = 0; w < n; ++w) j.m = fmaxf(j.m, one(at(w) + C::kCols * D + col));
#pragma unroll 4
    for (int w = 0; w < n; ++w) {
        const float* b = at(w);
        const float f = fast_exp2(one(b + C::kCols * D + col) - j.m);
        const float4 y = GLOBAL ? __ldcg(reinterpret_cast<const float4*>(b + e)) : *reinterpret_cast<const float4*>(b + e);
        j.l += f * one(b + C::kCols * (D + 1) + col);
        j.x = make_float4(j.x.x + f * y.x, j.x.y + f * y.y, j.x.z + f * y.z, j.x.w + f * y.w);
    }
    return j;
}

template <typename T, int FMT, int D, int NT, int PT>
__global__ void __launch_bounds__(WarpCfg<FMT, D, NT, PT>::kThreads, 1) kv_attn_lists_kernel(const AttnParams p, const ListWs ws)
{
    using C = WarpCfg<FMT, D, NT, PT>;
    using Tile = WarpTile<T, FMT, D, NT, PT, true>;
    constexpr int kTeam = C::kWarps / 2, kTeamThreads = 32 * kTeam;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    __shared__ int last_part[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = warp / kTeam, member = warp - team * kTeam, tt = tid - team * kTeamThreads;
    const b4_kv_attn& a = p.a;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(attn_smem);
    auto ring_of = [&](int w) { return attn_smem + (w < C::kBelow ? w * C::kRing : 2 * C::kTable - smem_at + (w - C::kBelow) * C::kRing); };
    auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kTeamThreads) : "memory"); };
    if (FMT == B4_KV_NF4) fill_levels<C>(attn_smem, smem_at, tid, Tile::kUp);
    kv_begin();
    if (FMT == B4_KV_NF4) __syncthreads();

    const int tiles = (p.group + C::kCols - 1) / C::kCols, per_token = p.l.kv_heads * tiles * p.parts;
    const long long items = (long long)a.total_q * per_token;
    Tile tile(p, ring_of(warp), lane);
    auto& u = tile.u;
    u.n = 1;
    for (long long item = blockIdx.x + (long long)team * gridDim.x; item < items; item += 2LL * gridDim.x) {
        const int token = (int)div64(item, per_token);
        int rest = (int)(item - (long long)token * per_token);
        const int seen = __ldg(a.ctx_len + token);
        if (seen < 0) continue;                                    // no query's row
        const int of_head = tiles * p.parts;
        u.head = rest / of_head;
        rest -= u.head * of_head;
        u.tile = rest / p.parts;
        const int part = rest - u.tile * p.parts;
        u.q0 = token;
        u.ctx = seen;
        // the list's chunks, one even where nothing is seen; a part that has less than one for each warp is left out
        const int chunks = max(1, (attn_held(p, seen) + kChunk - 1) / kChunk);
        const int parts = p.parts == 1 ? 1 : min(p.parts, (chunks + kTeam - 1) / kTeam), share = parts == 1 ? chunks : (chunks + parts - 1) / parts;
        const int c0 = min(chunks, part * share), c1 = min(chunks, c0 + share);
        if (part >= parts) continue;
        const int run = (share + kTeam - 1) / kTeam, first = min(c1, c0 + member * run), last = min(c1, first + run);
        const int busy = (c1 - c0 + run - 1) / run;                // warps with chunks
        if (first < last) {
            tile.walk(a.tables + (long long)token * a.table_stride + u.head * p.list_head, 0, first, last);
            const float vup = tile.finish();
            tile.store_piece(reinterpret_cast<float*>(tile.ring), vup);            // which is free
        }
        team_sync();

        // ---- join, and the part's piece or the outputs ----
        auto emit = [&](int e, const Joined& j) {
            const int c = u.tile * C::kCols + e / D, head = u.head * p.group + c;
            if (c >= p.group) return;
            const float inv = j.l > 0.0f ? 1.0f / j.l : 0.0f;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + token * a.out_stride_token + head * a.out_stride_head + e % D) =
                make_uint2(kv_round2<T>(j.x.x * inv, j.x.y * inv), kv_round2<T>(j.x.z * inv, j.x.w * inv));
            if (a.lse && e % D == 0) a.lse[(long long)token * a.heads + head] = j.l > 0.0f ? (j.m + fast_log2(j.l)) * kLn2 : -INFINITY;
        };
        const long long list = div64(item, p.parts);
        auto piece_of = [&](int k) { return ws.pieces + (list * p.parts + k) * C::kPiece; };
        for (int e = 4 * tt; e < C::kCols * D; e += 4 * kTeamThreads) {
            const Joined j = join_pieces<C, D, false>(e, busy, [&](int w) { return reinterpret_cast<const float*>(ring_of(team * kTeam + w)); });
            if (parts == 1) {
                emit(e, j);
            } else {
                float* dst = piece_of(part);
                *reinterpret_cast<float4*>(dst + e) = j.x;
                if (e % D == 0) {
                    dst[C::kCols * D + e / D] = j.m;
                    dst[C::kCols * (D + 1) + e / D] = j.l;
                }
            }
        }
        if (parts > 1) {
            team_sync();
            if (tt == 0) {
                last_part[team] = count_in(ws.count + list) == parts - 1;
                if (last_part[team]) ws.count[list] = 0;
            }
            team_sync();
            if (last_part[team])
                for (int e = 4 * tt; e < C::kCols * D; e += 4 * kTeamThreads) emit(e, join_pieces<C, D, true>(e, parts, piece_of));
        }
        team_sync();                                               // before the rings are filled again
    }
}

}  // namespace b4
