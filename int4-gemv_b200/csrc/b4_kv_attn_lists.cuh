// b4_kv_attn_lists.cuh -- attention over lists of pages, one for each query and kv
// head: the products and the softmax of b4_kv_attn_cols.cuh, with a schedule for lists.
//
// Split.  A list is short (tens of pages) and there are many, of lengths that are alike
// (a choice keeps as many pages for every query), so a list goes to a team of warps, a
// half or a quarter of a CTA's (TEAMS = 2 or 4, by the host's model of their times), which
// share its chunks in runs and join what they leave in shared memory: the teams of an SM's
// CTA work on lists of their own, one through its beginning and end while the others
// multiply.  The kernel over block tables gives every warp an equal run of all chunks
// instead: even for any lengths, for searches before and joins across CTAs after that cost
// lists of 32 pages of 64 as much as their products (64 heads over 8 x 128, 32 queries,
// INT4: 28.9 us).  Lists that are too few for one more round of all teams are shared by
// several, whose pieces the last to arrive joins in the list's order: the same bits every
// time.
//
// What bounds it.  Many lists: the products, a chunk's 600 instructions at 2.4 a cycle (16
// warps an SM, 2000 cycles for a warp alone, 3200 with three beside it on a scheduler), and
// 5700 cycles a list around them, half of which the other teams' products hide.  In two teams
// 32 queries over 32 pages of 64 (64 heads over 8 x 128, INT4) take 22.7 us, 69 MB, 3.0 TB/s;
// in four 64 over 64 pages 68.8 us, 275 MB, 4.0 TB/s, 96 over up to 64 pages of 16 (32 heads over
// 8 x 64, NF4 in bf16) 24.3 us, a chunk of 300 over 32 pages of 32 (28 heads over 4 x 128,
// INT4) 48.0 us, whose lists' 162 MB come from L2.  Few: latency, one query over 16 pages of
// 64 7.7 us.
#pragma once

#include "b4_kv_attn_cols.cuh"

namespace b4 {

struct ListWs {                // the workspace
    int* count;                // [shared lists] parts that have arrived
    float* pieces;             // [shared lists][parts]
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

template <typename T, int FMT, int D, int NT, int PT, int TEAMS>
__global__ void __launch_bounds__(WarpCfg<FMT, D, NT, PT>::kThreads, 1) kv_attn_lists_kernel(const AttnParams p, const ListWs ws)
{
    using C = WarpCfg<FMT, D, NT, PT>;
    using Tile = WarpTile<T, FMT, D, NT, PT, true>;
    constexpr int kTeam = C::kWarps / TEAMS, kTeamThreads = 32 * kTeam;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    __shared__ int last_part[TEAMS];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = warp / kTeam, member = warp - team * kTeam, tt = tid - team * kTeamThreads;
    const b4_kv_attn& a = p.a;
    const uint32_t smem_at = (uint32_t)__cvta_generic_to_shared(attn_smem);
    auto ring_of = [&](int w) { return attn_smem + (w < C::kBelow ? w * C::kRing : 2 * C::kTable - smem_at + (w - C::kBelow) * C::kRing); };
    auto team_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(kTeamThreads) : "memory"); };
    if (FMT == B4_KV_NF4) fill_levels<C>(attn_smem, smem_at, tid, Tile::kUp);
    kv_begin();
    if (FMT == B4_KV_NF4) __syncthreads();

    const int tiles = (p.group + C::kCols - 1) / C::kCols, per_token = p.l.kv_heads * tiles;
    const long long items = p.whole + ((long long)a.total_q * per_token - p.whole) * p.parts, step = (long long)TEAMS * gridDim.x;
    Tile tile(p, ring_of(warp), lane);
    typename Tile::Run run;
    auto& u = tile.u;
    u.n = 1;
    struct Item {
        long long id, list;
        int token, head, tile, part, parts, busy;                  // parts of its list, warps of this one with chunks
    };
    auto list_of = [&](long long item) { return item < p.whole ? item : p.whole + div64(item - p.whole, p.parts); };
    auto seen_of = [&](long long item) { return item < items ? __ldg(a.ctx_len + div64(list_of(item), per_token)) : -1; };
    // The first item with work from `item` on, whose query sees `seen`: asks for its first page ids and its queries.
    auto open = [&](long long item, int seen) {
        Item x = {};
        for (; item < items; item += step, seen = seen_of(item)) {
            if (seen < 0) continue;                                // no query's row
            x.list = list_of(item);
            x.token = (int)div64(x.list, per_token);
            const int rest = (int)(x.list - (long long)x.token * per_token), parts = item < p.whole ? 1 : p.parts;
            x.head = tiles == 1 ? rest : rest / tiles;
            x.tile = rest - x.head * tiles;
            x.part = parts == 1 ? 0 : (int)(item - p.whole - (x.list - p.whole) * parts);
            // the list's chunks, one even where nothing is seen; a part that would have less than one for each warp is left out
            const int chunks = max(1, (attn_held(p, seen) + kChunk - 1) / kChunk);
            x.parts = parts == 1 ? 1 : min(parts, (chunks + kTeam - 1) / kTeam);
            if (x.part >= x.parts) continue;
            const int share = x.parts == 1 ? chunks : (chunks + x.parts - 1) / x.parts;
            const int c0 = min(chunks, x.part * share), c1 = min(chunks, c0 + share);
            const int each = (share + kTeam - 1) / kTeam, first = min(c1, c0 + member * each);
            x.busy = (c1 - c0 + each - 1) / each;
            u.q0 = x.token;
            u.head = x.head;
            u.tile = x.tile;
            u.ctx = seen;
            tile.open(run, a.tables + (long long)x.token * a.table_stride + x.head * p.list_head, first, min(c1, first + each));
            break;
        }
        x.id = item;
        return x;
    };
    const long long start = blockIdx.x + (long long)team * gridDim.x;
    for (Item x = open(start, seen_of(start)), next; x.id < items; x = next) {
        const int next_seen = seen_of(x.id + step);
        if (run.first < run.last) {
            tile.walk(run);
            const float vup = tile.finish();
            tile.store_piece(reinterpret_cast<float*>(tile.ring), vup);            // which is free
        }
        next = open(x.id + step, next_seen);                       // on its way while the pieces are joined
        team_sync();

        // ---- join, and the part's piece or the outputs ----
        auto emit = [&](int e, const Joined& j) {
            const int c = x.tile * C::kCols + e / D, head = x.head * p.group + c;
            if (c >= p.group) return;
            const float inv = j.l > 0.0f ? 1.0f / j.l : 0.0f;
            *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + x.token * a.out_stride_token + head * a.out_stride_head + e % D) =
                make_uint2(kv_round2<T>(j.x.x * inv, j.x.y * inv), kv_round2<T>(j.x.z * inv, j.x.w * inv));
            if (a.lse && e % D == 0) a.lse[(long long)x.token * a.heads + head] = j.l > 0.0f ? (j.m + fast_log2(j.l)) * kLn2 : -INFINITY;
        };
        const int shared = (int)(x.list - p.whole);                // its number among the shared lists
        auto piece_of = [&](int k) { return ws.pieces + ((long long)shared * p.parts + k) * C::kPiece; };
        for (int e = 4 * tt; e < C::kCols * D; e += 4 * kTeamThreads) {
            const Joined j = join_pieces<C, D, false>(e, x.busy, [&](int w) { return reinterpret_cast<const float*>(ring_of(team * kTeam + w)); });
            if (x.parts == 1) {
                emit(e, j);
            } else {
                float* dst = piece_of(x.part);
                *reinterpret_cast<float4*>(dst + e) = j.x;
                if (e % D == 0) {
                    dst[C::kCols * D + e / D] = j.m;
                    dst[C::kCols * (D + 1) + e / D] = j.l;
                }
            }
        }
        if (x.parts > 1) {
            team_sync();
            if (tt == 0) {
                last_part[team] = count_in(ws.count + shared) == x.parts - 1;
                if (last_part[team]) ws.count[shared] = 0;
            }
            team_sync();
            if (last_part[team])
                for (int e = 4 * tt; e < C::kCols * D; e += 4 * kTeamThreads) emit(e, join_pieces<C, D, true>(e, x.parts, piece_of));
        }
        team_sync();                                               // before the rings are filled again
    }
}

}  // namespace b4
