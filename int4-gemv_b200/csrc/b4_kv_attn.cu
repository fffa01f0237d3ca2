// b4_kv_attn.cu -- attention over the 4-bit key/value cache.
#include <climits>
#include <cmath>

#include "b4_kv_attn_lists.cuh"
#include "b4_kv_attn_tile.cuh"
#include "b4_kv_attn_warp.cuh"
#include "b4_kv_overlap.h"

namespace b4 {
namespace {

int sm_count()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    return n;
}

// Which kernels run.  The warp kernel takes requests of few rows (queries x heads that
// share a kv head), in tiles of 8 or 16 that each read the cache, the tile kernel the
// others, whose time does not depend on the rows up to 128.  24 requests of 4000 tokens
// (INT4 in fp16, NF4 in bf16, NF4 in fp16): 4 kv heads x 128, 48 rows 67, 71 and 100 us
// against 69, 85 and 120, 64 rows 83, 87 and 125 against 69, 85 and 121; 8 kv heads x 64,
// 64 rows 83, 87 and 118 us against 96, 118 and 169, 80 rows 101, 105 and 144 against 96,
// 118 and 169.  So the warp kernel has up to 48 rows of 128, 64 of 64.
// max_q says which of the two the call needs: one where every request is of one
// kind by it, both (each skipping the other's requests) where it cannot be known.  In
// a call for both the warp kernel takes the smallest tile's rows alone: with tiles of 16
// and up to 48 rows, 31 single tokens behind 4000 and a chunk of 512 behind 2000 take
// 103 us for 87, 24 x 5 drafts and the chunk 127 for 110 (28 heads over 4 x 128, INT4).
struct Plan {
    bool warp, tile;
    int cols;               // the warp kernel's tile: 8 or 16 columns
    int above, upto;
};

Plan plan(const AttnParams& p)
{
    const long long most = (long long)std::max(1, p.a.max_q) * p.group;
    if (most <= (p.l.head_dim == 64 ? 64 : 48)) return {true, false, most <= 8 ? 8 : 16, INT_MAX, INT_MAX};
    if ((long long)p.a.n_req * p.a.max_q <= p.a.total_q || p.group > 16) return {false, true, 0, 0, 0};    // alike, or none of few rows
    const int cols = p.group <= 8 ? 8 : 16;
    return {true, true, cols, cols, cols};
}

// Workspace: the kernels' counters, then the pieces of the one that runs ([CTA][warp] first, [CTA][2] crossing; [CTA][2]
// crossing; lists: one for each team of warps), one CTA an SM.
constexpr int kMaxWarps = 16, kCounters = 4096, kListTeams = 4;
size_t ws_bytes_of(const AttnParams& p, int sms)
{
    const size_t row = (size_t)(p.l.head_dim + 2) * 4;
    if (p.lists) return 2 * kCounters + (size_t)(kListTeams * sms) * (p.group <= 8 ? 8 : 16) * row;
    const Plan w = plan(p);
    const size_t warp = w.warp ? (kMaxWarps + 2) * w.cols * row : 0, tile = w.tile ? 2 * kTileRows * row : 0;
    return 2 * kCounters + (size_t)sms * std::max(warp, tile);
}

template <typename T, int FMT, int D, int NT, int PT>
cudaError_t launch_warp(const AttnParams& p, void* ws, cudaStream_t st)
{
    using C = WarpCfg<FMT, D, NT, PT>;
    auto fn = kv_attn_warp_kernel<T, FMT, D, NT, PT>;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    const int sms = sm_count();
    WarpWs w;
    w.count = static_cast<int*>(ws);
    w.first = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 2 * kCounters);
    w.cross = w.first + (size_t)sms * C::kWarps * C::kPiece;
    return kv_launch(fn, dim3((unsigned)sms), C::kThreads, C::kSmem, st, p, w);
}

// How lists go to the teams of warps of every SM's CTA: whole ones round by round, each of those left for the last to as many
// teams as bring its time down; two teams or four, whichever takes less.  Times in hundreds of cycles as a profile has them:
// a chunk 20 where a warp has its scheduler for itself, 32 where four share it, a list's beginning and end 57, the join of
// several teams 30.  64 heads over 8 x 128, INT4, pages of 64: 8 lists of 64 pages take 10.5 us with two teams, 19.3 with
// four, 192 37.3 and 32.6, 256 of 32 22.7 and 26.7; 3200 of 16 (32 heads over 8 x 64) 82 and 69.
struct ListPlan {
    long long whole;
    int parts;
    double time;
};

ListPlan list_plan(long long lists, int teams, int chunks, int warps)
{
    const long long rounds = lists / teams;
    ListPlan best = {rounds * teams, 1, 0.0};
    const int rest = (int)(lists - best.whole);
    double least = 0.0;
    for (int n = 1; rest > 0 && n <= std::min((chunks + warps - 1) / warps, teams / rest); ++n) {
        const double each = (chunks + n * warps - 1) / (n * warps), time = each * (20.0 + 12.0 * rest * n / teams) + 57.0 + (n > 1 ? 30.0 : 0.0);
        if (n == 1 || time < least) {
            least = time;
            best.parts = n;
        }
    }
    best.time = rounds * ((chunks + warps - 1) / warps * 32.0 + 57.0) + least;
    return best;
}

template <typename T, int FMT, int D, int NT, int PT, int TEAMS>
cudaError_t launch_teams(AttnParams p, const ListPlan& plan, long long lists, int sms, void* ws, cudaStream_t st)
{
    using C = WarpCfg<FMT, D, NT, PT>;
    auto fn = kv_attn_lists_kernel<T, FMT, D, NT, PT, TEAMS>;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    p.whole = plan.whole;
    p.parts = plan.parts;
    ListWs w;
    w.count = static_cast<int*>(ws);
    w.pieces = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 2 * kCounters);
    return kv_launch(fn, dim3((unsigned)std::min<long long>(sms, p.whole + (lists - p.whole) * p.parts)), C::kThreads, C::kSmem, st, p, w);
}

template <typename T, int FMT, int D, int NT, int PT>
cudaError_t launch_lists(const AttnParams& p, void* ws, cudaStream_t st)
{
    constexpr int kWarps = WarpCfg<FMT, D, NT, PT>::kWarps;
    const int sms = sm_count();
    const long long lists = (long long)p.a.total_q * p.l.kv_heads * ((p.group + 8 * NT - 1) / (8 * NT));
    const int chunks = (int)std::min<long long>(std::max(1LL, ((long long)p.a.table_width * p.l.page_size + kChunk - 1) / kChunk), 1 << 20);
    const ListPlan two = list_plan(lists, 2 * sms, chunks, kWarps / 2), four = list_plan(lists, kListTeams * sms, chunks, kWarps / kListTeams);
    return four.time < two.time ? launch_teams<T, FMT, D, NT, PT, kListTeams>(p, four, lists, sms, ws, st)
                                : launch_teams<T, FMT, D, NT, PT, 2>(p, two, lists, sms, ws, st);
}

template <typename T, int FMT, int D>
cudaError_t launch_tile(const AttnParams& p, void* ws, cudaStream_t st)
{
    using C = TileCfg<T, FMT, D>;
    auto fn = kv_attn_tile_kernel<T, FMT, D>;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    TileWs w;
    w.count = reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + kCounters);
    w.cross = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 2 * kCounters);
    return kv_launch(fn, dim3((unsigned)sm_count()), kTileThreads, C::kSmem, st, p, w);
}

template <typename T, int FMT, int D>
cudaError_t launch(AttnParams p, void* ws, cudaStream_t st)
{
    if (p.lists) {
        if (p.l.page_size == 16) return p.group <= 8 ? launch_lists<T, FMT, D, 1, 16>(p, ws, st) : launch_lists<T, FMT, D, 2, 16>(p, ws, st);
        return p.group <= 8 ? launch_lists<T, FMT, D, 1, 32>(p, ws, st) : launch_lists<T, FMT, D, 2, 32>(p, ws, st);
    }
    const Plan w = plan(p);
    p.rows_above = w.above;
    p.rows_upto = w.upto;
    cudaError_t e = cudaSuccess;
    if (w.tile) e = launch_tile<T, FMT, D>(p, ws, st);
    if (w.warp && e == cudaSuccess) {
        if (p.l.page_size == 16) return w.cols == 8 ? launch_warp<T, FMT, D, 1, 16>(p, ws, st) : launch_warp<T, FMT, D, 2, 16>(p, ws, st);
        return w.cols == 8 ? launch_warp<T, FMT, D, 1, 32>(p, ws, st) : launch_warp<T, FMT, D, 2, 32>(p, ws, st);
    }
    return e;
}

template <typename T>
cudaError_t attention(const AttnParams& p, void* ws, cudaStream_t st)
{
    if (p.l.fmt == B4_KV_INT4) return p.l.head_dim == 64 ? launch<T, B4_KV_INT4, 64>(p, ws, st) : launch<T, B4_KV_INT4, 128>(p, ws, st);
    return p.l.head_dim == 64 ? launch<T, B4_KV_NF4, 64>(p, ws, st) : launch<T, B4_KV_NF4, 128>(p, ws, st);
}

int attn_params(const b4_kv_cache* cache, const b4_kv_attn* a, AttnParams* p)
{
    const int e = kv_layout(cache, &p->l);
    if (e != cudaSuccess) return e;
    if (!a || a->n_req < 0 || a->total_q < 0 || a->max_q < 0 || a->table_width < 0 || a->window < 0) return cudaErrorInvalidValue;
    if (a->heads < 1 || a->heads % p->l.kv_heads || a->heads / p->l.kv_heads > 64) return cudaErrorInvalidValue;
    if ((long long)a->total_q * (a->heads / p->l.kv_heads) > 0x7fffffffLL) return cudaErrorInvalidValue;
    if (a->dtype != B4_DTYPE_F16 && a->dtype != B4_DTYPE_BF16) return cudaErrorInvalidValue;
    if (a->flags & ~B4_KV_FULL || (a->flags & B4_KV_FULL && a->window > 0) || !std::isfinite(a->scale)) return cudaErrorInvalidValue;
    // the kernels count up to a block of 64 keys past a request's last
    if (a->table_stride < a->table_width || (long long)a->table_width * p->l.page_size > 0x80000000LL - 64) return cudaErrorInvalidValue;
    p->blocks = static_cast<const uint8_t*>(cache->blocks);
    p->a = *a;
    p->a.window = std::min(a->window, INT_MAX - a->total_q);       // a query's place, ctx - n + i + 1 > -total_q, less it fits an int
    p->group = a->heads / p->l.kv_heads;
    p->lists = false;
    p->parts = 1;
    p->whole = 0;
    p->list_head = 0;
    return cudaSuccess;
}

// a query's own lists: each query is a request of one
int list_params(const b4_kv_cache* cache, const b4_kv_attn* attn, AttnParams* p)
{
    if (!attn || attn->window != 0 || attn->flags != 0) return cudaErrorInvalidValue;
    b4_kv_attn a = *attn;
    a.n_req = a.total_q;
    a.max_q = 1;
    a.q_starts = nullptr;
    const int e = attn_params(cache, &a, p);
    p->lists = true;
    return e;
}

// outputs on what other teams read, or on one another: a query's own row alone may be where its output goes
bool outputs_in_the_way(const b4_kv_cache* cache, const AttnParams& p)
{
    const b4_kv_attn& a = p.a;
    const long long n = a.total_q, d = p.l.head_dim;
    const RowSet out = row_set(a.out, 2, a.out_stride_token, a.out_stride_head, n, a.heads, d), lse = row_set(a.lse, 4, a.lse ? n * a.heads : 0);
    const RowSet q = row_set(a.q, 2, a.q_stride_token, a.q_stride_head, n, a.heads, d);
    const bool in_place = a.out == a.q && (n == 1 || a.out_stride_token == a.q_stride_token) && (a.heads == 1 || a.out_stride_head == a.q_stride_head);
    if (rows_overlap(out) || rows_meet(out, lse) || (!in_place && rows_meet(out, q)) || rows_meet(lse, q)) return true;
    const RowSet reads[] = {row_set(a.tables, 4, a.table_stride, p.list_head, n, p.l.kv_heads, a.table_width), row_set(a.ctx_len, 4, n),
                            row_set(cache->blocks, p.l.block, (long long)p.l.n_pages * p.l.kv_heads)};
    for (const RowSet& r : reads)
        if (rows_meet(out, r) || rows_meet(lse, r)) return true;
    return false;
}

int attend(const AttnParams& p, void* ws, size_t ws_bytes, b4_stream_t stream)
{
    const b4_kv_attn& a = p.a;
    if (!a.q || !a.out || !a.ctx_len || (p.lists ? a.table_width > 0 && !a.tables : !a.tables || !a.q_starts)) return cudaErrorInvalidValue;
    const long long strides = a.q_stride_token | a.q_stride_head | a.out_stride_token | a.out_stride_head;
    if (!kv_aligned(a.q, 16) || !kv_aligned(a.out, 16) || strides % 8 != 0) return cudaErrorInvalidValue;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (!ws || !kv_aligned(ws, 16) || ws_bytes < ws_bytes_of(p, sm_count())) return cudaErrorInvalidValue;
    return a.dtype == B4_DTYPE_F16 ? attention<__half>(p, ws, st) : attention<__nv_bfloat16>(p, ws, st);
}

}  // namespace
}  // namespace b4

using namespace b4;

int b4::kv_attn_device_error(int clear)
{
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_error, sizeof(v)) != cudaSuccess) return -1;
    if (clear && v) {
        const int z = 0;
        if (cudaMemcpyToSymbol(g_device_error, &z, sizeof(z)) != cudaSuccess) return -1;
    }
    return v;
}

extern "C" {

int b4_kv_attention_workspace(const b4_kv_cache* cache, const b4_kv_attn* a, size_t* bytes)
{
    AttnParams p;
    const int e = attn_params(cache, a, &p);
    if (e != cudaSuccess) return e;
    if (!bytes) return cudaErrorInvalidValue;
    *bytes = a->total_q && a->n_req ? ws_bytes_of(p, sm_count()) : 0;
    return cudaSuccess;
}

int b4_kv_attention(const b4_kv_cache* cache, const b4_kv_attn* a, void* ws, size_t ws_bytes, b4_stream_t stream)
{
    AttnParams p;
    const int e = attn_params(cache, a, &p);
    if (e != cudaSuccess) return e;
    if (a->total_q == 0 || a->n_req == 0) return cudaSuccess;
    return attend(p, ws, ws_bytes, stream);
}

int b4_kv_attention_lists_workspace(const b4_kv_cache* cache, const b4_kv_attn* a, size_t* bytes)
{
    AttnParams p;
    const int e = list_params(cache, a, &p);
    if (e != cudaSuccess) return e;
    if (!bytes) return cudaErrorInvalidValue;
    *bytes = a->total_q ? ws_bytes_of(p, sm_count()) : 0;
    return cudaSuccess;
}

int b4_kv_attention_lists(const b4_kv_cache* cache, const b4_kv_attn* a, long long list_stride_head, void* ws, size_t ws_bytes,
                          b4_stream_t stream)
{
    AttnParams p;
    const int e = list_params(cache, a, &p);
    if (e != cudaSuccess) return e;
    if (list_stride_head < a->table_width) return cudaErrorInvalidValue;
    if (a->total_q == 0) return cudaSuccess;
    p.list_head = list_stride_head;
    if (outputs_in_the_way(cache, p)) return cudaErrorInvalidValue;
    return attend(p, ws, ws_bytes, stream);
}

}  // extern "C"
