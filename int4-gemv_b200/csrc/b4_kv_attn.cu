// b4_kv_attn.cu -- attention over the 4-bit key/value cache.
#include <climits>
#include <cmath>

#include "b4_kv_attn_tile.cuh"
#include "b4_kv_attn_warp.cuh"

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

// Workspace: the two kernels' counters, then the pieces of the one that runs
// ([CTA][warp] first, [CTA][2] crossing; [CTA][2] crossing), one CTA an SM.
constexpr int kMaxWarps = 16, kCounters = 4096;
size_t ws_bytes_of(const AttnParams& p, int sms)
{
    const Plan w = plan(p);
    const size_t row = (size_t)(p.l.head_dim + 2) * 4;
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
    return cudaSuccess;
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
    if (!a->q || !a->out || !a->tables || !a->ctx_len || !a->q_starts) return cudaErrorInvalidValue;
    const long long strides = a->q_stride_token | a->q_stride_head | a->out_stride_token | a->out_stride_head;
    if (!kv_aligned(a->q, 16) || !kv_aligned(a->out, 16) || strides % 8 != 0) return cudaErrorInvalidValue;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (!ws || !kv_aligned(ws, 16) || ws_bytes < ws_bytes_of(p, sm_count())) return cudaErrorInvalidValue;
    return a->dtype == B4_DTYPE_F16 ? attention<__half>(p, ws, st) : attention<__nv_bfloat16>(p, ws, st);
}

}  // extern "C"
