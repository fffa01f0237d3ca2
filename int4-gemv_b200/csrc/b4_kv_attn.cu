// b4_kv_attn.cu -- attention over the 4-bit key/value cache.
#include <cmath>

#include "b4_kv_attn_warp.cuh"

namespace b4 {
namespace {

// The least columns (queries x heads that share a kv head) of a tile that hold
// a request's queries, or 16 a tile.
int tile_cols(const AttnParams& p)
{
    const long long cols = (long long)std::max(1, p.a.max_q) * p.group;
    return cols <= 8 ? 8 : 16;
}

int sm_count()
{
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    return n;
}

// [counters][first pieces][crossing pieces], one CTA an SM
constexpr int kMaxWarps = 16;
size_t warp_ws_bytes(const AttnParams& p, int sms)
{
    const size_t piece = (size_t)tile_cols(p) * (p.l.head_dim + 2) * 4;
    return 4096 + (size_t)sms * (kMaxWarps + 2) * piece;
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
    w.first = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + 4096);
    w.cross = w.first + (size_t)sms * C::kWarps * C::kPiece;
    return kv_launch(fn, dim3((unsigned)sms), C::kThreads, C::kSmem, st, p, w);
}

template <typename T, int FMT, int D>
cudaError_t launch_cols(const AttnParams& p, void* ws, cudaStream_t st)
{
    const bool one = tile_cols(p) == 8;
    if (p.l.page_size == 16) return one ? launch_warp<T, FMT, D, 1, 16>(p, ws, st) : launch_warp<T, FMT, D, 2, 16>(p, ws, st);
    return one ? launch_warp<T, FMT, D, 1, 32>(p, ws, st) : launch_warp<T, FMT, D, 2, 32>(p, ws, st);
}

template <typename T>
cudaError_t attention(const AttnParams& p, void* ws, cudaStream_t st)
{
    if (p.l.fmt == B4_KV_INT4) return p.l.head_dim == 64 ? launch_cols<T, B4_KV_INT4, 64>(p, ws, st) : launch_cols<T, B4_KV_INT4, 128>(p, ws, st);
    return p.l.head_dim == 64 ? launch_cols<T, B4_KV_NF4, 64>(p, ws, st) : launch_cols<T, B4_KV_NF4, 128>(p, ws, st);
}

int attn_params(const b4_kv_cache* cache, const b4_kv_attn* a, AttnParams* p)
{
    const int e = kv_layout(cache, &p->l);
    if (e != cudaSuccess) return e;
    if (!a || a->n_req < 0 || a->total_q < 0 || a->max_q < 0 || a->table_width < 0 || a->window < 0) return cudaErrorInvalidValue;
    if (a->heads < 1 || a->heads % p->l.kv_heads || a->heads / p->l.kv_heads > 64) return cudaErrorInvalidValue;
    if (a->dtype != B4_DTYPE_F16 && a->dtype != B4_DTYPE_BF16) return cudaErrorInvalidValue;
    if (a->flags & ~B4_KV_FULL || (a->flags & B4_KV_FULL && a->window > 0) || !std::isfinite(a->scale)) return cudaErrorInvalidValue;
    if (a->table_stride < a->table_width || (long long)a->table_width * p->l.page_size > 0x7fffffffLL) return cudaErrorInvalidValue;
    p->blocks = static_cast<const uint8_t*>(cache->blocks);
    p->a = *a;
    p->group = a->heads / p->l.kv_heads;
    return cudaSuccess;
}

}  // namespace
}  // namespace b4

using namespace b4;

extern "C" {

int b4_kv_attention_workspace(const b4_kv_cache* cache, const b4_kv_attn* a, size_t* bytes)
{
    AttnParams p;
    const int e = attn_params(cache, a, &p);
    if (e != cudaSuccess) return e;
    if (!bytes) return cudaErrorInvalidValue;
    *bytes = a->total_q && a->n_req ? warp_ws_bytes(p, sm_count()) : 0;
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
    if (!ws || !kv_aligned(ws, 16) || ws_bytes < warp_ws_bytes(p, sm_count())) return cudaErrorInvalidValue;
    return a->dtype == B4_DTYPE_F16 ? attention<__half>(p, ws, st) : attention<__nv_bfloat16>(p, ws, st);
}

}  // extern "C"
