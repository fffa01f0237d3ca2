// b4_kv_attn.cu -- attention over the 4-bit key/value cache.
#include <cmath>

#include "b4_kv.cuh"

namespace b4 {
namespace {

struct AttnParams {
    KvLayout l;
    const uint8_t* blocks;
    b4_kv_attn a;
};

// The simple form: a warp per (query, head), one key at a time, the softmax's
// maximum and sum running (one pass); lane i holds columns i * D / 32 onward.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256) kv_attn_kernel(const AttnParams p)
{
    constexpr int C = D / 32;
    kv_begin();
    const int lane = threadIdx.x & 31;
    const b4_kv_attn& a = p.a;
    const long long rows = (long long)a.total_q * a.heads;
    for (long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < rows; i += (long long)gridDim.x * 8) {
        const int t = (int)(i / a.heads), h = (int)(i - (long long)t * a.heads), kvh = h / (a.heads / p.l.kv_heads);
        int r = 0;
        while (r < a.n_req - 1 && a.q_starts[r + 1] <= t) ++r;
        if (t < a.q_starts[r] || t >= a.q_starts[r + 1]) continue;
        const int ctx = max(0, min(a.ctx_len[r], a.table_width * p.l.page_size)), n = a.q_starts[r + 1] - a.q_starts[r];
        const int end = a.flags & B4_KV_FULL ? ctx : min(ctx, ctx - n + (t - a.q_starts[r]) + 1);
        const int begin = a.window > 0 ? max(0, end - a.window) : 0;
        const T* q = static_cast<const T*>(a.q) + t * a.q_stride_token + h * a.q_stride_head + lane * C;
        float qf[C], acc[C] = {}, m = -INFINITY, sum = 0.0f;
        for (int j = 0; j < C; ++j) qf[j] = kv_float(q[j]) * a.scale;
        for (int key = begin; key < end; ++key) {
            const int page = a.tables[r * a.table_stride + (key >> p.l.page_shift)], row = key & (p.l.page_size - 1);
            if (page < 0 || page >= p.l.n_pages) continue;
            const uint8_t* block = p.blocks + ((long long)page * p.l.kv_heads + kvh) * p.l.block;
            float s[2], kv[2][C];
            for (int o = 0; o < 2; ++o) {
                const int at = o * p.l.page_size + row;
                const uint8_t* sp = block + p.l.page_size * D;
                s[o] = FMT == B4_KV_INT4 ? __half2float(reinterpret_cast<const __half*>(sp)[at]) : reinterpret_cast<const float*>(sp)[at];
                for (int j = 0; j < C; ++j) {
                    const uint32_t c = block[at * (D / 2) + (lane * C + j) / 2] >> (4 * (j & 1)) & 15;
                    kv[o][j] = FMT == B4_KV_INT4 ? (float)c - 8.0f : c_nf4_table[c];
                }
            }
            float dot = 0.0f;
            for (int j = 0; j < C; ++j) dot = fmaf(qf[j], kv[0][j], dot);
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
            dot *= s[0];
            const float next = fmaxf(m, dot);
            const float keep = next == -INFINITY ? 0.0f : __expf(m - next), w = next == -INFINITY ? 0.0f : __expf(dot - next);
            sum = sum * keep + w;
            for (int j = 0; j < C; ++j) acc[j] = acc[j] * keep + w * s[1] * kv[1][j];
            m = next;
        }
        const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
        T* out = static_cast<T*>(a.out) + t * a.out_stride_token + h * a.out_stride_head + lane * C;
        for (int j = 0; j < C; ++j) out[j] = kv_round<T>(acc[j] * inv);
        if (a.lse && lane == 0) a.lse[i] = sum > 0.0f ? m + logf(sum) : -INFINITY;
    }
}

template <typename T, int FMT>
cudaError_t attention(const AttnParams& p, cudaStream_t st)
{
    const dim3 grid((unsigned)std::min<long long>(((long long)p.a.total_q * p.a.heads + 7) / 8, 1 << 20));
    return p.l.head_dim == 64 ? kv_launch(kv_attn_kernel<T, FMT, 64>, grid, 256, 0, st, p)
                              : kv_launch(kv_attn_kernel<T, FMT, 128>, grid, 256, 0, st, p);
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
    *bytes = 0;
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
    const bool i4 = p.l.fmt == B4_KV_INT4;
    if (a->dtype == B4_DTYPE_F16) return i4 ? attention<__half, B4_KV_INT4>(p, st) : attention<__half, B4_KV_NF4>(p, st);
    return i4 ? attention<__nv_bfloat16, B4_KV_INT4>(p, st) : attention<__nv_bfloat16, B4_KV_NF4>(p, st);
}

}  // extern "C"
