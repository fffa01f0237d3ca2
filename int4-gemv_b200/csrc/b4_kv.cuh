// b4_kv.cuh -- the 4-bit key/value cache: block layout and launch helpers shared
// by its kernels.
#pragma once

#include <cuda_bf16.h>

#include "b4_common.cuh"
#include "b4_internal.h"

namespace b4 {

// One kv head's part of a page (include/b4gemv.h): key codes, value codes, key
// scales, value scales.
struct KvLayout {
    int fmt, n_pages, page_size, page_shift, kv_heads, head_dim;
    int code_bytes, scale_bytes;      // of one token
    long long block;                  // bytes of a block
};

__host__ __device__ inline long long kv_block_bytes(int fmt, int page_size, int head_dim)
{
    return 2LL * page_size * (head_dim / 2 + (fmt == B4_KV_INT4 ? 2 : 4));
}

inline bool kv_shape_ok(int fmt, int page_size, int head_dim)
{
    return (fmt == B4_KV_INT4 || fmt == B4_KV_NF4) && (page_size == 16 || page_size == 32 || page_size == 64) &&
           (head_dim == 64 || head_dim == 128);
}

// cudaSuccess, or cudaErrorInvalidValue for a cache that the kernels cannot address
inline int kv_layout(const b4_kv_cache* c, KvLayout* l)
{
    if (!c || !c->blocks || reinterpret_cast<uintptr_t>(c->blocks) % 16 != 0) return cudaErrorInvalidValue;
    if (!kv_shape_ok(c->fmt, c->page_size, c->head_dim) || c->n_pages < 1 || c->kv_heads < 1 || c->kv_heads > 1024)
        return cudaErrorInvalidValue;
    if ((long long)c->n_pages * c->page_size > 0x7fffffffLL) return cudaErrorInvalidValue;
    l->fmt = c->fmt;
    l->n_pages = c->n_pages;
    l->page_size = c->page_size;
    l->page_shift = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : 6;
    l->kv_heads = c->kv_heads;
    l->head_dim = c->head_dim;
    l->code_bytes = c->head_dim / 2;
    l->scale_bytes = c->fmt == B4_KV_INT4 ? 2 : 4;
    l->block = kv_block_bytes(c->fmt, c->page_size, c->head_dim);
    return cudaSuccess;
}

inline bool kv_aligned(const void* p, unsigned a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// Launches a cache kernel as a programmatic dependent: each begins with
// kv_begin(), which lets the next launch start its prologue and then waits for
// the grid before it, so nothing is read or written too early.
template <typename... Params, typename... Args>
cudaError_t kv_launch(void (*fn)(Params...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args... args)
{
    cudaLaunchConfig_t lc = {};
    lc.gridDim = grid;
    lc.blockDim = dim3(threads);
    lc.dynamicSmemBytes = smem;
    lc.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = attr;
    lc.numAttrs = 1;
    return cudaLaunchKernelEx(&lc, fn, Params(args)...);
}

__device__ __forceinline__ void kv_begin()
{
    asm volatile("griddepcontrol.launch_dependents;");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

__device__ __forceinline__ float kv_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float kv_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float kv_float(float v) { return v; }

template <typename T> __device__ __forceinline__ T kv_round(float v);
template <> __device__ __forceinline__ __half kv_round<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 kv_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// two columns as T, packed
template <typename T> __device__ __forceinline__ uint32_t kv_round2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t kv_round2<__half>(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> __device__ __forceinline__ uint32_t kv_round2<__nv_bfloat16>(float lo, float hi)
{
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

}  // namespace b4
