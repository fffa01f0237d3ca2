// b4_kv_attn.cuh -- what the attention kernels over the 4-bit cache share: the
// parameters, a request's extent, and the fp16 operands made from 4-bit codes.
#pragma once

#include "b4_kv.cuh"

namespace b4 {

struct AttnParams {
    KvLayout l;
    const uint8_t* blocks;
    b4_kv_attn a;
    int group;              // query heads that share a kv head
};

constexpr int kChunk = 64;  // tokens that a warp takes at a time; a multiple of every page size

// What a launch needs of request r: its queries' first row and number, its tokens
// (those that the table can hold), and the chunks that any of its queries sees.
struct AttnReq {
    int q0, n, ctx, chunk0, chunks;
};

__device__ __forceinline__ AttnReq attn_request(const AttnParams& p, int r)
{
    const b4_kv_attn& a = p.a;
    AttnReq q;
    q.q0 = max(0, min(__ldg(a.q_starts + r), a.total_q));
    q.n = max(0, min(__ldg(a.q_starts + r + 1), a.total_q) - q.q0);
    q.ctx = max(0, min(__ldg(a.ctx_len + r), a.table_width * p.l.page_size));
    const int begin = a.window > 0 ? max(0, q.ctx - q.n + 1 - a.window) : 0;
    q.chunk0 = begin / kChunk;
    q.chunks = max(1, (q.ctx + kChunk - 1) / kChunk - q.chunk0);   // one even where nothing is seen: zeros are written
    return q;
}

__device__ __forceinline__ float fast_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float fast_log2(float x)
{
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The NF4 levels as fp16 operands.  fp16 has 11 bits, the levels 24: rounded as
// they are, the levels are off by 1.6e-4 of the code book's norm.  Times kNf4Up
// first, all 16 lie near fp16 numbers at once (6.3e-5; found by searching [1, 2) in
// steps of 2^-23), and 1 / kNf4Up goes into a factor that is applied in fp32 anyway.
constexpr float kNf4Up = 1.67766535282135f;

__device__ __forceinline__ uint32_t nf4_pair(uint32_t byte)
{
    const __half lo = __float2half_rn(c_nf4_table[byte & 15] * kNf4Up), hi = __float2half_rn(c_nf4_table[byte >> 4] * kNf4Up);
    return (uint32_t)__half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t a)
{
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}

__device__ __forceinline__ uint32_t pack_half2(float lo, float hi)
{
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^-e as a float, e an exponent field's offset: exact, for |e| <= 126
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

}  // namespace b4
