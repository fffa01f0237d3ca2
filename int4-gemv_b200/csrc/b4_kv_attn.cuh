// b4_kv_attn.cuh -- what the attention kernels over the 4-bit cache share: the
// parameters, a request's extent, and the fp16 operands made from 4-bit codes.
#pragma once

#include <type_traits>

#include "b4_kv.cuh"

namespace b4 {

struct AttnParams {
    KvLayout l;
    const uint8_t* blocks;
    b4_kv_attn a;
    int group;              // query heads that share a kv head
    int rows_above;         // the tile kernel takes requests of more rows (queries x group) than this, the warp kernel
    int rows_upto;          // those of at most this many
};

constexpr int kChunk = 32;  // tokens that a warp takes at a time: one page of 32, two of 16, half of one of 64

// What a launch needs of request r: its queries' first row and number, its tokens,
// which place the queries, and the chunks that any of its queries sees.
struct AttnReq {
    int q0, n, ctx, chunk0, chunks;
};

// The tokens that the table can hold: whole pages, so that those past it are masked as missing pages are.
__device__ __forceinline__ int attn_held(const AttnParams& p, int ctx) { return min(ctx, p.a.table_width * p.l.page_size); }

__device__ __forceinline__ int attn_first_chunk(const b4_kv_attn& a, int ctx, int n)
{
    return a.window > 0 ? max(0, ctx - n + 1 - a.window) / kChunk : 0;
}

__device__ __forceinline__ AttnReq attn_extent(const AttnParams& p, int q0, int n, int ctx)
{
    AttnReq q = {q0, n, ctx, attn_first_chunk(p.a, ctx, n), 1};
    q.chunks = max(1, (attn_held(p, ctx) + kChunk - 1) / kChunk - q.chunk0);      // one even where nothing is seen: zeros are written
    return q;
}

__device__ __forceinline__ AttnReq attn_request(const AttnParams& p, int r)
{
    const b4_kv_attn& a = p.a;
    const int q0 = __ldg(a.q_starts + r), q1 = __ldg(a.q_starts + r + 1), ctx = __ldg(a.ctx_len + r);
    const int from = max(0, min(q0, a.total_q));
    return attn_extent(p, from, max(0, min(q1, a.total_q) - from), max(0, ctx));
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

// a / b, a >= 0, b > 0; in 32 bits where both fit
__device__ __forceinline__ long long div64(long long a, long long b)
{
    return ((a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ uint32_t lds32(uint32_t at)
{
    uint32_t v;
    asm("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at));
    return v;
}

__device__ __forceinline__ uint2 lds64(uint32_t at)
{
    uint2 v;
    asm("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}

// 16 bytes from global memory to a shared address, past L1
__device__ __forceinline__ void copy_async16(uint32_t dst, const void* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Counts in at a segment that crosses CTAs: after it, what the CTAs that counted in before wrote is there.  By one thread,
// behind a barrier that puts its CTA's writes before it.
__device__ __forceinline__ int count_in(int* at)
{
    int n;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(n) : "l"(at) : "memory");
    return n;
}

// A maximum that no score has set yet: finite, so that differences with it are.
constexpr float kNoMax = -1e30f;

// A weight times a value scale goes to fp16 relative to the row's running maximum, which weights pass by 2^8 at most, and to
// 2^e, the least power above the value scales so far (kNoExp: none yet), times 2^kLift: below 2^15, so that fp16 holds its
// 11 bits down to 2^-21 of the largest weight times 2^e, and 2^-32 of it below that.
constexpr int kLift = 7, kNoExp = kLift - 126;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// The NF4 levels as fp16 operands.  fp16 has 11 bits, the levels 24: rounded as
// they are, the levels are off by 1.6e-4 of the code book's norm.  Times a factor in
// [1, 2) first, all 16 lie nearer to fp16 numbers, and its reciprocal goes into a
// factor that is applied in fp32 anyway.  kNf4Least leaves the least, 3.3e-5 in the mean
// square (6.3e-5 at most): where a low part follows (fp16 queries), which makes the levels
// exact to 2^-22.  kNf4Even, where none does (bf16), is off by 4e-5 in the mean square and
// by 9.3e-5 of a scale at most, whatever the codes; since a value's rounding is the same
// for every token of its code and does not average out, it is the factor, of 20 million,
// whose roundings sum to the least over codes as normal values and every code alike give
// them: 4e-7 to 1.1e-6 of a scale (kNf4Least: 1.1e-5).  Laplace values leave 4.7e-6,
// exponential ones 1.2e-5, 0.2 % of an output over 4000 tokens, which is bf16's own rounding.
constexpr float kNf4Least = 1.67766535282135f, kNf4Even = 1.6775788f;

__device__ __forceinline__ uint32_t nf4_pair(uint32_t byte, float up)
{
    const __half lo = __float2half_rn(c_nf4_table[byte & 15] * up), hi = __float2half_rn(c_nf4_table[byte >> 4] * up);
    return (uint32_t)__half_as_ushort(lo) | ((uint32_t)__half_as_ushort(hi) << 16);
}

// What the fp16 parts of nf4_pair leave of the levels: with it they are exact to 2^-22.
__device__ __forceinline__ uint32_t nf4_pair_low(uint32_t byte, float up)
{
    const float a = c_nf4_table[byte & 15] * up, b = c_nf4_table[byte >> 4] * up;
    const __half lo = __float2half_rn(a - __half2float(__float2half_rn(a))), hi = __float2half_rn(b - __half2float(__float2half_rn(b)));
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

// 2^e, |e| <= 126
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// W words of 8 query columns as fp16, negated where `negate`; the four lanes of a
// row (lane & ~3) hold it together.  Returns what a product with them lacks: 1, or
// for bf16 the power of two that was taken out of the row.
template <typename T, int W>
__device__ __forceinline__ float query_operand(uint4 (&v)[W], bool negate)
{
    float factor = 1.0f;
    const uint32_t sign = negate ? 0x80008000u : 0u;
    if (std::is_same<T, __nv_bfloat16>::value) {
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const uint32_t x[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, max(x[j] << 16 & 0x7fffffffu, x[j] & 0x7fff0000u));
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(top >> 23) - 127, -110), 126);
        const float up = pow2(10 - e);
        factor = pow2(e - 10);
#pragma unroll
        for (int i = 0; i < W; ++i) {
            uint32_t* x = reinterpret_cast<uint32_t*>(&v[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                x[j] = pack_half2(__uint_as_float(x[j] << 16) * up, __uint_as_float(x[j] & 0xffff0000u) * up);
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = make_uint4(v[i].x ^ sign, v[i].y ^ sign, v[i].z ^ sign, v[i].w ^ sign);
    return factor;
}

}  // namespace b4
