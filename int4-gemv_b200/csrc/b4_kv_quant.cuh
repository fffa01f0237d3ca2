// b4_kv_quant.cuh -- the cache's quantisers: a packed word of codes from 8 columns,
// shared by the kernels that write pages.
#pragma once

#include "b4_kv.cuh"

namespace b4 {

// (int)lround(q) + 8, clamped, as the weight quantiser rounds (half away from zero;
// a quotient that is no number or beyond long becomes code 8)
__device__ __forceinline__ int int4_code(float q)
{
    if (!(fabsf(q) < 0x1p63f)) return 8;
    return (int)min(15LL, max(0LL, llroundf(q) + 8));
}

// the first of the 16 levels at the least fp32 distance, as the weight quantiser scans
__device__ __forceinline__ int nf4_code(float norm)
{
    int best = 0;
    float bd = fabsf(__fsub_rn(norm, c_nf4_table[0]));
#pragma unroll
    for (int c = 1; c < 16; ++c) {
        const float d = fabsf(__fsub_rn(norm, c_nf4_table[c]));
        if (d < bd) {
            bd = d;
            best = c;
        }
    }
    return best;
}

// 8 columns of T as loaded, and as fp32
template <typename T, bool VEC>
struct Columns {
    uint4 raw[sizeof(T) / 2];
    __device__ void load(const T* p)
    {
        if (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
        } else {
            T* r = reinterpret_cast<T*>(raw);
#pragma unroll
            for (int i = 0; i < 8; ++i) r[i] = p[i];
        }
    }
    __device__ float get(int i) const { return kv_float(reinterpret_cast<const T*>(raw)[i]); }
};

// One packed word of INT4 codes.  The quotient by a product with the reciprocal is
// within 2 ulp of the fp32 division that defines the code, so a code is taken from
// it where it lies further than 1e-5 from a tie; the rest, and scales that are no
// normal fp16 number (there a quotient may pass 8), are divided.
__device__ __forceinline__ uint32_t int4_word(const float (&x)[8], float s)
{
    const float inv = __fdividef(1.0f, s);
    uint32_t w = 0;
    float worst = 0.0f, nans = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float y = x[j] * inv, r = y + 12582912.0f;           // 1.5 * 2^23: the integer nearest to y in the low bits
        worst = fmaxf(worst, fabsf(y - (r - 12582912.0f)));
        w |= (__float_as_uint(r) & 15u) << (4 * j);
        nans = fmaf(y, 0.0f, nans);
    }
    if (worst < 0.49999f && nans == 0.0f && s >= 6.1035156e-5f && s <= 65504.0f) return w ^ 0x88888888u;   // two's complement to code - 8
    w = 0;
#pragma unroll 1
    for (int j = 0; j < 8; ++j) w |= (uint32_t)int4_code(__fdiv_rn(x[j], s)) << (4 * j);
    return w;
}

// One packed word of NF4 codes.  [-1, 1] is cut into 31 bins of 1 / kBins with one boundary
// between two levels at most; lane b holds bin b's boundary and the level below it
// (codes below the boundary), so a code is a product, two shuffles and a
// comparison instead of a scan of 16 levels.  Quotients within 1e-6 of a boundary
// (and NaN) are divided and scanned as the definition says.
constexpr float kBins = 15.2f;         // less than the least distance between two boundaries; none lies at a bin's edge

__device__ __forceinline__ uint32_t nf4_word(const float (&x)[8], float s, float boundary, int below)
{
    const float inv = __fdividef(1.0f, s);
    uint32_t w = 0;
    float worst = 1.0f, nans = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float y = x[j] * inv;
        const int bin = (int)__float_as_uint(fmaf(y, kBins, 8388608.0f + 16.0f));          // low 5 bits: 16 + the integer nearest to kBins y
        const float d = y - __shfl_sync(0xffffffffu, boundary, bin);
        const int c = __shfl_sync(0xffffffffu, below, bin) + (d >= 0.0f);
        worst = fminf(worst, fabsf(d));
        nans = fmaf(y, 0.0f, nans);
        w |= (uint32_t)c << (4 * j);
    }
    if (worst > 1e-6f && nans == 0.0f && s > 1e-30f && s < 1e30f) return w;
    w = 0;
#pragma unroll 1
    for (int j = 0; j < 8; ++j) w |= (uint32_t)nf4_code(__fdiv_rn(x[j], s)) << (4 * j);
    return w;
}

// Lane b's part of nf4_word's table: bin b's boundary and the level below it.  By whole warps.
__device__ __forceinline__ void nf4_bins(float& boundary, int& below)
{
    const int lane = threadIdx.x & 31;
    const float start = (lane - 16.5f) / kBins, end = (lane - 15.5f) / kBins;
    // lane c: the boundary above level c; then the first at `start` or above by bisection
    const float level = c_nf4_table[lane & 15], above = __shfl_down_sync(0xffffffffu, level, 1);
    const float mid = lane < 15 ? 0.5f * (level + above) : INFINITY;
    boundary = 4.0f;
    below = 0;
#pragma unroll
    for (int step = 8; step > 0; step >>= 1)
        if (__shfl_sync(0xffffffffu, mid, below + step - 1) < start) below += step;
    const float next = __shfl_sync(0xffffffffu, mid, below);
    if (next < end) boundary = next;
}

// The word and the scale of 8 columns of a vector that TPV neighbouring lanes hold; returns the scale as the value
// that the codes are multiples of (`sh`: its fp16 form, INT4).
template <int FMT, int TPV>
__device__ __forceinline__ uint32_t quantised_word(const float (&x)[8], float boundary, int below, float& scale, __half& sh)
{
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
    for (int o = TPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (FMT == B4_KV_INT4) {
        // times fp32's 1/7 as torch divides by a number on the GPU: pages written by such a program have these bytes
        sh = __float2half_rn(amax > 0.0f ? __fmul_rn(amax, 1.0f / 7.0f) : 1.0f);
        scale = __half2float(sh);
        return int4_word(x, scale);
    }
    scale = amax > 0.0f ? amax : 1.0f;
    return nf4_word(x, scale, boundary, below);
}

}  // namespace b4
