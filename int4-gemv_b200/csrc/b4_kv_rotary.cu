// b4_kv_rotary.cu -- the quantising append with the rotary embedding of queries and
// keys on the way.
//
// Mathematics.  A position's angle is position * turns mod 2^64, in whole steps of
// 2^-64 turn: exact for any position, so what is rounded is the angle itself (to
// 2^-53 of half a turn), its sine and cosine, and the rotated column, once.  Keys are
// rotated in fp64: their 4-bit codes are then those of the exact rotation but where
// it lies within 2^-50 of a border, whatever computes it, for 2 DFMA a column of a few
// heads; queries, whose rounding to 16 bits is next, in fp32.
//
// Split.  A CTA takes up to 4 tokens: its threads compute the tokens' angles once,
// into shared memory, and its warps share the tokens' vectors (heads of q, k, v),
// 32 * 8 / D of one kind at a time, so that no warp holds two kinds.  The pair's other
// column is in a lane of the same vector, or in the same thread (adjacent pairs).
#include <climits>
#include <cmath>
#include <type_traits>

#include "b4_kv_quant.cuh"

namespace b4 {
namespace {

struct RotaryParams {
    KvLayout l;
    uint8_t* blocks;
    const void* src[3];                // q, k, v
    long long tok[3], head[3];         // their strides
    void* out;
    long long out_tok, out_head;
    const int32_t *positions, *slots;
    long long axis_stride;
    const uint64_t* turns;
    const uint8_t* axes;
    int n, heads, half, adjacent, n_axes;
    int tokens, parts;                 // of a CTA; CTAs that share a token's vectors
    float scale;
};

constexpr int kRotThreads = 256, kRotWarps = kRotThreads / 32, kRotTokens = 4, kRotHalf = 64;

template <typename T, typename O, int FMT, int D, bool VEC>
__global__ void __launch_bounds__(kRotThreads) kv_append_rotary_kernel(const RotaryParams p)
{
    constexpr int TPV = D / 8, VPW = 32 / TPV;         // threads a vector, vectors a warp
    constexpr int U = sizeof(T) == 2 ? 2 : 1;          // items a warp has in flight
    // pair i of a token at [i % 8][i / 8] (adjacent: [i % 4][i / 4]), so that lanes of neighbouring columns read neighbours
    __shared__ double2 turn64[kRotTokens][kRotHalf];
    __shared__ float2 turn32[kRotTokens][kRotHalf];
    float boundary = 4.0f;
    int below = 0;
    if (FMT == B4_KV_NF4) nf4_bins(boundary, below);
    kv_begin();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % TPV;
    const int t0 = blockIdx.x * p.tokens, n = min(p.tokens, p.n - t0);
    const int q_items = (p.heads + VPW - 1) / VPW, kv_items = (p.l.kv_heads + VPW - 1) / VPW, all = q_items + 2 * kv_items;
    const int step = kRotWarps * p.parts, items = n * all;

    struct Item {
        int token, kind, head;
        bool live;
    };
    auto item_of = [&](int i) {
        Item x;
        x.token = i / all;
        int w = i - x.token * all;
        x.kind = w < q_items ? 0 : w < q_items + kv_items ? 1 : 2;
        w -= x.kind == 0 ? 0 : x.kind == 1 ? q_items : q_items + kv_items;
        const int heads = x.kind == 0 ? p.heads : p.l.kv_heads;
        x.head = w * VPW + lane / TPV;
        x.live = x.head < heads;
        x.head = min(x.head, heads - 1);               // whole warps take part in the shuffles
        return x;
    };
    auto load = [&](const Item& x, Columns<T, VEC>& c) {
        c.load(static_cast<const T*>(p.src[x.kind]) + (t0 + x.token) * p.tok[x.kind] + x.head * p.head[x.kind] + sub * 8);
    };
    Item item[U];
    Columns<T, VEC> c[U];
    int at = warp * p.parts + blockIdx.y;              // asked for before the angles are computed
#pragma unroll
    for (int u = 0; u < U; ++u)
        if (at + u * step < items) {
            item[u] = item_of(at + u * step);
            load(item[u], c[u]);
        }

    const int per = p.adjacent ? 4 : 8;
    for (int e = threadIdx.x; e < n * p.half; e += kRotThreads) {
        const int token = e / p.half, i = e - token * p.half;
        const int axis = p.axes ? min((int)__ldg(p.axes + i), p.n_axes - 1) : 0;
        const long long pos = __ldg(p.positions + axis * p.axis_stride + t0 + token);
        const uint64_t phase = (uint64_t)pos * __ldg(reinterpret_cast<const unsigned long long*>(p.turns) + i);
        double s, co;
        sincospi((double)(int64_t)phase * 0x1p-63, &s, &co);
        s *= p.scale;
        co *= p.scale;
        const int place = i % per * (kRotHalf / 8) * (8 / per) + i / per;
        turn64[token][place] = make_double2(co, s);
        turn32[token][place] = make_float2((float)co, (float)s);
    }
    __syncthreads();

    // this lane's pairs: halves, h8 lanes hold the first columns and the next h8 the second; adjacent, four pairs a lane
    const int h8 = p.half / 8;
    const bool turns = sub < 2 * h8, second = !p.adjacent && sub >= h8;
    const int other = lane + (p.adjacent || !turns ? 0 : second ? -h8 : h8);
    const int block = p.adjacent ? sub : second ? sub - h8 : sub;

    for (; at < items; at += U * step) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at + u * step >= items) break;
            const Item x = item[u];
            float v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = c[u].get(j);
            if (x.kind < 2) {
                float w[8];                            // the pairs' other columns
                if (!p.adjacent) {
                    Columns<T, VEC> o;
#pragma unroll
                    for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
                        o.raw[i].x = __shfl_sync(0xffffffffu, c[u].raw[i].x, other);
                        o.raw[i].y = __shfl_sync(0xffffffffu, c[u].raw[i].y, other);
                        o.raw[i].z = __shfl_sync(0xffffffffu, c[u].raw[i].z, other);
                        o.raw[i].w = __shfl_sync(0xffffffffu, c[u].raw[i].w, other);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = o.get(j);
                }
                if (x.kind == 0 && turns) {
                    if (p.adjacent) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float2 t = turn32[x.token][j * 16 + block];
                            const float a = v[2 * j], b = v[2 * j + 1];
                            v[2 * j] = a * t.x - b * t.y;
                            v[2 * j + 1] = b * t.x + a * t.y;
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float2 t = turn32[x.token][j * 8 + block];
                            v[j] = v[j] * t.x + w[j] * (second ? t.y : -t.y);
                        }
                    }
                }
                if (x.kind == 1 && turns) {
                    if (p.adjacent) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const double2 t = turn64[x.token][j * 16 + block];
                            const double a = v[2 * j], b = v[2 * j + 1];
                            v[2 * j] = (float)(a * t.x - b * t.y);
                            v[2 * j + 1] = (float)(b * t.x + a * t.y);
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const double2 t = turn64[x.token][j * 8 + block];
                            v[j] = (float)((double)v[j] * t.x + (double)w[j] * (second ? t.y : -t.y));
                        }
                    }
                }
            }
            const int token = t0 + x.token;
            if (x.kind == 0) {
                if (x.live) {
                    O* dst = static_cast<O*>(p.out) + token * p.out_tok + x.head * p.out_head + sub * 8;
                    *reinterpret_cast<uint4*>(dst) = make_uint4(kv_round2<O>(v[0], v[1]), kv_round2<O>(v[2], v[3]), kv_round2<O>(v[4], v[5]),
                                                                kv_round2<O>(v[6], v[7]));
                }
            } else {
                float scale;
                __half sh;
                const uint32_t w = quantised_word<FMT, TPV>(v, boundary, below, scale, sh);
                const int slot = __ldg(p.slots + token), page = slot >> p.l.page_shift;
                if (x.live && slot >= 0 && page < p.l.n_pages) {
                    uint8_t* b = p.blocks + ((long long)page * p.l.kv_heads + x.head) * p.l.block;
                    const int row = (x.kind == 2 ? p.l.page_size : 0) + (slot & (p.l.page_size - 1));
                    reinterpret_cast<uint32_t*>(b + row * (D / 2))[sub] = w;
                    if (sub == 0) {
                        if (FMT == B4_KV_INT4) reinterpret_cast<__half*>(b + p.l.page_size * D)[row] = sh;
                        else reinterpret_cast<float*>(b + p.l.page_size * D)[row] = scale;
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int next = at + (U + u) * step;
            if (next < items) {
                item[u] = item_of(next);
                load(item[u], c[u]);
            }
        }
    }
}

template <typename T, typename O, int FMT, int D>
cudaError_t launch(RotaryParams p, bool vec, cudaStream_t st)
{
    constexpr int VPW = 256 / D;
    const int all = (p.heads + VPW - 1) / VPW + 2 * ((p.l.kv_heads + VPW - 1) / VPW);
    // few tokens: a token's vectors over as many CTAs as give each warp one; many: four tokens a CTA, their angles by one
    // pass of its threads
    const bool few = p.n < 148 * kRotTokens;
    p.tokens = few ? 1 : kRotTokens;
    p.parts = few ? std::max(1, std::min((all + kRotWarps - 1) / kRotWarps, 148 * 8 / p.n)) : 1;
    const dim3 grid((unsigned)((p.n + p.tokens - 1) / p.tokens), (unsigned)p.parts);
    return vec ? kv_launch(kv_append_rotary_kernel<T, O, FMT, D, true>, grid, kRotThreads, 0, st, p)
               : kv_launch(kv_append_rotary_kernel<T, O, FMT, D, false>, grid, kRotThreads, 0, st, p);
}

template <typename T, typename O>
cudaError_t launch(const RotaryParams& p, bool vec, cudaStream_t st)
{
    if (p.l.fmt == B4_KV_INT4) return p.l.head_dim == 64 ? launch<T, O, B4_KV_INT4, 64>(p, vec, st) : launch<T, O, B4_KV_INT4, 128>(p, vec, st);
    return p.l.head_dim == 64 ? launch<T, O, B4_KV_NF4, 64>(p, vec, st) : launch<T, O, B4_KV_NF4, 128>(p, vec, st);
}

}  // namespace
}  // namespace b4

using namespace b4;

extern "C" {

int b4_rotary_turns(const double* inv_freq, int n, uint64_t* turns)
{
    if (n < 0 || (n > 0 && (!inv_freq || !turns))) return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i)
        if (!std::isfinite(inv_freq[i])) return cudaErrorInvalidValue;
    for (int i = 0; i < n; ++i) {
        const double f = std::fabs(inv_freq[i] / 6.283185307179586476925287), part = f - std::floor(f);
        // 64 bits of the part: the upper 32, then what they leave, rounded; all else is exact
        const double hi = std::floor(part * 0x1p32), lo = std::nearbyint((part * 0x1p32 - hi) * 0x1p32);
        const uint64_t t = ((uint64_t)hi << 32) + (uint64_t)lo;
        turns[i] = inv_freq[i] < 0.0 ? 0 - t : t;
    }
    return cudaSuccess;
}

int b4_kv_append_rotary(const b4_kv_cache* cache, const b4_rotary* r, const b4_kv_rows* x, b4_stream_t stream)
{
    RotaryParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (!r || !x || x->n_tokens < 0 || x->heads < 0 || x->heads > 65536) return cudaErrorInvalidValue;
    if (r->dim < 16 || r->dim % 16 || r->dim > cache->head_dim || r->n_axes < 1 || r->n_axes > 256 || (r->flags & ~B4_ROTARY_ADJACENT) ||
        !std::isfinite(r->scale))
        return cudaErrorInvalidValue;
    if (x->dtype < B4_DTYPE_F16 || x->dtype > B4_DTYPE_F32) return cudaErrorInvalidValue;
    if (x->out_dtype != B4_DTYPE_F16 && x->out_dtype != B4_DTYPE_BF16) return cudaErrorInvalidValue;
    if (x->dtype != B4_DTYPE_F32 && x->dtype != x->out_dtype) return cudaErrorInvalidValue;
    if (x->n_tokens == 0) return cudaSuccess;
    const unsigned item = x->dtype == B4_DTYPE_F32 ? 4 : 2;
    if (!x->k || !x->v || !x->slots || !x->positions || !r->turns || (x->heads > 0 && (!x->q || !x->q_out))) return cudaErrorInvalidValue;
    if (!kv_aligned(x->k, item) || !kv_aligned(x->v, item) || !kv_aligned(x->slots, 4) || !kv_aligned(x->positions, 4) || !kv_aligned(r->turns, 8))
        return cudaErrorInvalidValue;
    if (x->heads > 0 && (!kv_aligned(x->q, item) || !kv_aligned(x->q_out, 16) || (x->out_stride_token | x->out_stride_head) % 8 != 0))
        return cudaErrorInvalidValue;
    if (r->n_axes > 1 && (!r->axes || x->position_stride < x->n_tokens)) return cudaErrorInvalidValue;
    p.blocks = static_cast<uint8_t*>(cache->blocks);
    p.src[0] = x->q;
    p.src[1] = x->k;
    p.src[2] = x->v;
    p.tok[0] = x->q_stride_token;
    p.tok[1] = x->k_stride_token;
    p.tok[2] = x->v_stride_token;
    p.head[0] = x->q_stride_head;
    p.head[1] = x->k_stride_head;
    p.head[2] = x->v_stride_head;
    p.out = x->q_out;
    p.out_tok = x->out_stride_token;
    p.out_head = x->out_stride_head;
    p.positions = x->positions;
    p.slots = x->slots;
    p.axis_stride = x->position_stride;
    p.turns = r->turns;
    p.axes = r->axes;
    p.n = x->n_tokens;
    p.heads = x->heads;
    p.half = r->dim / 2;
    p.n_axes = r->n_axes;
    p.adjacent = r->flags & B4_ROTARY_ADJACENT;
    p.scale = r->scale;
    long long strides = p.tok[1] | p.head[1] | p.tok[2] | p.head[2];
    bool vec = kv_aligned(x->k, 16) && kv_aligned(x->v, 16);
    if (x->heads > 0) {
        strides |= p.tok[0] | p.head[0];
        vec = vec && kv_aligned(x->q, 16);
    }
    vec = vec && strides * (long long)item % 16 == 0;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (x->dtype == B4_DTYPE_F16) return launch<__half, __half>(p, vec, st);
    if (x->dtype == B4_DTYPE_BF16) return launch<__nv_bfloat16, __nv_bfloat16>(p, vec, st);
    return x->out_dtype == B4_DTYPE_F16 ? launch<float, __half>(p, vec, st) : launch<float, __nv_bfloat16>(p, vec, st);
}

}  // extern "C"
