// b4_kv.cu -- the 4-bit key/value cache's bookkeeping: block tables and slots of a
// scheduling step, the quantising append, and the read-back.
#include <climits>

#include "b4_kv.cuh"

namespace b4 {
namespace {

// ---- block tables, slots, positions ----------------------------------------------
// Every CTA scans the requests' lengths itself (new tokens and new pages, both
// exclusive sums, in shared memory), so there is no second launch and no wait
// between CTAs; then the CTAs share the packed tokens (request found by binary
// search over the scanned starts) and the new table entries.  A slot in a new
// page comes straight from the ring, not through the table, which another CTA
// may still be writing.
constexpr int kTabThreads = 256;

__device__ __forceinline__ int sat(long long v) { return (int)(v > INT_MAX ? INT_MAX : v); }

__device__ __forceinline__ int pages_of(long long tokens, int page_size, int width)
{
    const long long p = (tokens + page_size - 1) / page_size;
    return (int)(p < width ? p : width);
}

struct TabLengths {
    long long cached, added;
    int held, fresh;
};

__device__ __forceinline__ TabLengths tab_lengths(const b4_kv_step& s, int r)
{
    TabLengths l;
    l.cached = max(__ldg(s.cached + r), 0);
    l.added = max(__ldg(s.added + r), 0);
    l.held = pages_of(l.cached, s.page_size, s.table_width);
    l.fresh = pages_of(l.cached + l.added, s.page_size, s.table_width) - l.held;
    return l;
}

__global__ void __launch_bounds__(kTabThreads) kv_tables_kernel(const b4_kv_step s)
{
    extern __shared__ int tab_smem[];
    int* start = tab_smem;                    // [n_req] first token of a request
    int* first = tab_smem + s.n_req;          // [n_req] its first new page, counted from the ring's place
    __shared__ long long warp_tok[kTabThreads / 32], warp_pag[kTabThreads / 32];
    kv_begin();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (s.n_req + kTabThreads - 1) / kTabThreads;
    const int r0 = min((int)threadIdx.x * per, s.n_req), r1 = min(r0 + per, s.n_req);
    long long tok = 0, pag = 0;
    for (int r = r0; r < r1; ++r) {
        const TabLengths l = tab_lengths(s, r);
        tok += l.added;
        pag += l.fresh;
    }
    long long it = tok, ip = pag;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, it, o), b = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) {
            it += a;
            ip += b;
        }
    }
    if (lane == 31) {
        warp_tok[warp] = it;
        warp_pag[warp] = ip;
    }
    __syncthreads();
    long long all_tok = 0, all_pag = 0, bt = it - tok, bp = ip - pag;
#pragma unroll
    for (int w = 0; w < kTabThreads / 32; ++w) {
        if (w < warp) {
            bt += warp_tok[w];
            bp += warp_pag[w];
        }
        all_tok += warp_tok[w];
        all_pag += warp_pag[w];
    }
    const bool writer = blockIdx.x == 0;
    for (int r = r0; r < r1; ++r) {
        const TabLengths l = tab_lengths(s, r);
        start[r] = sat(bt);
        first[r] = sat(bp);
        if (writer) {
            s.ctx_len[r] = sat(l.cached + l.added);
            s.q_starts[r] = sat(bt);
        }
        bt += l.added;
        bp += l.fresh;
    }
    __syncthreads();

    const int head = s.ring_size > 0 ? (int)((unsigned)max(__ldg(s.free_state), 0) % (unsigned)s.ring_size) : 0;
    const int left = min(max(__ldg(s.free_state + 1), 0), s.ring_size);
    if (writer && threadIdx.x == 0) {
        s.q_starts[s.n_req] = sat(all_tok);
        const int taken = (int)(all_pag < left ? all_pag : left);
        s.free_state_out[0] = s.ring_size > 0 ? (int)(((long long)head + taken) % s.ring_size) : 0;
        s.free_state_out[1] = left - taken;
        s.free_state_out[2] = sat(all_pag - taken);
    }
    auto ring = [&](int n) -> int {           // the n-th new page of the step
        if (n >= left) return -1;
        long long at = (long long)head + n;
        if (at >= s.ring_size) at -= s.ring_size;
        return __ldg(s.free_pages + at);
    };

    const int n_tok = sat(all_tok);
    for (long long i = (long long)blockIdx.x * kTabThreads + threadIdx.x; i < s.max_tokens;
         i += (long long)gridDim.x * kTabThreads) {
        int slot = -1, pos = 0;
        if (i < n_tok) {
            int lo = 0, hi = s.n_req;         // the last request that starts at or before i
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= i) lo = mid;
                else hi = mid;
            }
            const long long c = max(__ldg(s.cached + lo), 0), at = c + (i - start[lo]);
            const long long p = at / s.page_size;
            pos = sat(at);
            if (p < s.table_width) {
                const int held = pages_of(c, s.page_size, s.table_width);
                const int id = p < held ? s.tables[lo * s.table_stride + p] : ring(first[lo] + (int)p - held);
                if (id >= 0) slot = id * s.page_size + (int)(at - p * s.page_size);
            }
        }
        s.slots[i] = slot;
        s.positions[i] = pos;
    }
    const int warps = gridDim.x * (kTabThreads / 32);
    for (int r = blockIdx.x * (kTabThreads / 32) + warp; r < s.n_req; r += warps) {
        const TabLengths l = tab_lengths(s, r);
        for (int i = lane; i < l.fresh; i += 32) s.tables[r * s.table_stride + l.held + i] = ring(first[r] + i);
    }
}

// ---- append -------------------------------------------------------------------------
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

struct AppendParams {
    KvLayout l;
    uint8_t* blocks;
    const void *k, *v;
    long long k_tok, k_head, v_tok, v_head;
    const int32_t* slots;
    long long n;              // vectors: tokens * 2 * kv_heads
};

// Eight columns (one packed word) a thread, head_dim / 8 threads a vector.
template <typename T, int FMT, int D>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p)
{
    constexpr int TPV = D / 8;
    kv_begin();
    const int sub = threadIdx.x % TPV;
    for (long long b = (long long)blockIdx.x * (256 / TPV); b < p.n; b += (long long)gridDim.x * (256 / TPV)) {
        const long long v = b + threadIdx.x / TPV, i = v < p.n ? v : p.n - 1;   // whole warps take part in the shuffles
        const int token = (int)(i / (2 * p.l.kv_heads)), hv = (int)(i - (long long)token * (2 * p.l.kv_heads));
        const bool val = hv >= p.l.kv_heads;
        const int head = val ? hv - p.l.kv_heads : hv;
        const int slot = __ldg(p.slots + token);
        const int page = slot >> p.l.page_shift, row = slot & (p.l.page_size - 1);
        const bool live = v < p.n && slot >= 0 && page < p.l.n_pages;
        const T* src = val ? static_cast<const T*>(p.v) + token * p.v_tok + head * p.v_head
                           : static_cast<const T*>(p.k) + token * p.k_tok + head * p.k_head;
        float x[8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = live ? kv_float(src[sub * 8 + j]) : 0.0f;
            amax = fmaxf(amax, fabsf(x[j]));
        }
#pragma unroll
        for (int o = TPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (!live) continue;
        uint8_t* block = p.blocks + ((long long)page * p.l.kv_heads + head) * p.l.block;
        uint8_t* codes = block + ((val ? p.l.page_size : 0) + row) * (D / 2);
        uint8_t* scale = block + p.l.page_size * D + ((val ? p.l.page_size : 0) + row) * (FMT == B4_KV_INT4 ? 2 : 4);
        uint32_t w = 0;
        if (FMT == B4_KV_INT4) {
            const __half sh = __float2half_rn(amax > 0.0f ? __fmul_rn(amax, 1.0f / 7.0f) : 1.0f);
            const float s = __half2float(sh);
#pragma unroll
            for (int j = 0; j < 8; ++j) w |= (uint32_t)int4_code(__fdiv_rn(x[j], s)) << (4 * j);
            if (sub == 0) *reinterpret_cast<__half*>(scale) = sh;
        } else {
            const float s = amax > 0.0f ? amax : 1.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) w |= (uint32_t)nf4_code(__fdiv_rn(x[j], s)) << (4 * j);
            if (sub == 0) *reinterpret_cast<float*>(scale) = s;
        }
        reinterpret_cast<uint32_t*>(codes)[sub] = w;
    }
}

// ---- read-back --------------------------------------------------------------------
struct ReadParams {
    KvLayout l;
    const uint8_t* blocks;
    const int32_t* slots;
    float *k, *v;
    long long n;              // packed words: tokens * 2 * kv_heads * head_dim / 8
};

template <int FMT, int D>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p)
{
    constexpr int TPV = D / 8;
    kv_begin();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < p.n; i += (long long)gridDim.x * 256) {
        const int sub = (int)(i % TPV);
        const long long vec = i / TPV;
        const int token = (int)(vec / (2 * p.l.kv_heads)), hv = (int)(vec - (long long)token * (2 * p.l.kv_heads));
        const bool val = hv >= p.l.kv_heads;
        const int head = val ? hv - p.l.kv_heads : hv;
        const int slot = __ldg(p.slots + token);
        const int page = slot >> p.l.page_shift, row = slot & (p.l.page_size - 1);
        float x[8] = {};
        if (slot >= 0 && page < p.l.n_pages) {
            const uint8_t* block = p.blocks + ((long long)page * p.l.kv_heads + head) * p.l.block;
            const int at = (val ? p.l.page_size : 0) + row;
            const uint32_t w = reinterpret_cast<const uint32_t*>(block + at * (D / 2))[sub];
            const uint8_t* sp = block + p.l.page_size * D;
            const float s = FMT == B4_KV_INT4 ? __half2float(reinterpret_cast<const __half*>(sp)[at])
                                              : reinterpret_cast<const float*>(sp)[at];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = (w >> (4 * j)) & 15;
                x[j] = __fmul_rn(FMT == B4_KV_INT4 ? (float)(c - 8) : c_nf4_table[c], s);
            }
        }
        float4* o = reinterpret_cast<float4*>((val ? p.v : p.k) + ((long long)token * p.l.kv_heads + head) * D) + 2 * sub;
        o[0] = make_float4(x[0], x[1], x[2], x[3]);
        o[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

template <typename T, int FMT>
cudaError_t append(const AppendParams& p, cudaStream_t st)
{
    const int per = 256 / (p.l.head_dim / 8);
    const dim3 grid((unsigned)std::min<long long>((p.n + per - 1) / per, 148LL * 64));
    return p.l.head_dim == 64 ? kv_launch(kv_append_kernel<T, FMT, 64>, grid, 256, 0, st, p)
                              : kv_launch(kv_append_kernel<T, FMT, 128>, grid, 256, 0, st, p);
}

}  // namespace
}  // namespace b4

using namespace b4;

extern "C" {

int b4_kv_block_bytes(int fmt, int page_size, int head_dim, size_t* bytes)
{
    if (!bytes || !kv_shape_ok(fmt, page_size, head_dim)) return cudaErrorInvalidValue;
    *bytes = (size_t)kv_block_bytes(fmt, page_size, head_dim);
    return cudaSuccess;
}

int b4_kv_tables(const b4_kv_step* s, b4_stream_t stream)
{
    if (!s || s->n_req < 0 || s->n_req > B4_KV_MAX_REQUESTS || s->max_tokens < 0 || s->table_width < 0 || s->ring_size < 0)
        return cudaErrorInvalidValue;
    if (s->page_size != 16 && s->page_size != 32 && s->page_size != 64) return cudaErrorInvalidValue;
    if (s->table_stride < s->table_width || !s->q_starts || !s->free_state || !s->free_state_out) return cudaErrorInvalidValue;
    if (s->n_req > 0 && (!s->cached || !s->added || !s->ctx_len || (s->table_width > 0 && !s->tables))) return cudaErrorInvalidValue;
    if ((s->ring_size > 0 && !s->free_pages) || (s->max_tokens > 0 && (!s->slots || !s->positions))) return cudaErrorInvalidValue;
    if (s->free_state_out < s->free_state + 2 && s->free_state < s->free_state_out + 3) return cudaErrorInvalidValue;
    const size_t smem = 8 * (size_t)s->n_req;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 8 * B4_KV_MAX_REQUESTS);
        if (e != cudaSuccess) return e;
    }
    const long long want = ((long long)s->max_tokens + 4 * kTabThreads - 1) / (4 * kTabThreads);
    return kv_launch(kv_tables_kernel, dim3((unsigned)std::max<long long>(1, std::min<long long>(want, 148))), kTabThreads, smem,
                     reinterpret_cast<cudaStream_t>(stream), *s);
}

int b4_kv_append(const b4_kv_cache* cache, const void* k, const void* v, int dtype, long long k_stride_token,
                 long long k_stride_head, long long v_stride_token, long long v_stride_head, const int32_t* slots,
                 int n_tokens, b4_stream_t stream)
{
    AppendParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (n_tokens < 0 || dtype < B4_DTYPE_F16 || dtype > B4_DTYPE_F32) return cudaErrorInvalidValue;
    if (n_tokens == 0) return cudaSuccess;
    const unsigned item = dtype == B4_DTYPE_F32 ? 4 : 2;
    if (!k || !v || !slots || !kv_aligned(k, item) || !kv_aligned(v, item) || !kv_aligned(slots, 4)) return cudaErrorInvalidValue;
    p.blocks = static_cast<uint8_t*>(cache->blocks);
    p.k = k;
    p.v = v;
    p.k_tok = k_stride_token;
    p.k_head = k_stride_head;
    p.v_tok = v_stride_token;
    p.v_head = v_stride_head;
    p.slots = slots;
    p.n = 2LL * n_tokens * cache->kv_heads;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool i4 = cache->fmt == B4_KV_INT4;
    if (dtype == B4_DTYPE_F16) return i4 ? append<__half, B4_KV_INT4>(p, st) : append<__half, B4_KV_NF4>(p, st);
    if (dtype == B4_DTYPE_BF16) return i4 ? append<__nv_bfloat16, B4_KV_INT4>(p, st) : append<__nv_bfloat16, B4_KV_NF4>(p, st);
    return i4 ? append<float, B4_KV_INT4>(p, st) : append<float, B4_KV_NF4>(p, st);
}

int b4_kv_read(const b4_kv_cache* cache, const int32_t* slots, int n_tokens, float* k, float* v, b4_stream_t stream)
{
    ReadParams p;
    const int e = kv_layout(cache, &p.l);
    if (e != cudaSuccess) return e;
    if (n_tokens < 0) return cudaErrorInvalidValue;
    if (n_tokens == 0) return cudaSuccess;
    if (!slots || !k || !v || !kv_aligned(k, 16) || !kv_aligned(v, 16) || !kv_aligned(slots, 4)) return cudaErrorInvalidValue;
    p.blocks = static_cast<const uint8_t*>(cache->blocks);
    p.slots = slots;
    p.k = k;
    p.v = v;
    p.n = 2LL * n_tokens * cache->kv_heads * (cache->head_dim / 8);
    const dim3 grid((unsigned)std::min<long long>((p.n + 255) / 256, 148LL * 64));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (cache->fmt == B4_KV_INT4)
        return cache->head_dim == 64 ? kv_launch(kv_read_kernel<B4_KV_INT4, 64>, grid, 256, 0, st, p)
                                     : kv_launch(kv_read_kernel<B4_KV_INT4, 128>, grid, 256, 0, st, p);
    return cache->head_dim == 64 ? kv_launch(kv_read_kernel<B4_KV_NF4, 64>, grid, 256, 0, st, p)
                                 : kv_launch(kv_read_kernel<B4_KV_NF4, 128>, grid, 256, 0, st, p);
}

}  // extern "C"
