// b4_kv.cu -- the 4-bit key/value cache's bookkeeping: block tables and slots of a
// scheduling step, the quantising append, and the read-back.
#include <climits>

#include "b4_kv.cuh"

namespace b4 {
namespace {

// ---- block tables, slots, positions ----------------------------------------------
// Every CTA scans the requests' lengths itself (new tokens and new pages, both
// exclusive sums, in shared memory), so there is no second launch and no wait
// between CTAs; then the threads of the grid share the packed tokens and the new
// table entries, one each where the grid allows, and find their request by binary
// search in the sums: the time is a handful of dependent loads, whatever the
// requests' lengths (48 requests: 3.7 us; 700 with 175 thousand tokens: 9.0 us, 1.4 MB).  A slot in a new page comes straight from the ring, not through
// the table, which another CTA may still be writing.
constexpr int kTabThreads = 256, kTabGrid = 148 * 8;

__device__ __forceinline__ int sat(long long v) { return (int)(v > INT_MAX ? INT_MAX : v); }

__device__ __forceinline__ int pages_of(long long tokens, int shift, int width)
{
    const long long p = (tokens + (1 << shift) - 1) >> shift;
    return (int)(p < width ? p : width);
}

// the last of n ascending values that is at most x (values[0] <= x)
__device__ __forceinline__ int last_at_most(const int* values, int n, long long x)
{
    int lo = 0;
    for (int step = 1 << (31 - __clz(n)); step > 0; step >>= 1)
        if (lo + step < n && values[lo + step] <= x) lo += step;
    return lo;
}

__global__ void __launch_bounds__(kTabThreads) kv_tables_kernel(const b4_kv_step s, const int shift)
{
    extern __shared__ int tab_smem[];
    int* start = tab_smem;                    // [n_req] first token of a request
    int* first = start + s.n_req;             // [n_req] its first new page, counted from the ring's place
    int* cached = first + s.n_req;            // [n_req]
    __shared__ long long warp_tok[kTabThreads / 32], warp_pag[kTabThreads / 32];
    kv_begin();

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int ring_at = __ldg(s.free_state), ring_left = __ldg(s.free_state + 1);
    const int per = (s.n_req + kTabThreads - 1) / kTabThreads;
    const int r0 = min((int)threadIdx.x * per, s.n_req), r1 = min(r0 + per, s.n_req);
    long long tok = 0, pag = 0;
#pragma unroll 4
    for (int r = r0; r < r1; ++r) {           // sums within the thread
        const int c = max(__ldg(s.cached + r), 0), n = max(__ldg(s.added + r), 0);
        cached[r] = c;
        start[r] = n;
        tok += n;
        pag += pages_of((long long)c + n, shift, s.table_width) - pages_of(c, shift, s.table_width);
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
    for (int r = r0; r < r1; ++r) {           // the thread's own entries: exclusive sums over all
        const long long c = cached[r], n = start[r];
        const int fresh = pages_of(c + n, shift, s.table_width) - pages_of(c, shift, s.table_width);
        start[r] = sat(bt);
        first[r] = sat(bp);
        if (writer) {
            s.ctx_len[r] = sat(c + n);
            s.q_starts[r] = sat(bt);
        }
        bt += n;
        bp += fresh;
    }
    __syncthreads();

    const int head = s.ring_size > 0 ? (int)((unsigned)max(ring_at, 0) % (unsigned)s.ring_size) : 0;
    const int left = min(max(ring_left, 0), s.ring_size);
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

    const int n_tok = sat(all_tok), n_pag = sat(all_pag);
    const long long id0 = (long long)blockIdx.x * kTabThreads + threadIdx.x, ids = (long long)gridDim.x * kTabThreads;
    for (long long i = id0; i < s.max_tokens; i += ids) {
        int slot = -1, pos = 0;
        if (i < n_tok) {
            const int r = last_at_most(start, s.n_req, i);
            const long long c = cached[r], at = c + (i - start[r]), p = at >> shift;
            pos = sat(at);
            if (p < s.table_width) {
                const int held = pages_of(c, shift, s.table_width);
                const int id = p < held ? s.tables[r * s.table_stride + p] : ring(first[r] + (int)p - held);
                if (id >= 0) slot = (id << shift) + (int)(at & ((1 << shift) - 1));
            }
        }
        s.slots[i] = slot;
        s.positions[i] = pos;
    }
    for (long long i = id0; i < n_pag; i += ids) {
        const int r = last_at_most(first, s.n_req, i);
        s.tables[r * s.table_stride + pages_of(cached[r], shift, s.table_width) + (i - first[r])] = ring((int)i);
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

// Vectors (one token's keys or values of one head) are numbered token, then keys
// before values, then head; D / 8 threads hold one, a packed word each.
struct VectorIndex {
    int token, head;
    bool value;
};

__device__ __forceinline__ VectorIndex vector_index(long long i, int kv_heads, unsigned long long magic)
{
    VectorIndex v;
    v.token = (int)__umul64hi((unsigned long long)i, magic);       // i / (2 kv_heads): magic = 2^64 / (2 kv_heads) + 1, i < 2^42
    const int hv = (int)(i - (long long)v.token * (2 * kv_heads));
    v.value = hv >= kv_heads;
    v.head = v.value ? hv - kv_heads : hv;
    return v;
}

struct AppendParams {
    KvLayout l;
    uint8_t* blocks;
    const void *k, *v;
    long long k_tok, k_head, v_tok, v_head;
    const int32_t* slots;
    long long n;                       // vectors: tokens * 2 * kv_heads
    unsigned long long magic;
};

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

// Vectors a thread has in flight, U: two where 16-bit rows fill the GPU more than once (20011 tokens x 4 x 128, bf16 to
// NF4, append and read-back: 40 us against 47 with one), one otherwise (64 tokens x 8 x 128: 4.7 us against 6.7 with
// two; 6007 x 12 x 64 in fp32: 24.6 against 25.3).
constexpr long long kFewBlocks = 148 * 8;

// Bound by memory, 2.1 to 4.5 bytes a column, and at NF4 by issue, 32 instructions a code: 20011 tokens x 4 x 128 from
// bf16 in 29 us, 1.8 TB/s (ncu).
template <typename T, int FMT, int D, bool VEC, int U>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p)
{
    constexpr int TPV = D / 8, per = 256 / TPV;
    float boundary = 4.0f;
    int below = 0;
    if (FMT == B4_KV_NF4) {
        const int lane = threadIdx.x & 31;
        const float start = (lane - 16.5f) / kBins, end = (lane - 15.5f) / kBins;
        // lane c: the boundary above level c; then the first at `start` or above by bisection
        const float level = c_nf4_table[lane & 15], above = __shfl_down_sync(0xffffffffu, level, 1);
        const float mid = lane < 15 ? 0.5f * (level + above) : INFINITY;
#pragma unroll
        for (int step = 8; step > 0; step >>= 1)
            if (__shfl_sync(0xffffffffu, mid, below + step - 1) < start) below += step;
        const float next = __shfl_sync(0xffffffffu, mid, below);
        if (next < end) boundary = next;
    }
    kv_begin();
    const int sub = threadIdx.x % TPV;
    const long long first = (long long)blockIdx.x * (U * per) + threadIdx.x / TPV;
    Columns<T, VEC> c[U];
    uint8_t* block[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = min(first + u * per, p.n - 1);         // whole warps take part in the shuffles
        const VectorIndex v = vector_index(i, p.l.kv_heads, p.magic);
        const int slot = __ldg(p.slots + v.token), page = slot >> p.l.page_shift;
        const bool live = first + u * per < p.n && slot >= 0 && page < p.l.n_pages;
        const T* src = v.value ? static_cast<const T*>(p.v) + v.token * p.v_tok + v.head * p.v_head
                               : static_cast<const T*>(p.k) + v.token * p.k_tok + v.head * p.k_head;
        c[u].load(src + sub * 8);
        block[u] = live ? p.blocks + ((long long)page * p.l.kv_heads + v.head) * p.l.block : nullptr;
        at[u] = (v.value ? p.l.page_size : 0) + (slot & (p.l.page_size - 1));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[j] = c[u].get(j);
            amax = fmaxf(amax, fabsf(x[j]));
        }
#pragma unroll
        for (int o = TPV / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        uint32_t w;
        __half sh;
        if (FMT == B4_KV_INT4) {
            // times fp32's 1/7 as torch divides by a number on the GPU: pages written by such a program have these bytes
            sh = __float2half_rn(amax > 0.0f ? __fmul_rn(amax, 1.0f / 7.0f) : 1.0f);
            w = int4_word(x, __half2float(sh));
        } else {
            if (!(amax > 0.0f)) amax = 1.0f;
            w = nf4_word(x, amax, boundary, below);
        }
        if (!block[u]) continue;
        reinterpret_cast<uint32_t*>(block[u] + at[u] * (D / 2))[sub] = w;
        if (sub == 0) {
            if (FMT == B4_KV_INT4) reinterpret_cast<__half*>(block[u] + p.l.page_size * D)[at[u]] = sh;
            else reinterpret_cast<float*>(block[u] + p.l.page_size * D)[at[u]] = amax;
        }
    }
}

// ---- read-back --------------------------------------------------------------------
struct ReadParams {
    KvLayout l;
    const uint8_t* blocks;
    const int32_t* slots;
    float *k, *v;
    long long n;                       // vectors
    unsigned long long magic;
};

// Bound by its fp32 stores: the same tokens in 20 us, 4.65 TB/s (92.9 MB).
template <int FMT, int D, int U>
__global__ void __launch_bounds__(256) kv_read_kernel(const ReadParams p)
{
    constexpr int TPV = D / 8, per = 256 / TPV;
    const float level = c_nf4_table[threadIdx.x & 15];
    kv_begin();
    const int sub = threadIdx.x % TPV;
    const long long first = (long long)blockIdx.x * (U * per) + threadIdx.x / TPV;
    uint32_t w[U];
    float s[U];
    float* dst[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long i = min(first + u * per, p.n - 1);
        const VectorIndex v = vector_index(i, p.l.kv_heads, p.magic);
        const int slot = __ldg(p.slots + v.token), page = slot >> p.l.page_shift, row = slot & (p.l.page_size - 1);
        w[u] = FMT == B4_KV_INT4 ? 0x88888888u : 0x77777777u;      // zeros outside the cache
        s[u] = 0.0f;
        if (slot >= 0 && page < p.l.n_pages) {
            const uint8_t* block = p.blocks + ((long long)page * p.l.kv_heads + v.head) * p.l.block;
            const int at = (v.value ? p.l.page_size : 0) + row;
            w[u] = reinterpret_cast<const uint32_t*>(block + at * (D / 2))[sub];
            const uint8_t* sp = block + p.l.page_size * D;
            s[u] = FMT == B4_KV_INT4 ? __half2float(reinterpret_cast<const __half*>(sp)[at]) : reinterpret_cast<const float*>(sp)[at];
        }
        dst[u] = first + u * per < p.n ? (v.value ? p.v : p.k) + ((long long)v.token * p.l.kv_heads + v.head) * D + sub * 8 : nullptr;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const uint32_t c = w[u] >> (4 * j);
            x[j] = __fmul_rn(FMT == B4_KV_INT4 ? (float)((int)(c & 15) - 8) : __shfl_sync(0xffffffffu, level, c & 15), s[u]);
        }
        if (!dst[u]) continue;
        reinterpret_cast<float4*>(dst[u])[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(dst[u])[1] = make_float4(x[4], x[5], x[6], x[7]);
    }
}

// blocks of a launch over n vectors, u a thread, and the divisor's magic number
inline long long vector_blocks(long long n, int head_dim, int u)
{
    const int per = u * 256 / (head_dim / 8);
    return (n + per - 1) / per;
}

inline unsigned long long vector_magic(int kv_heads) { return ~0ULL / (2ULL * kv_heads) + 1; }

struct Ints {
    uintptr_t from, to;
    Ints(const int32_t* at, long long n) : from(reinterpret_cast<uintptr_t>(at)), to(from + 4 * n) {}
};

inline bool overlap(const Ints& a, const Ints& b) { return a.from < b.to && b.from < a.to && a.from < a.to && b.from < b.to; }

// whether a lies on entries of a step's tables
inline bool on_tables(const Ints& a, const b4_kv_step* s)
{
    if (s->n_req == 0 || s->table_width == 0 || !overlap(a, Ints(s->tables, (s->n_req - 1) * s->table_stride + s->table_width))) return false;
    const long long row = 4LL * s->table_width, stride = 4 * s->table_stride;
    const long long from = (long long)(a.from - reinterpret_cast<uintptr_t>(s->tables)), to = from + (long long)(a.to - a.from);
    const long long r = from < row ? 0 : (from - row) / stride + 1;        // the first row that ends after `from`
    return r < s->n_req && r * stride < to;
}

// What a step writes lies apart from what it reads, and from what else it writes: every CTA reads the lengths and the
// ring's place while the first one may have written its outputs.
inline bool step_apart(const b4_kv_step* s)
{
    const Ints out[] = {{s->ctx_len, s->n_req}, {s->q_starts, s->n_req + 1LL}, {s->slots, s->max_tokens}, {s->positions, s->max_tokens},
                        {s->free_state_out, 3}};
    const Ints in[] = {{s->cached, s->n_req}, {s->added, s->n_req}, {s->free_pages, s->ring_size}, {s->free_state, 2}};
    for (const Ints& o : out) {
        if (on_tables(o, s)) return false;
        for (const Ints& i : in)
            if (overlap(o, i)) return false;
        for (const Ints& p : out)
            if (&p < &o && overlap(o, p)) return false;
    }
    for (const Ints& i : in)
        if (on_tables(i, s)) return false;
    return true;
}

template <typename T, int FMT, int D, int U>
cudaError_t append_u(const AppendParams& p, bool vec, cudaStream_t st)
{
    const dim3 grid((unsigned)vector_blocks(p.n, D, U));
    return vec ? kv_launch(kv_append_kernel<T, FMT, D, true, U>, grid, 256, 0, st, p) : kv_launch(kv_append_kernel<T, FMT, D, false, U>, grid, 256, 0, st, p);
}

template <typename T, int FMT, int D>
cudaError_t append_d(const AppendParams& p, bool vec, cudaStream_t st)
{
    if constexpr (sizeof(T) == 2)
        if (vector_blocks(p.n, D, 1) > kFewBlocks) return append_u<T, FMT, D, 2>(p, vec, st);
    return append_u<T, FMT, D, 1>(p, vec, st);
}

template <int FMT, int D>
cudaError_t read_d(const ReadParams& p, cudaStream_t st)
{
    const long long few = vector_blocks(p.n, D, 1);
    if (few > kFewBlocks) return kv_launch(kv_read_kernel<FMT, D, 2>, dim3((unsigned)vector_blocks(p.n, D, 2)), 256, 0, st, p);
    return kv_launch(kv_read_kernel<FMT, D, 1>, dim3((unsigned)few), 256, 0, st, p);
}

template <typename T, int FMT>
cudaError_t append(const AppendParams& p, cudaStream_t st)
{
    const long long strides = p.k_tok | p.k_head | p.v_tok | p.v_head;
    const bool vec = kv_aligned(p.k, 16) && kv_aligned(p.v, 16) && strides * (long long)sizeof(T) % 16 == 0;
    return p.l.head_dim == 64 ? append_d<T, FMT, 64>(p, vec, st) : append_d<T, FMT, 128>(p, vec, st);
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
    if (!step_apart(s)) return cudaErrorInvalidValue;
    const size_t smem = 12 * (size_t)s->n_req;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kv_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 12 * B4_KV_MAX_REQUESTS);
        if (e != cudaSuccess) return e;
    }
    const long long want = ((long long)s->max_tokens + kTabThreads - 1) / kTabThreads;
    return kv_launch(kv_tables_kernel, dim3((unsigned)std::max<long long>(1, std::min<long long>(want, kTabGrid))), kTabThreads, smem,
                     reinterpret_cast<cudaStream_t>(stream), *s, s->page_size == 16 ? 4 : s->page_size == 32 ? 5 : 6);
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
    p.magic = vector_magic(cache->kv_heads);
    if (vector_blocks(p.n, cache->head_dim, 1) > 0x7fffffffLL) return cudaErrorInvalidValue;
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
    p.n = 2LL * n_tokens * cache->kv_heads;
    p.magic = vector_magic(cache->kv_heads);
    if (vector_blocks(p.n, cache->head_dim, 1) > 0x7fffffffLL) return cudaErrorInvalidValue;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (cache->fmt == B4_KV_INT4) return cache->head_dim == 64 ? read_d<B4_KV_INT4, 64>(p, st) : read_d<B4_KV_INT4, 128>(p, st);
    return cache->head_dim == 64 ? read_d<B4_KV_NF4, 64>(p, st) : read_d<B4_KV_NF4, 128>(p, st);
}

}  // extern "C"
