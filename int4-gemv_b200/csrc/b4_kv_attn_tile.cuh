// b4_kv_attn_tile.cuh -- attention over the 4-bit cache for many queries a request
// (prompt chunks, long drafts): products of 128 x 128 tiles on the tcgen05 pipe.
//
// Mathematics.  The queries that share a kv head (query tokens x heads of the
// group) are rows; a CTA takes 256 of them (two tiles of 128) through the keys in
// blocks of 64:
//   S = Q K^T  (Q, K in shared memory),  O += P V  (P in tensor memory, V in shared)
// with fp16 operands and fp32 accumulators in tensor memory.  Where a request has
// 128 rows or fewer, the two tiles are the same rows and take every other block: two
// streams, joined at the end.  K and V hold the bare levels (INT4: exact integers;
// NF4: rounded to fp16 with bf16 queries, in two fp16 parts with fp16 ones, each with its
// operands and products), so a token's key scale multiplies a column of S and
// its value scale a column of P, in fp32.  Softmax is the warp kernel's
// (b4_kv_attn_warp.cuh): a maximum that moves only when a score passes it by 2^8,
// weights relative to it and to a running power of two of the value scales, rounded
// to fp16 for the product.
//
// Roles.  Warps 0 and 2: a thread each issues a tile's products (one thread for both
// took 2.4 us a block over its chain of waits and issues).  Warp 1: the schedule.  Warps 4-7 and 8-11:
// softmax of the two tiles, a row a thread.  Warps 12-15: codes to fp16 operands, half
// a token a thread, in the 128-byte swizzle (the same bytes serve K, whose columns are
// the product's depth, and V, whose rows are).  K and V are rings of four, of two where
// levels have two parts.  A
// tile has two S of 64 columns of tensor memory (P takes half of one), so that the
// next block's scores are there when a block's weights are done: with one S of 128
// columns a block waited 4.1 us on the chain scores - softmax - outputs - scores,
// of which the products were 0.5.  The two O take the other 256 columns.
//
// A segment's end.  The next segment's queries are brought into their place, which the
// last scores have left, and its scores computed while this one's outputs go out.  The
// two streams of one row tile are joined in tensor memory: a warp reads the same rows
// of both outputs, so only maxima and sums pass through shared memory.
//
// Split.  The (request, row tile, head, key block) units of the whole call, only
// those that some row sees, form one sequence and every CTA gets an equal run of it;
// a segment (request, tile, head) that crosses CTAs is joined by the last of them to
// arrive, in order, as in the warp kernel.  A segment also costs what its begin and end
// cost: counted as kSegUnits blocks, since the first tiles of a prompt are many short
// segments (five prompts of 200 to 1500 tokens, NF4 in bf16, 64 heads over 8: 310 us without).
//
// What bounds it.  Two row tiles: some 1.6 us a block of 64 keys, of which the products
// are 0.75 (scores with 64 keys a product read Q anew for each: 48 cycles where 32
// multiply); the rest is the chain of a row's softmax, longest in the two quarters of
// the SM whose issue slots the products' warps share.  One row tile: the decoding
// warps, 1.1 us a block.  Two parts: the chain from a block's weights over the writing of
// the values after next, 2.8 us a block (LSU 60 % busy).  Measured (chunk of 2048 tokens
// behind 6000, 28 heads over 4 x 128, INT4): 272 us, 758 TFLOP/s, NF4 in bf16
// 300 us, in fp16 471; the five prompts: 168 us, in fp16 219.  Tried and left out (INT4
// chunk): the tiles half a block apart (289 us);
// the decoding warps in the other two quarters (287 us); scores issued only once the
// last ones are read (286 us).
//
// Every wait is bounded (2 s): one that runs out raises the device error flag and
// ends the CTA.
#pragma once

#include "b4_kv_attn.cuh"
#include "b4_tma.cuh"

namespace b4 {

constexpr int kTileRows = 256, kTileKeys = 64, kTileThreads = 512, kTileStages = 4;
// What a segment (a row tile and head) costs beside its blocks, in blocks' time: the five prompts of the comment above
// take 196 us with 2, 170 with 4, 177 with 6.
constexpr int kSegUnits = 4;

template <typename T, int FMT, int D>
struct TileCfg {
    static constexpr int kRow = D / 2, kScale = FMT == B4_KV_INT4 ? 2 : 4;
    static constexpr int kOperand = 128 * D * 2;                   // bytes of 128 queries of D fp16: D / 64 parts of 128 x 128 bytes
    static constexpr int kBlock = kTileKeys * D * 2;               // of a block's keys or values: parts of 64 x 128 bytes
    // NF4 with fp16 queries: levels in two fp16 parts, each with its operands and products; half as many stages of twice the size
    static constexpr int kParts = FMT == B4_KV_NF4 && std::is_same<T, __half>::value ? 2 : 1;
    static constexpr int kStages = kTileStages / kParts, kStage = kParts * kBlock;
    // Two stages: keys and values have barriers of their own, so that the keys of the block after next are written under a
    // block's softmax, its values still in place (chunk of 2048 behind 6000, NF4 in fp16: 542 us without, 470 to 483 with).
    static constexpr bool kSplit = kStages == 2;
    static constexpr float kUp = kParts == 2 ? kNf4Least : kNf4Even;
    // NF4: pairs of levels by byte, 256 rows of 16 copies (2 lanes a copy), or of 8 copies of both parts, at shared address
    // 16384, so that an OR makes a lookup's address; the operands follow it.  Without it they follow the static part.
    static constexpr int kTable = 16384, kStatic = 13312;
    static constexpr int kPiece = kTileRows * (D + 2);             // floats: output, maxima, sums
    static constexpr int kSmem = 2 * kOperand + 2 * kTileStages * kBlock + (FMT == B4_KV_NF4 ? 2 * kTable - kStatic : 1024);   // kStatic: less than the static part and the system's
};

struct TileSeg {               // a run's part of a segment
    int q0, n, ctx, head, tile, r, blk0, blk1;
    int first, last, end;      // whether it has the segment's first, last block; the run is over
    long long s0, s1;          // the segment's units of blocks (kSegUnits more follow, with nothing to do)
};

struct TileWs {
    int* count;
    float* cross;              // [grid][2] a CTA's part of a segment that began before it / goes on after it
};

// ---- tcgen05 ----------------------------------------------------------------------
// An operand's descriptor: start and leading byte offset in 16 bytes in the lower half;
// stride byte offset (1024: eight rows of 128 bytes), version 1 and the 128-byte
// swizzle in the upper.
__device__ __forceinline__ uint32_t umma_desc(uint32_t at, uint32_t lbo) { return (at >> 4) | (lbo >> 4) << 16; }
constexpr uint32_t kDescUpper = (1024 >> 4) | 1u << 14 | 2u << 29;

// fp32 accumulators, fp16 operands; `mn`: the right operand's rows are the product's depth
__host__ __device__ constexpr uint32_t umma_idesc(int m, int n, bool mn)
{
    return 1u << 4 | (mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}

__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add),
                 "r"(kDescUpper)
                 : "memory");
}

__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add)
{
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\tmov.b64 y, {%2, %5};\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add),
                 "r"(kDescUpper)
                 : "memory");
}

__device__ __forceinline__ void umma_commit(uint64_t* bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void tmem_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define B4_R8(r, i) "=r"((r)[i]), "=r"((r)[i + 1]), "=r"((r)[i + 2]), "=r"((r)[i + 3]), "=r"((r)[i + 4]), "=r"((r)[i + 5]), "=r"((r)[i + 6]), "=r"((r)[i + 7])
#define B4_W8(r, i) "r"((r)[i]), "r"((r)[i + 1]), "r"((r)[i + 2]), "r"((r)[i + 3]), "r"((r)[i + 4]), "r"((r)[i + 5]), "r"((r)[i + 6]), "r"((r)[i + 7])

// 32 columns of the warp's 32 lanes
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t at)
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : B4_R8(r, 0), B4_R8(r, 8), B4_R8(r, 16), B4_R8(r, 24)
        : "r"(at));
}

__device__ __forceinline__ void tmem_ld16(uint32_t* r, uint32_t at)
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : B4_R8(r, 0), B4_R8(r, 8)
                 : "r"(at));
}

__device__ __forceinline__ void tmem_st16(uint32_t at, const uint32_t* r)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
                 B4_W8(r, 0), B4_W8(r, 8)
                 : "memory");
}
#undef B4_R8
#undef B4_W8

__device__ __forceinline__ uint4 lds128(uint32_t at)
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// 16 bytes, or zeros
__device__ __forceinline__ void copy_async16_or_0(uint32_t dst, const void* src, bool there)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

__device__ __forceinline__ unsigned long long now_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ bool mbar_try_wait_long(uint64_t* bar, uint32_t phase)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(phase), "r"(20000u)             // the thread may sleep for 20 us
        : "memory");
    return ok != 0;
}

// Waits for a phase; false when the CTA gave up (here or elsewhere).
__device__ __forceinline__ bool tile_wait(uint64_t* bar, uint32_t phase, volatile int* dead)
{
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
        if (mbar_try_wait_long(bar, phase)) return true;
    const unsigned long long t0 = now_ns();
#pragma unroll 1
    while (!*dead) {
        if (mbar_try_wait_long(bar, phase)) return true;
        if (now_ns() - t0 > 2000000000ULL) {
            *dead = 1;
            atomicOr(&g_device_error, kErrMbarrierTimeout);
        }
    }
    return false;
}

// ... by a whole warp, with one answer
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t phase, volatile int* dead)
{
    return __all_sync(0xffffffffu, tile_wait(bar, phase, dead));
}

__device__ __forceinline__ bool elect_one()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

template <int R>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

// the blocks of keys that some row of a request's tile sees; one even where none is seen
__device__ __forceinline__ void tile_blocks(const AttnParams& p, int n, int ctx, int tile, int& b0, int& b1)
{
    const unsigned g = p.group;
    const int rows = n * p.group, t0 = (int)((unsigned)(tile * kTileRows) / g), t1 = (int)((unsigned)(min((tile + 1) * kTileRows, rows) - 1) / g);
    const int held = attn_held(p, ctx), end = p.a.flags & B4_KV_FULL ? held : max(0, min(held, ctx - n + t1 + 1));
    const int begin = p.a.window > 0 ? max(0, ctx - n + t0 + 1 - p.a.window) : 0;
    b0 = begin / kTileKeys;
    b1 = max(b0 + 1, (end + kTileKeys - 1) / kTileKeys);
}

template <typename T, int FMT, int D>
__global__ void __launch_bounds__(kTileThreads, 1) kv_attn_tile_kernel(const AttnParams p, const TileWs ws)
{
    using C = TileCfg<T, FMT, D>;
    constexpr int kStages = C::kStages;
    extern __shared__ __align__(1024) uint8_t tile_smem[];
    __shared__ uint64_t seg_full[2], seg_empty[2], q_full[2], s_full[2][2], p_full[2][2], o_done[2][2], q_both, q_free, tops, team, drain[2];
    __shared__ uint64_t full[kTileStages], empty[kTileStages], values_full[2], keys_empty[2];      // the last two: kSplit
    __shared__ TileSeg segs[2];
    __shared__ long long units_before[kTileThreads + 1];
    __shared__ int tiles_before[kTileThreads + 1];
    __shared__ long long warp_sum[kTileThreads / 32];
    __shared__ __align__(16) float key_scale[kTileStages][kTileKeys], value_scale[kTileStages][kTileKeys];
    __shared__ int value_exp[kTileStages], block_pages[kTileStages];
    __shared__ float value_top[2][2];
    __shared__ float q_factor[2][128], stream_max[2][128], stream_sum[2][128], stream_up[2][128];
    __shared__ uint32_t tmem_at;
    __shared__ volatile int dead;
    __shared__ int joins;

    const int tid = threadIdx.x, lane = tid & 31, warp_u = __shfl_sync(0xffffffffu, tid >> 5, 0), warp = warp_u;
    const b4_kv_attn& a = p.a;
    const uint32_t operands = FMT == B4_KV_NF4 ? 2 * C::kTable : (smem_addr(tile_smem) + 1023) & ~1023u;
    const uint32_t keys_at = operands + 2 * C::kOperand, values_at = keys_at + kStages * C::kStage;     // after Q of both tiles
    if (FMT == B4_KV_NF4 && (smem_addr(tile_smem) > C::kTable || smem_addr(tile_smem) < C::kStatic)) {   // the static part is not as kSmem takes it
        if (tid == 0) atomicOr(&g_device_error, kErrMbarrierTimeout);
        return;
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&seg_full[i], 1);
            mbar_init(&seg_empty[i], 14);
            mbar_init(&q_full[i], 4);
            for (int j = 0; j < 2; ++j) {
                mbar_init(&s_full[i][j], C::kSplit ? 2 : 1);
                mbar_init(&p_full[i][j], 4);
                mbar_init(&o_done[i][j], 1);
            }
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&full[i], 4);
            mbar_init(&empty[i], 2);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&values_full[i], 4);
            mbar_init(&keys_empty[i], 2);
        }
        mbar_init(&tops, 2);
        mbar_init(&team, 8);
        mbar_init(&q_both, 4);
        mbar_init(&q_free, 1);
        mbar_init(&drain[0], 1);
        mbar_init(&drain[1], 1);
        dead = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&tmem_at)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (FMT == B4_KV_NF4) {
        for (int i = tid; i < 256 * 4; i += kTileThreads) {
            const uint32_t v = nf4_pair(i >> 2, C::kUp), w = C::kParts == 2 ? nf4_pair_low(i >> 2, C::kUp) : v;
            asm volatile("st.shared.v4.u32 [%0], {%1, %2, %1, %2};" ::"r"(C::kTable + i * 16), "r"(v), "r"(w) : "memory");
        }
    }
    fence_mbar_init();
    kv_begin();

    // ---- the call's units: tiles of all requests, then each tile's heads and blocks ----
    auto taken = [&](const AttnReq& q) { return q.n * p.group > p.rows_above; };
    auto tiles_of = [&](int r) {
        const AttnReq q = attn_request(p, r);
        return taken(q) ? (q.n * p.group + kTileRows - 1) / kTileRows : 0;
    };
    auto scan = [&](long long v) {             // exclusive sums over the threads; the total comes back in all
        long long inc = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
        }
        __syncthreads();
        if (lane == 31) warp_sum[warp] = inc;
        __syncthreads();
        long long before = inc - v;
        for (int w = 0; w < warp; ++w) before += warp_sum[w];
        return before;
    };
    const int per = (a.n_req + kTileThreads - 1) / kTileThreads;
    {
        int mine = 0;
        for (int i = 0; i < per; ++i)
            if (tid * per + i < a.n_req) mine += tiles_of(tid * per + i);
        const long long before = scan(mine);
        tiles_before[tid] = (int)before;
        if (tid == kTileThreads - 1) tiles_before[kTileThreads] = (int)before + mine;
        __syncthreads();
    }
    const int all_tiles = tiles_before[kTileThreads];
    // a place in the sequence of tiles
    struct Cursor {
        int r, tile, tiles;
        AttnReq q;
    };
    auto seek = [&](int tile) {
        Cursor c;
        int lo = 0;
#pragma unroll 1
        for (int step = kTileThreads / 2; step > 0; step >>= 1)
            if (tiles_before[lo + step] <= tile) lo += step;
        c.r = lo * per;
        tile -= tiles_before[lo];
        for (;; ++c.r) {
            c.tiles = tiles_of(c.r);
            if (tile < c.tiles || c.r >= a.n_req - 1) break;
            tile -= c.tiles;
        }
        c.tile = tile;
        c.q = attn_request(p, c.r);
        return c;
    };
    auto next = [&](Cursor& c) {
        if (++c.tile < c.tiles) return;
        c.tile = 0;
        do {
            c.tiles = ++c.r < a.n_req ? tiles_of(c.r) : 1;
        } while (c.tiles == 0);
        if (c.r < a.n_req) c.q = attn_request(p, c.r);
    };
    const int t_first = (int)((long long)tid * all_tiles / kTileThreads), t_last = (int)((long long)(tid + 1) * all_tiles / kTileThreads);
    {
        long long mine = 0;
        if (t_first < t_last) {
            Cursor c = seek(t_first);
            for (int i = t_first; i < t_last; ++i) {
                int b0, b1;
                tile_blocks(p, c.q.n, c.q.ctx, c.tile, b0, b1);
                mine += (long long)(b1 - b0 + kSegUnits) * p.l.kv_heads;
                if (i + 1 < t_last) next(c);
            }
        }
        const long long before = scan(mine);
        units_before[tid] = before;
        if (tid == kTileThreads - 1) units_before[kTileThreads] = before + mine;
        tmem_before_sync();
        __syncthreads();
        tmem_after_sync();
    }
    const long long total = units_before[kTileThreads];
    const int ctas = (int)min((long long)gridDim.x, total), cta = blockIdx.x;
    const long long share = ctas > 0 ? total / ctas : 0, rest = ctas > 0 ? total - share * ctas : 0;
    const long long u0 = cta < ctas ? cta * share + min((long long)cta, rest) : 0, u1 = cta < ctas ? u0 + share + (cta < rest) : 0;
    auto owner = [&](long long u) { return (int)(u < rest * (share + 1) ? u / (share + 1) : rest + (u - rest * (share + 1)) / share); };
    const uint32_t tmem = tmem_at;

    if (warp < 4) {
        regs_down<64>();
        if (warp == 1) {
            // ---- schedule ----
            long long u = u0;
            int k = 0;
            Cursor c = {};
            long long at = 0;
            if (u < u1) {
                int lo = 0;
#pragma unroll 1
                for (int step = kTileThreads / 2; step > 0; step >>= 1)
                    if (units_before[lo + step] <= u) lo += step;
                at = units_before[lo];
                c = seek((int)((long long)lo * all_tiles / kTileThreads));
            }
            for (;;) {
                TileSeg s = {};
                if (u < u1 && c.r < a.n_req) {
                    int b0, b1;
                    tile_blocks(p, c.q.n, c.q.ctx, c.tile, b0, b1);
                    const long long blocks = b1 - b0, units = blocks + kSegUnits;
                    if (u >= at + units * p.l.kv_heads) {
                        at += units * p.l.kv_heads;
                        next(c);
                        continue;
                    }
                    s.q0 = c.q.q0;
                    s.n = c.q.n;
                    s.ctx = c.q.ctx;
                    s.tile = c.tile;
                    s.r = c.r;
                    s.head = (int)((u - at) / units);
                    s.s0 = at + s.head * units;
                    s.s1 = s.s0 + blocks;
                    if (u >= s.s1) {               // only of its end
                        u = s.s0 + units;
                        continue;
                    }
                    s.blk0 = b0 + (int)(u - s.s0);
                    const long long stop = min(s.s1, u1);
                    s.blk1 = s.blk0 + (int)(stop - u);
                    s.first = u == s.s0;
                    s.last = stop == s.s1;
                    u = s.last ? s.s0 + units : stop;
                } else {
                    s.end = 1;
                }
                if (k >= 2 && !warp_wait(&seg_empty[k & 1], (k >> 1) + 1 & 1, &dead)) break;
                if (lane == 0) {
                    segs[k & 1] = s;
                    mbar_arrive(&seg_full[k & 1]);
                }
                __syncwarp();
                ++k;
                if (s.end) break;
            }
        } else if (warp != 3) {
            // ---- products: one warp a tile ----
            // Everything that an instruction takes is the same in all lanes and known to be (values from shared memory come
            // through a shuffle), so that it sits in uniform registers; one elected lane issues.
            const int x = warp_u >> 1;
            constexpr uint32_t id_s = umma_idesc(128, kTileKeys, false), id_o = umma_idesc(128, D, true);
            constexpr uint32_t kPartQ = 128 * 128, kPartB = kTileKeys * 128;       // bytes from 64 columns to the next
            const uint32_t desc_k = umma_desc(keys_at, 16), desc_v = umma_desc(values_at, kPartB);
            const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0), s_at = tmem_u + x * 128, o_at = tmem_u + 256 + x * 128;
            int blocks_before = 0, cq = 0, shared = 0, cp = 0, cs = 0;             // blocks so far; the tile's queries, shared ones, weights, scores
            bool ok = true;
            for (int k = 0; ok; ++k) {
                if (!(ok = warp_wait(&seg_full[k & 1], k >> 1 & 1, &dead))) break;
                const TileSeg& g = segs[k & 1];
                const int blocks = __shfl_sync(0xffffffffu, g.blk1 - g.blk0, 0), end = __shfl_sync(0xffffffffu, g.end, 0);
                const bool two = __shfl_sync(0xffffffffu, g.n * p.group - g.tile * kTileRows, 0) > 128;
                if (elect_one()) mbar_arrive(&seg_empty[k & 1]);
                __syncwarp();
                if (end) break;
                // two tiles of rows: each takes every block; one: the tile's warp takes every other, and says so of the
                // others once they are there (a block is left when both warps have left it)
                const uint32_t desc_q = umma_desc(operands + (two ? x : 0) * C::kOperand, 16);
                // a tile's next block's scores are asked for before its weights are waited for, as far as the stages reach
                const int ahead = two || C::kSplit ? 1 : 2;
                bool queries = two || x == 0, add = false;
                if (!two && x == 1) {                              // the first tile's queries
                    if (!(ok = warp_wait(&q_both, shared++ & 1, &dead))) break;
                    if (blocks < 2) {
                        if (elect_one()) mbar_arrive(&q_free);
                        __syncwarp();
                    }
                }
#pragma unroll 1
                for (int i = -ahead; i < blocks; ++i) {
                    const int sb = i + ahead;
                    const bool taken = two || (i & 1) == x;
                    if (sb < blocks) {
                        const int b = blocks_before + sb, stage = b & (kStages - 1), buf = cs & 1;
                        if (!(ok = warp_wait(&full[stage], b / kStages & 1, &dead))) break;
                        if (two || (sb & 1) == x) {
                            if (queries) {
                                if (!(ok = warp_wait(&q_full[x], cq++ & 1, &dead))) break;
                                queries = false;
                            }
                            tmem_after_sync();
                            if (elect_one()) {
                                const uint32_t kd = desc_k + stage * (C::kStage >> 4);
#pragma unroll
                                for (int part = 0; part < C::kParts; ++part)
#pragma unroll
                                    for (int j = 0; j < D / 16; ++j)
                                        umma_ss(s_at + buf * 64, desc_q + (j >> 2) * (kPartQ >> 4) + (j & 3) * 2,
                                                kd + part * (C::kBlock >> 4) + (j >> 2) * (kPartB >> 4) + (j & 3) * 2, id_s, part > 0 || j > 0);
                                umma_commit(&s_full[x][buf]);
                                if (C::kSplit) {
                                    mbar_arrive(&s_full[x][buf]);  // the scales, too, are there for who waits for the scores
                                    umma_commit(&keys_empty[stage]);
                                }
                                if (!two && x == 1 && sb + 2 >= blocks) umma_commit(&q_free);
                            }
                            __syncwarp();
                            ++cs;
                        } else if (C::kSplit) {
                            if (elect_one()) mbar_arrive(&keys_empty[stage]);
                            __syncwarp();
                        }
                    }
                    if (i >= 0) {                                  // the block's operands are there since its scores
                        const int stage = (blocks_before + i) & (kStages - 1), buf = cp & 1;
                        if (C::kSplit && !(ok = warp_wait(&values_full[stage], (blocks_before + i) / kStages & 1, &dead))) break;
                        if (taken) {
                            if (!(ok = warp_wait(&p_full[x][buf], cp >> 1 & 1, &dead))) break;
                            ++cp;
                        }
                        tmem_after_sync();
                        if (elect_one()) {
                            if (taken) {
                                const uint32_t pa = s_at + buf * 64, v = desc_v + stage * (C::kStage >> 4);
#pragma unroll
                                for (int part = 0; part < C::kParts; ++part)
#pragma unroll
                                    for (int j = 0; j < kTileKeys / 16; ++j)
                                        umma_ts(o_at, pa + j * 8, v + part * (C::kBlock >> 4) + j * (2048 >> 4), id_o, add || part > 0 || j > 0);
                                umma_commit(&o_done[x][buf]);
                                umma_commit(&empty[stage]);
                            } else {
                                mbar_arrive(&empty[stage]);
                            }
                        }
                        __syncwarp();
                        add = add || taken;
                    }
                }
                blocks_before += blocks;
            }
            if (elect_one()) {
                umma_commit(&drain[x]);        // nothing in flight when the CTA ends
                for (int i = 0; i < 1 << 20 && !mbar_try_wait(&drain[x], 0); ++i) {}
            }
            __syncwarp();
        }
    } else if (warp >= 12) {
        // ---- codes to operands: half a token a thread (warps 12, 13 the first columns and the keys' scales, 14, 15 the others
        // and the values'); a block's codes are asked for while the one before is written, its page ids a block before that
        regs_down<96>();
        const int t = tid & 63, half = warp >> 1 & 1;
        constexpr int W = D / 16;              // words of half a token's codes
        constexpr int kPart = D == 128 ? kTileKeys * 128 : 0;      // D = 64: both halves lie in one part
        const uint32_t row_at = t * 128 + half * kPart, swizzle = (t & 7) << 4, chunk0 = D == 128 ? 0 : half * W;
        const int row = t & (p.l.page_size - 1);
        struct Codes {
            uint4 k[W / 4], v[W / 4];
            uint32_t scale;                    // the key's or the value's, as it lies there
            bool there;
        };
        TileSeg s = {};
        int k = -1, blk = 0, vexp = kNoExp, see_begin = 0, see_end = 0;
        bool ok = true;
        auto page_id = [&](int block) {
            const int token = block * kTileKeys + t;
            return block < s.blk1 && token < attn_held(p, s.ctx) ? __ldg(a.tables + (long long)s.r * a.table_stride + (token >> p.l.page_shift)) : -1;
        };
        auto load = [&](int page, Codes& c) {
            c.there = (unsigned)page < (unsigned)p.l.n_pages;
#pragma unroll
            for (int i = 0; i < W / 4; ++i) c.k[i] = c.v[i] = make_uint4(0, 0, 0, 0);
            c.scale = 0;
            if (!c.there) return;
            const uint8_t* b = p.blocks + ((long long)page * p.l.kv_heads + s.head) * p.l.block;
            const uint8_t* codes = b + row * C::kRow + half * (C::kRow / 2);
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                c.k[i] = __ldg(reinterpret_cast<const uint4*>(codes) + i);
                c.v[i] = __ldg(reinterpret_cast<const uint4*>(codes + p.l.page_size * C::kRow) + i);
            }
            const uint8_t* sp = b + p.l.page_size * D + (half * p.l.page_size + row) * C::kScale;
            c.scale = FMT == B4_KV_INT4 ? __ldg(reinterpret_cast<const uint16_t*>(sp)) : __ldg(reinterpret_cast<const uint32_t*>(sp));
        };
        auto write = [&](uint32_t to, const uint4 (&raw)[W / 4]) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
#pragma unroll
            for (int i = 0; i < W; ++i) {
                uint32_t h[4], low[4];
                if (FMT == B4_KV_INT4) {
                    int4_word_to_half2(w[i], h);
                } else if (C::kParts == 2) {
                    const uint32_t copy = C::kTable | (lane & 7) * 8;
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const uint2 x = lds64((b ? w[i] >> (8 * b - 6) : w[i] << 6) & 0x3fc0u | copy);
                        h[b] = x.x;
                        low[b] = x.y;
                    }
                } else {
                    const uint32_t copy = C::kTable | (lane & 15) * 4;
                    h[0] = lds32((w[i] << 6 & 0x3fc0u) | copy);
                    h[1] = lds32((w[i] >> 2 & 0x3fc0u) | copy);
                    h[2] = lds32((w[i] >> 10 & 0x3fc0u) | copy);
                    h[3] = lds32((w[i] >> 18 & 0x3fc0u) | copy);
                }
                asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + (((chunk0 + i) << 4) ^ swizzle)), "r"(h[0]), "r"(h[1]), "r"(h[2]),
                             "r"(h[3])
                             : "memory");
                if (C::kParts == 2)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + C::kBlock + (((chunk0 + i) << 4) ^ swizzle)), "r"(low[0]),
                                 "r"(low[1]), "r"(low[2]), "r"(low[3])
                                 : "memory");
            }
        };
        // the next segment, or the end of the run
        auto next_segment = [&]() {
            ++k;
            if (!(ok = warp_wait(&seg_full[k & 1], k >> 1 & 1, &dead))) return false;
            s = segs[k & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_empty[k & 1]);
            if (s.end) return false;
            const int last_row = min((s.tile + 1) * kTileRows, s.n * p.group) - 1;
            see_end = a.flags & B4_KV_FULL ? s.ctx : min(s.ctx, s.ctx - s.n + last_row / p.group + 1);
            see_begin = a.window > 0 ? s.ctx - s.n + s.tile * kTileRows / p.group + 1 - a.window : 0;
            return true;
        };
        Codes now, next;
        int id_next = -1;
        bool more = next_segment();
        if (more) {
            blk = s.blk0;
            const int id = page_id(blk);
            id_next = page_id(blk + 1);
            load(id, now);
        }
#pragma unroll 1
        for (int b = 0; more; ++b) {
            const int stage = b & (kStages - 1);
            if (blk + 1 < s.blk1) {
                load(id_next, next);
                id_next = page_id(blk + 2);
            }
            const int scales = b & (kTileStages - 1);
            if (b >= kStages && !(ok = warp_wait(C::kSplit ? &keys_empty[stage] : &empty[stage], (b / kStages + 1) & 1, &dead))) break;
            // scales: those of tokens that no row sees are 0, the values' relative to a running power of two
            const int token = blk * kTileKeys + t;
            const bool seen = now.there && token < see_end && token >= see_begin;
            const float scale = !seen ? 0.0f : FMT == B4_KV_INT4 ? __half2float(__ushort_as_half((unsigned short)now.scale)) : __uint_as_float(now.scale);
            if (half) {
                if (blk == s.blk0) vexp = kNoExp;
                const unsigned bits = __reduce_max_sync(0xffffffffu, scale < 3.4028235e38f ? __float_as_uint(fabsf(scale)) : 0u);
                if (lane == 0) {
                    value_top[b & 1][warp & 1] = __uint_as_float(bits);
                    mbar_arrive(&tops);
                }
                __syncwarp();
                if (!C::kSplit) write(values_at + stage * C::kStage + row_at, now.v);      // while the other warp's maximum comes
                if (!(ok = warp_wait(&tops, b & 1, &dead))) break;
                const float top = fmaxf(value_top[b & 1][0], value_top[b & 1][1]);
                vexp = max(vexp, (int)(__float_as_uint(top) >> 23) - 126);
                value_scale[scales][t] = fminf(scale * pow2(kLift - vexp), 3.4028235e38f);    // finite, so that a weight of 0 makes 0 of it
                if (t == 0) value_exp[scales] = vexp;
            } else {
                key_scale[scales][t] = scale;
                // tokens that are not there lie in whole pages of 16 at least: two bits a warp
                const unsigned pages = __ballot_sync(0xffffffffu, now.there);
                if (lane == 0) reinterpret_cast<uint8_t*>(&block_pages[scales])[warp & 1] = (uint8_t)((pages & 1) | (pages >> 16 & 1) << 1);
                if (!C::kSplit) write(values_at + stage * C::kStage + row_at, now.v);
            }
            write(keys_at + stage * C::kStage + row_at, now.k);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[stage]);
            if (C::kSplit) {
                if (b >= kStages && !(ok = warp_wait(&empty[stage], (b / kStages + 1) & 1, &dead))) break;
                write(values_at + stage * C::kStage + row_at, now.v);
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&values_full[stage]);
            }
            if (++blk < s.blk1) {
                now = next;
            } else {
                more = next_segment();
                if (more) {
                    blk = s.blk0;
                    const int id = page_id(blk);
                    id_next = page_id(blk + 1);
                    load(id, now);
                }
            }
        }
    } else {
        // ---- softmax: a row a thread ----
        regs_up<176>();
        const int x = (warp >> 2) - 1, t = tid & 127;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;          // 32 lanes a warp, lane in the upper half
        const uint32_t s_at = tmem + lanes + x * 128, o_at = tmem + lanes + 256 + x * 128;
        int cs = 0, ring0 = 0, teams = 0, shared = 0;      // this tile's blocks so far; all blocks; barriers' turns
        bool ok = true;
        TileSeg s;
        // A segment's queries to shared memory.  ask: copies in flight, a warp its 32 rows, D / 8 lanes a row.  put: each
        // thread turns its row into fp16 in the order of the decoded codes (bf16: times a power of two, as query_operand);
        // the factor that the row's products then lack is returned.  Where both tiles are the same rows, the first one's
        // warps do it, and the second's find the factors in q_factor.
        constexpr int kLanes = D / 8;
        constexpr bool kBf16 = std::is_same<T, __nv_bfloat16>::value;
        auto query_at = [&](int r, int c) { return operands + x * C::kOperand + (c >> 3) * 16384 + r * 128 + (((c & 7) ^ (r & 7)) << 4); };
        auto ask = [&](const TileSeg& g) {
            const int rows = g.n * p.group, from = g.tile * kTileRows;
            const bool two = rows - from > 128;
            if (!two && x == 1) return;
            const int row = from + (two ? x * 128 : 0) + t, token = row / p.group;
            const long long at = (g.q0 + token) * a.q_stride_token + (g.head * p.group + (row - token * p.group)) * a.q_stride_head;
            const unsigned in = __ballot_sync(0xffffffffu, row < rows);
#pragma unroll 4
            for (int i = lane / kLanes; i < 32; i += 32 / kLanes) {
                const long long src = __shfl_sync(0xffffffffu, at, i);
                const int ok = in >> i & 1;
                copy_async16_or_0(query_at((warp & 3) * 32 + i, lane & (kLanes - 1)),
                                  static_cast<const T*>(a.q) + (ok ? src + (lane & (kLanes - 1)) * 8 : 0), ok);
            }
        };
        auto put = [&](const TileSeg& g) -> float {
            const bool two = g.n * p.group - g.tile * kTileRows > 128;
            if (!two && x == 1) return 1.0f;
            const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;
            float factor = 1.0f, up = 1.0f;
            asm volatile("cp.async.wait_all;" ::: "memory");
            __syncwarp();
            if (kBf16) {
                uint32_t top = 0;
#pragma unroll 4
                for (int c = 0; c < kLanes; ++c) {
                    const uint4 v = lds128(query_at(t, c));
                    const uint32_t y[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) top = max(top, max(y[j] << 16 & 0x7fffffffu, y[j] & 0x7fff0000u));
                }
                const int e = min(max((int)(top >> 23) - 127, -110), 126);
                up = pow2(10 - e);
                factor = pow2(e - 10);
                if (!two) q_factor[shared & 1][t] = factor;
            }
            if (kBf16 || FMT == B4_KV_INT4 || sign) {
#pragma unroll 4
                for (int c = 0; c < kLanes; ++c) {
                    uint4 v = lds128(query_at(t, c));
                    if (kBf16) {
                        uint32_t* y = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                        for (int j = 0; j < 4; ++j) y[j] = pack_half2(__uint_as_float(y[j] << 16) * up, __uint_as_float(y[j] & 0xffff0000u) * up);
                    }
                    if (FMT == B4_KV_INT4) v = int4_pair_order(v);
                    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(query_at(t, c)), "r"(v.x ^ sign), "r"(v.y ^ sign), "r"(v.z ^ sign),
                                 "r"(v.w ^ sign)
                                 : "memory");
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&q_full[x]);
                if (!two) mbar_arrive(&q_both);
            }
            return factor;
        };
        auto together = [&]() {                // the eight softmax warps
            __syncwarp();
            if (lane == 0) mbar_arrive(&team);
            return warp_wait(&team, teams++ & 1, &dead);
        };
        auto fetch = [&](int k) {
            if (!(ok = warp_wait(&seg_full[k & 1], k >> 1 & 1, &dead))) return;
            s = segs[k & 1];
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_empty[k & 1]);
        };
        fetch(0);
        float factor = 1.0f;
        if (ok && !s.end) {
            ask(s);
            factor = put(s);
        }
#pragma unroll 1
        for (int k = 1; ok && !s.end; ++k) {
            const int blocks = s.blk1 - s.blk0, rows = s.n * p.group, row0 = s.tile * kTileRows;
            const bool two = rows - row0 > 128;
            const int row = row0 + (two ? x * 128 : 0) + t;
            const bool mine = row < rows;
            const int token = row / p.group, head = s.head * p.group + (row - token * p.group), q0 = s.q0;
            const bool whole = s.first && s.last, first = s.first;
            const long long s0 = s.s0, s1 = s.s1;
            const int lim = a.flags & B4_KV_FULL ? s.ctx : min(s.ctx, s.ctx - s.n + token + 1);
            const int from = a.window > 0 ? lim - a.window : 0;
            if (kBf16 && !two && x == 1) {
                if (!(ok = warp_wait(&q_both, shared & 1, &dead))) break;
                factor = q_factor[shared & 1][t];
            }
            const float qf = fmaxf(factor * (fabsf(a.scale) * kLog2e) * (FMT == B4_KV_NF4 ? 1.0f / C::kUp : 1.0f), 1e-30f);
            float m = kNoMax, l = 0.0f;
            int vexp = kNoExp;
            bool any = false;                  // whether O holds something
#pragma unroll 1
            for (int i = two ? 0 : x; i < blocks && ok; i += two ? 1 : 2, ++cs) {
                const int scales = (ring0 + i) & (kTileStages - 1), buf = cs & 1;
                if (!(ok = warp_wait(&s_full[x][buf], cs >> 1 & 1, &dead))) break;
                // the scales' writers; after the scores, so that the phase asked for is the last one done.  kSplit: the next one
                // may be done too, and the scores' barrier speaks for the scales
                if (!C::kSplit && !(ok = warp_wait(&full[scales], (ring0 + i) / kStages & 1, &dead))) break;
                tmem_after_sync();
                const int key0 = (s.blk0 + i) * kTileKeys, pages = block_pages[scales] & 0xffff, ve = value_exp[scales];
                const float4* ks = reinterpret_cast<const float4*>(key_scale[scales]);
                float2 v[kTileKeys / 2];       // the row's scores
                tmem_ld32(reinterpret_cast<uint32_t*>(v), s_at + buf * 64);
                tmem_ld32(reinterpret_cast<uint32_t*>(v) + 32, s_at + buf * 64 + 32);
                tmem_wait_ld();                // nothing between: the registers are the loads' until here
#pragma unroll
                for (int j = 0; j < kTileKeys / 4; ++j) {
                    const float4 f = ks[j];
                    v[2 * j] = __fmul2_rn(v[2 * j], make_float2(f.x, f.y));
                    v[2 * j + 1] = __fmul2_rn(v[2 * j + 1], make_float2(f.z, f.w));
                }
                if (__any_sync(0xffffffffu, key0 + kTileKeys > lim || key0 < from || pages != 0x0303)) {
                    const int hi = lim - key0, lo = from - key0;
#pragma unroll
                    for (int j = 0; j < kTileKeys; ++j) {
                        float& y = j & 1 ? v[j / 2].y : v[j / 2].x;
                        if (j >= hi || j < lo || !(pages >> ((j >> 5) * 8 + (j >> 4 & 1)) & 1)) y = -INFINITY;
                    }
                }
                float tops4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int j = 0; j < kTileKeys / 2; ++j) tops4[j & 3] = fmaxf(tops4[j & 3], fmaxf(v[j].x, v[j].y));
                const float top = fmaxf(fmaxf(tops4[0], tops4[1]), fmaxf(tops4[2], tops4[3]));
                if (__any_sync(0xffffffffu, top * qf > m + 8.0f) || ve != vexp) {
                    const float next = top == -INFINITY ? m : fmaxf(m, top * qf), keep_l = fast_exp2(m - next);
                    const float keep = keep_l * pow2(max(vexp - ve, -126));
                    m = next;
                    vexp = ve;
                    l *= keep_l;
                    if (any) {                 // two barriers in turn: the scores at hand say that the block before the last is done
                        if (!(ok = warp_wait(&o_done[x][cs - 1 & 1], (cs - 1) >> 1 & 1, &dead))) break;
                        tmem_after_sync();
#pragma unroll 1
                        for (int c = 0; c < D; c += 16) {
                            uint32_t o[16];
                            tmem_ld16(o, o_at + c);
                            tmem_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                            tmem_st16(o_at + c, o);
                        }
                        tmem_wait_st();
                    }
                }
                any = true;
                const float2 q2 = make_float2(qf, qf), m2 = make_float2(-m, -m);
                const float4* vs = reinterpret_cast<const float4*>(value_scale[scales]);
                float2 l2[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                uint32_t w[kTileKeys / 2];
#pragma unroll
                for (int j = 0; j < kTileKeys / 4; ++j) {
                    const float4 f = vs[j];
                    float2 e0 = __ffma2_rn(v[2 * j], q2, m2), e1 = __ffma2_rn(v[2 * j + 1], q2, m2);
                    e0 = make_float2(fast_exp2(e0.x), fast_exp2(e0.y));
                    e1 = make_float2(fast_exp2(e1.x), fast_exp2(e1.y));
                    l2[0] = __fadd2_rn(l2[0], e0);
                    l2[1] = __fadd2_rn(l2[1], e1);
                    e0 = __fmul2_rn(e0, make_float2(f.x, f.y));
                    e1 = __fmul2_rn(e1, make_float2(f.z, f.w));
                    w[2 * j] = pack_half2(e0.x, e0.y);
                    w[2 * j + 1] = pack_half2(e1.x, e1.y);
                }
                // the weights take the first 32 of the scores' 64 columns
                tmem_st16(s_at + buf * 64, w);
                tmem_st16(s_at + buf * 64 + 16, w + 16);
                l += (l2[0].x + l2[0].y) + (l2[1].x + l2[1].y);
                tmem_wait_st();
                tmem_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[x][buf]);
            }
            if (!ok) break;
            ring0 += blocks;
            // The next segment's queries, whose scores are then computed under this one's end.  Their place is free: the
            // tile's last scores have been read; one tile of rows: and the other stream's are done.
            fetch(k);
            if (!ok) break;
            if (!two && !(ok = warp_wait(&q_free, shared++ & 1, &dead))) break;
            if (!s.end) ask(s);
            if (any && !(ok = warp_wait(&o_done[x][cs - 1 & 1], (cs - 1) >> 1 & 1, &dead))) break;
            if (!s.end) factor = put(s);

            // ---- the segment's rows, or a piece of them: a row a thread; one tile of rows: half a row's columns, of both streams ----
            const float vup = any ? pow2(vexp - kLift) * (FMT == B4_KV_NF4 ? 1.0f / C::kUp : 1.0f) : 0.0f;
            float wa = vup, wb = 0.0f;
            if (!two) {
                stream_max[x][t] = m;
                stream_sum[x][t] = l;
                stream_up[x][t] = vup;
                if (!(ok = together())) break;
                const float m0 = stream_max[0][t], m1 = stream_max[1][t];
                m = fmaxf(m0, m1);
                wa = fast_exp2(m0 - m);
                wb = fast_exp2(m1 - m);
                l = wa * stream_sum[0][t] + wb * stream_sum[1][t];
                wa *= stream_up[0][t];
                wb *= stream_up[1][t];
            }
            tmem_after_sync();
            const float inv = !whole ? 1.0f : l > 0.0f ? 1.0f / l : 0.0f;
            wa *= inv;
            wb *= inv;
            const int c_begin = two ? 0 : x * (D / 2), c_end = two ? D : c_begin + D / 2, rows_of = two ? x : 0;
            auto piece_of = [&](int c, int begins) { return ws.cross + (((long long)c * 2 + begins) * 2 + rows_of) * (C::kPiece / 2); };
            float* const piece = piece_of(cta, first);             // [D / 4][128][4], maxima, sums
            T* const out = static_cast<T*>(a.out) + (q0 + token) * a.out_stride_token + head * a.out_stride_head;
            const uint32_t oa = two ? o_at : tmem + lanes + 256, ob = tmem + lanes + 256 + 128;
            auto store16 = [&](int c, const float* y) {
                uint32_t w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = kv_round2<T>(y[2 * j], y[2 * j + 1]);
                *reinterpret_cast<uint4*>(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                *reinterpret_cast<uint4*>(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
            };
#pragma unroll 1
            for (int c = c_begin; c < c_end; c += 16) {
                uint32_t o[16];
                float y[16];
                tmem_ld16(o, oa + c);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j)   // INT4: decoded columns (0, 4, 1, 5, 2, 6, 3, 7) of each eight
                    y[FMT == B4_KV_INT4 ? (j & 8) | (j >> 1 & 3) | (j & 1) << 2 : j] = __uint_as_float(o[j]) * wa;
                if (!two && blocks > 1) {
                    tmem_ld16(o, ob + c);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        float& z = y[FMT == B4_KV_INT4 ? (j & 8) | (j >> 1 & 3) | (j & 1) << 2 : j];
                        z = fmaf(__uint_as_float(o[j]), wb, z);
                    }
                }
                if (whole) {
                    if (mine) store16(c, y);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        *reinterpret_cast<float4*>(piece + ((c + j) / 4 * 128 + t) * 4) = make_float4(y[j], y[j + 1], y[j + 2], y[j + 3]);
                }
                __syncwarp();
            }
            tmem_before_sync();
            if (!two && !(ok = together())) break;                 // both streams' outputs are read
            if (whole) {
                if (mine && rows_of == x && a.lse)
                    a.lse[(long long)(q0 + token) * a.heads + head] = l > 0.0f ? (m + fast_log2(l)) * kLn2 : -INFINITY;
                continue;
            }
            if (rows_of == x) {
                piece[128 * D + t] = m;
                piece[128 * (D + 1) + t] = l;
            }
            // the last of the segment's CTAs joins them, in order
            const int f = owner(s0), parts = owner(s1 - 1) - f + 1;
            if (!(ok = together())) break;
            if (tid == 128) {
                joins = count_in(ws.count + f) == parts - 1;
                if (joins) ws.count[f] = 0;
            }
            if (!(ok = together())) break;
            const bool join = joins;
            if (!(ok = together())) break;     // before the flag is written again
            if (!join) continue;
            float jt = kNoMax, sum = 0.0f;
#pragma unroll 4
            for (int i = 0; i < parts; ++i) jt = fmaxf(jt, __ldcg(piece_of(f + i, i == 0) + 128 * D + t));
            constexpr int E = D / 2;           // columns at a time
#pragma unroll 1
            for (int c = c_begin; c < c_end; c += E) {
                float y[E];
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] = 0.0f;
                sum = 0.0f;
#pragma unroll 1
                for (int i = 0; i < parts; ++i) {
                    const float* b = piece_of(f + i, i == 0);
                    float4 z[E / 4];
#pragma unroll
                    for (int e = 0; e < E / 4; ++e) z[e] = __ldcg(reinterpret_cast<const float4*>(b) + (c / 4 + e) * 128 + t);
                    const float w = fast_exp2(__ldcg(b + 128 * D + t) - jt);
                    sum = fmaf(w, __ldcg(b + 128 * (D + 1) + t), sum);
#pragma unroll
                    for (int e = 0; e < E / 4; ++e) {
                        y[4 * e] = fmaf(w, z[e].x, y[4 * e]);
                        y[4 * e + 1] = fmaf(w, z[e].y, y[4 * e + 1]);
                        y[4 * e + 2] = fmaf(w, z[e].z, y[4 * e + 2]);
                        y[4 * e + 3] = fmaf(w, z[e].w, y[4 * e + 3]);
                    }
                }
                const float jinv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) y[e] *= jinv;
                if (mine) {
#pragma unroll
                    for (int e = 0; e < E; e += 16) store16(c + e, y + e);
                }
            }
            if (mine && rows_of == x && a.lse)
                a.lse[(long long)(q0 + token) * a.heads + head] = sum > 0.0f ? (jt + fast_log2(sum)) * kLn2 : -INFINITY;
        }
    }
    tmem_before_sync();
    __syncthreads();
    tmem_after_sync();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
}

}  // namespace b4
