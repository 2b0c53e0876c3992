// C[m, n] = T((sum_k A[m, k] B[n, k]) * (a_scales[m] * b_scales[n])): the
// product of 8-bit integer rows A (M x K, a scale per token) and B (N x K, a
// weight [out, in] with a scale per output channel), accumulated exactly in
// 32-bit integers (|sum| <= 2^14 K < 2^31 for K <= 131071) and rounded to T
// once, from the fp32 product of the sum and the two scales.
//
// Both operands are K-major, so a k block of 128 bytes is one 128-byte
// swizzled row: the tiles, descriptors and rings are those of a 16-bit
// product of half the depth (tcgen05.mma.kind::i8, 32 k per instruction).
// Two kernels:
//   * linear_int8_tile_kernel: BM x bn tiles (BM 64 or 128, bn 32 .. 256),
//     K split over a cluster of up to 8 CTAs; for decode batches, bound by
//     streaming B once, and for short prompts; also for operands that TMA cannot
//     address (a base or a row stride that is no multiple of 16 bytes), whose
//     rows its idle warps bring to shared memory instead;
//   * linear_int8_pair_kernel: two SMs per 256 x 256 tile
//     (cta_group::2), persistent, two accumulators; for prefill.
// Every mbarrier wait is bounded; on expiry the kernel records an error code
// (l2k_device_error) and leaves after its copies and MMAs have drained.
#include "common.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <type_traits>

namespace l2k
{

__device__ int g_int8_error = 0; // first error code recorded by a kernel of this file

namespace
{

constexpr int kBK = 128;     // k per block: one swizzled 128-byte row
constexpr int kMaxK = 131071;

enum Int8Error
{
    ERR_INT8_WAIT_LOAD = 0x701,
    ERR_INT8_WAIT_MMA = 0x702,
    ERR_INT8_WAIT_DONE = 0x703,
    ERR_INT8_SMEM_ALIGN = 0x704
};

__device__ __forceinline__ void int8_fail(int code, volatile int *abort_flag)
{
    atomicCAS(&g_int8_error, 0, code);
    *abort_flag = 1;
}

struct Int8Args
{
    const int8_t *a, *b;
    int64_t lda, ldb;
    const float *sa, *sb;
    void *c;
    int64_t ldc;
    int64_t m, n, k;
    int n_kb; // k blocks
    int n_nt; // pair kernel: column tiles
    int wide; // C rows are 16-byte aligned: 16-byte stores
    // tile kernel
    int bn;                           // columns per tile (a multiple of 32)
    int split;                        // CTAs per cluster sharing one C tile, each a K range
    int kb_per, kb_more;              // k blocks per rank; ranks that take one more
    int groups;                       // rings and accumulators per CTA
    int stages;                       // stages of all rings
    uint32_t stage_bytes, ring_bytes; // (TileShape)
};

// kind::i8: D s32 (2), A and B signed (1), both K-major.
__host__ __device__ constexpr uint32_t int8_instr_desc(uint32_t m, uint32_t n)
{
    return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

__device__ __forceinline__ void mma_i8(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc,
                                            uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same without ordering memory: only that every thread has got here.
__device__ __forceinline__ void cluster_barrier_relaxed()
{
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
}
__device__ __forceinline__ int64_t ceil_div_dev(int64_t a, int64_t b) { return (a + b - 1) / b; }
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr)
{
    uint32_t r;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(r) : "r"(addr) : "memory");
    return r;
}

// 16 consecutive accumulator columns of this thread's TMEM lane (no wait).
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}

// One thread of a converged warp, known to the compiler as one: the tensor-core
// and TMA instructions behind it are issued once. Behind a comparison with a
// thread index each took about 80 cycles to issue instead, which set the pace
// of the k loop (900 cycles a block, whatever its size).
__device__ __forceinline__ bool elect_one()
{
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// A whole warp's wait; the same answer in every lane. Bounded like mbar_wait,
// whose clock and flag are read only when the phase is not complete yet.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const volatile int *abort_flag)
{
    bool ok = mbar_try(bar, parity);
    if (!__all_sync(0xffffffffu, ok))
        ok = __all_sync(0xffffffffu, ok || mbar_wait(bar, parity, abort_flag));
    return ok;
}

// Columns [col, col + 8) of a row of C from their integer sums and b_scales: three
// fp32 roundings (the sum beyond 2^24, the product of the scales, the product of
// both) and one to T. `n`: columns of C from col on.
template <typename T>
__device__ __forceinline__ void store8(T *out, const uint32_t *r, float row_scale, const float *sb, int64_t n, bool wide)
{
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
        o[e] = from_f<T>(__fmul_rn((float)(int)r[e], __fmul_rn(row_scale, sb[e])));
    if (wide && n >= 8)
    {
        uint4 w[sizeof(T) / 2];
        __builtin_memcpy(w, o, sizeof(o));
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
            stg(out + 16 / sizeof(T) * i, w[i]);
    }
    else
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n)
                out[e] = o[e];
    }
}

// 32 consecutive columns of this lane's row, from their integer sums, into row
// `lane` of a 128-byte-swizzled staging tile, from its column c on. sb: the b_scale
// of the lane-th of these columns.
template <typename T>
__device__ __forceinline__ void scale_to_rows(const uint32_t (&r)[32], float row_scale, float sb, uint8_t *staging, int lane,
                                              int c)
{
    constexpr int N = Vec16<T>::N;
#pragma unroll
    for (int v = 0; v < 32 / N; ++v)
    {
        Vec16<T> o;
#pragma unroll
        for (int e = 0; e < N; ++e)
            o.v[e] = from_f<T>(__fmul_rn((float)(int)r[N * v + e],
                                         __fmul_rn(row_scale, __shfl_sync(0xffffffffu, sb, N * v + e))));
        const int unit = (c / N + v) ^ (lane & 7); // the 16-byte units of a row, permuted by the row
        *reinterpret_cast<uint4 *>(staging + 128 * lane + 16 * unit) = as_u4(o);
    }
}

template <typename T>
__device__ __forceinline__ T staged(const uint8_t *staging, int row, int col)
{
    constexpr int N = Vec16<T>::N;
    return *reinterpret_cast<const T *>(staging + 128 * row + 16 * ((col / N) ^ (row & 7)) + sizeof(T) * (col % N));
}

// ---------------------------------------------------------------------------
// One BM x bn tile per cluster of `split` CTAs, each a K range. Within a CTA the
// k blocks are dealt to `groups` (1, 2 or 4) of one producer and one MMA warp
// each, with a ring and an accumulator of their own, because one warp needs
// about 350 cycles for a block's wait, four MMAs and commit where the tensor
// cores need 32 to 128 per MMA. A producer warp initialises its own barriers and
// issues its first loads at once, before tensor memory is allocated. The
// epilogue adds the accumulators; integer sums do not depend on the dealing.
//
// split > 1 (or rows of C without 16-byte alignment, whose stores should be to
// neighbours): every rank leaves its partial tile in its own shared memory (the
// drained ring). After a cluster barrier each rank adds its rows [q rows_per,
// (q + 1) rows_per) into rank q's copy with one bulk reduction, and rank q
// scales and stores those rows once all have landed. A last barrier keeps every
// copy alive until it has been read. A rank that has failed takes the same steps, so
// that every reduction lands before its CTAs leave; each rank reads the others' failure
// flags while the reductions are on their way, and stores nothing if one is set.
//
// The A box has a.a_rows rows (m rounded up to 8). The MMA reads BM: the rest is
// whatever follows in shared memory (a stage lies BM rows from its end at the
// latest) and only reaches accumulator rows that are never read.
// ---------------------------------------------------------------------------
constexpr int kTThreads = 512;
constexpr int kTMaxStages = 32;
constexpr uint32_t kTRing = 208 * 1024; // bytes of shared memory for the ring at most
constexpr int kTMaxSmem = 227 * 1024;

// Shared memory: the ring (or the staged partial tile), bn scales, the barriers,
// the TMEM address and the abort flag.
struct TileShape
{
    int bm, bn, split, groups, stages;
    uint32_t stage_bytes, ring_bytes, smem_bytes;
    int a_rows;
};
inline TileShape tile_shape(int64_t m, int bm, int bn, int split, int groups, bool stage)
{
    TileShape t{bm, bn, split, groups, 0, 0, 0, 0, 0};
    t.a_rows = (int)std::min<int64_t>(bm, ceil_div(m, 8) * 8);
    t.stage_bytes = (uint32_t)(bn + t.a_rows) * 128;
    const uint32_t slack = (uint32_t)(bm - t.a_rows) * 128; // what the last stage's MMAs read past its A rows
    t.stages = (int)std::min<uint32_t>(kTMaxStages, (kTRing - slack) / t.stage_bytes) / groups * groups;
    const uint32_t staged = stage ? (uint32_t)bm * (bn + 4) * 4 : 0;
    t.ring_bytes = (std::max(t.stages * t.stage_bytes + slack, staged) + 1023) & ~1023u;
    t.smem_bytes = t.ring_bytes + 4 * (uint32_t)bn + 8 * (2 * kTMaxStages + 2) + 16;
    return t;
}

// Adds `bytes` of this CTA's shared memory at `src` to another CTA's at `dst`
// as 32-bit integers, signalling its mbarrier (both shared::cluster addresses).
__device__ __forceinline__ void bulk_add_s32(uint32_t dst, uint32_t src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.reduce.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes.add.s32 [%0], [%1], %2, "
                 "[%3];" ::"r"(dst),
                 "r"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// 16 bytes of a row from any address: those below `valid`, zeros behind. Reads the
// aligned words around them where these lie in [lo, hi), the operand's bytes.
__device__ __forceinline__ uint4 load_unaligned16(const int8_t *p, int64_t valid, uintptr_t lo, uintptr_t hi)
{
    uint32_t v[4] = {0, 0, 0, 0};
    const uintptr_t first = (uintptr_t)p & ~(uintptr_t)3;
    if (valid > 0 && first >= lo && first + 20 <= hi)
    {
        const uint32_t *w = reinterpret_cast<const uint32_t *>(first);
        const uint32_t shift = 8 * (uint32_t)((uintptr_t)p & 3);
        uint32_t x[5];
#pragma unroll
        for (int i = 0; i < 5; ++i)
            x[i] = ldg_coherent_u32(w + i);
#pragma unroll
        for (int i = 0; i < 4; ++i)
        {
            v[i] = __funnelshift_r(x[i], x[i + 1], shift);
            const int64_t n = valid - 4 * i; // bytes of the word that belong to the row
            v[i] = n >= 4 ? v[i] : n <= 0 ? 0u : v[i] & ((1u << (8 * n)) - 1);
        }
    }
    else if (valid > 0)
    {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < valid)
                v[e / 4] |= (uint32_t)(uint8_t)p[e] << (8 * (e & 3));
    }
    return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T, int BM, bool TMA>
__global__ void __launch_bounds__(kTThreads, 1)
    linear_int8_tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            const __grid_constant__ Int8Args a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    if (sbase & 1023u) // (the same in every CTA: the whole cluster leaves)
    {
        if (threadIdx.x == 0)
            atomicCAS(&g_int8_error, 0, ERR_INT8_SMEM_ALIGN);
        return;
    }
    const int bn = a.bn, split = a.split, groups = a.groups;
    const int depth = a.stages / groups; // stages of one group's ring
    float *sb = reinterpret_cast<float *>(smem + a.ring_bytes);
    const uint32_t bar_full = sbase + a.ring_bytes + 4 * bn; // + 8 * stage: the stage's tiles landed
    const uint32_t bar_freed = bar_full + 8 * kTMaxStages;   // + 8 * stage: the MMAs reading it completed
    const uint32_t bar_done = bar_freed + 8 * kTMaxStages;   // every group's MMAs completed
    const uint32_t bar_red = bar_done + 8;                   // the other ranks' rows have been added, their flags read
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + a.ring_bytes + 4 * bn + 8 * (2 * kTMaxStages + 2));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    const uint32_t abort_addr = smem_u32(tmem_slot + 1);

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0); // (uniform, known as such)
    const int rank = (int)blockIdx.x;
    const int64_t row0 = (int64_t)blockIdx.z * BM, col0 = (int64_t)blockIdx.y * bn;
    const int kb0 = rank * a.kb_per + min(rank, a.kb_more); // the first a.kb_more ranks take one k block more
    const int n_kb = a.kb_per + (rank < a.kb_more ? 1 : 0); // at least `groups`

    // warps 0 .. groups - 1: producers (without TMA: all warps but 4 .. 7, 12 / groups to a
    // group); warps 4 .. 3 + groups: MMA issuers
    const int group = TMA ? warp & 3 : warp & (groups - 1);
    const int count = group < groups ? (n_kb - group + groups - 1) / groups : 0; // the group's k blocks
    auto issue = [&](int i, int slot) { // the group's i-th k block into its ring's slot
        const int st = slot * groups + group;
        const uint32_t dst = sbase + st * a.stage_bytes;
        const uint32_t bar = bar_full + 8 * st;
        const int kx = (kb0 + i * groups + group) * kBK;
        mbar_expect_tx(bar, a.stage_bytes);
        tma_load_3d(dst, &tm_b, kx, (int)col0, 0, bar);
        tma_load_3d(dst + (uint32_t)bn * 128, &tm_a, kx, (int)row0, 0, bar);
    };
    int issued = 0; // producers: the group's k blocks whose loads were issued
    constexpr int kAtOnce = 2;
    pdl_trigger();
    if (warp < groups)
    {
        if (lane < depth)
        {
            mbar_init(bar_full + 8 * (lane * groups + group), TMA ? 1 : 12 / groups);
            mbar_init(bar_freed + 8 * (lane * groups + group), 1);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        pdl_wait();
        if constexpr (TMA)
        {
            issued = min(min(count, depth), kAtOnce);
            if (elect_one())
                for (int i = 0; i < issued; ++i)
                    issue(i, i);
            __syncwarp();
        }
    }
    else if (warp == 8)
    {
        if (elect_one())
        {
            mbar_init(bar_done, groups);
            mbar_init(bar_red, split);
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    else if (warp > 8)
    {
        pdl_wait();
        for (int i = tid - 9 * 32; i < bn; i += kTThreads - 9 * 32)
            sb[i] = col0 + i < a.n ? ldg_coherent_f32(a.sb + col0 + i) : 0.f;
    }
    pdl_wait(); // (every thread: the epilogue reads scales and writes C)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (!TMA && (warp < 4 || warp >= 8))
    {
        // ---- producers: the tiles' rows by plain loads, 8 lanes to a row's 128 bytes, into
        // the places that TMA's 128-byte swizzle gives them ----
        const int helpers = 12 / groups, helper = (warp < 4 ? warp : warp - 4) / groups;
        const int n_rows = (int)(a.stage_bytes / 128); // bn rows of B, then the rows of A
        const uintptr_t lo_a = (uintptr_t)a.a, hi_a = lo_a + (a.m - 1) * a.lda + a.k;
        const uintptr_t lo_b = (uintptr_t)a.b, hi_b = lo_b + (a.n - 1) * a.ldb + a.k;
        int slot = 0;
        uint32_t phase = 1; // (a fresh barrier's previous phase counts as complete)
        for (int i = 0; i < count; ++i)
        {
            const int st = slot * groups + group;
            if (!warp_wait(bar_freed + 8 * st, phase, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_MMA, abort_flag);
                break;
            }
            uint8_t *dst = smem + st * a.stage_bytes;
            const int64_t kx = (int64_t)(kb0 + i * groups + group) * kBK + 16 * (lane & 7);
#pragma unroll 4
            for (int r = 4 * helper + (lane >> 3); r < n_rows; r += 4 * helpers)
            {
                const bool of_b = r < bn;
                const int64_t row = of_b ? col0 + r : row0 + r - bn;
                const bool in = row < (of_b ? a.n : a.m);
                const int8_t *p = (of_b ? a.b + row * a.ldb : a.a + row * a.lda) + kx;
                const uint4 v = load_unaligned16(p, in ? a.k - kx : 0, of_b ? lo_b : lo_a, of_b ? hi_b : hi_a);
                *reinterpret_cast<uint4 *>(dst + 128 * r + 16 * ((lane & 7) ^ (r & 7))) = v;
            }
            fence_proxy_async(); // before the MMAs read them
            __syncwarp();
            if (lane == 0)
                mbar_arrive(bar_full + 8 * st);
            if (++slot == depth)
            {
                slot = 0;
                phase ^= 1;
            }
        }
    }
    else if (TMA && warp < groups)
    {
        // ---- producer: the rest of the group's k blocks ----
        int slot = issued;
        if (elect_one())
            for (; slot < depth && slot < count; ++slot)
                issue(slot, slot);
        __syncwarp();
        issued = min(count, depth);
        uint32_t phase = 0;
        slot = 0;
        for (int i = issued; i < count; ++i)
        {
            if (!warp_wait(bar_freed + 8 * (slot * groups + group), phase, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_MMA, abort_flag);
                break;
            }
            if (elect_one())
                issue(i, slot);
            __syncwarp();
            issued = i + 1;
            if (++slot == depth)
            {
                slot = 0;
                phase ^= 1;
            }
        }
    }
    else if (warp >= 4 && warp < 4 + groups)
    {
        // ---- MMA issuer ----
        const uint32_t idesc = int8_instr_desc(BM, (uint32_t)bn);
        const uint32_t acc = tmem + (uint32_t)(group * bn);
        int slot = 0, i = 0;
        uint32_t phase = 0;
        for (; i < count; ++i)
        {
            const int st = slot * groups + group;
            if (!warp_wait(bar_full + 8 * st, phase, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_LOAD, abort_flag);
                break;
            }
            tc_fence_after();
            if (elect_one())
            {
                const uint32_t pb = sbase + st * a.stage_bytes;
                const uint64_t da = smem_desc(pb + (uint32_t)bn * 128), db = smem_desc(pb);
#pragma unroll
                for (int k = 0; k < kBK / 32; ++k) // 32 bytes on along the rows: 2 units of 16
                    mma_i8(acc, da + 2u * k, db + 2u * k, idesc, (i | k) ? 1u : 0u);
                mma_commit(bar_freed + 8 * st);
                if (i + 1 == count)
                    mma_commit(bar_done);
            }
            __syncwarp();
            if (++slot == depth)
            {
                slot = 0;
                phase ^= 1;
            }
        }
        if (i < count && elect_one())
            mma_commit(bar_done); // after a failure: what was issued
        __syncwarp();
    }

    // warps of the same warp % 4 read TMEM lane quadrant warp % 4: row 32 quad + lane of the
    // tile, or (BM 64) row 16 quad + lane in lanes 0-15; they share its columns, 16 at a time
    const int quad = warp & 3, part = warp >> 2;
    const int lrow = BM == 64 ? 16 * quad + lane : 32 * quad + lane;
    const bool live = (BM == 128 || lane < 16) && row0 + lrow < a.m;
    const float row_scale = live ? ldg_coherent_f32(a.sa + row0 + lrow) : 0.f;
    if (!mbar_wait(bar_done, 0, abort_flag))
        int8_fail(ERR_INT8_WAIT_DONE, abort_flag);
    if (*abort_flag && warp < groups && lane == 0)
    {
        // after a failure the copies and MMAs in flight land before the ring is reused
        const int quiet = 0;
        for (int i = max(0, issued - depth); i < issued; ++i) // (none without TMA)
            mbar_wait(bar_full + 8 * ((i % depth) * groups + group), (i / depth) & 1, &quiet);
        mbar_wait(bar_done, 0, &quiet);
    }
    __syncwarp();
    tc_fence_after();
    // the integer sums of accumulator columns [c0, c0 + 16) of this thread's row
    auto load16 = [&](int c0, uint32_t(&r)[16]) {
        const uint32_t taddr = tmem + ((uint32_t)(32 * quad) << 16) + (uint32_t)c0;
        tmem_ld16_async(taddr, r);
        if (groups > 1)
        {
            uint32_t x[16];
            tmem_ld16_async(taddr + (uint32_t)bn, x);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
                r[e] += x[e];
        }
        if (groups > 2)
        {
            uint32_t x[16], y[16];
            tmem_ld16_async(taddr + (uint32_t)(2 * bn), x);
            tmem_ld16_async(taddr + (uint32_t)(3 * bn), y);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e)
                r[e] += x[e] + y[e];
        }
        tmem_wait_ld();
    };
    if (split == 1 && a.wide)
    {
        T *out = static_cast<T *>(a.c) + (row0 + lrow) * a.ldc + col0;
#pragma unroll 1
        for (int c0 = 16 * part; c0 < bn; c0 += 64)
        {
            uint32_t r[16];
            load16(c0, r);
            if (live && !*abort_flag)
            {
#pragma unroll
                for (int v = 0; v < 16; v += 8)
                    store8<T>(out + c0 + v, r + v, row_scale, sb + c0 + v, a.n - col0 - c0 - v, true);
            }
            __syncwarp();
        }
    }
    else
    {
        tc_fence_before();
        __syncthreads(); // (after a failure: the ring is quiet)
        tc_fence_after();
        const int stride = bn + 4; // integers per staged row (16-byte shift per row: no bank conflicts)
        const int m_tile = (int)std::min<int64_t>(BM, a.m - row0);
        const int rows_per = (m_tile + split - 1) / split;
        auto rows_of = [&](int q) { return max(0, min(m_tile, (q + 1) * rows_per) - q * rows_per); };
        const int mine = rows_of(rank);
        int *stage = reinterpret_cast<int *>(smem);
#pragma unroll 1
        for (int c0 = 16 * part; c0 < bn; c0 += 64)
        {
            uint32_t r[16];
            load16(c0, r);
            if (live)
            {
                int4 *dst = reinterpret_cast<int4 *>(stage + lrow * stride + c0);
#pragma unroll
                for (int v = 0; v < 4; ++v)
                    dst[v] = make_int4((int)r[4 * v], (int)r[4 * v + 1], (int)r[4 * v + 2], (int)r[4 * v + 3]);
            }
            __syncwarp();
        }
        fence_proxy_async(); // the staged rows, before the bulk reductions from and to them
        if (tid == 0 && mine > 0)
            mbar_expect_tx(bar_red, (uint32_t)((split - 1) * mine * stride * 4));
        __syncwarp();
        cluster_barrier(); // every rank's partial is in its shared memory
        if (warp < split && warp != rank && elect_one())
        {
            if (rows_of(warp) > 0)
            {
                const uint32_t src = sbase + (uint32_t)(warp * rows_per * stride) * 4;
                bulk_add_s32(cluster_addr(src, (uint32_t)warp), src, (uint32_t)(rows_of(warp) * stride * 4),
                             cluster_addr(bar_red, (uint32_t)warp));
            }
            if (ld_cluster_u32(cluster_addr(abort_addr, (uint32_t)warp)) != 0) // (its partial is incomplete)
                *abort_flag = 1;
            mbar_arrive(bar_red);
        }
        __syncwarp();
        const int quiet = 0; // (after a failure too: what is being added here lands first)
        if (mine > 0 && !mbar_wait(bar_red, 0, &quiet))
            int8_fail(ERR_INT8_WAIT_DONE, abort_flag);
        // this rank's rows in runs of 8 columns; a warp's lanes take neighbouring runs
        const int runs = bn / 8, items = runs * mine;
        if (!*abort_flag)
            for (int i = tid; i < items; i += kTThreads)
            {
                const int rr = rank * rows_per + i / runs, c = (i % runs) * 8;
                uint32_t r[8];
                *reinterpret_cast<int4 *>(r) = *reinterpret_cast<const int4 *>(stage + rr * stride + c);
                *reinterpret_cast<int4 *>(r + 4) = *reinterpret_cast<const int4 *>(stage + rr * stride + c + 4);
                store8<T>(static_cast<T *>(a.c) + (row0 + rr) * a.ldc + col0 + c, r,
                          ldg_coherent_f32(a.sa + row0 + rr), sb + c, a.n - col0 - c, a.wide);
            }
        __syncwarp();
        cluster_barrier_relaxed(); // no rank leaves while another may still read its partial
    }

    // -------- teardown --------
    tc_fence_before();
    __syncthreads();
    if (warp == 8)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// ---------------------------------------------------------------------------
// Two SMs per 256 x 256 tile (tcgen05.mma.cta_group::2, M = 256, N = 256):
// CTA rank r of the pair holds rows [128 r, 128 r + 128) of the A tile and of
// the B tile in its shared memory, at the same offsets, and receives rows
// [128 r, 128 r + 128) of the accumulator in its tensor memory. Warp 0 of each
// CTA streams its halves through the ring, the loads completing on rank 0's
// "full" barrier; warp 1 of rank 0 issues the MMAs and commits to both CTAs'
// "empty" and "accumulator full" barriers; warps 2-9 of each CTA scale and
// store their 128 rows while the next tile's MMAs fill the other accumulator,
// and release theirs on rank 0's "accumulator empty" barrier. The pairs walk
// the tiles persistently.
// ---------------------------------------------------------------------------
constexpr int kPThreads = 64 + 256;                 // producer warp, MMA warp, epilogue warps
constexpr int kPStages = 6;
constexpr uint32_t kPHalf = 128 * 128;              // one CTA's half of an operand: 128 rows x 128 k
constexpr uint32_t kPStageBytes = 2 * kPHalf;
constexpr uint32_t kPOffOut = kPStages * kPStageBytes;    // 32 rows x 128 bytes of C per epilogue warp
constexpr uint32_t kPOffBar = kPOffOut + 8 * 4096;
constexpr uint32_t kPOffMisc = kPOffBar + 8 * (2 * kPStages + 4);
constexpr uint32_t kPSmemBytes = kPOffMisc + 16;

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar_cluster)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, "
                 "{%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(map), "r"(x), "r"(y), "r"(0), "r"(bar_cluster)
                 : "memory");
}
// Arrives on the mbarrier at `bar` (same offset) in both CTAs of the pair once
// the MMAs issued so far have completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::
                     "r"(bar),
                 "h"((uint16_t)3)
                 : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster)
{
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster) : "memory");
}

// The tile's row and column of tiles: bands of 16 columns, each walked row by row,
// so that the tiles in flight (74 on B200) share 16 tiles of B and about 5 of A in
// L2 (row by row over all columns: 8192 x 27648 x 5120 885 us, 743 in bands).
constexpr int64_t kPBand = 16;
struct TileAt
{
    int64_t row, col;
};
__device__ __forceinline__ TileAt tile_at(int64_t tile, int64_t m_tiles, int64_t n_tiles)
{
    const int64_t band = tile / (m_tiles * kPBand), rest = tile - band * m_tiles * kPBand;
    const int64_t width = n_tiles - band * kPBand < kPBand ? n_tiles - band * kPBand : kPBand;
    return TileAt{rest / width, band * kPBand + rest % width};
}

template <typename T>
__global__ void __launch_bounds__(kPThreads, 1)
    linear_int8_pair_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            const __grid_constant__ CUtensorMap tm_c, const __grid_constant__ Int8Args a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const bool leader = rank == 0;
    const uint32_t bar_full = sbase + kPOffBar;             // + 8 * stage (rank 0's are the live ones)
    const uint32_t bar_empty = bar_full + 8 * kPStages;     // + 8 * stage
    const uint32_t bar_acc_full = bar_empty + 8 * kPStages; // + 8 * accumulator
    const uint32_t bar_acc_empty = bar_acc_full + 16;       // + 8 * accumulator (rank 0's are the live ones)
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + kPOffMisc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(smem + kPOffMisc + 8);

    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0); // (uniform, known as such)
    const int64_t m_tiles = ceil_div_dev(a.m, 256), n_tiles = m_tiles * a.n_nt;
    const int64_t cluster_id = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
    const int n_kb = a.n_kb;
    const bool misaligned = (sbase & 1023u) != 0; // uniform over the cluster (same layout); acted on after the sync

    if (tid == 0)
    {
        for (int i = 0; i < kPStages; ++i)
        {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_empty + 8 * i, 1);
        }
        for (int b = 0; b < 2; ++b)
        {
            mbar_init(bar_acc_full + 8 * b, 1);
            mbar_init(bar_acc_empty + 8 * b, 2 * 8); // both CTAs' epilogue warps
        }
        *abort_flag = misaligned ? 1 : 0;
        if (misaligned)
            atomicCAS(&g_int8_error, 0, ERR_INT8_SMEM_ALIGN);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1)
    {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    pdl_trigger();
    tc_fence_before();
    __syncthreads();
    pdl_wait();
    cluster_barrier(); // both CTAs' barriers are initialized and the tensor memory allocated
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t full0 = cluster_addr(bar_full, 0);           // rank 0's full barriers
    const uint32_t acc_empty0 = cluster_addr(bar_acc_empty, 0); // rank 0's accumulator-empty barriers

    int64_t issued = 0;    // producer: k blocks whose loads were issued
    int64_t mma_done = -1; // rank 0's MMA warp: the last k block whose MMAs were committed
    if (warp == 0)
    {
        int st = 0;
        uint32_t phase = 1; // (a fresh barrier's previous phase counts as complete)
        for (int64_t tile = cluster_id; tile < n_tiles && !misaligned; tile += n_clusters)
        {
            const TileAt t = tile_at(tile, m_tiles, a.n_nt);
            const int row0 = (int)t.row * 256 + 128 * (int)rank, col0 = (int)t.col * 256 + 128 * (int)rank;
            int kb = 0;
            for (; kb < n_kb; ++kb)
            {
                if (!warp_wait(bar_empty + 8 * st, phase, abort_flag))
                {
                    int8_fail(ERR_INT8_WAIT_MMA, abort_flag);
                    break;
                }
                if (elect_one())
                {
                    const uint32_t dst = sbase + st * kPStageBytes;
                    if (leader)
                        mbar_expect_tx(bar_full + 8 * st, 2 * kPStageBytes); // both CTAs' halves
                    tma_load_pair(dst, &tm_a, kb * kBK, row0, full0 + 8 * st);
                    tma_load_pair(dst + kPHalf, &tm_b, kb * kBK, col0, full0 + 8 * st);
                }
                __syncwarp();
                ++issued;
                if (++st == kPStages)
                {
                    st = 0;
                    phase ^= 1;
                }
            }
            if (kb < n_kb)
                break;
        }
    }
    else if (warp == 1)
    {
        if (leader)
        {
            const uint32_t idesc = int8_instr_desc(256, 256);
            int st = 0;
            uint32_t phase = 0;
            int64_t lt = 0;
            for (int64_t tile = cluster_id; tile < n_tiles && !misaligned; tile += n_clusters, ++lt)
            {
                const int buf = (int)(lt & 1);
                if (!warp_wait(bar_acc_empty + 8 * buf, (uint32_t)((lt >> 1) & 1) ^ 1u, abort_flag))
                {
                    int8_fail(ERR_INT8_WAIT_DONE, abort_flag);
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem + (uint32_t)(buf * 256);
                int kb = 0;
                for (; kb < n_kb; ++kb)
                {
                    if (!warp_wait(bar_full + 8 * st, phase, abort_flag))
                    {
                        int8_fail(ERR_INT8_WAIT_LOAD, abort_flag);
                        break;
                    }
                    tc_fence_after();
                    if (elect_one())
                    {
                        const uint32_t pa = sbase + st * kPStageBytes;
                        const uint64_t da = smem_desc(pa), db = smem_desc(pa + kPHalf);
#pragma unroll
                        for (int k = 0; k < kBK / 32; ++k) // 32 bytes on along the rows: 2 units of 16
                            mma_i8_pair(acc, da + 2u * k, db + 2u * k, idesc, (kb | k) ? 1u : 0u);
                        mma_commit_pair(bar_empty + 8 * st); // both CTAs may refill the stage
                        if (kb + 1 == n_kb)
                            mma_commit_pair(bar_acc_full + 8 * buf);
                    }
                    __syncwarp();
                    ++mma_done;
                    if (++st == kPStages)
                    {
                        st = 0;
                        phase ^= 1;
                    }
                }
                if (kb < n_kb)
                    break;
            }
        }
    }
    else
    {
        // epilogue warps 2..: TMEM lane quadrant warp % 4 holds rows 32 (warp % 4) + lane of this CTA's half;
        // the two warps of a quadrant share its columns
        const int quad = warp & 3, part = (warp - 2) >> 2;
        uint8_t *staging = smem + kPOffOut + 4096 * (warp - 2);
        int64_t lt = 0;
        for (int64_t tile = cluster_id; tile < n_tiles && !*abort_flag; tile += n_clusters, ++lt)
        {
            const int buf = (int)(lt & 1);
            const TileAt t = tile_at(tile, m_tiles, a.n_nt);
            const int64_t row = t.row * 256 + 128 * (int64_t)rank + 32 * quad + lane, col0 = t.col * 256 + 128 * part;
            const bool store = row < a.m;
            const float row_scale = store ? ldg_coherent_f32(a.sa + row) : 0.f;
            float sb[4]; // the scales of this warp's columns 32 i + lane
#pragma unroll
            for (int i = 0; i < 4; ++i)
                sb[i] = col0 + 32 * i + lane < a.n ? ldg_coherent_f32(a.sb + col0 + 32 * i + lane) : 0.f;
            if (!mbar_wait(bar_acc_full + 8 * buf, (uint32_t)(lt >> 1) & 1u, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_DONE, abort_flag);
                break;
            }
            __syncwarp();
            tc_fence_after();
            const uint32_t taddr = tmem + (uint32_t)(buf * 256 + 128 * part) + ((uint32_t)(32 * quad) << 16);
            if (a.wide)
            {
                // through shared memory (128-byte swizzle) and TMA, 32 rows x 128 bytes at a time:
                // whole lines, where each lane's own 16-byte stores touch 32 lines per instruction
                constexpr int kCols = 128 / (int)sizeof(T); // columns per store: 64 or 32
#pragma unroll
                for (int c0 = 0; c0 < 128; c0 += kCols)
                {
                    bulk_wait_read_0(); // the previous store has read the staging rows
                    __syncwarp();
#pragma unroll
                    for (int h = 0; h < kCols; h += 32)
                    {
                        uint32_t r[32];
                        tmem_ld32_async(taddr + (uint32_t)(c0 + h), r);
                        tmem_wait_ld();
                        scale_to_rows<T>(r, row_scale, sb[(c0 + h) / 32], staging, lane, h);
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (col0 + c0 < a.n && row - lane < a.m && elect_one())
                        tma_store_3d(&tm_c, smem_u32(staging), (int)(col0 + c0), (int)(row - lane), 0);
                    bulk_commit(); // (an empty group in the other lanes)
                }
            }
            else
            {
                // rows of no 16-byte alignment: staged the same way, then a row at a time, a warp's
                // lanes storing neighbouring elements
                const int64_t rows = a.m - (row - lane);
                T *out = static_cast<T *>(a.c) + (row - lane) * a.ldc + col0;
#pragma unroll
                for (int c0 = 0; c0 < 128; c0 += 32)
                {
                    uint32_t r[32];
                    tmem_ld32_async(taddr + (uint32_t)c0, r);
                    tmem_wait_ld();
                    scale_to_rows<T>(r, row_scale, sb[c0 / 32], staging, lane, 0);
                    __syncwarp();
                    const bool in = col0 + c0 + lane < a.n;
                    for (int i = 0; i < 32 && i < rows; ++i)
                        if (in)
                            out[i * a.ldc + c0 + lane] = staged<T>(staging, i, lane);
                    __syncwarp();
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive_cluster(acc_empty0 + 8 * buf);
        }
        bulk_wait_read_0(); // the last stores have read their rows
    }

    // -------- teardown: after a failure, copies and MMAs in flight land first --------
    if (*abort_flag)
    {
        const int quiet = 0;
        if (tid == 32 && leader && mma_done >= 0)
            mbar_wait(bar_empty + 8 * (int)(mma_done % kPStages), (uint32_t)(mma_done / kPStages) & 1u, &quiet);
        if (tid == 0 && leader)
            for (int64_t it = issued > kPStages ? issued - kPStages : 0; it < issued; ++it)
                mbar_wait(bar_full + 8 * (int)(it % kPStages), (uint32_t)(it / kPStages) & 1u, &quiet);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_barrier(); // no CTA leaves while its peer may still signal its barriers or read its tensor memory
    if (warp == 1)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

int cuda_status(cudaError_t e)
{
    if (e == cudaSuccess)
        return L2K_OK;
    (void)cudaGetLastError(); // (else the next launch would report it again)
    return set_error(L2K_ERR_CUDA, "l2k_linear_int8: %s", cudaGetErrorString(e));
}

// K = 0: every sum is 0, every element 0 times its scales.
template <typename T>
__global__ void linear_int8_empty_kernel(const Int8Args a)
{
    for (int64_t row = blockIdx.y; row < a.m; row += gridDim.y)
        for (int64_t col = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; col < a.n; col += (int64_t)gridDim.x * blockDim.x)
            static_cast<T *>(a.c)[row * a.ldc + col] = from_f<T>(__fmul_rn(0.f, __fmul_rn(a.sa[row], a.sb[col])));
}

template <typename T, int BM, bool TMA>
int launch_tile(Int8Args a, int bn, int split, int groups, cudaStream_t stream)
{
    while (groups > 1 && (groups * bn > 512 || groups > a.n_kb / split)) // 512 TMEM columns, a k block for each
        groups /= 2;
    const TileShape t = tile_shape(a.m, BM, bn, split, groups, split > 1 || !a.wide);
    a.bn = bn;
    a.split = split;
    a.kb_per = a.n_kb / split;
    a.kb_more = a.n_kb % split;
    a.groups = groups;
    a.stages = t.stages;
    a.stage_bytes = t.stage_bytes;
    a.ring_bytes = t.ring_bytes;
    CUtensorMap ma = {}, mb = {};
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t m = (uint64_t)a.m, n = (uint64_t)a.n, k = (uint64_t)a.k, lda = (uint64_t)a.lda, ldb = (uint64_t)a.ldb;
    if (TMA && (!make_map(&ma, dt, a.a, k, m, 1, lda, lda * m, (uint32_t)t.a_rows, kBK) ||
                !make_map(&mb, dt, a.b, k, n, 1, ldb, ldb * n, (uint32_t)bn, kBK)))
        return set_error(L2K_ERR_CUDA, "l2k_linear_int8: tensor map encoding failed");
    auto kernel = linear_int8_tile_kernel<T, BM, TMA>;
    const int st = cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTMaxSmem));
    if (st != L2K_OK)
        return st;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)split, (unsigned)ceil_div(a.n, bn), (unsigned)ceil_div(a.m, BM));
    cfg.blockDim = dim3(kTThreads);
    cfg.dynamicSmemBytes = t.smem_bytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = pdl_attribute();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, ma, mb, a));
}

// The two-SM kernel: 256 x 256 tiles over clusters of two CTAs.
template <typename T>
int launch_pair(Int8Args a, cudaStream_t stream)
{
    a.n_nt = (int)ceil_div(a.n, 256);
    CUtensorMap ma, mb;
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t m = (uint64_t)a.m, n = (uint64_t)a.n, k = (uint64_t)a.k, lda = (uint64_t)a.lda, ldb = (uint64_t)a.ldb;
    if (!make_map(&ma, dt, a.a, k, m, 1, lda, lda * m, 128, kBK) ||
        !make_map(&mb, dt, a.b, k, n, 1, ldb, ldb * n, 128, kBK))
        return set_error(L2K_ERR_CUDA, "l2k_linear_int8: tensor map encoding failed");
    CUtensorMap mc = {};
    if (a.wide)
    {
        const CUtensorMapDataType ct = std::is_same<T, float>::value   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                       : std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                        : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        const uint64_t ldc_bytes = (uint64_t)a.ldc * sizeof(T);
        if (!make_map(&mc, ct, a.c, n, m, 1, ldc_bytes, ldc_bytes * m, 32, 128 / sizeof(T)))
            return set_error(L2K_ERR_CUDA, "l2k_linear_int8: tensor map encoding failed");
    }
    auto kernel = linear_int8_pair_kernel<T>;
    const int st =
        cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kPSmemBytes));
    if (st != L2K_OK)
        return st;
    const int64_t tiles = ceil_div(a.m, 256) * a.n_nt;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * std::min<int64_t>(tiles, num_sms() / 2)));
    cfg.blockDim = dim3(kPThreads);
    cfg.dynamicSmemBytes = kPSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = pdl_attribute();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, ma, mb, mc, a));
}

// Which kernel, and its tiles.
struct Plan
{
    int bm, bn, split, groups; // bm 256: the two-SM kernel
};

// Clusters of `split` CTAs of the tile kernel that the device runs at once (one CTA
// per SM; cached per device).
template <typename T>
int resident_clusters(int split)
{
    static std::mutex mu;
    static int cache[64][9] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
        return 1;
    std::lock_guard<std::mutex> lock(mu);
    int &c = cache[dev][split];
    if (c == 0)
    {
        auto kernel = linear_int8_tile_kernel<T, 128, true>;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)split);
        cfg.blockDim = dim3(kTThreads);
        cfg.dynamicSmemBytes = kTRing;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = (unsigned)split;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kTMaxSmem) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess)
            (void)cudaGetLastError();
        c = n > 0 ? n : 1;
    }
    return c;
}

// The least estimated time, in SM clocks. The estimate was fitted to 2 900 timings
// (165 sizes of 1 to 3000 rows, 300 to 32000 columns and 512 to 13824 k, under
// every tile, split and group count): its choice takes 0.9 % longer than the best
// of each size on the average, 16 % at worst. A tile's k block takes the longest
// of its MMAs (2 bn), its issue (450 shared by the groups) and its bytes at 79 per
// clock from L2; a wave of tiles ends with its last stores (15.5 bn, and 2.2 bn for
// each further accumulator); the product takes at least its bytes at 3657 per clock
// from HBM, and 0.62 of the shorter of the two on top of the longer; then 5300 for
// launch, first loads and teardown, and for the reduction over a cluster 740 and a
// quarter of the tile's elements. The two-SM kernel: 438 a k block, 11000 once.
// Without TMA only the tile kernel, at 15 bytes per clock for what its warps move.
template <typename T>
Plan estimate(int64_t m, int64_t n, int n_kb, bool tma)
{
    const int64_t pairs = num_sms() / 2;
    const double dram = ((double)(m + n) * n_kb * kBK + 2.0 * m * n) / 3657.0;
    auto together = [&](double run) { return std::max(run, dram) + 0.62 * std::min(run, dram); };
    Plan best{256, 256, 1, 1};
    double best_t = together((double)ceil_div(ceil_div(m, 256) * ceil_div(n, 256), pairs) * n_kb * 438.0) + 11040.0;
    const int bm = m <= 64 ? 64 : 128;
    const int64_t mt = ceil_div(m, bm), a_rows = std::min<int64_t>(bm, ceil_div(m, 8) * 8);
    if (tma && (mt > 65535 || ceil_div(n, 32) > 65535 || mt * ceil_div(n, 256) > 16 * pairs))
        return best; // (many tiles: far in the two-SM kernel's range)
    if (!tma)
    {
        best = Plan{bm, 256, 1, 2};
        best_t = 1e300;
    }
    const double move = tma ? 79.0 : 15.0;
    for (int bn = 32; bn <= 256; bn += 32)
        for (int split = 1; split <= 8 && split <= n_kb; ++split)
        {
            const int64_t tiles = mt * ceil_div(n, bn), resident = resident_clusters<T>(split);
            if (split > 1 && tiles > resident)
                break; // a second wave of split tiles
            const double waves = (double)ceil_div(tiles, resident), per = (double)ceil_div(n_kb, split);
            for (int groups = bn < 128 ? 2 : 1; groups <= (bn <= 96 ? 4 : 2); groups *= 2)
            {
                if (groups > 1 && groups > n_kb / split)
                    continue;
                const double kb = std::max({2.0 * bn, 450.0 / groups, (double)(bn + a_rows) * 128 / move});
                const double run = waves * (per * kb + (15.5 + 2.2 * (groups - 1)) * bn);
                const double t = together(run) + 5337.0 + (split > 1 ? 737.0 + 0.255 * bm * bn : 0.0);
                if (t < best_t)
                {
                    best_t = t;
                    best = Plan{bm, bn, split, groups};
                }
            }
            if (bn < 128 && n_kb / split < 2) // too few k blocks for two groups
            {
                const double run = waves * (per * std::max(450.0, (double)(bn + a_rows) * 128 / move) + 15.5 * bn);
                const double t = together(run) + 5337.0 + (split > 1 ? 737.0 + 0.255 * bm * bn : 0.0);
                if (t < best_t)
                {
                    best_t = t;
                    best = Plan{bm, bn, split, 1};
                }
            }
        }
    return best;
}

// estimate(), remembered for the sizes last asked for (a pure function of them and
// the device's SM count).
template <typename T>
Plan plan(int64_t m, int64_t n, int n_kb, bool tma)
{
    struct Entry
    {
        int64_t m = -1, n = 0;
        int n_kb = 0;
        bool tma = false;
        Plan p{};
    };
    static thread_local Entry cache[64];
    Entry &e = cache[(uint64_t)(m * 31 + n * 7 + n_kb) % 64];
    if (e.m != m || e.n != n || e.n_kb != n_kb || e.tma != tma)
        e = Entry{m, n, n_kb, tma, estimate<T>(m, n, n_kb, tma)};
    return e.p;
}

template <typename T, bool TMA>
int launch_planned(const Int8Args &a, cudaStream_t stream)
{
    const Plan t = plan<T>(a.m, a.n, a.n_kb, TMA);
    if (t.bm == 64)
        return launch_tile<T, 64, TMA>(a, t.bn, t.split, t.groups, stream);
    if (t.bm == 128)
        return launch_tile<T, 128, TMA>(a, t.bn, t.split, t.groups, stream);
    return launch_pair<T>(a, stream); // (only with TMA)
}

template <typename T>
int launch_linear(const Int8Args &p, cudaStream_t stream)
{
    Int8Args a = p;
    a.wide = (a.ldc * (int64_t)sizeof(T)) % 16 == 0 && is_aligned(a.c, 16);
    a.n_kb = (int)ceil_div(a.k, kBK);
    if (a.k == 0)
    {
        const dim3 grid((unsigned)std::min<int64_t>(ceil_div(a.n, 256), 1024), (unsigned)std::min<int64_t>(a.m, 65535));
        linear_int8_empty_kernel<T><<<grid, 256, 0, stream>>>(a);
        return check_launch("l2k_linear_int8");
    }
    if (is_aligned(a.a, 16) && is_aligned(a.b, 16) && a.lda % 16 == 0 && a.ldb % 16 == 0)
    {
        if (encode_fn() == nullptr)
            return set_error(L2K_ERR_CUDA, "l2k_linear_int8: the driver has no tensor map encoder");
        return launch_planned<T, true>(a, stream);
    }
    // operands that TMA cannot address: slabs of rows and columns within the grid's limits
    const int64_t rows = (int64_t)65535 * 64, cols = (int64_t)65535 * 32;
    for (int64_t r = 0; r < a.m; r += rows)
        for (int64_t c = 0; c < a.n; c += cols)
        {
            Int8Args s = a;
            s.m = std::min(rows, a.m - r);
            s.n = std::min(cols, a.n - c);
            s.a = a.a + r * a.lda;
            s.b = a.b + c * a.ldb;
            s.sa = a.sa + r;
            s.sb = a.sb + c;
            s.c = static_cast<T *>(a.c) + r * a.ldc + c;
            const int st = launch_planned<T, false>(s, stream);
            if (st != L2K_OK)
                return st;
        }
    return L2K_OK;
}

} // namespace

int read_int8_error(bool clear)
{
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_int8_error, sizeof(int)) != cudaSuccess)
        return -1;
    if (clear && v)
    {
        const int zero = 0;
        if (cudaMemcpyToSymbol(g_int8_error, &zero, sizeof(int)) != cudaSuccess)
            return -1;
    }
    return v;
}

} // namespace l2k

extern "C" int l2k_linear_int8(int64_t m, int64_t n, int64_t k, const int8_t *a, int64_t lda, const float *a_scales,
                               const int8_t *b, int64_t ldb, const float *b_scales, void *c, int64_t ldc, int dtype,
                               l2k_stream_t stream)
{
    using namespace l2k;
    L2K_REQUIRE(dtype_ok(dtype), "l2k_linear_int8: unsupported dtype %d", dtype);
    L2K_REQUIRE(m >= 0 && n >= 0 && k >= 0, "l2k_linear_int8: negative size");
    L2K_REQUIRE(lda >= k && ldb >= k && ldc >= n, "l2k_linear_int8: leading dimension too small");
    if (m == 0 || n == 0)
        return L2K_OK;
    L2K_REQUIRE(a_scales && b_scales && c && (k == 0 || (a && b)), "l2k_linear_int8: null pointer");
    L2K_REQUIRE(is_aligned(a_scales, 4) && is_aligned(b_scales, 4) && is_aligned(c, dtype_size(dtype)),
                "l2k_linear_int8: c or the scales are not aligned to their elements");
    L2K_REQUIRE_SHAPE(k <= kMaxK, "l2k_linear_int8: k > %d could overflow a 32-bit sum", kMaxK);
    L2K_REQUIRE_SHAPE(m < (int64_t(1) << 31) && n < (int64_t(1) << 31) &&
                          ceil_div(m, 64) * ceil_div(n, 32) < (int64_t(1) << 28),
                      "l2k_linear_int8: m or n too large");
    Int8Args p{};
    p.a = a;
    p.b = b;
    p.lda = lda;
    p.ldb = ldb;
    p.sa = a_scales;
    p.sb = b_scales;
    p.c = c;
    p.ldc = ldc;
    p.m = m;
    p.n = n;
    p.k = k;
    L2K_DISPATCH(dtype, { return launch_linear<T>(p, stream); });
    return L2K_OK;
}
