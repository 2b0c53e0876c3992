// C[m, n] = T((sum_k A[m, k] B[n, k]) * (a_scales[m] * b_scales[n])): the
// product of 8-bit integer rows A (M x K, a scale per token) and B (N x K, a
// weight [out, in] with a scale per output channel), accumulated exactly in
// 32-bit integers (|sum| <= 2^14 K < 2^31 for K <= 131071) and rounded to T
// once, from the fp32 product of the sum and the two scales.
//
// Both operands are K-major, so a k block of 128 bytes is one 128-byte
// swizzled row: the tiles, descriptors and rings are those of a 16-bit
// product of half the depth (tcgen05.mma.kind::i8, 32 k per instruction).
// Three kernels:
//   * linear_int8_tile_kernel: BM x bn tiles (BM 64 or 128, bn 32 .. 256),
//     K split over a cluster of up to 8 CTAs; for decode batches, bound by
//     streaming B once, and for short prompts;
//   * linear_int8_pair_kernel: two SMs per 256 x 256 tile
//     (cta_group::2), persistent, two accumulators; for prefill;
//   * linear_int8_any_kernel: CUDA cores (dp4a), any alignment: rows that
//     TMA cannot address (a base or a row stride that is no multiple of 16).
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
    const int8_t *a, *b; // (the CUDA-core kernel)
    int64_t lda, ldb;
    const float *sa, *sb;
    void *c;
    int64_t ldc;
    int64_t m, n, k;
    int n_kb;   // k blocks
    int n_nt;   // column tiles
    int bn;     // tile kernel: columns per tile (a multiple of 32)
    int split;  // tile kernel: CTAs per cluster sharing one C tile, each a K range
    int stages; // tile kernel: ring depth
    int a_rows; // tile kernel: rows of the A box (the tile's other rows are never stored)
    int wide;   // C rows are 16-byte aligned: 16-byte stores
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
__device__ __forceinline__ int4 ld_cluster_i4(uint32_t addr)
{
    int4 v;
    asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
    return r;
}

// Columns [col, col + 32) of a row of C from their integer sums: two fp32
// roundings (the sum beyond 2^24, the product with the scales, whose own
// product is a third) and one to T.
template <typename T>
__device__ __forceinline__ void store_scaled(const Int8Args &a, const uint32_t (&r)[32], int64_t row, int64_t col,
                                             float row_scale)
{
    constexpr int N = Vec16<T>::N;
    T *out = static_cast<T *>(a.c) + row * a.ldc;
#pragma unroll
    for (int v = 0; v < 32 / N; ++v)
    {
        const int64_t cv = col + N * v;
        if (cv >= a.n)
            break;
        if (a.wide && cv + N <= a.n)
        {
            Vec16<T> o;
#pragma unroll
            for (int e = 0; e < N; ++e)
                o.v[e] = from_f<T>(__fmul_rn((float)(int)r[N * v + e], __fmul_rn(row_scale, __ldg(a.sb + cv + e))));
            stg(out + cv, as_u4(o));
        }
        else
        {
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (cv + e < a.n)
                    out[cv + e] =
                        from_f<T>(__fmul_rn((float)(int)r[N * v + e], __fmul_rn(row_scale, __ldg(a.sb + cv + e))));
        }
    }
}

// ---------------------------------------------------------------------------
// One BM x bn tile per cluster. Thread 0 initialises the barriers and issues
// the first stages' loads before tensor memory is allocated, so the first
// tiles are in flight during the set-up. With split > 1 every rank writes its
// integer partial tile to its own shared memory (the drained ring), and after
// a cluster barrier each rank sums the 32-column chunks dealt to it over all
// ranks' copies; a second barrier keeps every copy alive until its readers
// are done. Integer sums do not depend on the split.
// ---------------------------------------------------------------------------
constexpr int kTThreads = 256;
constexpr int kTMaxStages = 16;
constexpr int kTRing = 200 * 1024; // bytes of shared memory for the ring at most
constexpr uint32_t kTTmemCols = 256;

template <int BM>
struct TileCfg
{
    static constexpr uint32_t kATile = BM * 128;
    static uint32_t stage_bytes(int bn) { return kATile + (uint32_t)bn * 128; }
    static int stages(int bn) { return (int)std::min<uint32_t>(kTMaxStages, kTRing / stage_bytes(bn)); }
    // the ring (or the staged partial tile), then the barriers
    static uint32_t ring_bytes(int bn)
    {
        return std::max<uint32_t>(stages(bn) * stage_bytes(bn), (uint32_t)BM * (bn + 4) * 4 + 1008) & ~1023u;
    }
    static uint32_t smem_bytes(int bn) { return ring_bytes(bn) + 8 * (2 * kTMaxStages + 1) + 24; }
};

template <typename T, int BM>
__global__ void __launch_bounds__(kTThreads, 1)
    linear_int8_tile_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                            const __grid_constant__ Int8Args a, const uint32_t off_bar)
{
    constexpr uint32_t kATile = BM * 128;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t sbase = smem_u32(smem);
    if (sbase & 1023u) // (the same in every CTA: the whole cluster leaves)
    {
        if (threadIdx.x == 0)
            atomicCAS(&g_int8_error, 0, ERR_INT8_SMEM_ALIGN);
        return;
    }
    const int stages = a.stages, bn = a.bn, split = a.split;
    const uint32_t stage_bytes = kATile + (uint32_t)bn * 128;
    const uint32_t bar_full = sbase + off_bar;             // + 8 * stage: the stage's tiles landed
    const uint32_t bar_freed = bar_full + 8 * kTMaxStages; // + 8 * stage: the MMAs reading it completed
    const uint32_t bar_done = bar_freed + 8 * kTMaxStages; // every MMA completed
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + off_bar + 8 * (2 * kTMaxStages + 1));
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 2);

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rank = (int)(blockIdx.x % split);
    const int tile = (int)(blockIdx.x / split);
    const int64_t row0 = (int64_t)(tile / a.n_nt) * BM;
    const int64_t col0 = (int64_t)(tile % a.n_nt) * bn;
    const int kb0 = (int)((int64_t)rank * a.n_kb / split);
    const int n_kb = (int)((int64_t)(rank + 1) * a.n_kb / split) - kb0; // at least 1 (split <= n_kb)

    auto issue = [&](int kb) {
        const int st = kb % stages;
        const uint32_t dst = sbase + st * stage_bytes;
        const uint32_t bar = bar_full + 8 * st;
        mbar_expect_tx(bar, (uint32_t)(a.a_rows + bn) * 128);
        tma_load_3d(dst + kATile, &tm_b, (kb0 + kb) * kBK, (int)col0, 0, bar);
        tma_load_3d(dst, &tm_a, (kb0 + kb) * kBK, (int)row0, 0, bar);
    };

    int issued = 0; // thread 0: k blocks whose loads were issued
    if (tid == 0)
    {
        for (int i = 0; i < stages; ++i)
        {
            mbar_init(bar_full + 8 * i, 1);
            mbar_init(bar_freed + 8 * i, 1);
        }
        mbar_init(bar_done, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (; issued < n_kb && issued < stages; ++issued)
            issue(issued);
    }
    if (warp == 1)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (tid == 0)
    {
        // ---- producer: the rest of the ring ----
        for (int kb = issued; kb < n_kb && !*abort_flag; ++kb)
        {
            if (!mbar_wait(bar_freed + 8 * (kb % stages), ((kb / stages) - 1) & 1, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_MMA, abort_flag);
                break;
            }
            issue(kb);
            issued = kb + 1;
        }
    }
    else if (tid == 32)
    {
        // ---- MMA issuer ----
        const uint32_t idesc = int8_instr_desc(BM, (uint32_t)bn);
        for (int kb = 0; kb < n_kb && !*abort_flag; ++kb)
        {
            const int st = kb % stages;
            if (!mbar_wait(bar_full + 8 * st, (kb / stages) & 1, abort_flag))
            {
                int8_fail(ERR_INT8_WAIT_LOAD, abort_flag);
                break;
            }
            tc_fence_after();
            const uint32_t pa = sbase + st * stage_bytes, pb = pa + kATile;
#pragma unroll
            for (int k = 0; k < kBK / 32; ++k)
                mma_i8(tmem, smem_desc(pa + 32u * k), smem_desc(pb + 32u * k), idesc, (kb | k) ? 1u : 0u);
            mma_commit(bar_freed + 8 * st);
        }
        mma_commit(bar_done);
    }
    __syncwarp();

    // warps w and w + 4 read TMEM lane quadrant w: row 32 w + lane of the tile,
    // or (BM 64) row 16 w + lane in lanes 0-15; each takes every other chunk
    const int quad = warp & 3, half = warp >> 2;
    const int lrow = BM == 64 ? 16 * quad + lane : 32 * quad + lane;
    const bool live = (BM == 128 || lane < 16) && row0 + lrow < a.m;
    const float row_scale = live ? __ldg(a.sa + row0 + lrow) : 0.f;
    if (!mbar_wait(bar_done, 0, abort_flag))
        int8_fail(ERR_INT8_WAIT_DONE, abort_flag);
    if (tid == 0 && *abort_flag)
    {
        // after a failure the copies and MMAs in flight land before the ring is reused
        const int quiet = 0;
        for (int kb = std::max(0, issued - stages); kb < issued; ++kb)
            mbar_wait(bar_full + 8 * (kb % stages), (kb / stages) & 1, &quiet);
        mbar_wait(bar_done, 0, &quiet);
    }
    __syncwarp();
    tc_fence_after();
    const uint32_t taddr = tmem + ((uint32_t)(32 * quad) << 16);
    if (split == 1)
    {
#pragma unroll 1
        for (int c0 = 32 * half; c0 < bn; c0 += 64)
        {
            uint32_t r[32];
            tmem_ld32_async(taddr + (uint32_t)c0, r);
            tmem_wait_ld();
            if (live && !*abort_flag)
                store_scaled<T>(a, r, row0 + lrow, col0 + c0, row_scale);
            __syncwarp();
        }
    }
    else
    {
        tc_fence_before();
        __syncthreads(); // (after a failure: the ring is quiet)
        tc_fence_after();
        const int stride = bn + 4; // integers per staged row (16-byte shift per row: no bank conflicts)
        int *stage = reinterpret_cast<int *>(smem);
#pragma unroll 1
        for (int c0 = 32 * half; c0 < bn; c0 += 64)
        {
            uint32_t r[32];
            tmem_ld32_async(taddr + (uint32_t)c0, r);
            tmem_wait_ld();
            if (live)
            {
                int4 *dst = reinterpret_cast<int4 *>(stage + lrow * stride + c0);
#pragma unroll
                for (int v = 0; v < 8; ++v)
                    dst[v] = make_int4((int)r[4 * v], (int)r[4 * v + 1], (int)r[4 * v + 2], (int)r[4 * v + 3]);
            }
            __syncwarp();
        }
        cluster_barrier(); // every rank's partial is in its shared memory
        // the tile's (row, 32-column chunk) items, dealt over the cluster's threads
        // so that a warp's lanes hold consecutive rows of one chunk
        const int m_tile = (int)std::min<int64_t>(BM, a.m - row0);
        const int items = (bn / 32) * BM;
        if (!*abort_flag)
            for (int i = rank * kTThreads + tid; i < items; i += split * kTThreads)
            {
                const int rr = i % BM, c0 = (i / BM) * 32;
                if (rr >= m_tile || col0 + c0 >= a.n)
                    continue;
                uint32_t r[32] = {};
                const uint32_t off = smem_u32(stage + rr * stride + c0);
#pragma unroll 1
                for (int q = 0; q < split; ++q)
                {
                    const uint32_t peer = cluster_addr(off, (uint32_t)q);
                    int4 x[8];
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                        x[v] = ld_cluster_i4(peer + 16 * v);
#pragma unroll
                    for (int v = 0; v < 8; ++v)
                    {
                        r[4 * v] += (uint32_t)x[v].x;
                        r[4 * v + 1] += (uint32_t)x[v].y;
                        r[4 * v + 2] += (uint32_t)x[v].z;
                        r[4 * v + 3] += (uint32_t)x[v].w;
                    }
                }
                store_scaled<T>(a, r, row0 + rr, col0 + c0, __ldg(a.sa + row0 + rr));
            }
        __syncwarp();
        cluster_barrier(); // no rank leaves while another may still read its partial
    }

    // -------- teardown --------
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
    {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTTmemCols));
    }
}

// ---------------------------------------------------------------------------
// CUDA cores: 64 x 64 tiles of C, 32 k per step, each thread 4 x 4 sums. Rows
// may start at any byte; bytes past K are zero.
// ---------------------------------------------------------------------------
constexpr int kATileRows = 64, kAStep = 32;

template <typename T>
__global__ void __launch_bounds__(256) linear_int8_any_kernel(const Int8Args a)
{
    __shared__ int sa[kAStep / 4][kATileRows + 1], sb[kAStep / 4][kATileRows + 1];
    const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
    const int64_t row0 = (int64_t)blockIdx.y * kATileRows, col0 = (int64_t)blockIdx.x * kATileRows;
    int acc[4][4] = {};
    // word w (4 bytes of k) of one of the tile's rows
    auto word = [&](const int8_t *base, int64_t ld, int64_t row, int64_t rows, int64_t k0) -> int {
        uint32_t v = 0;
        if (row < rows)
            for (int e = 0; e < 4; ++e)
                if (k0 + e < a.k)
                    v |= (uint32_t)(uint8_t)base[row * ld + k0 + e] << (8 * e);
        return (int)v;
    };
    for (int64_t k0 = 0; k0 < a.k; k0 += kAStep)
    {
#pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            const int w = tid & 7, r = (tid >> 3) + 32 * i;
            sa[w][r] = word(a.a, a.lda, row0 + r, a.m, k0 + 4 * w);
            sb[w][r] = word(a.b, a.ldb, col0 + r, a.n, k0 + 4 * w);
        }
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kAStep / 4; ++w)
        {
            int x[4], y[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
            {
                x[i] = sa[w][ty + 16 * i];
                y[i] = sb[w][tx + 16 * i];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[i][j] = __dp4a(x[i], y[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
        {
            const int64_t row = row0 + ty + 16 * i, col = col0 + tx + 16 * j;
            if (row < a.m && col < a.n)
                static_cast<T *>(a.c)[row * a.ldc + col] =
                    from_f<T>(__fmul_rn((float)acc[i][j], __fmul_rn(a.sa[row], a.sb[col])));
        }
}

template <typename T>
int launch_any(const Int8Args &a, cudaStream_t stream)
{
    // gridDim.y is limited to 65535: longer products go in slabs of rows
    const int64_t slab = (int64_t)65535 * kATileRows;
    for (int64_t r = 0; r < a.m; r += slab)
    {
        Int8Args s = a;
        s.m = std::min(slab, a.m - r);
        s.a = a.a + r * a.lda;
        s.sa = a.sa + r;
        s.c = static_cast<T *>(a.c) + r * a.ldc;
        const dim3 grid((unsigned)ceil_div(a.n, kATileRows), (unsigned)ceil_div(s.m, kATileRows));
        linear_int8_any_kernel<T><<<grid, 256, 0, stream>>>(s);
    }
    return check_launch("l2k_linear_int8");
}

template <typename T, int BM>
int launch_tile(Int8Args a, int bn, int split, cudaStream_t stream)
{
    using C = TileCfg<BM>;
    a.bn = bn;
    a.split = split;
    a.stages = C::stages(bn);
    a.a_rows = (int)std::min<int64_t>(BM, ceil_div(a.m, 8) * 8);
    a.n_nt = (int)ceil_div(a.n, bn);
    CUtensorMap ma, mb;
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t m = (uint64_t)a.m, n = (uint64_t)a.n, k = (uint64_t)a.k, lda = (uint64_t)a.lda, ldb = (uint64_t)a.ldb;
    if (!make_map(&ma, dt, a.a, k, m, 1, lda, lda * m, (uint32_t)a.a_rows, kBK) ||
        !make_map(&mb, dt, a.b, k, n, 1, ldb, ldb * n, (uint32_t)bn, kBK))
        return set_error(L2K_ERR_CUDA, "l2k_linear_int8: tensor map encoding failed");
    auto kernel = linear_int8_tile_kernel<T, BM>;
    const uint32_t smem = C::smem_bytes(bn);
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess)
        return set_error(L2K_ERR_CUDA, "l2k_linear_int8: %s", cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ceil_div(a.m, BM) * a.n_nt * split));
    cfg.blockDim = dim3(kTThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kernel, ma, mb, a, C::ring_bytes(bn));
    if (e != cudaSuccess)
        return set_error(L2K_ERR_CUDA, "l2k_linear_int8: %s", cudaGetErrorString(e));
    return check_launch("l2k_linear_int8");
}

template <typename T>
int launch_linear(const Int8Args &p, cudaStream_t stream)
{
    Int8Args a = p;
    a.wide = (a.ldc * (int64_t)sizeof(T)) % 16 == 0 && is_aligned(a.c, 16);
    a.n_kb = (int)ceil_div(a.k, kBK);
    const bool tc = a.k > 0 && is_aligned(a.a, 16) && is_aligned(a.b, 16) && a.lda % 16 == 0 && a.ldb % 16 == 0 &&
                    encode_fn() != nullptr;
    if (!tc)
        return launch_any<T>(a, stream);
    if (a.m <= 64)
        return launch_tile<T, 64>(a, 64, 1, stream);
    return launch_tile<T, 128>(a, 128, 1, stream);
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
