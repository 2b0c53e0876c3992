// Rows to 8 bits: the three operators whose result feeds l2k_linear_int8.
//
//   l2k_quantize_rows_int8:             y = x
//   l2k_fused_add_residual_rmsnorm_int8: x += residual (if ADD), y = x w / rms(x)
//   l2k_swiglu_int8:                    y = silu(gate) * up
// and for each row, with a = max |y_j|,
//   scale = a / 127,   q_j = the integer nearest 127 y_j / a (ties to even).
// A row of zeros gives q = 0 and scale 0; a row holding a NaN or an infinity
// gives q = 0 and scale NaN, so that every product of that row is NaN.
//
// The norm's 1 / rms(x) > 0 multiplies every y_j and a alike: it cancels in
// q_j = rne(127 x_j w_j / max |x w|) and is left to the scale. x_j w_j is
// exact in fp32 for 16-bit data and in fp64 for fp32 data, so q does not
// depend on the order in which the squares are summed. SwiGLU's y is the fp32
// value of silu_mul, not rounded to T first (one rounding fewer than
// l2k_swiglu followed by l2k_quantize_rows_int8). Sums and maxima are fp32 or
// wider.
//
// 127 y / a is evaluated as fma(y, 127 / a, 1.5 * 2^23), whose low byte is the
// rounded integer: its error is below 127 * 2^-24 = 2^-17 (the rounded
// reciprocal), so only values within 2^-14 of a border between two integers
// can land on the wrong side; those few are divided in fp64.
#include "common.cuh"

#include <algorithm>
#include <type_traits>

namespace l2k
{
namespace
{

constexpr float kRmsEps = 1e-5f;
constexpr int kMaxThreads = 1024;

enum Source
{
    SRC_ROWS = 0,
    SRC_NORM = 1,
    SRC_NORM_ADD = 2,
    SRC_SWIGLU = 3
};

struct RowArgs
{
    const void *x;        // SRC_ROWS / SRC_SWIGLU: the input (SwiGLU rows: 2 * dim)
    void *xio;            // SRC_NORM*: the residual stream (written with ADD)
    const void *residual; // SRC_NORM_ADD
    const void *w;        // SRC_NORM*
    int8_t *q;
    float *scales;
    int64_t n_rows, dim;
};

// The type the row's values are held in: fp64 for the products x w of fp32
// data (exact), fp32 otherwise (exact for x and for 16-bit x w).
template <typename T, int SRC>
struct RowValue
{
    using type =
        std::conditional_t<std::is_same<T, float>::value && (SRC == SRC_NORM || SRC == SRC_NORM_ADD), double, float>;
};

// |y| as an unsigned integer of the same order; NaN above infinity above all
// finite values.
__device__ __forceinline__ uint32_t mag_bits(float y) { return __float_as_uint(y) & 0x7fffffffu; }
__device__ __forceinline__ uint64_t mag_bits(double y)
{
    return (uint64_t)__double_as_longlong(y) & 0x7fffffffffffffffull;
}
__device__ __forceinline__ float from_bits(uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ double from_bits(uint64_t b) { return __longlong_as_double((long long)b); }
__device__ __forceinline__ bool finite_bits(uint32_t b) { return b < 0x7f800000u; }
__device__ __forceinline__ bool finite_bits(uint64_t b) { return b < 0x7ff0000000000000ull; }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ uint64_t warp_max_bits(uint64_t v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = max((unsigned long long)v, (unsigned long long)__shfl_xor_sync(0xffffffffu, (unsigned long long)v, o));
    return v;
}

// The largest magnitude and (norms) the sum of squares over the block; one
// barrier, every thread gets both.
template <typename Bits, bool SUM>
__device__ __forceinline__ void block_reduce(Bits &top, float &sq)
{
    __shared__ Bits s_top[kMaxThreads / 32];
    __shared__ float s_sq[kMaxThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    top = warp_max_bits(top);
    if (SUM)
        sq = warp_sum(sq);
    if (n_warps == 1)
        return;
    if (lane == 0)
    {
        s_top[warp] = top;
        if (SUM)
            s_sq[warp] = sq;
    }
    __syncthreads();
    top = warp_max_bits(lane < n_warps ? s_top[lane] : Bits(0));
    if (SUM)
        sq = warp_sum(lane < n_warps ? s_sq[lane] : 0.f);
}

// What a row's values are divided by, and its scale.
template <typename V>
struct Quantizer
{
    V a;          // max |y| of the finite row, before 1 / rms
    float r;      // 127 / a, or 0 where only the fp64 division is used
    bool dead;    // every q of the row is 0
    float scale;
};

template <typename V, typename Bits>
__device__ __forceinline__ Quantizer<V> make_quantizer(Bits top, float inv_rms)
{
    Quantizer<V> z;
    z.a = from_bits(top);
    z.dead = !finite_bits(top) || top == 0;
    // outside 2^-100 .. 2^100 the reciprocal or the values could leave the range of fp32
    z.r = !z.dead && z.a >= (V)0x1p-100 && z.a <= (V)0x1p100 ? (float)((V)127 / z.a) : 0.f;
    z.scale = finite_bits(top) ? (float)(z.a * (V)inv_rms / (V)127) : __uint_as_float(0x7fc00000u);
    return z;
}

// Correctly rounded 127 y / a: 127 y is exact in fp64 for fp32 y, and a
// quotient of 24- and 32-bit integers that is no border between two integers
// is further from one than fp64 rounds.
template <typename V>
__device__ __noinline__ int quantize_exact(V y, V a)
{
    return __double2int_rn(__ddiv_rn(__dmul_rn((double)y, 127.0), (double)a));
}

// The 8-bit values of N consecutive y, packed low byte first.
template <typename V, int N>
__device__ __forceinline__ void quantize(const V (&y)[N], const Quantizer<V> &z, uint32_t (&bytes)[(N + 3) / 4])
{
    constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds to an integer held in the low bits
    uint32_t b[N];
    float worst = 0.f;
#pragma unroll
    for (int e = 0; e < N; ++e)
    {
        const float f = (float)y[e];
        const float t = __fmaf_rn(f, z.r, kMagic);
        worst = fmaxf(worst, fabsf(__fmaf_rn(f, z.r, -__fsub_rn(t, kMagic))));
        b[e] = __float_as_uint(t);
    }
    if (z.dead)
    {
#pragma unroll
        for (int e = 0; e < N; ++e)
            b[e] = 0;
    }
    else if (worst > 0.5f - 0x1p-14f || z.r == 0.f)
    {
#pragma unroll
        for (int e = 0; e < N; ++e)
            b[e] = (uint32_t)quantize_exact(y[e], z.a);
    }
#pragma unroll
    for (int i = 0; i < (N + 3) / 4; ++i)
    {
        uint32_t v = b[4 * i] & 0xffu;
        if (4 * i + 3 < N)
            v = __byte_perm(__byte_perm(b[4 * i], b[4 * i + 1], 0x0040), __byte_perm(b[4 * i + 2], b[4 * i + 3], 0x0040),
                            0x5410);
        bytes[i] = v;
    }
}

// 8 consecutive elements from a 16-byte aligned address.
template <typename T>
struct Raw8
{
    uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p, bool keep)
{
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        r.v[i] = keep ? ldg_keep(p + 16 / sizeof(T) * i) : ldg_coherent(p + 16 / sizeof(T) * i);
    return r;
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, T (&v)[8])
{
    __builtin_memcpy(v, &r, sizeof(r));
}

// One row per CTA, held in registers: thread t takes the groups of 8 elements
// t, t + blockDim.x, ... (NV of them at most).
template <typename T, int SRC, int NV>
__global__ void __launch_bounds__(kMaxThreads) rows_int8_kernel(const RowArgs a)
{
    using V = typename RowValue<T, SRC>::type;
    using Bits = std::conditional_t<sizeof(V) == 8, uint64_t, uint32_t>;
    constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    const int64_t row = blockIdx.x;
    const int n_groups = (int)(a.dim / 8);
    const T *src = static_cast<const T *>(kNorm ? a.xio : a.x) + row * a.dim * (SRC == SRC_SWIGLU ? 2 : 1);
    const T *add = SRC == SRC_NORM_ADD ? static_cast<const T *>(a.residual) + row * a.dim : nullptr;
    const T *w = static_cast<const T *>(a.w);

    V y[NV][8];
    Bits top = 0;
    float sq = 0.f;
    Raw8<T> in[NV], in2[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < n_groups)
        {
            in[j] = load8(src + 8 * g, false);
            if (SRC == SRC_NORM_ADD)
                in2[j] = load8(add + 8 * g, false);
            if (SRC == SRC_SWIGLU)
                in2[j] = load8(src + a.dim + 8 * g, false);
        }
    }
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            y[j][e] = (V)0;
        if (g >= n_groups)
            continue;
        T v[8], u[8];
        unpack8(in[j], v);
        if constexpr (SRC == SRC_ROWS)
        {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[j][e] = to_f(v[e]);
        }
        else if constexpr (SRC == SRC_SWIGLU)
        {
            unpack8(in2[j], u);
#pragma unroll
            for (int e = 0; e < 8; ++e)
                y[j][e] = silu_mul<T>(to_f(v[e]), to_f(u[e]));
        }
        else
        {
            if constexpr (SRC == SRC_NORM_ADD)
            {
                unpack8(in2[j], u);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = from_f<T>(__fadd_rn(to_f(v[e]), to_f(u[e])));
                Raw8<T> o;
                __builtin_memcpy(&o, v, sizeof(o));
                T *dst = static_cast<T *>(a.xio) + row * a.dim + 8 * g;
#pragma unroll
                for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
                    stg(dst + 16 / sizeof(T) * i, o.v[i]);
            }
            unpack8(load8(w + 8 * g, true), u);
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                const float f = to_f(v[e]);
                sq = fmaf(f, f, sq);
                y[j][e] = (V)f * (V)to_f(u[e]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
            top = max(top, mag_bits(y[j][e]));
    }
    block_reduce<Bits, kNorm>(top, sq);
    float inv_rms = 1.f;
    if (kNorm)
        inv_rms = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sq, (float)a.dim), kRmsEps)));
    const Quantizer<V> z = make_quantizer<V>(top, inv_rms);
    int8_t *q = a.q + row * a.dim;
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < n_groups)
        {
            uint32_t b[2];
            quantize<V, 8>(y[j], z, b);
            *reinterpret_cast<uint2 *>(q + 8 * g) = make_uint2(b[0], b[1]);
        }
    }
    if (threadIdx.x == 0)
        a.scales[row] = z.scale;
}

// Any length and alignment: two passes over the row, an element at a time
// (the second re-reads it, normally from L1 or L2, and recomputes y).
template <typename T, int SRC>
__global__ void __launch_bounds__(kMaxThreads) rows_int8_any_kernel(const RowArgs a)
{
    using V = typename RowValue<T, SRC>::type;
    using Bits = std::conditional_t<sizeof(V) == 8, uint64_t, uint32_t>;
    constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    const int64_t row = blockIdx.x;
    const T *src = static_cast<const T *>(kNorm ? a.xio : a.x) + row * a.dim * (SRC == SRC_SWIGLU ? 2 : 1);
    const T *add = SRC == SRC_NORM_ADD ? static_cast<const T *>(a.residual) + row * a.dim : nullptr;
    const T *w = static_cast<const T *>(a.w);
    T *xio = static_cast<T *>(a.xio) + row * a.dim;
    auto value = [&](int64_t d, float f) -> V {
        if constexpr (SRC == SRC_SWIGLU)
            return silu_mul<T>(f, to_f(src[a.dim + d]));
        else if constexpr (kNorm)
            return (V)f * (V)to_f(w[d]);
        else
            return f;
    };
    Bits top = 0;
    float sq = 0.f;
    for (int64_t d = threadIdx.x; d < a.dim; d += blockDim.x)
    {
        float f;
        if constexpr (SRC == SRC_NORM_ADD)
        {
            const T s = from_f<T>(__fadd_rn(to_f(xio[d]), to_f(add[d])));
            xio[d] = s;
            f = to_f(s);
        }
        else
            f = to_f(src[d]);
        sq = fmaf(f, f, sq);
        top = max(top, mag_bits(value(d, f)));
    }
    block_reduce<Bits, kNorm>(top, sq);
    float inv_rms = 1.f;
    if (kNorm)
        inv_rms = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sq, (float)a.dim), kRmsEps)));
    const Quantizer<V> z = make_quantizer<V>(top, inv_rms);
    int8_t *q = a.q + row * a.dim;
    for (int64_t d = threadIdx.x; d < a.dim; d += blockDim.x)
    {
        // (with ADD: this thread's own store of the first pass)
        const V y[1] = {value(d, to_f(kNorm ? xio[d] : src[d]))};
        uint32_t b[1];
        quantize<V, 1>(y, z, b);
        q[d] = (int8_t)(b[0] & 0xffu);
    }
    if (threadIdx.x == 0)
        a.scales[row] = z.scale;
}

template <typename T, int SRC, int NV>
int launch_rows_nv(const RowArgs &a, int64_t groups, cudaStream_t stream)
{
    const int threads = (int)(ceil_div(ceil_div(groups, NV), 32) * 32);
    rows_int8_kernel<T, SRC, NV><<<(unsigned)a.n_rows, threads, 0, stream>>>(a);
    return L2K_OK;
}

template <typename T, int SRC>
int launch_rows(const RowArgs &a, const char *name, cudaStream_t stream)
{
    const bool vec = a.dim % 8 == 0 && is_aligned(a.x, 16) && is_aligned(a.xio, 16) && is_aligned(a.residual, 16) &&
                     is_aligned(a.w, 16) && is_aligned(a.q, 8);
    const int64_t groups = a.dim / 8;
    if (vec && groups <= kMaxThreads)
        launch_rows_nv<T, SRC, 1>(a, groups, stream);
    else if (vec && groups <= 2 * kMaxThreads)
        launch_rows_nv<T, SRC, 2>(a, groups, stream);
    else
    {
        const int threads = (int)std::min<int64_t>(kMaxThreads, ceil_div(a.dim, 32) * 32);
        rows_int8_any_kernel<T, SRC><<<(unsigned)a.n_rows, threads, 0, stream>>>(a);
    }
    return check_launch(name);
}

// Checks common to the three entries; returns L2K_OK with *done set when
// nothing is left to do.
int check_rows(const RowArgs &a, int dtype, const char *name, cudaStream_t stream, bool *done)
{
    *done = true;
    L2K_REQUIRE(a.n_rows >= 0 && a.dim >= 0, "%s: negative size", name);
    L2K_REQUIRE(dtype_ok(dtype), "%s: unsupported dtype %d", name, dtype);
    if (a.n_rows == 0)
        return L2K_OK;
    L2K_REQUIRE(a.scales, "%s: null pointer", name);
    if (a.dim == 0) // rows without elements: scale 0
    {
        const cudaError_t e = cudaMemsetAsync(a.scales, 0, (size_t)a.n_rows * sizeof(float), stream);
        return e == cudaSuccess ? L2K_OK : set_error(L2K_ERR_CUDA, "%s: %s", name, cudaGetErrorString(e));
    }
    L2K_REQUIRE_SHAPE(a.n_rows < (int64_t(1) << 31), "%s: more than 2^31 - 1 rows", name);
    *done = false;
    return L2K_OK;
}

} // namespace
} // namespace l2k

extern "C" int l2k_quantize_rows_int8(const void *x, int8_t *q, float *scales, int64_t num_rows, int64_t dim,
                                      int dtype, l2k_stream_t stream)
{
    using namespace l2k;
    const char *name = "l2k_quantize_rows_int8";
    const RowArgs a{x, nullptr, nullptr, nullptr, q, scales, num_rows, dim};
    bool done;
    const int st = check_rows(a, dtype, name, stream, &done);
    if (done)
        return st;
    L2K_REQUIRE(x && q, "%s: null pointer", name);
    L2K_DISPATCH(dtype, { return launch_rows<T, SRC_ROWS>(a, name, stream); });
    return L2K_OK;
}

extern "C" int l2k_fused_add_residual_rmsnorm_int8(const void *weights, void *x, const void *residual, int8_t *q,
                                                   float *scales, int64_t num_tokens, int64_t embed_dim,
                                                   int add_residual, int dtype, l2k_stream_t stream)
{
    using namespace l2k;
    const char *name = "l2k_fused_add_residual_rmsnorm_int8";
    const RowArgs a{nullptr, x, add_residual ? residual : nullptr, weights, q, scales, num_tokens, embed_dim};
    bool done;
    const int st = check_rows(a, dtype, name, stream, &done);
    if (done)
        return st;
    L2K_REQUIRE(weights && x && q && (residual || !add_residual), "%s: null pointer", name);
    L2K_REQUIRE(!add_residual || x != residual, "%s: x and residual must be distinct buffers", name);
    L2K_DISPATCH(dtype, {
        return add_residual ? launch_rows<T, SRC_NORM_ADD>(a, name, stream) : launch_rows<T, SRC_NORM>(a, name, stream);
    });
    return L2K_OK;
}

extern "C" int l2k_swiglu_int8(const void *input, int8_t *q, float *scales, int64_t num_tokens,
                               int64_t intermediate_size, int dtype, l2k_stream_t stream)
{
    using namespace l2k;
    const char *name = "l2k_swiglu_int8";
    const RowArgs a{input, nullptr, nullptr, nullptr, q, scales, num_tokens, intermediate_size};
    bool done;
    const int st = check_rows(a, dtype, name, stream, &done);
    if (done)
        return st;
    L2K_REQUIRE(input && q, "%s: null pointer", name);
    L2K_DISPATCH(dtype, { return launch_rows<T, SRC_SWIGLU>(a, name, stream); });
    return L2K_OK;
}
