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
// value of silu * up, not rounded to T first (one rounding fewer than
// l2k_swiglu followed by l2k_quantize_rows_int8). Sums and maxima are fp32 or
// wider.
//
// 127 y / a is evaluated as fma(y, 127 / a, 1.5 * 2^23), whose low byte is the
// rounded integer: its error is at most 127 * 2^-23 (the rounded reciprocal, and
// y of fp64 products), so only values within 2^-14 of a border between two
// integers can land on the wrong side; those are compared with the border exactly, in fp64.
// Values of 16 bits need no second look (kShort).
//
// Three kernels:
//   * rows_int8_stream_kernel, for many rows: CTAs stay on their SM and walk the
//     rows; one thread keeps a ring of rows in flight with bulk copies into
//     shared memory, so loads go on while a row is reduced and written (with a
//     row's loads issued by the threads that then wait for its reduction, DRAM
//     idled between them: 16384 x 4096 bf16 rows ran at 2.8 TB/s);
//   * rows_int8_kernel, for few rows: one row per CTA, straight into registers;
//   * rows_int8_any_kernel: rows longer than the others hold.
#include "common.cuh"
#include "tcgen05.cuh" // mbarriers

#include <algorithm>
#include <type_traits>

namespace l2k
{

__device__ int g_int8_rows_error = 0; // first error code recorded by a kernel of this file

namespace
{

constexpr int ERR_INT8_ROWS_WAIT = 0x801;
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

// The largest |y| so far: fp32 with NaN above everything, or the bits of an fp64
// (whose order, for magnitudes, is theirs as integers, NaN above infinity).
struct TopF
{
    using Bits = uint32_t;
    float v = 0.f;
    __device__ __forceinline__ void add(float a, float b)
    {
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(v), "f"(a), "f"(b));
    }
    __device__ __forceinline__ Bits bits() const { return __float_as_uint(v) & 0x7fffffffu; }
};
struct TopD
{
    using Bits = unsigned long long;
    Bits v = 0;
    __device__ __forceinline__ static Bits mag(double y)
    {
        return (Bits)__double_as_longlong(y) & 0x7fffffffffffffffull;
    }
    __device__ __forceinline__ void add(double a, double b) { v = max(v, max(mag(a), mag(b))); }
    __device__ __forceinline__ Bits bits() const { return v; }
};
template <typename V>
using Top = std::conditional_t<sizeof(V) == 8, TopD, TopF>;

__device__ __forceinline__ float from_bits(uint32_t b) { return __uint_as_float(b); }
__device__ __forceinline__ double from_bits(unsigned long long b) { return __longlong_as_double((long long)b); }
__device__ __forceinline__ bool finite_bits(uint32_t b) { return b < 0x7f800000u; }
__device__ __forceinline__ bool finite_bits(unsigned long long b) { return b < 0x7ff0000000000000ull; }
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t v) { return __reduce_max_sync(0xffffffffu, v); }
__device__ __forceinline__ unsigned long long warp_max_bits(unsigned long long v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The largest magnitude and (norms) the sum of squares over the block; one
// barrier, every thread gets both. A caller's consecutive rows alternate `buf`,
// so that a warp that is a row ahead does not overwrite what another still reads.
template <typename Bits, bool SUM>
__device__ __forceinline__ void block_reduce(Bits &top, float &sq, int buf)
{
    __shared__ Bits s_top[2][kMaxThreads / 32];
    __shared__ float s_sq[2][kMaxThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n_warps = blockDim.x >> 5;
    top = warp_max_bits(top);
    if (SUM)
        sq = warp_sum(sq);
    if (n_warps == 1)
    {
        __syncwarp();
        return;
    }
    if (lane == 0)
    {
        s_top[buf][warp] = top;
        if (SUM)
            s_sq[buf][warp] = sq;
    }
    __syncthreads();
    top = warp_max_bits(lane < n_warps ? s_top[buf][lane] : Bits(0));
    if (SUM)
        sq = warp_sum(lane < n_warps ? s_sq[buf][lane] : 0.f);
}

// What a row's values are divided by, and its scale.
template <typename V>
struct Quantizer
{
    V a;           // max |y| of the row, before 1 / rms
    float r, r_lo; // 127 / a to 48 bits; r = 0 where it or the values could leave the range of fp32
    bool dead;     // every q of the row is 0
    float scale;
};

template <typename V, typename Bits>
__device__ __forceinline__ Quantizer<V> make_quantizer(Bits top, float inv_rms)
{
    Quantizer<V> z;
    z.a = from_bits(top);
    z.dead = !finite_bits(top) || top == 0;
    z.r = !z.dead && z.a >= (V)0x1p-100 && z.a <= (V)0x1p100 ? (float)((V)127 / z.a) : 0.f;
    z.r_lo = __fdividef(__fmaf_rn(-z.r, (float)z.a, 127.f), (float)z.a); // (of 16-bit a: an exact remainder)
    z.scale = finite_bits(top) ? (float)(z.a * (V)inv_rms / (V)127) : __uint_as_float(0x7fc00000u);
    return z;
}

// 127 y / a, rounded once: 127 y of an fp32 y is exact in fp64, and a quotient of a
// 32- and a 24-bit integer that is no border between two integers is further from
// one than fp64 rounds.
__device__ __noinline__ uint32_t quantize_divided(float y, float a)
{
    return (uint32_t)__double2int_rn(__ddiv_rn(__dmul_rn((double)y, 127.0), (double)a));
}

// For the 48-bit products of fp32 norms: 127 y takes 55 bits, two more than fp64 has
// (an exact half of the largest came out as 63 instead of 64 for one in eight pairs
// of x and w). So the side of a border k + 1/2 is the sign of 127 |y| - (k + 1/2) a:
// both less p, the second one's fp64 value, which leaves a few bits of either next to
// the border, and the sign in any case. k is the quotient in fp32, rounded down; next
// to an integer either neighbour leads to the same result. (An fp64 division here took
// registers from the callers: 8192 x 5120 fp32 norms 107 us, 95 without.)
__device__ __noinline__ uint32_t quantize_divided(double y, double a)
{
    const double m = fabs(y), unit = __hiloint2double(0x7fe00000 - (__double2hiint(a) & 0x7ff00000), 0); // a unit: 1 to 2
    const float k = floorf(__fdividef(127.f * (float)__dmul_rn(m, unit), (float)__dmul_rn(a, unit)));
    const double h = (double)k + 0.5, p = __dmul_rn(h, a);
    const double past = __dsub_rn(__fma_rn(127.0, m, -p), __fma_rn(h, a, -p));
    const int q = (int)k + (past > 0.0 || (past == 0.0 && ((int)k & 1)) ? 1 : 0);
    return (uint32_t)(y < 0.0 ? -q : q);
}

// The same for a value that lies next to the border k + 1/2, k >= 0: which side.
__device__ __noinline__ uint32_t quantize_at_border(float y, float a, float r)
{
    const float k = floorf(fabsf(__fmul_rn(y, r)));
    const double v = 127.0 * (double)fabsf(y), border = ((double)k + 0.5) * (double)a; // (31 and 32 bits: exact)
    const int q = (int)k + (v > border || (v == border && ((int)k & 1)) ? 1 : 0);
    return (uint32_t)(y < 0.f ? -q : q);
}
__device__ __forceinline__ uint32_t quantize_at_border(double y, double a, float)
{
    return quantize_divided(y, a);
}

// Two fp32 operations at once.
__device__ __forceinline__ unsigned long long bits2(const float2 &v)
{
    unsigned long long u;
    __builtin_memcpy(&u, &v, 8);
    return u;
}
__device__ __forceinline__ float2 floats2(unsigned long long u)
{
    float2 v;
    __builtin_memcpy(&v, &u, 8);
    return v;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    unsigned long long d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)), "l"(bits2(c)));
    return floats2(d);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    unsigned long long d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
    return floats2(d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    unsigned long long d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(bits2(a)), "l"(bits2(b)));
    return floats2(d);
}

constexpr float kMagic = 12582912.f; // 1.5 * 2^23: adding it rounds to an integer held in the low bits
constexpr float kBorder = 0.5f - 0x1p-14f;

// Values of at most 16 bits (bf16 values and their products, f16 values) whose
// row's largest has no more: 254 y and the odd multiples of a differ by more than
// half a step of fp32 unless they are equal, so the fp32 nearest to 127 y / a is a
// border k + 1/2 only where the quotient is, and adding kMagic then rounds ties to
// even. 0.5 % of a bf16 row's values are ties: looking at each of them again cost
// more than the whole fast path.
template <typename T, int SRC>
constexpr bool kShort = SRC != SRC_SWIGLU &&
                        (std::is_same<T, __nv_bfloat16>::value || (std::is_same<T, __half>::value && SRC == SRC_ROWS));

// The low byte of the result holds the 8-bit value of y.
template <bool SHORT, typename V>
__device__ __forceinline__ uint32_t quantize1(V y, const Quantizer<V> &z)
{
    if (z.dead)
        return 0u;
    if (z.r == 0.f)
        return quantize_divided(y, z.a);
    if constexpr (SHORT)
        return __float_as_uint(__fadd_rn(__fmaf_rn(y, z.r, __fmul_rn(y, z.r_lo)), kMagic));
    else
    {
        const float t = __fmaf_rn((float)y, z.r, kMagic);
        if (fabsf(__fmaf_rn((float)y, z.r, -__fsub_rn(t, kMagic))) > kBorder)
            return quantize_at_border(y, z.a, z.r);
        return __float_as_uint(t);
    }
}

// The 8-bit values of 8 consecutive y, packed low byte first.
template <bool SHORT, typename V>
__device__ __forceinline__ uint2 quantize8(const V (&y)[8], const Quantizer<V> &z)
{
    if (z.dead) // (the whole row; padding is common)
        return make_uint2(0u, 0u);
    uint32_t b[8];
    if (z.r == 0.f) // (the whole row)
    {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            b[e] = quantize_divided(y[e], z.a);
    }
    else
    {
        const float2 r2 = make_float2(z.r, z.r), magic2 = make_float2(kMagic, kMagic);
        if constexpr (SHORT)
        {
            const float2 lo2 = make_float2(z.r_lo, z.r_lo);
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                const float2 f = make_float2(y[e], y[e + 1]);
                const float2 t = add2(fma2(f, r2, mul2(f, lo2)), magic2);
                b[e] = __float_as_uint(t.x);
                b[e + 1] = __float_as_uint(t.y);
            }
        }
        else
        {
            const float2 minus2 = make_float2(-1.f, -1.f);
            float off = 0.f; // the largest distance from the integer rounded to
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                const float2 f = make_float2((float)y[e], (float)y[e + 1]);
                const float2 t = fma2(f, r2, magic2);
                const float2 d = fma2(f, r2, fma2(t, minus2, magic2));
                asm("max.abs.f32 %0, %1, %2, %3;" : "=f"(off) : "f"(off), "f"(d.x), "f"(d.y));
                b[e] = __float_as_uint(t.x);
                b[e + 1] = __float_as_uint(t.y);
            }
            if (off > kBorder)
            {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    b[e] = quantize1<false>(y[e], z);
            }
        }
    }
    uint2 w;
    w.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    w.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
    return w;
}

// 8 consecutive elements from a 16-byte aligned address.
template <typename T>
struct Raw8
{
    uint4 v[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p)
{
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        r.v[i] = ldg_coherent(p + 16 / sizeof(T) * i);
    return r;
}
template <typename T>
__device__ __forceinline__ Raw8<T> load8_shared(const uint8_t *p)
{
    Raw8<T> r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        r.v[i] = *reinterpret_cast<const uint4 *>(p + 16 * i);
    return r;
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const Raw8<T> &r)
{
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        stg(p + 16 / sizeof(T) * i, r.v[i]);
}
// The same values, unknown as such to the compiler.
template <typename T>
__device__ __forceinline__ void opaque(Raw8<T> &r)
{
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
        asm("" : "+r"(r.v[i].x), "+r"(r.v[i].y), "+r"(r.v[i].z), "+r"(r.v[i].w));
}
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T> &r, T (&v)[8])
{
    __builtin_memcpy(v, &r, sizeof(r));
}

template <typename T>
__device__ __forceinline__ float2 pair(const T (&v)[8], int e)
{
    return make_float2(to_f(v[e]), to_f(v[e + 1]));
}

// The largest magnitude of 16-bit values, two at a time (the sign that the instruction
// gives is not used): 16384 x 4096 bf16 rows 38 us, 41 through fp32. Packed additions
// and products in the norms, a fifth fewer instructions, were not kept: 8192 x 11008 111
// us against 125, but 16384 x 4096 88 against 76, launches back to back.
template <typename T>
struct TopPacked
{
    using Bits = uint32_t;
    uint32_t v = 0;
    __device__ __forceinline__ void add(const Raw8<T> &r)
    {
#pragma unroll
        for (uint32_t x : {r.v[0].x, r.v[0].y, r.v[0].z, r.v[0].w})
            if constexpr (std::is_same<T, __half>::value)
                asm("max.NaN.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(v) : "r"(x));
            else
                asm("max.NaN.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(v) : "r"(x));
    }
    __device__ __forceinline__ Bits bits() const
    {
        T e[2];
        __builtin_memcpy(e, &v, sizeof(e));
        TopF top;
        top.add(to_f(e[0]), to_f(e[1]));
        return top.bits();
    }
};

// silu(g) * u in fp32 by the fast exponential and reciprocal, for every type (fp32 too,
// where l2k_swiglu takes expf and an IEEE reciprocal). Relative error, in half steps of
// fp32 (2^-24): 1.23 |g| from the exponential's rounded argument and factor, 4 and 2
// for the two approximations, 3 for the sum and the products, so at most 1.25 |g| + 9.
// In a row's 8-bit values an element's error and the largest's count 127 times each:
// 1.4e-4 of a step next to g = 0, 7e-4 at |g| = 32, 1.7e-3 at 80, which moves a byte only
// where 127 y / a lies that close to a border. 0 where 1 + exp(-g) passes 2^126
// (g < -87.33), whose reciprocal is flushed.
__device__ __forceinline__ float2 silu_up2(float2 g, float2 u)
{
    const float2 x = mul2(g, make_float2(-1.4426950408889634f, -1.4426950408889634f));
    float2 e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(x.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(x.y));
    const float2 d = add2(e, make_float2(1.f, 1.f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
    return mul2(mul2(g, r), u);
}
__device__ __forceinline__ float silu_up(float g, float u)
{
    return silu_up2(make_float2(g, g), make_float2(u, u)).x;
}

// y of 8 elements of a row (or with ADD of the sum to write back) and the norm's weights.
template <typename T, int SRC, typename V>
__device__ __forceinline__ void values8(const Raw8<T> &in, const Raw8<T> &w, V (&y)[8])
{
    T v[8], u[8];
    unpack8(in, v);
    unpack8(w, u);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        y[e] = SRC == SRC_ROWS ? (V)to_f(v[e]) : (V)to_f(v[e]) * (V)to_f(u[e]);
}

// What a thread holds of 8 elements from the first look at them to the second:
// SwiGLU's y, and fp64 products where the registers allow (NV <= 2: 137 us for
// 16384 x 4096 fp32 norms, 154 when they are computed twice); else the inputs, half
// the registers or less, from which y is computed again.
template <typename T, int SRC, int NV>
struct Held
{
    using V = typename RowValue<T, SRC>::type;
    static constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    static constexpr bool kPacked = SRC == SRC_ROWS && sizeof(T) == 2;
    using RowTop = std::conditional_t<kPacked, TopPacked<T>, Top<V>>;
    static constexpr bool kKeep = SRC == SRC_SWIGLU || (sizeof(V) == 8 && NV <= 2);
    Raw8<T> in;
    V y[8];

    // The first look: in2 is the residual, or SwiGLU's up half; with ADD `in`
    // becomes the sum to write back.
    __device__ __forceinline__ void look(const Raw8<T> &first, const Raw8<T> &in2, const Raw8<T> &w, RowTop &top, float &sq)
    {
        T v[8], u[8];
        if constexpr (SRC == SRC_SWIGLU)
        {
            unpack8(first, v);
            unpack8(in2, u);
#pragma unroll
            for (int e = 0; e < 8; e += 2)
            {
                const float2 t = silu_up2(pair(v, e), pair(u, e));
                y[e] = t.x;
                y[e + 1] = t.y;
            }
#pragma unroll
            for (int e = 0; e < 8; e += 2)
                top.add(y[e], y[e + 1]);
        }
        else
        {
            unpack8(first, v);
            if constexpr (SRC == SRC_NORM_ADD)
            {
                unpack8(in2, u);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[e] = from_f<T>(__fadd_rn(to_f(v[e]), to_f(u[e])));
            }
            __builtin_memcpy(&in, v, sizeof(in));
            if constexpr (kNorm)
            {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    sq = fmaf(to_f(v[e]), to_f(v[e]), sq);
            }
            if constexpr (kPacked)
                top.add(in);
            else
            {
                V t[8];
                values8<T, SRC>(in, w, t);
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (kKeep)
                        y[e] = t[e];
#pragma unroll
                for (int e = 0; e < 8; e += 2)
                    top.add(t[e], t[e + 1]);
            }
        }
    }
    __device__ __forceinline__ uint2 quantized(const Raw8<T> &w, const Quantizer<V> &z) const
    {
        if constexpr (kKeep)
            return quantize8<false>(y, z);
        else
        {
            V t[8];
            Raw8<T> again = in, w_again = w;
            opaque(again); // (else the compiler keeps the first look's products instead)
            opaque(w_again);
            values8<T, SRC>(again, w_again, t);
            return quantize8<kShort<T, SRC>>(t, z);
        }
    }
};

__device__ __forceinline__ float inv_rms_of(float sq, int64_t dim)
{
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(sq, (float)dim), kRmsEps)));
}

// One row per CTA: thread t takes the groups of 8 elements t, t + blockDim.x, ...
// (NV of them at most).
template <typename T, int SRC, int NV>
__global__ void __launch_bounds__(kMaxThreads) rows_int8_kernel(const RowArgs a)
{
    using V = typename RowValue<T, SRC>::type;
    constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    const int64_t row = blockIdx.x;
    const int n_groups = (int)(a.dim / 8);
    const T *src = static_cast<const T *>(kNorm ? a.xio : a.x) + row * a.dim * (SRC == SRC_SWIGLU ? 2 : 1);
    const T *add = SRC == SRC_NORM_ADD ? static_cast<const T *>(a.residual) + row * a.dim : nullptr;
    T *xio = static_cast<T *>(a.xio) + row * a.dim;

    pdl_trigger();
    pdl_wait();
    Raw8<T> in[NV], in2[NV], w[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < n_groups)
        {
            in[j] = load8(src + 8 * g);
            if (SRC == SRC_NORM_ADD)
                in2[j] = load8(add + 8 * g);
            if (SRC == SRC_SWIGLU)
                in2[j] = load8(src + a.dim + 8 * g);
            if (kNorm)
                w[j] = load8(static_cast<const T *>(a.w) + 8 * g);
        }
    }
    Held<T, SRC, NV> held[NV];
    typename Held<T, SRC, NV>::RowTop top;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < n_groups)
        {
            held[j].look(in[j], in2[j], w[j], top, sq);
            if (SRC == SRC_NORM_ADD)
                store8(xio + 8 * g, held[j].in);
        }
    }
    auto bits = top.bits();
    block_reduce<decltype(bits), kNorm>(bits, sq, 0);
    const Quantizer<V> z = make_quantizer<V>(bits, kNorm ? inv_rms_of(sq, a.dim) : 1.f);
    int8_t *q = a.q + row * a.dim;
#pragma unroll
    for (int j = 0; j < NV; ++j)
    {
        const int g = threadIdx.x + j * blockDim.x;
        if (g < n_groups)
            *reinterpret_cast<uint2 *>(q + 8 * g) = held[j].quantized(w[j], z);
    }
    if (threadIdx.x == 0)
        a.scales[row] = z.scale;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

// The rows blockIdx.x, blockIdx.x + gridDim.x, ... through a ring of `depth`
// stages, each one row's inputs (x, then the residual; or SwiGLU's gate and up
// halves). A stage is refilled once the row's reduction has shown that every
// thread has read it. Each thread holds NV groups of 8 elements.
//
// Aligned rows (16-byte aligned, a multiple of 8 elements): 16-byte accesses.
// RAGGED: rows of any length and alignment, in 16-byte accesses too (an element at a
// time, 16384 x 1023 bf16 rows took 25 us, norms 61, SwiGLU 41; now 20, 39, 32; 4099 x
// 13799: 82, 197, 126, now 44, 114, 85):
// - A CTA's rows lie a multiple of 8 rows apart, so all of them lie alike with respect
//   to the units of 8 elements in memory.
// - The groups are cut where q's bytes (norms: the row that is written back) can be
//   stored together. The first group may begin before the row and the last end behind
//   it; where the two parts fit into one group they share the first, so there are no
//   more groups than in an aligned row (with one more, 16384 x 1023 bf16 rows took
//   31.6 us: a warp for one group).
// - The copy takes the units that the row touches; what belongs to the rows next to it
//   is not used. Elements of 16-byte units that reach out of the tensor are added by
//   the threads.
// - An x, or an up half, that lies otherwise than the groups is moved into place in
//   registers. A residual that lies otherwise than x is read an element at a time, and
//   so a norm's q is written where it lies otherwise than x.
constexpr int kMaxDepth = 8;
constexpr int kStreamThreads = 512;

__device__ __forceinline__ uintptr_t down16(uintptr_t p) { return p & ~(uintptr_t)15; }
__device__ __forceinline__ uintptr_t up16(uintptr_t p) { return (p + 15) & ~(uintptr_t)15; }

// Elements [pos, pos + 8) at p, where p + pos - shift is a unit of 8 elements (shift: 0
// to 7, the same in every thread): aligned 16-byte loads, moved into place by selects
// (a switch over the shift was 5 to 15 % slower). CHECK: loads that begin outside
// [0, end) are left out.
template <typename T, bool CHECK>
__device__ __forceinline__ Raw8<T> load8_shifted(const uint8_t *p, int pos, int shift, int end)
{
    constexpr int kVec = 16 / sizeof(T), kLoads = 8 / kVec + 1, kWords = 8 * sizeof(T) / 4;
    shift %= kVec;
    const int first = pos - shift;
    if (!CHECK && shift == 0)
        return load8_shared<T>(p + first * (int)sizeof(T));
    uint32_t w[4 * kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
    {
        uint4 v = {};
        const int e = first + kVec * i;
        if ((!CHECK || (e >= 0 && e < end)) && (i < kLoads - 1 || shift))
            v = *reinterpret_cast<const uint4 *>(p + e * (int)sizeof(T));
        __builtin_memcpy(w + 4 * i, &v, sizeof(v));
    }
    const int by = shift * (int)sizeof(T); // bytes
#pragma unroll
    for (int step = 2; step; step /= 2)
        if (by & (4 * step))
        {
#pragma unroll
            for (int i = 0; i < kWords + step - 1 + (sizeof(T) == 2); ++i)
                w[i] = i + step < 4 * kLoads ? w[i + step] : 0;
        }
    if (sizeof(T) == 2 && (by & 2))
    {
#pragma unroll
        for (int i = 0; i < kWords; ++i)
            w[i] = __funnelshift_r(w[i], w[i + 1], 16);
    }
    Raw8<T> r;
    __builtin_memcpy(&r, w, sizeof(r));
    return r;
}

// THREADS: the most threads of a launch; below kStreamThreads the instantiation is held
// to the registers with which an SM takes two such CTAs (448: 72, 320: 96).
template <typename T, int SRC, int NV, bool RAGGED, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS < kStreamThreads ? 2 : 1)
    rows_int8_stream_kernel(const RowArgs a, const int depth, const uint32_t input_bytes)
{
    using V = typename RowValue<T, SRC>::type;
    constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    constexpr int kCopies = SRC == SRC_NORM_ADD ? 2 : 1;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ __align__(8) uint64_t s_full[kMaxDepth];
    __shared__ int s_abort;
    const int tid = threadIdx.x, n_threads = blockDim.x;
    const int dim = (int)a.dim;
    const int64_t row_bytes = a.dim * (int64_t)sizeof(T) * (SRC == SRC_SWIGLU ? 2 : 1);
    const void *const base = kNorm ? a.xio : a.x;
    const uint32_t stage_bytes = input_bytes * kCopies;
    const int64_t n_mine = (a.n_rows - blockIdx.x + gridDim.x - 1) / gridDim.x; // (gridDim.x <= n_rows)
    auto place = [&](const void *tensor) { // of this CTA's rows in their units of 8 elements
        return RAGGED ? (int)((((uintptr_t)tensor + blockIdx.x * row_bytes) / sizeof(T)) & 7) : 0;
    };
    const int off = place(base);
    const int cut = kNorm ? off : RAGGED ? (int)(((uintptr_t)a.q + blockIdx.x * a.dim) & 7) : 0;
    const int off2 = SRC == SRC_NORM_ADD ? place(a.residual) : 0;
    const bool q_aligned = !RAGGED || (((uintptr_t)a.q + blockIdx.x * a.dim - cut) & 7) == 0;
    const int n_elements = (dim + 7) / 8 * 8; // of all groups
    auto mine = [&](int j) { return 8 * (j * n_threads + tid) < dim; };
    // The first element of group j; below 0 in a ragged row's first group, where an
    // element e < 0 stands for e + n_elements. Thread 0 begins with the last group, so
    // that the partial ones are its first and thread 1's.
    auto at = [&](int j) {
        const int e = 8 * (j * n_threads + tid) - cut;
        return !RAGGED ? e : j == 0 && tid == 0 ? e + n_elements - 8 : e - 8;
    };
    auto partial = [&](int j, int e) { return RAGGED && j == 0 && (e < 0 || e + 8 > dim); };
    auto element = [&](int e, int i) { return e + i < 0 ? e + i + n_elements : e + i; }; // (in the row if < dim)
    auto gather = [&](const T *p, int e) {
        T v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = element(e, i) < dim ? p[element(e, i)] : from_f<T>(0.f);
        Raw8<T> r;
        __builtin_memcpy(&r, v, sizeof(r));
        return r;
    };
    // A partial group: `own` as it lies, with the elements before the row from `last`.
    auto join = [&](int e, const Raw8<T> &own, const Raw8<T> &last) {
        T v[8], l[8];
        unpack8(own, v);
        unpack8(last, l);
#pragma unroll
        for (int i = 0; i < 8; ++i)
        {
            v[i] = e + i < 0 ? l[i] : v[i];
            v[i] = element(e, i) < dim ? v[i] : from_f<T>(0.f);
        }
        Raw8<T> r;
        __builtin_memcpy(&r, v, sizeof(r));
        return r;
    };
    constexpr uint32_t kUnit = 8 * sizeof(T);
    auto unit_bytes = [&](int c) { return ((uint32_t)row_bytes + c * (uint32_t)sizeof(T) + kUnit - 1) / kUnit * kUnit; };
    const int n_end = dim >= 8 ? 1 : 8; // rows at each end of the tensor whose units may reach out
    auto at_end = [&](int64_t row) { return row < n_end || row >= a.n_rows - n_end; };
    // Bytes [at, at + n) of the n of a row's units at p are in the tensor's whole 16-byte units.
    auto clip = [&](const void *tensor, const uint8_t *p, uint32_t &at, uint32_t &n) {
        const uintptr_t first = up16((uintptr_t)tensor), end = down16((uintptr_t)tensor + a.n_rows * row_bytes);
        const uintptr_t lo = (uintptr_t)p < (uintptr_t)tensor ? first : (uintptr_t)p;
        const uintptr_t hi = (uintptr_t)p + n < end ? (uintptr_t)p + n : end;
        at = (uint32_t)(lo - (uintptr_t)p);
        n = hi > lo ? (uint32_t)(hi - lo) : 0;
    };
    // Elements that clip leaves out, from global memory.
    auto complete = [&](const void *tensor, int64_t row, int c, uint8_t *stage) {
        const T *src = reinterpret_cast<const T *>(static_cast<const uint8_t *>(tensor) + row * row_bytes);
        uint32_t at = 0, n = unit_bytes(c);
        clip(tensor, reinterpret_cast<const uint8_t *>(src - c), at, n);
        for (int e = tid; e < (int)(row_bytes / (int)sizeof(T)); e += n_threads)
            if ((uint32_t)(c + e) * sizeof(T) < at || (uint32_t)(c + e) * sizeof(T) >= at + n)
                reinterpret_cast<T *>(stage)[c + e] = src[e];
    };
    auto issue = [&](int64_t it, int slot) {
        const int64_t row = blockIdx.x + it * gridDim.x;
        const uint32_t dst = smem_u32(ring) + slot * stage_bytes, bar = smem_u32(&s_full[slot]);
        if constexpr (RAGGED)
        {
            const uint8_t *x = static_cast<const uint8_t *>(base) + row * row_bytes - off * (int)sizeof(T);
            const uint8_t *r = static_cast<const uint8_t *>(a.residual) + row * row_bytes - off2 * (int)sizeof(T);
            uint32_t at_x = 0, at_r = 0, nx = unit_bytes(off), nr = kCopies == 2 ? unit_bytes(off2) : 0;
            if (at_end(row))
            {
                clip(base, x, at_x, nx);
                if (kCopies == 2)
                    clip(a.residual, r, at_r, nr);
            }
            mbar_expect_tx(bar, nx + nr);
            if (nx)
                bulk_load(dst + at_x, x + at_x, nx, bar);
            if (nr)
                bulk_load(dst + input_bytes + at_r, r + at_r, nr, bar);
        }
        else
        {
            mbar_expect_tx(bar, stage_bytes);
            bulk_load(dst, static_cast<const uint8_t *>(base) + row * row_bytes, input_bytes, bar);
            if (kCopies == 2)
                bulk_load(dst + input_bytes, static_cast<const uint8_t *>(a.residual) + row * row_bytes, input_bytes, bar);
        }
    };
    int64_t issued = n_mine < depth ? n_mine : depth; // (thread 0's)
    pdl_trigger();
    if (tid == 0)
    {
        for (int i = 0; i < depth; ++i)
            mbar_init(smem_u32(&s_full[i]), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        pdl_wait();
        for (int i = 0; i < (int)issued; ++i)
            issue(i, i);
    }
    pdl_wait();
    Raw8<T> w[NV];
    if (kNorm)
    {
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            if (!mine(j))
                continue;
            const T *from = static_cast<const T *>(a.w);
            if constexpr (RAGGED)
            {
                const int e = at(j), shift = (int)(((uintptr_t)from / sizeof(T) - cut) & 7), first = e - shift;
                w[j] = first >= 0 && first + 16 <= dim
                           ? load8_shifted<T, false>(reinterpret_cast<const uint8_t *>(from), e, shift, dim)
                           : gather(from, e);
            }
            else
                w[j] = load8(from + at(j));
        }
    }
    __syncthreads();
    const volatile int *abort_flag = &s_abort;

    int slot = 0;
    uint32_t phase = 0;
    for (int64_t it = 0; it < n_mine; ++it)
    {
        const int64_t row = blockIdx.x + it * gridDim.x;
        const uint32_t bar = smem_u32(&s_full[slot]);
        if (!mbar_try(bar, phase) && !mbar_wait(bar, phase, abort_flag))
        {
            atomicCAS(&g_int8_rows_error, 0, ERR_INT8_ROWS_WAIT);
            s_abort = 1;
        }
        const bool arrived = !*abort_flag; // (a row that has not arrived is not written back)
        uint8_t *stage = ring + slot * stage_bytes;
        Held<T, SRC, NV> held[NV];
        typename Held<T, SRC, NV>::RowTop top;
        float sq = 0.f;
        if constexpr (RAGGED)
        {
            if (at_end(row))
            {
                if (arrived)
                {
                    complete(base, row, off, stage);
                    if (kCopies == 2)
                        complete(a.residual, row, off2, stage + input_bytes);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // (the slot is copied to again)
                __syncthreads();
            }
            T *out = static_cast<T *>(a.xio) + row * a.dim;
#pragma unroll
            for (int j = 0; j < NV; ++j)
            {
                int e = at(j);
                asm volatile("" : "+r"(e)); // (addresses are not held over the rows)
                if (!mine(j))
                    continue;
                const int end = off + dim * (SRC == SRC_SWIGLU ? 2 : 1), shift = kNorm ? 0 : (off - cut) & 7;
                auto load = [&](auto check, int pos, int shift) {
                    return load8_shifted<T, decltype(check)::value>(stage, pos, shift, end);
                };
                Raw8<T> in, in2;
                if (!partial(j, e))
                {
                    in = load(std::false_type(), off + e, shift);
                    if (SRC == SRC_SWIGLU)
                        in2 = load(std::false_type(), off + dim + e, (shift + dim) & 7);
                }
                else
                {
                    const std::true_type check;
                    const int last = e + n_elements;
                    const bool wraps = e < 0 && last < dim;
                    in = load(check, off + e, shift);
                    in = join(e, in, wraps ? load(check, off + last, shift) : in);
                    if (SRC == SRC_SWIGLU)
                    {
                        in2 = load(check, off + dim + e, (shift + dim) & 7);
                        in2 = join(e, in2, wraps ? load(check, off + dim + last, (shift + dim) & 7) : in2);
                    }
                }
                if (SRC == SRC_NORM_ADD)
                {
                    const T *p = reinterpret_cast<const T *>(stage + input_bytes) + off2;
                    in2 = off2 == off && !partial(j, e) ? load8_shared<T>(reinterpret_cast<const uint8_t *>(p + e)) : gather(p, e);
                }
                held[j].look(in, in2, w[j], top, sq); // (zeros beside the row add nothing)
                if (SRC == SRC_NORM_ADD && arrived)
                {
                    if (!partial(j, e))
                        store8(out + e, held[j].in);
                    else
                    {
                        T v[8];
                        unpack8(held[j].in, v);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (element(e, i) < dim)
                                out[element(e, i)] = v[i];
                    }
                }
            }
        }
        else
        {
#pragma unroll
            for (int j = 0; j < NV; ++j)
            {
                const int e = at(j);
                if (!mine(j))
                    continue;
                const uint8_t *p = stage + (uint32_t)e * sizeof(T);
                Raw8<T> in = load8_shared<T>(p), in2;
                if (SRC == SRC_NORM_ADD)
                    in2 = load8_shared<T>(p + input_bytes);
                if (SRC == SRC_SWIGLU)
                    in2 = load8_shared<T>(p + (uint32_t)dim * sizeof(T));
                held[j].look(in, in2, w[j], top, sq);
                if (SRC == SRC_NORM_ADD && arrived)
                    store8(static_cast<T *>(a.xio) + row * a.dim + e, held[j].in);
            }
        }
        auto bits = top.bits();
        block_reduce<decltype(bits), kNorm>(bits, sq, (int)(it & 1));
        if (*abort_flag)
            break; // (set before the barrier: the same answer in every thread)
        if (tid == 0 && issued < n_mine)
            issue(issued++, slot);
        const Quantizer<V> z = make_quantizer<V>(bits, kNorm ? inv_rms_of(sq, a.dim) : 1.f);
        int8_t *q = a.q + row * a.dim;
#pragma unroll
        for (int j = 0; j < NV; ++j)
        {
            if (!mine(j))
                continue;
            const uint2 b = held[j].quantized(w[j], z);
            int e = at(j);
            if (RAGGED)
                asm volatile("" : "+r"(e));
            if (q_aligned && !partial(j, e))
                *reinterpret_cast<uint2 *>(q + e) = b;
            else
            {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (element(e, i) < dim)
                        q[element(e, i)] = (int8_t)((i < 4 ? b.x : b.y) >> (8 * (i & 3)));
            }
        }
        if (tid == 0)
            a.scales[row] = z.scale;
        if (++slot == depth)
        {
            slot = 0;
            phase ^= 1;
        }
    }
    if (*abort_flag && tid == 0)
    {
        // after a failure the copies in flight land before the CTA leaves
        const int quiet = 0;
        for (int64_t i = issued > depth ? issued - depth : 0; i < issued; ++i)
            mbar_wait(smem_u32(&s_full[i % depth]), (uint32_t)(i / depth) & 1u, &quiet);
    }
}

// Any length: two passes over the row, an element at a time (the second re-reads
// it, normally from L1 or L2, and recomputes y).
template <typename T, int SRC>
__global__ void __launch_bounds__(kMaxThreads) rows_int8_any_kernel(const RowArgs a)
{
    using V = typename RowValue<T, SRC>::type;
    constexpr bool kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    const int64_t row = blockIdx.x;
    const T *src = static_cast<const T *>(kNorm ? a.xio : a.x) + row * a.dim * (SRC == SRC_SWIGLU ? 2 : 1);
    const T *add = SRC == SRC_NORM_ADD ? static_cast<const T *>(a.residual) + row * a.dim : nullptr;
    const T *w = static_cast<const T *>(a.w);
    T *xio = static_cast<T *>(a.xio) + row * a.dim;
    auto value = [&](int64_t d, float f) -> V {
        if constexpr (SRC == SRC_SWIGLU)
            return silu_up(f, to_f(src[a.dim + d]));
        else if constexpr (kNorm)
            return (V)f * (V)to_f(w[d]);
        else
            return f;
    };
    pdl_trigger();
    pdl_wait();
    Top<V> top;
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
        top.add(value(d, f), (V)0);
    }
    auto bits = top.bits();
    block_reduce<decltype(bits), kNorm>(bits, sq, 0);
    const Quantizer<V> z = make_quantizer<V>(bits, kNorm ? inv_rms_of(sq, a.dim) : 1.f);
    int8_t *q = a.q + row * a.dim;
    for (int64_t d = threadIdx.x; d < a.dim; d += blockDim.x) // (with ADD: this thread's own stores of the first pass)
        q[d] = (int8_t)(quantize1<kShort<T, SRC>>(value(d, to_f(kNorm ? xio[d] : src[d])), z) & 0xffu);
    if (threadIdx.x == 0)
        a.scales[row] = z.scale;
}

constexpr int64_t kSmemPerSM = 220 * 1024;

int cuda_status(cudaError_t e)
{
    if (e == cudaSuccess)
        return L2K_OK;
    (void)cudaGetLastError(); // (else the next launch would report it again)
    return set_error(L2K_ERR_CUDA, "int8 rows: %s", cudaGetErrorString(e));
}

template <typename... P, typename... A>
int launch_pdl(void (*kernel)(P...), unsigned grid, int threads, size_t smem, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = pdl_attribute();
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, P(args)...));
}

// CTAs of `threads` threads that an SM's registers hold: 16384 in each of its four
// parts, allocated in units of 256 for a warp.
template <typename T, int SRC, int NV, bool RAGGED, int THREADS>
int stream_resident(int threads)
{
    static const int regs = [] {
        cudaFuncAttributes f;
        return cudaFuncGetAttributes(&f, rows_int8_stream_kernel<T, SRC, NV, RAGGED, THREADS>) == cudaSuccess ? f.numRegs
                                                                                                              : 128;
    }();
    return std::max(1, 4 * (16384 / ((regs * 32 + 255) / 256 * 256)) / (threads / 32));
}

// The stream kernel on as many CTAs as an SM holds, with a ring that keeps about
// 96 KB an SM in flight (64 to 128 KB measured the same within 2 %, 200 KB up to
// 15 % slower) and at least two rows of each CTA where they fit.
template <typename T, int SRC, int NV, bool RAGGED, int THREADS>
int launch_stream_nv(const RowArgs &a, int64_t input_bytes, int64_t stage_bytes, cudaStream_t stream)
{
    auto kernel = rows_int8_stream_kernel<T, SRC, NV, RAGGED, THREADS>;
    const int threads = (int)(ceil_div(ceil_div(a.dim, 8 * NV), 32) * 32);
    const int64_t resident = std::min(16, stream_resident<T, SRC, NV, RAGGED, THREADS>(threads));
    const int64_t per_sm = std::max<int64_t>(1, std::min(resident, kSmemPerSM / (2 * stage_bytes)));
    const int64_t fits = kSmemPerSM / (per_sm * stage_bytes); // at least 1 (stage_bytes <= kSmemPerSM)
    const int depth = (int)std::min({std::max<int64_t>(96 * 1024 / (per_sm * stage_bytes), 2), fits, (int64_t)kMaxDepth});
    const int st = cuda_status(
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemPerSM));
    if (st != L2K_OK)
        return st;
    const int64_t most = per_sm * num_sms();
    const int64_t grid = std::min<int64_t>(a.n_rows, RAGGED ? std::max<int64_t>(8, most / 8 * 8) : most);
    return launch_pdl(kernel, (unsigned)grid, threads, (size_t)(depth * stage_bytes), stream, a, depth, (uint32_t)input_bytes);
}

// Groups per thread: one for the shortest rows (a warp or less); four for 16-bit
// rows (the reduction's fixed cost of about 60 instructions a warp is shared by
// four groups: 16384 x 4096 bf16 rows 40 us, 44 with two, eight no faster), two where a few rows per
// SM leave threads idle (512 rows: 4.0 us, 4.7 with one); two for fp32 rows (53 us,
// 60 with four) and one for fp32 SwiGLU (90 us, 99 with two) and a few ragged
// rows; more where the row needs it. CTAs of 352 to 448 threads would leave an SM
// one of them at the 86 to 96 registers of the plain instantiation: 4099 x 13824 f16
// SwiGLU 75 us, 56 with two; 8192 x 11008 bf16 rows 74, 55 with two; likewise fp32
// norms of 288 to 320 threads (8192 x 5120: 114 us, 95 with two), and fp32 ragged rows
// of any length (16384 x 4095 SwiGLU 230 us at 115 registers, 116 at 72; 16-bit ones
// without gain: 16384 x 1023 rows 29 us, 19 without). 16-bit norms stay at
// their 122 to 126: held to 80 they spill (16384 x 4096: 94 us against 76).
template <typename T, int SRC, bool RAGGED>
int launch_stream(const RowArgs &a, int64_t input_bytes, int64_t stage_bytes, cudaStream_t stream)
{
    constexpr bool kWide = sizeof(T) == 4, kNorm = SRC == SRC_NORM || SRC == SRC_NORM_ADD;
    const int64_t groups = ceil_div(a.dim, 8);
    const bool few = a.n_rows <= 4 * num_sms();
    const int want = groups <= 32 || (kWide && SRC == SRC_SWIGLU) || (RAGGED && few) ? 1
                     : kWide || groups <= 64 || (few && !kNorm)                      ? 2
                                                                                     : 4;
    constexpr int kMost = RAGGED && !kNorm && kWide ? 448 : kStreamThreads;
    if (want == 1 && groups <= kMost)
        return launch_stream_nv<T, SRC, 1, RAGGED, kMost>(a, input_bytes, stage_bytes, stream);
    if constexpr (kNorm && kWide)
        if (groups > 2 * 256 && groups <= 2 * 320)
            return launch_stream_nv<T, SRC, 2, RAGGED, 320>(a, input_bytes, stage_bytes, stream);
    if (want <= 2 && groups <= 2 * kMost)
        return launch_stream_nv<T, SRC, 2, RAGGED, kMost>(a, input_bytes, stage_bytes, stream);
    if constexpr (!kNorm)
        if (groups > 4 * 320 && groups <= 4 * 448)
            return launch_stream_nv<T, SRC, 4, RAGGED, 448>(a, input_bytes, stage_bytes, stream);
    return launch_stream_nv<T, SRC, 4, RAGGED, kStreamThreads>(a, input_bytes, stage_bytes, stream);
}

template <typename T, int SRC>
int launch_rows(const RowArgs &a, const char *name, cudaStream_t stream)
{
    const bool vec = a.dim % 8 == 0 && is_aligned(a.x, 16) && is_aligned(a.xio, 16) && is_aligned(a.residual, 16) &&
                     is_aligned(a.w, 16) && is_aligned(a.q, 8);
    constexpr int64_t kUnit = 8 * sizeof(T);
    const int64_t groups = ceil_div(a.dim, 8);
    const int64_t row_bytes = a.dim * (SRC == SRC_SWIGLU ? 2 : 1) * (int64_t)sizeof(T);
    // (without alignment: the units of 8 elements that a row touches)
    const int64_t input_bytes = vec ? row_bytes : (row_bytes + 7 * (int64_t)sizeof(T) + kUnit - 1) / kUnit * kUnit;
    const int64_t stage_bytes = input_bytes * (SRC == SRC_NORM_ADD ? 2 : 1);
    const bool stream_fits = groups <= 4 * kStreamThreads && stage_bytes <= kSmemPerSM;
    int st = L2K_OK;
    if (vec && a.n_rows <= 2 * num_sms() && groups <= 2 * kMaxThreads)
    {
        // few rows: latency, so as many threads as there are groups
        if (groups <= kMaxThreads)
            st = launch_pdl(rows_int8_kernel<T, SRC, 1>, (unsigned)a.n_rows, (int)(ceil_div(groups, 32) * 32), 0, stream, a);
        else
            st = launch_pdl(rows_int8_kernel<T, SRC, 2>, (unsigned)a.n_rows, (int)(ceil_div(groups, 64) * 32), 0, stream, a);
    }
    else if (stream_fits)
        st = vec ? launch_stream<T, SRC, false>(a, input_bytes, stage_bytes, stream)
                 : launch_stream<T, SRC, true>(a, input_bytes, stage_bytes, stream);
    else
        st = launch_pdl(rows_int8_any_kernel<T, SRC>, (unsigned)a.n_rows, kMaxThreads, 0, stream, a);
    return st != L2K_OK ? st : check_launch(name);
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
        return cuda_status(cudaMemsetAsync(a.scales, 0, (size_t)a.n_rows * sizeof(float), stream));
    }
    const uintptr_t es = dtype_size(dtype);
    L2K_REQUIRE(is_aligned(a.x, es) && is_aligned(a.xio, es) && is_aligned(a.residual, es) && is_aligned(a.w, es) &&
                    is_aligned(a.scales, 4),
                "%s: a tensor is not aligned to its elements", name);
    L2K_REQUIRE_SHAPE(a.n_rows < (int64_t(1) << 31), "%s: more than 2^31 - 1 rows", name);
    *done = false;
    return L2K_OK;
}

} // namespace

int read_int8_rows_error(bool clear)
{
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_int8_rows_error, sizeof(int)) != cudaSuccess)
        return -1;
    if (clear && v)
    {
        const int zero = 0;
        if (cudaMemcpyToSymbol(g_int8_rows_error, &zero, sizeof(int)) != cudaSuccess)
            return -1;
    }
    return v;
}

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
