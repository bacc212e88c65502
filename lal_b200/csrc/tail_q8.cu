/*
 * tail_q8.cu -- rows quantized to 8 bits as they are computed: what feeds the
 * 4-bit products of a layer (tail_q4.cu).
 *
 *   NormRow    h = x + residual (rounded to its type), v = h * w,
 *              scale = max|v| / sqrt(mean h^2 + eps) / 127
 *   SwigluRow  v = gate / (1 + exp(-gate)) * up, scale = max|v| / 127
 *
 * and q = rint(127 v / max|v|), ties to even, as in 64 bits: the norm's factor
 * cancels in q, so one reduction gives both the sum of squares and max|v|.
 *
 * v is computed in 32 bits.  Where 127 v / max|v| then lies so near a border
 * between two steps that the rounding of v could have moved it across, the
 * element is computed again in 64 bits; rows whose largest value is outside
 * the comfortable range of 32 bits take 64 bits throughout.  So q does not
 * depend on the order of the sum, on the launch's shape or on how v is split
 * over threads.
 */
#include "tail_layer.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>

using namespace lal;

namespace {

struct RowParams {
    const void *a, *b; /* x and the residual, or gate and up */
    void *h;
    const float *w;
    long long a_stride, b_stride, h_stride, q_stride;
    int n;
    float eps;
    int8_t *q;
    float *scale;
    int parts;   /* CTAs a row */
    float inv_n; /* 1 / n */
};

/* What few elements need, out of line: inlined for each of a thread's elements
 * it would fill the instruction cache. */
__device__ __noinline__ double silu64(double g, double u) { return g / (1.0 + exp(-g)) * u; }
__device__ __noinline__ int round64(double v, double top) { return (int)rint(127.0 * v / top); }

constexpr float kFltMax = 3.4028234663852886e38f;
/* max|v| in 32 bits at or above kWideHi or (not zero) below kWideLo: the row
 * is computed in 64 bits, clear of overflow and of denormal rounding */
constexpr float kWideHi = 1e37f, kWideLo = 1e-30f;

/* Eight elements of a row as they lie in memory. */
template <typename T> union Eight {
    uint4 q[sizeof(T) / 2];
    uint32_t w[2 * sizeof(T)];
    unsigned short s[4 * sizeof(T)];
    T e[8];
    __device__ Eight() {}
};

/* From p on, of which `n` exist (the others 0).  kWide: all do, at a 16-byte
 * boundary; else as wide as p's alignment allows (rows of 16-bit elements may
 * begin at any even address). */
template <bool kWide, typename T> __device__ __forceinline__ void get8(const T *p, int n, Eight<T> &v) {
    const unsigned at = (unsigned)(uintptr_t)p;
    if (kWide || (n == 8 && (at & 15) == 0)) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) v.q[i] = ((const uint4 *)p)[i];
    } else if (n == 8 && (sizeof(T) == 4 || (at & 3) == 0)) {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) v.w[i] = ((const uint32_t *)p)[i];
    } else if (n == 8) {
        const uint32_t *w = (const uint32_t *)(p + 1);
        const uint32_t m0 = w[0], m1 = w[1], m2 = w[2];
        const uint32_t first = ((const unsigned short *)p)[0], last = ((const unsigned short *)p)[7];
        v.w[0] = first | m0 << 16;
        v.w[1] = __funnelshift_r(m0, m1, 16);
        v.w[2] = __funnelshift_r(m1, m2, 16);
        v.w[3] = m2 >> 16 | last << 16;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v.e[i] = i < n ? p[i] : from_f32<T>(0.0f);
    }
}
template <bool kWide, typename T> __device__ __forceinline__ void put8(T *p, int n, const Eight<T> &v) {
    const unsigned at = (unsigned)(uintptr_t)p;
    if (kWide || (n == 8 && (at & 15) == 0)) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)p)[i] = v.q[i];
    } else if (n == 8 && (sizeof(T) == 4 || (at & 3) == 0)) {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) ((uint32_t *)p)[i] = v.w[i];
    } else if (n == 8) {
        p[0] = v.e[0];
#pragma unroll
        for (int i = 0; i < 3; ++i) ((uint32_t *)(p + 1))[i] = __funnelshift_r(v.w[i], v.w[i + 1], 16);
        p[7] = v.e[7];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = v.e[i];
    }
}
template <typename T> __device__ __forceinline__ void to8(const Eight<T> &v, float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = to_f32(v.e[i]);
}
/* a + b, rounded to the type.  (16-bit sums rounded once are those rounded to
 * fp32 first: where fp32 rounds, the smaller term is below 2^-13 of the larger
 * and the sum far from halfway between two 16-bit numbers.) */
__device__ __forceinline__ void add8(Eight<float> &a, const Eight<float> &b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.e[i] = __fadd_rn(a.e[i], b.e[i]);
}
template <typename T> __device__ __forceinline__ void add8(Eight<T> &a, const Eight<T> &b) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        T2 u, v;
        memcpy(&u, &a.w[i], 4);
        memcpy(&v, &b.w[i], 4);
        u = __hadd2_rn(u, v);
        memcpy(&a.w[i], &u, 4);
    }
}

/* n of eight bytes */
template <bool kWide> __device__ __forceinline__ void put_q8(int8_t *p, int n, const uint32_t (&w)[2]) {
    const unsigned at = (unsigned)(uintptr_t)p;
    if (kWide || (n == 8 && (at & 7) == 0)) {
        *(uint2 *)p = make_uint2(w[0], w[1]);
    } else if (n == 8 && (at & 3) == 0) {
        ((uint32_t *)p)[0] = w[0];
        ((uint32_t *)p)[1] = w[1];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = (int8_t)(w[i / 4] >> (8 * (i % 4)));
    }
}

/* What the two kinds of rows have of their own: v of eight elements in 32
 * bits, v of one in 64. */
template <typename T, bool kWide_> struct NormRow {
    static constexpr bool kWide = kWide_;
    const T *x, *r;
    T *h;
    const float *w;
    int n;
    /* v: 2^-24; 127 / max|v|: 2 * 2^-24; their product: 2^-24; times 127: below 3.1e-5 */
    static constexpr float kBorder = 4e-5f;
    static constexpr float kRelative = 0.0f;
    static constexpr bool kNorm = true;
    __device__ NormRow(const RowParams &p, int at)
        : x((const T *)p.a + (size_t)at * p.a_stride),
          r(p.b != nullptr ? (const T *)p.b + (size_t)at * p.b_stride : nullptr),
          h(p.h != nullptr ? (T *)p.h + (size_t)at * p.h_stride : nullptr), w(p.w), n(p.n) {}
    /* adds the residual, stores the sum, adds its squares to `sum` */
    __device__ void load(int i, float (&v)[8], double &sum) const {
        const int m = min(8, n - i);
        Eight<T> a;
        get8<kWide>(x + i, m, a);
        Eight<float> u;
        get8<kWide>(w + i, m, u);
        if (r != nullptr) {
            Eight<T> b;
            get8<kWide>(r + i, m, b);
            add8(a, b);
        }
        if (h != nullptr) put8<kWide>(h + i, m, a);
        to8(a, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = fma((double)v[j], (double)v[j], sum);
            v[j] = __fmul_rn(v[j], u.e[j]);
        }
    }
    /* the same v again, by the thread that loaded it */
    __device__ void again(int i, float (&v)[8]) const {
        const int m = min(8, n - i);
        Eight<T> a;
        get8<kWide>(h != nullptr ? (const T *)h + i : x + i, m, a);
        Eight<float> u;
        get8<kWide>(w + i, m, u);
        to8(a, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], u.e[j]);
    }
    __device__ double v64(int i) const { return (double)to_f32(h != nullptr ? h[i] : x[i]) * (double)w[i]; }
};

template <typename T, bool kWide_> struct SwigluRow {
    static constexpr bool kWide = kWide_;
    const T *g, *u;
    int n;
    /* Relative errors: exp(-gate) 2^-22 of ex2 and 2^-23 around it, 1 + e 2^-24, its reciprocal 2^-23,
     * two products 2^-24 each, 127 / max|v| 2^-23, the product with it 2^-24: below 1e-6 */
    static constexpr float kRelative = 1.2e-6f;
    static constexpr float kBorder = 0.0f;
    static constexpr bool kNorm = false;
    __device__ SwigluRow(const RowParams &p, int at)
        : g((const T *)p.a + (size_t)at * p.a_stride), u((const T *)p.b + (size_t)at * p.b_stride),
          n(p.n) {}
    __device__ void load(int i, float (&v)[8], double &) const {
        const int m = min(8, n - i);
        float up[8], low = 0.0f;
        Eight<T> a, b;
        get8<kWide>(g + i, m, a);
        get8<kWide>(u + i, m, b);
        to8(a, v);
        to8(b, up);
#pragma unroll
        for (int j = 0; j < 8; ++j) low = fminf(low, v[j]);
        if (low < -80.0f) { /* there 1 + exp(-gate) leaves the reciprocal's range */
#pragma unroll 1
            for (int j = 0; j < m; ++j) {
                const float w = (float)v64(i + j);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    if (k == j) v[k] = w;
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            /* exp(-g) = 2^hi (1 + lo ln 2), hi + lo = -g log2 e */
            constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596303e-8f, kLn2 = 0.693147182f;
            const float hi = __fmul_rn(v[j], -kLog2e);
            const float lo = fmaf(v[j], -kLog2eLow, fmaf(v[j], -kLog2e, -hi));
            float e, r;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(hi));
            e = fmaf(__fmul_rn(e, lo), kLn2, e);
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.0f, e)));
            /* gate * up first: where that is subnormal v is too, far below any row's step, while gate * r
             * may be subnormal and v large.  Gates above 2.36e38 give NaN (hi overflows), products that
             * overflow infinity: such rows find their maximum, and store() such elements, in 64 bits. */
            v[j] = __fmul_rn(__fmul_rn(v[j], up[j]), r);
        }
    }
    __device__ void again(int i, float (&v)[8]) const {
        double none;
        load(i, v, none);
    }
    __device__ double v64(int i) const {
        const float a = to_f32(g[i]), b = to_f32(u[i]);
        return a == 0.0f || b == 0.0f ? (double)a * (double)b : silu64((double)a, (double)b);
    }
};

/* Doubles that are not negative, NaN above all, order as their bits. */
__device__ __forceinline__ unsigned long long abs_bits(double v) {
    return (unsigned long long)__double_as_longlong(v) & 0x7fffffffffffffffull;
}

__device__ __forceinline__ double of_bits(unsigned long long b) {
    double v;
    memcpy(&v, &b, sizeof v);
    return v;
}

/* max with NaN above all */
__device__ __forceinline__ float max_nan(float a, float b) {
    float v;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(v) : "f"(a), "f"(b));
    return v;
}

constexpr int kMaxParts = 8; /* CTAs of a row: a portable cluster */

/* A row's statistics: across a CTA, then across the CTAs of the row. */
struct RowShared {
    double sums[32];
    unsigned tops[32];
    unsigned long long top; /* max|v| of this CTA's part, in 64 bits */
    double part_sum[kMaxParts];
    unsigned long long part_top[kMaxParts];
};

__device__ __forceinline__ bool row_wide(float top32) { return !(top32 < kWideHi && top32 >= kWideLo); }

/* The row's max|v| in 64 bits and sum of squares, in every thread, from each
 * thread's largest |v| in 32 bits `m` and `sum`.  Only elements whose |v| may
 * be the largest (its error is below 1e-6) are computed in 64 bits; `best(least)`
 * is their largest, as bits, of the thread's elements not below `least`. */
template <bool kNorm, bool kCluster, typename Best>
__device__ __forceinline__ double row_stat(RowShared &sh, int parts, int part, float m, double &sum, Best best) {
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned top_warp = __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu);
    if (kNorm)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        sh.tops[warp] = top_warp;
        sh.sums[warp] = sum;
    }
    if (threadIdx.x == 0) sh.top = 0;
    __syncthreads();
    const float top32 = __uint_as_float(__reduce_max_sync(0xffffffffu, lane < warps ? sh.tops[lane] : 0u));
    const float least = row_wide(top32) ? 0.0f : top32 * (1.0f - 4e-6f);
    if (!(m < least)) {
        const unsigned long long b = best(least);
        if (b) atomicMax(&sh.top, b);
    }
    if (kNorm && warp == 0) {
        sum = lane < warps ? sh.sums[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sh.part_sum[part] = sum;
    }
    __syncthreads();
    if (!kCluster) {
        if (kNorm) sum = sh.part_sum[0];
        return of_bits(sh.top);
    }
    /* to every CTA of the row, once all have begun; none leaves before all have written */
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (threadIdx.x < parts) {
        uint32_t at;
        const unsigned long long top = sh.top;
        const uint32_t here = (uint32_t)__cvta_generic_to_shared(&sh.part_top[part]);
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(here), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(top) : "memory");
        if (kNorm) {
            const uint32_t here_s = (uint32_t)__cvta_generic_to_shared(&sh.part_sum[part]);
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(here_s), "r"(threadIdx.x));
            asm volatile("st.shared::cluster.b64 [%0], %1;" ::"r"(at), "l"(__double_as_longlong(sh.part_sum[part])) : "memory");
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const unsigned long long top = lane < parts ? sh.part_top[lane] : 0;
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(top >> 32));
    const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(top >> 32) == high ? (unsigned)top : 0u);
    if (kNorm) {
        sum = 0.0;
        for (int i = 0; i < parts; ++i) sum += sh.part_sum[i];
    }
    return of_bits((unsigned long long)high << 32 | low);
}

/* A row's quantizer, once max|v| and the sum of squares are known. */
template <typename Row> struct RowQuant {
    double top, sum;
    float r32; /* 127 / top */
    bool wide, fits; /* fits: fp32 holds the scale; else the row is NaN */

    __device__ double factor(const RowParams &p) const {
        return Row::kNorm ? 1.0 / sqrt(sum / p.n + (double)p.eps) : 1.0;
    }
    __device__ RowQuant(const RowParams &p, double top_, double sum_) : top(top_), sum(sum_) {
        float about = (float)top;
        wide = row_wide(about);
        r32 = __fdiv_rn(127.0f, about);
        if (Row::kNorm) about *= rsqrtf((float)sum * p.inv_n + p.eps);
        fits = about < 1e38f || top == 0.0 || top * factor(p) <= (double)kFltMax;
    }
    /* 1.5 * 2^23: added, it leaves the nearest integer in the low bits */
    static constexpr float kRound = 12582912.0f;
    /* how far t may be from the nearest integer, u - kRound */
    static __device__ __forceinline__ float off_centre(float t, float u) {
        const float d = __fsub_rn(t, __fsub_rn(u, kRound));
        return Row::kRelative > 0.0f ? fabsf(d) + fabsf(__fmul_rn(t, Row::kRelative)) : fabsf(d);
    }
    /* q of the eight elements from i on */
    __device__ void store(const RowParams &p, const Row &row, int8_t *q, int i, const float (&v)[8]) const {
        float u[8], far = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = __fmul_rn(v[j], r32);
            u[j] = __fadd_rn(t, kRound);
            far = max_nan(far, off_centre(t, u[j])); /* a v that 32 bits do not have goes to 64 */
        }
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
            w[h] = __byte_perm(__byte_perm(__float_as_uint(u[4 * h]), __float_as_uint(u[4 * h + 1]), 0x0040),
                               __byte_perm(__float_as_uint(u[4 * h + 2]), __float_as_uint(u[4 * h + 3]), 0x0040), 0x5410);
        const bool none = !fits || top == 0.0;
        if (none) w[0] = w[1] = 0;
        const int n = Row::kWide ? 8 : min(8, p.n - i);
        put_q8<Row::kWide>(q + i, n, w);
        if ((wide || !(far < 0.5f - Row::kBorder)) && !none) { /* next to a border: 64 bits decide */
            unsigned near = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float t = __fmul_rn(v[j], r32);
                near |= (wide || !(off_centre(t, __fadd_rn(t, kRound)) < 0.5f - Row::kBorder) ? 1u : 0u) << j;
            }
            near &= (1u << n) - 1u;
            for (; near != 0; near &= near - 1) {
                const int j = i + __ffs(near) - 1;
                q[j] = (int8_t)round64(row.v64(j), top);
            }
        }
    }
    __device__ float scale(const RowParams &p) const {
        return !fits ? __int_as_float(0x7fc00000) : top == 0.0 ? 0.0f : (float)(top * factor(p) / 127.0);
    }
};

/* A row a CTA, or (kCluster) a cluster: 8 kC elements a thread, which stay in
 * registers between the statistics and the quantizer.  Norm of 4096x3584 bf16
 * with its residual 26.4 us (0.60 of the measured HBM rate; fp32 35.5, 0.82),
 * SwiGLU of 512x18944 bf16 24.6 us (0.30; fp32 28.6, 0.47): bounded by latency, a
 * row's loads, barriers and stores one after the other with nothing of the next
 * row in flight (the instructions, 27 and 39 an element, are 10 us of issue at
 * most).  One row of 3584 and of 18944: 2.4 and 3.0 us. */
template <typename Row, int kC, int kMaxThreads, int kMinCtas, bool kCluster>
__global__ void __launch_bounds__(kMaxThreads, kMinCtas) row_q8_kernel(const RowParams p) {
    after_previous();
    __shared__ RowShared sh;
    const int parts = kCluster ? p.parts : 1, part = kCluster ? blockIdx.x % parts : 0;
    const int at = kCluster ? blockIdx.x / parts : blockIdx.x;
    if (kCluster) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    const Row row(p, at);
    const int first = part * blockDim.x * (8 * kC);
    float v[kC][8], m = 0.0f;
    double sum = 0.0;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        const int i = first + (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
        if (i < p.n) row.load(i, v[c], sum);
    }
#pragma unroll
    for (int c = 0; c < kC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[c][j]));
    const double top = row_stat<Row::kNorm, kCluster>(sh, parts, part, m, sum, [&](float least) {
        unsigned long long best = 0;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int i = first + (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < p.n && !(fabsf(v[c][j]) < least)) best = max(best, abs_bits(row.v64(i + j)));
        }
        return best;
    });
    const RowQuant<Row> rq(p, top, sum);
    int8_t *q = p.q + (size_t)at * p.q_stride;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        const int i = first + (c * blockDim.x + threadIdx.x) * 8;
        if (i < p.n) rq.store(p, row, q, i, v[c]);
    }
    if (part == 0 && threadIdx.x == 0) p.scale[at] = rq.scale(p);
}

/* Rows longer than that: one CTA, and every element is visited again. */
constexpr int kLongThreads = 512;
template <typename Row> __global__ void __launch_bounds__(kLongThreads) row_q8_long_kernel(const RowParams p) {
    after_previous();
    __shared__ RowShared sh;
    const Row row(p, blockIdx.x);
    double sum = 0.0;
    float v[8], m = 0.0f;
    for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
        row.load(i, v, sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(v[j]));
    }
    const double top = row_stat<Row::kNorm, false>(sh, 1, 0, m, sum, [&](float least) {
        unsigned long long best = 0;
        for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
            row.again(i, v);
            for (int j = 0; j < 8; ++j)
                if (i + j < p.n && !(fabsf(v[j]) < least)) best = max(best, abs_bits(row.v64(i + j)));
        }
        return best;
    });
    const RowQuant<Row> rq(p, top, sum);
    int8_t *q = p.q + (size_t)blockIdx.x * p.q_stride;
    for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
        row.again(i, v);
        rq.store(p, row, q, i, v);
    }
    if (threadIdx.x == 0) p.scale[blockIdx.x] = rq.scale(p);
}

template <typename Row, int kC, int kMaxThreads, int kMinCtas>
cudaError_t launch_parts(RowParams p, int rows, int parts, cudaStream_t st) {
    const int eights = (p.n + 7) / 8;
    const int threads = ((eights + parts * kC - 1) / (parts * kC) + 31) / 32 * 32;
    p.parts = parts;
    return launch_early(parts == 1 ? row_q8_kernel<Row, kC, kMaxThreads, kMinCtas, false>
                                   : row_q8_kernel<Row, kC, kMaxThreads, kMinCtas, true>,
                        dim3((unsigned)(rows * parts)), threads, 0, st, parts, p);
}

constexpr int kFewN = 8192, kFewPart = 2048;
template <typename Row> cudaError_t launch_row(RowParams p, int rows, int num_sms, cudaStream_t st) {
    p.inv_n = 1.0f / (float)p.n;
    /* Few rows: a thread takes 8 elements, and a long row is spread over as
     * many SMs as a cluster has (SwiGLU of one row of 18944: 8.7 us in one CTA,
     * 3.0 over a cluster).  Many: 16 elements, and no more CTAs a row than its
     * registers need; SwiGLU's in smaller CTAs (512 rows: 24.6 us against 31.4 with
     * CTAs of 512 threads), the norm's in larger ones (26.4 against 27.4). */
    if (rows < 2 * num_sms) {
        if (p.n <= kFewN) return launch_parts<Row, 1, 1024, 1>(p, rows, 1, st);
        if (p.n <= kMaxParts * 8192) return launch_parts<Row, 1, 1024, 1>(p, rows, std::min(kMaxParts, (p.n + kFewPart - 1) / kFewPart), st);
    } else if (p.n <= kMaxParts * 8192 && rows <= 0x7fffffff / kMaxParts) {
        if (Row::kNorm) return launch_parts<Row, 2, 512, 2>(p, rows, (p.n + 8191) / 8192, st);
        if (p.n <= kMaxParts * 4096) return launch_parts<Row, 2, 256, 5>(p, rows, (p.n + 4095) / 4096, st);
    }
    return launch_early(row_q8_long_kernel<Row>, dim3((unsigned)rows), kLongThreads, 0, st, 1, p);
}

/* kWide where every row of every buffer begins at a 16-byte boundary (q: 8)
 * and ends at a whole eight: no test of alignment or of the end an element.
 * Against the other form on the same rows, us: norm 4096x3584 bf16 26.4 and
 * 27.8, fp32 35.5 and 36.8; SwiGLU 512x18944 bf16 24.6 and 24.8, fp32 28.6 and
 * 27.7.  Norm of rows that are not aligned 31.7. */
template <template <typename, bool> class Row, typename T>
cudaError_t launch_rows(const RowParams &p, int rows, int num_sms, cudaStream_t st) {
    const long long strides = p.a_stride | p.b_stride | (p.h != nullptr ? p.h_stride : 0);
    const bool wide = p.n % 8 == 0 && (((uintptr_t)p.a | (uintptr_t)p.b | (uintptr_t)p.h | (uintptr_t)p.w) & 15) == 0 &&
                      strides * (long long)sizeof(T) % 16 == 0 && ((uintptr_t)p.q | (uintptr_t)p.q_stride) % 8 == 0;
    return wide ? launch_row<Row<T, true>>(p, rows, num_sms, st) : launch_row<Row<T, false>>(p, rows, num_sms, st);
}

}  // namespace

extern "C" {

int lal_tail_add_rms_norm_q8(const void *d_x, int64_t x_stride, const void *d_residual,
                             int64_t residual_stride, void *d_h, int64_t h_stride, int dtype,
                             const float *d_norm_w, float eps, int rows, int n_embd, int8_t *d_q,
                             int64_t q_stride, float *d_scale, void *stream) {
    static const char *op = "add_rms_norm_q8";
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (rows < 0 || n_embd < 1 || n_embd > kLayerMaxDim)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: %d rows of %d", op, rows, n_embd);
    if (!(eps >= 0.0f && eps <= kFltMax))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: eps %g", op, (double)eps);
    if (rows == 0) return LAL_TAIL_OK;
    if (!d_x || !d_norm_w || !d_q || !d_scale)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (d_residual && !d_h)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a residual, and no d_h for the sum", op);
    if (x_stride < n_embd || q_stride < n_embd || (d_residual && residual_stride < n_embd) ||
        (d_h && h_stride < n_embd))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below n_embd %d", op, n_embd);
    const uintptr_t m = (uintptr_t)d_x | (uintptr_t)d_residual | (uintptr_t)d_h;
    if (m % size != 0 || (uintptr_t)d_norm_w % 4 != 0 || (uintptr_t)d_scale % 4 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    /* the sum may take the place of x or of the residual, and nothing else may meet */
    const Span x(d_x, rows, n_embd, x_stride, size), r(d_residual, rows, n_embd, residual_stride, size),
        h(d_h, rows, n_embd, h_stride, size), w(d_norm_w, 1, n_embd, n_embd, 4),
        q(d_q, rows, n_embd, q_stride, 1), s(d_scale, 1, rows, rows, 4);
    if (!all_fit({x, r, h, q})) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride beyond the address space", op);
    const bool h_on_x = d_h == d_x && h_stride == x_stride;
    const bool h_on_r = d_residual && d_h == d_residual && h_stride == residual_stride;
    if ((!h_on_x && h.meets(x)) || (!h_on_r && h.meets(r)) || h.meets(w) || h.meets(q) || h.meets(s) ||
        q.meets(x) || q.meets(r) || q.meets(w) || q.meets(s) || s.meets(x) || s.meets(r) || s.meets(w))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_x", "d_residual", "d_h", "d_norm_w", "d_q", "d_scale"};
    const void *ptrs[] = {d_x, d_residual, d_h, d_norm_w, d_q, d_scale};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 6)) return rc;
    const RowParams p = {d_x, d_residual, d_h, d_norm_w, x_stride, residual_stride, h_stride, q_stride,
                         n_embd, eps, d_q, d_scale, 1, 0.0f};
    cudaStream_t st = (cudaStream_t)stream;
    return launched(op, dtype == LAL_TAIL_F32    ? launch_rows<NormRow, float>(p, rows, dev.num_sms(), st)
                        : dtype == LAL_TAIL_BF16 ? launch_rows<NormRow, __nv_bfloat16>(p, rows, dev.num_sms(), st)
                                                 : launch_rows<NormRow, __half>(p, rows, dev.num_sms(), st));
}

int lal_tail_swiglu_q8(const void *d_gate, int64_t gate_stride, const void *d_up, int64_t up_stride,
                       int dtype, int rows, int n, int8_t *d_q, int64_t q_stride, float *d_scale,
                       void *stream) {
    static const char *op = "swiglu_q8";
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (rows < 0 || n < 1 || n > kLayerMaxDim) return layer_fail(LAL_TAIL_ERR_ARG, "%s: %d rows of %d", op, rows, n);
    if (rows == 0) return LAL_TAIL_OK;
    if (!d_gate || !d_up || !d_q || !d_scale)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (gate_stride < n || up_stride < n || q_stride < n)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below n %d", op, n);
    if (((uintptr_t)d_gate | (uintptr_t)d_up) % size != 0 || (uintptr_t)d_scale % 4 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    const Span g(d_gate, rows, n, gate_stride, size), u(d_up, rows, n, up_stride, size),
        q(d_q, rows, n, q_stride, 1), s(d_scale, 1, rows, rows, 4);
    if (!all_fit({g, u, q})) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride beyond the address space", op);
    if (q.meets(g) || q.meets(u) || q.meets(s) || s.meets(g) || s.meets(u))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_gate", "d_up", "d_q", "d_scale"};
    const void *ptrs[] = {d_gate, d_up, d_q, d_scale};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const RowParams p = {d_gate, d_up, nullptr, nullptr, gate_stride, up_stride, 0, q_stride,
                         n, 0.0f, d_q, d_scale, 1, 0.0f};
    cudaStream_t st = (cudaStream_t)stream;
    return launched(op, dtype == LAL_TAIL_F32    ? launch_rows<SwigluRow, float>(p, rows, dev.num_sms(), st)
                        : dtype == LAL_TAIL_BF16 ? launch_rows<SwigluRow, __nv_bfloat16>(p, rows, dev.num_sms(), st)
                                                 : launch_rows<SwigluRow, __half>(p, rows, dev.num_sms(), st));
}

}  // extern "C"
