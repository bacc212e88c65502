/*
 * tail_q8.cu -- rows quantized to 8 bits as they are computed: what feeds the
 * 4-bit products of a layer (tail_q4.cu).
 *
 *   norm_q8_kernel    h = x + residual (rounded to its type), v = h * w,
 *                     scale = max|v| / sqrt(mean h^2 + eps) / 127
 *   swiglu_q8_kernel  v = gate / (1 + exp(-gate)) * up, scale = max|v| / 127
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

#include <cmath>

using namespace lal;

namespace {

constexpr int kRowThreads = 256;
constexpr float kFltMax = 3.4028234663852886e38f;
/* |v| in 32 bits at or above kWideHi or (not zero) below kWideLo: the row is
 * computed in 64 bits, clear of overflow and of denormal rounding */
constexpr float kWideHi = 1e37f, kWideLo = 1e-30f;

/* One element of a row, in 32 and in 64 bits. */
template <typename T> struct NormRow {
    const T *x, *r;
    T *h;
    const float *w;
    /* |error of v()| <= 2^-24, of 127/max|v| 2^-24, of their product 2^-24: 3 * 2^-24 * 127 < 3e-5 */
    static constexpr float kBorder = 3e-5f;
    static constexpr bool kNorm = true;
    struct Elem {
        float h, w;
        __device__ float v() const { return __fmul_rn(h, w); }
        __device__ double v64() const { return (double)h * (double)w; }
        __device__ bool zero() const { return h == 0.0f || w == 0.0f; }
    };
    /* first visit: adds the residual and stores the sum */
    __device__ Elem first(int i) const {
        float a = to_f32(x[i]);
        if (r != nullptr) a = to_f32(from_f32<T>(__fadd_rn(a, to_f32(r[i]))));
        if (h != nullptr) h[i] = from_f32<T>(a);
        return {a, __ldg(w + i)};
    }
    /* second visit, by the thread that made the first */
    __device__ Elem again(int i) const { return {to_f32(h != nullptr ? h[i] : x[i]), __ldg(w + i)}; }
};

template <typename T> struct SwigluRow {
    const T *g, *u;
    /* expf 2 ulp, 1 + e, the division and the product 0.5 ulp each (2^-23), then as above:
     * (3.5 * 2^-23 + 2 * 2^-24) * 127 < 7e-5 */
    static constexpr float kBorder = 1e-4f;
    static constexpr bool kNorm = false;
    struct Elem {
        float g, u;
        __device__ float v() const { return __fmul_rn(__fdiv_rn(g, 1.0f + expf(-g)), u); }
        __device__ double v64() const { return (double)g / (1.0 + exp(-(double)g)) * (double)u; }
        __device__ bool zero() const { return g == 0.0f || u == 0.0f; }
    };
    __device__ Elem first(int i) const { return {to_f32(g[i]), to_f32(u[i])}; }
    __device__ Elem again(int i) const { return first(i); }
};

/* A thread's part of a row's statistics. */
struct RowStat {
    double sum = 0.0;   /* of h^2 */
    double top = 0.0;   /* max|v| in 64 bits; NaN or infinite if a v is */
    float top32 = 0.0f;
    bool wide = false;

    template <typename E> __device__ void take(const E &e) {
        const float a = fabsf(e.v());
        if (!(a < kWideHi)) { /* NaN and infinities too */
            wide = true;
            const double d = fabs(e.v64());
            if (!(d <= top)) top = top != top ? top : d;
        } else if (a >= top32 * (1.0f - 1e-5f)) {
            /* may be the largest: 64 bits decide (|error of v()| < 1e-6) */
            if (a >= kWideLo || (top32 < 1e-25f && !e.zero())) {
                const double d = fabs(e.v64());
                if (d > top) top = d;
            }
            top32 = fmaxf(top32, a);
        } else if (a < kWideLo && top32 < 1e-25f && !e.zero()) {
            const double d = fabs(e.v64());
            if (d > top) top = d;
        }
    }
};

__device__ __forceinline__ double max_or_nan(double a, double b) { return a != a || a > b ? a : b; }

/* The row's statistics, in every thread. */
__device__ __forceinline__ void block_stat(RowStat &s) {
    __shared__ double sums[kRowThreads / 32], tops[kRowThreads / 32];
    __shared__ int wides[kRowThreads / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s.sum += __shfl_xor_sync(0xffffffffu, s.sum, o);
        s.top = max_or_nan(s.top, __shfl_xor_sync(0xffffffffu, s.top, o));
    }
    const bool wide = __any_sync(0xffffffffu, s.wide);
    if ((threadIdx.x & 31) == 0) {
        sums[threadIdx.x >> 5] = s.sum;
        tops[threadIdx.x >> 5] = s.top;
        wides[threadIdx.x >> 5] = wide;
    }
    __syncthreads();
    s.sum = 0.0;
    s.top = 0.0;
    s.wide = false;
#pragma unroll
    for (int i = 0; i < kRowThreads / 32; ++i) {
        s.sum += sums[i];
        s.top = max_or_nan(s.top, tops[i]);
        s.wide |= wides[i] != 0;
    }
    if (s.top < (double)kWideLo) s.wide = true;
}

/* A row's quantizer, once its statistics are known. */
struct RowQuant {
    double top;
    float r32;     /* 127 / top */
    float scale;
    bool wide, empty; /* empty: every q is 0 */

    /* factor: what v is still to be multiplied by (the norm's) */
    __device__ RowQuant(const RowStat &s, double factor) : top(s.top), wide(s.wide) {
        const double size = s.top == 0.0 ? 0.0 : s.top * factor; /* no eps: 0, not 0 * infinity */
        const bool fine = size <= (double)kFltMax; /* false for NaN */
        empty = !fine || s.top == 0.0;
        scale = fine ? (float)(size / 127.0) : __int_as_float(0x7fc00000);
        r32 = empty ? 0.0f : (float)(127.0 / s.top);
    }
    template <typename E> __device__ int q(const E &e, float border) const {
        if (empty) return 0;
        if (!wide) {
            const float t = __fmul_rn(e.v(), r32);
            const float n = rintf(t);
            if (fabsf(t - n) < 0.5f - border) return (int)n;
        }
        return (int)rint(127.0 * e.v64() / top);
    }
};

struct RowParams {
    const void *a, *b; /* x and the residual, or gate and up */
    void *h;
    const float *w;
    long long a_stride, b_stride, h_stride, q_stride;
    int n;
    float eps;
    int8_t *q;
    float *scale;
};

template <typename Row> __device__ __forceinline__ void row_q8(const Row &row, const RowParams &p) {
    RowStat s;
    for (int i = threadIdx.x; i < p.n; i += kRowThreads) {
        const auto e = row.first(i);
        if constexpr (Row::kNorm) s.sum += (double)e.h * (double)e.h;
        s.take(e);
    }
    block_stat(s);
    const RowQuant rq(s, Row::kNorm ? 1.0 / sqrt(s.sum / p.n + (double)p.eps) : 1.0);
    int8_t *q = p.q + (size_t)blockIdx.x * p.q_stride;
    for (int i = threadIdx.x; i < p.n; i += kRowThreads) q[i] = (int8_t)rq.q(row.again(i), Row::kBorder);
    if (threadIdx.x == 0) p.scale[blockIdx.x] = rq.scale;
}

/* One CTA a row, two visits to each element. */
template <typename T>
__global__ void __launch_bounds__(kRowThreads) norm_q8_kernel(const RowParams p) {
    const size_t i = blockIdx.x;
    const NormRow<T> row = {(const T *)p.a + i * p.a_stride,
                            p.b != nullptr ? (const T *)p.b + i * p.b_stride : nullptr,
                            p.h != nullptr ? (T *)p.h + i * p.h_stride : nullptr, p.w};
    row_q8(row, p);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) swiglu_q8_kernel(const RowParams p) {
    const size_t i = blockIdx.x;
    const SwigluRow<T> row = {(const T *)p.a + i * p.a_stride, (const T *)p.b + i * p.b_stride};
    row_q8(row, p);
}

template <typename T> cudaError_t launch_norm(const RowParams &p, int rows, cudaStream_t st) {
    norm_q8_kernel<T><<<rows, kRowThreads, 0, st>>>(p);
    return cudaGetLastError();
}
template <typename T> cudaError_t launch_swiglu(const RowParams &p, int rows, cudaStream_t st) {
    swiglu_q8_kernel<T><<<rows, kRowThreads, 0, st>>>(p);
    return cudaGetLastError();
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
    if (rows < 0 || n_embd < 1)
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
                         n_embd, eps, d_q, d_scale};
    cudaStream_t st = (cudaStream_t)stream;
    return launched(op, dtype == LAL_TAIL_F32    ? launch_norm<float>(p, rows, st)
                        : dtype == LAL_TAIL_BF16 ? launch_norm<__nv_bfloat16>(p, rows, st)
                                                 : launch_norm<__half>(p, rows, st));
}

int lal_tail_swiglu_q8(const void *d_gate, int64_t gate_stride, const void *d_up, int64_t up_stride,
                       int dtype, int rows, int n, int8_t *d_q, int64_t q_stride, float *d_scale,
                       void *stream) {
    static const char *op = "swiglu_q8";
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (rows < 0 || n < 1) return layer_fail(LAL_TAIL_ERR_ARG, "%s: %d rows of %d", op, rows, n);
    if (rows == 0) return LAL_TAIL_OK;
    if (!d_gate || !d_up || !d_q || !d_scale)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (gate_stride < n || up_stride < n || q_stride < n)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below n %d", op, n);
    if (((uintptr_t)d_gate | (uintptr_t)d_up) % size != 0 || (uintptr_t)d_scale % 4 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    const Span g(d_gate, rows, n, gate_stride, size), u(d_up, rows, n, up_stride, size),
        q(d_q, rows, n, q_stride, 1), s(d_scale, 1, rows, rows, 4);
    if (q.meets(g) || q.meets(u) || q.meets(s) || s.meets(g) || s.meets(u))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_gate", "d_up", "d_q", "d_scale"};
    const void *ptrs[] = {d_gate, d_up, d_q, d_scale};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const RowParams p = {d_gate, d_up, nullptr, nullptr, gate_stride, up_stride, 0, q_stride,
                         n, 0.0f, d_q, d_scale};
    cudaStream_t st = (cudaStream_t)stream;
    return launched(op, dtype == LAL_TAIL_F32    ? launch_swiglu<float>(p, rows, st)
                        : dtype == LAL_TAIL_BF16 ? launch_swiglu<__nv_bfloat16>(p, rows, st)
                                                 : launch_swiglu<__half>(p, rows, st));
}

}  // extern "C"
