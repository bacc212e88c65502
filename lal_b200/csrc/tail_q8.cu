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

#include <cmath>
#include <cstring>

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
};

/* What few elements need, out of line: inlined for each of a thread's elements
 * it would fill the instruction cache. */
__device__ __noinline__ double silu64(double g, double u) { return g / (1.0 + exp(-g)) * u; }
__device__ __noinline__ int round64(double v, double top) { return (int)rint(127.0 * v / top); }

constexpr float kFltMax = 3.4028234663852886e38f;
/* max|v| in 32 bits at or above kWideHi or (not zero) below kWideLo: the row
 * is computed in 64 bits, clear of overflow and of denormal rounding */
constexpr float kWideHi = 1e37f, kWideLo = 1e-30f;

/* Eight elements of a row from p on, of which `n` exist, as wide as p's
 * alignment allows (rows of 16-bit elements may begin at any even address). */
template <typename T> __device__ __forceinline__ void get8(const T *p, int n, float (&v)[8]) {
    if (n < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
        return;
    }
    const unsigned at = (unsigned)(uintptr_t)p;
    union Raw {
        uint4 q[sizeof(T) / 2];
        uint32_t w[2 * sizeof(T)];
        T e[8];
        __device__ Raw() {}
    } raw;
    if ((at & 15) == 0) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw.q[i] = ((const uint4 *)p)[i];
    } else if (sizeof(T) == 4 || (at & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) raw.w[i] = ((const uint32_t *)p)[i];
    } else {
        raw.e[0] = p[0];
        const uint32_t *w = (const uint32_t *)(p + 1);
        const uint32_t m0 = w[0], m1 = w[1], m2 = w[2];
        const unsigned short last = ((const unsigned short *)p)[7];
        const uint32_t first = *(const unsigned short *)&raw.e[0];
        raw.w[0] = first | m0 << 16;
        raw.w[1] = __funnelshift_r(m0, m1, 16);
        raw.w[2] = __funnelshift_r(m1, m2, 16);
        raw.w[3] = m2 >> 16 | (uint32_t)last << 16;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f32(raw.e[i]);
}

template <typename T> __device__ __forceinline__ void put8(T *p, int n, const float (&v)[8]) {
    if (n < 8) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
        return;
    }
    const unsigned at = (unsigned)(uintptr_t)p;
    union Raw {
        uint4 q[sizeof(T) / 2];
        uint32_t w[2 * sizeof(T)];
        T e[8];
        __device__ Raw() {}
    } raw;
#pragma unroll
    for (int i = 0; i < 8; ++i) raw.e[i] = from_f32<T>(v[i]);
    if ((at & 15) == 0) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4 *)p)[i] = raw.q[i];
    } else if (sizeof(T) == 4 || (at & 3) == 0) {
#pragma unroll
        for (int i = 0; i < 2 * (int)sizeof(T); ++i) ((uint32_t *)p)[i] = raw.w[i];
    } else {
        p[0] = raw.e[0];
#pragma unroll
        for (int i = 0; i < 3; ++i) ((uint32_t *)(p + 1))[i] = __funnelshift_r(raw.w[i], raw.w[i + 1], 16);
        p[7] = raw.e[7];
    }
}

__device__ __forceinline__ void put8(int8_t *p, int n, const int (&q)[8]) {
    const unsigned at = (unsigned)(uintptr_t)p;
    if (n == 8 && (at & 3) == 0) {
        uint32_t w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            w[i] = (q[4 * i] & 255) | (q[4 * i + 1] & 255) << 8 | (q[4 * i + 2] & 255) << 16 | (uint32_t)q[4 * i + 3] << 24;
        if ((at & 7) == 0) {
            *(uint2 *)p = make_uint2(w[0], w[1]);
        } else {
            ((uint32_t *)p)[0] = w[0];
            ((uint32_t *)p)[1] = w[1];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = (int8_t)q[i];
}

/* What the two kinds of rows have of their own: v of eight elements in 32
 * bits, v of one in 64. */
template <typename T> struct NormRow {
    const T *x, *r;
    T *h;
    const float *w;
    int n;
    /* v: 2^-24; 127 / max|v|: 2 * 2^-24; their product: 2^-24; times 127: below 3.1e-5 */
    static constexpr float kBorder = 4e-5f;
    static constexpr bool kNorm = true;
    __device__ NormRow(const RowParams &p)
        : x((const T *)p.a + (size_t)blockIdx.x * p.a_stride),
          r(p.b != nullptr ? (const T *)p.b + (size_t)blockIdx.x * p.b_stride : nullptr),
          h(p.h != nullptr ? (T *)p.h + (size_t)blockIdx.x * p.h_stride : nullptr), w(p.w), n(p.n) {}
    /* adds the residual, stores the sum, adds its squares to `sum` */
    __device__ void load(int i, float (&v)[8], double &sum) const {
        const int m = min(8, n - i);
        get8(x + i, m, v);
        float u[8];
        if (r != nullptr) {
            get8(r + i, m, u);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(from_f32<T>(__fadd_rn(v[j], u[j])));
        }
        if (h != nullptr) put8(h + i, m, v);
        get8(w + i, m, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum = fma((double)v[j], (double)v[j], sum);
            v[j] = __fmul_rn(v[j], u[j]);
        }
    }
    /* the same v again, by the thread that loaded it */
    __device__ void again(int i, float (&v)[8]) const {
        const int m = min(8, n - i);
        float u[8];
        get8(h != nullptr ? (const T *)h + i : x + i, m, v);
        get8(w + i, m, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], u[j]);
    }
    __device__ double v64(int i) const { return (double)to_f32(h != nullptr ? h[i] : x[i]) * (double)w[i]; }
};

template <typename T> struct SwigluRow {
    const T *g, *u;
    int n;
    /* expf 2 ulp, 1 + e 0.5, __fdividef 2, the product 0.5 (5 * 2^-23), 127 / max|v| and the
     * product with it 3 * 2^-24; times 127: below 1e-4 */
    static constexpr float kBorder = 1.2e-4f;
    static constexpr bool kNorm = false;
    __device__ SwigluRow(const RowParams &p)
        : g((const T *)p.a + (size_t)blockIdx.x * p.a_stride), u((const T *)p.b + (size_t)blockIdx.x * p.b_stride),
          n(p.n) {}
    __device__ void load(int i, float (&v)[8], double &) const {
        const int m = min(8, n - i);
        float up[8];
        get8(g + i, m, v);
        get8(u + i, m, up);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gate = v[j];
            v[j] = __fmul_rn(__fdividef(gate, 1.0f + expf(-gate)), up[j]);
            /* there 1 + exp(-gate) leaves what __fdividef takes */
            if (gate < -80.0f) v[j] = (float)silu64((double)gate, (double)up[j]);
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

/* A row's statistics across the CTA. */
struct RowShared {
    double sums[32], sum;
    unsigned tops[32];
    unsigned long long top;
};

/* The largest |v| in 32 bits (as its bits) in every thread; the sum of `sum`
 * in sh.sum after the next barrier. */
template <bool kNorm> __device__ __forceinline__ unsigned row_top32(RowShared &sh, double sum, unsigned m) {
    const int warps = blockDim.x >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    m = __reduce_max_sync(0xffffffffu, m);
    if (kNorm)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
        sh.tops[warp] = m;
        sh.sums[warp] = sum;
    }
    if (threadIdx.x == 0) sh.top = 0;
    __syncthreads();
    if (kNorm && warp == 0) {
        sum = lane < warps ? sh.sums[lane] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) sh.sum = sum;
    }
    return __reduce_max_sync(0xffffffffu, lane < warps ? sh.tops[lane] : 0u);
}

/* Who may have the largest |v|: 64 bits decide (|error of v| < 1e-6). */
__device__ __forceinline__ bool row_wide(float top32) { return !(top32 < kWideHi && top32 >= kWideLo); }
__device__ __forceinline__ float row_least(float top32) { return row_wide(top32) ? 0.0f : top32 * (1.0f - 4e-6f); }

/* A row's quantizer, once max|v| and the sum of squares are known. */
template <typename Row> struct RowQuant {
    double top;
    float r32; /* 127 / top */
    bool wide, fits; /* fits: fp32 holds the scale; else the row is NaN */

    __device__ double factor(const RowParams &p, double sum) const {
        return Row::kNorm ? 1.0 / sqrt(sum / p.n + (double)p.eps) : 1.0;
    }
    __device__ RowQuant(const RowParams &p, const RowShared &sh, bool wide_)
        : top(of_bits(sh.top)), wide(wide_) {
        r32 = __fdiv_rn(127.0f, (float)top);
        float about = (float)top;
        if (Row::kNorm) about *= rsqrtf((float)(sh.sum * (1.0 / p.n)) + p.eps);
        fits = about < 1e38f || top == 0.0 || top * factor(p, sh.sum) <= (double)kFltMax;
    }
    __device__ void store(const RowParams &p, const Row &row, int i, const float (&v)[8]) const {
        int out[8];
        unsigned near = 0; /* elements next to a border */
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float t = __fmul_rn(v[j], r32), n = rintf(t);
            if (!(fabsf(t - n) < 0.5f - Row::kBorder)) near |= 1u << j;
            out[j] = (int)n;
        }
        if (wide) near = 255;
        if (!fits || top == 0.0) {
            near = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) out[j] = 0;
        }
        int8_t *q = p.q + (size_t)blockIdx.x * p.q_stride + i;
        put8(q, min(8, p.n - i), out);
        for (; near != 0; near &= near - 1) {
            const int j = __ffs(near) - 1;
            if (i + j < p.n) q[j] = (int8_t)round64(row.v64(i + j), top);
        }
    }
    __device__ float scale(const RowParams &p, double sum) const {
        return !fits ? __int_as_float(0x7fc00000) : top == 0.0 ? 0.0f : (float)(top * factor(p, sum) / 127.0);
    }
};

/* One CTA a row, 8 kC elements a thread, which stay in registers between the
 * statistics and the quantizer. */
template <typename Row, int kC, int kMaxThreads>
__global__ void __launch_bounds__(kMaxThreads) row_q8_kernel(const RowParams p) {
    __shared__ RowShared sh;
    const Row row(p);
    float v[kC][8];
    double sum = 0.0;
    unsigned m = 0;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        const int i = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
        if (i < p.n) row.load(i, v[c], sum);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(fabsf(v[c][j])));
    }
    const float top32 = __uint_as_float(row_top32<Row::kNorm>(sh, sum, m)), least = row_least(top32);
    if (!(__uint_as_float(m) < least)) {
        unsigned long long best = 0;
#pragma unroll
        for (int c = 0; c < kC; ++c) {
            const int i = (c * blockDim.x + threadIdx.x) * 8;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < p.n && !(fabsf(v[c][j]) < least)) best = max(best, abs_bits(row.v64(i + j)));
        }
        if (best) atomicMax(&sh.top, best);
    }
    __syncthreads();
    const RowQuant<Row> rq(p, sh, row_wide(top32));
#pragma unroll
    for (int c = 0; c < kC; ++c) {
        const int i = (c * blockDim.x + threadIdx.x) * 8;
        if (i < p.n) rq.store(p, row, i, v[c]);
    }
    if (threadIdx.x == 0) p.scale[blockIdx.x] = rq.scale(p, sh.sum);
}

/* Rows longer than a CTA's registers hold: every element is visited again. */
constexpr int kLongThreads = 512;
template <typename Row> __global__ void __launch_bounds__(kLongThreads) row_q8_long_kernel(const RowParams p) {
    __shared__ RowShared sh;
    const Row row(p);
    double sum = 0.0;
    unsigned m = 0;
    float v[8];
    for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
        row.load(i, v, sum);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j < p.n) m = max(m, __float_as_uint(fabsf(v[j])));
    }
    const float top32 = __uint_as_float(row_top32<Row::kNorm>(sh, sum, m)), least = row_least(top32);
    if (!(__uint_as_float(m) < least)) {
        unsigned long long best = 0;
        for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
            row.again(i, v);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j < p.n && !(fabsf(v[j]) < least)) best = max(best, abs_bits(row.v64(i + j)));
        }
        if (best) atomicMax(&sh.top, best);
    }
    __syncthreads();
    const RowQuant<Row> rq(p, sh, row_wide(top32));
    for (int i = threadIdx.x * 8; i < p.n; i += kLongThreads * 8) {
        row.again(i, v);
        rq.store(p, row, i, v);
    }
    if (threadIdx.x == 0) p.scale[blockIdx.x] = rq.scale(p, sh.sum);
}

template <typename Row> cudaError_t launch_rows(const RowParams &p, int rows, cudaStream_t st) {
    const int eights = (p.n + 7) / 8;
    auto threads = [&](int c) { return ((eights + c - 1) / c + 31) / 32 * 32; };
    if (eights <= 1024)
        row_q8_kernel<Row, 1, 1024><<<rows, threads(1), 0, st>>>(p);
    else if (eights <= 2048)
        row_q8_kernel<Row, 2, 1024><<<rows, threads(2), 0, st>>>(p);
    else if (eights <= 4 * 640)
        row_q8_kernel<Row, 4, 640><<<rows, threads(4), 0, st>>>(p);
    else
        row_q8_long_kernel<Row><<<rows, kLongThreads, 0, st>>>(p);
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
    return launched(op, dtype == LAL_TAIL_F32    ? launch_rows<NormRow<float>>(p, rows, st)
                        : dtype == LAL_TAIL_BF16 ? launch_rows<NormRow<__nv_bfloat16>>(p, rows, st)
                                                 : launch_rows<NormRow<__half>>(p, rows, st));
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
    return launched(op, dtype == LAL_TAIL_F32    ? launch_rows<SwigluRow<float>>(p, rows, st)
                        : dtype == LAL_TAIL_BF16 ? launch_rows<SwigluRow<__nv_bfloat16>>(p, rows, st)
                                                 : launch_rows<SwigluRow<__half>>(p, rows, st));
}

}  // extern "C"
