/*
 * tail_q4.cu -- weights in 4 bits with a scale (and, on demand, a minimum) per
 * group of columns: the quantizer, the read-back and the product with 8-bit
 * vectors.
 *
 * Layout.  A row is ceil(cols / 32) blocks of 16 bytes; byte j of a block
 * holds column j in its low half and column j + 16 in its high half, so a
 * 32-bit word, masked, is four consecutive columns, and shifted by 4 and
 * masked the four that lie 16 further: both are operands of a 4-way int8 dot
 * product as they are.  Scales (and minima) are f16, [rows][ceil(cols / group)].
 *
 *   symmetric     w = s * (q - 8)
 *   with minimum  w = s * q + m
 */
#include "tail_layer.h"

using namespace lal;

namespace {

constexpr int kQ4Block = 32; /* columns of a 16-byte block */

__host__ __device__ inline int q4_blocks(int cols) { return (cols + kQ4Block - 1) / kQ4Block; }

/* ---------------------------------------------------------- quantizer --- */

/* v >= 0 in f16, rounded up: with a scale that is not below max|w| / 7 no
 * weight is clamped.  Infinite when v is above f16's range. */
__device__ __forceinline__ __half half_up(double v) {
    const __half h = __double2half(v);
    return (double)__half2float(h) < v ? __ushort_as_half(__half_as_ushort(h) + 1) : h;
}
/* v >= 0 in f16, rounded down */
__device__ __forceinline__ __half half_down(double v) {
    const __half h = __double2half(v);
    return (double)__half2float(h) > v ? __ushort_as_half(__half_as_ushort(h) - 1) : h;
}

/* rint((w - m) / s) of the quotient in 64 bits: 32 bits where they cannot be
 * on the wrong side of a border (the quotient is below 16, its error below
 * 16 * 2 * 2^-24 < 2e-6) */
__device__ __forceinline__ int q4_round(float w, float m, float s) {
    const float t = __fdiv_rn(__fsub_rn(w, m), s);
    const float n = rintf(t);
    if (fabsf(t - n) < 0.5f - 4e-6f) return (int)n;
    return (int)rint(((double)w - (double)m) / (double)s);
}

struct QuantParams {
    const void *w;
    long long w_stride;
    int rows, cols, group;
    uint8_t *q;
    __half *scale, *min;
};

/* A warp takes a group: lane j the columns j, j + 32, ... */
template <typename T, bool kMin>
__global__ void __launch_bounds__(256) quantize_q4_kernel(const QuantParams p) {
    const int lane = threadIdx.x & 31;
    const int groups = (p.cols + p.group - 1) / p.group;
    const long long at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= (long long)p.rows * groups) return;
    const int row = (int)(at / groups), g = (int)(at - (long long)row * groups);
    const T *w = (const T *)p.w + (size_t)row * p.w_stride;
    const int c0 = g * p.group, c1 = min(p.cols, c0 + p.group);
    float hi = -INFINITY, lo = INFINITY;
    bool bad = false;
    for (int c = c0 + lane; c < c1; c += 32) {
        const float v = to_f32(w[c]);
        bad |= !(fabsf(v) <= 3.4028234663852886e38f);
        hi = fmaxf(hi, v);
        lo = fminf(lo, v);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    bad = __any_sync(0xffffffffu, bad);
    __half s, m = __float2half_rn(0.0f);
    if (kMin) {
        m = lo < 0.0f ? __hneg(half_up(-(double)lo)) : half_down((double)lo);
        s = half_up(((double)hi - (double)__half2float(m)) / 15.0);
        bad |= __hisinf(m) != 0;
    } else {
        s = half_up((double)fmaxf(hi, -lo) / 7.0);
    }
    bad |= __hisinf(s) != 0;
    const float sf = __half2float(s), mf = __half2float(m);
    for (int c = c0 + lane; c < c0 + p.group && c / kQ4Block < q4_blocks(p.cols); c += 32) {
        int q = kMin ? 0 : 8;
        if (c < c1 && !bad && sf > 0.0f) {
            const int n = q4_round(to_f32(w[c]), kMin ? mf : 0.0f, sf);
            q = kMin ? max(0, min(15, n)) : max(-7, min(7, n)) + 8;
        }
        const int up = __shfl_down_sync(0xffffffffu, q, 16);
        if (lane < 16)
            p.q[(size_t)row * q4_blocks(p.cols) * 16 + c / kQ4Block * 16 + lane] = (uint8_t)(q | up << 4);
    }
    if (lane == 0) {
        const __half nan = __ushort_as_half(0x7e00);
        p.scale[(size_t)row * groups + g] = bad ? nan : s;
        if (kMin) p.min[(size_t)row * groups + g] = bad ? nan : m;
    }
}

/* ---------------------------------------------------------- read-back --- */
struct BackParams {
    const uint8_t *q;
    const __half *scale, *min;
    int rows, cols, group;
    void *w;
    long long w_stride;
};

/* A thread takes four consecutive columns. */
template <typename T, bool kMin>
__global__ void __launch_bounds__(256) dequantize_q4_kernel(const BackParams p) {
    const int quads = (p.cols + 3) / 4;
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    if (at >= (long long)p.rows * quads) return;
    const int row = (int)(at / quads), c = (int)(at - (long long)row * quads) * 4;
    const int groups = (p.cols + p.group - 1) / p.group;
    const size_t block = (size_t)row * q4_blocks(p.cols) + c / kQ4Block;
    const uint32_t word = __ldg((const uint32_t *)(p.q + block * 16) + (c % 16) / 4);
    const uint32_t four = (c % kQ4Block >= 16 ? word >> 4 : word) & 0x0f0f0f0fu;
    const float s = __half2float(p.scale[(size_t)row * groups + c / p.group]);
    const float m = kMin ? __half2float(p.min[(size_t)row * groups + c / p.group]) : 0.0f;
    T *w = (T *)p.w + (size_t)row * p.w_stride + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float q = (float)((four >> (8 * j)) & 15u);
        /* s * q is exact in 32 bits (11 and 4 bits): one rounding */
        const float v = kMin ? fmaf(s, q, m) : __fmul_rn(s, q - 8.0f);
        if (c + j < p.cols) w[j] = from_f32<T>(v);
    }
}

/* ------------------------------------------------------------ product --- */
struct MatvecParams {
    const int8_t *x;
    long long x_stride;
    const float *sx;
    const uint8_t *q;
    const __half *scale, *min;
    int streams, rows, cols, group;
    void *y;
    long long y_stride;
};

/* four consecutive columns of a vector, zeros behind its end */
__device__ __forceinline__ int x_word(const int8_t *x, int c, int cols) {
    uint32_t v = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (c + j < cols) v |= (uint32_t)(uint8_t)x[c + j] << (8 * j);
    return (int)v;
}

/* A warp takes a row and up to kB streams; a lane takes every 32nd block of
 * the row.  The dots of a block are exact integers; their scaled sum is in
 * 32-bit floats. */
template <typename T, int kB, bool kMin>
__global__ void __launch_bounds__(256) q4_matvec_kernel(const MatvecParams p) {
    const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= p.rows) return;
    const int b0 = blockIdx.y * kB;
    const int blocks = q4_blocks(p.cols), groups = (p.cols + p.group - 1) / p.group;
    const uint4 *q = (const uint4 *)p.q + (size_t)row * blocks;
    float acc[kB] = {};
    for (int k = lane; k < blocks; k += 32) {
        const uint4 v = __ldg(q + k);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        const size_t g = (size_t)row * groups + k * kQ4Block / p.group;
        const float s = __half2float(p.scale[g]);
        const float m = kMin ? __half2float(p.min[g]) : __fmul_rn(s, -8.0f);
#pragma unroll
        for (int b = 0; b < kB; ++b) {
            if (b0 + b >= p.streams) break;
            const int8_t *x = p.x + (size_t)(b0 + b) * p.x_stride;
            int dot = 0, sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lo = x_word(x, k * kQ4Block + 4 * i, p.cols);
                const int hi = x_word(x, k * kQ4Block + 16 + 4 * i, p.cols);
                dot = __dp4a((int)(w[i] & 0x0f0f0f0fu), lo, dot);
                dot = __dp4a((int)((w[i] >> 4) & 0x0f0f0f0fu), hi, dot);
                sum = __dp4a(0x01010101, lo, __dp4a(0x01010101, hi, sum));
            }
            if (kMin)
                acc[b] = fmaf(m, (float)sum, fmaf(s, (float)dot, acc[b]));
            else
                acc[b] = fmaf(s, (float)(dot - 8 * sum), acc[b]);
        }
    }
#pragma unroll
    for (int b = 0; b < kB; ++b) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) acc[b] += __shfl_xor_sync(0xffffffffu, acc[b], o);
        if (lane == 0 && b0 + b < p.streams)
            ((T *)p.y)[(size_t)(b0 + b) * p.y_stride + row] =
                from_f32<T>(__fmul_rn(p.sx[b0 + b], acc[b]));
    }
}

template <typename T, bool kMin> cudaError_t launch_matvec(const MatvecParams &p, cudaStream_t st) {
    const unsigned gx = (unsigned)((p.rows + 7) / 8);
    if (p.streams == 1)
        q4_matvec_kernel<T, 1, kMin><<<dim3(gx, 1), 256, 0, st>>>(p);
    else
        q4_matvec_kernel<T, 8, kMin><<<dim3(gx, (p.streams + 7) / 8), 256, 0, st>>>(p);
    return cudaGetLastError();
}

/* calls f with the type of `dtype` and the truth of `min` as constants */
template <typename F> cudaError_t by_type(int dtype, bool min, F f) {
    if (dtype == LAL_TAIL_F32)
        return min ? f(float{}, std::true_type{}) : f(float{}, std::false_type{});
    if (dtype == LAL_TAIL_BF16)
        return min ? f(__nv_bfloat16{}, std::true_type{}) : f(__nv_bfloat16{}, std::false_type{});
    return min ? f(__half{}, std::true_type{}) : f(__half{}, std::false_type{});
}

int check_weights(const char *op, const lal_tail_q4 *w) {
    if (!w) return layer_fail(LAL_TAIL_ERR_ARG, "%s: null weights", op);
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: groups of %d columns (32, 64 or 128)", op, w->group);
    if (w->rows < 0 || w->cols < 1)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: weights of %d x %d", op, w->rows, w->cols);
    if (w->rows > 0 && (!w->d_q || !w->d_scale))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer in the weights", op);
    if ((uintptr_t)w->d_q % 16 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: d_q is not aligned to 16 bytes", op);
    if (((uintptr_t)w->d_scale | (uintptr_t)w->d_min) % 2 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: scales are not aligned to 2 bytes", op);
    return LAL_TAIL_OK;
}

struct WeightSpans {
    Span q, s, m;
    explicit WeightSpans(const lal_tail_q4 *w) {
        const long long groups = (w->cols + w->group - 1LL) / w->group, bytes = 16LL * q4_blocks(w->cols);
        q = Span(w->d_q, w->rows, bytes, bytes, 1);
        s = Span(w->d_scale, w->rows, groups, groups, 2);
        m = Span(w->d_min, w->rows, groups, groups, 2);
    }
    bool meets(const Span &o) const { return q.meets(o) || s.meets(o) || m.meets(o); }
    bool meet_each_other() const { return q.meets(s) || q.meets(m) || s.meets(m); }
};

}  // namespace

extern "C" {

int lal_tail_quantize_q4(const lal_tail_q4 *w, const void *d_w, int64_t w_stride, int dtype, void *stream) {
    static const char *op = "quantize_q4";
    if (const int rc = check_weights(op, w)) return rc;
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (w->rows == 0) return LAL_TAIL_OK;
    if (!d_w) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (w_stride < w->cols) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below cols %d", op, w->cols);
    if ((uintptr_t)d_w % size != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    const WeightSpans spans(w);
    if (spans.meets(Span(d_w, w->rows, w->cols, w_stride, size)) || spans.meet_each_other())
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_w", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_w, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const QuantParams p = {d_w, w_stride, w->rows, w->cols, w->group, w->d_q, (__half *)w->d_scale,
                           (__half *)w->d_min};
    const long long warps = (long long)w->rows * ((w->cols + w->group - 1LL) / w->group);
    if ((warps + 7) / 8 > 0x7fffffffLL)
        return layer_fail(LAL_TAIL_ERR_UNSUPPORTED, "%s: weights of %d x %d", op, w->rows, w->cols);
    return launched(op, by_type(dtype, w->d_min != nullptr, [&](auto t, auto min) {
        quantize_q4_kernel<decltype(t), decltype(min)::value>
            <<<(unsigned)((warps + 7) / 8), 256, 0, (cudaStream_t)stream>>>(p);
        return cudaGetLastError();
    }));
}

int lal_tail_dequantize_q4(const lal_tail_q4 *w, void *d_w, int64_t w_stride, int dtype, void *stream) {
    static const char *op = "dequantize_q4";
    if (const int rc = check_weights(op, w)) return rc;
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (w->rows == 0) return LAL_TAIL_OK;
    if (!d_w) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (w_stride < w->cols) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below cols %d", op, w->cols);
    if ((uintptr_t)d_w % size != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    if (WeightSpans(w).meets(Span(d_w, w->rows, w->cols, w_stride, size)))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_w", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_w, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const BackParams p = {w->d_q, (const __half *)w->d_scale, (const __half *)w->d_min, w->rows, w->cols,
                          w->group, d_w, w_stride};
    const long long threads = (long long)w->rows * ((w->cols + 3LL) / 4);
    if ((threads + 255) / 256 > 0x7fffffffLL)
        return layer_fail(LAL_TAIL_ERR_UNSUPPORTED, "%s: weights of %d x %d", op, w->rows, w->cols);
    return launched(op, by_type(dtype, w->d_min != nullptr, [&](auto t, auto min) {
        dequantize_q4_kernel<decltype(t), decltype(min)::value>
            <<<(unsigned)((threads + 255) / 256), 256, 0, (cudaStream_t)stream>>>(p);
        return cudaGetLastError();
    }));
}

int lal_tail_q4_matvec(const lal_tail_q4 *w, const int8_t *d_xq, int64_t xq_stride, const float *d_scale_x,
                       int n_streams, void *d_y, int64_t y_stride, int dtype, void *stream) {
    static const char *op = "q4_matvec";
    if (const int rc = check_weights(op, w)) return rc;
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (n_streams < 0 || n_streams > LAL_TAIL_Q4_MAX_STREAMS)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: %d streams (at most %d)", op, n_streams,
                          LAL_TAIL_Q4_MAX_STREAMS);
    if (w->rows == 0 || n_streams == 0) return LAL_TAIL_OK;
    if (!d_xq || !d_scale_x || !d_y) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (xq_stride < w->cols || y_stride < w->rows)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below the weights' %d x %d", op, w->rows, w->cols);
    if ((uintptr_t)d_y % size != 0 || (uintptr_t)d_scale_x % 4 != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    const Span y(d_y, n_streams, w->rows, y_stride, size);
    if (y.meets(Span(d_xq, n_streams, w->cols, xq_stride, 1)) ||
        y.meets(Span(d_scale_x, 1, n_streams, n_streams, 4)) || WeightSpans(w).meets(y))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_xq", "d_scale_x", "d_y", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_xq, d_scale_x, d_y, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 6)) return rc;
    const MatvecParams p = {d_xq, xq_stride, d_scale_x, w->d_q, (const __half *)w->d_scale,
                            (const __half *)w->d_min, n_streams, w->rows, w->cols, w->group, d_y, y_stride};
    return launched(op, by_type(dtype, w->d_min != nullptr, [&](auto t, auto min) {
        return launch_matvec<decltype(t), decltype(min)::value>(p, (cudaStream_t)stream);
    }));
}

}  // extern "C"
