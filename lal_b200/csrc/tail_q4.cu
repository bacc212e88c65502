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
#include "tail_device.cuh"
#include "tail_layer.h"

#include <algorithm>
#include <type_traits>

namespace lal {
namespace {

constexpr int kQ4Block = 32; /* columns of a 16-byte block */

__host__ __device__ inline int q4_blocks(int cols) { return (cols + kQ4Block - 1) / kQ4Block; }

/* ---------------------------------------------------------- quantizer --- */

/* rint((w - m) / s) exactly, ties to even, from n that is off by one at most:
 * w - m as the sum of two fp32 numbers, less n s (11 and 4 bits: exact), against
 * half a step.  Near half a step the difference has no more than 24 bits. */
__device__ __forceinline__ float q4_exact(float w, float m, float s, float n) {
    const float d = __fsub_rn(w, m), bb = __fsub_rn(d, w);
    const float low = __fadd_rn(__fsub_rn(w, __fsub_rn(d, bb)), -__fadd_rn(m, bb));
    const float e = fmaf(-n, s, d), half = __fmul_rn(0.5f, s);
    const float over = __fadd_rn(__fsub_rn(e, half), low), under = __fadd_rn(__fadd_rn(e, half), low);
    const bool odd = (__float2int_rn(n) & 1) != 0;
    if (over > 0.0f || (over == 0.0f && odd)) n += 1.0f;
    if (under < 0.0f || (under == 0.0f && odd)) n -= 1.0f;
    return n;
}

/* The smallest f16 s with k s >= x: rounded up, so no weight is clamped.  k s is
 * an fp32 number (11 and 4 bits), so it compares exactly; the nearest f16 to
 * x / k is s or one step below.  Infinite above f16's range. */
__device__ __forceinline__ __half f16_step_up(float x, float k, float k_inv) {
    const __half h = __float2half_rn(__fmul_rn(x, k_inv));
    return __fmul_rn(k, __half2float(h)) < x ? __ushort_as_half((unsigned short)(__half_as_ushort(h) + 1)) : h;
}
/* the largest f16 not above x */
__device__ __forceinline__ __half f16_floor(float x) {
    const __half h = __float2half_rn(x);
    const unsigned short b = __half_as_ushort(h);
    return __half2float(h) > x ? __ushort_as_half((unsigned short)(b & 0x8000 ? b + 1 : b - 1)) : h;
}

/* Four elements from p on, of which n (may be below 0) exist. */
template <typename T> __device__ __forceinline__ void get4(const T *p, int n, bool aligned, float (&v)[4]) {
    if (n >= 4 && aligned) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = *(const float4 *)p;
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
            const uint2 w = *(const uint2 *)p;
            unpack16<T>(w.x, v[0], v[1]);
            unpack16<T>(w.y, v[2], v[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}
/* to p, aligned to four elements */
template <typename T> __device__ __forceinline__ void put4(T *p, int n, const float (&v)[4]) {
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) {
            *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            union Raw {
                uint2 w;
                T e[4];
                __device__ Raw() {}
            } raw;
#pragma unroll
            for (int i = 0; i < 4; ++i) raw.e[i] = from_f32<T>(v[i]);
            *(uint2 *)p = raw.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < n) p[i] = from_f32<T>(v[i]);
    }
}

/* Four elements as they lie in memory. */
template <typename T> union Four {
    uint32_t w[sizeof(T)];
    T e[4];
    __device__ Four() {}
};

/* Both directions: four lanes a block, a warp takes kRun runs of 256 columns of
 * a row, all their loads at once.  Bounded by HBM: 18944x3584 fp32 to 4 bits 53
 * us (0.88 of the measured rate; with minima and groups of 32 69), back 47.3
 * (0.99); bf16 60 us (108), bounded by instructions, and 32.  Of fp32, lane u of
 * a block has columns 4u .. 4u + 3 and 16 + 4u .., which are the word u; of 16-bit
 * numbers eight columns in a row, 16 bytes, and half a word's worth goes over to
 * another lane. */
constexpr int kRun = 4;
constexpr int kQ4Warps = 8;
struct ConvertParams {
    uint8_t *q;
    __half *scale, *min;
    int rows, cols, group;
    void *w;
    long long w_stride;
    int aligned; /* rows of w are aligned to 16 bytes */
};
/* warps: kRun * 256 columns of a row each */
__host__ __device__ inline int q4_row_warps(int cols) { return (cols + kRun * 256 - 1) / (kRun * 256); }
inline long long q4_ctas(int rows, int cols) { return ((long long)rows * q4_row_warps(cols) + kQ4Warps - 1) / kQ4Warps; }

template <typename T, int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kQ4Warps) quantize_q4_kernel(const ConvertParams p) {
    after_previous();
    const int lane = threadIdx.x & 31, nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    constexpr bool kRow8 = sizeof(T) == 2;
    const int per_row = q4_row_warps(p.cols);
    const long long at = (long long)blockIdx.x * kQ4Warps + (threadIdx.x >> 5);
    const int row = (int)(at / per_row), c0 = (int)(at - (long long)row * per_row) * (kRun * 256);
    if (row >= p.rows) return;
    float v[kRun][8];
    const T *const w0 = (const T *)p.w + (size_t)row * p.w_stride + c0 + (lane >> 2) * 32 + (lane & 3) * (kRow8 ? 8 : 4);
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        if (c0 + u * 256 >= p.cols) break;
        const int c = c0 + u * 256 + (lane >> 2) * 32 + (lane & 3) * (kRow8 ? 8 : 4);
        const T *w = w0 + u * 256;
        float lo[4], hi[4];
        if constexpr (kRow8) {
            if (p.aligned && c + 8 <= p.cols) {
                const uint4 x = *(const uint4 *)w;
                unpack16<T>(x.x, lo[0], lo[1]);
                unpack16<T>(x.y, lo[2], lo[3]);
                unpack16<T>(x.z, hi[0], hi[1]);
                unpack16<T>(x.w, hi[2], hi[3]);
            } else {
                get4(w, p.cols - c, false, lo);
                get4(w + 4, p.cols - c - 4, false, hi);
            }
        } else {
            get4(w, p.cols - c, p.aligned, lo);
            get4(w + 16, p.cols - c - 16, p.aligned, hi);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = lo[i], v[u][4 + i] = hi[i];
    }
    uint32_t *const q0 = (uint32_t *)p.q + ((size_t)row * nb + c0 / kQ4Block + (lane >> 2)) * 4;
    const size_t s0 = (size_t)row * groups;
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        if (c0 + u * 256 >= p.cols) break;
        const int c = c0 + u * 256 + (lane >> 2) * 32; /* the block's first column */
        /* max|w|, NaN above all; what does not exist is 0 to it, and left out of the extremes */
        float top = 0.0f, hi = -INFINITY, lo = INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[u][i])));
        if (kMin) {
            if (c0 + u * 256 + 256 <= p.cols) {
#pragma unroll
                for (int i = 0; i < 8; ++i) hi = fmaxf(hi, v[u][i]), lo = fminf(lo, v[u][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c + (kRow8 ? (lane & 3) * 8 + i : (lane & 3) * 4 + (i < 4 ? i : 12 + i)) < p.cols) hi = fmaxf(hi, v[u][i]), lo = fminf(lo, v[u][i]);
            }
        }
        unsigned worst = __float_as_uint(top) & 0x7fffffffu;
#pragma unroll
        for (int o = kGroup / 16; o > 0; o >>= 1) { /* 4 lanes a block */
            worst = max(worst, __shfl_xor_sync(0xffffffffu, worst, o));
            if (kMin) {
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            }
        }
        __half s, m = __float2half_rn(0.0f);
        if (kMin) {
            m = f16_floor(lo);
            s = f16_step_up(__fsub_ru(hi, __half2float(m)), 15.0f, 1.0f / 15.0f);
        } else {
            s = f16_step_up(__uint_as_float(worst), 7.0f, 1.0f / 7.0f);
        }
        const bool bad = worst >= 0x7f800000u || __hisinf(s) != 0 || (kMin && __hisinf(m) != 0);
        const float sf = __half2float(s), mf = __half2float(m);
        uint32_t low = 0, high = 0;
        if (!bad && sf > 0.0f) {
            float r, far = 0.0f;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(sf));
            constexpr float kRound = 12582912.0f; /* 1.5 * 2^23: added, it leaves the nearest integer in the low bits */
            uint32_t n[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float t = __fmul_rn(kMin ? __fsub_rn(v[u][i], mf) : v[u][i], r);
                /* 11 bits by 11: the quotient is halfway between two steps, and then this is it, or 2^-12 away */
                if (kRow8 && !kMin) t = fmaf(fmaf(-t, sf, v[u][i]), r, t);
                const float x = __fadd_rn(t, kRound);
                if (!kRow8 || kMin) far = fmaxf(far, fabsf(__fsub_rn(t, __fsub_rn(x, kRound))));
                n[i] = __float_as_uint(x);
            }
            /* three roundings of a quotient below 16, 2^-22 of it together: below 4e-6 */
            if (!(far < 0.5f - 8e-6f))
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    n[i] = __float_as_uint(__fadd_rn(
                        q4_exact(v[u][i], mf, sf, __fsub_rn(__uint_as_float(n[i]), kRound)), kRound));
            low = __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
            high = __byte_perm(__byte_perm(n[4], n[5], 0x0040), __byte_perm(n[6], n[7], 0x0040), 0x5410);
        }
        int place = lane & 3;
        if (kRow8) {
            /* lanes 0 and 1 have columns 0-15, a word's low halves; 2 and 3 the high ones: lanes 0, 2, 1, 3 end with words 0, 1, 2, 3 */
            const bool first = place < 2;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, first ? high : low, 2);
            (first ? high : low) = got;
            place = (place & 1) * 2 + (place >> 1);
        }
        /* -7 .. 7, plus 8: the sign bit of four turned */
        const uint32_t word = ((low & 0x0f0f0f0fu) | ((high << 4) & 0xf0f0f0f0u)) ^ (kMin ? 0u : 0x88888888u);
        if (c / kQ4Block < nb) {
            q0[u * 32 + place] = word;
            if ((lane & 3) == 0 && c % kGroup == 0) {
                const __half nan = __ushort_as_half(0x7e00);
                p.scale[s0 + c / kGroup] = bad ? nan : s;
                if (kMin) p.min[s0 + c / kGroup] = bad ? nan : m;
            }
        }
    }
}

template <typename T, int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kQ4Warps) dequantize_q4_kernel(const ConvertParams p) {
    after_previous();
    const int lane = threadIdx.x & 31, nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int per_row = q4_row_warps(p.cols);
    const long long at = (long long)blockIdx.x * kQ4Warps + (threadIdx.x >> 5);
    const int row = (int)(at / per_row), c0 = (int)(at - (long long)row * per_row) * (kRun * 256);
    if (row >= p.rows) return;
    const uint32_t *const q0 = (const uint32_t *)p.q + ((size_t)row * nb + c0 / kQ4Block) * 4 + lane;
    const size_t s0 = (size_t)row * groups;
    __shared__ __align__(16) T lines[kQ4Warps][256]; /* for rows that are not aligned */
    T *const line = lines[threadIdx.x >> 5];
    uint32_t word[kRun];
    float s[kRun], m[kRun];
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        const int c = c0 + u * 256 + (lane >> 2) * 32;
        word[u] = 0;
        if (c >= p.cols) continue;
        word[u] = q0[u * 32];
        s[u] = __half2float(p.scale[s0 + c / kGroup]);
        m[u] = kMin ? __half2float(p.min[s0 + c / kGroup]) : 0.0f;
    }
    T *const w0 = (T *)p.w + (size_t)row * p.w_stride + c0;
#pragma unroll
    for (int u = 0; u < kRun; ++u) {
        const int c = (lane >> 2) * 32 + (lane & 3) * 4, left = p.cols - c0 - u * 256;
        if (left <= 0) break;
        T *const w = w0 + u * 256;
        float v[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = (float)((word[u] >> (8 * i + 4 * h)) & 15u);
                /* s * q is exact in 32 bits (11 and 4 bits): one rounding */
                v[h][i] = kMin ? fmaf(s[u], q, m[u]) : __fmul_rn(s[u], q - 8.0f);
            }
        if (sizeof(T) == 2 && p.aligned && left >= 256) {
            /* an even lane gives its high columns and takes its neighbour's low ones: eight in a row, 16 bytes */
            Four<T> own[2], got;
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) own[h].e[i] = from_f32<T>(v[h][i]);
            const bool h = (lane & 1) != 0;
            got.w[0] = __shfl_xor_sync(0xffffffffu, h ? own[0].w[0] : own[1].w[0], 1);
            got.w[1] = __shfl_xor_sync(0xffffffffu, h ? own[0].w[1] : own[1].w[1], 1);
            const uint4 x = h ? make_uint4(got.w[0], got.w[1], own[1].w[0], own[1].w[1])
                              : make_uint4(own[0].w[0], own[0].w[1], got.w[0], got.w[1]);
            *(uint4 *)(w + (lane >> 2) * 32 + (lane & 1) * 16 + (lane & 2) * 4) = x;
            continue;
        }
        if (!p.aligned) __syncwarp();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (p.aligned) put4(w + c + 16 * h, left - c - 16 * h, v[h]);
            else put4(line + c + 16 * h, 4, v[h]);
        }
        if (!p.aligned) { /* consecutive lanes, consecutive elements */
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 256; i += 32)
                if (i + lane < left) w[i + lane] = line[i + lane];
        }
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
    int dtype;
};

/* ---- up to sixteen streams at a time: mma.sync m16n8k32 on int8 ----
 *
 * A warp takes 16 kMT rows and every warps_k-th stage of 256 columns; the rows'
 * 4-bit words, their scales and the vectors go through a ring of shared memory
 * of its own (cp.async, no barrier of the CTA until the warps' sums are joined).
 * Large weights are read at 0.76 to 0.86 of the measured HBM rate (152064x3584
 * with one stream 55 us, with sixteen 58); few rows are bounded by a warp's
 * instructions a stage, about 22 a block and 16 rows (3584x18944 with eight
 * streams and minima 11.8 us, 0.55), the smallest by latency (3584x3584 3.6 us).  A
 * block's word t of row g, shifted and masked, is that lane's part of the A
 * operand for columns 4t.. and 16 + 4t..: q - 8 in the upper half of a byte is
 * 16 (q - 8) as int8, so the dots come out 16 times too large, which the results
 * take back.  The dots of a group are exact int32 (below 2^24), and are scaled
 * and added in fp32.  With a minimum, w = s q + m: A holds q itself, and a second
 * product with rows of ones gives the sums of the vectors.  (s (q - 8) and 8 s + m
 * would cancel where q is small, and leave 8 s of rounding: 3% of the result for
 * groups of one large weight and many small ones.) */
constexpr int kStageBlocks = 8;               /* 256 columns */
/* 16 bytes to shared memory, the last 16 - n of them zeros */
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async16_l1(uint32_t dst, const void *src, int n) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

/* the same from zero */
__device__ __forceinline__ void mma_s8_zero(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=r"(c[0]), "=r"(c[1]), "=r"(c[2]), "=r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0));
}

/* Four weights of a word, of columns j .. j + 3 or of those 16 further, as int8:
 * 16 (q - 8), or with minima q itself.  kUnit takes the 16 out of the results. */
template <bool kMin> __device__ __forceinline__ uint32_t low_weights(uint32_t w) {
    return kMin ? w & 0x0f0f0f0fu : ((w << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
}
template <bool kMin> __device__ __forceinline__ uint32_t high_weights(uint32_t w) {
    return kMin ? (w >> 4) & 0x0f0f0f0fu : (w & 0xf0f0f0f0u) ^ 0x80808080u;
}
template <bool kMin> constexpr float kUnit = kMin ? 1.0f : 0.0625f;

/* 16 columns c0 .. of kCount vectors, `step` bytes apart and aligned to 16 bytes,
 * of which n exist (of vector j to dst(j)); zeros behind their end. */
template <int kCount, typename Dst>
__device__ __forceinline__ void stage_x(Dst dst, const int8_t *x, size_t step, int n, int c0, int cols) {
    const int bytes = max(0, min(16, cols - c0));
    if (bytes > 0) x += c0;
#pragma unroll
    for (int j = 0; j < kCount; ++j, x += step)
        if (j < n) cp_async16_l1(smem_u32(dst(j)), x, bytes);
}

__device__ __forceinline__ void store_y(const MatvecParams &p, int b, int row, float v) {
    const size_t at = (size_t)b * p.y_stride + row;
    v = __fmul_rn(p.sx[b], v);
    if (p.dtype == LAL_TAIL_F32)
        ((float *)p.y)[at] = v;
    else if (p.dtype == LAL_TAIL_BF16)
        ((__nv_bfloat16 *)p.y)[at] = __float2bfloat16_rn(v);
    else
        ((__half *)p.y)[at] = __float2half_rn(v);
}

/* A warp's results from mma accumulators: 16 kMT rows from row0 (`rows` of them
 * exist) by 8 kNT streams from b0 (nx exist).  Written out once for each type,
 * with addresses moved on: code that runs once a tile is fetched for it alone. */
template <typename T, bool kMin, int kMT, int kNT>
__device__ __forceinline__ void store_tile_as(const MatvecParams &p, int b0, int nx, int row0, int rows,
                                              const float (&acc)[kMT][kNT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    T *y = (T *)p.y + (size_t)(b0 + 2 * t) * p.y_stride + row0 + g;
    const float *sx = p.sx + b0 + 2 * t;
#pragma unroll
    for (int n = 0; n < kNT; ++n, y += 8 * p.y_stride) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if (8 * n + 2 * t + c >= nx) break;
            const float s = sx[8 * n + c];
#pragma unroll
            for (int r = 0; r < 2 * kMT; ++r)
                if (g + 8 * r < rows)
                    y[c * p.y_stride + 8 * r] = from_f32<T>(__fmul_rn(s, __fmul_rn(kUnit<kMin>, acc[r >> 1][n][2 * (r & 1) + c])));
        }
    }
}
template <bool kMin, int kMT, int kNT>
__device__ __forceinline__ void store_tile(const MatvecParams &p, int b0, int nx, int row0, int rows,
                                           const float (&acc)[kMT][kNT][4]) {
    if (p.dtype == LAL_TAIL_F32) store_tile_as<float, kMin>(p, b0, nx, row0, rows, acc);
    else if (p.dtype == LAL_TAIL_BF16) store_tile_as<__nv_bfloat16, kMin>(p, b0, nx, row0, rows, acc);
    else store_tile_as<__half, kMin>(p, b0, nx, row0, rows, acc);
}

/* kCount words from an even offset on */
template <int kCount> __device__ __forceinline__ void shifted_words(uint32_t (&w)[kCount], const uint8_t *from, uint32_t off) {
    const uint32_t *at = (const uint32_t *)(from + (off & ~3u));
    uint32_t a = at[0];
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
        const uint32_t b = at[i + 1];
        w[i] = __funnelshift_r(a, b, 8 * (off & 2));
        a = b;
    }
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

/* How a warp's ring is filled.  kAligned: vectors and rows of scales begin at
 * 16-byte boundaries (scales: of a stage's size) and lie as ldmatrix wants
 * them.  kAny: the aligned 16-byte pieces around them are copied as they are
 * (each holds a byte of its row, so none lies outside memory), and their
 * offsets are taken at the reading, so these copies are asynchronous too.  kMany
 * (aligned, 32 rows a warp, tiles for several waves): more warps with shorter
 * rings; 58 us against 66 for 152064x3584 g128 and sixteen streams, but 19.3
 * against 14.8 for 37888x3584, one wave. */
enum MmaFill { kAligned, kMany, kAny };

/* What a warp's ring holds a stage: weights of 16 kMT rows, their scales (and
 * minima), the part of 8 kNT vectors. */
template <int kMT, int kNT, int kGroup, bool kMin, MmaFill kFill> struct MmaStage {
    static constexpr int kGroups = kStageBlocks * kQ4Block / kGroup;
    /* bytes of a row's scales, of a vector's part; kAny: two and seventeen pieces, eight rows in different banks */
    static constexpr int kSRow = kFill == kAny ? 48 : kGroups * 2;
    static constexpr int kXRow = kStageBlocks * 32 + (kFill == kAny ? 16 : 0);
    static constexpr int kScale = 16 * kMT * kSRow;
    static constexpr int kS = 16 * kMT * 128, kX = (kS + (kMin ? 2 : 1) * kScale + 127) / 128 * 128;
    static constexpr int kBytes = (kX + 8 * kNT * kXRow + 127) / 128 * 128;
    static constexpr int kWarps = kFill == kMany ? 12 : 8, kCtas = kMT * kNT == 1 ? 2 : 1;
    static constexpr int kDepth = kFill == kMany || (kFill == kAny && kMT * kNT != 2) ? 2 : 3;
    static constexpr int kSmem = kWarps * kDepth * kBytes;
    static_assert(kCtas * (kSmem + 1024) <= 228 * 1024, "CTAs of an SM");
};

template <int kMT, int kNT, int kGroup, bool kMin, MmaFill kFill>
__global__ void __launch_bounds__(kFill == kMany ? 384 : 256, kMT * kNT == 1 ? 2 : 1) q4_mma_kernel(const MatvecParams p, int x_base, int warps_k, int height) {
    extern __shared__ __align__(128) uint8_t smem[];
    using Stage = MmaStage<kMT, kNT, kGroup, kMin, kFill>;
    constexpr int kDepth = Stage::kDepth, kWarps = Stage::kWarps;
    constexpr int kPer = kGroup / kQ4Block, kGroups = Stage::kGroups; /* blocks of a group, groups of a stage */
    constexpr int kRows = 16 * kMT, kStreams = 8 * kNT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = warp % warps_k;
    const int row0 = (blockIdx.x * (kWarps / warps_k) + warp / warps_k) * height;
    const int b0 = x_base + blockIdx.y * kStreams, nx = min(kStreams, p.streams - b0);
    const int nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int stages = (nb + kStageBlocks - 1) / kStageBlocks;
    uint8_t *const ring = smem + warp * kDepth * Stage::kBytes;
    const uint32_t ring32 = smem_u32(ring);

    float acc[kMT][kNT][4] = {};
    const bool live = row0 < p.rows;
    if (live) {
        const int rows = min(height, p.rows - row0);
        /* ---- loads: this lane's share of a stage, its sources moved on by warps_k stages ---- */
        /* block lane & 7 of rows lane / 8, + 4, ...; in place block ^ (row mod 8) */
        const int w_r = lane >> 3, w_k = lane & 7;
        const uint32_t w_to = ring32 + w_r * 128 + ((w_k ^ w_r) << 4);
        const uint8_t *w_src = p.q + ((size_t)(row0 + w_r) * nb + wk * kStageBlocks + w_k) * 16;
        const size_t w_step = (size_t)nb * 64;
        /* 16 bytes lane & 15 of vectors lane / 16, + 2, ...; in place piece ^ (vector mod 8) */
        const int x_n = lane >> 4, x_c = lane & 15;
        const int8_t *x_src = p.x + (size_t)(b0 + x_n) * p.x_stride;
        const size_t x_step = (size_t)2 * p.x_stride;
        /* a row's scales of a stage, one copy (kAny: two): lane has rows lane, + 32, the minima after the scales */
        constexpr int kCopies = kRows * (kMin ? 2 : 1);
        auto load = [&](int st, int slot) {
            const uint32_t base = slot * Stage::kBytes;
            const int k0 = st * kStageBlocks;
            if (k0 + w_k < nb) {
#pragma unroll
                for (int j = 0; j < 4 * kMT; ++j)
                    if (w_r + 4 * j < rows) cp_async16((w_to + base + j * 512) ^ (j & 1 ? 64 : 0), w_src + j * w_step, 16);
            }
            w_src += (size_t)warps_k * (kStageBlocks * 16);
            const int c0 = k0 * kQ4Block + x_c * 16;
            uint8_t *const x_to = ring + base + Stage::kX + x_n * Stage::kXRow;
            if constexpr (kFill != kAny) {
                stage_x<4 * kNT>([&](int j) { return x_to + j * 512 + ((x_c ^ ((x_n + 2 * j) & 7)) << 4); }, x_src, x_step,
                                 (nx - x_n + 1) >> 1, c0, p.cols);
            } else {
                /* pieces x_c, and by the last lane of a row the seventeenth, from the boundary at or before column 256 st */
                const int8_t *x = x_src;
#pragma unroll
                for (int j = 0; j < 4 * kNT; ++j, x += x_step) {
                    if (x_n + 2 * j >= nx) break;
                    const int8_t *from = x + k0 * kQ4Block, *end = x + p.cols;
                    from -= (uintptr_t)from & 15;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int piece = e ? 16 : x_c;
                        if (e && x_c != 15) break;
                        const int8_t *src = from + piece * 16;
                        const int n = (int)max(0LL, min(16LL, (long long)(end - src)));
                        cp_async16_l1(smem_u32(x_to + j * 2 * Stage::kXRow + piece * 16), n > 0 ? src : from, n);
                    }
                }
            }
            const int g0 = st * kGroups;
#pragma unroll
            for (int i = lane; i < kCopies; i += 32) {
                const unsigned short *row = (const unsigned short *)(i < kRows ? p.scale : p.min) +
                                            (size_t)(row0 + min(i % kRows, rows - 1)) * groups;
                uint8_t *to = ring + base + Stage::kS + i * Stage::kSRow;
                if constexpr (kFill == kAny) {
                    const uint8_t *from = (const uint8_t *)(row + g0), *end = (const uint8_t *)(row + groups);
                    const int off = (int)((uintptr_t)from & 15);
                    from -= off;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (e && off + 2 * kGroups <= 16) break; /* within the first */
                        const int n = (int)max(0LL, min(16LL, (long long)(end - from) - 16 * e));
                        cp_async16_l1(smem_u32(to + 16 * e), n > 0 ? from + 16 * e : from, n);
                    }
                } else { /* a row of scales is whole stages (all_aligned) */
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(row + g0), "n"(2 * kGroups) : "memory");
                }
            }
        };
        /* weights on their way into L2 while the kernel before ends; nothing is read yet */
#pragma unroll
        for (int j = 0; j < 4 * kMT; ++j)
            if (wk * kStageBlocks + w_k < nb && w_r + 4 * j < rows) prefetch_l2(w_src + j * w_step);
        after_previous();
        int ahead = wk;
#pragma unroll
        for (int i = 0; i < kDepth - 1; ++i, ahead += warps_k) {
            if (ahead < stages) load(ahead, i);
            cp_async_commit();
        }
        /* ldmatrix addresses: rows lane mod 16, block lane / 16 of a pair; vectors lane mod 8, piece lane / 8 of a pair's four */
        const uint32_t a_at = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
        const uint32_t x_at = Stage::kX + (lane & 7) * 256 + (((lane >> 3) ^ (lane & 7)) << 4);
        /* kAny: this lane's first word of vector 8 n + g, and the bits to shift it by */
        uint32_t x_any[kNT], x_shift[kNT];
        if constexpr (kFill == kAny) {
#pragma unroll
            for (int n = 0; n < kNT; ++n) {
                const int v = min(8 * n + g, nx - 1); /* vectors that are not there: any, their sums are dropped */
                const uint32_t off = (uint32_t)(uintptr_t)(p.x + (size_t)(b0 + v) * p.x_stride) & 15;
                x_any[n] = Stage::kX + v * Stage::kXRow + (off & ~3u) + 4 * t;
                x_shift[n] = 8 * (off & 3);
            }
        }
        int slot = 0;
        for (int st = wk; st < stages; st += warps_k, ahead += warps_k) {
            cp_async_wait<kDepth - 2>();
            __syncwarp();
            if (ahead < stages) load(ahead, slot == 0 ? kDepth - 1 : slot - 1);
            cp_async_commit();
            const uint32_t at = ring32 + slot * Stage::kBytes;
            using Pack = std::conditional_t<kGroups == 8, uint4, std::conditional_t<kGroups == 4, uint2, uint32_t>>;
            union Row {
                Pack all;
                uint32_t word[kGroups / 2];
                __half one[kGroups];
                __device__ Row() {}
            } scale[kMT][2], low[kMT][2]; /* of rows g and g + 8 */
            const uint8_t *sc = ring + slot * Stage::kBytes + Stage::kS + g * Stage::kSRow;
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint8_t *at_s = sc + (16 * m + 8 * h) * Stage::kSRow;
                    if constexpr (kFill != kAny) {
                        scale[m][h].all = *(const Pack *)at_s;
                        if (kMin) low[m][h].all = *(const Pack *)(at_s + Stage::kScale);
                    } else {
                        /* rows that are not there: any offset within the copy */
                        const size_t i = (size_t)(row0 + min(g + 16 * m + 8 * h, rows - 1)) * groups + st * kGroups;
                        const uint32_t off = (uint32_t)(uintptr_t)(p.scale + i) & 15, off_m = (uint32_t)(uintptr_t)(p.min + i) & 15;
                        shifted_words(scale[m][h].word, at_s, off);
                        if (kMin) shifted_words(low[m][h].word, at_s + Stage::kScale, off_m);
                    }
                }
            int c[kMT][kNT][4], cx[kNT][4];
#pragma unroll
            for (int pair = 0; pair < kStageBlocks / 2; ++pair) {
                /* blocks behind the row's end hold zeros in the vectors; groups behind it (kAny) scales of zero */
                uint32_t w[kMT][4], x[kNT][4];
#pragma unroll
                for (int m = 0; m < kMT; ++m) ldmatrix4(w[m], (at + a_at + m * 2048) ^ (pair << 5));
#pragma unroll
                for (int n = 0; n < kNT; ++n) {
                    if constexpr (kFill != kAny) {
                        ldmatrix4(x[n], ((at + x_at + n * 2048) ^ ((pair & 1) << 6)) + (pair >> 1) * 128);
                    } else {
                        const uint8_t *from = ring + slot * Stage::kBytes + x_any[n] + pair * 64;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            x[n][i] = __funnelshift_r(*(const uint32_t *)(from + 16 * i), *(const uint32_t *)(from + 16 * i + 4), x_shift[n]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const int block = 2 * pair + k;
                    const bool begin = block % kPer == 0;
                    if (kMin) {
                        const uint32_t ones[4] = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
#pragma unroll
                        for (int n = 0; n < kNT; ++n) {
                            if (begin) mma_s8_zero(cx[n], ones, x[n][2 * k], x[n][2 * k + 1]);
                            else mma_s8(cx[n], ones, x[n][2 * k], x[n][2 * k + 1]);
                        }
                    }
#pragma unroll
                    for (int m = 0; m < kMT; ++m) {
                        const uint32_t w0 = w[m][2 * k], w1 = w[m][2 * k + 1];
                        const uint32_t a[4] = {low_weights<kMin>(w0), low_weights<kMin>(w1), high_weights<kMin>(w0), high_weights<kMin>(w1)};
#pragma unroll
                        for (int n = 0; n < kNT; ++n) {
                            if (begin) mma_s8_zero(c[m][n], a, x[n][2 * k], x[n][2 * k + 1]);
                            else mma_s8(c[m][n], a, x[n][2 * k], x[n][2 * k + 1]);
                        }
                        if (block % kPer != kPer - 1) continue;
                        const int gr = block / kPer;
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float s = __half2float(scale[m][h].one[gr]);
                            const float l = kMin ? __half2float(low[m][h].one[gr]) : 0.0f;
#pragma unroll
                            for (int n = 0; n < kNT; ++n)
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    acc[m][n][2 * h + i] = fmaf(s, (float)c[m][n][2 * h + i], acc[m][n][2 * h + i]);
                                    if (kMin) acc[m][n][2 * h + i] = fmaf(l, (float)cx[n][i], acc[m][n][2 * h + i]);
                                }
                        }
                    }
                }
            }
            slot = slot + 1 == kDepth ? 0 : slot + 1;
        }
        cp_async_wait<0>();
    } else {
        after_previous();
    }
    if (warps_k == 1) {
        if (live) store_tile<kMin>(p, b0, nx, row0, min(height, p.rows - row0), acc);
        return;
    }
    /* the warps of a row tile, in order; their sums take the rings' place */
    __syncthreads();
    float(*part)[kRows * kStreams] = (float(*)[kRows * kStreams])smem;
#pragma unroll
    for (int m = 0; m < kMT; ++m)
#pragma unroll
        for (int n = 0; n < kNT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                part[warp][(8 * n + 2 * t + (i & 1)) * kRows + 16 * m + g + (i >> 1) * 8] = acc[m][n][i];
    __syncthreads();
    const int tiles = kWarps / warps_k;
    for (int i = threadIdx.x; i < tiles * kRows * nx; i += 32 * kWarps) {
        const int r = i % kRows, b = i / kRows % nx, tile = i / kRows / nx;
        const int row = (blockIdx.x * tiles + tile) * height + r;
        if (r >= height || row >= p.rows) continue;
        float sum = 0.0f;
        for (int w = 0; w < warps_k; ++w) sum += part[tile * warps_k + w][b * kRows + r];
        store_y(p, b0 + b, row, kUnit<kMin> * sum);
    }
}

template <int kMT, int kNT, int kGroup, bool kMin, MmaFill kFill>
cudaError_t launch_mma(const MatvecParams &p, int x_base, int num_sms, cudaStream_t st) {
    /* warps of a row tile: as many as fit the SMs at once, no more than there are stages */
    using Stage = MmaStage<kMT, kNT, kGroup, kMin, kFill>;
    constexpr int kRows = 16 * kMT, kWarps = Stage::kWarps, kWarpsSm = Stage::kCtas * kWarps;
    const int tiles = (p.rows + kRows - 1) / kRows, stages = (q4_blocks(p.cols) + kStageBlocks - 1) / kStageBlocks;
    int wk = 1;
    while (kFill != kMany && wk < kWarps && 2 * wk <= stages && (long long)tiles * 2 * wk <= (long long)kWarpsSm * num_sms) wk *= 2;
    /* rows of a tile: fewer than it holds where that gives every SM some */
    const int at_once = num_sms * (kWarpsSm / wk), waves = (tiles + at_once - 1) / at_once;
    const int height = waves > 1 ? kRows : std::max((p.rows + at_once - 1) / at_once, std::min(p.rows, kRows / 2));
    const int n = (p.rows + height - 1) / height, per = kWarps / wk;
    constexpr int smem = Stage::kSmem;
    const cudaError_t e = raise_smem((const void *)q4_mma_kernel<kMT, kNT, kGroup, kMin, kFill>, smem);
    if (e != cudaSuccess) return e;
    return launch_early(q4_mma_kernel<kMT, kNT, kGroup, kMin, kFill>,
                        dim3((n + per - 1) / per, (p.streams - x_base + 8 * kNT - 1) / (8 * kNT)), 32 * kWarps, smem, st, 1, p,
                        x_base, wk, height);
}

/* ---- 33 streams and more: tcgen05.mma kind::i8 ----
 *
 * 37888x3584 g128 with 64 streams 30.5 us, 0.38 of HBM's rate and 0.34 of the
 * bf16 one; bounded by what the warps' roles take in turn a stage (with their
 * arithmetic, products and vectors taken out it still takes 21 us).
 *
 * A CTA takes tiles of 128 rows by up to 64 streams.  The weights are the A
 * operand and lie in tensor memory: a thread of the eight unpacking warps has a
 * row, reads its 16-byte blocks from a ring of its warp's own (cp.async) and
 * stores 16 (q - 8), or with minima q, as int8, eight columns of tensor memory a
 * block.  The vectors are the B operand, in shared memory with the 128-byte
 * swizzle.  One thread issues the products, two groups of columns at a time into two of kTcD
 * accumulators; sixteen warps read finished ones (int32, exact), scale them
 * by the row's scales of the groups and add them in fp32 registers, while the
 * next groups are multiplied.  So every scale is applied in fp32, the weights are
 * read once, and only the unpacked weights' 8-bit form is ever written on the
 * chip.  With few tiles, the K range of a tile is split over a cluster of
 * CTAs, whose sums are exchanged and added in order over distributed shared
 * memory.
 *
 * Every wait is bounded; one that runs out makes the tile's results NaN. */
constexpr int kTcUnpack = 8, kTcEpi = 16, kTcLoad = 4;
constexpr int kTcIssue = kTcUnpack + kTcEpi; /* the warp that issues the products */
constexpr int kTcWarps = kTcIssue + 1 + kTcLoad;
constexpr int kTcA = 4;        /* stages of unpacked weights in tensor memory, 64 columns each */
constexpr int kTcD = 4;        /* accumulators, handed over in pairs: 30.6 us against 35.1 one by one, groups of 32 53.6 against 69.8 */
constexpr int kTcPairs = kTcD / 2;
constexpr int kTcWDepth = 6;   /* stages of a warp's weight ring */
constexpr int kTcXDepth = 4;   /* stages of the vectors */
constexpr int kTcHalf = kStageBlocks / 2;         /* blocks of a stage that an unpacking warp has */
constexpr int kTcWStage = 32 * kTcHalf * 16;
constexpr int kTcMaxSplit = 8;
constexpr int kTcStreams = 64;

struct TcShared {
    uint64_t a_full[kTcA], a_empty[kTcA], x_full[kTcXDepth], x_empty[kTcXDepth], d_full[kTcPairs], d_empty[kTcPairs], drain;
    uint32_t tmem;
    int abort, never;
};

constexpr int kTcXStage = kTcStreams * kStageBlocks * 32;
template <int kGroup, bool kMin> constexpr int tc_smem() {
    constexpr int kGroups = kStageBlocks * kQ4Block / kGroup; /* of a stage: scales (and minima), sums of the vectors */
    return 1024 + kTcUnpack * kTcWDepth * kTcWStage +
           kTcXDepth * (kTcXStage + 128 * kGroups * (kMin ? 4 : 2) + (kMin ? kGroups * kTcStreams * 4 : 0));
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
/* arrive on bar when every tcgen05.mma this thread issued before has completed */
__device__ __forceinline__ void tc_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
/* Shared-memory descriptor of rows of 128 bytes with the 128-byte swizzle
 * (8-row groups 1024 bytes apart): its low word from the address in units of
 * 16 bytes, to which a K step of 32 bytes adds 2, and its high word. */
constexpr uint32_t kTcDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t tc_desc_low(uint32_t at) { return ((at >> 4) & 0x3FFFu) | 1u << 16; }
/* D[tensor memory] (+)= A[tensor memory] * B[shared memory]^T, int8 x int8 -> int32 */
__device__ __forceinline__ void tc_mma_i8_ta(uint32_t d, uint32_t a, uint32_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "mov.b64 b, {%2, %6};\n\t"
                 "tcgen05.mma.cta_group::1.kind::i8 [%0], [%1], b, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
                 "r"(a), "r"(bdesc), "r"(idesc), "r"(accumulate), "r"(0), "r"(kTcDescHigh));
}
/* int32 accumulators, signed int8 operands, both K-major, 128 rows by n */
__device__ constexpr uint32_t tc_idesc(int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void tc_store8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(at), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tc_load16(uint32_t at, int (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
    /* the wait names the registers, so that nothing reads them before it */
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

/* A thread's results, n of kCount streams from b0, of a row. */
template <typename T, bool kMin, int kCount>
__device__ __forceinline__ void store_row(const MatvecParams &p, int b0, int n, int row, const float (&acc)[kCount]) {
    T *y = (T *)p.y + (size_t)b0 * p.y_stride + row;
#pragma unroll
    for (int j = 0; j < kCount; ++j, y += p.y_stride)
        if (j < n) *y = from_f32<T>(__fmul_rn(p.sx[b0 + j], __fmul_rn(kUnit<kMin>, acc[j])));
}

/* The stages of a CTA in order: every tile's range of K. */
struct TcWalk {
    int tile, st, n = 0;
    __device__ TcWalk(int tile0, int st0) : tile(tile0), st(st0) {}
    __device__ void next(int st0, int st1, int tile_step) {
        ++n;
        if (++st == st1) st = st0, tile += tile_step;
    }
};

/* A bounded wait, as mbar_wait, that reads a clock only once it has waited long. */
__device__ __forceinline__ bool tc_wait(uint64_t *b, uint32_t parity, volatile int *abort_flag) {
    constexpr long long kClocks = 4000000000LL; /* about two seconds */
    long long t0 = 0;
    for (uint32_t it = 1; !mbar_try(b, parity); ++it) {
        if ((it & 255u) != 0) continue;
        if (*abort_flag) return false;
        const long long now = clock64();
        if (t0 == 0) t0 = now;
        if (now - t0 > kClocks) return false;
    }
    return true;
}

template <int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kTcWarps, 1) q4_tc_kernel(const MatvecParams p, int splits, int x_base) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ TcShared sh;
    constexpr int kPer = kGroup / kQ4Block, kGroups = kStageBlocks / kPer; /* blocks a group, groups a stage */
    constexpr int kN = kTcStreams, kMine = kN / (kTcEpi / 4);              /* streams of a tile, of an epilogue warp */
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *xring = smem;                                      /* kTcXDepth stages of two swizzled tiles */
    uint8_t *wring = xring + kTcXDepth * kTcXStage;        /* of each unpacking warp */
    uint8_t *sring = wring + kTcUnpack * kTcWDepth * kTcWStage; /* scales: [kTcXDepth][1, or 2 with minima][128][kGroups] */
    float *xsums = (float *)(sring + kTcXDepth * 128 * kGroups * (kMin ? 4 : 2)); /* [kTcXDepth][kGroups][kN] */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort_flag = &sh.abort, *never = &sh.never;
    const int b0 = x_base + blockIdx.y * kN, nx = min(kN, p.streams - b0);
    const int nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int all = (nb + kStageBlocks - 1) / kStageBlocks; /* stages of a row */
    const int tiles = (p.rows + 127) / 128;
    /* this CTA's tiles, and its stages of each */
    const int split = (int)(blockIdx.x % splits), tile0 = (int)(blockIdx.x / splits), tile_step = (int)(gridDim.x / splits);
    const int st0 = (int)((long long)all * split / splits), st1 = (int)((long long)all * (split + 1) / splits);
    const int my_tiles = tile0 < tiles ? (tiles - 1 - tile0) / tile_step + 1 : 0;
    const int per = st1 - st0, total = my_tiles * per;

    if (threadIdx.x == 0) {
        for (int i = 0; i < kTcA; ++i) mbar_init(&sh.a_full[i], kTcUnpack), mbar_init(&sh.a_empty[i], 1);
        for (int i = 0; i < kTcXDepth; ++i)
            mbar_init(&sh.x_full[i], kTcLoad), mbar_init(&sh.x_empty[i], kTcEpi);
        for (int i = 0; i < kTcPairs; ++i) mbar_init(&sh.d_full[i], 1), mbar_init(&sh.d_empty[i], kTcEpi);
        mbar_init(&sh.drain, 1);
        sh.abort = sh.never = 0;
        mbar_fence_init();
    }
    constexpr int kCols = 512;
    static_assert(64 * kTcA + kTcD * kN <= kCols, "tensor memory");
    if (warp == kTcIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    after_previous();
    const uint32_t tmem = sh.tmem, tmem_d = tmem + 64 * kTcA; /* the A operands, then the accumulators */

    float acc[kMine]; /* of an epilogue thread */

    if (warp < kTcUnpack) {
        /* ---- weights: 4 bits in global memory -> int8 in tensor memory;
         * rows of one quarter of tensor memory, half of a stage's blocks ---- */
        uint8_t *ring = wring + warp * kTcWDepth * kTcWStage;
        const int quad = warp & 3, half = warp >> 2;
        const uint32_t to = tmem + ((uint32_t)(quad * 32) << 16) + half * (kTcHalf * 8);
        const int k = half * kTcHalf + (lane & 3); /* this lane's block of a stage, of rows lane / 4, + 8, ... */
        const uint32_t dst = smem_u32(ring) + lane * 16; /* 4 blocks a row; swizzled by the row's pair */
        TcWalk ahead(tile0, st0);
        auto load = [&](int slot) {
            if (ahead.n < total) {
                const int row0 = ahead.tile * 128 + quad * 32 + (lane >> 2), kb = ahead.st * kStageBlocks + k;
                const uint32_t to_slot = (dst + slot * kTcWStage) ^ (((lane >> 3) & 3) << 4);
                if (row0 + 24 < p.rows && kb < nb) {
                    const uint8_t *src = p.q + ((size_t)row0 * nb + kb) * 16;
                    const size_t step = (size_t)nb * 128; /* 8 rows */
#pragma unroll
                    for (int j = 0; j < 4; ++j) cp_async16(to_slot + j * 512, src + j * step, 16);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        cp_async16(to_slot + j * 512, p.q + ((size_t)min(row0 + 8 * j, p.rows - 1) * nb + min(kb, nb - 1)) * 16,
                                   kb < nb ? 16 : 0);
                }
            }
            ahead.next(st0, st1, tile_step);
            cp_async_commit();
        };
        for (int i = 0; i < kTcWDepth - 1; ++i) load(i);
        int slot = 0;
        for (int it = 0; it < total; ++it) {
            cp_async_wait<kTcWDepth - 2>();
            __syncwarp();
            load(slot == 0 ? kTcWDepth - 1 : slot - 1);
            uint4 v[kTcHalf];
            const uint8_t *row = ring + slot * kTcWStage + lane * 64;
#pragma unroll
            for (int i = 0; i < kTcHalf; ++i) v[i] = *(const uint4 *)(row + ((i ^ ((lane >> 1) & 3)) << 4));
            slot = slot + 1 == kTcWDepth ? 0 : slot + 1;
            const int buf = it % kTcA;
            const bool ok = it < kTcA || tc_wait(&sh.a_empty[buf], ((it / kTcA) & 1) ^ 1, abort_flag);
            if (!__all_sync(0xffffffffu, ok)) { /* a warp leaves as one: what follows is for all its lanes */
                *abort_flag = 1;
                break;
            }
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kTcHalf; ++i) {
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[j] = low_weights<kMin>(w[j]);
                    o[4 + j] = high_weights<kMin>(w[j]);
                }
                tc_store8(to + buf * 64 + i * 8, o);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.a_full[buf]);
        }
        cp_async_wait<0>();
    } else if (warp < kTcIssue) {
        /* ---- accumulators: scaled and added ---- */
        const int quad = warp & 3, part = (warp - kTcUnpack) >> 2;
        const uint32_t lanes = tmem_d + ((uint32_t)(quad * 32) << 16) + part * kMine;
        /* a row's scales (and minima) of a stage */
        using Pack = std::conditional_t<kGroups == 8, uint4, std::conditional_t<kGroups == 4, uint2, uint32_t>>;
        union Row {
            Pack all;
            unsigned short one[kGroups];
            __device__ Row() {}
        } scale, low;
        bool ok = true;
        TcWalk at(tile0, st0);
        for (int d = 0, xs = 0, xs_round = 0; at.n < total; at.next(st0, st1, tile_step)) {
            if (at.st == st0)
#pragma unroll
                for (int j = 0; j < kMine; ++j) acc[j] = 0.0f;
            if (!tc_wait(&sh.x_full[xs], xs_round & 1, abort_flag)) ok = false;
            const Pack *sc = (const Pack *)sring + xs * (kMin ? 256 : 128) + quad * 32 + lane;
            scale.all = sc[0];
            if (kMin) low.all = sc[128];
#pragma unroll
            for (int pair = 0; pair < kGroups / 2; ++pair, ++d) {
                const int buf = d % kTcPairs;
                if (ok && !tc_wait(&sh.d_full[buf], (d / kTcPairs) & 1, abort_flag)) ok = false;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int gr = 2 * pair + h;
                    int c[kMine];
                    tc_load16(lanes + (2 * buf + h) * kN, c);
                    if (h == 1) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sh.d_empty[buf]);
                    }
                    const float s = __half2float(__ushort_as_half(scale.one[gr]));
#pragma unroll
                    for (int j = 0; j < kMine; ++j) acc[j] = fmaf(s, (float)c[j], acc[j]);
                    if (kMin) {
                        const float m = __half2float(__ushort_as_half(low.one[gr]));
                        const float4 *sum = (const float4 *)(xsums + (xs * kGroups + gr) * kN + part * kMine);
#pragma unroll
                        for (int j = 0; j < kMine; j += 4) {
                            const float4 v = sum[j / 4];
                            acc[j] = fmaf(m, v.x, acc[j]);
                            acc[j + 1] = fmaf(m, v.y, acc[j + 1]);
                            acc[j + 2] = fmaf(m, v.z, acc[j + 2]);
                            acc[j + 3] = fmaf(m, v.w, acc[j + 3]);
                        }
                    }
                }
            }
            if (!ok) break;
            /* the stage's products are complete, its vectors and scales read */
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.x_empty[xs]);
            if (++xs == kTcXDepth) xs = 0, ++xs_round;
            if (splits == 1 && at.st == st1 - 1) {
                const int row = at.tile * 128 + quad * 32 + lane;
                if (row < p.rows) {
                    if (p.dtype == LAL_TAIL_F32) store_row<float, kMin>(p, b0 + part * kMine, nx - part * kMine, row, acc);
                    else if (p.dtype == LAL_TAIL_BF16) store_row<__nv_bfloat16, kMin>(p, b0 + part * kMine, nx - part * kMine, row, acc);
                    else store_row<__half, kMin>(p, b0 + part * kMine, nx - part * kMine, row, acc);
                }
            }
        }
        if (!ok) {
#pragma unroll
            for (int j = 0; j < kMine; ++j) acc[j] = __int_as_float(0x7fc00000);
            /* loud: every tile of this CTA */
            if (splits == 1)
                for (int t = 0; t < my_tiles; ++t) {
                    const int row = (tile0 + t * tile_step) * 128 + quad * 32 + lane;
                    if (row < p.rows)
                        for (int j = 0; j < kMine; ++j)
                            if (part * kMine + j < nx) store_y(p, b0 + part * kMine + j, row, acc[0]);
                }
        }
    } else if (warp == kTcIssue) {
        /* ---- products ---- */
        if (lane == 0) {
            bool ok = true;
            const uint32_t x0 = tc_desc_low(smem_u32(xring));
            int xs = 0, xs_round = 0;
            for (int it = 0, d = 0; it < total && ok; ++it) {
                const int buf = it % kTcA;
                if (!tc_wait(&sh.x_full[xs], xs_round & 1, abort_flag) ||
                    !tc_wait(&sh.a_full[buf], (it / kTcA) & 1, abort_flag)) {
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t xt = x0 + xs * (kTcXStage >> 4);
#pragma unroll
                for (int pair = 0; pair < kGroups / 2; ++pair, ++d) {
                    const int d_buf = d % kTcPairs;
                    if (d >= kTcPairs && !tc_wait(&sh.d_empty[d_buf], ((d / kTcPairs) & 1) ^ 1, abort_flag)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int k = 2 * pair * kPer; k < 2 * (pair + 1) * kPer; ++k)
                        tc_mma_i8_ta(tmem_d + (2 * d_buf + k / kPer % 2) * kN, tmem + buf * 64 + k * 8,
                                     xt + (k / 4) * (kN * 128 >> 4) + (k % 4) * 2, tc_idesc(kN), k % kPer != 0);
                    tc_commit(&sh.d_full[d_buf]);
                }
                tc_commit(&sh.a_empty[buf]);
                if (++xs == kTcXDepth) xs = 0, ++xs_round;
            }
            /* every product issued is complete before the tensor memory is freed */
            tc_commit(&sh.drain);
            if (!tc_wait(&sh.drain, 0u, never)) *abort_flag = 1;
        }
    } else {
        /* ---- vectors, and (with minima) their sums; scales ---- */
        const int lw = warp - kTcIssue - 1;
        /* a loader warp has every kTcLoad-th pair of rows: 16 lanes a row */
        const int n0 = lw * 2 + (lane >> 4);
        const int8_t *x0 = p.x + (size_t)(b0 + min(n0, nx - 1)) * p.x_stride;
        const size_t x_step = (size_t)(2 * kTcLoad) * p.x_stride;
        const uint32_t d0 = ((lane & 15) >> 3) * kN * 128 + n0 * 128 + (((lane & 7) ^ (n0 & 7)) << 4);
        static_assert(2 * kTcLoad == 8, "a lane's rows are 8 apart: the same place in the swizzle");
        TcWalk ahead(tile0, st0);
        auto load = [&](int xs, int round) -> bool {
            if (ahead.n < total) {
                if (round > 0 && !tc_wait(&sh.x_empty[xs], (round & 1) ^ 1, abort_flag)) return false;
                const int c0 = ahead.st * kStageBlocks * kQ4Block + (lane & 15) * 16;
                uint8_t *dst = xring + xs * kTcXStage + d0;
                const int n = (nx - n0 + 2 * kTcLoad - 1) / (2 * kTcLoad); /* this lane's vectors, four at a time */
                stage_x<4>([&](int j) { return dst + j * 1024; }, x0, x_step, min(n, 4), c0, p.cols);
                if (n > 4)
                    stage_x<4>([&](int j) { return dst + 4096 + j * 1024; }, x0 + 4 * x_step, x_step, n - 4, c0, p.cols);
                /* the scales of row 32 lw + lane: as many stages ahead, their latency is HBM's */
                const int row = min(ahead.tile * 128 + lw * 32 + lane, p.rows - 1), g0 = ahead.st * kGroups;
#pragma unroll
                for (int m = 0; m < (kMin ? 2 : 1); ++m) {
                    const unsigned short *src = (const unsigned short *)(m ? p.min : p.scale) + (size_t)row * groups + g0;
                    uint8_t *to = sring + ((xs * (kMin ? 2 : 1) + m) * 128 + lw * 32 + lane) * (2 * kGroups);
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(to)), "l"(src), "n"(2 * kGroups) : "memory");
                }
            }
            ahead.next(st0, st1, tile_step);
            cp_async_commit();
            return true;
        };
        for (int i = 0; i < kTcXDepth - 1; ++i) load(i, 0);
        for (int it = 0, xs = 0, xl = kTcXDepth - 1, round = 0; it < total; ++it) {
            cp_async_wait<kTcXDepth - 2>();
            __syncwarp();
            if (kMin) {
                /* the sum of each group of this warp's rows */
                const uint8_t *st = xring + xs * kTcXStage;
                for (int i = lane; i < kN / kTcLoad * kGroups; i += 32) {
                    const int gr = i % kGroups, pair = i / kGroups;
                    const int n = (pair >> 1) * 2 * kTcLoad + lw * 2 + (pair & 1);
                    if (n >= nx) continue;
                    int sum = 0;
#pragma unroll
                    for (int j = 0; j < kPer * 2; ++j) {
                        const int c = gr * kPer * 2 + j;
                        const uint4 v = *(const uint4 *)(st + (c >> 3) * kN * 128 + n * 128 + (((c & 7) ^ (n & 7)) << 4));
                        sum = __dp4a((int)v.x, 0x01010101, __dp4a((int)v.y, 0x01010101, sum));
                        sum = __dp4a((int)v.z, 0x01010101, __dp4a((int)v.w, 0x01010101, sum));
                    }
                    xsums[(xs * kGroups + gr) * kN + n] = (float)sum;
                }
            }
            /* the copies (and stores) become visible to the tensor core */
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.x_full[xs]);
            const bool ok = load(xl, round);
            if (++xs == kTcXDepth) xs = 0;
            if (++xl == kTcXDepth) xl = 0, ++round;
            if (!__all_sync(0xffffffffu, ok)) {
                *abort_flag = 1;
                break;
            }
        }
        cp_async_wait<0>();
    }

    __syncwarp();
    if (splits > 1) {
        /* The CTAs of a tile: each gets every part's sums of kN / splits
         * streams, [part][stream][128 rows] where the rings were, and adds
         * them in order. */
        const int mine = kN / splits;
        float *parts = (float *)smem;
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (warp >= kTcUnpack && warp < kTcIssue) {
            const int quad = warp & 3, part = (warp - kTcUnpack) >> 2;
#pragma unroll
            for (int j = 0; j < kMine; ++j) {
                const int n = part * kMine + j;
                const uint32_t here = smem_u32(parts + ((size_t)split * mine + n % mine) * 128 + quad * 32 + lane);
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(here), "r"(n / mine));
                asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(per > 0 ? acc[j] : 0.0f) : "memory");
            }
        }
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        for (int i = threadIdx.x; i < mine * 128; i += 32 * kTcWarps) {
            const int n = split * mine + (i >> 7), row = tile0 * 128 + (i & 127);
            if (n >= nx || row >= p.rows) continue;
            float sum = 0.0f;
            for (int s = 0; s < splits; ++s) sum += parts[((size_t)s * mine + (i >> 7)) * 128 + (i & 127)];
            store_y(p, b0 + n, row, kUnit<kMin> * sum);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kTcIssue) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols) : "memory");
    }
}

template <int kGroup, bool kMin>
cudaError_t launch_tc(const MatvecParams &p, int x_base, int chunks, int num_sms, cudaStream_t st) {
    const int tiles = (p.rows + 127) / 128, stages = (q4_blocks(p.cols) + kStageBlocks - 1) / kStageBlocks;
    /* CTAs of a tile: as many as leave each an SM and two stages */
    int splits = 1;
    while (splits < kTcMaxSplit && (long long)tiles * chunks * splits * 2 <= num_sms && splits * 4 <= stages) splits *= 2;
    const void *fn = (const void *)q4_tc_kernel<kGroup, kMin>;
    constexpr int smem = tc_smem<kGroup, kMin>();
    cudaError_t e = raise_smem(fn, smem);
    if (e != cudaSuccess) return e;
    return launch_early(q4_tc_kernel<kGroup, kMin>,
                        dim3((unsigned)(splits > 1 ? tiles * splits : std::min(tiles, num_sms)), (unsigned)chunks), 32 * kTcWarps,
                        smem, st, splits, p, splits, x_base);
}

/* ---- 17 to 32 streams, many rows: the same products, the vectors shared by a CTA ----
 *
 * 37888x3584 g128 with 32 streams 21.7 us, 0.53 of HBM's rate; bounded by the
 * ldmatrix traffic of the vectors and the latency of eight warps an SM.
 *
 * A CTA of eight warps takes a range of rows, 32 a warp and tile, by up to 8
 * kNT streams.  A warp's weights and scales go through a ring of its own, as
 * above; the vectors' part of a stage is loaded once for all (a barrier a
 * stage), so that a stage's 8 kNT vectors serve 256 rows.  A CTA's ring runs on
 * over its tiles. */
constexpr int kWideDepth = 4;
constexpr int kWideMT = 2, kWideNT = 4;

struct WideShape {
    int range, height; /* rows of a CTA; of a warp and tile */
};

template <int kGroup, bool kMin> struct WideStage {
    static constexpr int kMT = kWideMT, kNT = kWideNT;
    static constexpr int kGroups = kStageBlocks * kQ4Block / kGroup;
    static constexpr int kWarps = 16 / kMT, kThreads = 32 * kWarps, kRows = 16 * kMT; /* rows of a warp */
    static constexpr int kA = kRows * 128, kScale = kRows * kGroups * 2;
    static constexpr int kW = (kA + (kMin ? 2 : 1) * kScale + 127) / 128 * 128; /* of a warp */
    static constexpr int kX = 8 * kNT * kStageBlocks * 32;
    static constexpr int kSmem = kWideDepth * (kX + kWarps * kW);
    static_assert(kSmem <= 227 * 1024, "one CTA an SM");
};

template <int kGroup, bool kMin>
__global__ void __launch_bounds__(512 / kWideMT, 1) q4_wide_kernel(const MatvecParams p, const WideShape h, int b0) {
    extern __shared__ __align__(128) uint8_t smem[];
    using Stage = WideStage<kGroup, kMin>;
    constexpr int kMT = kWideMT, kNT = kWideNT;
    constexpr int kWarps = Stage::kWarps, kGroups = Stage::kGroups, kPer = kGroup / kQ4Block;
    constexpr int kUnit = kPer < 2 ? 2 : kPer;        /* blocks between two readings of the scales */
    constexpr int kUnitGroups = kUnit / kPer, kUnits = kStageBlocks / kUnit;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int nx = p.streams - b0; /* at most 8 kNT */
    const int nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int stages = (nb + kStageBlocks - 1) / kStageBlocks; /* of a row */
    const int first = blockIdx.x * h.range, end = min(p.rows, first + h.range), tile_rows = kWarps * h.height;
    const int tiles = (end - first + tile_rows - 1) / tile_rows, total = tiles * stages;
    const uint32_t x_ring = smem_u32(smem), w_ring = x_ring + kWideDepth * Stage::kX + warp * kWideDepth * Stage::kW;

    /* ---- loads ---- */
    const int w_r = lane >> 3, w_k = lane & 7;
    const uint32_t w_to = w_ring + w_r * 128 + ((w_k ^ w_r) << 4);
    const size_t w_step = (size_t)nb * 64;
    const uint8_t *w_src = nullptr;
    const int x_n = threadIdx.x >> 4, x_c = threadIdx.x & 15; /* kXRows vectors at a time */
    constexpr int kXRows = Stage::kThreads / 16;
    const uint32_t x_to = x_ring + x_n * 256 + ((x_c ^ (x_n & 7)) << 4);
    const int8_t *const x_src = p.x + (size_t)(b0 + min(x_n, nx - 1)) * p.x_stride;
    const size_t x_step = (size_t)kXRows * p.x_stride;
    size_t s_row = 0;
    int l_row = first + warp * h.height, l_st = 0, l_slot = 0, l_left = total, l_rows = 0;
    auto load = [&] {
        if (l_left > 0) {
            if (l_st == 0) { /* a tile begins */
                l_rows = min(h.height, end - l_row); /* may be below 1 */
                w_src = p.q + ((size_t)(l_row + w_r) * nb + w_k) * 16;
                s_row = (size_t)(l_row + lane) * groups;
                l_row += tile_rows;
            }
            const int k0 = l_st * kStageBlocks;
            const uint32_t base = l_slot * Stage::kW;
            if (k0 + w_k < nb) {
#pragma unroll
                for (int j = 0; j < 4 * kMT; ++j)
                    if (w_r + 4 * j < l_rows) cp_async16((w_to + base + j * 512) ^ (j & 1 ? 64 : 0), w_src + j * w_step, 16);
            }
            w_src += kStageBlocks * 16;
            const int c0 = k0 * kQ4Block + x_c * 16;
            const uint32_t to = x_to + l_slot * Stage::kX;
            stage_x<8 * kNT / kXRows>([&](int j) { return smem + (to - x_ring) + j * (kXRows * 256); }, x_src, x_step,
                                      (nx - x_n + kXRows - 1) / kXRows, c0, p.cols);
            if (lane < l_rows) {
                const int g0 = l_st * kGroups;
#pragma unroll
                for (int m = 0; m < (kMin ? 2 : 1); ++m) {
                    const unsigned short *src = (const unsigned short *)(m ? p.min : p.scale) + s_row + g0;
                    const uint32_t dst = w_ring + base + Stage::kA + m * Stage::kScale + lane * (2 * kGroups);
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(2 * kGroups) : "memory");
                }
            }
            --l_left;
            if (++l_slot == kWideDepth) l_slot = 0;
            if (++l_st == stages) l_st = 0;
        }
        cp_async_commit();
    };
    after_previous();
    for (int i = 0; i < kWideDepth - 1; ++i) load();

    /* ---- products ---- */
    const uint32_t a_at = w_ring + (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    const uint32_t x_at = x_ring + (lane & 7) * 256 + (((lane >> 3) ^ (lane & 7)) << 4);
    const uint32_t s_at = w_ring + Stage::kA + g * (2 * kGroups);
    float acc[kMT][kNT][4];
    int slot = 0, st = 0, row0 = first + warp * h.height;
    for (int it = 0; it < total; ++it) {
        cp_async_wait<kWideDepth - 2>();
        __syncthreads();
        load();
        if (st == 0)
#pragma unroll
            for (int m = 0; m < kMT; ++m)
#pragma unroll
                for (int n = 0; n < kNT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.0f;
        if (row0 < end) {
            /* blocks behind the row's end hold zeros in the vectors */
            const uint32_t at = slot * Stage::kW, xt = slot * Stage::kX;
#pragma unroll 1
            for (int u = 0; u < kUnits; ++u) {
                uint32_t a[kMT][kUnit][4];
#pragma unroll
                for (int m = 0; m < kMT; ++m)
#pragma unroll
                    for (int q = 0; q < kUnit / 2; ++q) {
                        uint32_t w[4];
                        ldmatrix4(w, (a_at + at + m * 2048) ^ ((u * (kUnit / 2) + q) << 5));
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            a[m][2 * q + k][0] = low_weights<kMin>(w[2 * k]);
                            a[m][2 * q + k][1] = low_weights<kMin>(w[2 * k + 1]);
                            a[m][2 * q + k][2] = high_weights<kMin>(w[2 * k]);
                            a[m][2 * q + k][3] = high_weights<kMin>(w[2 * k + 1]);
                        }
                    }
                float s[kMT][2][kUnitGroups], l[kMT][2][kUnitGroups];
#pragma unroll
                for (int m = 0; m < kMT; ++m)
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t from = s_at + at + (16 * m + 8 * r) * (2 * kGroups) + u * (2 * kUnitGroups);
                        uint32_t v, w = 0;
                        if (kUnitGroups == 2) {
                            asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
                            if (kMin) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(from + Stage::kScale) : "memory");
                        } else {
                            asm volatile("ld.shared.u16 %0, [%1];" : "=r"(v) : "r"(from) : "memory");
                            if (kMin) asm volatile("ld.shared.u16 %0, [%1];" : "=r"(w) : "r"(from + Stage::kScale) : "memory");
                        }
#pragma unroll
                        for (int k = 0; k < kUnitGroups; ++k) {
                            s[m][r][k] = __half2float(__ushort_as_half((unsigned short)(v >> (16 * k))));
                            if (kMin) l[m][r][k] = __half2float(__ushort_as_half((unsigned short)(w >> (16 * k))));
                        }
                    }
                /* kB eights of vectors at once: as many independent products again */
                constexpr int kB = 2;
#pragma unroll
                for (int n0 = 0; n0 < kNT; n0 += kB) {
                    uint32_t x[kB][kUnit / 2][4];
#pragma unroll
                    for (int n = 0; n < kB; ++n)
#pragma unroll
                        for (int q = 0; q < kUnit / 2; ++q) {
                            const int pair = u * (kUnit / 2) + q;
                            ldmatrix4(x[n][q], ((x_at + xt + (n0 + n) * 2048) ^ ((pair & 1) << 6)) + (pair >> 1) * 128);
                        }
#pragma unroll
                    for (int k = 0; k < kUnitGroups; ++k) {
                        int c[kB][kMT][4], cx[kB][4];
#pragma unroll
                        for (int j = 0; j < kPer; ++j) {
                            const int i = k * kPer + j;
#pragma unroll
                            for (int n = 0; n < kB; ++n) {
                                const uint32_t x0 = x[n][i / 2][2 * (i % 2)], x1 = x[n][i / 2][2 * (i % 2) + 1];
                                if (kMin) {
                                    const uint32_t ones[4] = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
                                    if (j == 0) mma_s8_zero(cx[n], ones, x0, x1);
                                    else mma_s8(cx[n], ones, x0, x1);
                                }
#pragma unroll
                                for (int m = 0; m < kMT; ++m) {
                                    if (j == 0) mma_s8_zero(c[n][m], a[m][i], x0, x1);
                                    else mma_s8(c[n][m], a[m][i], x0, x1);
                                }
                            }
                        }
#pragma unroll
                        for (int n = 0; n < kB; ++n)
#pragma unroll
                            for (int m = 0; m < kMT; ++m)
#pragma unroll
                                for (int i = 0; i < 4; ++i) {
                                    float &to = acc[m][n0 + n][i];
                                    to = fmaf(s[m][i >> 1][k], (float)c[n][m][i], to);
                                    if (kMin) to = fmaf(l[m][i >> 1][k], (float)cx[n][i & 1], to);
                                }
                    }
                }
            }
        }
        if (++slot == kWideDepth) slot = 0;
        if (++st < stages) continue;
        st = 0;
        store_tile<kMin>(p, b0, nx, row0, min(h.height, end - row0), acc);
        row0 += tile_rows;
    }
    cp_async_wait<0>();
}

template <int kGroup, bool kMin>
cudaError_t launch_wide(const MatvecParams &p, int x_base, int num_sms, cudaStream_t st) {
    /* equal ranges of rows, so that every SM reads as much; tiles as equal as they go */
    using Stage = WideStage<kGroup, kMin>;
    constexpr int kTile = Stage::kRows * Stage::kWarps;
    WideShape h;
    h.range = std::max((p.rows + num_sms - 1) / num_sms, std::min(p.rows, kTile / 2));
    const int n = (h.range + kTile - 1) / kTile;
    h.height = (h.range + n * Stage::kWarps - 1) / (n * Stage::kWarps);
    const cudaError_t e = raise_smem((const void *)q4_wide_kernel<kGroup, kMin>, Stage::kSmem);
    if (e != cudaSuccess) return e;
    return launch_early(q4_wide_kernel<kGroup, kMin>, dim3((p.rows + h.range - 1) / h.range), Stage::kThreads, Stage::kSmem, st,
                        1, p, h, x_base);
}

/* Whether every vector begins at a 16-byte boundary and every row of scales at
 * one of a stage's copy, 512 / group bytes, of which it then holds whole ones.
 * (So columns that are no multiple of 256, but for a last stage whose groups
 * are all begun, count as not aligned.) */
inline bool all_aligned(const MatvecParams &p) {
    const int groups = (p.cols + p.group - 1) / p.group, copy = 2 * kStageBlocks * kQ4Block / p.group;
    return (uintptr_t)p.x % 16 == 0 && (p.streams == 1 || p.x_stride % 16 == 0) &&
           ((uintptr_t)p.scale | (uintptr_t)p.min | (uintptr_t)groups * 2) % copy == 0;
}

/* Which kernel for the last (at most 64) streams, from x_base on.  Measured on a
 * B200, back to back, us:
 *   streams  weights            mma    shared vectors  tcgen05
 *   16       152064x3584 g128   58     92              114
 *   16       37888x3584  g32    23.9   27.3            52.7
 *   32       37888x3584  g128   27.7   21.7            29.8
 *   32       37888x3584  g32    42.8   28.8            52.9
 *   32       3584x3584   g32    10.5   25.4            14.1
 *   64       37888x3584  g128   54.0                   30.6
 *   64       37888x3584  g32    79.1                   53.4
 *   64       3584x3584   g32    19.3                   14.5
 * so mma up to 16 streams; of 17 to 32, shared vectors where every SM has 128
 * rows and mma, 16 at a time, where it has fewer; tcgen05 beyond (and for whole
 * 64s).  What is not aligned takes mma, 16 streams at a time: 37888x3584 g128
 * 31.7 us with 16 (aligned 14.8), 62 with 32 and 124 with 64. */
template <int kGroup, bool kMin>
cudaError_t launch_streams(const MatvecParams &p, int x_base, int num_sms, cudaStream_t st) {
    const int n = p.streams - x_base;
    const bool large = (long long)p.rows * p.cols >= (long long)num_sms * 256 * 1024;
    const bool waves = (p.rows + 31) / 32 >= 2 * num_sms * 12; /* of 32 rows, 12 warps an SM */
    if (!all_aligned(p)) {
        if (n > 8) return launch_mma<2, 2, kGroup, kMin, kAny>(p, x_base, num_sms, st);
        return large ? launch_mma<2, 1, kGroup, kMin, kAny>(p, x_base, num_sms, st)
                     : launch_mma<1, 1, kGroup, kMin, kAny>(p, x_base, num_sms, st);
    }
    if (n > 32) return launch_tc<kGroup, kMin>(p, x_base, 1, num_sms, st);
    if (n > 16 && p.rows >= 128 * num_sms) return launch_wide<kGroup, kMin>(p, x_base, num_sms, st);
    if (n > 8)
        return waves ? launch_mma<2, 2, kGroup, kMin, kMany>(p, x_base, num_sms, st)
                     : launch_mma<2, 2, kGroup, kMin, kAligned>(p, x_base, num_sms, st);
    /* 32 rows a warp share its part of the vectors: fewer instructions, but half the warps.  Eight
     * streams, us: 14.0 against 18.4 for 37888x3584 g32, 11.8 against 15.6 for 3584x18944 with minima,
     * 3.3 against 2.9 for 5000x1024 */
    if (waves) return launch_mma<2, 1, kGroup, kMin, kMany>(p, x_base, num_sms, st);
    if (large) return launch_mma<2, 1, kGroup, kMin, kAligned>(p, x_base, num_sms, st);
    return launch_mma<1, 1, kGroup, kMin, kAligned>(p, x_base, num_sms, st);
}

template <int kGroup, bool kMin> cudaError_t launch_matvec(const MatvecParams &p, int num_sms, cudaStream_t st) {
    const int whole = all_aligned(p) ? p.streams / kTcStreams : 0;
    if (whole > 0) {
        const cudaError_t e = launch_tc<kGroup, kMin>(p, 0, whole, num_sms, st);
        if (e != cudaSuccess || whole * kTcStreams == p.streams) return e;
    }
    return launch_streams<kGroup, kMin>(p, whole * kTcStreams, num_sms, st);
}

template <int kGroup> cudaError_t launch_matvec(const MatvecParams &p, int num_sms, cudaStream_t st) {
    return p.min != nullptr ? launch_matvec<kGroup, true>(p, num_sms, st) : launch_matvec<kGroup, false>(p, num_sms, st);
}

/* one of the conversions' kernels by type, group and minimum */
template <typename T, int kGroup>
cudaError_t launch_convert(const ConvertParams &p, bool back, cudaStream_t st) {
    return launch_early(back ? (p.min ? dequantize_q4_kernel<T, kGroup, true> : dequantize_q4_kernel<T, kGroup, false>)
                             : (p.min ? quantize_q4_kernel<T, kGroup, true> : quantize_q4_kernel<T, kGroup, false>),
                        dim3((unsigned)q4_ctas(p.rows, p.cols)), 32 * kQ4Warps, 0, st, 1, p);
}
template <typename T> cudaError_t launch_convert(const ConvertParams &p, bool back, cudaStream_t st) {
    return p.group == 32   ? launch_convert<T, 32>(p, back, st)
           : p.group == 64 ? launch_convert<T, 64>(p, back, st)
                           : launch_convert<T, 128>(p, back, st);
}

int check_weights(const char *op, const lal_tail_q4 *w) {
    if (!w) return layer_fail(LAL_TAIL_ERR_ARG, "%s: null weights", op);
    if (w->group != 32 && w->group != 64 && w->group != 128)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: groups of %d columns (32, 64 or 128)", op, w->group);
    if (w->rows < 0 || w->cols < 1 || w->rows > kLayerMaxDim || w->cols > kLayerMaxDim)
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

int convert_q4(const char *op, const lal_tail_q4 *w, void *d_w, int64_t w_stride, int dtype, bool back, void *stream) {
    if (const int rc = check_weights(op, w)) return rc;
    const int size = dtype_size(dtype);
    if (size == 0) return layer_fail(LAL_TAIL_ERR_ARG, "%s: dtype %d", op, dtype);
    if (w->rows == 0) return LAL_TAIL_OK;
    if (!d_w) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a null pointer", op);
    if (w_stride < w->cols) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride below cols %d", op, w->cols);
    if ((uintptr_t)d_w % size != 0)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: a pointer is not aligned to its type", op);
    const WeightSpans spans(w);
    const Span values(d_w, w->rows, w->cols, w_stride, size);
    if (!values.fits) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride beyond the address space", op);
    if (spans.meets(values) || spans.meet_each_other())
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: buffers overlap", op);
    if (q4_ctas(w->rows, w->cols) > 0x7fffffffLL)
        return layer_fail(LAL_TAIL_ERR_UNSUPPORTED, "%s: weights of %d x %d", op, w->rows, w->cols);
    static const char *const names[] = {"d_w", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_w, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const ConvertParams p = {w->d_q, (__half *)w->d_scale, (__half *)w->d_min, w->rows, w->cols, w->group, d_w, w_stride,
                             ((uintptr_t)d_w | (uintptr_t)w_stride * size) % 16 == 0};
    cudaStream_t st = (cudaStream_t)stream;
    return launched(op, dtype == LAL_TAIL_F32    ? launch_convert<float>(p, back, st)
                        : dtype == LAL_TAIL_BF16 ? launch_convert<__nv_bfloat16>(p, back, st)
                                                 : launch_convert<__half>(p, back, st));
}

}  // namespace
}  // namespace lal

using namespace lal;

extern "C" {

int lal_tail_quantize_q4(const lal_tail_q4 *w, const void *d_w, int64_t w_stride, int dtype, void *stream) {
    return convert_q4("quantize_q4", w, (void *)d_w, w_stride, dtype, false, stream);
}

int lal_tail_dequantize_q4(const lal_tail_q4 *w, void *d_w, int64_t w_stride, int dtype, void *stream) {
    return convert_q4("dequantize_q4", w, d_w, w_stride, dtype, true, stream);
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
    const Span y(d_y, n_streams, w->rows, y_stride, size), x(d_xq, n_streams, w->cols, xq_stride, 1);
    if (!all_fit({y, x})) return layer_fail(LAL_TAIL_ERR_ARG, "%s: a stride beyond the address space", op);
    if (y.meets(x) ||
        y.meets(Span(d_scale_x, 1, n_streams, n_streams, 4)) || WeightSpans(w).meets(y))
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: an output overlaps another buffer", op);
    static const char *const names[] = {"d_xq", "d_scale_x", "d_y", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_xq, d_scale_x, d_y, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 6)) return rc;
    const MatvecParams p = {d_xq, xq_stride, d_scale_x, w->d_q, (const __half *)w->d_scale,
                            (const __half *)w->d_min, n_streams, w->rows, w->cols, w->group, d_y, y_stride, dtype};
    cudaStream_t st = (cudaStream_t)stream;
    const int sms = dev.num_sms();
    return launched(op, w->group == 32   ? launch_matvec<32>(p, sms, st)
                        : w->group == 64 ? launch_matvec<64>(p, sms, st)
                                         : launch_matvec<128>(p, sms, st));
}

}  // extern "C"
