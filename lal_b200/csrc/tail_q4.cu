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

/* rint((w - m) / s) of the quotient in 64 bits: 32 bits where they cannot be
 * on the wrong side of a border (the quotient is below 16, and three roundings
 * of 2^-24 each are below 3e-6) */
__device__ __noinline__ int q4_round64(float w, float m, float s) {
    return (int)rint(((double)w - (double)m) / (double)s);
}
__device__ __forceinline__ int q4_round(float w, float m, float s, float r) {
    const float t = __fmul_rn(__fsub_rn(w, m), r);
    const float n = rintf(t);
    if (fabsf(t - n) < 0.5f - 4e-6f) return (int)n;
    return q4_round64(w, m, s);
}

/* Four elements from p on, of which n (may be below 0) exist. */
template <typename T> __device__ __forceinline__ void get4(const T *p, int n, bool aligned, float (&v)[4]) {
    if (n >= 4 && aligned) {
        if constexpr (sizeof(T) == 4) {
            const float4 f = __ldg((const float4 *)p);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
            union Raw {
                uint2 w;
                T e[4];
                __device__ Raw() {}
            } raw;
            raw.w = __ldg((const uint2 *)p);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_f32(raw.e[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? to_f32(p[i]) : 0.0f;
    }
}
template <typename T> __device__ __forceinline__ void put4(T *p, int n, bool aligned, const float (&v)[4]) {
    if (n >= 4 && aligned) {
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

/* Both directions: a lane takes a 32-bit word, columns 4u .. 4u + 3 and 16 +
 * 4u .. of a block; a warp takes kRun runs of 256 columns of a row, all their
 * loads at once. */
constexpr int kRun = 4;
constexpr int kQ4Warps = 8;
struct ConvertParams {
    uint8_t *q;
    __half *scale, *min;
    int rows, cols, group;
    void *w;
    long long w_stride;
    int aligned; /* rows of w are aligned to four elements */
};
inline long long q4_runs(int rows, int cols) { return (long long)rows * ((cols + 255) / 256); }
inline unsigned q4_ctas(int rows, int cols) {
    return (unsigned)((q4_runs(rows, cols) + kRun * kQ4Warps - 1) / (kRun * kQ4Warps));
}

template <typename T, int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kQ4Warps) quantize_q4_kernel(const ConvertParams p) {
    const int lane = threadIdx.x & 31, nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int per_row = (p.cols + 255) / 256;
    const long long run0 = ((long long)blockIdx.x * kQ4Warps + (threadIdx.x >> 5)) * kRun;
    float v[kRun][8];
    int row = (int)(run0 / per_row), seg = (int)(run0 - (long long)row * per_row);
    const int row_0 = row, seg_0 = seg;
    auto step = [&] {
        if (++seg == per_row) seg = 0, ++row;
    };
#pragma unroll
    for (int u = 0; u < kRun; ++u, step()) {
        if (row >= p.rows) break;
        const int c = seg * 256 + (lane >> 2) * 32 + (lane & 3) * 4;
        const T *w = (const T *)p.w + (size_t)row * p.w_stride + c;
        float lo[4], hi[4];
        get4(w, p.cols - c, p.aligned, lo);
        get4(w + 16, p.cols - c - 16, p.aligned, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[u][i] = lo[i], v[u][4 + i] = hi[i];
    }
    row = row_0, seg = seg_0;
#pragma unroll
    for (int u = 0; u < kRun; ++u, step()) {
        if (row >= p.rows) break;
        const int c = seg * 256 + (lane >> 2) * 32 + (lane & 3) * 4;
        /* what does not exist is 0 to the absolute largest, and left out of the extremes */
        float hi = -INFINITY, lo = INFINITY, top = 0.0f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool in = c + (i < 4 ? i : 12 + i) < p.cols;
            const float a = fabsf(v[u][i]);
            bad |= !(a <= 3.4028234663852886e38f);
            top = fmaxf(top, a);
            if (kMin && in) hi = fmaxf(hi, v[u][i]), lo = fminf(lo, v[u][i]);
        }
        int worst = bad ? 0x7f800000 : __float_as_int(top);
#pragma unroll
        for (int o = kGroup / 16; o > 0; o >>= 1) { /* 4 lanes a block */
            worst = max(worst, __shfl_xor_sync(0xffffffffu, worst, o));
            if (kMin) {
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            }
        }
        bad = worst >= 0x7f800000;
        /* Rounded outwards step by step, which is rounding outwards once: f16
         * numbers and their multiples by 7 or 15 are fp32 numbers too. */
        __half s, m = __float2half_rn(0.0f);
        if (kMin) {
            m = __float2half_rd(lo);
            s = __float2half_ru(__fdiv_ru(__fsub_ru(hi, __half2float(m)), 15.0f));
            bad |= __hisinf(m) != 0;
        } else {
            s = __float2half_ru(__fdiv_ru(__int_as_float(worst), 7.0f));
        }
        bad |= __hisinf(s) != 0;
        const float sf = __half2float(s), mf = __half2float(m);
        const bool some = !bad && sf > 0.0f;
        const float r = some ? __frcp_rn(sf) : 0.0f;
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            int q = kMin ? 0 : 8;
            if (some) {
                const int n = q4_round(v[u][i], mf, sf, r);
                q = kMin ? max(0, min(15, n)) : max(-7, min(7, n)) + 8;
            }
            word |= (uint32_t)q << (i < 4 ? 8 * i : 8 * (i - 4) + 4);
        }
        if (c / kQ4Block < nb) {
            ((uint32_t *)p.q)[((size_t)row * nb + c / kQ4Block) * 4 + (lane & 3)] = word;
            if (c % kGroup == 0) {
                const __half nan = __ushort_as_half(0x7e00);
                p.scale[(size_t)row * groups + c / kGroup] = bad ? nan : s;
                if (kMin) p.min[(size_t)row * groups + c / kGroup] = bad ? nan : m;
            }
        }
    }
}

template <typename T, int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kQ4Warps) dequantize_q4_kernel(const ConvertParams p) {
    const int lane = threadIdx.x & 31, nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int per_row = (p.cols + 255) / 256;
    const long long run0 = ((long long)blockIdx.x * kQ4Warps + (threadIdx.x >> 5)) * kRun;
    int row = (int)(run0 / per_row), seg = (int)(run0 - (long long)row * per_row);
    const int row_0 = row, seg_0 = seg;
    auto step = [&] {
        if (++seg == per_row) seg = 0, ++row;
    };
    uint32_t word[kRun];
    float s[kRun], m[kRun];
#pragma unroll
    for (int u = 0; u < kRun; ++u, step()) {
        const int c = seg * 256 + (lane >> 2) * 32;
        if (row >= p.rows) break;
        if (c >= p.cols) continue;
        word[u] = __ldg((const uint32_t *)p.q + ((size_t)row * nb + c / kQ4Block) * 4 + (lane & 3));
        s[u] = __half2float(p.scale[(size_t)row * groups + c / kGroup]);
        m[u] = kMin ? __half2float(p.min[(size_t)row * groups + c / kGroup]) : 0.0f;
    }
    row = row_0, seg = seg_0;
#pragma unroll
    for (int u = 0; u < kRun; ++u, step()) {
        const int c = seg * 256 + (lane >> 2) * 32 + (lane & 3) * 4;
        if (row >= p.rows) break;
        if (c >= p.cols) continue;
        T *w = (T *)p.w + (size_t)row * p.w_stride + c;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float q = (float)((word[u] >> (8 * i + 4 * h)) & 15u);
                /* s * q is exact in 32 bits (11 and 4 bits): one rounding */
                v[i] = kMin ? fmaf(s[u], q, m[u]) : __fmul_rn(s[u], q - 8.0f);
            }
            put4(w + 16 * h, p.cols - c - 16 * h, p.aligned, v);
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

/* ---- up to eight streams: mma.sync m16n8k32 on int8 ----
 *
 * A warp takes 16 rows and every kWarpsK-th stage of 256 columns; the rows'
 * 4-bit words and the vectors go through a ring of shared memory of its own
 * (cp.async, no barrier of the CTA until the warps' sums are joined).  A
 * block's word t of row g, shifted and masked, is that lane's part of the A
 * operand for columns 4t.. and 16 + 4t..: q - 8 in the upper half of a byte is
 * 16 (q - 8) as int8, so the dots come out 16 times too large and the scales
 * carry 1/16.  The dots of a group are exact int32 (below 2^24), and are
 * scaled and added in fp32.  With a minimum, w = s (q - 8) + (8 s + m): a
 * second product with rows of 16 gives 16 times the sums of the vectors. */
constexpr int kMmaWarps = 8;
constexpr int kMmaStreams = 8;
constexpr int kStageBlocks = 8;               /* 256 columns */
constexpr int kStageARow = kStageBlocks * 16; /* block k of row r in place k ^ (r mod 8): no bank conflicts */
constexpr int kStageA = 16 * kStageARow;
constexpr int kStageS = 2 * 16 * 2 * kStageBlocks; /* scales and minima, groups of 32 */
constexpr int kStageXRow = kStageBlocks * 32 + 16; /* rows 16 bytes apart mod 128 */
constexpr int kMmaSmem = 113 * 1024 - 1024; /* two CTAs an SM */
static_assert(kMmaWarps * 3 * (kStageA + kStageS + 8 * kStageXRow) <= kMmaSmem, "up to eight streams, three stages");
static_assert(kMmaWarps * 4 * (kStageA + kStageS + 3 * kStageXRow) <= kMmaSmem, "up to three streams, four stages");

/* 16 (or 4) bytes to shared memory, the last 16 - n of them zeros */
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

/* n (0 to 16) columns c0 .. of a vector's row to 16 bytes of shared memory,
 * zeros behind them.  Rows that are not aligned to 16 bytes are read as aligned
 * words and shifted, byte by byte at the row's ends (no byte outside the row is
 * read). */
__device__ __forceinline__ void stage_x16(uint8_t *dst, const int8_t *row, int c0, int cols, bool aligned) {
    const int n = max(0, min(16, cols - c0));
    const int8_t *src = row + (n > 0 ? c0 : 0);
    if (aligned) {
        cp_async16_l1(smem_u32(dst), src, n);
        return;
    }
    uint32_t v[4] = {0, 0, 0, 0};
    if (c0 >= 4 && c0 + 20 <= cols) {
        const unsigned off = (unsigned)((uintptr_t)src & 3);
        const uint32_t *w = (const uint32_t *)(src - off);
        uint32_t a = __ldg(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = __ldg(w + i + 1);
            v[i] = __funnelshift_r(a, b, 8 * off);
            a = b;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < n) v[i / 4] |= (uint32_t)(uint8_t)__ldg(src + i) << (8 * (i % 4));
    }
    *(uint4 *)dst = make_uint4(v[0], v[1], v[2], v[3]);
}

__device__ __forceinline__ void store_y(const MatvecParams &p, int b, int row, float v) {
    const size_t at = (size_t)b * p.y_stride + row;
    v = __fmul_rn(__ldg(p.sx + b), v);
    if (p.dtype == LAL_TAIL_F32)
        ((float *)p.y)[at] = v;
    else if (p.dtype == LAL_TAIL_BF16)
        ((__nv_bfloat16 *)p.y)[at] = __float2bfloat16_rn(v);
    else
        ((__half *)p.y)[at] = __float2half_rn(v);
}

/* ---- one or two streams: 4-way int8 dot products ----
 *
 * A warp takes kR rows; a lane takes every 32nd block of each (16 bytes, all
 * kR loads at once), eight dp4a a block and stream, and one scaled addition
 * in fp32.  The vectors lie in shared memory as two planes, columns 0-15 and
 * 16-31 of the blocks, so that a warp's 16-byte reads have no bank conflicts.
 * With few rows the K range of a row is split over warps of the CTA. */
constexpr int kDotWarps = 8;

template <int kB, int kR, bool kMin>
__global__ void __launch_bounds__(32 * kDotWarps) q4_dot_kernel(const MatvecParams p, int warps_k, int group_shift) {
    extern __shared__ __align__(16) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nb = q4_blocks(p.cols), groups = ((nb - 1) >> group_shift) + 1;
    uint4 *xs = (uint4 *)smem; /* [kB][2][nb] */
    int *sums = (int *)(smem + (size_t)kB * nb * 32); /* [kB][nb] */
    const bool x_aligned = (((uintptr_t)p.x | (uintptr_t)p.x_stride) & 15) == 0;
    for (int c = threadIdx.x; c < kB * nb * 2; c += 32 * kDotWarps) {
        const int b = kB == 1 ? 0 : c / (nb * 2), i = c - b * nb * 2;
        stage_x16((uint8_t *)(xs + (size_t)(b * 2 + (i & 1)) * nb + (i >> 1)), p.x + b * p.x_stride, i * 16, p.cols,
                  x_aligned);
    }
    const int wk = warp % warps_k;
    const int row0 = (blockIdx.x * (kDotWarps / warps_k) + warp / warps_k) * kR;
    const uint4 *q[kR];
    const __half *s[kR], *m[kR];
#pragma unroll
    for (int r = 0; r < kR; ++r) {
        const int row = min(row0 + r, p.rows - 1);
        q[r] = (const uint4 *)p.q + (size_t)row * nb;
        s[r] = p.scale + (size_t)row * groups;
        m[r] = p.min + (size_t)row * groups;
    }
    cp_async_commit();
    cp_async_wait<0>();
    __syncthreads();
    if (kMin) {
        for (int c = threadIdx.x; c < kB * nb; c += 32 * kDotWarps) {
            const int b = kB == 1 ? 0 : c / nb, i = c - b * nb;
            const uint4 lo = xs[(size_t)(b * 2) * nb + i], hi = xs[(size_t)(b * 2 + 1) * nb + i];
            int sum = 0;
            for (uint32_t v : {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w}) sum = __dp4a((int)v, 0x10101010, sum);
            sums[c] = sum; /* 16 times the sum, as the dots */
        }
        __syncthreads();
    }
    float acc[kR][kB] = {};
    constexpr int kU = kR >= 4 ? 1 : 4 / kR; /* blocks of a row in flight */
    if (row0 < p.rows) {
        for (int k0 = wk * 32 + lane; k0 < nb; k0 += 32 * kU * warps_k) {
            uint4 v[kU][kR];
            float sc[kU][kR], lo[kU][kR];
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int k = k0 + 32 * u * warps_k;
#pragma unroll
                for (int r = 0; r < kR; ++r) {
                    if (k >= nb) break;
                    v[u][r] = __ldg(q[r] + k);
                    sc[u][r] = __half2float(__ldg(s[r] + (k >> group_shift)));
                    if (kMin) lo[u][r] = __half2float(__ldg(m[r] + (k >> group_shift)));
                }
            }
#pragma unroll
            for (int u = 0; u < kU; ++u) {
                const int k = k0 + 32 * u * warps_k;
                if (k >= nb) break;
#pragma unroll
                for (int b = 0; b < kB; ++b) {
                    const uint4 xl = xs[(size_t)(b * 2) * nb + k], xh = xs[(size_t)(b * 2 + 1) * nb + k];
                    const uint32_t x0[4] = {xl.x, xl.y, xl.z, xl.w}, x1[4] = {xh.x, xh.y, xh.z, xh.w};
                    const float sum = kMin ? (float)sums[b * nb + k] : 0.0f;
#pragma unroll
                    for (int r = 0; r < kR; ++r) {
                        const uint32_t w[4] = {v[u][r].x, v[u][r].y, v[u][r].z, v[u][r].w};
                        int dot = 0;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            dot = __dp4a((int)(((w[i] << 4) & 0xf0f0f0f0u) ^ 0x80808080u), (int)x0[i], dot);
                            dot = __dp4a((int)((w[i] & 0xf0f0f0f0u) ^ 0x80808080u), (int)x1[i], dot);
                        }
                        acc[r][b] = fmaf(sc[u][r], (float)dot, acc[r][b]);
                        if (kMin) acc[r][b] = fmaf(fmaf(8.0f, sc[u][r], lo[u][r]), sum, acc[r][b]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < kR; ++r)
#pragma unroll
        for (int b = 0; b < kB; ++b) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) acc[r][b] += __shfl_xor_sync(0xffffffffu, acc[r][b], o);
            acc[r][b] *= 0.0625f;
        }
    if (warps_k == 1) {
        if (lane == 0)
#pragma unroll
            for (int r = 0; r < kR; ++r)
#pragma unroll
                for (int b = 0; b < kB; ++b)
                    if (row0 + r < p.rows) store_y(p, b, row0 + r, acc[r][b]);
        return;
    }
    /* the warps of a row, in order */
    __shared__ float part[kDotWarps][kR * kB];
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < kR * kB; ++i) part[warp][i] = acc[i / kB][i % kB];
    __syncthreads();
    const int tiles = kDotWarps / warps_k;
    for (int i = threadIdx.x; i < tiles * kR * kB; i += 32 * kDotWarps) {
        const int tile = i / (kR * kB), j = i % (kR * kB);
        const int row = (blockIdx.x * tiles + tile) * kR + j / kB;
        float sum = 0.0f;
        for (int w = 0; w < warps_k; ++w) sum += part[tile * warps_k + w][j];
        if (row < p.rows) store_y(p, j % kB, row, sum);
    }
}

constexpr int kDotSmem = 96 * 1024;

inline int dot_smem(const MatvecParams &p, int streams) {
    const long long n = (long long)streams * q4_blocks(p.cols) * (32 + (p.min ? 4 : 0));
    return n > kDotSmem ? -1 : (int)n;
}

template <int kB, int kR, bool kMin> cudaError_t launch_dot(const MatvecParams &p, int num_sms, cudaStream_t st) {
    const int nb = q4_blocks(p.cols), tiles = (p.rows + kR - 1) / kR;
    int wk = 1;
    while (wk < kDotWarps && 32 * wk < nb && (long long)tiles * wk < 16LL * num_sms) wk *= 2;
    const void *fn = (const void *)q4_dot_kernel<kB, kR, kMin>;
    cudaError_t e = raise_smem(fn, kDotSmem);
    if (e != cudaSuccess) return e;
    const int per = kDotWarps / wk, shift = p.group == 32 ? 0 : p.group == 64 ? 1 : 2;
    q4_dot_kernel<kB, kR, kMin><<<(tiles + per - 1) / per, 32 * kDotWarps, dot_smem(p, kB), st>>>(p, wk, shift);
    return cudaGetLastError();
}

template <int kB> cudaError_t launch_dot(const MatvecParams &p, int num_sms, cudaStream_t st) {
    /* rows a warp: four once that leaves 24 warps an SM */
    const int per_warp = p.rows / (24 * num_sms);
    if (p.min)
        return per_warp >= 4   ? launch_dot<kB, 4, true>(p, num_sms, st)
               : per_warp >= 2 ? launch_dot<kB, 2, true>(p, num_sms, st)
                               : launch_dot<kB, 1, true>(p, num_sms, st);
    return per_warp >= 4   ? launch_dot<kB, 4, false>(p, num_sms, st)
           : per_warp >= 2 ? launch_dot<kB, 2, false>(p, num_sms, st)
                           : launch_dot<kB, 1, false>(p, num_sms, st);
}

template <int kGroup, bool kMin, int kDepth>
__global__ void __launch_bounds__(32 * kMmaWarps, 2) q4_mma_kernel(const MatvecParams p, int warps_k) {
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int kPer = kGroup / kQ4Block;             /* blocks of a group */
    constexpr int kGroups = kStageBlocks / kPer;        /* groups of a stage */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int wk = warp % warps_k;
    const int row0 = (blockIdx.x * (kMmaWarps / warps_k) + warp / warps_k) * 16;
    const int b0 = blockIdx.y * kMmaStreams, nx = min(kMmaStreams, p.streams - b0);
    const int nb = q4_blocks(p.cols), groups = (p.cols + kGroup - 1) / kGroup;
    const int stages = (nb + kStageBlocks - 1) / kStageBlocks;
    const int stage_bytes = kStageA + kStageS + min(kMmaStreams, p.streams) * kStageXRow;
    uint8_t *ring = smem + warp * kDepth * stage_bytes;

    float acc[4] = {};
    const bool live = row0 < p.rows;
    if (live) {
        /* this lane's share of a stage: four 16-byte blocks of weights, up to four of the vectors */
        const uint8_t *qsrc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            qsrc[j] = p.q + ((size_t)min(row0 + (lane >> 3) + 4 * j, p.rows - 1) * nb + (lane & 7)) * 16;
        const uint32_t qdst = (lane >> 3) * kStageARow + ((lane & 7) ^ (lane >> 3)) * 16;
        const int8_t *xrow = p.x + (size_t)(b0 + min(lane >> 4, nx - 1)) * p.x_stride;
        const bool x_aligned = (((uintptr_t)p.x | (uintptr_t)p.x_stride) & 15) == 0;
        /* scales of lane's row, kGroups a stage: one copy where every row's are aligned to it */
        const unsigned short *ssrc = (const unsigned short *)(lane < 16 ? p.scale : p.min) +
                                     (size_t)min(row0 + (lane & 15), p.rows - 1) * groups;
        const bool s_aligned = ((((uintptr_t)p.scale | (kMin ? (uintptr_t)p.min : 0) | (uintptr_t)(groups * 2)) & (2 * kGroups - 1)) == 0);
        auto load = [&](int st, int slot) {
            uint8_t *a = ring + slot * stage_bytes;
            const int k0 = st * kStageBlocks;
            const bool in = k0 + (lane & 7) < nb;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                cp_async16(smem_u32(a + ((qdst + 4 * j * kStageARow) ^ (j & 1 ? 64 : 0))), in ? qsrc[j] + (size_t)k0 * 16 : p.q, in ? 16 : 0);
            if (kMin || lane < 16) {
                /* [16 rows][kGroups] scales, then minima */
                unsigned short *d = (unsigned short *)(a + kStageA) + lane * kGroups;
                const int g0 = st * kGroups;
                if (s_aligned && g0 + kGroups <= groups) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(smem_u32(d)), "l"(ssrc + g0),
                                 "n"(2 * kGroups)
                                 : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < kGroups; ++i)
                        if (g0 + i < groups) d[i] = __ldg(ssrc + g0 + i);
                }
            }
            const int8_t *xr = xrow;
            for (int c = lane; c < nx * 16; c += 32, xr += 2 * p.x_stride)
                stage_x16(a + kStageA + kStageS + (c >> 4) * kStageXRow + (c & 15) * 16, xr,
                          k0 * kQ4Block + (c & 15) * 16, p.cols, x_aligned);
        };
#pragma unroll
        for (int i = 0; i < kDepth - 1; ++i) {
            if (wk + i * warps_k < stages) load(wk + i * warps_k, i);
            cp_async_commit();
        }
        int slot = 0;
        const int xg = min(g, nx - 1); /* vectors that are not there: any, their sums are dropped */
        for (int st = wk; st < stages; st += warps_k) {
            cp_async_wait<kDepth - 2>();
            __syncwarp();
            {
                const int next = st + (kDepth - 1) * warps_k;
                if (next < stages) load(next, slot == 0 ? kDepth - 1 : slot - 1);
                cp_async_commit();
            }
            const uint8_t *a = ring + slot * stage_bytes + g * kStageARow + 4 * t;
            const uint32_t turn = g * 16;
            const uint8_t *x = ring + slot * stage_bytes + kStageA + kStageS + xg * kStageXRow + 4 * t;
            /* the scales (and minima) of rows g and g + 8 */
            using Pack = std::conditional_t<kGroups == 8, uint4, std::conditional_t<kGroups == 4, uint2, uint32_t>>;
            const Pack *sc = (const Pack *)(ring + slot * stage_bytes + kStageA) + g;
            union Row {
                Pack all;
                __half one[kGroups];
                __device__ Row() {}
            } scale[2], low[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                scale[h].all = sc[8 * h];
                if (kMin) low[h].all = sc[16 + 8 * h];
            }
            const int left = nb - st * kStageBlocks; /* blocks from this stage on */
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr) {
                if (gr * kPer >= left) break;
                int c[4] = {}, cx[4] = {};
#pragma unroll
                for (int k = gr * kPer; k < (gr + 1) * kPer; ++k) {
                    /* blocks behind the row's end hold zeros in the vectors */
                    const uint32_t w0 = *(const uint32_t *)(a + (k * 16 ^ turn)),
                                   w1 = *(const uint32_t *)(a + 8 * kStageARow + (k * 16 ^ turn));
                    const uint32_t x0 = *(const uint32_t *)(x + k * 32), x1 = *(const uint32_t *)(x + k * 32 + 16);
                    const uint32_t av[4] = {((w0 << 4) & 0xf0f0f0f0u) ^ 0x80808080u, ((w1 << 4) & 0xf0f0f0f0u) ^ 0x80808080u,
                                            (w0 & 0xf0f0f0f0u) ^ 0x80808080u, (w1 & 0xf0f0f0f0u) ^ 0x80808080u};
                    mma_s8(c, av, x0, x1);
                    if (kMin) {
                        const uint32_t ones[4] = {0x10101010u, 0x10101010u, 0x10101010u, 0x10101010u};
                        mma_s8(cx, ones, x0, x1);
                    }
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float s = __half2float(scale[h].one[gr]);
#pragma unroll
                    for (int i = 0; i < 2; ++i) acc[2 * h + i] = fmaf(s, (float)c[2 * h + i], acc[2 * h + i]);
                    if (kMin) {
                        const float m = fmaf(8.0f, s, __half2float(low[h].one[gr]));
#pragma unroll
                        for (int i = 0; i < 2; ++i) acc[2 * h + i] = fmaf(m, (float)cx[i], acc[2 * h + i]);
                    }
                }
            }
            slot = slot + 1 == kDepth ? 0 : slot + 1;
        }
        cp_async_wait<0>();
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] *= 0.0625f;
    }
    if (warps_k == 1) {
        if (live)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = row0 + g + (i >> 1) * 8, b = 2 * t + (i & 1);
                if (row < p.rows && b < nx) store_y(p, b0 + b, row, acc[i]);
            }
        return;
    }
    /* the warps of a row tile, in order; their sums take the rings' place */
    __syncthreads();
    float(*part)[16 * kMmaStreams] = (float(*)[16 * kMmaStreams])smem;
#pragma unroll
    for (int i = 0; i < 4; ++i) part[warp][(2 * t + (i & 1)) * 16 + g + (i >> 1) * 8] = acc[i];
    __syncthreads();
    const int tiles = kMmaWarps / warps_k;
    for (int i = threadIdx.x; i < tiles * 16 * nx; i += 32 * kMmaWarps) {
        const int r = i & 15, b = (i >> 4) % nx, tile = (i >> 4) / nx;
        const int row = (blockIdx.x * tiles + tile) * 16 + r;
        if (row >= p.rows) continue;
        float sum = 0.0f;
        for (int w = 0; w < warps_k; ++w) sum += part[tile * warps_k + w][b * 16 + r];
        store_y(p, b0 + b, row, sum);
    }
}

template <int kGroup, bool kMin, int kDepth>
cudaError_t launch_mma(const MatvecParams &p, int num_sms, cudaStream_t st) {
    /* warps of a row tile: enough that the tiles' warps fill the SMs (16 a SM),
     * no more than there are stages */
    const int tiles = (p.rows + 15) / 16, stages = (q4_blocks(p.cols) + kStageBlocks - 1) / kStageBlocks;
    int wk = 1;
    while (wk < kMmaWarps && 2 * wk <= stages && (long long)tiles * wk < 16LL * num_sms) wk *= 2;
    const int smem = kMmaWarps * kDepth * (kStageA + kStageS + std::min(kMmaStreams, p.streams) * kStageXRow);
    const void *fn = (const void *)q4_mma_kernel<kGroup, kMin, kDepth>;
    cudaError_t e = raise_smem(fn, kMmaSmem);
    if (e != cudaSuccess) return e;
    const int per = kMmaWarps / wk;
    q4_mma_kernel<kGroup, kMin, kDepth>
        <<<dim3((tiles + per - 1) / per, (p.streams + kMmaStreams - 1) / kMmaStreams), 32 * kMmaWarps, smem, st>>>(p, wk);
    return cudaGetLastError();
}

/* ---- nine streams and more: tcgen05.mma kind::i8 ----
 *
 * A CTA takes tiles of 128 rows by up to kN streams.  The weights are the A
 * operand and lie in tensor memory: a thread of the four unpacking warps has a
 * row, reads its 16-byte blocks from a ring of its warp's own (cp.async) and
 * stores 16 (q - 8) as int8, eight columns of tensor memory a block.  The
 * vectors are the B operand, in shared memory with the 128-byte swizzle.  One
 * thread issues the products, a group of columns at a time into one of kD
 * accumulators; eight warps read a finished one (int32, exact), scale it by
 * the row's scale of the group and add it in fp32 registers, while the next
 * groups are multiplied.  So every scale is applied in fp32, the weights are
 * read once, and only the unpacked weights' 8-bit form is ever written on the
 * chip.  With few tiles, the K range of a tile is split over a cluster of
 * CTAs, whose sums are exchanged and added in order over distributed shared
 * memory.
 *
 * Every wait is bounded; one that runs out makes the tile's results NaN. */
constexpr int kTcUnpack = 8, kTcEpi = 16, kTcLoad = 4;
constexpr int kTcIssue = kTcUnpack + kTcEpi; /* the warp that issues the products */
constexpr int kTcWarps = kTcIssue + 1 + kTcLoad;
constexpr int kTcD = 4;        /* accumulators */
constexpr int kTcWDepth = 6;   /* stages of a warp's weight ring */
constexpr int kTcXDepth = 4;   /* stages of the vectors */
constexpr int kTcHalf = kStageBlocks / 2;         /* blocks of a stage that an unpacking warp has */
constexpr int kTcWStage = 32 * kTcHalf * 16;
constexpr int kTcMaxSplit = 8;

struct TcShared {
    uint64_t a_full[2], a_empty[2], x_full[kTcXDepth], x_empty[kTcXDepth], d_full[kTcD], d_empty[kTcD], drain;
    uint32_t tmem;
    int abort, never;
};

__host__ __device__ constexpr int tc_x_stage(int n) { return n * kStageBlocks * 32; }
__host__ __device__ constexpr int tc_sum_bytes(int n, int group) { return kTcXDepth * (kStageBlocks * 32 / group) * n * 4; }
template <int kN, int kGroup, bool kMin> constexpr int tc_smem() {
    return 1024 + kTcUnpack * kTcWDepth * kTcWStage + kTcXDepth * tc_x_stage(kN) + (kMin ? tc_sum_bytes(kN, kGroup) : 0);
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
template <int kCount> __device__ __forceinline__ void tc_load(uint32_t at, int (&r)[kCount]) {
    if constexpr (kCount == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                     "%14, %15}, [%16];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                       "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                     : "r"(at));
    else if constexpr (kCount == 8)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                     : "r"(at));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                     : "r"(at));
    /* the wait names the registers, so that nothing reads them before it */
    if constexpr (kCount == 16)
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                       "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                     :
                     : "memory");
    else if constexpr (kCount == 8)
        asm volatile("tcgen05.wait::ld.sync.aligned;"
                     : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                     :
                     : "memory");
    else
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]) : : "memory");
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

template <int kN, int kGroup, bool kMin>
__global__ void __launch_bounds__(32 * kTcWarps, 1) q4_tc_kernel(const MatvecParams p, int splits, int x_base) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ TcShared sh;
    constexpr int kPer = kGroup / kQ4Block, kGroups = kStageBlocks / kPer; /* blocks a group, groups a stage */
    constexpr int kMine = kN / (kTcEpi / 4);                               /* streams of an epilogue warp */
    uint8_t *smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t *xring = smem;                                      /* kTcXDepth stages of two swizzled tiles */
    uint8_t *wring = xring + kTcXDepth * tc_x_stage(kN);        /* of each unpacking warp */
    float *xsums = (float *)(wring + kTcUnpack * kTcWDepth * kTcWStage); /* [kTcXDepth][kGroups][kN] */
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
        for (int i = 0; i < 2; ++i) mbar_init(&sh.a_full[i], kTcUnpack), mbar_init(&sh.a_empty[i], 1);
        for (int i = 0; i < kTcXDepth; ++i)
            mbar_init(&sh.x_full[i], kTcLoad), mbar_init(&sh.x_empty[i], 1 + (kMin ? kTcEpi : 0));
        for (int i = 0; i < kTcD; ++i) mbar_init(&sh.d_full[i], 1), mbar_init(&sh.d_empty[i], kTcEpi);
        mbar_init(&sh.drain, 1);
        sh.abort = sh.never = 0;
        mbar_fence_init();
    }
    constexpr int kCols = 128 + kTcD * kN <= 256 ? 256 : 512;
    if (warp == kTcIssue) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)), "n"(kCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem, tmem_d = tmem + 128; /* two A operands of 64 columns, then the accumulators */

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
            const int buf = it & 1;
            if (it >= 2 && !tc_wait(&sh.a_empty[buf], ((it >> 1) & 1) ^ 1, abort_flag)) {
                *abort_flag = 1;
                break;
            }
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int i = 0; i < kTcHalf; ++i) {
                const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    o[j] = ((w[j] << 4) & 0xf0f0f0f0u) ^ 0x80808080u;
                    o[4 + j] = (w[j] & 0xf0f0f0f0u) ^ 0x80808080u;
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
        /* a row's scales (and minima) of a stage, one load where all rows' are aligned to it */
        using Pack = std::conditional_t<kGroups == 8, uint4, std::conditional_t<kGroups == 4, uint2, uint32_t>>;
        union Row {
            Pack all;
            unsigned short one[kGroups];
            __device__ Row() {}
        } scale, low, scale_next, low_next;
        const bool s_aligned =
            (((uintptr_t)p.scale | (kMin ? (uintptr_t)p.min : 0) | (uintptr_t)(groups * 2)) & (2 * kGroups - 1)) == 0;
        TcWalk ahead(tile0, st0);
        auto load_scales = [&] {
            if (ahead.n < total) {
                const int row = min(ahead.tile * 128 + quad * 32 + lane, p.rows - 1), g0 = ahead.st * kGroups;
                const size_t at = (size_t)row * groups + g0;
                if (s_aligned && g0 + kGroups <= groups) {
                    scale_next.all = __ldg((const Pack *)(p.scale + at));
                    if (kMin) low_next.all = __ldg((const Pack *)(p.min + at));
                } else {
#pragma unroll
                    for (int i = 0; i < kGroups; ++i) {
                        scale_next.one[i] = g0 + i < groups ? __ldg((const unsigned short *)p.scale + at + i) : 0;
                        if (kMin) low_next.one[i] = g0 + i < groups ? __ldg((const unsigned short *)p.min + at + i) : 0;
                    }
                }
            }
            ahead.next(st0, st1, tile_step);
        };
        load_scales();
        bool ok = true;
        TcWalk at(tile0, st0);
        for (int d = 0, xs = 0, xs_round = 0; at.n < total; at.next(st0, st1, tile_step)) {
            if (at.st == st0)
#pragma unroll
                for (int j = 0; j < kMine; ++j) acc[j] = 0.0f;
            scale.all = scale_next.all;
            if (kMin) low.all = low_next.all;
            load_scales();
            if (kMin && !tc_wait(&sh.x_full[xs], xs_round & 1, abort_flag)) ok = false;
#pragma unroll
            for (int gr = 0; gr < kGroups; ++gr, ++d) {
                const int buf = d % kTcD;
                if (ok && !tc_wait(&sh.d_full[buf], (d / kTcD) & 1, abort_flag)) ok = false;
                if (!__all_sync(0xffffffffu, ok)) {
                    ok = false;
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                int c[kMine];
                tc_load<kMine>(lanes + buf * kN, c);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.d_empty[buf]);
                const float s = __half2float(__ushort_as_half(scale.one[gr]));
#pragma unroll
                for (int j = 0; j < kMine; ++j) acc[j] = fmaf(s, (float)c[j], acc[j]);
                if (kMin) {
                    const float m = fmaf(8.0f, s, __half2float(__ushort_as_half(low.one[gr])));
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
            if (!ok) break;
            if (kMin) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.x_empty[xs]);
                if (++xs == kTcXDepth) xs = 0, ++xs_round;
            }
            if (splits == 1 && at.st == st1 - 1) {
                const int row = at.tile * 128 + quad * 32 + lane;
                if (row < p.rows)
#pragma unroll
                    for (int j = 0; j < kMine; ++j)
                        if (part * kMine + j < nx) store_y(p, b0 + part * kMine + j, row, 0.0625f * acc[j]);
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
                const int buf = it & 1;
                if (!tc_wait(&sh.x_full[xs], xs_round & 1, abort_flag) ||
                    !tc_wait(&sh.a_full[buf], (it >> 1) & 1, abort_flag)) {
                    *abort_flag = 1;
                    break;
                }
                tc_fence_after();
                const uint32_t xt = x0 + xs * (tc_x_stage(kN) >> 4);
#pragma unroll
                for (int gr = 0; gr < kGroups; ++gr, ++d) {
                    const int acc_buf = d % kTcD;
                    if (d >= kTcD && !tc_wait(&sh.d_empty[acc_buf], ((d / kTcD) & 1) ^ 1, abort_flag)) {
                        *abort_flag = 1;
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll
                    for (int k = gr * kPer; k < (gr + 1) * kPer; ++k)
                        tc_mma_i8_ta(tmem_d + acc_buf * kN, tmem + buf * 64 + k * 8, xt + (k / 4) * (kN * 128 >> 4) + (k % 4) * 2,
                                     tc_idesc(kN), k != gr * kPer);
                    tc_commit(&sh.d_full[acc_buf]);
                }
                tc_commit(&sh.a_empty[buf]);
                tc_commit(&sh.x_empty[xs]);
                if (++xs == kTcXDepth) xs = 0, ++xs_round;
            }
            /* every product issued is complete before the tensor memory is freed */
            tc_commit(&sh.drain);
            if (!tc_wait(&sh.drain, 0u, never)) *abort_flag = 1;
        }
    } else {
        /* ---- vectors, and (with minima) their sums ---- */
        const int lw = warp - kTcIssue - 1;
        const bool x_aligned = (((uintptr_t)p.x | (uintptr_t)p.x_stride) & 15) == 0;
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
                uint8_t *dst = xring + xs * tc_x_stage(kN) + d0;
                const int8_t *x = x0;
                if (x_aligned && c0 + 16 <= p.cols) {
                    x += c0;
                    for (int n = n0; n < nx; n += 2 * kTcLoad, x += x_step, dst += 1024) cp_async16_l1(smem_u32(dst), x, 16);
                } else {
                    for (int n = n0; n < nx; n += 2 * kTcLoad, x += x_step, dst += 1024) stage_x16(dst, x, c0, p.cols, x_aligned);
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
                /* 16 times the sum of each group of this warp's rows */
                const uint8_t *st = xring + xs * tc_x_stage(kN);
                for (int i = lane; i < kN / kTcLoad * kGroups; i += 32) {
                    const int gr = i % kGroups, pair = i / kGroups;
                    const int n = (pair >> 1) * 2 * kTcLoad + lw * 2 + (pair & 1);
                    if (n >= nx) continue;
                    int sum = 0;
#pragma unroll
                    for (int j = 0; j < kPer * 2; ++j) {
                        const int c = gr * kPer * 2 + j;
                        const uint4 v = *(const uint4 *)(st + (c >> 3) * kN * 128 + n * 128 + (((c & 7) ^ (n & 7)) << 4));
                        sum = __dp4a((int)v.x, 0x10101010, __dp4a((int)v.y, 0x10101010, sum));
                        sum = __dp4a((int)v.z, 0x10101010, __dp4a((int)v.w, 0x10101010, sum));
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
            store_y(p, b0 + n, row, 0.0625f * sum);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kTcIssue) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols) : "memory");
    }
}

template <int kN, int kGroup, bool kMin>
cudaError_t launch_tc(const MatvecParams &p, int x_base, int chunks, int num_sms, cudaStream_t st) {
    const int tiles = (p.rows + 127) / 128, stages = (q4_blocks(p.cols) + kStageBlocks - 1) / kStageBlocks;
    /* CTAs of a tile: as many as leave each an SM and two stages */
    int splits = 1;
    while (splits < kTcMaxSplit && (long long)tiles * chunks * splits * 2 <= num_sms && splits * 4 <= stages) splits *= 2;
    const void *fn = (const void *)q4_tc_kernel<kN, kGroup, kMin>;
    constexpr int smem = tc_smem<kN, kGroup, kMin>();
    cudaError_t e = raise_smem(fn, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(splits > 1 ? tiles * splits : std::min(tiles, num_sms)), (unsigned)chunks);
    cfg.blockDim = dim3(32 * kTcWarps);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, q4_tc_kernel<kN, kGroup, kMin>, p, splits, x_base);
}

template <int kGroup, bool kMin>
cudaError_t launch_tc_all(const MatvecParams &p, int num_sms, cudaStream_t st) {
    /* whole chunks of 64 streams, then the smallest tile that has the rest */
    const int whole = p.streams / 64, rest = p.streams % 64;
    if (whole > 0) {
        const cudaError_t e = launch_tc<64, kGroup, kMin>(p, 0, whole, num_sms, st);
        if (e != cudaSuccess || rest == 0) return e;
    }
    return rest <= 16   ? launch_tc<16, kGroup, kMin>(p, whole * 64, 1, num_sms, st)
           : rest <= 32 ? launch_tc<32, kGroup, kMin>(p, whole * 64, 1, num_sms, st)
                        : launch_tc<64, kGroup, kMin>(p, whole * 64, 1, num_sms, st);
}

template <int kGroup, bool kMin> cudaError_t launch_matvec(const MatvecParams &p, int num_sms, cudaStream_t st) {
    if (p.streams > kMmaStreams) return launch_tc_all<kGroup, kMin>(p, num_sms, st);
    return p.streams <= 3 ? launch_mma<kGroup, kMin, 4>(p, num_sms, st) : launch_mma<kGroup, kMin, 3>(p, num_sms, st);
}

template <int kGroup> cudaError_t launch_matvec(const MatvecParams &p, int num_sms, cudaStream_t st) {
    return p.min != nullptr ? launch_matvec<kGroup, true>(p, num_sms, st) : launch_matvec<kGroup, false>(p, num_sms, st);
}

/* one of the conversions' kernels by type, group and minimum */
template <typename T, int kGroup>
cudaError_t launch_convert(const ConvertParams &p, bool back, cudaStream_t st) {
    const unsigned n = q4_ctas(p.rows, p.cols);
    if (back && p.min) dequantize_q4_kernel<T, kGroup, true><<<n, 32 * kQ4Warps, 0, st>>>(p);
    else if (back) dequantize_q4_kernel<T, kGroup, false><<<n, 32 * kQ4Warps, 0, st>>>(p);
    else if (p.min) quantize_q4_kernel<T, kGroup, true><<<n, 32 * kQ4Warps, 0, st>>>(p);
    else quantize_q4_kernel<T, kGroup, false><<<n, 32 * kQ4Warps, 0, st>>>(p);
    return cudaGetLastError();
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
    if (spans.meets(Span(d_w, w->rows, w->cols, w_stride, size)) || spans.meet_each_other())
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: buffers overlap", op);
    if (q4_runs(w->rows, w->cols) / (kRun * kQ4Warps) >= 0x7fffffffLL)
        return layer_fail(LAL_TAIL_ERR_UNSUPPORTED, "%s: weights of %d x %d", op, w->rows, w->cols);
    static const char *const names[] = {"d_w", "d_q", "d_scale", "d_min"};
    const void *ptrs[] = {d_w, w->d_q, w->d_scale, w->d_min};
    CallDevice dev;
    if (const int rc = dev.enter(op, names, ptrs, 4)) return rc;
    const ConvertParams p = {w->d_q, (__half *)w->d_scale, (__half *)w->d_min, w->rows, w->cols, w->group, d_w, w_stride,
                             ((uintptr_t)d_w | (uintptr_t)w_stride * size) % (4 * size) == 0};
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
    const Span y(d_y, n_streams, w->rows, y_stride, size);
    if (y.meets(Span(d_xq, n_streams, w->cols, xq_stride, 1)) ||
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
    if (n_streams == 1 && dot_smem(p, n_streams) >= 0) return launched(op, launch_dot<1>(p, sms, st));
    return launched(op, w->group == 32   ? launch_matvec<32>(p, sms, st)
                        : w->group == 64 ? launch_matvec<64>(p, sms, st)
                                         : launch_matvec<128>(p, sms, st));
}

}  // extern "C"
