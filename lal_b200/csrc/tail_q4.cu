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

#include <algorithm>
#include <type_traits>

using namespace lal;

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

__device__ __forceinline__ uint32_t smem_u32(const void *p) {
    return (uint32_t)__cvta_generic_to_shared(p);
}
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

template <int kGroup, bool kMin> cudaError_t launch_matvec(const MatvecParams &p, int num_sms, cudaStream_t st) {
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
