/*
 * tail_layer.h -- what the layer operators (tail_q8.cu, tail_q4.cu) share:
 * their types, the checks of their device pointers and the device that a call
 * runs on.  Not installed.
 */
#pragma once

#include "../../include/lal_tail.h"
#include "tail_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <initializer_list>

namespace lal {

inline int layer_fail(int code, const char *fmt, ...) {
    char buf[256];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return set_error(code, buf);
}

/* Rows and columns of a call: indexes rounded up to a tile stay within int. */
constexpr int kLayerMaxDim = 1 << 30;

inline int dtype_size(int dtype) {
    return dtype == LAL_TAIL_F32 ? 4 : dtype == LAL_TAIL_BF16 || dtype == LAL_TAIL_F16 ? 2 : 0;
}

/* The bytes that `rows` rows of `n` elements, `stride` elements apart, span;
 * `fits` where they end within the address space.  Rows that lie between
 * another buffer's, `step` bytes apart as those are, do not meet them. */
struct Span {
    uintptr_t lo = 0, hi = 0, width = 0, step = 0; /* step 0: one row */
    bool fits = true;
    Span() {}
    Span(const void *p, long long rows, long long n, long long stride, int size) {
        if (p == nullptr || rows < 1) return;
        const unsigned __int128 end = (uintptr_t)p + ((unsigned __int128)(rows - 1) * (unsigned long long)stride + n) * size;
        fits = end <= UINTPTR_MAX;
        lo = (uintptr_t)p;
        hi = fits ? (uintptr_t)end : UINTPTR_MAX;
        width = (uintptr_t)n * size;
        step = fits && rows > 1 ? (uintptr_t)stride * size : 0;
    }
    bool meets(const Span &o) const {
        if (!(lo < o.hi && o.lo < hi)) return false;
        const uintptr_t s = step != 0 ? step : o.step;
        if (s == 0 || (o.step != 0 && o.step != s)) return true;
        const uintptr_t at = o.lo >= lo ? (o.lo - lo) % s : (s - (lo - o.lo) % s) % s; /* of o's rows behind these */
        return at < width || o.width > s - at;
    }
};
inline bool all_fit(std::initializer_list<Span> spans) {
    for (const Span &s : spans)
        if (!s.fits) return false;
    return true;
}

/* The device whose memory p is; host memory is refused here, before a kernel
 * could fault on it. */
inline int pointer_device(const char *op, const char *what, const void *p, int *dev) {
    cudaPointerAttributes a;
    const cudaError_t e = cudaPointerGetAttributes(&a, p);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return layer_fail(LAL_TAIL_ERR_CUDA, "%s: %s: %s", op, what, cudaGetErrorString(e));
    }
    if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
        return layer_fail(LAL_TAIL_ERR_ARG, "%s: %s is not device memory", op, what);
    *dev = a.device;
    return LAL_TAIL_OK;
}

/* Makes the device of a call's memory current while the call launches, and
 * the caller's device again after it. */
class CallDevice {
    int before_ = -1, dev_ = -1;

  public:
    /* every pointer that is not null has to be memory of one device */
    int enter(const char *op, const char *const *names, const void *const *ptrs, int n) {
        int dev = -1;
        for (int i = 0; i < n; ++i) {
            if (ptrs[i] == nullptr) continue;
            int d = -1;
            const int rc = pointer_device(op, names[i], ptrs[i], &d);
            if (rc != LAL_TAIL_OK) return rc;
            if (dev >= 0 && d != dev)
                return layer_fail(LAL_TAIL_ERR_ARG, "%s: %s is on device %d, other memory on device %d",
                                  op, names[i], d, dev);
            dev = d;
        }
        int now = -1;
        cudaError_t e = cudaGetDevice(&now);
        if (e == cudaSuccess && now != dev) {
            e = cudaSetDevice(dev);
            if (e == cudaSuccess) before_ = now;
        }
        if (e != cudaSuccess) {
            (void)cudaGetLastError();
            return layer_fail(LAL_TAIL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
        }
        dev_ = dev;
        return LAL_TAIL_OK;
    }
    int num_sms() const {
        int n = 0;
        if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev_) != cudaSuccess || n < 1) {
            (void)cudaGetLastError();
            n = 148;
        }
        return n;
    }
    ~CallDevice() {
        if (before_ >= 0) cudaSetDevice(before_);
    }
};

inline int launched(const char *op, cudaError_t e) {
    if (e == cudaSuccess) return LAL_TAIL_OK;
    (void)cudaGetLastError(); /* reported here; leave no stale error behind */
    return layer_fail(LAL_TAIL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
}

#if defined(__CUDACC__)
/* Launches `kernel` (over clusters of `cluster` CTAs) so that it may begin
 * while the kernel before it on the stream ends: every thread of it calls
 * after_previous() before it reads or writes anything that a call may share,
 * and what that kernel may have written is read by ordinary loads: it is not
 * constant over this kernel's life, as __ldg wants it. */
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, A &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}
/* The kernel before has completed and its writes are visible; the next may begin. */
__device__ __forceinline__ void after_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
/* two 16-bit numbers of a word */
template <typename T> __device__ __forceinline__ void unpack16(uint32_t w, float &a, float &b);
template <> __device__ __forceinline__ void unpack16<__nv_bfloat16>(uint32_t w, float &a, float &b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
}
template <> __device__ __forceinline__ void unpack16<__half>(uint32_t w, float &a, float &b) {
    a = __half2float(__ushort_as_half((unsigned short)w));
    b = __half2float(__ushort_as_half((unsigned short)(w >> 16)));
}
#endif

}  // namespace lal
