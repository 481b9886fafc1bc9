// Host helpers shared by the serving operators (mk_serve.cu, mk_sample.cu, mk_attend.cu).
#pragma once
#include <cstdarg>
#include <cstdio>
#include <cstring>

#include <cuda_runtime.h>

#include "../../include/mk_b200.h"
#include "../../include/mk_serve.h"

int mk_set_error(int code, const char* text);       // mk_api.cu: the text behind mk_last_error()

namespace mkv {

inline int vfail(int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return mk_set_error(code, buf);
}
#define MKV_CUDA(call)                                                                      \
    do {                                                                                    \
        cudaError_t err__ = (call);                                                         \
        if (err__ != cudaSuccess)                                                           \
            return mkv::vfail(MK_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(err__)); \
    } while (0)

// The caller's current device, again on every way out.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device) err = cudaSetDevice(device);
        else if (err == cudaSuccess) before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};
#define MKV_DEVICE(d)                                                                                   \
    mkv::DeviceGuard guard__(d);                                                                        \
    if (guard__.err != cudaSuccess) return mkv::vfail(MK_ERR_CUDA, "device %d: %s", d, cudaGetErrorString(guard__.err))

// Launches in clusters of `ranks` CTAs along x; `chained`: the kernel waits for the one before it by itself.
template <class Kernel, class... Args>
inline cudaError_t launch(Kernel fn, dim3 grid, int threads, size_t smem, int ranks, bool chained, cudaStream_t st, const Args&... args) {
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (ranks > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = ranks;
        attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
        n++;
    }
    if (chained) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cfg.attrs = attr;
    cfg.numAttrs = n;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

inline bool aligned(uint64_t p, int n) { return (p & (uint64_t)(n - 1)) == 0; }

// What every call that takes a cache asks of it; null if it is fine.
inline const char* bad_cache(const mk_cache& c) {
    if (c.type != MKV_BF16 && c.type != MKV_F16 && c.type != MKV_INT4) return "cache type";
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return "head dim (64, 128 or 256)";
    if (c.page < 16 || (c.page & (c.page - 1))) return "page size (a power of two, 16 or more)";
    if (c.pages < 1 || c.kv_heads < 1 || (int64_t)c.pages * c.page > INT32_MAX) return "pages or KV heads";
    if (!c.k || !c.v || !aligned(c.k, 16) || !aligned(c.v, 16)) return "cache address (16-byte aligned)";
    if (c.type == MKV_INT4) return !c.k_scales || !c.v_scales || !aligned(c.k_scales, 16) || !aligned(c.v_scales, 16) ? "scales (16-byte aligned)" : nullptr;
    if (c.s_page < 0 || c.s_head < 0 || c.s_pos < 0 || c.s_page % 8 || c.s_head % 8 || c.s_pos % 8) return "cache strides (multiples of 8 elements)";
    if ((c.pages > 1 && !c.s_page) || (c.kv_heads > 1 && !c.s_head) || !c.s_pos) return "cache strides (rows on top of one another)";
    return nullptr;
}

}  // namespace mkv
