// What the drafted-token operators (rope_kv.cu, tree_attention.cu, sample.cu) share: the checks of
// their argument blocks and the conversions of their three value types.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <initializer_list>
#include <vector>

namespace sdy {

inline int value_bytes(int type) { return type == T_F32 ? 4 : 2; }

// Ordinal of the device that the driver knows `p` to belong to (false: it knows no such memory).
bool pointer_device(const void *p, int *device);

// True when the kernels of the current device may use `p`: memory of that device, managed memory,
// or pinned host memory mapped there. A pointer of another device or of pageable host memory would
// fault in the kernel, so it is refused here.
// (The driver's one-attribute query answers for memory of the current device in a fraction of the
// full query's time; a call makes up to nine.)
inline bool device_pointer(const char *fn, const char *name, const void *p) {
    int at_device = -1, current = -1;
    if (pointer_device(p, &at_device) && cudaGetDevice(&current) == cudaSuccess && at_device == current) return true;
    cudaPointerAttributes at;
    if (!SDY_CUDA(cudaPointerGetAttributes(&at, p))) return false;
    int dev = -1;
    if (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeHost && at.devicePointer == p)) return true;
    if (at.type == cudaMemoryTypeDevice) {
        if (!SDY_CUDA(cudaGetDevice(&dev))) return false;
        if (at.device == dev) return true;
    }
    set_error("%s: %s is not memory of the current device", fn, name);
    return false;
}

struct Axis {
    int64_t stride, count;
};
// True when the elements of an output with these axes above a contiguous run of `inner` elements
// cannot coincide: each axis steps over all that the smaller ones span.
inline bool disjoint(std::initializer_list<Axis> axes, int64_t inner) {
    std::vector<Axis> a(axes);
    std::sort(a.begin(), a.end(), [](const Axis &x, const Axis &y) { return x.stride < y.stride; });
    int64_t span = inner;
    for (const Axis &x : a) {
        if (x.count <= 1) continue;
        if (x.stride < span || x.stride > (int64_t)1 << 48) return false;
        span += x.stride * (x.count - 1);
    }
    return true;
}
inline bool strides_fit(std::initializer_list<int64_t> s) {
    for (int64_t v : s)
        if (v < 0 || v > (int64_t)1 << 48) return false;
    return true;
}

#ifdef __CUDACC__
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f32(float x);
template <> __device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
#endif

}  // namespace sdy
