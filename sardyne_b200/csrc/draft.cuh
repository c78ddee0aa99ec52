// What the drafted-token operators (rope_kv.cu, tree_attention.cu, sample.cu) share: the checks of
// their argument blocks and the conversions of their three value types.
#pragma once
#include "common.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <initializer_list>

namespace sdy {

inline int value_bytes(int type) { return type == T_F32 ? 4 : 2; }

// Ordinal of the device that the driver knows `p` to belong to (false: it knows no such memory).
bool pointer_device(const void *p, int *device);

struct Pointer {
    const char *name;
    const void *p;
};
// True when the kernels of the current device may use every pointer that is set: memory of that
// device, managed memory, or pinned host memory mapped there. A pointer of another device or of
// pageable host memory would fault in the kernel, so it is refused here. (The driver's one-attribute
// query answers for memory of the current device in a tenth of a microsecond, the full query in
// three times that; a call has up to nine pointers.)
inline bool device_pointers(const char *fn, std::initializer_list<Pointer> all) {
    int current = -1;
    if (!SDY_CUDA(cudaGetDevice(&current))) return false;
    for (const Pointer &x : all) {
        int at_device = -1;
        if (!x.p || (pointer_device(x.p, &at_device) && at_device == current)) continue;
        cudaPointerAttributes at;
        if (!SDY_CUDA(cudaPointerGetAttributes(&at, x.p))) return false;
        if (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeHost && at.devicePointer == x.p)) continue;
        set_error("%s: %s is not memory of the current device", fn, x.name);
        return false;
    }
    return true;
}

struct Axis {
    int64_t stride, count;
};
// True when the elements of an output with these axes (three at most) above a contiguous run of `inner`
// elements cannot coincide: each axis steps over all that the smaller ones span.
inline bool disjoint(std::initializer_list<Axis> axes, int64_t inner) {
    Axis a[3];  // sorted by stride
    int n = 0;
    for (const Axis &x : axes) {
        if (x.count <= 1 || n == 3) continue;
        int i = n++;
        for (; i > 0 && a[i - 1].stride > x.stride; i--) a[i] = a[i - 1];
        a[i] = x;
    }
    int64_t span = inner;
    for (int i = 0; i < n; i++) {
        if (a[i].stride < span || a[i].stride > (int64_t)1 << 48) return false;
        span += a[i].stride * (a[i].count - 1);
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
