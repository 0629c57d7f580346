// Host-side launch helpers of the decoding operators, and the device-side end of their launches.
#pragma once

#include "l2d_internal.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <atomic>

namespace l2d {

constexpr int kMaxDevices = 64;

// The device's SM count, looked up once per device; a negative status if there is no such device.
inline int device_sms(int device, int *sms) {
    static std::atomic<int> known[kMaxDevices];
    if (device >= 0 && device < kMaxDevices) {
        const int n = known[device].load(std::memory_order_relaxed);
        if (n) {
            *sms = n;
            return L2D_OK;
        }
    }
    int ndev = 0;
    if (cudaGetDeviceCount(&ndev) != cudaSuccess || ndev == 0) {
        cudaGetLastError();
        return set_error(L2D_ERR_NO_DEVICE, "no CUDA device");
    }
    if (device < 0 || device >= ndev || device >= kMaxDevices)
        return set_error(L2D_ERR_INVALID, "device %d out of range", device);
    L2D_CUDA_TRY(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, device));
    known[device].store(*sms, std::memory_order_relaxed);
    return L2D_OK;
}

inline bool misaligned(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes != 0; }

// Makes `device` current for a scope.
struct OnDevice {
    int prev = -1;
    cudaError_t err = cudaSuccess;
    explicit OnDevice(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device) err = cudaSetDevice(device);
        else prev = -1;
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// Launches `k` on `stream` of the current device.  Programmatic dependent launch: after a kernel that
// releases its dependents early (those of these operators, and the GEMV's), this one's blocks become
// resident while that kernel drains, and wait for all of it with wait_for_previous() before their first
// access to global memory; after any other kernel this is an ordinary stream-ordered launch.
template <typename... P, typename... A>
cudaError_t launch_clusters(void (*k)(P...), dim3 grid, int cluster, int block, size_t smem, void *stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, static_cast<P>(args)...);
}

template <typename... P, typename... A>
cudaError_t launch(void (*k)(P...), dim3 grid, int block, size_t smem, void *stream, A... args) {
    return launch_clusters(k, grid, 1, block, smem, stream, args...);
}

// Raises a kernel's dynamic shared memory limit on the current device, once per device.  `done` is the
// kernel's own record.
template <typename K>
cudaError_t allow_smem(K *k, int bytes, int device, std::atomic<uint64_t> &done) {
    const uint64_t bit = 1ull << device;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

namespace dev {

// Waits until every kernel before this one on the stream has completed and its writes are visible, then
// lets the next kernel's blocks become resident.  In that order: a kernel that starts on the release
// finds everything before this kernel complete: only what this kernel itself writes (results, and new keys and values)
// may change under a resident block that still waits, and must not be read by loads for read-only data (__ldg, .nc).
// Weights, scales and page tables may, no kernel that releases early writes them.
__device__ __forceinline__ void wait_for_previous() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ float widen(T v);
template <>
__device__ __forceinline__ float widen<float>(float v) { return v; }
template <>
__device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T narrow(float v);
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element `i` of an array whose type is only known at run time.
__device__ __forceinline__ float load_as_float(const void *p, int dtype, int64_t i) {
    if (dtype == L2D_F32) return static_cast<const float *>(p)[i];
    if (dtype == L2D_F16) return __half2float(static_cast<const __half *>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
}

__device__ __forceinline__ void store_as(void *p, int dtype, int64_t i, float v) {
    if (dtype == L2D_F32) static_cast<float *>(p)[i] = v;
    else if (dtype == L2D_F16) static_cast<__half *>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
}

}  // namespace dev
}  // namespace l2d
