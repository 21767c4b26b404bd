/* Shared pieces of the operator kernels: element access, launches, argument errors. */
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "emmyrt_ops.h"

#define EMMY_EXPORT extern "C" __attribute__((visibility("default")))

/* records the text of a failure and returns its status */
int ops_fail(int status, const char *format, ...);
int ops_cuda(cudaError_t e, const char *what);
int ops_sm_count(int device, int *out);

/* makes `device` current for the lifetime of the object */
struct DeviceScope {
    int before = -1;
    cudaError_t status;
    explicit DeviceScope(int device) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device)
            status = cudaSetDevice(device);
        else
            before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) cudaSetDevice(before);
    }
};

/* Launches with programmatic dependent launch: every kernel here calls enter_grid() before it
 * touches memory, so its set-up overlaps the tail of the stream's previous kernel. */
template <typename... Params, typename... Args>
static inline cudaError_t launch(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, uint64_t stream,
                                 Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = (cudaStream_t)(uintptr_t)stream;
    cudaLaunchAttribute pdl = {};
    pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    pdl.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &pdl;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

static __device__ __forceinline__ void enter_grid() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

static inline bool aligned(uint64_t pointer, uint64_t bytes) { return pointer % bytes == 0; }
static inline int elem_size(int dtype) { return dtype == EMMY_OPS_F32 ? 4 : 2; }
static inline bool known_dtype(int dtype) { return dtype >= EMMY_OPS_F32 && dtype <= EMMY_OPS_BF16; }

static __device__ __forceinline__ float to_f32(float v) { return v; }
static __device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
static __device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> static __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

/* V consecutive elements that are loaded and stored in one access */
template <typename T, int V> struct alignas(sizeof(T) * V) Pack {
    T at[V];
};
