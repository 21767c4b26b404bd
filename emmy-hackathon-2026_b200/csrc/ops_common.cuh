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

/* a pair of f32 that one instruction works on */
struct Two {
    uint64_t v;
    __device__ __forceinline__ Two() {}
    __device__ __forceinline__ explicit Two(uint64_t both) : v(both) {}
    __device__ __forceinline__ Two(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ float2 get() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Two operator*(Two a, Two b) {
    Two d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
    Two d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
    return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
    Two d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return d;
}

/* a / b for a below 2^31 without a division: the upper half of a * inverse, shifted (exact: inverse = ceil(2^(31 + s) / b) with
 * 2^s >= b); b = 1: inverse = 0 */
struct Divisor {
    uint32_t by, inverse, shift;
    Divisor(uint32_t b = 1) : by(b), inverse(0), shift(0) {
        if (b == 1) return;
        uint32_t s = 1;
        while ((1u << s) < b) ++s;
        inverse = (uint32_t)((((uint64_t)1 << (31 + s)) + b - 1) / b);
        shift = s - 1;
    }
    __device__ __forceinline__ uint32_t divides(uint32_t a) const { return inverse ? __umulhi(a, inverse) >> shift : a; }
};

/* the values of an access in f32, and back with one rounding each */
template <typename T, int V> static __device__ __forceinline__ void unpack(const Pack<T, V> &q, float (&f)[V]) {
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = to_f32(q.at[i]);
}
template <int V> static __device__ __forceinline__ void unpack(const Pack<__nv_bfloat16, V> &q, float (&f)[V]) {
    if (V % 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = to_f32(q.at[i]);
    } else {
        const uint32_t *u = (const uint32_t *)&q;
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
}
template <int V> static __device__ __forceinline__ void pack(const float (&f)[V], Pack<float, V> &q) {
#pragma unroll
    for (int i = 0; i < V; ++i) q.at[i] = f[i];
}
template <int V> static __device__ __forceinline__ void pack(const float (&f)[V], Pack<__half, V> &q) {
    if (V % 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) q.at[i] = __float2half_rn(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) ((__half2 *)&q)[i] = __floats2half2_rn(f[2 * i], f[2 * i + (V > 1)]);
    }
}
template <int V> static __device__ __forceinline__ void pack(const float (&f)[V], Pack<__nv_bfloat16, V> &q) {
    if (V % 2) {
#pragma unroll
        for (int i = 0; i < V; ++i) q.at[i] = __float2bfloat16_rn(f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) ((__nv_bfloat162 *)&q)[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + (V > 1)]);
    }
}

/* v / s, correctly rounded, with r = 1 / s correctly rounded.  By Markstein's theorem (IBM J. Res. Dev. 34, 1990) the
 * quotient q0 = v r is put right by one step, q0 + (v - s q0) r with both sums fused, where nothing underflows: for s
 * within 2^-60 .. 2^60 and quotients that are not below 2^-60 of interest.  Three instructions. */
static __device__ __forceinline__ float quotient(float v, float s, float r) {
    const float q = v * r;
    return fmaf(fmaf(-s, q, v), r, q);
}
