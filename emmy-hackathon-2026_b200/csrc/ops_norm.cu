/*
 * Norms after and before a block, with its gate and residual scale, in one pass:
 *
 *     y = x + scale * gate * N(block),   h = N(y)
 *
 * The bytes bound it: x and block are read once, y and h written once; the row stays in
 * registers between its two norms.  A row belongs to a group of 8 .. 1024 threads with at
 * most 16 elements each (32-bit sums: shuffles inside a warp, shared memory across the
 * warps of a row).  The layer norm's variance is taken about the mean of the registers'
 * values, not as a difference of two sums, which would lose it when the mean is large.
 */
#include "ops_common.cuh"

namespace {

struct Vector {          /* a weight, bias or gate row of any element type; 0 pointer: none */
    const char *at;
    int dtype;
};

struct NormParams {
    const char *x, *block;
    char *y, *h;
    int64_t x_stride, block_stride, y_stride, h_stride, gate_stride, rows_per_gate, rows;
    Vector post_weight, post_bias, gate, pre_weight, pre_bias;
    int dim, group, layer, post_norm, wide;
    float eps, scale;
};

template <int V> __device__ __forceinline__ void load_vector(const Vector &w, int64_t e, bool wide, float (&out)[V]) {
    if (w.dtype == EMMY_OPS_F32) {
        const float *p = (const float *)w.at + e;
        if (V >= 4 && wide) {
#pragma unroll
            for (int i = 0; i < V; i += 4) {
                const float4 q = *(const float4 *)(p + (V >= 4 ? i : 0));
                out[i] = q.x;
                if (V >= 4) out[i + 1] = q.y, out[i + 2] = q.z, out[i + 3] = q.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = p[i];
        }
    } else if (w.dtype == EMMY_OPS_F16) {
        const __half *p = (const __half *)w.at + e;
        if (V > 1 && wide) {
            const Pack<__half, V> q = *(const Pack<__half, V> *)p;
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_f32(q.at[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_f32(p[i]);
        }
    } else {
        const __nv_bfloat16 *p = (const __nv_bfloat16 *)w.at + e;
        if (V > 1 && wide) {
            const Pack<__nv_bfloat16, V> q = *(const Pack<__nv_bfloat16, V> *)p;
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_f32(q.at[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[i] = to_f32(p[i]);
        }
    }
}

/* the sum over a row's group of threads, to each of them */
__device__ __forceinline__ float group_sum(float v, int group, float *shared) {
    for (int d = min(group, 32) / 2; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    if (group > 32) {
        const int warp = threadIdx.x >> 5, warps = group >> 5, first = warp & ~(warps - 1);
        __syncthreads();                        /* the last sum's readers are done */
        if ((threadIdx.x & 31) == 0) shared[warp] = v;
        __syncthreads();
        v = shared[first + (threadIdx.x & (warps - 1))];
        for (int d = warps / 2; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    }
    return v;
}

/* V elements an access, N accesses a thread */
template <typename T, int V, int N>
__global__ void __launch_bounds__(1024) residual_norm(NormParams p) {
    __shared__ float shared[32];
    enter_grid();
    const int group = p.group, lane = threadIdx.x & (group - 1);
    const int64_t row = (int64_t)blockIdx.x * (blockDim.x / group) + threadIdx.x / group;
    const bool live = row < p.rows;
    const float inv_dim = 1.0f / p.dim;
    Pack<T, V> x[N];
    float b[N][V];
    bool in[N];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int e = (n * group + lane) * V;
        in[n] = live && e < p.dim;
        if (in[n]) {
            const Pack<T, V> q = *(const Pack<T, V> *)((const T *)p.block + row * p.block_stride + e);
            x[n] = *(const Pack<T, V> *)((const T *)p.x + row * p.x_stride + e);
#pragma unroll
            for (int i = 0; i < V; ++i) b[n][i] = to_f32(q.at[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) b[n][i] = 0.0f;
        }
    }
    auto statistics = [&](float &mean, float &rstd) {
        mean = 0.0f;
        if (p.layer) {
            float s = 0.0f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int i = 0; i < V; ++i) s += b[n][i];
            mean = group_sum(s, group, shared) * inv_dim;
        }
        float s = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (in[n]) {
#pragma unroll
                for (int i = 0; i < V; ++i) s += (b[n][i] - mean) * (b[n][i] - mean);
            }
        rstd = 1.0f / sqrtf(group_sum(s, group, shared) * inv_dim + p.eps);
    };
    float mean, rstd;
    if (p.post_norm) {
        statistics(mean, rstd);
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (in[n]) {
                const int e = (n * group + lane) * V;
                float w[V];
#pragma unroll
                for (int i = 0; i < V; ++i) b[n][i] = (b[n][i] - mean) * rstd;
                if (p.post_weight.at) {
                    load_vector(p.post_weight, e, p.wide, w);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[n][i] *= w[i];
                }
                if (p.post_bias.at) {
                    load_vector(p.post_bias, e, p.wide, w);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[n][i] += w[i];
                }
            }
    }
    const int64_t gate_row = p.gate.at && live ? row / p.rows_per_gate * p.gate_stride : 0;
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (in[n]) {
            const int e = (n * group + lane) * V;
            if (p.gate.at) {
                float w[V];
                load_vector(p.gate, gate_row + e, p.wide, w);
#pragma unroll
                for (int i = 0; i < V; ++i) b[n][i] *= w[i];
            }
            Pack<T, V> q;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                b[n][i] = fmaf(p.scale, b[n][i], to_f32(x[n].at[i]));
                q.at[i] = from_f32<T>(b[n][i]);
            }
            *(Pack<T, V> *)((T *)p.y + row * p.y_stride + e) = q;
        }
    if (!p.h) return;
    statistics(mean, rstd);
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (in[n]) {
            const int e = (n * group + lane) * V;
            float w[V];
#pragma unroll
            for (int i = 0; i < V; ++i) b[n][i] = (b[n][i] - mean) * rstd;
            if (p.pre_weight.at) {
                load_vector(p.pre_weight, e, p.wide, w);
#pragma unroll
                for (int i = 0; i < V; ++i) b[n][i] *= w[i];
            }
            if (p.pre_bias.at) {
                load_vector(p.pre_bias, e, p.wide, w);
#pragma unroll
                for (int i = 0; i < V; ++i) b[n][i] += w[i];
            }
            Pack<T, V> q;
#pragma unroll
            for (int i = 0; i < V; ++i) q.at[i] = from_f32<T>(b[n][i]);
            *(Pack<T, V> *)((T *)p.h + row * p.h_stride + e) = q;
        }
}

template <typename T, int V, int N> cudaError_t go(const NormParams &p, int threads, uint64_t stream) {
    const int64_t rows = threads / p.group;
    return launch(residual_norm<T, V, N>, dim3((unsigned)((p.rows + rows - 1) / rows)), dim3(threads), 0, stream, p);
}

/* Accesses of 16 bytes where every row allows them, else of 4, else of one element.  A thread
 * takes 8 elements, and 16 only where 1024 threads would not cover the row otherwise. */
template <typename T> cudaError_t dispatch(NormParams &p, int bytes, uint64_t stream) {
    const int per = p.dim > 8192 ? 16 : 8;
    int group = 8;
    while ((int64_t)group * per < p.dim) group *= 2;
    p.group = group;
    const int threads = group < 128 ? 128 : group;
    constexpr int W = 16 / sizeof(T);
    if (bytes == 16) return per == 16 ? go<T, W, 16 / W>(p, threads, stream) : go<T, W, 8 / W>(p, threads, stream);
    if (bytes == 4 && sizeof(T) == 2)
        return per == 16 ? go<T, 2, 8>(p, threads, stream) : go<T, 2, 4>(p, threads, stream);
    return per == 16 ? go<T, 1, 16>(p, threads, stream) : go<T, 1, 8>(p, threads, stream);
}

}  // namespace

EMMY_EXPORT int emmy_ops_residual_norm(const emmy_ops_norm_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (!known_dtype(a->dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", a->dtype);
    if (a->dim < 1 || a->dim > EMMY_OPS_NORM_MAX_DIM)
        return ops_fail(EMMY_RT_EINVAL, "dim %lld is not in 1 .. %d", (long long)a->dim, EMMY_OPS_NORM_MAX_DIM);
    if (a->rows < 0 || a->rows > 0x7fffffffLL) return ops_fail(EMMY_RT_EINVAL, "rows %lld", (long long)a->rows);
    if (a->kind != EMMY_OPS_NORM_RMS && a->kind != EMMY_OPS_NORM_LAYER)
        return ops_fail(EMMY_RT_EINVAL, "norm kind %d", a->kind);
    if (a->rows == 0) return 0;
    if (!a->x || !a->block || !a->y) return ops_fail(EMMY_RT_EINVAL, "x, block and y are needed");
    if (a->gate && a->rows_per_gate < 1) return ops_fail(EMMY_RT_EINVAL, "rows_per_gate %lld", (long long)a->rows_per_gate);
    const int64_t strides[] = {a->x_stride, a->block_stride, a->y_stride, a->h ? a->h_stride : a->dim};
    for (int64_t s : strides)
        if (s < a->dim && a->rows > 1) return ops_fail(EMMY_RT_EINVAL, "rows overlap: stride %lld", (long long)s);
    const uint64_t rows_at[] = {a->x, a->block, a->y, a->h};
    const int es = elem_size(a->dtype);
    int bytes = 16;
    for (int i = 0; i < 4; ++i) {
        if (!aligned(rows_at[i], es)) return ops_fail(EMMY_RT_EINVAL, "an operand is not aligned to its elements");
        while (bytes > es && (!aligned(rows_at[i], bytes) || (a->rows > 1 && strides[i] * es % bytes) || a->dim * es % bytes))
            bytes = bytes == 16 ? 4 : es;
    }
    NormParams p = {};
    const struct { uint64_t at; int dtype; Vector *to; int64_t stride; } vectors[] = {
        {a->post_norm ? a->post_weight : 0, a->post_weight_dtype, &p.post_weight, 0},
        {a->post_norm ? a->post_bias : 0, a->post_bias_dtype, &p.post_bias, 0},
        {a->gate, a->gate_dtype, &p.gate, a->gate_stride},
        {a->h ? a->pre_weight : 0, a->pre_weight_dtype, &p.pre_weight, 0},
        {a->h ? a->pre_bias : 0, a->pre_bias_dtype, &p.pre_bias, 0}};
    p.wide = 1;
    for (auto &v : vectors) {
        if (!v.at) continue;
        if (!known_dtype(v.dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", v.dtype);
        const int size = elem_size(v.dtype);
        if (!aligned(v.at, size)) return ops_fail(EMMY_RT_EINVAL, "an operand is not aligned to its elements");
        /* one access covers `bytes / es` elements of a vector, in 16 bytes at most */
        int64_t access = (int64_t)bytes / es * size;
        if (access > 16) access = 16;
        if (!aligned(v.at, access) || v.stride * size % access) p.wide = 0;
        v.to->at = (const char *)(uintptr_t)v.at;
        v.to->dtype = v.dtype;
    }
    p.x = (const char *)(uintptr_t)a->x;
    p.block = (const char *)(uintptr_t)a->block;
    p.y = (char *)(uintptr_t)a->y;
    p.h = (char *)(uintptr_t)a->h;
    p.x_stride = a->x_stride, p.block_stride = a->block_stride, p.y_stride = a->y_stride, p.h_stride = a->h_stride;
    p.gate_stride = a->gate_stride, p.rows_per_gate = a->rows_per_gate, p.rows = a->rows;
    p.dim = (int)a->dim, p.layer = a->kind, p.post_norm = a->post_norm != 0, p.eps = a->eps, p.scale = a->scale;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    cudaError_t e = a->dtype == EMMY_OPS_F32    ? dispatch<float>(p, bytes, stream)
                    : a->dtype == EMMY_OPS_F16 ? dispatch<__half>(p, bytes, stream)
                                               : dispatch<__nv_bfloat16>(p, bytes, stream);
    return ops_cuda(e, "residual norm");
}
