/*
 * Norms after and before a block, with its gate and residual scale, in one pass:
 *
 *     y = x + scale * gate * N(block),   h = N(y)
 *
 * x and block are read once, y and h written once; the row stays in registers between its two norms.  A row belongs to 8, 16 or 32 lanes of a warp, or to a
 * block of threads of its own; a thread holds 8 elements of it, or 32 where there are rows
 * enough to fill the GPU: fewer warps then have to meet at a row's sums (one barrier each), and
 * more bytes are under way for each of them.  32-bit sums: shuffles inside a warp, shared
 * memory across a row's warps.  The layer norm's variance is taken about the mean of the
 * registers' values, not as a difference of two sums, which would lose it when the mean is large.
 * Few rows are bound by the launch (8 rows 3.1 us), many by latency and not by their bytes: 8192 x 4096 in bf16, both norms layer
 * norms, takes 73 us (3.7 TB/s), as 104 registers leave 16 warps an SM, which wait for four sums in sequence and five vectors
 * through L1.
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
    int64_t x_stride, block_stride, y_stride, h_stride, gate_stride, rows;
    int rows_per_gate;
    Vector post_weight, post_bias, gate, pre_weight, pre_bias;
    int dim, group, layer, post_norm, wide;
    float eps, scale;
};

/* A thread's elements: N accesses of V, at e[n], as E = N V values in a row; in pairs (Two) where an access has pairs, else one
 * by one. */
template <bool PAIRS> struct Unit {
    using type = Two;
    static constexpr int SIZE = 2;
};
template <> struct Unit<false> {
    using type = float;
    static constexpr int SIZE = 1;
};
__device__ __forceinline__ float fma2(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float total(float v) { return v; }
__device__ __forceinline__ float total(Two v) { return v.get().x + v.get().y; }
template <typename U> __device__ __forceinline__ U both(float a, float b);
template <> __device__ __forceinline__ float both<float>(float a, float) { return a; }
template <> __device__ __forceinline__ Two both<Two>(float a, float b) { return Two(a, b); }
__device__ __forceinline__ float value(float v, int) { return v; }
__device__ __forceinline__ float value(Two v, int i) { return i ? v.get().y : v.get().x; }

/* Runs op(first element of an access, its V values) over a thread's piece of a vector.  The choice of its type stands outside
 * the loops, so that as many loads as registers allow are under way at once. */
template <int V, int N, typename W, typename Op>
__device__ __forceinline__ void each_as(const W *w, const int (&e)[N], bool wide, Op op) {
    constexpr int A = 16 / (int)sizeof(W) < V ? 16 / (int)sizeof(W) : V;        /* elements an access */
    Pack<W, A> q[N][V / A];
    if (V == 1 || wide) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < V / A; ++i) q[n][i] = *(const Pack<W, A> *)(w + e[n] + i * A);
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < V; ++i) q[n][i / A].at[i % A] = w[e[n] + i];
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float f[V];
#pragma unroll
        for (int i = 0; i < V / A; ++i) {
            float part[A];
            unpack(q[n][i], part);
#pragma unroll
            for (int j = 0; j < A; ++j) f[i * A + j] = part[j];
        }
        op(n * V, f);
    }
}
template <int V, int N, typename Op>
__device__ __forceinline__ void each(const Vector &w, int64_t skip, const int (&e)[N], bool wide, Op op) {
    if (w.dtype == EMMY_OPS_F32)
        each_as<V>((const float *)w.at + skip, e, wide, op);
    else if (w.dtype == EMMY_OPS_F16)
        each_as<V>((const __half *)w.at + skip, e, wide, op);
    else
        each_as<V>((const __nv_bfloat16 *)w.at + skip, e, wide, op);
}

/* the sum over a row's threads, to each of them; `shared`: 32 floats of this sum's own */
__device__ __forceinline__ float row_sum(float v, int group, float *shared) {
    for (int d = min(group, 32) / 2; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    if (group > 32) {           /* the row is this block of threads */
        const int lane = threadIdx.x & 31;
        if (lane == 0) shared[threadIdx.x >> 5] = v;
        __syncthreads();
        v = lane < group >> 5 ? shared[lane] : 0.0f;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
    }
    return v;
}

template <typename T, int V, int N>
__global__ void __launch_bounds__(N * V > 16 ? 512 : 1024) residual_norm(NormParams p) {
    /* few elements a thread: rows are few too, and the weights are fetched before the sums they wait for */
    constexpr int E = N * V, K = Unit<V % 2 == 0>::SIZE;
    using U = typename Unit<V % 2 == 0>::type;
    constexpr bool EARLY = E <= 8;
    __shared__ float shared[4][32];
    enter_grid();
    const int group = p.group, lane = group > 32 ? threadIdx.x : threadIdx.x & (group - 1);
    const int64_t place = group > 32 ? blockIdx.x : (int64_t)blockIdx.x * (blockDim.x / group) + threadIdx.x / group;
    const int64_t row = min(place, p.rows - 1);
    const float inv_dim = 1.0f / p.dim;
    /* Accesses past the row take its last one once more: no branch stands between the loads, and only the sums and the
     * stores ask what is in the row. */
    int e[N];
    bool in[N];
    Pack<T, V> x[N], raw[N];
    U b[E / K];
    float w[EARLY ? E : 1];
    const T *const from = (const T *)p.block + row * p.block_stride, *const stream = (const T *)p.x + row * p.x_stride;
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int at = (n * group + lane) * V;
        in[n] = at < p.dim && place < p.rows;
        e[n] = min(at, p.dim - V);
        raw[n] = *(const Pack<T, V> *)(from + e[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) x[n] = *(const Pack<T, V> *)(stream + e[n]);
    auto early = [&](const Vector &v) {
        each<V>(v, 0, e, p.wide, [&](int at, const float (&f)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[EARLY ? at + i : 0] = f[i];
        });
    };
    if (EARLY && p.post_weight.at) early(p.post_weight);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float f[V];
        unpack(raw[n], f);
#pragma unroll
        for (int i = 0; i < V / K; ++i) b[n * V / K + i] = both<U>(f[K * i], f[K * i + K - 1]);
    }
    /* op over an access's values and V others */
    auto with = [&](int at, const float (&f)[V], auto op) {
#pragma unroll
        for (int i = 0; i < V / K; ++i) b[at / K + i] = op(b[at / K + i], both<U>(f[K * i], f[K * i + K - 1]));
    };
    auto product = [](U a, U c) { return a * c; };
    auto sum = [](U a, U c) { return a + c; };
    /* the sum over the row of each(b) */
    auto over_row = [&](float *shared, auto each) {
        float all = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            U s = both<U>(0.0f, 0.0f);
#pragma unroll
            for (int i = 0; i < V / K; ++i) s = each(b[n * V / K + i], s);
            all += in[n] ? total(s) : 0.0f;
        }
        return row_sum(all, group, shared);
    };
    /* (b - mean) / deviation, in place */
    auto normalise = [&](int first) {
        if (p.layer) {
            const float mean = over_row(shared[first], [](U v, U s) { return s + v; }) * inv_dim;
#pragma unroll
            for (int i = 0; i < E / K; ++i) b[i] = b[i] + both<U>(-mean, -mean);
        }
        const float r = rsqrtf(over_row(shared[first + 1], [](U v, U s) { return fma2(v, v, s); }) * inv_dim + p.eps);
#pragma unroll
        for (int i = 0; i < E / K; ++i) b[i] = b[i] * both<U>(r, r);
    };
    auto weigh = [&](const Vector &v) {
        if (EARLY) {
#pragma unroll
            for (int i = 0; i < E / K; ++i) b[i] = b[i] * both<U>(w[EARLY ? K * i : 0], w[EARLY ? K * i + K - 1 : 0]);
        } else {
            each<V>(v, 0, e, p.wide, [&](int at, const float (&f)[V]) { with(at, f, product); });
        }
    };
    auto store = [&](char *to, int64_t stride) {
        T *const y = (T *)to + row * stride;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float f[V];
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = value(b[(n * V + i) / K], i % K);
            Pack<T, V> q;
            pack(f, q);
            if (in[n]) *(Pack<T, V> *)(y + e[n]) = q;
        }
    };
    if (p.post_norm) normalise(0);
    if (p.post_weight.at) weigh(p.post_weight);
    if (p.post_bias.at) each<V>(p.post_bias, 0, e, p.wide, [&](int at, const float (&f)[V]) { with(at, f, sum); });
    if (p.gate.at) {
        const int64_t skip = (int64_t)((uint32_t)row / (uint32_t)p.rows_per_gate) * p.gate_stride;
        each<V>(p.gate, skip, e, p.wide, [&](int at, const float (&f)[V]) { with(at, f, product); });
    }
    const U scale = both<U>(p.scale, p.scale);
#pragma unroll
    for (int n = 0; n < N; ++n) {
        float f[V];
        unpack(x[n], f);
        with(n * V, f, [&](U a, U c) { return fma2(scale, a, c); });
    }
    store(p.y, p.y_stride);
    if (!p.h) return;
    if (EARLY && p.pre_weight.at) early(p.pre_weight);
    normalise(2);
    if (p.pre_weight.at) weigh(p.pre_weight);
    if (p.pre_bias.at) each<V>(p.pre_bias, 0, e, p.wide, [&](int at, const float (&f)[V]) { with(at, f, sum); });
    store(p.h, p.h_stride);
}

template <typename T, int V, int N> cudaError_t go(NormParams &p, uint64_t stream) {
    const int threads = (p.dim + V * N - 1) / (V * N);
    p.group = threads <= 8 ? 8 : threads <= 16 ? 16 : (threads + 31) / 32 * 32;
    const int block = p.group > 32 ? p.group : 128, rows = p.group > 32 ? 1 : 128 / p.group;
    return launch(residual_norm<T, V, N>, dim3((unsigned)((p.rows + rows - 1) / rows)), dim3(block), 0, stream, p);
}

/* Accesses of 16 bytes where every row allows them, else of 4, else of one element.  8 elements a thread while the rows
 * do not fill the GPU (they are bound by the chain from load to store), where accesses are narrow, and up to 128 elements a
 * row, of which 32 each would leave half of the 8 lanes idle (200000 rows of 64 in bf16: 44 us, 20 with 8 each); else
 * 32, over which a row's sums and addresses cost little (100000 rows of 200: 44 us, 56 with 8 each); 16 in narrow accesses
 * for rows that 1024 threads of 8 would not hold.  Those keep to the 64 registers of 1024 threads by spilling, 16 to 24 bytes in
 * pairs and about 300 in single elements: 2861 rows of 11727 in bf16 take 243 us, of 11728 in 16-byte accesses 85. */
template <typename T> cudaError_t dispatch(NormParams &p, int bytes, int sms, uint64_t stream) {
    const bool many = p.dim > 8192 || (p.dim > 128 && p.rows * p.dim > (int64_t)sms * 4096 * 2);
    constexpr int W = 16 / sizeof(T);
    const bool large = p.dim > 8192;
    if (bytes == 16) return many ? go<T, W, 32 / W>(p, stream) : go<T, W, 8 / W>(p, stream);
    if constexpr (sizeof(T) == 2)
        if (bytes == 4) return large ? go<T, 2, 8>(p, stream) : go<T, 2, 4>(p, stream);
    return large ? go<T, 1, 16>(p, stream) : go<T, 1, 8>(p, stream);
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
    for (int i = 0; i < 4; ++i)         /* x and block may be one row for all */
        if (strides[i] < a->dim && a->rows > 1 && !(i < 2 && strides[i] == 0))
            return ops_fail(EMMY_RT_EINVAL, "rows overlap: stride %lld", (long long)strides[i]);
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
    p.gate_stride = a->gate_stride, p.rows = a->rows;
    p.rows_per_gate = (int)(a->rows_per_gate < a->rows ? a->rows_per_gate : a->rows);
    p.dim = (int)a->dim, p.layer = a->kind, p.post_norm = a->post_norm != 0, p.eps = a->eps, p.scale = a->scale;
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    cudaError_t e = a->dtype == EMMY_OPS_F32    ? dispatch<float>(p, bytes, sms, stream)
                    : a->dtype == EMMY_OPS_F16 ? dispatch<__half>(p, bytes, sms, stream)
                                               : dispatch<__nv_bfloat16>(p, bytes, sms, stream);
    return ops_cuda(e, "residual norm");
}
