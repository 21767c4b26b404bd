/*
 * Writing keys and values into the 4-bit cache.
 *
 *     least = f16(min v), step = f16((max v - min v) / 15), level = rint((v - least) / step) in 0 .. 15
 *
 * over each token's head vector v.  Levels are taken against the rounded least and step, so
 * what the rounding moved is made good by the levels.  Values beyond the range of f16
 * saturate; a vector with a NaN gets a NaN step and reads back as NaN.
 *
 * The bytes bound it.  dim / 8 lanes hold a vector, eight elements each: one 16-byte load,
 * shuffles for the least and the largest, one 4-byte store of eight levels.
 */
#include "ops_common.cuh"

namespace {

struct AppendParams {
    const char *x[2];
    char *level[2], *stored[2];
    __half2 *meta[2];
    int64_t token[2], head[2], slots_in_cache;
    const void *slots;
    int tokens, heads, page, slots_64, wide;
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

/* DIM / 8 lanes a vector; blocks of threads y = 0 take keys, y = 1 values */
template <typename T, int DIM>
__global__ void __launch_bounds__(256) cache4_append(AppendParams p) {
    constexpr int LANES = DIM / 8;
    constexpr float LARGEST = 65504.0f;
    enter_grid();
    const int lane = threadIdx.x % LANES, which = blockIdx.y;
    const uint32_t item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, token = item / (uint32_t)p.heads;
    const int head = item - token * p.heads;
    const bool live = token < (uint32_t)p.tokens;
    int64_t slot = -1;
    if (live) slot = p.slots_64 ? ((const int64_t *)p.slots)[token] : ((const int32_t *)p.slots)[token];
    float v[8];
    if (live) {
        const T *x = (const T *)p.x[which] + token * p.token[which] + head * p.head[which] + lane * 8;
        if (p.wide) {
            constexpr int V = 16 / sizeof(T);
            Pack<T, V> q[8 / V];
#pragma unroll
            for (int i = 0; i < 8 / V; ++i) q[i] = *(const Pack<T, V> *)(x + i * V);
#pragma unroll
            for (int i = 0; i < 8 / V; ++i) {
                float f[V];
                unpack(q[i], f);
#pragma unroll
                for (int j = 0; j < V; ++j) v[i * V + j] = f[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(x[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    auto extremes = [&](float &low, float &high) {
        low = high = v[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) low = fminf(low, v[i]), high = max_or_nan(high, v[i]);
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) {
            low = fminf(low, __shfl_xor_sync(~0u, low, d));
            high = max_or_nan(high, __shfl_xor_sync(~0u, high, d));
        }
    };
    float low, high;
    extremes(low, high);
    const bool nan = high != high;
    if (__any_sync(~0u, nan || low < -LARGEST || high > LARGEST)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fminf(fmaxf(v[i], -LARGEST), LARGEST);      /* a NaN becomes a number, too */
        extremes(low, high);
    }
    const __half least = __float2half_rn(low);
    const __half step = nan ? __ushort_as_half(0x7fff) : __float2half_rn(__fdiv_rn(high - low, 15.0f));
    const float z = __half2float(least), s = __half2float(step), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
    /* The level to the nearest even by adding 1.5 2^23, whose last bit is 1; four levels make 16 bits, exact in f32.  With a
     * step of 0 (or NaN) all levels are 0: r is 0. */
    constexpr float ROUND = 12582912.0f;
    float n[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = s > 0.0f ? quotient(v[i] - z, s, r) : 0.0f;
        n[i] = (fminf(fmaxf(q, 0.0f), 15.0f) + ROUND) - ROUND;
    }
    if (!live) return;
    if (slot >= 0 && slot < p.slots_in_cache) {
        const int64_t page = slot <= 0xffffffffll ? (uint32_t)slot / (uint32_t)p.page : slot / p.page, row = slot - page * p.page;
        const int64_t to = (page * p.heads + head) * p.page + row;
        const float first = fmaf(fmaf(fmaf(n[3], 16.0f, n[2]), 16.0f, n[1]), 16.0f, n[0]);
        const float second = fmaf(fmaf(fmaf(n[7], 16.0f, n[6]), 16.0f, n[5]), 16.0f, n[4]);
        *(uint32_t *)(p.level[which] + to * (DIM / 2) + lane * 4) = (uint32_t)first | (uint32_t)second << 16;
        if (lane == 0) p.meta[which][to] = __halves2half2(step, least);
    }
    if (p.stored[which]) {
        constexpr int V = 16 / sizeof(T);
        T *out = (T *)p.stored[which] + ((int64_t)token * p.heads + head) * DIM + lane * 8;
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; ++j) f[j] = fmaf(n[i + j], s, z);
            Pack<T, V> q;
            pack(f, q);
            *(Pack<T, V> *)(out + i) = q;
        }
    }
}

template <typename T> cudaError_t dispatch(const AppendParams &p, int dim, uint64_t stream) {
    const int64_t items = (int64_t)p.tokens * p.heads, per = 256 / (dim / 8);
    const dim3 grid((unsigned)((items + per - 1) / per), 2);
    return dim == 64 ? launch(cache4_append<T, 64>, grid, dim3(256), 0, stream, p)
                     : launch(cache4_append<T, 128>, grid, dim3(256), 0, stream, p);
}

}  // namespace

int ops_check_cache4(const emmy_ops_cache4 &c) {
    if (c.dim != 64 && c.dim != 128) return ops_fail(EMMY_RT_EINVAL, "head dim %d is not 64 or 128", c.dim);
    if (c.heads < 1 || c.heads > 4096 || c.page < 1 || c.page > (1 << 20) || c.pages < 0 || c.pages > 0x7fffffffLL)
        return ops_fail(EMMY_RT_EINVAL, "cache of %lld pages, %d heads, %d rows a page", (long long)c.pages, c.heads, c.page);
    if (c.pages && (!c.k || !c.v || !c.k_meta || !c.v_meta)) return ops_fail(EMMY_RT_EINVAL, "the cache has no memory");
    if (!aligned(c.k, 16) || !aligned(c.v, 16) || !aligned(c.k_meta, 4) || !aligned(c.v_meta, 4))
        return ops_fail(EMMY_RT_EINVAL, "the cache's levels start on 16 bytes, its steps on 4");
    return 0;
}

EMMY_EXPORT int emmy_ops_cache4_append(const emmy_ops_cache4_append_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (int e = ops_check_cache4(a->cache)) return e;
    if (!known_dtype(a->dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", a->dtype);
    if (a->tokens < 0 || a->tokens > 0x7fffffffLL) return ops_fail(EMMY_RT_EINVAL, "tokens %lld", (long long)a->tokens);
    if (a->tokens == 0) return 0;
    const int es = elem_size(a->dtype);
    if (a->tokens * a->cache.heads > 0x7fffff00LL)
        return ops_fail(EMMY_RT_EINVAL, "%lld tokens of %d heads are too many for one call", (long long)a->tokens, a->cache.heads);
    if (!a->k || !a->v || !a->slots || !aligned(a->k, es) || !aligned(a->v, es) || !aligned(a->slots, a->slots_64 ? 8 : 4))
        return ops_fail(EMMY_RT_EINVAL, "k, v and slots are needed, aligned to their elements");
    if (!aligned(a->k_stored, 16) || !aligned(a->v_stored, 16))
        return ops_fail(EMMY_RT_EINVAL, "k_stored and v_stored start on 16 bytes");
    AppendParams p = {};
    p.x[0] = (const char *)(uintptr_t)a->k, p.x[1] = (const char *)(uintptr_t)a->v;
    p.level[0] = (char *)(uintptr_t)a->cache.k, p.level[1] = (char *)(uintptr_t)a->cache.v;
    p.meta[0] = (__half2 *)(uintptr_t)a->cache.k_meta, p.meta[1] = (__half2 *)(uintptr_t)a->cache.v_meta;
    p.stored[0] = (char *)(uintptr_t)a->k_stored, p.stored[1] = (char *)(uintptr_t)a->v_stored;
    p.token[0] = a->k_token, p.token[1] = a->v_token, p.head[0] = a->k_head, p.head[1] = a->v_head;
    p.tokens = (int)a->tokens, p.slots_in_cache = a->cache.pages * a->cache.page;
    p.slots = (const void *)(uintptr_t)a->slots, p.slots_64 = a->slots_64 != 0;
    p.heads = a->cache.heads, p.page = a->cache.page;
    p.wide = aligned(a->k, 16) && aligned(a->v, 16);
    const int64_t strides[] = {a->k_token, a->k_head, a->v_token, a->v_head};
    for (int64_t s : strides) p.wide = p.wide && s * es % 16 == 0;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    const int dim = a->cache.dim;
    cudaError_t e = a->dtype == EMMY_OPS_F32   ? dispatch<float>(p, dim, stream)
                    : a->dtype == EMMY_OPS_F16 ? dispatch<__half>(p, dim, stream)
                                               : dispatch<__nv_bfloat16>(p, dim, stream);
    return ops_cuda(e, "append to the 4-bit cache");
}
