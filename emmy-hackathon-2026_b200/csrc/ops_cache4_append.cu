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
    int64_t token[2], head[2], tokens, slots_in_cache;
    const void *slots;
    int heads, page, slots_64, wide;
};

template <typename T, int DIM>
__global__ void __launch_bounds__(256) cache4_append(AppendParams p) {
    constexpr int LANES = DIM / 8;
    constexpr float LARGEST = 65504.0f;
    enter_grid();
    const int lane = threadIdx.x % LANES;
    const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
    const int64_t vectors = p.tokens * p.heads;
    const int which = item >= vectors;             /* keys first, then values */
    const int64_t at = which ? item - vectors : item;
    const int64_t token = at / p.heads;
    const int head = (int)(at - token * p.heads);
    const bool live = token < p.tokens;
    int64_t slot = -1;
    if (live) slot = p.slots_64 ? ((const int64_t *)p.slots)[token] : ((const int32_t *)p.slots)[token];
    float v[8];
    if (live) {
        const T *x = (const T *)p.x[which] + token * p.token[which] + head * p.head[which] + lane * 8;
        if (p.wide) {
            if (sizeof(T) == 2) {
                const Pack<T, 8> q = *(const Pack<T, 8> *)x;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_f32(q.at[i]);
            } else {
                const Pack<T, 4> q[2] = {*(const Pack<T, 4> *)x, *(const Pack<T, 4> *)(x + 4)};
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = to_f32(q[i / 4].at[i % 4]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = to_f32(x[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
    float low = LARGEST, high = -LARGEST;
    int nan = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        nan |= v[i] != v[i];
        v[i] = fminf(fmaxf(v[i], -LARGEST), LARGEST);
        low = fminf(low, v[i]);
        high = fmaxf(high, v[i]);
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d >>= 1) {
        low = fminf(low, __shfl_xor_sync(~0u, low, d));
        high = fmaxf(high, __shfl_xor_sync(~0u, high, d));
        nan |= __shfl_xor_sync(~0u, nan, d);
    }
    const __half least = __float2half_rn(low);
    const __half step = nan ? __ushort_as_half(0x7fff) : __float2half_rn((high - low) / 15.0f);
    const float z = __half2float(least), s = __half2float(step);
    uint32_t levels = 0;
    float said[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float n = s > 0.0f ? fminf(fmaxf(rintf((v[i] - z) / s), 0.0f), 15.0f) : 0.0f;
        levels |= (uint32_t)n << 4 * i;
        said[i] = fmaf(n, s, z);
    }
    if (!live) return;
    if (slot >= 0 && slot < p.slots_in_cache) {
        const int64_t page = slot / p.page, row = slot - page * p.page;
        const int64_t to = (page * p.heads + head) * p.page + row;
        *(uint32_t *)(p.level[which] + to * (DIM / 2) + lane * 4) = levels;
        if (lane == 0) p.meta[which][to] = __halves2half2(step, least);
    }
    if (p.stored[which]) {
        T *out = (T *)p.stored[which] + (token * p.heads + head) * DIM + lane * 8;
        if (sizeof(T) == 2) {
            Pack<T, 8> q;
#pragma unroll
            for (int i = 0; i < 8; ++i) q.at[i] = from_f32<T>(said[i]);
            *(Pack<T, 8> *)out = q;
        } else {
            Pack<T, 4> q[2];
#pragma unroll
            for (int i = 0; i < 8; ++i) q[i / 4].at[i % 4] = from_f32<T>(said[i]);
            *(Pack<T, 4> *)out = q[0];
            *(Pack<T, 4> *)(out + 4) = q[1];
        }
    }
}

template <typename T> cudaError_t dispatch(const AppendParams &p, int dim, uint64_t stream) {
    const int64_t items = 2 * p.tokens * p.heads, per = 256 / (dim / 8);
    const dim3 grid((unsigned)((items + per - 1) / per));
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
    if (2 * a->tokens * a->cache.heads > 0x7fffffffLL * 8)
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
    p.tokens = a->tokens, p.slots_in_cache = a->cache.pages * a->cache.page;
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
