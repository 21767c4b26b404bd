/*
 * Writing keys and values into the 4-bit cache.
 *
 *     least = f16(min v), step = f16((max v - min v) / 15), level = rint((v - least) / step) in 0 .. 15
 *
 * over each token's head vector v.  Levels are taken against the rounded least and step, so
 * what the rounding moved is made good by the levels.  Values beyond the range of f16
 * saturate; a vector with a NaN gets a NaN step and reads back as NaN.
 *
 * Bytes and instructions bound it alike.  dim / 8 lanes hold a vector, eight elements each: one 16-byte load,
 * shuffles for the least and the largest, one 4-byte store of eight levels.  16384 tokens of 8 heads of 128, with
 * the stored values, take 38.5 us (3.9 TB/s); 310 instructions a vector, with divisions for the indexes and the extremes
 * in f32, took 52.7 us at 80 % of the issue slots, and two vectors a thread are no faster.
 */
#include "ops_common.cuh"

namespace {

struct AppendParams {
    const char *x[2];
    char *level[2], *stored[2];
    __half2 *meta[2];
    int64_t token[2], head[2], slots_in_cache;
    const void *slots;
    int tokens, slots_64, wide;
    Divisor heads, page;
};

__device__ __forceinline__ float max_or_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ __half2 lesser(__half2 a, __half2 b) { return __hmin2_nan(a, b); }
__device__ __forceinline__ __nv_bfloat162 lesser(__nv_bfloat162 a, __nv_bfloat162 b) { return __hmin2_nan(a, b); }
template <typename T> struct PairOf;
template <> struct PairOf<__half> { using type = __half2; };
template <> struct PairOf<__nv_bfloat16> { using type = __nv_bfloat162; };

/* The least and the largest of LANES threads' 8 values.  In 16 bits two at a time, and the largest as the least of the values with
 * their signs turned: both in one shuffle.  NaN if any is. */
template <int LANES, typename T, int V, int N> __device__ __forceinline__ void extremes(const Pack<T, V> (&q)[N], float &low, float &high) {
    if constexpr (sizeof(T) == 2) {
        using Pair = typename PairOf<T>::type;
        const uint32_t *u = (const uint32_t *)&q[0];
        auto pair = [](uint32_t v) { return *(const Pair *)&v; };
        auto bits = [](Pair v) { return *(const uint32_t *)&v; };
        Pair a = lesser(lesser(pair(u[0]), pair(u[1])), lesser(pair(u[2]), pair(u[3])));
        constexpr uint32_t SIGNS = 0x80008000u;
        Pair b = lesser(lesser(pair(u[0] ^ SIGNS), pair(u[1] ^ SIGNS)), lesser(pair(u[2] ^ SIGNS), pair(u[3] ^ SIGNS)));
        a = lesser(pair(__byte_perm(bits(a), bits(b), 0x5410)), pair(__byte_perm(bits(a), bits(b), 0x7632)));
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) a = lesser(a, pair(__shfl_xor_sync(~0u, bits(a), d)));
        low = to_f32(a.x), high = -to_f32(a.y);
    } else {
        low = high = q[0].at[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) low = fminf(low, q[i / V].at[i % V]), high = max_or_nan(high, q[i / V].at[i % V]);
#pragma unroll
        for (int d = LANES / 2; d > 0; d >>= 1) {
            low = fminf(low, __shfl_xor_sync(~0u, low, d));
            high = max_or_nan(high, __shfl_xor_sync(~0u, high, d));
        }
    }
}

/* DIM / 8 lanes a vector; blocks of threads y = 0 take keys, y = 1 values */
template <typename T, int DIM> __global__ void __launch_bounds__(256) cache4_append(AppendParams p) {
    constexpr int LANES = DIM / 8, V = 16 / sizeof(T);
    constexpr float LARGEST = 65504.0f;
    enter_grid();
    const int lane = threadIdx.x % LANES, which = blockIdx.y;
    const uint32_t item = blockIdx.x * (256 / LANES) + threadIdx.x / LANES, own = p.heads.divides(item), head = item - own * p.heads.by;
    const uint32_t token = min(own, (uint32_t)p.tokens - 1);       /* past the end: the last one's once more, not stored */
    const int64_t slot = p.slots_64 ? ((const int64_t *)p.slots)[token] : ((const int32_t *)p.slots)[token];
    const T *x = (const T *)p.x[which] + token * p.token[which] + head * p.head[which] + lane * 8;
    Pack<T, V> raw[8 / V];
    if (p.wide) {
#pragma unroll
        for (int i = 0; i < 8 / V; ++i) raw[i] = *(const Pack<T, V> *)(x + i * V);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i / V].at[i % V] = x[i];
    }
    float low, high, v[8];
    extremes<LANES>(raw, low, high);
#pragma unroll
    for (int i = 0; i < 8 / V; ++i) {
        float f[V];
        unpack(raw[i], f);
#pragma unroll
        for (int j = 0; j < V; ++j) v[i * V + j] = f[j];
    }
    const bool nan = low != low || high != high;
    if (__any_sync(~0u, nan || low < -LARGEST || high > LARGEST)) {
        Pack<float, 4> held[2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            held[i / 4].at[i % 4] = v[i] = fminf(fmaxf(v[i], -LARGEST), LARGEST);      /* a NaN becomes a number, too */
        extremes<LANES>(held, low, high);
    }
    const __half least = __float2half_rn(low);
    /* a difference below 2^-60, which quotient() is not made for, gives a step of 0 in any case */
    constexpr float FIFTEENTH = 1.0f / 15.0f;
    const __half step = nan ? __ushort_as_half(0x7fff) : __float2half_rn(quotient(high - low, 15.0f, FIFTEENTH));
    const float z = __half2float(least), s = __half2float(step), r = s > 0.0f ? __frcp_rn(s) : 0.0f;
    /* The level to the nearest even by adding 1.5 2^23: it then is in the last bits, and eight of them are shifted into a
     * word.  With a step of 0 or NaN the quotient is 0 or NaN, and the level 0. */
    constexpr float ROUND = 12582912.0f;
    constexpr uint32_t ROUND_BITS = 0x4b400000u * 0x11111111u;     /* what the eight sums' upper bits make of it */
    Two n[4];
    uint32_t word = 0;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const Two d = Two(v[2 * i], v[2 * i + 1]) + Two(-z, -z), q0 = d * Two(r, r);
        const float2 q = fma2(fma2(Two(-s, -s), q0, d), Two(r, r), q0).get();
        n[i] = Two(fminf(fmaxf(q.x, 0.0f), 15.0f), fminf(fmaxf(q.y, 0.0f), 15.0f)) + Two(ROUND, ROUND);
        const float2 f = n[i].get();
        word = word * 256 + (__float_as_uint(f.y) * 16 + __float_as_uint(f.x));
    }
    if (own >= (uint32_t)p.tokens) return;
    if (slot >= 0 && slot < p.slots_in_cache) {
        const int64_t page = slot < 0x80000000ll ? p.page.divides((uint32_t)slot) : slot / p.page.by;
        const int64_t to = (page * p.heads.by + head) * p.page.by + (slot - page * p.page.by);
        *(uint32_t *)(p.level[which] + to * (DIM / 2) + lane * 4) = word - ROUND_BITS;
        if (lane == 0) p.meta[which][to] = __halves2half2(step, least);
    }
    if (p.stored[which]) {
        T *out = (T *)p.stored[which] + ((int64_t)token * p.heads.by + head) * DIM + lane * 8;
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            float f[V];
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 both = fma2(n[(i + j) / 2] + Two(-ROUND, -ROUND), Two(s, s), Two(z, z)).get();
                f[j] = both.x, f[j + 1] = both.y;
            }
            Pack<T, V> q;
            pack(f, q);
            *(Pack<T, V> *)(out + i) = q;
        }
    }
}

template <typename T> cudaError_t dispatch(const AppendParams &p, int dim, uint64_t stream) {
    const int64_t items = (int64_t)p.tokens * p.heads.by, per = 256 / (dim / 8);
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
    p.heads = Divisor(a->cache.heads), p.page = Divisor(a->cache.page);
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
