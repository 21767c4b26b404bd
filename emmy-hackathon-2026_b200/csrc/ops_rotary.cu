/*
 * Rotary positions:  (a, b) -> magnitude * (a cos t - b sin t, a sin t + b cos t) for each pair
 * of a head, t = position * frequency.
 *
 * The angle is kept in turns as a 64-bit fraction: position * turns wraps exactly where the
 * angle does, so a far position keeps the precision of a near one (a 32-bit product of a
 * position of 2^20 would be off by 0.03 radians).  Its upper 32 bits go to sincospif in f32, whose 24 bits make an f32 result
 * off by 5.6e-8 of the norm, where cosines of 64 bits leave 4.2e-8; 16-bit results are off by their own rounding.
 *
 * Every element is read and written once.  A block takes a few tokens, computes their cosines and sines once into
 * shared memory, and every head of both tensors uses them.  16384 tokens of 40 heads of 128, 64 of them rotated, take
 * 65 us in bf16 (5.1 TB/s): instructions bound it as much as bytes (three integer divisions a thread were 3 us).
 */
#include "ops_common.cuh"

namespace {

struct RotaryParams {
    const char *x[2];
    char *out[2];
    int64_t x_token[2], x_head[2], out_token[2], out_head[2];
    int heads[2];
    const void *positions;
    const uint64_t *turns;
    int64_t tokens;
    int positions_64, rest, per_block, transpose;
    Divisor pairs, per_head, all_heads;     /* per_head: accesses (of V pairs, or V copied elements) a head */
    int side;                               /* heads that 256 threads take side by side, or 1 */
    float magnitude;
};

/* V pairs a step (half: V elements of either half; interleaved: 2 V consecutive elements).  A thread keeps its place in the
 * heads and goes over the block's (token, head) pairs, AT_ONCE of them under way; the first ones' loads are issued before the
 * angles are worked out. */
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(256) rotary(RotaryParams p) {
    constexpr int AT_ONCE = 2;
    extern __shared__ __align__(16) float2 table[];             /* [per_block][pairs] (cos, sin) */
    enter_grid();
    const int64_t first = (int64_t)blockIdx.x * p.per_block;
    const int live = (int)min((int64_t)p.per_block, p.tokens - first);
    const int pairs = p.pairs.by, units = pairs / V, per_head = p.per_head.by, heads = p.all_heads.by, side = p.side;
    const int own = p.per_head.divides(threadIdx.x), second = HALF ? pairs : V;    /* from an access to its partner */
    struct Item {
        int token, head;
    };
    const int over = p.all_heads.divides(own);
    Item next = {over, own - over * heads};
    if (own >= side) next.token = live;                         /* no place: nothing to do */
    auto advance = [&] {
        next.head += side;
        while (next.head >= heads) next.head -= heads, ++next.token;
    };
    int unit = threadIdx.x - own * per_head;
    Item item[AT_ONCE];
    Pack<T, V> a[AT_ONCE], b[AT_ONCE];
    auto element = [&] { return unit >= units ? 2 * pairs + (unit - units) * V : HALF ? unit * V : 2 * unit * V; };
    auto load = [&] {
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            item[i] = next;
            if (next.token < live) {
                const int which = next.head >= p.heads[0], h = which ? next.head - p.heads[0] : next.head;
                const T *x = (const T *)p.x[which] + (first + next.token) * p.x_token[which] + h * p.x_head[which] + element();
                a[i] = *(const Pack<T, V> *)x;
                if (unit < units) b[i] = *(const Pack<T, V> *)(x + second);
                advance();
            }
        }
    };
    load();
    for (int i = threadIdx.x; i < live * pairs; i += blockDim.x) {
        const int token = p.pairs.divides(i), pair = i - token * pairs;
        const int64_t position = p.positions_64 ? ((const int64_t *)p.positions)[first + token]
                                                : ((const int32_t *)p.positions)[first + token];
        const uint64_t turn = (uint64_t)position * p.turns[pair];
        float s, c;
        sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
        table[i] = make_float2(c * p.magnitude, (p.transpose ? -s : s) * p.magnitude);
    }
    __syncthreads();
    while (true) {
        while (item[0].token < live) {
#pragma unroll
            for (int i = 0; i < AT_ONCE; ++i) {
                if (item[i].token >= live) continue;
                const int which = item[i].head >= p.heads[0], h = which ? item[i].head - p.heads[0] : item[i].head;
                T *out = (T *)p.out[which] + (first + item[i].token) * p.out_token[which] + h * p.out_head[which] + element();
                if (unit >= units) {
                    *(Pack<T, V> *)out = a[i];
                    continue;
                }
                const float2 *cs = table + item[i].token * pairs + unit * V;
                float u[V], v[V], ru[V], rv[V];
                unpack(a[i], u);
                unpack(b[i], v);
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    /* pair j: u[j] and v[j], or elements 2 j and 2 j + 1 of u and v in a row */
                    const float2 q = cs[j];
                    const int k = 2 * j, l = 2 * j + 1;
                    const float c = HALF ? u[j] : k < V ? u[k % V] : v[k % V], d = HALF ? v[j] : l < V ? u[l % V] : v[l % V];
                    const float rc = c * q.x - d * q.y, rd = c * q.y + d * q.x;
                    (HALF ? ru[j] : k < V ? ru[k % V] : rv[k % V]) = rc;
                    (HALF ? rv[j] : l < V ? ru[l % V] : rv[l % V]) = rd;
                }
                Pack<T, V> ra, rb;
                pack(ru, ra);
                pack(rv, rb);
                *(Pack<T, V> *)out = ra;
                *(Pack<T, V> *)(out + second) = rb;
            }
            load();
        }
        /* more places in a head than threads: the next ones, from the first head on */
        if (side > 1 || (unit += blockDim.x) >= per_head) return;
        next = {0, 0};
        load();
    }
}

template <typename T, int V> cudaError_t go(RotaryParams &p, int layout, bool copies, int sms, uint64_t stream) {
    /* tokens a block: about two (token, head) pairs for each of its 256 threads where there are many tokens, one token
     * where there are few, as long as the table fits 32 KB.  More would fill the threads better and wait longer for angles: 16384
     * tokens of 40 heads take 69 us with one token a block and 77 with two. */
    const int pairs = p.pairs.by, per_head = pairs / V + (copies ? p.rest / V : 0);
    p.per_head = Divisor(per_head), p.all_heads = Divisor(p.heads[0] + p.heads[1]);
    p.side = per_head < 256 ? 256 / per_head : 1;
    const int64_t per_token = (int64_t)(p.heads[0] + p.heads[1]) * per_head;
    int64_t per = (512 + per_token / 2) / per_token;
    const int64_t spread = p.tokens / (sms * 4), most = 32768 / ((int64_t)pairs * 8);
    if (per > spread) per = spread;
    if (per > most) per = most;
    p.per_block = per < 1 ? 1 : (int)per;
    const dim3 grid((unsigned)((p.tokens + p.per_block - 1) / p.per_block));
    const size_t smem = (size_t)p.per_block * pairs * 8;
    return layout == EMMY_OPS_ROTARY_HALF ? launch(rotary<T, V, true>, grid, dim3(256), smem, stream, p)
                                          : launch(rotary<T, V, false>, grid, dim3(256), smem, stream, p);
}

}  // namespace

EMMY_EXPORT int emmy_ops_rotary(const emmy_ops_rotary_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (!known_dtype(a->dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", a->dtype);
    if (a->rotary < 2 || a->rotary % 2 || a->rotary > a->dim || a->dim > 8192)
        return ops_fail(EMMY_RT_EINVAL, "rotary %d of dim %d", a->rotary, a->dim);
    if (a->layout != EMMY_OPS_ROTARY_HALF && a->layout != EMMY_OPS_ROTARY_INTERLEAVED)
        return ops_fail(EMMY_RT_EINVAL, "layout %d", a->layout);
    if (a->tokens < 0 || a->tokens > 0x7fffffffLL) return ops_fail(EMMY_RT_EINVAL, "tokens %lld", (long long)a->tokens);
    if (a->heads[0] < 0 || a->heads[1] < 0 || (int64_t)(a->heads[0] + (int64_t)a->heads[1]) * a->dim > (1 << 24))
        return ops_fail(EMMY_RT_EINVAL, "heads %d and %d", a->heads[0], a->heads[1]);
    if (a->tokens == 0 || (a->heads[0] == 0 && a->heads[1] == 0)) return 0;
    if (!a->positions || !a->turns || !aligned(a->positions, a->positions_64 ? 8 : 4) || !aligned(a->turns, 8))
        return ops_fail(EMMY_RT_EINVAL, "positions and turns are needed, aligned to their elements");
    const int es = elem_size(a->dtype);
    RotaryParams p = {};
    int bytes = 16;
    bool copies = false;
    for (int i = 0; i < 2; ++i) {
        p.heads[i] = a->heads[i];
        if (!a->heads[i]) continue;
        if (!a->x[i] || !a->out[i] || !aligned(a->x[i], es) || !aligned(a->out[i], es))
            return ops_fail(EMMY_RT_EINVAL, "x and out are needed, aligned to their elements");
        const int64_t strides[] = {a->x_token[i], a->x_head[i], a->out_token[i], a->out_head[i]};
        while (bytes > es) {
            bool ok = aligned(a->x[i], bytes) && aligned(a->out[i], bytes);
            for (int64_t s : strides) ok = ok && s * es % bytes == 0;
            if (ok) break;
            bytes = bytes == 16 && es == 2 ? 4 : es;
        }
        p.x[i] = (const char *)(uintptr_t)a->x[i];
        p.out[i] = (char *)(uintptr_t)a->out[i];
        p.x_token[i] = a->x_token[i], p.x_head[i] = a->x_head[i];
        p.out_token[i] = a->out_token[i], p.out_head[i] = a->out_head[i];
        copies |= a->x[i] != a->out[i] || a->x_token[i] != a->out_token[i] || a->x_head[i] != a->out_head[i];
    }
    const int pairs = a->rotary / 2;
    p.pairs = Divisor(pairs);
    p.rest = a->dim - a->rotary;
    while (bytes > es && (pairs % (bytes / es) || p.rest % (bytes / es))) bytes = bytes == 16 && es == 2 ? 4 : es;
    p.positions = (const void *)(uintptr_t)a->positions;
    p.turns = (const uint64_t *)(uintptr_t)a->turns;
    p.tokens = a->tokens, p.positions_64 = a->positions_64 != 0, p.transpose = a->transpose != 0;
    p.magnitude = a->magnitude;
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    cudaError_t e;
    if (a->dtype == EMMY_OPS_F32)
        e = bytes == 16 ? go<float, 4>(p, a->layout, copies, sms, stream) : go<float, 1>(p, a->layout, copies, sms, stream);
    else if (a->dtype == EMMY_OPS_F16)
        e = bytes == 16  ? go<__half, 8>(p, a->layout, copies, sms, stream)
            : bytes == 4 ? go<__half, 2>(p, a->layout, copies, sms, stream)
                         : go<__half, 1>(p, a->layout, copies, sms, stream);
    else
        e = bytes == 16  ? go<__nv_bfloat16, 8>(p, a->layout, copies, sms, stream)
            : bytes == 4 ? go<__nv_bfloat16, 2>(p, a->layout, copies, sms, stream)
                         : go<__nv_bfloat16, 1>(p, a->layout, copies, sms, stream);
    return ops_cuda(e, "rotary");
}
