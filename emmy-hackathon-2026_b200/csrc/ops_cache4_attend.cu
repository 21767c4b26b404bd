/*
 * Attention over the paged 4-bit cache.
 *
 * For one key / value head the queries are the rows (token, head of the group); with n the
 * levels, s and z the steps and least values of a cached token t:
 *
 *     score[t, r] = scale * (s_k[t] * sum_d q[r, d] n_k[t, d] + z_k[t] * sum_d q[r, d])
 *     out[r, d]   = (sum_t (p[t, r] s_v[t]) n_v[t, d] + sum_t p[t, r] z_v[t]) / sum_t p[t, r]
 *
 * so the products run on the bare levels, and steps and least values are applied to the
 * scores and probabilities, once per token instead of once per element.
 *
 * The bytes of the cache bound it: a token is (dim / 2 + 4) * 2 bytes per head.  A level in
 * bits 0..3 of a 16-bit half IS an f16 number, level * 2^-24 (a subnormal one), and one in
 * bits 4..7 is level * 2^-20; the tensor cores multiply subnormal f16 exactly.  So unpacking a key
 * is one AND per two elements and one shift per eight, with no conversion; the powers of two
 * are put into q's odd elements and into the results.  The queries are scaled by a power of
 * two per row so that their largest element is just below 2^14, which leaves f16 no less exact
 * than the 16-bit type they come in.
 *
 * Products are transposed: keys and values are the left operand (m16 n8 k16), queries the
 * right one, so a group of 8 rows fills the narrow side and no half of a tile is idle.
 * S^T = K Q^T has tokens as rows; movmatrix turns P^T into the right operand of
 * O^T = V^T P^T.  The order of the dims in Q K^T and of the tokens in V^T P^T is free, and is
 * chosen so that each thread's share of a token is consecutive bytes.
 *
 * Work is a list of tiles of 128 tokens over all (sequence, head, group of rows), cut into
 * equal runs, one for each block, whatever the lengths are.  A block's two warps take 64
 * tokens of each tile with their own running maxima and sums and their own ring of
 * asynchronous copies, and join at the end of a sequence; a sequence that runs over several
 * blocks leaves 32-bit partial sums in the workspace, which a second kernel joins in order.
 * 64 sequences of up to 16384 tokens (10500 on average), 8 heads of 128 under 32, take 151 us (4.8 TB/s; the loads alone 128); one
 * of 1000 tokens takes 6.9 us, most of it the chain from lengths to pages to tokens, twice.  All of a tile's tokens are
 * computed for all rows, and every 8 or 16 rows read the cache again, so a prompt is far from what it could be: 2048 tokens
 * over 8192 held ones take 1.6 ms, 195 TFLOP/s of what they see.
 */
#include "ops_common.cuh"

int ops_check_cache4(const emmy_ops_cache4 &c);

namespace {

constexpr int WARPS = 2, WARP_TOKENS = 64, TILE = WARPS * WARP_TOKENS, STAGES = 2, MT = WARP_TOKENS / 16;
/* what registers and shared memory let an SM hold of 8-row and of 16-row blocks */
template <int NT> constexpr int BLOCKS_PER_SM = NT == 1 ? 6 : 4;
constexpr int MAX_BATCH = 4096;
constexpr uint32_t NOT_FINITE = 0x7c00;      /* magnitudes of f16 from here on are infinity and NaN */

struct AttendParams {
    const char *k, *v;
    const __half2 *k_meta, *v_meta;
    const char *q;
    char *out;
    const int32_t *table, *lengths;
    float *partial;                     /* [blocks][2][rows][dim], then [blocks][2][rows][2] (max, sum) */
    int64_t pages, q_batch, q_token, q_head, out_batch, out_token, out_head, table_stride;
    int batch, tokens, heads, group, row_groups, page, max_positions;
    uint32_t page_inverse, page_shift;  /* position / page without a division */
    int q_wide, out_wide;               /* rows allow accesses of 16 and of 8 bytes */
    float scale_log2;
};

/* where tile `t` of the list lies */
struct Place {
    int sequence, head, row_group, tile, tiles, length;
};

__device__ __forceinline__ int sequence_length(const AttendParams &p, int b) {
    return max(0, min(p.lengths[b], p.max_positions));
}
__device__ __forceinline__ int sequence_tiles(int length) { return max(1, (length + TILE - 1) / TILE); }

/* exclusive sums of the sequences' tiles into shared memory; all threads of the block */
__device__ __forceinline__ int sum_tiles(const AttendParams &p, int32_t *before, int *warp_sums) {
    int carry = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    for (int base = 0; base < p.batch; base += blockDim.x) {
        const int b = base + threadIdx.x;
        const int own = b < p.batch ? sequence_tiles(sequence_length(p, b)) : 0;
        int upto = own;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(~0u, upto, d);
            if (lane >= d) upto += o;
        }
        if (lane == 31) warp_sums[warp] = upto;
        __syncthreads();
        int pre = carry, all = 0;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) pre += warp_sums[w];
            all += warp_sums[w];
        }
        if (b < p.batch) before[b] = pre + upto - own;
        carry += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) before[p.batch] = carry;
    __syncthreads();
    return carry;
}

/* The list's tiles in equal runs: block i's starts at i * each + min(i, more). */
struct Runs {
    int each, more;
    __device__ Runs(int tiles, int blocks) : each(tiles / blocks), more(tiles - tiles / blocks * blocks) {}
    __device__ int start(int block) const { return block * each + min(block, more); }
    /* the block that has tile t */
    __device__ int of(int t) const {
        const int edge = more * (each + 1);
        return t < edge ? t / (each + 1) : more + (t - edge) / max(each, 1);
    }
};

__device__ __forceinline__ Place find(const AttendParams &p, const int32_t *before, int t) {
    const int per = p.heads * p.row_groups;
    int lo = 0, hi = p.batch - 1;
    while (lo < hi) {                   /* the last sequence that starts at or before t */
        const int mid = (lo + hi + 1) / 2;
        if (before[mid] * per <= t) lo = mid; else hi = mid - 1;
    }
    Place at;
    at.sequence = lo;
    at.tiles = before[lo + 1] - before[lo];
    const int r = t - before[lo] * per, segment = r / at.tiles;
    at.tile = r - segment * at.tiles;
    at.head = segment / p.row_groups;
    at.row_group = segment - at.head * p.row_groups;
    at.length = sequence_length(p, lo);
    return at;
}

__device__ __forceinline__ void advance(const AttendParams &p, const int32_t *before, Place &at) {
    if (++at.tile < at.tiles) return;
    at.tile = 0;
    if (++at.row_group < p.row_groups) return;
    at.row_group = 0;
    if (++at.head < p.heads) return;
    at.head = 0;
    if (++at.sequence >= p.batch) return;
    at.tiles = before[at.sequence + 1] - before[at.sequence];
    at.length = sequence_length(p, at.sequence);
}

__device__ __forceinline__ void copy16(uint32_t to, const void *from, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void *from, bool live) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
/* d = a b */
__device__ __forceinline__ void mma_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %0;" : "+r"(v));
    return v;
}
__device__ __forceinline__ uint32_t packed(float low, float high) {
    const __half2 h = __floats2half2_rn(low, high);
    return *(const uint32_t *)&h;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ float reciprocal_approx(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* The token that row r (0 .. 7) of an eight-token group stands for.  A warp reads a token's keys by
 * r = lane / 4 and its values by the pairs r = 2 (lane % 4) + {0, 1}; these orders (with the
 * swizzle below at dim 128) put both into different banks. */
template <int DIM> __device__ __forceinline__ int token_of(int r) {
    return DIM == 128 ? r ^ ((r >> 1) & 1) : (r & 1 ? 4 + ((r >> 1) ^ 2) : r >> 1);
}
template <int DIM> __device__ __forceinline__ int swizzled(int token, int byte) {
    return DIM == 128 ? byte ^ ((token & 4) << 3) : byte;
}

template <int DIM> struct alignas(16) Stage {
    unsigned char k[WARP_TOKENS * DIM / 2], v[WARP_TOKENS * DIM / 2];
    __half2 k_meta[WARP_TOKENS], v_meta[WARP_TOKENS];
    uint64_t held;                      /* bit t: token t is in the sequence, on a page of the cache */
};

/* a token's (step, step, least, least) in f32, for instructions that work on pairs */
struct Doubled {
    ulonglong2 k, v;
};
static_assert(sizeof(Doubled) * WARP_TOKENS <= sizeof(Stage<64>::k), "they take the place of keys that have been read");

template <int DIM, int NT> struct Shared {
    Stage<DIM> ring[WARPS][STAGES];     /* a warp's partial results lie in the stage that it used last */
    float top[WARPS][8 * NT], sum[WARPS][8 * NT];
    int warp_sums[WARPS];
    int32_t before[];
};

template <typename T, int DIM, int NT, bool WHOLE>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS_PER_SM<NT>) cache4_attend(AttendParams p) {
    extern __shared__ __align__(16) unsigned char raw[];
    Shared<DIM, NT> &sh = *(Shared<DIM, NT> *)raw;
    constexpr int ROWS = 8 * NT, WORDS = DIM / 32, ROW_BYTES = DIM / 2, OT = DIM / 16, OUT_ROW = DIM + 4;
    static_assert(ROWS * OUT_ROW * 4 <= (int)sizeof(Stage<DIM>), "a stage holds a warp's results");
    /* p s_v goes to f16, off by up to 2^-12 of itself.  Of an f16 result that was 3.2e-4 of the norm beside 2.1e-4 from the result's
     * own rounding, so there sum p and sum p z take the p that the rounded product stands for: what is left is 2^-12 of the values'
     * distance from their mean (2.5e-4 in all at 16 sequences of up to 5000).  A bf16 result keeps the 2^-12 of p s n: 1.687e-3 of
     * the norm in all, where its own rounding alone is 1.658e-3 (64 sequences of up to 16384).  Both halves of p s_v in the
     * products would leave 1.660e-3 and take 14 us of 150 more. */
    constexpr bool EXACT = sizeof(T) == 2 && !__is_same(T, __nv_bfloat16);
    /* the join may start only when what this kernel waits for is there: it reads the lengths before it waits */
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int total = sum_tiles(p, sh.before, sh.warp_sums);
    const Runs runs(total * p.heads * p.row_groups, gridDim.x);
    const int first = runs.start(blockIdx.x), last = runs.start(blockIdx.x + 1);
    if (first >= last) return;
    Place ahead = find(p, sh.before, first), at = ahead;
    int issued = first;

    /* The copies' side.  rows: where this lane's tokens (lane and lane + 32) lie in the cache (rows of pages x heads x
     * page), -1 for nowhere.  WHOLE: pages are a multiple of a warp's tokens, which then are consecutive rows of
     * one page: rows[0] is the first one's, the same for all lanes, and rows behind a sequence's end come along. */
    auto lookup = [&](const Place &place, int i) -> int64_t {
        const int position = place.tile * TILE + warp * WARP_TOKENS + (WHOLE ? 0 : lane + 32 * i);
        if (position >= place.length) return -1;
        const int page = p.page_inverse ? __umulhi(position, p.page_inverse) >> p.page_shift : position;
        const int64_t index = p.table[place.sequence * p.table_stride + page];
        if (index < 0 || index >= p.pages) return -1;
        return (index * p.heads + place.head) * p.page + (position - page * p.page);
    };
    int64_t rows[2];
    auto look = [&] {
        rows[0] = lookup(ahead, 0);
        if (!WHOLE) rows[1] = lookup(ahead, 1);
    };
    look();
    auto issue = [&](int stage) {
        if (issued < last) {
            Stage<DIM> &s = sh.ring[warp][stage];
            constexpr int CHUNKS = ROW_BYTES / 16, PER = 32 / CHUNKS;     /* an access of the warp: PER tokens */
            const uint32_t k_to = (uint32_t)__cvta_generic_to_shared(s.k), v_to = (uint32_t)__cvta_generic_to_shared(s.v);
            const uint32_t k_meta_to = (uint32_t)__cvta_generic_to_shared(&s.k_meta[lane]);
            const uint32_t v_meta_to = (uint32_t)__cvta_generic_to_shared(&s.v_meta[lane]);
            uint64_t held;
            if (WHOLE) {
                const int left = ahead.length - ahead.tile * TILE - warp * WARP_TOKENS;
                held = rows[0] < 0 ? 0 : left >= 64 ? ~0ull : (1ull << left) - 1;
                if (rows[0] >= 0) {
                    const int64_t offset = rows[0] * ROW_BYTES + lane * 16;
                    const char *k = p.k + offset, *v = p.v + offset;
                    const uint32_t to = lane / CHUNKS * ROW_BYTES + swizzled<DIM>(lane / CHUNKS, lane % CHUNKS * 16);
#pragma unroll
                    for (int i = 0; i < WARP_TOKENS / PER; ++i) {
                        copy16(k_to + to + i * 512, k + i * 512, true);
                        copy16(v_to + to + i * 512, v + i * 512, true);
                    }
                    const __half2 *k_meta = p.k_meta + rows[0] + lane, *v_meta = p.v_meta + rows[0] + lane;
                    copy4(k_meta_to, k_meta, true), copy4(k_meta_to + 128, k_meta + 32, true);
                    copy4(v_meta_to, v_meta, true), copy4(v_meta_to + 128, v_meta + 32, true);
                }
            } else {
#pragma unroll
                for (int i = 0; i < WARP_TOKENS / PER; ++i) {
                    const int token = i * PER + lane / CHUNKS, byte = lane % CHUNKS * 16;
                    const int64_t from = __shfl_sync(~0u, rows[i * PER / 32], token & 31);
                    const uint32_t to = token * ROW_BYTES + swizzled<DIM>(token, byte);
                    const int64_t offset = (from < 0 ? 0 : from) * ROW_BYTES + byte;
                    copy16(k_to + to, p.k + offset, from >= 0);
                    copy16(v_to + to, p.v + offset, from >= 0);
                }
                held = __ballot_sync(~0u, rows[0] >= 0) | (uint64_t)__ballot_sync(~0u, rows[1] >= 0) << 32;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    copy4(k_meta_to + 128 * i, p.k_meta + (rows[i] < 0 ? 0 : rows[i]), rows[i] >= 0);
                    copy4(v_meta_to + 128 * i, p.v_meta + (rows[i] < 0 ? 0 : rows[i]), rows[i] >= 0);
                }
            }
            if (lane == 0) s.held = held;
            if (++issued < last) {
                advance(p, sh.before, ahead);
                look();
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int s = 0; s < STAGES - 1; ++s) issue(s);

    uint32_t qf[NT][2 * WORDS][2];
    Two o[NT][OT][2];
    float top[NT][2];
    Two least[NT], sum[NT], by[NT], base[NT];
    int sees[NT][2];
    int v_exponent = 0, all_see = 0;
    int segment_start = first, stage = 0;
    for (int t = first; t < last; ++t) {
        if (t == first || at.tile == 0) {
            /* a new (sequence, head, group of rows): its queries */
            segment_start = t;
            v_exponent = -16;
            all_see = at.length - p.tokens + 1;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int own = at.row_group * ROWS + n * 8 + r, rows = p.tokens * p.group;
                float v[8 * WORDS], largest = 0.0f, all = 0.0f;
                const int token = own / p.group;
                if (own < rows) {
                    const T *q = (const T *)p.q + at.sequence * p.q_batch + token * p.q_token +
                                 (int64_t)(at.head * p.group + own - token * p.group) * p.q_head + c * 8 * WORDS;
                    if (p.q_wide) {
#pragma unroll
                        for (int w = 0; w < WORDS; ++w) {
                            const Pack<T, 8> x = *(const Pack<T, 8> *)(q + 8 * w);
#pragma unroll
                            for (int i = 0; i < 8; ++i) v[8 * w + i] = to_f32(x.at[i]);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8 * WORDS; ++i) v[i] = to_f32(q[i]);
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8 * WORDS; ++i) v[i] = 0.0f;
                }
#pragma unroll
                for (int i = 0; i < 8 * WORDS; ++i) largest = fmaxf(largest, fabsf(v[i])), all += v[i];
#pragma unroll
                for (int d = 1; d < 4; d <<= 1) {
                    largest = fmaxf(largest, __shfl_xor_sync(~0u, largest, d));
                    all += __shfl_xor_sync(~0u, all, d);
                }
                const float sign = p.scale_log2 < 0.0f ? -1.0f : 1.0f;
                const int exponent = max((int)(__float_as_uint(largest) >> 23) - 127, -100);
                const float up = __uint_as_float((uint32_t)(127 + 13 - min(exponent, 127)) << 23);
#pragma unroll
                for (int w = 0; w < WORDS; ++w)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int e = 8 * w + 2 * i;
                        const float low = sign * up, high = low * 0x1p-4f;
                        qf[n][2 * w + i][0] = packed(v[e] * low, v[e + 4] * low);
                        qf[n][2 * w + i][1] = packed(v[e + 1] * high, v[e + 5] * high);
                    }
                /* of the rows that this thread has in the scores: 2 c and 2 c + 1 */
                const float mine = fmaxf(fabsf(p.scale_log2) / up, 0x1p-126f), mine0 = sign * up * all;
                by[n] = Two(__shfl_sync(~0u, mine, 8 * c), __shfl_sync(~0u, mine, 8 * c + 4));
                base[n] = Two(__shfl_sync(~0u, mine0, 8 * c), __shfl_sync(~0u, mine0, 8 * c + 4));
                sum[n] = least[n] = Two(0.0f, 0.0f);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = at.row_group * ROWS + n * 8 + 2 * c + i;
                    sees[n][i] = row < rows ? at.length - p.tokens + row / p.group + 1 : 0;
                    top[n][i] = -INFINITY;
                }
#pragma unroll
                for (int i = 0; i < OT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[n][i][j] = Two(0.0f, 0.0f);
            }
        }
        issue((stage + STAGES - 1) % STAGES);
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();
        Stage<DIM> &s = sh.ring[warp][stage];
        /* S^T = K Q^T, in two independent chains of products at a time */
        float score[MT][NT][4];
#pragma unroll
        for (int m = 0; m < MT; m += 2) {
            Pack<uint32_t, WORDS> x[2][2];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int token = 16 * (m + j) + 8 * h + token_of<DIM>(r);
                    x[j][h] = *(const Pack<uint32_t, WORDS> *)(s.k + token * ROW_BYTES + swizzled<DIM>(token, c * 4 * WORDS));
                }
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t a = x[j][0].at[w] >> 8 * i, b = x[j][1].at[w] >> 8 * i;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint32_t *q = qf[n][2 * w + i];
                            if (w + i == 0)
                                mma_first(score[m + j][n], a & 0x000f000f, b & 0x000f000f, a & 0x00f000f0, b & 0x00f000f0, q[0], q[1]);
                            else
                                mma(score[m + j][n], a & 0x000f000f, b & 0x000f000f, a & 0x00f000f0, b & 0x00f000f0, q[0], q[1]);
                        }
                    }
        }
        /* p times the value's step goes to f16: a power of two brings the largest step met so far near 2^14, so a product is lost
         * below 2^-39 of that step */
        float rescale = 1.0f;
        /* A hidden token's probability is 0, and 0 times infinity is no 0: where a value of such a tile is not finite, the
         * products leave it out, and the rows that see it take it by itself. */
        bool guarded = false;
        Doubled *const doubled = (Doubled *)s.k;
        __syncwarp();                   /* all lanes are done with the keys */
        {
            const bool lives[2] = {(s.held >> lane & 1) != 0, (s.held >> (lane + 32) & 1) != 0};
            const __half2 vm[2] = {s.v_meta[lane], s.v_meta[lane + 32]}, zero = __halves2half2(__half(), __half());
            __half2 of_v[2] = {lives[0] ? vm[0] : zero, lives[1] ? vm[1] : zero};
            /* the largest step's bits; NOT_FINITE and more where a step or a least value is infinite or NaN */
            auto step_bits = [&](int i) { return (uint32_t)__half_as_ushort(__low2half(of_v[i])) & 0x7fff; };
            auto least_bits = [&](int i) { return (uint32_t)__half_as_ushort(__high2half(of_v[i])) & 0x7fff; };
            auto either = [&](int i) { return least_bits(i) >= NOT_FINITE ? NOT_FINITE : step_bits(i); };
            uint32_t bits = __reduce_max_sync(~0u, max(either(0), either(1)));
            if (bits >= NOT_FINITE) {
                guarded = s.held != ~0ull || at.tile * TILE + (warp + 1) * WARP_TOKENS > all_see;
                uint32_t finite = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (step_bits(i) < NOT_FINITE) finite = max(finite, step_bits(i));
                    if (guarded && max(step_bits(i), least_bits(i)) >= NOT_FINITE) of_v[i] = zero;
                }
                bits = __reduce_max_sync(~0u, finite);
            }
            const int exponent = (int)(bits >> 10) - 15;
            if (exponent > v_exponent) {
                rescale = v_exponent < -15 ? 1.0f : exp2_approx((float)(v_exponent - exponent));
                v_exponent = exponent;
            }
            const float up = __uint_as_float((uint32_t)(127 + 14 - v_exponent) << 23);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float2 k = __half22float2(s.k_meta[lane + 32 * i]), v = __half22float2(of_v[i]);
                const float k_step = k.x * 0x1p24f, v_step = v.x * up;
                Doubled &to = doubled[lane + 32 * i];
                to.k = make_ulonglong2(Two(k_step, k_step).v, Two(k.y, k.y).v);
                to.v = make_ulonglong2(Two(v_step, v_step).v, Two(v.y, v.y).v);
            }
            __syncwarp();
        }
        /* logits to base 2, all but the factor `by` of their row, and the running maximum */
        const int from = at.tile * TILE + warp * WARP_TOKENS;
        const uint64_t held = s.held;
        const bool full = held == ~0ull && from + WARP_TOKENS <= all_see;      /* nothing is hidden from any row */
        float next[NT][2], shrink[NT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const ulonglong2 k = doubled[16 * m + 8 * h + token_of<DIM>(r)].k;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float *x = &score[m][n][2 * h];
                    const float2 y = fma2(Two(k.x), Two(x[0], x[1]), Two(k.y) * base[n]).get();
                    x[0] = y.x, x[1] = y.y;
                }
            }
        if (!full) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int token = 16 * m + 8 * h + token_of<DIM>(r);
                    const int place = held >> token & 1 ? from + token : 0x7fffffff;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (place >= sees[n][i]) score[m][n][2 * h + i] = -INFINITY;
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                next[n][i] = top[n][i];
#pragma unroll
                for (int m = 0; m < MT; ++m) next[n][i] = fmaxf(next[n][i], fmaxf(score[m][n][i], score[m][n][2 + i]));
            }
        Two minus[NT];                  /* less the maximum, in the exponent */
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float2 f = by[n].get();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) next[n][i] = fmaxf(next[n][i], __shfl_xor_sync(~0u, next[n][i], d));
                const float ref = next[n][i] == -INFINITY ? 0.0f : next[n][i];
                shrink[n][i] = exp2_approx((top[n][i] - ref) * (i ? f.y : f.x));
                top[n][i] = next[n][i];
                next[n][i] = -ref * (i ? f.y : f.x);
            }
            minus[n] = Two(next[n][0], next[n][1]);
        }
        Two keep[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const Two f(shrink[n][0], shrink[n][1]);
            sum[n] = sum[n] * f;
            least[n] = least[n] * f;
            keep[n] = f * Two(rescale, rescale);
        }
        if (guarded) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int token = 16 * m + 8 * h + token_of<DIM>(r);
                    const float2 v = __half22float2(s.v_meta[token]);
                    if (!(held >> token & 1) || (fabsf(v.x) < INFINITY && fabsf(v.y) < INFINITY)) continue;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 x = fma2(by[n], Two(score[m][n][2 * h], score[m][n][2 * h + 1]), minus[n]).get();
                        least[n] = least[n] + Two(from + token < sees[n][0] ? exp2_approx(x.x) * (v.x + v.y) : 0.0f,
                                                  from + token < sees[n][1] ? exp2_approx(x.y) * (v.x + v.y) : 0.0f);
                    }
                }
        }
        uint32_t pf[MT][NT][2];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const ulonglong2 v = doubled[16 * m + 8 * h + token_of<DIM>(r)].v;
                const float inverse = EXACT ? reciprocal_approx(Two(v.x).get().x) : 0.0f;      /* off by 2^-23: as p itself */
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 x = fma2(by[n], Two(score[m][n][2 * h], score[m][n][2 * h + 1]), minus[n]).get();
                    float e[2] = {exp2_approx(x.x), exp2_approx(x.y)};
                    const float2 y = (Two(e[0], e[1]) * Two(v.x)).get();
                    const __half2 ps = __floats2half2_rn(y.x, y.y);
                    pf[m][n][h] = transposed(*(const uint32_t *)&ps);
                    if (EXACT) {
                        const float2 rounded = __half22float2(ps);
                        if (rounded.x >= 0x1p-14f) e[0] = rounded.x * inverse;
                        if (rounded.y >= 0x1p-14f) e[1] = rounded.y * inverse;
                    }
                    const Two e2(e[0], e[1]);
                    sum[n] = sum[n] + e2;
                    least[n] = fma2(e2, Two(v.y), least[n]);
                }
            }
        /* V^T P^T of the tile.  The tensor cores' sums lose what lies below their last bit, always towards zero; kept over a
         * run of 147 tiles that was 3.4e-5 of sum p s n, or 2 % of a result that sum p z nearly cancels (131072 positions).  So a
         * tile's sums are its own, and join the others by instructions that round to nearest (149 -> 151 us; 157 with all of 128
         * dims at a time, whose sums registers do not hold beside the others). */
        constexpr int PARTS = DIM == 128 ? 2 : 1, WORDS_EACH = WORDS / 2 / PARTS;      /* dims in parts */
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
            float fresh[NT][OT / PARTS][4];
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                Pack<uint32_t, WORDS_EACH> x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = 16 * m + 8 * (i >> 1) + token_of<DIM>(2 * c + (i & 1));
                    x[i] = *(const Pack<uint32_t, WORDS_EACH> *)(s.v + token * ROW_BYTES + swizzled<DIM>(token, r * 2 * WORDS) + 4 * WORDS_EACH * part);
                }
#pragma unroll
                for (int w = 0; w < WORDS_EACH; ++w)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const uint32_t a = __byte_perm(x[0].at[w], x[1].at[w], half ? 0x7632 : 0x5410);
                        const uint32_t b = __byte_perm(x[2].at[w], x[3].at[w], half ? 0x7632 : 0x5410);
                        /* bytes 0 and 2, then 1 and 3; the even dim's level alone, and the whole byte,
                         * 16 times the odd dim's level more: the even sum is taken out at the end */
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const uint32_t u = __byte_perm(a, 0, i ? 0x4341 : 0x4240), v = __byte_perm(b, 0, i ? 0x4341 : 0x4240);
                            const int d = 4 * w + 2 * half + i;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                if (m == 0)
                                    mma_first(fresh[n][d], u & 0x000f000f, u, v & 0x000f000f, v, pf[m][n][0], pf[m][n][1]);
                                else
                                    mma(fresh[n][d], u & 0x000f000f, u, v & 0x000f000f, v, pf[m][n][0], pf[m][n][1]);
                                if (m == MT - 1)
#pragma unroll
                                    for (int j = 0; j < 2; ++j) {
                                        Two &to = o[n][OT / PARTS * part + d][j];
                                        to = fma2(to, keep[n], Two(fresh[n][d][2 * j], fresh[n][d][2 * j + 1]));
                                    }
                            }
                        }
                    }
            }
        }
        __syncwarp();                   /* all lanes are done with the stage before it is filled again */

        if (at.tile + 1 == at.tiles || t + 1 == last) {
            /* the warps' sums joined */
            const float down = __uint_as_float((uint32_t)(127 - 14 + v_exponent) << 23);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float2 s2 = sum[n].get(), l2 = least[n].get(), f2 = by[n].get();
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float all = i ? s2.y : s2.x, bottom = i ? l2.y : l2.x;
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) {
                        all += __shfl_xor_sync(~0u, all, d);
                        bottom += __shfl_xor_sync(~0u, bottom, d);
                    }
                    if (r == 0) {
                        sh.top[warp][8 * n + 2 * c + i] = top[n][i] == -INFINITY ? -INFINITY : top[n][i] * (i ? f2.y : f2.x);
                        sh.sum[warp][8 * n + 2 * c + i] = all;
                    }
                    /* this thread's dims: 2 OT from 2 OT r on, of row 2 c + i */
                    float *to = (float *)&sh.ring[warp][stage] + (8 * n + 2 * c + i) * OUT_ROW + 2 * OT * r;
#pragma unroll
                    for (int j = 0; j < OT; ++j) {
                        const float2 even = o[n][j][0].get(), whole = o[n][j][1].get();
                        const float a = i ? even.y : even.x, b = i ? whole.y : whole.x;
                        to[2 * j] = fmaf(a * 0x1p24f, down, bottom);
                        to[2 * j + 1] = fmaf((b - a) * 0x1p20f, down, bottom);
                    }
                }
            }
            __syncthreads();
            const bool whole = at.tile + 1 == at.tiles && t - segment_start + 1 == at.tiles;
            const int rows = p.tokens * p.group;
            const int64_t slot = (int64_t)blockIdx.x * 2 + (segment_start != first);
            for (int i = threadIdx.x; i < ROWS * DIM / 4; i += WARPS * 32) {
                const int n = i / (DIM / 4), e = i % (DIM / 4) * 4, own = at.row_group * ROWS + n;
                float high = -INFINITY;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) high = fmaxf(high, sh.top[w][n]);
                const float ref = high == -INFINITY ? 0.0f : high;
                float all = 0.0f;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    const float f = exp2_approx(sh.top[w][n] - ref);
                    const float4 x = *(const float4 *)((const float *)&sh.ring[w][stage] + n * OUT_ROW + e);
                    all = fmaf(f, sh.sum[w][n], all);
                    v.x = fmaf(f, x.x, v.x), v.y = fmaf(f, x.y, v.y), v.z = fmaf(f, x.z, v.z), v.w = fmaf(f, x.w, v.w);
                }
                if (whole) {
                    if (own < rows) {
                        const float inv = all > 0.0f || all != all ? 1.0f / all : 0.0f;
                        const int token = own / p.group;
                        T *out = (T *)p.out + at.sequence * p.out_batch + token * p.out_token +
                                 (int64_t)(at.head * p.group + own - token * p.group) * p.out_head + e;
                        const Pack<T, 4> y = {from_f32<T>(v.x * inv), from_f32<T>(v.y * inv), from_f32<T>(v.z * inv),
                                              from_f32<T>(v.w * inv)};
                        if (p.out_wide)
                            *(Pack<T, 4> *)out = y;
                        else
                            out[0] = y.at[0], out[1] = y.at[1], out[2] = y.at[2], out[3] = y.at[3];
                    }
                } else {
                    *(float4 *)(p.partial + (slot * ROWS + n) * DIM + e) = v;
                    if (e == 0) {
                        float *stat = p.partial + (int64_t)gridDim.x * 2 * ROWS * DIM + (slot * ROWS + n) * 2;
                        stat[0] = high, stat[1] = all;
                    }
                }
            }
            __syncthreads();
        }
        stage = (stage + 1) % STAGES;
        if (t + 1 < last) advance(p, sh.before, at);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

/* joins the runs of a segment that several blocks of the first kernel shared, in their order */
template <typename T, int DIM, int NT>
__global__ void __launch_bounds__(128) cache4_join(AttendParams p, int blocks) {
    constexpr int ROWS = 8 * NT;
    __shared__ int sums[2][4];
    __shared__ float tops[4], totals[4], parts[4][DIM];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int per = p.heads * p.row_groups, sequence = blockIdx.x / per, segment = blockIdx.x - sequence * per;
    int before = 0, total = 0;
    for (int b = threadIdx.x; b < p.batch; b += 128) {
        const int n = sequence_tiles(sequence_length(p, b));
        total += n;
        if (b < sequence) before += n;
    }
    before = __reduce_add_sync(~0u, before);
    total = __reduce_add_sync(~0u, total);
    if ((threadIdx.x & 31) == 0) sums[0][threadIdx.x >> 5] = before, sums[1][threadIdx.x >> 5] = total;
    __syncthreads();
    before = sums[0][0] + sums[0][1] + sums[0][2] + sums[0][3];
    total = sums[1][0] + sums[1][1] + sums[1][2] + sums[1][3];
    const Runs runs(total * per, blocks);
    const int own_tiles = sequence_tiles(sequence_length(p, sequence));
    const int start = before * per + segment * own_tiles;
    const int a = runs.of(start), z = runs.of(start + own_tiles - 1);
    asm volatile("griddepcontrol.wait;" ::: "memory");     /* the parts are written */
    if (a == z) return;
    const float *stats = p.partial + (int64_t)blocks * 2 * ROWS * DIM;
    const int head = segment / p.row_groups, row_group = segment - head * p.row_groups, rows = p.tokens * p.group;
    /* a row of the segment to each block of the grid's second dimension: its warps take every fourth run */
    const int n = blockIdx.y, own = row_group * ROWS + n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (own >= rows) return;
    constexpr int PER = DIM / 32;
    float high = -INFINITY, all = 0.0f, v[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) v[j] = 0.0f;
#pragma unroll 4
    for (int block = a + warp; block <= z; block += 4) {
        const int64_t slot = block * 2 + (runs.start(block) < start);
        const float2 stat = *(const float2 *)(stats + (slot * ROWS + n) * 2);
        const Pack<float, PER> x = *(const Pack<float, PER> *)(p.partial + (slot * ROWS + n) * DIM + lane * PER);
        const float top = stat.x, next = fmaxf(high, top), ref = next == -INFINITY ? 0.0f : next;
        const float f = exp2_approx(high - ref), g = exp2_approx(top - ref);
        all = fmaf(g, stat.y, all * f);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = fmaf(g, x.at[j], v[j] * f);
        high = next;
    }
    if (lane == 0) tops[warp] = high, totals[warp] = all;
#pragma unroll
    for (int j = 0; j < PER; ++j) parts[warp][lane * PER + j] = v[j];
    __syncthreads();
    float best = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w) best = fmaxf(best, tops[w]);
    const float ref = best == -INFINITY ? 0.0f : best;
    float sum = 0.0f, out = 0.0f;
    const int e = threadIdx.x;
    if (e >= DIM) return;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float f = exp2_approx(tops[w] - ref);
        sum = fmaf(f, totals[w], sum);
        out = fmaf(f, parts[w][e], out);
    }
    const int token = own / p.group;
    ((T *)p.out)[sequence * p.out_batch + token * p.out_token + (int64_t)(head * p.group + own - token * p.group) * p.out_head + e] =
        from_f32<T>(sum > 0.0f || sum != sum ? out / sum : 0.0f);
}

template <typename T, int DIM, int NT, bool WHOLE> int go(const AttendParams &p, int sms, int device, uint64_t stream) {
    const size_t smem = sizeof(Shared<DIM, NT>) + 4 * ((size_t)p.batch + 1);
    static uint64_t allowed;                 /* devices whose limit is raised */
    if (!(__atomic_load_n(&allowed, __ATOMIC_ACQUIRE) >> device & 1)) {
        cudaError_t e = cudaFuncSetAttribute(cache4_attend<T, DIM, NT, WHOLE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)(sizeof(Shared<DIM, NT>) + 4 * (MAX_BATCH + 1)));
        if (e != cudaSuccess) return ops_cuda(e, "shared memory of the attention");
        __atomic_fetch_or(&allowed, 1ull << device, __ATOMIC_RELEASE);
    }
    /* as many blocks as run at once: the list of a long batch takes shared memory too */
    const int fit = (int)((228 * 1024) / (smem + 1024)), blocks = sms * (fit < BLOCKS_PER_SM<NT> ? fit : BLOCKS_PER_SM<NT>);
    cudaError_t e = launch(cache4_attend<T, DIM, NT, WHOLE>, dim3(blocks), dim3(WARPS * 32), smem, stream, p);
    if (e != cudaSuccess) return ops_cuda(e, "attention over the 4-bit cache");
    e = launch(cache4_join<T, DIM, NT>, dim3((unsigned)(p.batch * p.heads * p.row_groups), 8 * NT), dim3(128), 0, stream, p, blocks);
    return ops_cuda(e, "joining the attention's parts");
}

template <typename T, int DIM> int by_shape(const AttendParams &p, int nt, int sms, int device, uint64_t stream) {
    if (p.page % WARP_TOKENS == 0)
        return nt == 1 ? go<T, DIM, 1, true>(p, sms, device, stream) : go<T, DIM, 2, true>(p, sms, device, stream);
    return nt == 1 ? go<T, DIM, 1, false>(p, sms, device, stream) : go<T, DIM, 2, false>(p, sms, device, stream);
}

uint64_t workspace(int sms, int dim) {
    const int rows = 8 * (BLOCKS_PER_SM<1> > 2 * BLOCKS_PER_SM<2> ? BLOCKS_PER_SM<1> : 2 * BLOCKS_PER_SM<2>);
    return (uint64_t)sms * rows * 2 * (dim + 2) * 4;
}

}  // namespace

EMMY_EXPORT int emmy_ops_cache4_attend_workspace(int dim, int device, uint64_t *bytes) {
    if (!bytes || (dim != 64 && dim != 128)) return ops_fail(EMMY_RT_EINVAL, "head dim %d is not 64 or 128", dim);
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    *bytes = workspace(sms, dim);
    return 0;
}

EMMY_EXPORT int emmy_ops_cache4_attend(const emmy_ops_cache4_attend_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (int e = ops_check_cache4(a->cache)) return e;
    if (a->dtype != EMMY_OPS_F16 && a->dtype != EMMY_OPS_BF16)
        return ops_fail(EMMY_RT_EINVAL, "element type %d: queries are f16 or bf16", a->dtype);
    if (a->batch < 0 || a->batch > MAX_BATCH) return ops_fail(EMMY_RT_EINVAL, "batch %d is not in 0 .. %d", a->batch, MAX_BATCH);
    if (a->tokens < 0 || a->q_heads < 1 || a->q_heads % a->cache.heads)
        return ops_fail(EMMY_RT_EINVAL, "%d tokens of %d heads over %d heads of the cache", a->tokens, a->q_heads, a->cache.heads);
    const int group = a->q_heads / a->cache.heads;
    if ((int64_t)a->tokens * group > (1 << 20)) return ops_fail(EMMY_RT_EINVAL, "%d tokens a sequence", a->tokens);
    if (a->max_pages < 0 || (int64_t)a->max_pages * a->cache.page > 0x7fffff00LL)
        return ops_fail(EMMY_RT_EINVAL, "%d pages of %d rows a sequence", a->max_pages, a->cache.page);
    if (a->batch == 0 || a->tokens == 0) return 0;
    if (!a->q || !a->out || !a->lengths || (a->max_pages && !a->table) || !a->workspace || !aligned(a->workspace, 16))
        return ops_fail(EMMY_RT_EINVAL, "q, out, table, lengths and a workspace (on 16 bytes) are needed");
    if (!aligned(a->q, 2) || !aligned(a->out, 2) || !aligned(a->table, 4) || !aligned(a->lengths, 4))
        return ops_fail(EMMY_RT_EINVAL, "an operand is not aligned to its elements");
    const int rows = a->tokens * group, nt = rows <= 8 ? 1 : 2;
    AttendParams p = {};
    p.k = (const char *)(uintptr_t)a->cache.k, p.v = (const char *)(uintptr_t)a->cache.v;
    p.k_meta = (const __half2 *)(uintptr_t)a->cache.k_meta, p.v_meta = (const __half2 *)(uintptr_t)a->cache.v_meta;
    p.q = (const char *)(uintptr_t)a->q, p.out = (char *)(uintptr_t)a->out;
    p.table = (const int32_t *)(uintptr_t)a->table, p.lengths = (const int32_t *)(uintptr_t)a->lengths;
    p.partial = (float *)(uintptr_t)a->workspace;
    p.pages = a->cache.pages;
    p.q_batch = a->q_batch, p.q_token = a->q_token, p.q_head = a->q_head;
    p.out_batch = a->out_batch, p.out_token = a->out_token, p.out_head = a->out_head, p.table_stride = a->table_stride;
    p.q_wide = aligned(a->q, 16) && !((p.q_batch | p.q_token | p.q_head) & 7);
    p.out_wide = aligned(a->out, 8) && !((p.out_batch | p.out_token | p.out_head) & 3);
    p.batch = a->batch, p.tokens = a->tokens, p.heads = a->cache.heads, p.group = group;
    p.row_groups = (rows + 8 * nt - 1) / (8 * nt), p.page = a->cache.page;
    p.max_positions = a->cache.pages ? a->max_pages * a->cache.page : 0;     /* nothing to see in a cache without pages */
    p.scale_log2 = (float)(a->scale * 1.4426950408889634);
    if ((int64_t)p.batch * p.heads * p.row_groups > 0x7fffffffLL / ((int64_t)p.max_positions / TILE + 1))
        return ops_fail(EMMY_RT_EINVAL, "%d sequences of %d positions are too many for one call", p.batch, p.max_positions);
    if (p.page > 1) {                   /* ceil(2^(31 + s) / page), 2^s >= page: exact below 2^31 */
        uint32_t shift = 1;
        while ((1u << shift) < (uint32_t)p.page) ++shift;
        p.page_inverse = (uint32_t)((((uint64_t)1 << (31 + shift)) + p.page - 1) / p.page);
        p.page_shift = shift - 1;
    }
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    if (a->workspace_bytes < workspace(sms, a->cache.dim))
        return ops_fail(EMMY_RT_ESCRATCH, "a workspace of %llu bytes is too small", (unsigned long long)a->workspace_bytes);
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    const bool f16 = a->dtype == EMMY_OPS_F16;
    if (a->cache.dim == 64)
        return f16 ? by_shape<__half, 64>(p, nt, sms, device, stream) : by_shape<__nv_bfloat16, 64>(p, nt, sms, device, stream);
    return f16 ? by_shape<__half, 128>(p, nt, sms, device, stream) : by_shape<__nv_bfloat16, 128>(p, nt, sms, device, stream);
}
