/*
 * FP8 (e4m3) products with a scale for each block of 128.
 *
 *     y[m, n] = sum_b sx[b, m] sw[n / 128, b] sum_{k in block b} xq[m, k] wq[n, k]
 *
 * x is quantised per row and 128 columns, W per 128 x 128 block:
 *     s = amax / 448 (1 where that is 0),  q = e4m3(v / s), nearest even.
 *
 * The row quantiser is bound by its issue slots as much as by its bytes (65 % and 52 %), few_rows (up to 16 rows of x) by waits for
 * W and by the conversions that mma.sync makes of e4m3, at half of what DRAM gives, and many_rows by the tensor cores and the
 * scaled sums beside them; join_parts adds up products that many_rows cut along k.
 */
#include "ops_common.cuh"
#include "ops_wait.cuh"

namespace {

constexpr int BLOCK = 128;
constexpr float E4M3_MAX = 448.0f;

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t low, high;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(d), "f"(c));
    return low | (uint32_t)high << 16;
}

/* |v| as an ordered integer: a NaN is the largest */
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
/* largest / 448, correctly rounded; 1 where that is 0 */
__device__ __forceinline__ float scale_of(uint32_t largest) {
    const float a = __uint_as_float(largest);
    constexpr float R = 1.0f / E4M3_MAX;
    if (a >= 0x1p-60f && a <= 0x1p100f) return quotient(a, E4M3_MAX, R);
    const float s = __fdiv_rn(a, E4M3_MAX);
    return s == 0.0f ? 1.0f : s;
}
/* of two 16-bit floats side by side: the larger magnitudes, each in its half */
__device__ __forceinline__ uint32_t larger2(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("max.u16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
template <typename T> __device__ __forceinline__ uint32_t largest_of(uint32_t two) {       /* as f32 bits */
    const uint32_t one = max(two & 0xffff, two >> 16);
    return sizeof(T) == 4 ? two : __float_as_uint(to_f32(*(const T *)&one));
}

template <typename T> __device__ __forceinline__ void load8(const T *x, int64_t e, int64_t end, bool wide, float (&v)[8]) {
    if (wide && e + 8 <= end) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += V) {
            const Pack<T, V> q = *(const Pack<T, V> *)(x + e + i);
#pragma unroll
            for (int j = 0; j < V; ++j) v[i + j] = to_f32(q.at[j]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = e + i < end ? to_f32(x[e + i]) : 0.0f;
    }
}

/* v / s for N values of a block's scale, two at a time.  With divisions the quantiser took 39 us for 4096 x 8192 in bf16, now 20 us
 * (5.1 TB/s). */
template <int N> __device__ __forceinline__ void divide(float (&v)[N], float s) {
    if (s >= 0x1p-60f && s <= 0x1p60f) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const Two both(v[i], v[i + 1]), q = both * Two(r, r);
            const float2 f = fma2(fma2(Two(-s, -s), q, both), Two(r, r), q).get();
            v[i] = f.x, v[i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fdiv_rn(v[i], s);
    }
}

/* ---- quantisers ---------------------------------------------------------------------- */

struct QuantRowsParams {
    const char *x;
    uint8_t *q;
    float *s;
    int64_t rows, cols, x_stride, q_stride, s_stride;
    int across;
};

/* 16 lanes a block of 128, eight elements each; 1 << across blocks of a row side by side in a block of threads, which
 * takes QUANT_ROWS rows for each of its 16 groups of lanes, all loads before the first use.  A: the elements of an
 * access, which rows, their ends and the pointer allow.  BARE: a single row that is not padded; asking every row for its end
 * took 4096 x 8192 from 20.2 to 22.0 us. */
constexpr int QUANT_ROWS = 4;
template <typename T, int A, bool BARE = false> __global__ void __launch_bounds__(256) quantize_rows(QuantRowsParams p) {
    enter_grid();
    const int group = threadIdx.x / 16, lane = threadIdx.x & 15, down = 16 >> p.across;
    const int64_t b = ((int64_t)blockIdx.y << p.across) + (group & ((1 << p.across) - 1)), e = b * BLOCK + lane * 8;
    const int64_t first = (int64_t)blockIdx.x * (down * QUANT_ROWS) + (group >> p.across);
    const int left = (int)min((int64_t)(QUANT_ROWS * 16), p.rows - first);       /* rows from `first` on */
    Pack<T, A> x[QUANT_ROWS][8 / A];
    const T *from = (const T *)p.x + first * p.x_stride + e;
#pragma unroll
    for (int i = 0; i < QUANT_ROWS; ++i, from += down * p.x_stride)
#pragma unroll
        for (int j = 0; j < 8 / A; ++j) {
#pragma unroll
            for (int k = 0; k < A; ++k) x[i][j].at[k] = from_f32<T>(0.0f);
            if (i * down < left && e + j * A < p.cols) x[i][j] = *(const Pack<T, A> *)(from + j * A);
        }
    float *scale = p.s + b * p.s_stride + first;
    uint8_t *to = p.q + first * p.q_stride + e;
    const bool stores = e < ((p.cols + 15) & ~15ll);    /* columns past the end, up to a multiple of 16, become zero */
#pragma unroll
    for (int i = 0; i < QUANT_ROWS; ++i, to += down * p.q_stride) {
        float v[8];
        uint32_t largest = 0;
        if (sizeof(T) == 2 && A > 1) {
            const uint32_t *two = (const uint32_t *)&x[i][0];
            largest = larger2(larger2(two[0] & 0x7fff7fff, two[1] & 0x7fff7fff), larger2(two[2] & 0x7fff7fff, two[3] & 0x7fff7fff));
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) largest = larger2(largest, __shfl_xor_sync(~0u, largest, d));
            largest = largest_of<T>(largest);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) largest = max(largest, magnitude(to_f32(x[i][j / A].at[j % A])));
#pragma unroll
            for (int d = 8; d > 0; d >>= 1) largest = max(largest, __shfl_xor_sync(~0u, largest, d));
        }
#pragma unroll
        for (int j = 0; j < 8; j += A) {
            float f[A];
            unpack(x[i][j / A], f);
#pragma unroll
            for (int k = 0; k < A; ++k) v[j + k] = f[k];
        }
        if (i * down >= left || b * BLOCK >= p.cols) continue;
        const float s = scale_of(largest);
        if (lane == 0) scale[i * down] = s;
        divide(v, s);
        const uint2 eight = make_uint2(e4m3x4(v[0], v[1], v[2], v[3]), e4m3x4(v[4], v[5], v[6], v[7]));
        if (BARE) {
            for (int j = 0; j < 8 && e + j < p.cols; ++j) to[j] = (uint8_t)((j < 4 ? eight.x : eight.y) >> 8 * (j & 3));
        } else if (stores) {
            *(uint2 *)to = eight;
        }
    }
}

struct QuantBlocksParams {
    const char *w;
    uint8_t *q;
    float *s;
    int64_t rows, cols, w_stride, q_stride, s_stride;
    int wide;
};

/* a block of threads for each 128 x 128 block: 16 threads a row, 16 rows at a time, values kept in registers */
template <typename T> __global__ void __launch_bounds__(256) quantize_blocks(QuantBlocksParams p) {
    __shared__ uint32_t warps[8];
    enter_grid();
    const int64_t row0 = (int64_t)blockIdx.y * BLOCK + threadIdx.x / 16, e = (int64_t)blockIdx.x * BLOCK + (threadIdx.x & 15) * 8;
    uint32_t largest = 0;
    float v[8][8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = row0 + 16 * i;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        if (row < p.rows) load8((const T *)p.w + row * p.w_stride, e, p.cols, p.wide, v[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) largest = max(largest, magnitude(v[i][j]));
    }
    largest = __reduce_max_sync(~0u, largest);
    if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = largest;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) largest = max(largest, warps[i]);
    const float s = scale_of(largest);
    if (threadIdx.x == 0) p.s[blockIdx.y * p.s_stride + blockIdx.x] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = row0 + 16 * i;
        if (row >= p.rows) continue;
        divide(v[i], s);
        const uint2 q = make_uint2(e4m3x4(v[i][0], v[i][1], v[i][2], v[i][3]), e4m3x4(v[i][4], v[i][5], v[i][6], v[i][7]));
        uint8_t *to = p.q + row * p.q_stride + e;
        if (e + 8 <= p.cols) {
            *(uint2 *)to = q;
        } else {
            for (int j = 0; j < 8 && e + j < p.cols; ++j) to[j] = (uint8_t)((j < 4 ? q.x : q.y) >> 8 * (j & 3));
        }
    }
}

/* ---- few rows of x -------------------------------------------------------------------- */

struct FewParams {
    const uint8_t *x, *w;
    const float *sx, *sw;
    char *y;
    int64_t x_stride, w_stride, sx_stride, sw_stride, y_stride;
    int m, n, k, stages;
    int64_t raw_stride;                 /* of x before quantisation, where the product quantises it itself */
    int raw_wide;
    uint8_t *xq;                        /* where the first block of threads leaves what it quantised */
    float *xs;
    int64_t xq_stride, xs_stride;
};

__device__ __forceinline__ void mma_e4m3(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

/* 16 rows of W a block of threads; its 8 or 16 warps take every 8th or 16th block of 128 columns and join at the end.  W and x come
 * through a ring of asynchronous copies in shared memory, FEW_STAGES blocks of a warp ahead: what is under way decides the rate
 * at so little work a byte, and registers for it would halve what runs at once.  A thread takes 16 consecutive bytes of a row;
 * the order of the columns inside a product is the same for x and W, and free.  1 x 16384 x 8192 reads W at 50 % of what DRAM gives
 * and issues in 45 % of its slots: a warp waits for its own copies and for its chain of products, whose e4m3 is converted
 * in the general pipes. */
template <int NT> struct alignas(16) FewStage {
    unsigned char w[16][BLOCK], x[8 * NT][BLOCK];
    float sx[8 * NT], sw, unused[3];
};
/* two or three blocks of threads an SM: 1 x 4096 x 14336 took 16.0 us, 22.1 with two stages, 16.4 with four; 1 x 4096 x 4096 takes
 * 6.5 us, 6.8 with four */
constexpr int FEW_STAGES = 3;

__device__ __forceinline__ void copy_async16(const void *shared, const void *from, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
                 ::"r"((uint32_t)__cvta_generic_to_shared(shared)), "l"(from), "r"(bytes) : "memory");
}

/* X: the type of an x that is not quantised yet, of up to 2 rows: a warp quantises what it takes, 4 elements a lane, which
 * saves the launch of the quantiser (1 x 4321 x 648: 4.4 -> 3.0 us); the first block of threads leaves it in p.xq and p.xs.  Quantised:
 * p.x and p.sx have it. */
struct Quantised {};
constexpr int FUSED_ROWS = 2;

template <typename T, int NT, typename X, int FEW_WARPS> __global__ void __launch_bounds__(32 * FEW_WARPS) few_rows(FewParams p) {
    constexpr int STAGES = FEW_STAGES;
    constexpr bool FUSED = !__is_same(X, Quantised);
    extern __shared__ __align__(128) unsigned char raw[];           /* [warps][stages] */
    __shared__ float parts[FEW_WARPS][16][8 * NT + 1];
    enter_grid();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    const int n0 = blockIdx.x * 16, blocks = (p.k + BLOCK - 1) / BLOCK, steps = (blocks - warp + FEW_WARPS - 1) / FEW_WARPS;
    FewStage<NT> *const ring = (FewStage<NT> *)raw + warp * p.stages;
    /* A copy of the warp has four rows' 128 bytes; the 16 bytes `piece` of a row lie at a place that depends on the row's
     * parity, as the reads below take two rows' halves at a time. */
    const int down = lane >> 3, piece = lane & 7, place = (piece ^ ((down & 1) * 4)) * 16;
    const uint8_t *w_row[4], *x_row[2 * NT];
#pragma unroll
    for (int i = 0; i < 4; ++i) w_row[i] = p.w + (int64_t)min(n0 + down + 4 * i, p.n - 1) * p.w_stride;
#pragma unroll
    for (int i = 0; i < 2 * NT; ++i) x_row[i] = p.x + (int64_t)min(down + 4 * i, p.m - 1) * p.x_stride;
    const float *sw = p.sw + (n0 / BLOCK) * p.sw_stride;
    auto issue = [&](int step, int stage) {
        if (step < steps) {
            FewStage<NT> &s = ring[stage];
            const int b = warp + FEW_WARPS * step, k = b * BLOCK + piece * 16, bytes = max(0, min(16, p.k - k)), at = bytes ? k : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) copy_async16(&s.w[down + 4 * i][place], w_row[i] + at, bytes);
            if (!FUSED)
#pragma unroll
                for (int i = 0; i < 2 * NT; ++i) copy_async16(&s.x[down + 4 * i][place], x_row[i] + at, down + 4 * i < p.m ? bytes : 0);
            if (!FUSED && lane < 2 * NT) {
                const int rest = max(0, min(4, p.m - 4 * lane));
                copy_async16(&s.sx[4 * lane], p.sx + b * p.sx_stride + (rest ? 4 * lane : 0), 4 * rest);
            } else if (lane == 31) {
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;"
                             ::"r"((uint32_t)__cvta_generic_to_shared(&s.sw)), "l"(sw + b) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 0; i < p.stages; ++i) issue(i, i);
    /* FUSED: four elements of each row of x, a block ahead; rows that are not there stay zero */
    float ahead[FUSED ? FUSED_ROWS : 1][4];
    auto fetch = [&](int step) {
        if constexpr (FUSED) {
            const int e = (warp + FEW_WARPS * step) * BLOCK + 4 * lane;
#pragma unroll
            for (int m = 0; m < FUSED_ROWS; ++m) {
                ahead[m][0] = ahead[m][1] = ahead[m][2] = ahead[m][3] = 0.0f;
                if (m >= p.m || step >= steps) continue;
                const X *x = (const X *)p.x + m * p.raw_stride + e;
                if (p.raw_wide && e + 4 <= p.k) {
                    const Pack<X, 4> q = *(const Pack<X, 4> *)x;
                    unpack(q, ahead[m]);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (e + i < p.k) ahead[m][i] = to_f32(x[i]);
                }
            }
        }
    };
    auto quantise = [&](FewStage<NT> &s, int step) {
        if constexpr (FUSED) {
            const int b = warp + FEW_WARPS * step, e = b * BLOCK + 4 * lane;
#pragma unroll
            for (int m = 0; m < FUSED_ROWS; ++m) {
                if (m >= p.m) break;
                uint32_t largest = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) largest = max(largest, magnitude(ahead[m][i]));
                const float scale = scale_of(__reduce_max_sync(~0u, largest));
                float (&v)[4] = ahead[m];
                divide(v, scale);
                const uint32_t four = e4m3x4(v[0], v[1], v[2], v[3]);
                *(uint32_t *)&s.x[m][((lane >> 2) ^ ((m & 1) * 4)) * 16 + (lane & 3) * 4] = four;
                if (lane == 0) s.sx[m] = scale;
                if (blockIdx.x == 0) {
                    if (e < ((p.k + 15) & ~15)) *(uint32_t *)(p.xq + m * p.xq_stride + e) = four;   /* zeros up to a multiple of 16 */
                    if (lane == 0) p.xs[b * p.xs_stride + m] = scale;
                }
            }
        }
    };
    if (FUSED) {
        for (int i = 0; i < p.stages; ++i) {
            const uint4 zero = make_uint4(0, 0, 0, 0);
            *(uint4 *)&ring[i].x[lane >> 3][(lane & 7) * 16] = zero, *(uint4 *)&ring[i].x[4 + (lane >> 3)][(lane & 7) * 16] = zero;
            if (lane < 8) ring[i].sx[lane] = 0.0f;
        }
        __syncwarp();
        fetch(0);
    }
    float acc[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[t][i] = 0.0f;
    const int low = (c ^ ((r & 1) * 4)) * 16, high = ((c + 4) ^ ((r & 1) * 4)) * 16;
    for (int step = 0, stage = 0; step < steps; ++step) {
        if (FUSED) {
            quantise(ring[stage], step);
            fetch(step + 1);
        }
        if (p.stages == STAGES)
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        else
            asm volatile("cp.async.wait_all;" ::: "memory");
        __syncwarp();
        const FewStage<NT> &s = ring[stage];
        const uint4 a0 = *(const uint4 *)&s.w[r][low], a1 = *(const uint4 *)&s.w[r + 8][low];
        const uint4 a2 = *(const uint4 *)&s.w[r][high], a3 = *(const uint4 *)&s.w[r + 8][high];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const uint4 x0 = *(const uint4 *)&s.x[8 * t + r][low], x1 = *(const uint4 *)&s.x[8 * t + r][high];
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma_e4m3(d, a0.x, a1.x, a0.y, a1.y, x0.x, x0.y);
            mma_e4m3(d, a0.z, a1.z, a0.w, a1.w, x0.z, x0.w);
            mma_e4m3(d, a2.x, a3.x, a2.y, a3.y, x1.x, x1.y);
            mma_e4m3(d, a2.z, a3.z, a2.w, a3.w, x1.z, x1.w);
            const float2 sx = *(const float2 *)&s.sx[8 * t + 2 * c];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = fmaf(s.sw * (i & 1 ? sx.y : sx.x), d[i], acc[t][i]);
        }
        __syncwarp();
        issue(step + p.stages, stage);
        stage = stage + 1 == p.stages ? 0 : stage + 1;
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) parts[warp][r + 8 * (i >> 1)][8 * t + 2 * c + (i & 1)] = acc[t][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * 8 * NT; i += 32 * FEW_WARPS) {
        const int n = i & 15, m = i >> 4;
        if (m >= p.m || n0 + n >= p.n) continue;
        float s = 0.0f;
#pragma unroll
        for (int v = 0; v < FEW_WARPS; ++v) s += parts[v][n][m];
        ((T *)p.y)[m * p.y_stride + n0 + n] = from_f32<T>(s);
    }
}

template <typename T, int NT, typename X, int WARPS> cudaError_t go_warps(FewParams p, int device, uint64_t stream) {
    static uint64_t allowed;
    constexpr size_t STAGE = WARPS * sizeof(FewStage<NT>);
    if (!(__atomic_load_n(&allowed, __ATOMIC_ACQUIRE) >> device & 1)) {
        cudaError_t e = cudaFuncSetAttribute(few_rows<T, NT, X, WARPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_STAGES * STAGE);
        if (e != cudaSuccess) return e;
        __atomic_fetch_or(&allowed, 1ull << device, __ATOMIC_RELEASE);
    }
    /* as many stages as a warp has blocks, up to all: short rows leave the room to more blocks of threads */
    const int steps = ((p.k + BLOCK - 1) / BLOCK + WARPS - 1) / WARPS;
    p.stages = steps < FEW_STAGES ? steps : FEW_STAGES;
    return launch(few_rows<T, NT, X, WARPS>, dim3((unsigned)((p.n + 15) / 16)), dim3(32 * WARPS), p.stages * STAGE, stream, p);
}
/* 16 warps a block of threads where there is a block for each SM at most, and rows have more than 8 blocks of 128 to share: 1 x 1024 x
 * 8192 takes 6.7 us, with 8 warps 9.8; 8 x 1321 x 6450 7.3 and 9.9; where SMs hold several blocks 8 warps are as fast. */
template <typename T, int NT, typename X = Quantised> cudaError_t go_few(const FewParams &p, int device, uint64_t stream) {
    int sms;
    if (ops_sm_count(device, &sms)) return cudaErrorInvalidDevice;
    return p.n <= 16 * sms && p.k > 8 * BLOCK ? go_warps<T, NT, X, 16>(p, device, stream) : go_warps<T, NT, X, 8>(p, device, stream);
}

/* ---- many rows of x: tcgen05 ------------------------------------------------------------ */

/* A tile of 128 rows of x (256 on a pair of SMs) by BN columns of y.  Warp 0 copies, warp 1 multiplies, warps 4 and on scale:
 * the tensor core sums a block of 128 columns into tensor memory, and the scaling warps add scale times that to the
 * tile's sums in registers while the next block's product runs (tensor memory holds 512 / BN blocks).  Operands
 * arrive by TMA in 128-byte rows with the 128-byte swizzle; every wait gives up after 2 s.
 * 8192 x 8192 x 8192 takes 483 to 512 us from box to box (2.15 to 2.28 PFLOP/s), and took 418 where it took 483 with the scaled sums
 * left out: what is left of the distance to the e4m3 rate is the sums' issue slots and the power limit. */
struct ManyParams {
    const float *sw;
    char *y;
    unsigned *status;
    int64_t sw_stride, y_stride, split_stride;
    int m, n, k_blocks, m_tiles, n_tiles, wide, even, splits, per_split;
};

struct TensorMap {
    alignas(64) unsigned char bytes[128];
};

template <bool PAIR>
__device__ __forceinline__ void tma_load(uint32_t to, const TensorMap *map, int x, int y, uint32_t barrier) {
    if (PAIR)
        asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(barrier) : "memory");
    else
        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                     ::"r"(to), "l"(map), "r"(x), "r"(y), "r"(barrier) : "memory");
}
/* A block's product: four steps of 32 bytes along the rows.  Operands are K-major rows of 128 bytes with the 128-byte
 * swizzle, eight rows 1024 bytes apart: the descriptors differ in the low words (address / 16) alone. */
template <bool PAIR> __device__ __forceinline__ void multiply_block(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
    constexpr uint32_t HIGH = (1024u >> 4) | (1u << 14) | (2u << 29);
#define EMMY_STEPS(CG)                                                                                                  \
    asm volatile("{\n.reg .pred first, later;\n.reg .b32 x, y;\n.reg .b64 u, v;\n"                                        \
                 "setp.ne.u32 first, %3, %3;\nsetp.eq.u32 later, %3, %3;\n"                                              \
                 "mov.b64 u, {%1, %4};\nmov.b64 v, {%2, %4};\n"                                                           \
                 "tcgen05.mma.cta_group::" CG ".kind::f8f6f4 [%0], u, v, %3, first;\n"                                    \
                 "add.u32 x, %1, 2;\nadd.u32 y, %2, 2;\nmov.b64 u, {x, %4};\nmov.b64 v, {y, %4};\n"                       \
                 "tcgen05.mma.cta_group::" CG ".kind::f8f6f4 [%0], u, v, %3, later;\n"                                    \
                 "add.u32 x, %1, 4;\nadd.u32 y, %2, 4;\nmov.b64 u, {x, %4};\nmov.b64 v, {y, %4};\n"                       \
                 "tcgen05.mma.cta_group::" CG ".kind::f8f6f4 [%0], u, v, %3, later;\n"                                    \
                 "add.u32 x, %1, 6;\nadd.u32 y, %2, 6;\nmov.b64 u, {x, %4};\nmov.b64 v, {y, %4};\n"                       \
                 "tcgen05.mma.cta_group::" CG ".kind::f8f6f4 [%0], u, v, %3, later;\n}"                                   \
                 ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(HIGH) : "memory")
    if (PAIR)
        EMMY_STEPS("2");
    else
        EMMY_STEPS("1");
#undef EMMY_STEPS
}
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t barrier) {
    if (PAIR)
        asm volatile("{\n.reg .b16 m;\nmov.b16 m, 3;\n"
                     "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n}"
                     ::"r"(barrier) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
}
/* to this block's barrier alone */
template <bool PAIR> __device__ __forceinline__ void commit_here(uint32_t barrier) {
    if (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(barrier) : "memory");
    else
        commit<false>(barrier);
}
__device__ __forceinline__ void tensor_load(uint32_t address, uint32_t (&u)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
                   "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
                   "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
                   "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
                 : "r"(address));
}
/* the loads before it are done; `u` passes through, so that no use of it moves ahead of the wait */
__device__ __forceinline__ void tensor_wait(uint32_t (&u)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]),
                   "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15]), "+r"(u[16]),
                   "+r"(u[17]), "+r"(u[18]), "+r"(u[19]), "+r"(u[20]), "+r"(u[21]), "+r"(u[22]), "+r"(u[23]), "+r"(u[24]),
                   "+r"(u[25]), "+r"(u[26]), "+r"(u[27]), "+r"(u[28]), "+r"(u[29]), "+r"(u[30]), "+r"(u[31])::"memory");
}
__device__ __forceinline__ void tensor_load(uint32_t address, uint32_t (&u)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
                   "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
                 : "r"(address));
}
/* the loads before it are done; `u` passes through, so that no use of it moves ahead of the wait */
__device__ __forceinline__ void tensor_wait(uint32_t (&u)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(u[0]), "+r"(u[1]), "+r"(u[2]), "+r"(u[3]), "+r"(u[4]), "+r"(u[5]), "+r"(u[6]), "+r"(u[7]), "+r"(u[8]),
                   "+r"(u[9]), "+r"(u[10]), "+r"(u[11]), "+r"(u[12]), "+r"(u[13]), "+r"(u[14]), "+r"(u[15])::"memory");
}
/* a pair of f32 sums: sum += s v */
__device__ __forceinline__ void add_scaled(uint64_t &sum, uint64_t s, uint32_t v0, uint32_t v1) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "r"(v0), "r"(v1));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(sum) : "l"(s), "l"(v));
}

__device__ __forceinline__ float half_of(uint64_t v, int high) {
    float a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
    return high ? b : a;
}

template <int BN, bool PAIR> struct ManyShape {
    static constexpr int ROWS = PAIR ? 256 : 128;                     /* of a tile */
    static constexpr int B_ROWS = PAIR ? BN / 2 : BN;                 /* rows of W that one SM copies */
    static constexpr int A_BYTES = 128 * BLOCK, B_BYTES = B_ROWS * BLOCK, STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = STAGE > 40960 ? 4 : STAGE >= 32768 ? 6 : 8;
    static constexpr int BUFFERS = 512 / BN > 4 ? 4 : 512 / BN;
    /* x's scales have a ring of their own, in runs of SCALE_RUN places that the scaling warps hand back by a barrier each (runs of
     * 2 take 1 % longer at 8192^3, of 4 0.3 %).  The copies are at most STAGES blocks ahead of the products, and these BUFFERS
     * ahead of the scaling, so they find the next run free: nothing waits there. */
    static constexpr int SCALES = 24, SCALE_RUN = 8;
    static_assert(STAGES + BUFFERS <= SCALES - SCALE_RUN, "the scales' ring");
    static constexpr int COLUMNS = BN * BUFFERS < 32 ? 32 : BN * BUFFERS;
    static constexpr int SCALE_WARPS = BN >= 128 ? 8 : 4;
    static constexpr int PER = BN / (SCALE_WARPS / 4);                /* columns a scaling thread */
    static constexpr int CHUNK = PER >= 64 ? 32 : 16, CHUNKS = PER / CHUNK;   /* columns a load of tensor memory */
    static constexpr int THREADS = 128 + 32 * SCALE_WARPS;
    static constexpr bool SPLIT = PER == 128;     /* the scaling warps need more registers than an even share */
    static constexpr int STORE_ROW = 80;           /* 64 bytes of a row of y, and 16 that keep its neighbours in other banks */
    static constexpr int SMEM = STAGES * STAGE + 1024 + SCALE_WARPS * 32 * STORE_ROW;
};

template <typename T, int BN, bool PAIR>
__global__ void __launch_bounds__(ManyShape<BN, PAIR>::THREADS, 1)
    many_rows(const __grid_constant__ TensorMap x_map, const __grid_constant__ TensorMap w_map,
              const __grid_constant__ TensorMap s_map, ManyParams p) {
    using S = ManyShape<BN, PAIR>;
    extern __shared__ unsigned char raw[];
    __shared__ uint64_t full[S::STAGES], empty[S::STAGES], summed[S::BUFFERS], read[S::BUFFERS], scaled[S::SCALES / S::SCALE_RUN], ended[2];
    __shared__ alignas(128) float scales[S::SCALES][128];      /* of x: a block's 128 rows, copied with its operands */
    __shared__ uint32_t tensor_base;
    __shared__ volatile unsigned abort;
    __shared__ uint32_t next_stage, next_phase;         /* of the copies, when they ended */
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t ring = (shared_address(raw) + 1023) & ~1023u;
    uint32_t rank = 0;
    if (PAIR) asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&full[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&empty[i])));
        }
        for (int i = 0; i < S::BUFFERS; ++i) {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&summed[i])));
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(&read[i])), "r"(S::SCALE_WARPS * (PAIR ? 2 : 1)));
        }
        for (int i = 0; i < S::SCALES / S::SCALE_RUN; ++i)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(&scaled[i])), "r"(S::SCALE_WARPS));
        for (int i = 0; i < 2; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&ended[i])));
        abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\nfence.proxy.async.shared::cta;" ::: "memory");
    }
    if (PAIR) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    if (warp == 1) {
        const uint32_t to = shared_address(&tensor_base);
        if (PAIR)
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n"
                         "tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::"r"(to), "n"(S::COLUMNS) : "memory");
        else
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n"
                         "tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::"r"(to), "n"(S::COLUMNS) : "memory");
    }
    enter_grid();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t base = tensor_base;
    const int worker = PAIR ? blockIdx.x / 2 : blockIdx.x, workers = PAIR ? gridDim.x / 2 : gridDim.x;
    const int tiles = p.m_tiles * p.n_tiles * p.splits;

    /* tiles that run together share rows and columns: groups of 16 row tiles, column by column */
    struct Unit { int m0, n0, from, to, split; };
    auto place = [&](int t) {
        Unit u;
        u.split = t % p.splits, t /= p.splits;
        u.from = u.split * p.per_split, u.to = min(u.from + p.per_split, p.k_blocks);
        const int group = t / (16 * p.n_tiles), first = group * 16, rows = min(16, p.m_tiles - first);
        const int r = t - first * p.n_tiles;
        u.n0 = r / rows * BN;
        u.m0 = (first + r % rows) * S::ROWS;
        return u;
    };

    if (warp < 4 && S::SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 0) {
        if (lane == 0) {
            uint32_t leader = shared_address(&full[0]);
            if (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %0, 0;" : "+r"(leader));
            int stage = 0, slot = 0;
            uint32_t phase = 0, slot_phase = 0;
            bool ok = true;
            for (int t = worker; t < tiles && ok; t += workers) {
                const Unit u = place(t);
                const int m0 = u.m0 + (PAIR ? 128 * rank : 0), n0 = u.n0 + (PAIR ? S::B_ROWS * rank : 0);
                for (int b = u.from; b < u.to; ++b) {
                    if (!(ok = wait_for(shared_address(&empty[stage]), phase ^ 1, &abort, p.status, 1))) break;
                    if (slot % S::SCALE_RUN == 0 &&
                        !(ok = wait_for(shared_address(&scaled[slot / S::SCALE_RUN]), slot_phase ^ 1, &abort, p.status, 1))) break;
                    if (rank == 0)      /* both copies of a pair complete on the leader's barrier */
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                                     ::"r"(shared_address(&full[stage])), "r"((S::STAGE + 512) * (PAIR ? 2 : 1)) : "memory");
                    const uint32_t to = ring + stage * S::STAGE, barrier = leader + 8 * stage;
                    tma_load<PAIR>(to, &x_map, b * BLOCK, m0, barrier);
                    tma_load<PAIR>(to + S::A_BYTES, &w_map, b * BLOCK, n0, barrier);
                    tma_load<PAIR>(shared_address(scales[slot]), &s_map, m0, b, barrier);
                    if (++slot == S::SCALES) slot = 0, slot_phase ^= 1;
                    if (++stage == S::STAGES) stage = 0, phase ^= 1;
                }
            }
            next_stage = stage, next_phase = phase;
        }
    } else if (warp == 1 || warp == 3) {
        /* Two threads issue the products, every other block each: issuing one takes a thread longer than the tensor core
         * takes to run it. */
        if (lane == 0 && rank == 0) {
            constexpr uint32_t idesc = 1u << 4 | (uint32_t)(BN >> 3) << 17 | (uint32_t)(S::ROWS >> 4) << 24;
            const uint32_t full0 = shared_address(&full[0]), empty0 = shared_address(&empty[0]);
            const uint32_t summed0 = shared_address(&summed[0]), read0 = shared_address(&read[0]);
            const uint32_t a0 = (1u << 16) | ring >> 4, b0 = a0 + (S::A_BYTES >> 4);
            int stage = warp >> 1, buffer = warp >> 1, skip = warp >> 1;
            uint32_t phase = 0, buffer_phase = 0;
            bool ok = true;
            static_assert(S::STAGES % 2 == 0 && S::BUFFERS % 2 == 0, "every other stage and buffer");
            for (int t = worker; t < tiles && ok; t += workers) {
                const Unit u = place(t);
                /* blocks of later tiles, as far as they matter: a stage that is not filled again is not handed back either, so
                 * that no arrival is under way when the block of threads ends */
                int rest = 0;
                for (int later = t + workers; later < tiles && rest < S::STAGES; later += workers) {
                    const int from = later % p.splits * p.per_split;
                    rest += min(from + p.per_split, p.k_blocks) - from;
                }
                const int hand_back = u.to + rest - S::STAGES;
                int b = u.from + skip;
                for (; b < u.to; b += 2) {
                    if (!(ok = wait_for_both(read0 + 8 * buffer, buffer_phase ^ 1, full0 + 8 * stage, phase, &abort, p.status, 2))) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    multiply_block<PAIR>(base + buffer * BN, a0 + stage * (S::STAGE >> 4), b0 + stage * (S::STAGE >> 4), idesc);
                    commit<PAIR>(summed0 + 8 * buffer);
                    if (b < hand_back) commit<PAIR>(empty0 + 8 * stage);
                    if ((stage += 2) >= S::STAGES) stage -= S::STAGES, phase ^= 1;
                    if ((buffer += 2) >= S::BUFFERS) buffer -= S::BUFFERS, buffer_phase ^= 1;
                }
                skip = b - u.to;        /* the next tile's first block is the other thread's, or this one's */
            }
        }
    } else if (warp >= 4) {
        if (S::SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");      /* 256 of them, and 128 with 40: 384 of 168 */
        const int quarter = warp & 3, half = (warp - 4) >> 2;
        const uint32_t mine = base + (uint32_t)(quarter * 32) * 65536 + half * S::PER;
        uint32_t leader = shared_address(&read[0]);
        if (PAIR) asm volatile("mapa.shared::cluster.u32 %0, %0, 0;" : "+r"(leader));
        int buffer = 0, slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = worker; t < tiles && ok; t += workers) {
            const Unit u = place(t);
            const int row = u.m0 + 128 * rank + 32 * quarter + lane, col = u.n0 + half * S::PER;
            const float *sw = p.sw + (int64_t)(min(col, p.n - 1) / BLOCK) * p.sw_stride;
            uint64_t sum[S::PER / 2];
#pragma unroll
            for (int i = 0; i < S::PER / 2; ++i) sum[i] = 0;
            float next_w = sw[u.from];
            /* a load of tensor memory is under way while the one before it is added, from block to block too */
            uint32_t v[2][S::CHUNK];
            auto begin = [&] {
                if (!wait_for(shared_address(&summed[buffer]), phase, &abort, p.status, 4)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                tensor_load(mine + buffer * BN, v[0]);
                return true;
            };
            if (!(ok = begin())) continue;
#pragma unroll 1
            for (int b = u.from; b < u.to; ++b) {
                const float one = next_w * scales[slot][32 * quarter + lane];
                if (slot % S::SCALE_RUN == S::SCALE_RUN - 1) {
                    /* the run has been read, by all lanes: copies may write it again */
                    __syncwarp();
                    if (lane == 0)
                        asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"(shared_address(&scaled[slot / S::SCALE_RUN])) : "memory");
                }
                if (b + 1 < u.to) next_w = sw[b + 1];
                slot = slot + 1 == S::SCALES ? 0 : slot + 1;
                uint64_t s;
                asm("mov.b64 %0, {%1, %1};" : "=l"(s) : "f"(one));
#pragma unroll
                for (int c = 0; c < S::CHUNKS; ++c) {
                    tensor_wait(v[c & 1]);
                    if (c + 1 < S::CHUNKS) {
                        tensor_load(mine + buffer * BN + (c + 1) * S::CHUNK, v[(c + 1) & 1]);
                    } else {
                        /* All of the block is in registers.  A relaxed arrive is enough: the fences of tcgen05 on both sides order the
                         * loads before the next product, and nothing else rests on it. */
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) {
                            if (PAIR)
                                asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader + 8 * buffer) : "memory");
                            else
                                asm volatile("mbarrier.arrive.relaxed.cta.shared::cta.b64 _, [%0];" ::"r"(leader + 8 * buffer) : "memory");
                        }
                        if (++buffer == S::BUFFERS) buffer = 0, phase ^= 1;
                        if (b + 1 < u.to) ok = begin();
                    }
#pragma unroll
                    for (int i = 0; i < S::CHUNK; i += 2)
                        add_scaled(sum[(c * S::CHUNK + i) / 2], s, v[c & 1][i], v[c & 1][i + 1]);
                }
                if (!ok) break;
            }
            if (!ok) continue;
            /* 64 bytes of 32 rows at a time through shared memory, so that a store has whole sectors of a row */
            constexpr int V = 16 / sizeof(T), WIDE = 64 / sizeof(T);
            unsigned char *const rows = raw + (ring - shared_address(raw)) + S::STAGES * S::STAGE + (warp - 4) * 32 * S::STORE_ROW;
            const int row0 = row - lane;
            T *const y = (T *)p.y + u.split * p.split_stride;
#pragma unroll
            for (int c = 0; c < S::PER; c += WIDE) {
#pragma unroll
                for (int i = 0; i < WIDE; i += V) {
                    Pack<T, V> q;
#pragma unroll
                    for (int j = 0; j < V; ++j) q.at[j] = from_f32<T>(half_of(sum[(c + i + j) / 2], j & 1));
                    *(Pack<T, V> *)(rows + lane * S::STORE_ROW + i * sizeof(T)) = q;
                }
                __syncwarp();
                if (p.wide && col + c + WIDE <= p.n) {
                    const int piece = lane & 3;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int at = 8 * i + (lane >> 2);
                        if (row0 + at < p.m)
                            *(Pack<T, V> *)(y + (row0 + at) * p.y_stride + col + c + piece * V) =
                                *(const Pack<T, V> *)(rows + at * S::STORE_ROW + piece * 16);
                    }
                } else if (sizeof(T) == 2 && p.even && col + c + WIDE <= p.n) {
                    /* rows that start on 4 bytes: pairs, two rows at a time */
                    const int e = 2 * (lane & 15);
#pragma unroll 4
                    for (int at = lane >> 4; at < 32; at += 2)
                        if (row0 + at < p.m)
                            *(uint32_t *)(y + (row0 + at) * p.y_stride + col + c + e) = *(const uint32_t *)(rows + at * S::STORE_ROW + 2 * e);
                } else {
                    constexpr int AT_ONCE = 32 / WIDE;
                    const int e = lane % WIDE;
                    if (col + c + e < p.n)
                        for (int at = lane / WIDE; at < 32 && row0 + at < p.m; at += AT_ONCE)
                            y[(row0 + at) * p.y_stride + col + c + e] = *(const T *)(rows + at * S::STORE_ROW + e * sizeof(T));
                }
                __syncwarp();
            }
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    /* Where a wait gave up, whoever's: copies under way must not arrive in shared memory that is no longer this block's, nor products
     * in tensor memory that has been freed, so both are waited for.  A pair's copies all complete on the leader's barriers, and
     * its products are the leader's; it gives up where the other block does, as each waits for the other.  What was never
     * copied ends by the limit, which is one for all stages. */
    if (abort) {
        if (rank == 0 && lane == 0 && warp == 0) {
            uint32_t stage = next_stage, phase = next_phase;
            const uint64_t start = now_ns();
            for (int i = 0; i < S::STAGES; ++i) {
                wait_for_end(shared_address(&full[stage]), phase ^ 1, start);
                if (++stage == S::STAGES) stage = 0, phase ^= 1;
            }
        } else if (rank == 0 && lane == 0 && (warp == 1 || warp == 3)) {
            const uint32_t end = shared_address(&ended[warp >> 1]);
            commit_here<PAIR>(end);
            wait_for_end(end, 0, now_ns());
        }
        __syncthreads();
    }
    if (PAIR) asm volatile("barrier.cluster.arrive.release;\nbarrier.cluster.wait.acquire;" ::: "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 1) {
        if (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(S::COLUMNS));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(S::COLUMNS));
    }
}

/* y = the sum of the parts of a product that was cut along its columns, in their order */
struct JoinParams {
    const float *parts;
    char *y;
    int64_t part_stride, split_stride, y_stride;
    int m, n, splits;
};
template <typename T> __global__ void __launch_bounds__(256) join_parts(JoinParams p) {
    enter_grid();
    const int col = (blockIdx.x * 256 + threadIdx.x) * 4, row = blockIdx.y;
    if (col >= p.n) return;
    const float *from = p.parts + row * p.part_stride + col;       /* rows of the parts are whole fours */
    float4 s = *(const float4 *)from;
    for (int i = 1; i < p.splits; ++i) {
        const float4 v = *(const float4 *)(from + i * p.split_stride);
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    T *y = (T *)p.y + row * p.y_stride + col;
    const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (col + j < p.n) y[j] = from_f32<T>(v[j]);
}

int encode(TensorMap *map, uint64_t at, int64_t cols, int64_t rows, int64_t stride, int box_rows, bool scales = false) {
    const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)stride};
    const unsigned box[2] = {BLOCK, (unsigned)box_rows}, steps[2] = {1, 1};
    /* bytes with the 128-byte swizzle, or f32 without one; no interleave, 256-byte L2 promotion, zeros outside */
    if (int e = emmy_rt_tensor_map_encode_tiled(map, scales ? 7 : 0, 2, at, dims, strides, box, steps, 0, scales ? 0 : 3, 3, 0))
        return ops_fail(e, "tensor map: %s", emmy_rt_last_error());
    return 0;
}

template <typename T, int BN, bool PAIR> int go_many(const emmy_ops_blockfp8_args *a, ManyParams p, int device, uint64_t stream) {
    using S = ManyShape<BN, PAIR>;
    static uint64_t allowed;
    if (!(__atomic_load_n(&allowed, __ATOMIC_ACQUIRE) >> device & 1)) {
        cudaError_t e = cudaFuncSetAttribute(many_rows<T, BN, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
        if (e != cudaSuccess) return ops_cuda(e, "shared memory of the FP8 product");
        __atomic_fetch_or(&allowed, 1ull << device, __ATOMIC_RELEASE);
    }
    TensorMap x, w, scales;
    if (int e = encode(&x, a->xq, a->k, a->m, a->xq_stride, 128)) return e;
    if (int e = encode(&w, a->wq, a->k, a->n, a->wq_stride, S::B_ROWS)) return e;
    if (int e = encode(&scales, a->xs, a->m, (a->k + BLOCK - 1) / BLOCK, a->xs_stride * 4, 1, true)) return e;
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    p.m_tiles = (int)((a->m + S::ROWS - 1) / S::ROWS);
    p.n_tiles = (int)((a->n + BN - 1) / BN);
    const int64_t tiles = (int64_t)p.m_tiles * p.n_tiles * p.splits;
    const int workers = PAIR ? sms / 2 : sms, blocks = (int)(tiles < workers ? tiles : workers) * (PAIR ? 2 : 1);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks), cfg.blockDim = dim3(S::THREADS), cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = (cudaStream_t)(uintptr_t)stream;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = PAIR ? 2 : 1, attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    cfg.attrs = attributes, cfg.numAttrs = 2;
    return ops_cuda(cudaLaunchKernelEx(&cfg, many_rows<T, BN, PAIR>, x, w, scales, p), "FP8 product");
}

template <typename T> int by_tile(int which, const emmy_ops_blockfp8_args *a, const ManyParams &p, int device, uint64_t stream) {
    switch (which) {
    case 0: return go_many<T, 32, false>(a, p, device, stream);
    case 1: return go_many<T, 64, false>(a, p, device, stream);
    case 2: return go_many<T, 128, false>(a, p, device, stream);
    default: return go_many<T, 256, true>(a, p, device, stream);
    }
}

template <typename T> int product(const emmy_ops_blockfp8_args *a, int device, uint64_t stream) {
    /* Up to 8 rows, and up to 16 where W is small: 16 x 4096 x 4096 takes 7.6 us here and 8.8 us in tiles cut in four,
     * 16 x 4096 x 14336 20.9 us here and 18.1 us there. */
    if (a->m <= 8 || (a->m <= 16 && a->n * a->k <= (1 << 25))) {
        FewParams p = {(const uint8_t *)(uintptr_t)a->xq, (const uint8_t *)(uintptr_t)a->wq, (const float *)(uintptr_t)a->xs,
                       (const float *)(uintptr_t)a->ws, (char *)(uintptr_t)a->y, a->xq_stride, a->wq_stride, a->xs_stride,
                       a->ws_stride, a->y_stride, (int)a->m, (int)a->n, (int)a->k};
        const cudaError_t e = a->m <= 8 ? go_few<T, 1>(p, device, stream) : go_few<T, 2>(p, device, stream);
        return ops_cuda(e, "FP8 product of few rows");
    }
    ManyParams p = {};
    p.sw = (const float *)(uintptr_t)a->ws, p.y = (char *)(uintptr_t)a->y;
    p.status = (unsigned *)(uintptr_t)a->status;
    p.sw_stride = a->ws_stride, p.y_stride = a->y_stride;
    p.m = (int)a->m, p.n = (int)a->n, p.k_blocks = (int)((a->k + BLOCK - 1) / BLOCK);
    p.wide = aligned(a->y, 16) && a->y_stride * sizeof(T) % 16 == 0;
    p.even = aligned(a->y, 4) && a->y_stride * sizeof(T) % 4 == 0;
    int sms;
    if (int e = ops_sm_count(device, &sms)) return e;
    /* The tiles and the cut along k that take least.  Measured at 782 choices for 90 products of 17 to 2000 rows, a round of
     * tiles takes 300 ns a block of 128 columns (tiles 32 and 64 wide) to 490 (256, on pairs of SMs) and 0.7 to 2.9 us
     * beside them: the wider the tile, the less a column of y costs, as long as there are tiles for all SMs.  Where there
     * are not, k is cut into parts that SMs take beside each other; joining them takes 1.2 us and 1.3 us for a million
     * elements.  The fit is off by 6 %; what it chooses is 1.1 % slower than the fastest on average (with powers of two
     * alone as cuts 3.8 %). */
    const int64_t rows = (a->m + 127) / 128, pairs = (a->m + 255) / 256, part_row = (a->n + 3) / 4 * 4;
    const struct { int64_t tiles, workers, block_ns, round_ns; } shapes[] = {{rows * ((a->n + 31) / 32), sms, 300, 700},
                                                                              {rows * ((a->n + 63) / 64), sms, 300, 1060},
                                                                              {rows * ((a->n + 127) / 128), sms, 417, 1570},
                                                                              {pairs * ((a->n + 255) / 256), sms / 2, 490, 2900}};
    int best = 0, splits = 1;
    int64_t least = INT64_MAX;
    for (int i = 0; i < (rows > 1 ? 4 : 3); ++i) {
        const auto &f = shapes[i];
        for (int cut = 1; cut <= 16 && (cut == 1 || cut * 4 <= p.k_blocks); ++cut) {
            if (cut > 1 && (f.tiles > f.workers || a->m > 65535 || cut * a->m * part_row * 4 > (a->parts ? (int64_t)a->parts_bytes : 0))) break;
            const int64_t per = (p.k_blocks + cut - 1) / cut, rounds = (f.tiles * cut + f.workers - 1) / f.workers;
            const int64_t cost = rounds * (per * f.block_ns + f.round_ns) + (cut > 1 ? 1200 + cut * a->m * part_row / 760 : 0);
            if (cost < least) least = cost, best = i, splits = cut;
        }
    }
    p.per_split = (p.k_blocks + splits - 1) / splits;
    p.splits = splits = (p.k_blocks + p.per_split - 1) / p.per_split;
    if (splits == 1) return by_tile<T>(best, a, p, device, stream);
    JoinParams j = {(const float *)(uintptr_t)a->parts, p.y, part_row, a->m * part_row, p.y_stride, p.m, p.n, splits};
    p.y = (char *)(uintptr_t)a->parts, p.y_stride = part_row, p.split_stride = j.split_stride, p.wide = 1;
    if (int e = by_tile<float>(best, a, p, device, stream)) return e;
    return ops_cuda(launch(join_parts<T>, dim3((unsigned)((a->n + 1023) / 1024), (unsigned)a->m), dim3(256), 0, stream, j),
                    "joining the FP8 product's parts");
}

/* shared: all rows may be one (stride 0) */
int check_matrix(const char *name, uint64_t at, int64_t rows, int64_t cols, int64_t stride, int size, int multiple, bool shared = false) {
    if (rows < 0 || cols < 1 || rows > 0x7fffff00LL || cols > 0x7fffff00LL)
        return ops_fail(EMMY_RT_EINVAL, "%s of %lld x %lld", name, (long long)rows, (long long)cols);
    if (rows > 1 && stride < cols && !(shared && stride == 0)) return ops_fail(EMMY_RT_EINVAL, "%s: rows overlap: stride %lld", name, (long long)stride);
    if (!at || !aligned(at, size * multiple)) return ops_fail(EMMY_RT_EINVAL, "%s is needed, on %d bytes", name, size * multiple);
    if (stride % multiple) return ops_fail(EMMY_RT_EINVAL, "%s: rows are not a multiple of %d elements apart", name, multiple);
    return 0;
}

template <typename T> cudaError_t go_fused(const FewParams &p, int dtype, int device, uint64_t stream) {
    return dtype == EMMY_OPS_F32   ? go_few<T, 1, float>(p, device, stream)
           : dtype == EMMY_OPS_F16 ? go_few<T, 1, __half>(p, device, stream)
                                   : go_few<T, 1, __nv_bfloat16>(p, device, stream);
}

int check_product(const emmy_ops_blockfp8_args *a) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (!known_dtype(a->dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", a->dtype);
    const int es = elem_size(a->dtype);
    const int64_t k_blocks = (a->k + BLOCK - 1) / BLOCK, n_blocks = (a->n + BLOCK - 1) / BLOCK;
    if (a->n < 1) return ops_fail(EMMY_RT_EINVAL, "n %lld", (long long)a->n);
    if (int e = check_matrix("xq", a->m ? a->xq : 16, a->m, a->k, a->xq_stride, 1, 16)) return e;
    if (int e = check_matrix("wq", a->wq, a->n, a->k, a->wq_stride, 1, 16)) return e;
    if (a->xq_stride < (a->k + 15) / 16 * 16 || a->wq_stride < (a->k + 15) / 16 * 16)
        return ops_fail(EMMY_RT_EINVAL, "rows of xq and wq are not padded to 16 bytes");
    if (int e = check_matrix("xs", a->m ? a->xs : 16, k_blocks, a->m > 0 ? a->m : 1, a->xs_stride, 4, 4)) return e;
    if (a->xs_stride < 4) return ops_fail(EMMY_RT_EINVAL, "rows of xs are %lld apart", (long long)a->xs_stride);
    if (int e = check_matrix("ws", a->ws, n_blocks, k_blocks, a->ws_stride, 4, 1)) return e;
    if (int e = check_matrix("y", a->m ? a->y : 16, a->m, a->n, a->y_stride, es, 1)) return e;
    if (a->parts && !aligned(a->parts, 16)) return ops_fail(EMMY_RT_EINVAL, "parts start on 16 bytes");
    if (!a->status || !aligned(a->status, 4)) return ops_fail(EMMY_RT_EINVAL, "a status word is needed");
    if (((a->m + 127) / 128) * ((a->n + 31) / 32) > 0x7fffffffLL)
        return ops_fail(EMMY_RT_EINVAL, "y of %lld x %lld", (long long)a->m, (long long)a->n);
    return 0;
}

}  // namespace

EMMY_EXPORT int emmy_ops_blockfp8_quantize(const emmy_ops_blockfp8_quantize_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    if (!known_dtype(a->dtype)) return ops_fail(EMMY_RT_EINVAL, "element type %d", a->dtype);
    const int es = elem_size(a->dtype);
    const int64_t row_blocks = a->square ? (a->rows + BLOCK - 1) / BLOCK : a->rows, col_blocks = (a->cols + BLOCK - 1) / BLOCK;
    if (int e = check_matrix("x", a->rows ? a->x : 16, a->rows, a->cols, a->x_stride, es, 1, true)) return e;
    /* a single row that is not in padded rows: no column past its last one is written */
    const int64_t padded = (a->cols + 15) / 16 * 16;
    const bool bare = a->rows == 1 && a->q_stride < padded;
    const int64_t q_stride = bare ? padded : a->q_stride;
    if (int e = check_matrix("q", a->rows ? a->q : 16, a->rows, a->cols, q_stride, 1, 16)) return e;
    if (q_stride < padded) return ops_fail(EMMY_RT_EINVAL, "rows of q are not padded to 16 bytes");
    if (int e = check_matrix("s", a->rows ? a->s : 16, a->square ? row_blocks : col_blocks, a->square ? col_blocks : a->rows > 0 ? a->rows : 1,
                             a->s_stride, 4, 1))
        return e;
    if (a->rows == 0) return 0;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    const int wide = aligned(a->x, 16) && a->x_stride * es % 16 == 0;
    cudaError_t e;
    if (a->square) {
        if (row_blocks > 65535) return ops_fail(EMMY_RT_EINVAL, "%lld rows of a weight", (long long)a->rows);
        QuantBlocksParams p = {(const char *)(uintptr_t)a->x, (uint8_t *)(uintptr_t)a->q, (float *)(uintptr_t)a->s, a->rows, a->cols,
                               a->x_stride, q_stride, a->s_stride, wide};
        const dim3 grid((unsigned)col_blocks, (unsigned)row_blocks);
        e = a->dtype == EMMY_OPS_F32   ? launch(quantize_blocks<float>, grid, dim3(256), 0, stream, p)
            : a->dtype == EMMY_OPS_F16 ? launch(quantize_blocks<__half>, grid, dim3(256), 0, stream, p)
                                       : launch(quantize_blocks<__nv_bfloat16>, grid, dim3(256), 0, stream, p);
    } else {
        int across = 0;
        while (across < 4 && (1 << across) < col_blocks) ++across;
        const int64_t down = (16 >> across) * QUANT_ROWS, tall = (col_blocks + (1 << across) - 1) >> across;
        if (tall > 65535) return ops_fail(EMMY_RT_EINVAL, "%lld columns", (long long)a->cols);
        QuantRowsParams p = {(const char *)(uintptr_t)a->x, (uint8_t *)(uintptr_t)a->q, (float *)(uintptr_t)a->s, a->rows, a->cols,
                             a->x_stride, q_stride, a->s_stride, across};
        const dim3 grid((unsigned)((a->rows + down - 1) / down), (unsigned)tall);
        auto fits = [&](int bytes) { return aligned(a->x, bytes) && a->x_stride * es % bytes == 0 && a->cols * es % bytes == 0; };
        const int access = fits(16) ? 16 : fits(4) ? 4 : es;
        auto go = [&](auto kernel) { return launch(kernel, grid, dim3(256), 0, stream, p); };
        if (bare)
            e = a->dtype == EMMY_OPS_F32   ? go(quantize_rows<float, 1, true>)
                : a->dtype == EMMY_OPS_F16 ? go(quantize_rows<__half, 1, true>)
                                           : go(quantize_rows<__nv_bfloat16, 1, true>);
        else if (a->dtype == EMMY_OPS_F32)
            e = access == 16 ? go(quantize_rows<float, 4>) : go(quantize_rows<float, 1>);
        else if (a->dtype == EMMY_OPS_F16)
            e = access == 16 ? go(quantize_rows<__half, 8>) : access == 4 ? go(quantize_rows<__half, 2>) : go(quantize_rows<__half, 1>);
        else
            e = access == 16  ? go(quantize_rows<__nv_bfloat16, 8>)
                : access == 4 ? go(quantize_rows<__nv_bfloat16, 2>)
                              : go(quantize_rows<__nv_bfloat16, 1>);
    }
    return ops_cuda(e, "FP8 quantisation");
}

EMMY_EXPORT int emmy_ops_blockfp8_product(const emmy_ops_blockfp8_args *a, int device, uint64_t stream) {
    if (int e = check_product(a)) return e;
    if (a->m == 0) return 0;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    return a->dtype == EMMY_OPS_F32   ? product<float>(a, device, stream)
           : a->dtype == EMMY_OPS_F16 ? product<__half>(a, device, stream)
                                      : product<__nv_bfloat16>(a, device, stream);
}

EMMY_EXPORT int emmy_ops_blockfp8_linear(const emmy_ops_blockfp8_linear_args *a, int device, uint64_t stream) {
    if (!a) return ops_fail(EMMY_RT_EINVAL, "no arguments");
    const emmy_ops_blockfp8_args &q = a->product;
    if (int e = check_product(&q)) return e;
    const emmy_ops_blockfp8_quantize_args x = {a->x, q.xq, q.xs, a->x_stride, q.xq_stride, q.xs_stride, q.m, q.k, a->x_dtype, 0};
    /* One launch or two: in one, every 16 rows of W quantise x again, which shows where there are many or rows are long.  Device
     * times in one launch and in two: 2 x 1000 x 1000 3.1 and 3.7 us, 1 x 6144 x 2048 6.0 and 6.7, 1 x 4096 x 4096 6.5 and 6.2 (and
     * 2.5 us less of the host's time), 2 x 4096 x 4096 7.8 and 6.9, 2 x 14336 x 4096 27 and 19. */
    if (q.m > FUSED_ROWS || q.m * q.n * q.k > (1 << 24) || !known_dtype(a->x_dtype)) {
        if (int e = emmy_ops_blockfp8_quantize(&x, device, stream)) return e;
        return emmy_ops_blockfp8_product(&q, device, stream);
    }
    const int es = elem_size(a->x_dtype);
    if (int e = check_matrix("x", q.m ? a->x : 16, q.m, q.k, a->x_stride, es, 1, true)) return e;
    if (q.m == 0) return 0;
    DeviceScope scope(device);
    if (scope.status != cudaSuccess) return ops_cuda(scope.status, "device");
    FewParams p = {(const uint8_t *)(uintptr_t)a->x, (const uint8_t *)(uintptr_t)q.wq, nullptr, (const float *)(uintptr_t)q.ws,
                   (char *)(uintptr_t)q.y, 0, q.wq_stride, 0, q.ws_stride, q.y_stride, (int)q.m, (int)q.n, (int)q.k, 0, a->x_stride,
                   aligned(a->x, 4 * es) && a->x_stride % 4 == 0, (uint8_t *)(uintptr_t)q.xq, (float *)(uintptr_t)q.xs, q.xq_stride,
                   q.xs_stride};
    const cudaError_t e = q.dtype == EMMY_OPS_F32   ? go_fused<float>(p, a->x_dtype, device, stream)
                          : q.dtype == EMMY_OPS_F16 ? go_fused<__half>(p, a->x_dtype, device, stream)
                                                    : go_fused<__nv_bfloat16>(p, a->x_dtype, device, stream);
    return ops_cuda(e, "FP8 product of few rows");
}
