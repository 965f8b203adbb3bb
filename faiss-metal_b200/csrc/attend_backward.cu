// Gradient of attention.  With s = scale q k^T, p = exp(s - lse), dp = do v^T, ds = p (dp - delta), delta = rowsum(do o):
//   dv = p^T do, dk = scale ds^T q   (summed over the query heads of a key head)      grad_kernel<KEYS = true>
//   dq = scale ds k                                                                  grad_kernel<KEYS = false>
// Scores are computed twice (7 products instead of 5) so that every sum has one owner: adding dq tile by tile from the key side
// would take atomics, whose order changes results.
#include "attention_mma.cuh"

#include <math.h>

namespace b200f {

namespace {

// ---- grad_kernel ------------------------------------------------------------------------------
// A CTA keeps a pair of tiles of 128 rows (A1, A2) and streams pairs of 64 rows (B1, B2) past them:
//   KEYS:  A1 = k, A2 = v, B1 = q, B2 = do     S = A1 B1^T, P' = A2 B2^T, acc1 (dk) += ds B1, acc2 (dv) += p B2
//   else:  A1 = q, A2 = do, B1 = k, B2 = v     acc1 (dq) += ds B1
// S and P' have two buffers, each with its own group of four warps (a row of A a thread) that turns them into p and ds in place; the
// tensor cores compute the next pair of scores and add the previous pair's products meanwhile.
// Products of 64 columns with both operands in shared memory run at 2/3 of the full rate, which its bandwidth bounds: KEYS spends 1,280
// of its 1,326 cycles a tile on them (1,024 at full rate), tensor memory being full.  Without acc2 there is room: A1 and A2 lie in
// tensor memory, and 768 of a tile's 923 cycles are the tensor cores'.
// Measured (bf16, d = 128, 8 x 2,048 queries of 16 heads on 4 key heads, 4,096 keys): 1,650 us, 830 TFLOP/s of the 5 products that the
// gradient needs, 1,160 of the 7 that run, at the clock that the power limit leaves.
constexpr int GRAD_THREADS = 384;   // TMA, MMA, two spare warps; 2 x 4 warps
constexpr int GRAD_ROWS = 64;       // rows of a streamed tile
constexpr int GRAD_MAX_STAGES = 8;
// Tiles whose products are summed up in tensor memory, 2^15 rows; then the sums go to memory and start from 0 (see SUM_TILES in attend.cu).  Even:
// the same group of warps does it every time.
constexpr int GRAD_SUM_TILES = 512;
template <int DP>
constexpr int GRAD_A_BYTES = DP / 64 * ATT_CHUNK;
template <int DP>
constexpr int GRAD_B_BYTES = DP / 64 * GRAD_ROWS * 128;
// Statistics of a streamed tile (see grad_stat_kernel), GRAD_ROWS of each: bf16 two floats; fp16 two floats and a 16-bit word, which the keys'
// pass takes, and two more floats.
template <typename T>
constexpr int GRAD_STATS = (std::is_same<T, __half>::value ? 18 : 8) * GRAD_ROWS / 4;   // floats
template <typename T>
constexpr int GRAD_KEY_STAT_BYTES = (std::is_same<T, __half>::value ? 10 : 8) * GRAD_ROWS;
constexpr int GRAD_STAT_BYTES = GRAD_KEY_STAT_BYTES<__half>;   // room for them in a stage
constexpr int STAT_DELTA = GRAD_ROWS, STAT_MOVED = 2 * GRAD_ROWS, STAT_ALONE = 5 * GRAD_ROWS / 2, STAT_FACTOR = 7 * GRAD_ROWS / 2;
template <int DP, bool KEYS>
constexpr int GRAD_STAGES = DP == 64 ? 8 : KEYS ? 4 : 6;
template <int DP, bool KEYS>
constexpr int GRAD_SM_RING = KEYS ? 2 * GRAD_A_BYTES<DP> : 0;
template <int DP, bool KEYS>
constexpr int GRAD_SM_STAT = GRAD_SM_RING<DP, KEYS> + GRAD_STAGES<DP, KEYS> * 2 * GRAD_B_BYTES<DP>;
template <int DP, bool KEYS>
constexpr int GRAD_SM_BAR = GRAD_SM_STAT<DP, KEYS> + GRAD_STAGES<DP, KEYS> * GRAD_STAT_BYTES;
template <int DP, bool KEYS>
constexpr int GRAD_SMEM = GRAD_SM_BAR<DP, KEYS> + (2 * GRAD_MAX_STAGES + 8) * 8 + 16;
static_assert(GRAD_SMEM<128, true> <= 232448 && GRAD_SMEM<128, false> <= 232448 && GRAD_SMEM<64, true> <= 232448, "shared memory of a CTA");
static_assert(GRAD_SM_STAT<64, false> >= 256 * 128, "the results' stage");
constexpr uint32_t TG_S = 0, TG_P = 128, TG_ACC1 = 256, TG_ACC2 = 384;   // S and P' of buffer b at + 64 b
constexpr uint32_t TG_A1 = 384, TG_A2 = 448;                             // not KEYS

struct GradParams {
    AttMap km, vm, qm, gm;
    AttView q, g;            // queries and output gradients (KEYS = false: A1 and A2 are read with plain loads)
    AttLengths len;
    RowTiles rt;             // query rows in tiles of GRAD_ROWS
    const float* stat;       // [unit][tile][GRAD_STATS]
    const uint32_t* range;   // fp16: [2][unit], see UnitRange
    int64_t units;
    int64_t queries;
    int heads, kv_heads, group, d;
    float scale;
    int splits;              // ranges of the streamed tiles
    int64_t blocks;          // blocks of 128 rows a unit
    uint16_t* out1;          // dk or dq; dense
    uint16_t* out2;          // dv
    float* part;             // splits > 1: [split][out1 | out2] in fp32
    float* sums;             // one range of more than GRAD_SUM_TILES tiles: [out1 | out2] in fp32
    int64_t part_stride, part2;
    int32_t* status;
};

// fp16: powers of two keep what is rounded to 16 bits clear of subnormals and of overflow.
// Weights are held 2^12 up: n of them, each 1 / n, are normal numbers up to n = 2^26.
// A row's score gradients are at most |do| |v - o| <= 2 |do| max |v|, over the values that its sequence sees.  With |do| < 2^ld, |v| < 2^lv and
// |q| < 2^lq (the largest entry) the factor 2^(13 - lv - ld) brings that bound to [2^12, 2^14), whatever other rows hold.  dq takes
// it as it is: a row is a thread's own.  dk adds up rows of different factors 2^e, so that the rows of q take the rest 2^x of a common 2^E, e + x = E
// (grad_stat_kernel writes them, exactly but for entries below 2^-22 of the row's largest): E is the largest for which no row of the unit passes
// 2^15 with x, and a row's own factor is kept unless |do| |q| is below 2^-17 of the unit's largest (the largest entry of 2^x q stays at 2^-3
// or more).  One factor for the call, from the largest |do|, lost rows 2^10 below it to subnormals (grad_q 12 % off at 4,096 keys).
// Terms below 2^-26 of their row's bound lose bits still: weights of 2^-22 and less where a value row is much longer than those that count.
constexpr int WEIGHT_BITS = 12, DS_BITS = 13, Q_BITS = 15, Q_LEAST_BITS = -2;
__device__ __forceinline__ float power_of_2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // |e| <= 126
// |x| < 2^(this), at least half of that
__device__ __forceinline__ int bits_above(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 126; }
// of a norm, from its square
__device__ __forceinline__ int norm_bits(float square) { return (bits_above(square) + 1) >> 1; }
__device__ __forceinline__ bool usable(float largest) { return largest > 0.f && largest < CUDART_INF_F; }
// 8 entries of an fp16 row: their squares added, their largest magnitude (INF where one is not finite)
__device__ __forceinline__ void add_square(const uint4& x, float* square) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = to_f32<__half>((uint16_t)w[e]), b = to_f32<__half>((uint16_t)(w[e] >> 16));
        *square = fmaf(a, a, fmaf(b, b, *square));
    }
}
__device__ __forceinline__ void add_largest(const uint4& x, float* top) {
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float a = fabsf(to_f32<__half>((uint16_t)w[e])), b = fabsf(to_f32<__half>((uint16_t)(w[e] >> 16)));
        *top = a + b != a + b ? CUDART_INF_F : fmaxf(*top, fmaxf(a, b));
    }
}

// Of the finite rows of a (sequence, key head): the largest ld + lq, and the largest lv.  Held 256 up, 0: none.
struct UnitRange {
    int row, value;
    __device__ __forceinline__ int common() const { return DS_BITS + Q_BITS - value - row; }   // E
};
__device__ __forceinline__ UnitRange unit_range(const uint32_t* range, int64_t units, int64_t unit) {
    const int row = (int)__ldcg(range + unit), value = (int)__ldcg(range + units + unit);
    return UnitRange{row ? row - 256 : 0, value ? value - 256 : 0};
}

// Score gradients of 32 columns from `col` on, ds = p (dp - delta), and the weights p.  KEYS: the columns' statistics lie at `mstat` in shared
// memory, minus log-sums, minus deltas and, fp16, what undoes the move of the query row, 2^-x: c and `factor` are of rows that were not
// moved, the deltas hold their factor already (16 bits are enough for a power of two, and the products leave shared memory little time: the
// case measured above in fp16, L2 flushed in between, 1,610 us with both factors read as floats, 1,570 so, 1,475 without any).  Else the row's own.  Steps by groups, as in weigh32.
template <typename T, bool KEYS>
__device__ __forceinline__ void grad32(const uint32_t (&s)[32], const uint32_t (&dp)[32], float c, float factor, uint32_t mstat, int col,
                                       float mlse, float mdelta, uint32_t (&wp)[16], uint32_t (&ws)[16]) {
    constexpr bool HALF = std::is_same<T, __half>::value;
#pragma unroll
    for (int g = 0; g < 16; g += 4) {
        float2 l[4], d[4], y[4], c2[4], f2[4];
        auto columns = [&](int at, float2 (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const uint4 a = lds128(mstat + (at + col + 2 * (g + e)) * 4);
                x[e] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
                x[e + 1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
            }
        };
#pragma unroll
        for (int e = 0; e < 4; e++)
            l[e] = make_float2(mlse, mlse), d[e] = make_float2(mdelta, mdelta), c2[e] = make_float2(c, c), f2[e] = make_float2(factor, factor);
        if (KEYS) {
            columns(0, l);
            columns(STAT_DELTA, d);
            if (HALF) {
                const uint4 a = lds128(mstat + STAT_MOVED * 4 + (col + 2 * g) * 2);
                const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 m = make_float2(__uint_as_float(w[e] << 16), __uint_as_float(w[e] & 0xffff0000u));
                    c2[e] = mul2(c2[e], m);
                    f2[e] = mul2(f2[e], m);
                }
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            y[e] = fma2(make_float2(__uint_as_float(s[2 * (g + e)]), __uint_as_float(s[2 * (g + e) + 1])), c2[e], l[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e].x = ex2(y[e].x);
            y[e].y = ex2(y[e].y);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float2 x = make_float2(__uint_as_float(dp[2 * (g + e)]), __uint_as_float(dp[2 * (g + e) + 1]));
            if (!HALF) d[e] = add2(x, d[e]);
            else d[e] = KEYS ? fma2(x, f2[e], d[e]) : mul2(add2(x, d[e]), f2[e]);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
            d[e] = mul2(y[e], d[e]);
            wp[g + e] = pack2<T>(y[e].x, y[e].y);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) ws[g + e] = pack2<T>(d[e].x, d[e].y);
    }
}

template <typename T, int DP, bool KEYS>
__device__ __forceinline__ void grad_item(const CUtensorMap& map_k, const CUtensorMap& map_v, const CUtensorMap& map_q, const CUtensorMap& map_g,
                                          const GradParams& p, uint8_t* smem, uint32_t item) {
    const CUtensorMap &map_b1 = KEYS ? map_q : map_k, &map_b2 = KEYS ? map_g : map_v;
    constexpr int STAGES = GRAD_STAGES<DP, KEYS>, ABYTES = GRAD_A_BYTES<DP>, BBYTES = GRAD_B_BYTES<DP>, CHUNKS = DP / 64;
    constexpr int RING = GRAD_SM_RING<DP, KEYS>;
    constexpr bool HALF = std::is_same<T, __half>::value;
    const uint32_t sbase = smem_u32(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar_full = sbase + GRAD_SM_BAR<DP, KEYS>, bar_empty = bar_full + GRAD_MAX_STAGES * 8;
    const uint32_t bar_a = bar_empty + GRAD_MAX_STAGES * 8, bar_s = bar_a + 8, bar_d = bar_s + 16, bar_p = bar_d + 16, bar_done = bar_p + 16;
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(smem + GRAD_SM_BAR<DP, KEYS> + (2 * GRAD_MAX_STAGES + 8) * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    const uint32_t ring = sbase + RING;

    // ---- this CTA's item: a block of 128 rows of A, a range of B's tiles
    const uint32_t rest = item / (uint32_t)p.blocks, blk = item - rest * (uint32_t)p.blocks;
    const uint32_t unit = rest / (uint32_t)p.splits;
    const int sp = (int)(rest - unit * p.splits);
    const int64_t b = unit / (uint32_t)p.kv_heads;
    const int kvh = (int)(unit - (uint32_t)b * p.kv_heads);
    const int64_t len = p.len.of(b);
    const int64_t row0 = (int64_t)blk * 128;
    const int64_t tiles = KEYS ? (row0 < len ? p.rt.tiles : 0) : (len + GRAD_ROWS - 1) / GRAD_ROWS;
    const int64_t per = (tiles + p.splits - 1) / p.splits;
    const int first = (int)min(tiles, per * sp);
    const int n = (int)min(tiles - first, per);

    if (n == 0) {   // nothing is seen: zeros
        const int vecs = p.d / 8, piece = threadIdx.x % vecs;
        for (int x = threadIdx.x / vecs; x < 128; x += GRAD_THREADS / vecs) {
            const int64_t row = row0 + x;
            if (threadIdx.x >= GRAD_THREADS / vecs * vecs || row >= (KEYS ? p.len.n : (int64_t)p.queries * p.group)) break;
            const uint32_t t = (uint32_t)row / (uint32_t)p.group, g = (uint32_t)row - t * (uint32_t)p.group;
            const int64_t at = (KEYS ? ((b * p.len.n + row) * p.kv_heads + kvh) * p.d
                                     : ((b * p.queries + t) * p.heads + kvh * p.group + g) * p.d) + piece * 8;
            const float none[8] = {};
            if (p.part) {
                st_global_v8(p.part + sp * p.part_stride + at, none);
                if (KEYS) st_global_v8(p.part + sp * p.part_stride + p.part2 + at, none);
            } else {
                *reinterpret_cast<uint4*>(p.out1 + at) = make_uint4(0, 0, 0, 0);
                if (KEYS) *reinterpret_cast<uint4*>(p.out2 + at) = make_uint4(0, 0, 0, 0);
            }
        }
        return;
    }
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
        }
        mbar_init(bar_a, 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(bar_s + t * 8, 1);
            mbar_init(bar_d + t * 8, 1);
            mbar_init(bar_p + t * 8, 4);
        }
        mbar_init(bar_done, 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_ptr)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (KEYS) {
        // slots that no box fills hold zeros: they are K rows of the products
        const int fill = p.rt.gb * p.rt.bt;
        if (fill < GRAD_ROWS) {
            for (int s = warp; s < 2 * STAGES; s += GRAD_THREADS / 32) zero_tile_rows(smem + RING + s * BBYTES, CHUNKS, fill, GRAD_ROWS);
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status); };
    auto waits = [&](uint32_t bar, uint32_t parity) { return (bool)__all_sync(0xffffffffu, wait(bar, parity)); };
    // what a thread of the two groups of four warps owns: a key, or a packed query row
    const int wg = (warp - 4) >> 2, ew = warp & 3;
    const uint32_t lanes = (uint32_t)(ew * 32) << 16;
    const int64_t r = row0 + ew * 32 + lane;
    const bool live = KEYS ? r < p.len.n : r < (int64_t)p.queries * p.group;
    int t = 0, g = 0;
    if (!KEYS && live) {
        t = (int)((uint32_t)r / (uint32_t)p.group);
        g = (int)((uint32_t)r - (uint32_t)t * p.group);
    }
    if (!KEYS) {
        // A1 and A2 to tensor memory: four warps each, a row a thread
        if (warp >= 4) {
            const AttView& src = wg ? p.g : p.q;
            const uint4* const row = reinterpret_cast<const uint4*>(src.at(b, t, kvh * p.group + g));
#pragma unroll
            for (int c = 0; c < DP / 64; c++) {
                uint32_t x[32];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    uint4 y = make_uint4(0, 0, 0, 0);
                    if (live && (8 * c + e) * 8 < p.d) y = __ldg(row + 8 * c + e);
                    x[4 * e] = y.x;
                    x[4 * e + 1] = y.y;
                    x[4 * e + 2] = y.z;
                    x[4 * e + 3] = y.w;
                }
                tc_st32(tmem + (wg ? TG_A2 : TG_A1) + 32 * c + lanes, x);
            }
            tc_wait_st();
            tc_fence_before();
        }
        if (warp != 0) asm volatile("bar.sync 1, %0;" ::"n"(GRAD_THREADS - 32) : "memory");
        tc_fence_after();
    }

    if (warp == 0) {
        if (elect_one()) {
            bool ok = true;
            if (KEYS) {
                mbar_arrive_expect_tx(bar_a, 2 * ABYTES);
                for (int c = 0; c < CHUNKS; c++)
                    for (int h = 0; h < 128; h += GRAD_ROWS) {
                        tma_load_4d(sbase + c * ATT_CHUNK + h * 128, &map_k, bar_a, c * 64, (int)row0 + h, kvh * p.km.head_step,
                                    (int)b * p.km.batch_step);
                        tma_load_4d(sbase + ABYTES + c * ATT_CHUNK + h * 128, &map_v, bar_a, c * 64, (int)row0 + h, kvh * p.vm.head_step,
                                    (int)b * p.vm.batch_step);
                    }
            }
            const uint32_t bytes = KEYS ? 2 * CHUNKS * p.rt.gb * p.rt.bt * 128 + GRAD_KEY_STAT_BYTES<T> : 2 * BBYTES;
            int slot = 0;
            uint32_t phase = 0;
            for (int i = 0; i < n && ok; i++) {
                ok = wait(bar_empty + slot * 8, phase ^ 1);
                if (!ok) break;
                const uint32_t full = bar_full + slot * 8, b1 = ring + slot * 2 * BBYTES, b2 = b1 + BBYTES;
                mbar_arrive_expect_tx(full, bytes);
                const int tile = first + i;
                if (KEYS) {
                    const int block = tile / p.rt.gchunks, g0 = (tile - block * p.rt.gchunks) * p.rt.gb, t0 = block * p.rt.bt;
                    for (int c = 0; c < CHUNKS; c++) {
                        tma_load_5d(b1 + c * GRAD_ROWS * 128, &map_b1, full, c * 64, g0, t0, kvh * p.qm.head_step,
                                    (int)b * p.qm.batch_step);
                        tma_load_5d(b2 + c * GRAD_ROWS * 128, &map_b2, full, c * 64, g0, t0, kvh * p.gm.head_step,
                                    (int)b * p.gm.batch_step);
                    }
                    bulk_load(sbase + GRAD_SM_STAT<DP, KEYS> + slot * GRAD_STAT_BYTES,
                              p.stat + ((int64_t)unit * p.rt.tiles + tile) * GRAD_STATS<T>, GRAD_KEY_STAT_BYTES<T>, full);
                } else {
                    for (int c = 0; c < CHUNKS; c++) {
                        tma_load_4d(b1 + c * GRAD_ROWS * 128, &map_b1, full, c * 64, tile * GRAD_ROWS, kvh * p.km.head_step,
                                    (int)b * p.km.batch_step);
                        tma_load_4d(b2 + c * GRAD_ROWS * 128, &map_b2, full, c * 64, tile * GRAD_ROWS, kvh * p.vm.head_step,
                                    (int)b * p.vm.batch_step);
                    }
                }
                if (++slot == STAGES) {
                    slot = 0;
                    phase ^= 1;
                }
            }
            if (!ok) {   // let the copies in flight land before shared memory goes away
                const long long t0 = clock64();
                while (clock64() - t0 < 2000000LL) {
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // every wait is voted on: control flow stays uniform
        const bool leader = elect_one();
        bool ok = !KEYS || waits(bar_a, 0);
        const int tail = (int)(len & (GRAD_ROWS - 1));
        const int boundary = !KEYS && len < p.len.n && tail ? (int)(len / GRAD_ROWS) - first : -1;
        int slot = 0, used = 0;
        uint32_t phase = 0;
        auto scores = [&](int i) {   // S and P' of the next stage
            if (!waits(bar_full + slot * 8, phase)) return false;
            // keys behind the sequence's end, within the tensor: K rows of the products
            if (!KEYS && i == boundary) zero_tile_rows(smem + RING + slot * 2 * BBYTES, CHUNKS, tail, GRAD_ROWS);
            const uint32_t b1 = ring + slot * 2 * BBYTES, x = 64 * (i & 1);
            if (KEYS) mma_rows<T, DP, GRAD_ROWS>(leader, tmem + TG_S + x, sbase, b1);
            else mma_rows_ts<T, DP, GRAD_ROWS>(leader, tmem + TG_S + x, tmem + TG_A1, b1);
            tc_commit_by<false>(leader, bar_s + (i & 1) * 8);
            if (KEYS) mma_rows<T, DP, GRAD_ROWS>(leader, tmem + TG_P + x, sbase + ABYTES, b1 + BBYTES);
            else mma_rows_ts<T, DP, GRAD_ROWS>(leader, tmem + TG_P + x, tmem + TG_A2, b1 + BBYTES);
            tc_commit_by<false>(leader, bar_d + (i & 1) * 8);
            if (++slot == STAGES) {
                slot = 0;
                phase ^= 1;
            }
            return true;
        };
        ok = ok && scores(0) && (n < 2 || scores(1));
        for (int i = 0; i < n && ok; i++) {
            ok = waits(bar_p + (i & 1) * 8, (i >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b1 = ring + used * 2 * BBYTES, x = 64 * (i & 1);
            const bool add = i % GRAD_SUM_TILES != 0;
            mma_weights<T, DP, GRAD_ROWS>(leader, tmem + TG_ACC1, tmem + TG_P + x, b1, add);
            if (KEYS) mma_weights<T, DP, GRAD_ROWS>(leader, tmem + TG_ACC2, tmem + TG_S + x, b1 + BBYTES, add);
            tc_commit_by<false>(leader, bar_empty + used * 8);
            if (++used == STAGES) used = 0;
            if (i + 2 < n) ok = scores(i + 2);
        }
        tc_commit_by<false>(leader, bar_done);
        if (!ok) {   // let the MMAs in flight retire before tensor memory goes away
            const long long t0 = clock64();
            while (clock64() - t0 < 200000LL) {
            }
        }
    } else if (warp >= 4) {
        const float c = p.scale * kLog2e;
        float mlse = 0.f, mdelta = 0.f, factor = 1.f;
        if (!KEYS && live) {
            const int64_t place = p.rt.place(t, g);
            const float* const st = p.stat + ((int64_t)unit * p.rt.tiles + place / GRAD_ROWS) * GRAD_STATS<T> + place % GRAD_ROWS;
            mlse = __ldcg(st);
            mdelta = __ldcg(st + (HALF ? STAT_ALONE : STAT_DELTA));
            if (HALF) factor = __ldcg(st + STAT_FACTOR);
        }
        if (KEYS && HALF) factor = power_of_2(unit_range(p.range, p.units, unit).common() - WEIGHT_BITS);
        bool ok = true;
        const int64_t at = KEYS ? ((b * p.len.n + r) * p.kv_heads + kvh) * p.d : ((b * p.queries + t) * p.heads + kvh * p.group + g) * p.d;
        // where this row's sums are kept
        auto kept = [&](bool second) { return (p.part ? p.part + sp * p.part_stride : p.sums) + (second ? p.part2 : 0) + at; };
        for (int i = wg; i < n; i += 2) {
            ok = wait(bar_s + wg * 8, (i >> 1) & 1);
            // the stage's statistics: complete since the scores are there, and not refilled before this tile's products
            if (KEYS) ok = ok && wait(bar_full + (i % STAGES) * 8, (i / STAGES) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ts = tmem + TG_S + 64 * wg + lanes, tp = tmem + TG_P + 64 * wg + lanes;
            const uint32_t stat = sbase + GRAD_SM_STAT<DP, KEYS> + (i % STAGES) * GRAD_STAT_BYTES;
            const int lim = KEYS ? GRAD_ROWS : (int)(len - (int64_t)(first + i) * GRAD_ROWS);
            uint32_t s[2][32];
            tc_ld32(ts, s[0]);
            tc_ld32(ts + 32, s[1]);
            ok = waits(bar_d + wg * 8, (i >> 1) & 1);
            if (!ok) break;
            tc_fence_after();
            uint32_t dp[2][32];
            tc_ld32(tp, dp[0]);
            tc_wait_ld32(s[0]);
            tc_wait_ld32(s[1]);
            tc_wait_ld32(dp[0]);
            tc_ld32(tp + 32, dp[1]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint32_t wp[16], ws[16];
                if (h == 1) tc_wait_ld32(dp[1]);
                grad32<T, KEYS>(s[h], dp[h], c, factor, stat, 32 * h, mlse, mdelta, wp, ws);
                if (!KEYS && lim < GRAD_ROWS) {   // keys behind the end
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        if (32 * h + 2 * e >= lim) ws[e] = 0;
                        else if (32 * h + 2 * e + 1 >= lim) ws[e] &= 0xffffu;
                    }
                }
                if (KEYS) tc_st16(ts + 16 * h, wp);
                // the second half's P' is in registers by now, or on its way to them: the first half's ds overwrites the first quarter
                tc_st16(tp + 16 * h, ws);
            }
            tc_wait_st();
            if (i > 0 && i % GRAD_SUM_TILES == 0) {
                // once the previous tile's products are done, which give their stage back: this tile's wait for bar_p, so that it is not given back again
                ok = waits(bar_empty + ((i - 1) % STAGES) * 8, ((i - 1) / STAGES) & 1);
                if (!ok) break;
                tc_fence_after();
#pragma unroll 1
                for (int ch = 0; ch < (KEYS ? 2 : 1) * DP / 16; ch++) {
                    const bool second = ch >= DP / 16;
                    const int col = (ch - (second ? DP / 16 : 0)) * 16;
                    uint32_t o[16];
                    tc_ld16_wait(tmem + (second ? TG_ACC2 : TG_ACC1) + lanes + col, o);
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        if (live && col + e < p.d) {
                            float4* const x = reinterpret_cast<float4*>(kept(second) + col + e);
                            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (i > GRAD_SUM_TILES) y = *x;
                            *x = make_float4(y.x + __uint_as_float(o[e]), y.y + __uint_as_float(o[e + 1]), y.z + __uint_as_float(o[e + 2]),
                                             y.w + __uint_as_float(o[e + 3]));
                        }
                }
            }
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if(lane == 0, bar_p + wg * 8);
        }
        if (n > GRAD_SUM_TILES) asm volatile("bar.sync 2, 256;" ::: "memory");   // one group's sums, read by both
        // ------------------------------ results: KEYS: a group of warps an accumulator, else half of its columns each
        if (ok) ok = wait(bar_done, 0);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            const bool zero = KEYS && r >= len;
            const float mul = (KEYS && wg == 1) ? 1.f : p.scale;
            float undo = 1.f;   // of the powers of two
            if (HALF) undo = KEYS && wg ? power_of_2(-WEIGHT_BITS) : power_of_2(-WEIGHT_BITS) / factor;
            const uint32_t acc = tmem + (KEYS && wg ? TG_ACC2 : TG_ACC1) + lanes;
            constexpr int COLS = KEYS ? DP : DP / 2;
            const int col0 = KEYS ? 0 : wg * COLS;
            uint8_t* const stage = smem + (warp - 4) * 32 * COLS * 2;   // tiles are done with
#pragma unroll 1
            for (int ch = 0; ch < COLS / 32; ch++) {
                const int col = col0 + 32 * ch;
                uint32_t o[32];
                tc_ld32(acc + col, o);
                tc_wait_ld32(o);
                if (n > GRAD_SUM_TILES && live) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4)
                        if (col + e < p.d) {
                            const float4 y = *reinterpret_cast<const float4*>(kept(KEYS && wg) + col + e);
                            o[e] = __float_as_uint(__uint_as_float(o[e]) + y.x);
                            o[e + 1] = __float_as_uint(__uint_as_float(o[e + 1]) + y.y);
                            o[e + 2] = __float_as_uint(__uint_as_float(o[e + 2]) + y.z);
                            o[e + 3] = __float_as_uint(__uint_as_float(o[e + 3]) + y.w);
                        }
                }
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = zero ? 0u : __float_as_uint(__uint_as_float(o[e]) * undo * mul);
                if (!p.part) {
                    stage_columns32<T, COLS>(stage, o, 4 * ch);
                } else if (live) {
                    float* const po = p.part + sp * p.part_stride + (KEYS && wg ? p.part2 : 0) + at;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (col + e < p.d) {
                            const float v[8] = {__uint_as_float(o[e]),     __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                                __uint_as_float(o[e + 3]), __uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]),
                                                __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])};
                            st_global_v8(po + col + e, v);
                        }
                }
            }
            if (!p.part) store_rows<COLS>(stage, KEYS && wg ? p.out2 : p.out1, live ? at : -1, col0, p.d);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// Items of the keys first, which take longest, then those of the query rows: one launch, one tail.
template <typename T, int DP>
__global__ void __launch_bounds__(GRAD_THREADS, 1)
grad_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_q,
            const __grid_constant__ CUtensorMap map_g, const __grid_constant__ GradParams keys, const __grid_constant__ GradParams rows,
            uint32_t key_items) {
    extern __shared__ __align__(1024) uint8_t smem[];
    pdl_wait();
    pdl_trigger();
    if ((smem_u32(smem) & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(keys.status, kDevErrSmemAlign);
        return;
    }
    if (blockIdx.x < key_items) grad_item<T, DP, true>(map_k, map_v, map_q, map_g, keys, smem, blockIdx.x);
    else grad_item<T, DP, false>(map_k, map_v, map_q, map_g, rows, smem, blockIdx.x - key_items);
}

// ---- fp16: grad_range_kernel: the units' largest rows (UnitRange) --------------------------------
// A CTA takes rows of a unit, of do and q or of v, LANES lanes a row and eight loads a lane.  A maximum does not depend on the order.  Rows that
// are not finite, or zero, do not count: their terms are NaN, or 0, whatever the factors.
template <int LANES>
constexpr int RANGE_ROWS = 4 * 256 / LANES;   // of queries; twice as many of values
template <int LANES>
__global__ void __launch_bounds__(256, 5) grad_range_kernel(AttView g, AttView q, AttView v, AttLengths len, uint32_t units, uint32_t kv_heads,
                                                            uint32_t group, int d, uint32_t* range) {
    constexpr int ROWS = RANGE_ROWS<LANES>;
    const int sub = threadIdx.x % LANES, slot = threadIdx.x / LANES;
    const uint32_t rows = (uint32_t)len.queries * group;
    const uint32_t row_blocks = (rows + ROWS - 1) / ROWS, blocks = row_blocks + (uint32_t)((len.n + 2 * ROWS - 1) / (2 * ROWS));
    for (uint32_t item = blockIdx.x; item < units * blocks; item += gridDim.x) {   // below 2^31: b200f_attend_backward sees to it
        const uint32_t unit = item / blocks, block = item - unit * blocks, b = unit / kv_heads, kvh = unit - b * kv_heads;
        uint32_t most = 0;
        auto take = [&](auto query_c, uint32_t row0, uint32_t end) __attribute__((always_inline)) {
            constexpr bool query = decltype(query_c)::value;
            constexpr int N = query ? 4 : 8;
            uint4 x[N], y[4];
#pragma unroll
            for (int k = 0; k < N; k++) {
                const uint32_t r = row0 + 256 / LANES * k + slot;
                x[k] = make_uint4(0, 0, 0, 0);
                if (query) y[k % 4] = make_uint4(0, 0, 0, 0);
                if (r < end && sub * 8 < d) {
                    const uint32_t t = query ? r / group : r, h = query ? kvh * group + (r - t * group) : kvh;
                    x[k] = *reinterpret_cast<const uint4*>((query ? g : v).at(b, t, h) + sub * 8);
                    if (query) y[k % 4] = *reinterpret_cast<const uint4*>(q.at(b, t, h) + sub * 8);
                }
            }
#pragma unroll
            for (int k = 0; k < N; k++) {
                float square = 0.f, top = 1.f;
                add_square(x[k], &square);
                if (query) top = 0.f, add_largest(y[k % 4], &top);
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) {
                    square += __shfl_xor_sync(0xffffffffu, square, o);
                    if (query) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                }
                if (usable(square) && usable(top)) most = max(most, 256u + norm_bits(square) + (query ? bits_above(top) : 0));
            }
        };
        if (block < row_blocks) {
            take(std::true_type(), block * ROWS, rows);
        } else {
            const uint32_t row0 = (block - row_blocks) * 2 * ROWS, end = (uint32_t)len.of(b);
            if (row0 >= end) continue;
            take(std::false_type(), row0, end);
        }
        most = __reduce_max_sync(0xffffffffu, most);
        uint32_t* const to = range + (block < row_blocks ? 0 : units) + unit;
        if ((threadIdx.x & 31) == 0 && most) atomicMax(to, most);
    }
}

// ---- grad_stat_kernel: what the gradients need of every query row, LANES lanes a slot ----------------------
// Of every slot minus the log-sum in base 2 (-INF: no row, or nothing to be seen) and minus delta.  fp16: the log-sum's weight is 2^WEIGHT_BITS up and
// delta is multiplied by the factor 2^(e - WEIGHT_BITS) of the keys' pass; then 2^-x (as bf16), minus delta as it is, the factor of dq; and the query
// rows 2^x q, dense, go to moved_q.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) grad_stat_kernel(AttView g, AttView q, const uint16_t* out, const float* lse, RowTiles rt, uint32_t units,
                                                        int heads, int kv_heads, int d, float c, float* stat, const uint32_t* range,
                                                        uint16_t* moved_q) {
    constexpr bool HALF = std::is_same<T, __half>::value;
    constexpr int SLOTS = 256 / LANES;   // of a CTA, all of one tile
    const int sub = threadIdx.x % LANES;
    const uint32_t tile_of = blockIdx.x / (GRAD_ROWS / SLOTS), unit = tile_of / (uint32_t)rt.tiles;
    const int slot = (int)(blockIdx.x % (GRAD_ROWS / SLOTS)) * SLOTS + threadIdx.x / LANES;
    int t, gg;
    const bool live = rt.at((int)(tile_of - unit * rt.tiles), slot, &t, &gg);
    float dot = 0.f, square = 0.f, top = 0.f;
    const uint32_t b = unit / (uint32_t)kv_heads;
    const int h = (int)(unit - b * kv_heads) * rt.group + (live ? gg : 0);
    const int64_t row = live ? ((int64_t)b * rt.queries + t) * heads + h : 0;
    const bool mine = live && sub * 8 < d;
    uint4 z = make_uint4(0, 0, 0, 0);
    if (mine) {
        const uint4 x = *reinterpret_cast<const uint4*>(g.at(b, t, h) + sub * 8);
        const uint4 y = *reinterpret_cast<const uint4*>(out + row * d + sub * 8);
        if (HALF) z = *reinterpret_cast<const uint4*>(q.at(b, t, h) + sub * 8);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            dot = fmaf(to_f32<T>((uint16_t)xs[e]), to_f32<T>((uint16_t)ys[e]), dot);
            dot = fmaf(to_f32<T>((uint16_t)(xs[e] >> 16)), to_f32<T>((uint16_t)(ys[e] >> 16)), dot);
        }
        if (HALF) {
            add_square(x, &square);
            add_largest(z, &top);
        }
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        dot += __shfl_xor_sync(0xffffffffu, dot, o);
        if (HALF) {
            square += __shfl_xor_sync(0xffffffffu, square, o);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        }
    }
    // exponents: the query row's move x, with which its score gradients have e = common - x (at most `alone`), and those for dq
    int x = 0, e = 0, alone = 0;
    if (HALF && live) {
        const UnitRange u = unit_range(range, units, unit);
        if (usable(square)) {
            alone = DS_BITS - u.value - norm_bits(square);
            x = u.common() - alone;
            if (!usable(top)) x = max(x, 0);   // zeros do not mind
            else if (c <= 1e30f) x = max(x, Q_LEAST_BITS - bits_above(top));
            else x = min(max(x, 0), Q_BITS - bits_above(top));   // c 2^-x stays finite
        }
        e = u.common() - x;
    }
    if (sub == 0) {
        const float l = live ? lse[row] * kLog2e : CUDART_INF_F;
        float* const st = stat + (int64_t)tile_of * GRAD_STATS<T> + slot;
        // -INF either way where nothing is to be seen
        st[0] = l == -CUDART_INF_F ? l : (HALF ? (float)WEIGHT_BITS - l : -l);
        const float delta = live ? -dot : 0.f;
        st[STAT_DELTA] = HALF ? delta * power_of_2(e - WEIGHT_BITS) : delta;
        if (HALF) {
            reinterpret_cast<uint16_t*>(st - slot + STAT_MOVED)[slot] = (uint16_t)(__float_as_uint(power_of_2(-x)) >> 16);
            st[STAT_ALONE] = delta;
            st[STAT_FACTOR] = power_of_2(alone - WEIGHT_BITS);
        }
    }
    if (HALF && mine) {
        const float f = power_of_2(x);
        auto moved = [&](uint32_t w) { return pack2<T>(to_f32<T>((uint16_t)w) * f, to_f32<T>((uint16_t)(w >> 16)) * f); };
        *reinterpret_cast<uint4*>(moved_q + row * d + sub * 8) = make_uint4(moved(z.x), moved(z.y), moved(z.z), moved(z.w));
    }
}

// Sums of partial gradients, in order.
template <typename T>
__global__ void __launch_bounds__(256) grad_join_kernel(const float* part, int splits, int64_t stride, int64_t n1, int64_t n2, uint16_t* out1,
                                                        uint16_t* out2) {
    pdl_wait();
    pdl_trigger();
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= n1 + n2) return;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < splits; k++) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(part + k * stride + i));
        s.x += x.x;
        s.y += x.y;
        s.z += x.z;
        s.w += x.w;
    }
    *reinterpret_cast<uint2*>(i < n1 ? out1 + i : out2 + (i - n1)) = make_uint2(pack2<T>(s.x, s.y), pack2<T>(s.z, s.w));
}

// ---- host ---------------------------------------------------------------------------------------

struct GradPlan {
    RowTiles rt;
    int64_t key_blocks, row_blocks;
    int key_splits, row_splits;
    bool key_sums, row_sums;   // one range, whose sums are moved
    size_t range_bytes, stat_bytes, moved_bytes, key_part_bytes, scratch;
};
// Ranges of the streamed tiles: where an item would take more than twice an SM's share of the work, as many as bring it down to that, of
// at least MIN_TILES tiles of 64 rows.
constexpr int MIN_TILES = 8;
GradPlan plan_grad(const B200FAttendBackwardArgs& a) {
    GradPlan pl{};
    const int group = a.heads / a.kv_heads;
    const int64_t units = a.batch * a.kv_heads, sm = cached_sm_count();
    pl.rt = row_tiles(GRAD_ROWS, a.queries, group);
    pl.key_blocks = ceil_div64(a.n, 128);
    pl.row_blocks = ceil_div64(a.queries * group, 128);
    // what an SM has to do, in tiles (a tile of the keys takes 1.4 of the rows')
    const int64_t row_tiles = ceil_div64(a.n, GRAD_ROWS);
    const int64_t share = (units * pl.key_blocks * pl.rt.tiles * 7 / 5 + units * pl.row_blocks * row_tiles) / sm;
    auto splits = [&](int64_t tiles, int64_t most) {
        if (most < MIN_TILES) most = MIN_TILES;
        return (int)(tiles > 2 * most ? ceil_div64(tiles, most) : 1);
    };
    // with nothing on one side there are no sums on the other to cut
    pl.key_splits = a.n > 0 ? splits(pl.rt.tiles, share * 5 / 7) : 1;
    pl.row_splits = a.queries > 0 ? splits(row_tiles, share) : 1;
    const bool half = a.storage == B200F_STORAGE_F16;
    const int64_t keys = units * a.n * a.d, rows = a.batch * a.queries * a.heads * a.d;
    pl.range_bytes = half ? (size_t)round_up64(2 * units * 4, 256) : 0;
    pl.stat_bytes = (size_t)round_up64(units * pl.rt.tiles * 4 * (half ? GRAD_STATS<__half> : GRAD_STATS<__nv_bfloat16>), 256);
    pl.moved_bytes = half ? (size_t)round_up64(rows * 2, 256) : 0;
    pl.key_sums = a.n > 0 && pl.key_splits == 1 && pl.rt.tiles > GRAD_SUM_TILES;
    pl.row_sums = a.queries > 0 && pl.row_splits == 1 && row_tiles > GRAD_SUM_TILES;
    pl.key_part_bytes = pl.key_splits > 1 || pl.key_sums ? (size_t)round_up64(pl.key_splits * 2 * keys * 4, 256) : 0;
    pl.scratch = 256 + pl.range_bytes + pl.stat_bytes + pl.moved_bytes + pl.key_part_bytes + (pl.row_splits > 1 || pl.row_sums ? (size_t)pl.row_splits * rows * 4 : 0);
    return pl;
}

int check_grad(const B200FAttendBackwardArgs* a) {
    if (!a) return B200F_ERR_BAD_ARG;
    return att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale);
}

template <typename T, int DP>
int launch_grad(const CUtensorMap* maps, const GradParams& keys, const GradParams& rows, int64_t key_items, int64_t row_items, cudaStream_t st) {
    constexpr int SMEM = GRAD_SMEM<DP, true> > GRAD_SMEM<DP, false> ? GRAD_SMEM<DP, true> : GRAD_SMEM<DP, false>;
    static bool attr_set[kMaxDevices] = {false};
    const int slot = device_slot();
    if (!attr_set[slot]) {
        B200F_CUDA_TRY(cudaFuncSetAttribute(grad_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        attr_set[slot] = true;
    }
    const cudaError_t e = launch_kernel(grad_kernel<T, DP>, dim3((unsigned)(key_items + row_items)), GRAD_THREADS, SMEM, Launch(st), maps[0],
                                        maps[1], maps[2], maps[3], keys, rows, (uint32_t)key_items);
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return B200F_ERR_CUDA;
    }
    count_launch();
    return B200F_OK;
}

template <typename T>
int launch_backward(const B200FAttendBackwardArgs& a, const GradPlan& pl, GradParams p, const uint16_t* out, uint8_t* scratch, const AttView& k,
                    const AttView& v) {
    constexpr bool HALF = std::is_same<T, __half>::value;
    uint32_t* const range = reinterpret_cast<uint32_t*>(scratch);
    float* const stat = reinterpret_cast<float*>(scratch + pl.range_bytes);
    uint16_t* const moved_q = reinterpret_cast<uint16_t*>(scratch + pl.range_bytes + pl.stat_bytes);
    float* const part = reinterpret_cast<float*>(scratch + pl.range_bytes + pl.stat_bytes + pl.moved_bytes);
    p.stat = stat;
    p.range = range;
    const cudaStream_t st = (cudaStream_t)a.stream;
    const int64_t units = a.batch * a.kv_heads;
    if (pl.rt.tiles > 0) {
        if (HALF) {
            B200F_CUDA_TRY(cudaMemsetAsync(range, 0, 2 * units * 4, st));
            const int64_t per = a.d <= 64 ? RANGE_ROWS<8> : RANGE_ROWS<16>, most = (int64_t)cached_sm_count() * 24;
            const int64_t items = units * (ceil_div64(a.queries * pl.rt.group, per) + ceil_div64(a.n, 2 * per));
            auto* const kernel = a.d <= 64 ? grad_range_kernel<8> : grad_range_kernel<16>;
            kernel<<<(unsigned)(items < most ? items : most), 256, 0, st>>>(p.g, p.q, v, p.len, (uint32_t)units, (uint32_t)a.kv_heads,
                                                                            (uint32_t)pl.rt.group, a.d, range);
            count_launch();
            B200F_LAUNCH_CHECK();
        }
        auto* const kernel = a.d <= 64 ? grad_stat_kernel<T, 8> : grad_stat_kernel<T, 16>;
        const int64_t blocks = units * pl.rt.tiles * (GRAD_ROWS * (a.d <= 64 ? 8 : 16) / 256);
        kernel<<<(unsigned)blocks, 256, 0, st>>>(p.g, p.q, out, a.lse, pl.rt, (uint32_t)units, a.heads, a.kv_heads, a.d, a.scale * kLog2e, stat, range,
                                                 moved_q);
        count_launch();
        B200F_LAUNCH_CHECK();
    }
    CUtensorMap maps[4] = {};
    int rc = B200F_OK;
    if (a.n > 0) {
        rc = make_rows_map(&maps[0], &p.km, k, a.storage, a.d, a.n, a.kv_heads, a.batch, GRAD_ROWS);
        if (rc == B200F_OK) rc = make_rows_map(&maps[1], &p.vm, v, a.storage, a.d, a.n, a.kv_heads, a.batch, GRAD_ROWS);
    }
    if (rc == B200F_OK && a.queries > 0) {
        const AttView moved{moved_q, a.queries * a.heads * a.d, (int64_t)a.heads * a.d, a.d};
        rc = make_queries_map(&maps[2], &p.qm, HALF ? moved : p.q, a.storage, a.d, pl.rt, a.kv_heads, a.batch);
        if (rc == B200F_OK) rc = make_queries_map(&maps[3], &p.gm, p.g, a.storage, a.d, pl.rt, a.kv_heads, a.batch);
    }
    if (rc != B200F_OK) return rc;
    const int64_t keys = units * a.n * a.d, rows = a.batch * a.queries * a.heads * a.d;
    GradParams pk = p, pr = p;
    pk.splits = pl.key_splits;
    pk.blocks = pl.key_blocks;
    pk.out1 = static_cast<uint16_t*>(a.grad_k);
    pk.out2 = static_cast<uint16_t*>(a.grad_v);
    pk.part = pl.key_splits > 1 ? part : nullptr;
    pk.sums = pl.key_sums ? part : nullptr;
    pk.part_stride = 2 * keys;
    pk.part2 = keys;
    pr.splits = pl.row_splits;
    pr.blocks = pl.row_blocks;
    pr.out1 = static_cast<uint16_t*>(a.grad_q);
    pr.out2 = nullptr;
    pr.part = pl.row_splits > 1 ? part + pl.key_part_bytes / 4 : nullptr;
    pr.sums = pl.row_sums ? part + pl.key_part_bytes / 4 : nullptr;
    pr.part_stride = rows;
    pr.part2 = 0;
    rc = a.d > 64 ? launch_grad<T, 128>(maps, pk, pr, units * pl.key_blocks * pl.key_splits, units * pl.row_blocks * pl.row_splits, st)
                  : launch_grad<T, 64>(maps, pk, pr, units * pl.key_blocks * pl.key_splits, units * pl.row_blocks * pl.row_splits, st);
    auto join = [&](const GradParams& q, int64_t n1, int64_t n2) {
        const cudaError_t e = launch_kernel(grad_join_kernel<T>, dim3((unsigned)ceil_div64((n1 + n2) / 4, 256)), 256, 0, Launch(st),
                                            static_cast<const float*>(q.part), q.splits, n1 + n2, n1, n2, q.out1, q.out2);
        if (e != cudaSuccess) {
            (void)cudaGetLastError();
            return B200F_ERR_CUDA;
        }
        count_launch();
        return B200F_OK;
    };
    if (rc == B200F_OK && pk.part) rc = join(pk, keys, keys);
    if (rc == B200F_OK && pr.part) rc = join(pr, rows, 0);
    return rc;
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" size_t b200f_attend_backward_scratch_bytes(const B200FAttendBackwardArgs* a) {
    return check_grad(a) == B200F_OK ? plan_grad(*a).scratch : 0;
}

extern "C" int b200f_attend_backward(const B200FAttendBackwardArgs* a) {
    const int rc = check_grad(a);
    if (rc != B200F_OK) return rc;
    if (a->batch == 0 || (a->queries == 0 && a->n == 0)) return B200F_OK;
    const AttView g = att_view(a->grad_out, a->grad_out_stride), q = att_view(a->q, a->q_stride);
    const AttView k = att_view(a->k, a->k_stride), v = att_view(a->v, a->v_stride);
    auto aligned = [](const void* x) { return x && (reinterpret_cast<uintptr_t>(x) & 15) == 0; };
    const int group = a->heads / a->kv_heads;
    if (!a->status ||
        (a->queries > 0 && (!att_view_ok(g, a->batch, a->queries, a->heads) || !att_view_ok(q, a->batch, a->queries, a->heads) ||
                            (group > 1 && (q.sh == 0 || g.sh == 0)) || !aligned(a->out) || !a->lse || !aligned(a->grad_q))) ||
        (a->n > 0 && (!att_view_ok(k, a->batch, a->n, a->kv_heads) || !att_view_ok(v, a->batch, a->n, a->kv_heads) ||
                      !aligned(a->grad_k) || !aligned(a->grad_v))))
        return B200F_ERR_BAD_ARG;
    const GradPlan pl = plan_grad(*a);
    if (!a->scratch || (reinterpret_cast<uintptr_t>(a->scratch) & 255) != 0 || a->scratch_bytes < pl.scratch) return B200F_ERR_SCRATCH;
    const int64_t units = a->batch * a->kv_heads, lim = 0x7fffffff;
    if (units * pl.key_blocks * pl.key_splits + units * pl.row_blocks * pl.row_splits > lim / 2 ||
        units * pl.rt.tiles * GRAD_ROWS / 16 > lim || units * a->n * a->d / 512 > lim)
        return B200F_ERR_UNSUPPORTED;
    GradParams p{};
    p.q = q;
    p.g = g;
    p.len = AttLengths{a->key_lengths, a->n, a->queries, 0};
    p.rt = pl.rt;
    p.units = units;
    p.queries = a->queries;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = group;
    p.d = a->d;
    p.scale = a->scale;
    p.status = a->status;
    const uint16_t* const out = static_cast<const uint16_t*>(a->out);
    uint8_t* const scratch = static_cast<uint8_t*>(a->scratch);
    return a->storage == B200F_STORAGE_F16 ? launch_backward<__half>(*a, pl, p, out, scratch, k, v)
                                           : launch_backward<__nv_bfloat16>(*a, pl, p, out, scratch, k, v);
}
