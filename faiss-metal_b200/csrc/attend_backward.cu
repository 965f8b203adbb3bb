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
// Measured (bf16, d = 128, 8 x 2,048 queries of 16 heads on 4 key heads, 4,096 keys): 1,660 us, 830 TFLOP/s of the 5 products that the
// gradient needs, 1,160 of the 7 that run, at the clock that the power limit leaves.
constexpr int GRAD_THREADS = 384;   // TMA, MMA, two spare warps; 2 x 4 warps
constexpr int GRAD_ROWS = 64;       // rows of a streamed tile
constexpr int GRAD_MAX_STAGES = 8;
template <int DP>
constexpr int GRAD_A_BYTES = DP / 64 * ATT_CHUNK;
template <int DP>
constexpr int GRAD_B_BYTES = DP / 64 * GRAD_ROWS * 128;
constexpr int GRAD_STAT_BYTES = GRAD_ROWS * 8;
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
    const float* stat;       // [unit][tile]: of every slot minus the lse in base 2 (-INF: no row), then minus delta
    const uint32_t* gmax;    // fp16: bit pattern of the largest |do|
    int64_t queries;
    int heads, kv_heads, group, d;
    float scale;
    int splits;              // ranges of the streamed tiles
    int64_t blocks;          // blocks of 128 rows a unit
    uint16_t* out1;          // dk or dq; dense
    uint16_t* out2;          // dv
    float* part;             // splits > 1: [split][out1 | out2] in fp32
    int64_t part_stride, part2;
    int32_t* status;
};

// fp16 score gradients are multiplied by a power of two that brings the largest element of do into [2^-3, 2^-2): they stay clear of fp16's
// subnormals.  |ds| <= |do| |v - o| <= 2^-2 sqrt(128) * 2 max |v|, below 65504 while a value row's norm is below 11,500.
__device__ __forceinline__ float grad_factor(uint32_t max_bits) {
    const int e = (int)(max_bits >> 23) - 127;
    return max_bits == 0 || e > 126 ? 1.f : exp2f((float)min(max(-3 - e, -100), 100));
}

// Score gradients of 32 columns, ds = p (dp - delta), and the weights p; mstat = minus log-sums and deltas, of the columns (KEYS; an
// address in shared memory, the deltas behind the log-sums) or the row's.  Steps by groups, as in weigh32.
template <typename T, bool KEYS>
__device__ __forceinline__ void grad32(const uint32_t (&s)[32], const uint32_t (&dp)[32], float c, float factor, uint32_t mstat, float mlse,
                                       float mdelta, uint32_t (&wp)[16], uint32_t (&ws)[16]) {
    constexpr bool HALF = std::is_same<T, __half>::value;
    const float2 c2 = make_float2(c, c), f2 = make_float2(factor, factor);
#pragma unroll
    for (int g = 0; g < 16; g += 4) {
        float2 l[4], d[4], y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) l[e] = make_float2(mlse, mlse), d[e] = make_float2(mdelta, mdelta);
        if (KEYS) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const uint4 a = lds128(mstat + (2 * (g + e)) * 4), b = lds128(mstat + GRAD_ROWS * 4 + (2 * (g + e)) * 4);
                l[e] = make_float2(__uint_as_float(a.x), __uint_as_float(a.y));
                l[e + 1] = make_float2(__uint_as_float(a.z), __uint_as_float(a.w));
                d[e] = make_float2(__uint_as_float(b.x), __uint_as_float(b.y));
                d[e + 1] = make_float2(__uint_as_float(b.z), __uint_as_float(b.w));
            }
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            y[e] = fma2(make_float2(__uint_as_float(s[2 * (g + e)]), __uint_as_float(s[2 * (g + e) + 1])), c2, l[e]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e].x = ex2(y[e].x);
            y[e].y = ex2(y[e].y);
        }
#pragma unroll
        for (int e = 0; e < 4; e++) d[e] = add2(make_float2(__uint_as_float(dp[2 * (g + e)]), __uint_as_float(dp[2 * (g + e) + 1])), d[e]);
        if (HALF) {
#pragma unroll
            for (int e = 0; e < 4; e++) d[e] = mul2(d[e], f2);
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
            const uint32_t bytes = KEYS ? 2 * CHUNKS * p.rt.gb * p.rt.bt * 128 + GRAD_STAT_BYTES : 2 * BBYTES;
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
                              p.stat + ((int64_t)unit * p.rt.tiles + tile) * 2 * GRAD_ROWS, GRAD_STAT_BYTES, full);
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
            mma_weights<T, DP, GRAD_ROWS>(leader, tmem + TG_ACC1, tmem + TG_P + x, b1, i > 0);
            if (KEYS) mma_weights<T, DP, GRAD_ROWS>(leader, tmem + TG_ACC2, tmem + TG_S + x, b1 + BBYTES, i > 0);
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
        const float factor = HALF ? grad_factor(__ldcg(p.gmax)) : 1.f;
        float mlse = 0.f, mdelta = 0.f;
        if (!KEYS && live) {
            const int64_t place = p.rt.place(t, g);
            const float* const st = p.stat + ((int64_t)unit * p.rt.tiles + place / GRAD_ROWS) * 2 * GRAD_ROWS + place % GRAD_ROWS;
            mlse = __ldcg(st);
            mdelta = __ldcg(st + GRAD_ROWS);
        }
        bool ok = true;
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
                grad32<T, KEYS>(s[h], dp[h], c, factor, stat + 32 * h * 4, mlse, mdelta, wp, ws);
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
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if(lane == 0, bar_p + wg * 8);
        }
        // ------------------------------ results: KEYS: a group of warps an accumulator, else half of its columns each
        if (ok) ok = wait(bar_done, 0);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            tc_fence_after();
            const bool zero = KEYS && r >= len;
            const float mul = (KEYS && wg == 1) ? 1.f : p.scale / factor;
            const int64_t at = KEYS ? ((b * p.len.n + r) * p.kv_heads + kvh) * p.d
                                    : ((b * p.queries + t) * p.heads + kvh * p.group + g) * p.d;
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
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = zero ? 0u : __float_as_uint(__uint_as_float(o[e]) * mul);
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

// ---- grad_stat_kernel: what the gradients need of every query row, 16 lanes a slot ----------------------
template <typename T>
__global__ void __launch_bounds__(256) grad_stat_kernel(AttView g, const uint16_t* out, const float* lse, RowTiles rt, int64_t units, int heads,
                                                        int kv_heads, int d, float* stat, uint32_t* gmax) {
    const int sub = threadIdx.x & 15;
    const int64_t i = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    const bool in = i < units * rt.tiles * rt.slots;
    const int64_t tile_of = in ? i / rt.slots : 0, unit = tile_of / rt.tiles;
    int t, gg;
    const bool live = in && rt.at((int)(tile_of - unit * rt.tiles), (int)(i % rt.slots), &t, &gg);
    float dot = 0.f;
    uint32_t top = 0;
    const int h = (int)(unit % kv_heads) * rt.group + (live ? gg : 0);
    const int64_t b = unit / kv_heads;
    const int64_t row = live ? (b * rt.queries + t) * heads + h : 0;
    if (live && sub * 8 < d) {
        const uint4 x = *reinterpret_cast<const uint4*>(g.at(b, t, h) + sub * 8);
        const uint4 y = *reinterpret_cast<const uint4*>(out + row * d + sub * 8);
        const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = to_f32<T>((uint16_t)xs[e]), c = to_f32<T>((uint16_t)(xs[e] >> 16));
            dot = fmaf(a, to_f32<T>((uint16_t)ys[e]), dot);
            dot = fmaf(c, to_f32<T>((uint16_t)(ys[e] >> 16)), dot);
            top = max(top, max(__float_as_uint(a) & 0x7fffffffu, __float_as_uint(c) & 0x7fffffffu));
        }
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    if (in && sub == 0) {
        const float l = live ? lse[row] * kLog2e : CUDART_INF_F;
        float* const st = stat + tile_of * 2 * rt.slots + i % rt.slots;
        st[0] = l == -CUDART_INF_F ? l : -l;   // -INF either way where nothing is to be seen
        st[rt.slots] = live ? -dot : 0.f;
    }
    if (gmax) {   // the largest finite one; the order does not matter
        if (top >= 0x7f800000u) top = 0;
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0 && top > __ldcg(gmax)) atomicMax(gmax, top);
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
    size_t stat_bytes, key_part_bytes, scratch;
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
    pl.stat_bytes = (size_t)round_up64(units * pl.rt.tiles * GRAD_ROWS * 8, 256);
    const int64_t keys = units * a.n * a.d, rows = a.batch * a.queries * a.heads * a.d;
    pl.key_part_bytes = pl.key_splits > 1 ? (size_t)round_up64(pl.key_splits * 2 * keys * 4, 256) : 0;
    pl.scratch = 256 + pl.stat_bytes + pl.key_part_bytes + (pl.row_splits > 1 ? (size_t)pl.row_splits * rows * 4 : 0);
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
int launch_backward(const B200FAttendBackwardArgs& a, const GradPlan& pl, GradParams p, const uint16_t* out, float* stat, uint32_t* gmax,
                    float* part, const AttView& k, const AttView& v) {
    const cudaStream_t st = (cudaStream_t)a.stream;
    const int64_t units = a.batch * a.kv_heads;
    if (pl.rt.tiles > 0) {
        if (gmax) B200F_CUDA_TRY(cudaMemsetAsync(gmax, 0, 4, st));
        const int64_t slots = units * pl.rt.tiles * GRAD_ROWS;
        grad_stat_kernel<T><<<(unsigned)ceil_div64(slots, 16), 256, 0, st>>>(p.g, out, a.lse, pl.rt, units, a.heads, a.kv_heads, a.d, stat, gmax);
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
        rc = make_queries_map(&maps[2], &p.qm, p.q, a.storage, a.d, pl.rt, a.kv_heads, a.batch);
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
    pk.part_stride = 2 * keys;
    pk.part2 = keys;
    pr.splits = pl.row_splits;
    pr.blocks = pl.row_blocks;
    pr.out1 = static_cast<uint16_t*>(a.grad_q);
    pr.out2 = nullptr;
    pr.part = pl.row_splits > 1 ? part + pl.key_part_bytes / 4 : nullptr;
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
    if (units * pl.key_blocks * pl.key_splits + units * pl.row_blocks * pl.row_splits > lim ||
        units * pl.rt.tiles * GRAD_ROWS / 16 > lim || units * a->n * a->d / 512 > lim)
        return B200F_ERR_UNSUPPORTED;
    uint8_t* const scratch = static_cast<uint8_t*>(a->scratch);
    uint32_t* const gmax = a->storage == B200F_STORAGE_F16 ? reinterpret_cast<uint32_t*>(scratch) : nullptr;
    float* const stat = reinterpret_cast<float*>(scratch + 256);
    float* const part = reinterpret_cast<float*>(scratch + 256 + pl.stat_bytes);
    GradParams p{};
    p.q = q;
    p.g = g;
    p.len = AttLengths{a->key_lengths, a->n, a->queries, 0};
    p.rt = pl.rt;
    p.stat = stat;
    p.gmax = gmax;
    p.queries = a->queries;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = group;
    p.d = a->d;
    p.scale = a->scale;
    p.status = a->status;
    const uint16_t* const out = static_cast<const uint16_t*>(a->out);
    return gmax ? launch_backward<__half>(*a, pl, p, out, stat, gmax, part, k, v)
                : launch_backward<__nv_bfloat16>(*a, pl, p, out, stat, gmax, part, k, v);
}
