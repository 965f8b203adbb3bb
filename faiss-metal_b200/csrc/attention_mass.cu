// Accumulated attention weight: m_j += sum over query rows of exp(scale q.k_j - lse).
#include "attention_mma.cuh"

#include <math.h>

namespace b200f {

namespace {

// ---- mass_kernel ------------------------------------------------------------------------------
// Scores with the keys in the rows of the tile, S = K Q^T, so that a key belongs to a thread and its weights are added up in a
// register.  FEW (all query rows of a key head in one tile): the queries stay in shared memory, key tiles stream past: one read of
// the keys is the bound.  Else a key tile stays and tiles of query rows stream past; exponentials bound it.  S has two buffers, each with
// its own four warps.  Two CTAs share an SM, so that one's start and end hide behind the other.
// Measured: FEW (bf16, d = 128, 32 sequences of one query, 32 heads on 8 key heads, up to 8,192 keys) 57 us, 5.7 TB/s; else (fp16, d = 64, 2 x 1,111
// queries, 16 heads on 4 key heads, 2,049 keys) 37 us.  A quarter of the exponentials by ex2_fma, or loads of S in two buffers: 7 %
// slower.
constexpr int MASS_THREADS = 384;   // TMA, MMA, two warps for log-sums; 2 x 4 warps
constexpr int MASS_SLOTS = 128;     // query rows of a tile
constexpr int MASS_RING = 5;        // streamed tiles at most: what half an SM's shared memory takes (launch_mass)
constexpr int MASS_STATS = 4;       // query tiles whose log-sums are fetched ahead
constexpr int MASS_STAT = MASS_STATS * MASS_SLOTS * 8;

struct MassParams {
    AttMap km, qm;
    AttLengths len;
    RowTiles rt;
    const float* lse;
    const float* mass_in;
    float* mass_out;
    float* part;             // several ranges of query rows: sums [split][unit][n]
    int64_t queries, units;
    int heads, kv_heads, group;
    float scale;
    int cols;                // columns of S: the filled slots, rounded up
    int blocks;              // FEW: chunks of `chunk` key tiles a unit; else key tiles
    int chunk;
    int splits;
    int ring, a_off, ring_off, stage;   // shared memory: the tile that stays, the ring and a stage of it
    int stat_off, bar_off;
    int tmem_cols;
    int32_t* status;
};

// minus the log-sum (base 2; -INF: no row) and end of visible keys of a slot
__device__ __forceinline__ void slot_stat(const MassParams& p, int64_t b, int kvh, int64_t len, int tile, int slot, float* lse2, int* end) {
    int t, g;
    float l = CUDART_INF_F;
    int e = 0;
    if (p.rt.at(tile, slot, &t, &g)) {
        l = __ldg(p.lse + (b * p.queries + t) * p.heads + kvh * p.group + g) * kLog2e;
        if (l == -CUDART_INF_F) l = CUDART_INF_F;
        e = (int)p.len.seen(len, t);
    }
    lse2[slot] = -l;
    end[slot] = e;
}

template <typename T, int DP, bool FEW>
__global__ void __launch_bounds__(MASS_THREADS, 2)
mass_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_q, const MassParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ float other[128];
    constexpr int CHUNKS = DP / 64;
    const uint32_t sbase = smem_u32(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar_full = sbase + p.bar_off, bar_empty = bar_full + MASS_RING * 8, bar_a = bar_empty + MASS_RING * 8;
    const uint32_t bar_s = bar_a + 8, bar_free = bar_s + 16, bar_stat = bar_free + 16, bar_used = bar_stat + MASS_STATS * 8;
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(smem + p.bar_off + (2 * MASS_RING + 5 + 2 * MASS_STATS) * 8);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
    float* const stat_lse = reinterpret_cast<float*>(smem + p.stat_off);            // [MASS_STATS][MASS_SLOTS]
    int* const stat_end = reinterpret_cast<int*>(smem + p.stat_off) + MASS_STATS * MASS_SLOTS;

    if ((sbase & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(p.status, kDevErrSmemAlign);
        return;
    }
    int64_t item = blockIdx.x;
    const int blk = (int)(item % p.blocks);
    item /= p.blocks;
    const int sp = (int)(item % p.splits);
    const int64_t unit = item / p.splits;
    const int kvh = (int)(unit % p.kv_heads);
    const int64_t b = unit / p.kv_heads;
    const int64_t len = p.len.of(b);
    // streamed tiles first .. first + n
    int64_t first;
    int n;
    if (FEW) {
        first = (int64_t)blk * p.chunk;
        const int64_t last = min(first + p.chunk, (len + 127) / 128);
        n = last > first ? (int)(last - first) : 0;
        // keys behind the end keep what they have
        const int64_t j1 = min((first + p.chunk) * 128, p.len.n);
        for (int64_t j = max(first * 128, len) + threadIdx.x; j < j1; j += MASS_THREADS)
            p.mass_out[unit * p.len.n + j] = p.mass_in ? p.mass_in[unit * p.len.n + j] : 0.f;
        if (n == 0) return;
    } else {
        const int64_t key0 = (int64_t)blk * 128;
        // row tiles in front of `skip` see nothing of this key tile
        int64_t skip = 0;
        if (p.len.causal) skip = max(key0 - len + p.queries, (int64_t)0) / p.rt.bt * p.rt.gchunks;
        const int64_t tiles = key0 < len ? max(p.rt.tiles - skip, (int64_t)0) : 0;
        const int64_t per = (tiles + p.splits - 1) / p.splits;
        first = min(tiles, per * sp);
        n = (int)(min(tiles, first + per) - first);
        first += skip;
    }

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < p.ring; s++) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
        }
        mbar_init(bar_a, 1);
        for (int t = 0; t < 2; t++) {
            mbar_init(bar_s + t * 8, 1);
            mbar_init(bar_free + t * 8, 4);
        }
        for (int t = 0; t < MASS_STATS; t++) {
            mbar_init(bar_stat + t * 8, 2);
            mbar_init(bar_used + t * 8, 4);
        }
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_ptr)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    {
        // query slots that no box fills hold zeros: NaN in them would come through the sums
        const int fill = p.rt.gb * p.rt.bt;
        if (fill < p.cols) {
            if (FEW) {
                if (warp == 2) zero_tile_rows(smem + p.a_off, CHUNKS, fill, p.cols);
            } else if (warp >= 2 && warp < 2 + p.ring) {
                zero_tile_rows(smem + p.ring_off + (warp - 2) * p.stage, CHUNKS, fill, p.cols);
            }
        }
    }
    if (FEW && threadIdx.x >= 128 && threadIdx.x < 128 + MASS_SLOTS) slot_stat(p, b, kvh, len, 0, threadIdx.x - 128, stat_lse, stat_end);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status); };

    if (warp == 0) {
        if (elect_one() && n > 0) {
            bool ok = true;
            auto keys = [&](uint32_t dst, uint32_t bar, int64_t tile) {
                mbar_arrive_expect_tx(bar, CHUNKS * ATT_CHUNK);
                for (int c = 0; c < CHUNKS; c++)
                    tma_load_4d(dst + c * ATT_CHUNK, &map_k, bar, c * 64, (int)tile * 128, kvh * p.km.head_step, (int)b * p.km.batch_step);
            };
            auto queries = [&](uint32_t dst, uint32_t bar, int64_t tile) {
                mbar_arrive_expect_tx(bar, CHUNKS * p.rt.gb * p.rt.bt * 128);
                for (int c = 0; c < CHUNKS; c++)
                    tma_load_5d(dst + c * p.cols * 128, &map_q, bar, c * 64, (int)(tile % p.rt.gchunks) * p.rt.gb,
                                (int)(tile / p.rt.gchunks) * p.rt.bt, kvh * p.qm.head_step, (int)b * p.qm.batch_step);
            };
            if (FEW) queries(sbase + p.a_off, bar_a, 0);
            else keys(sbase + p.a_off, bar_a, blk);
            int slot = 0;
            uint32_t phase = 0;
            for (int i = 0; i < n && ok; i++) {
                ok = wait(bar_empty + slot * 8, phase ^ 1);
                if (!ok) break;
                if (FEW) keys(sbase + p.ring_off + slot * p.stage, bar_full + slot * 8, first + i);
                else queries(sbase + p.ring_off + slot * p.stage, bar_full + slot * 8, first + i);
                if (++slot == p.ring) {
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
        const bool leader = elect_one();
        // waits are voted on: control flow stays uniform, and one that ran out ends the loop of all lanes, with nothing committed
        bool ok = n == 0 || __all_sync(0xffffffffu, wait(bar_a, 0));
        int slot = 0;
        uint32_t phase = 0;
        const uint32_t idesc = att_idesc<T>(16, false) - (2u << 17) + ((uint32_t)(p.cols >> 3) << 17);
        for (int i = 0; i < n && ok; i++) {
            ok = __all_sync(0xffffffffu, wait(bar_full + slot * 8, phase) && wait(bar_free + (i & 1) * 8, ((i >> 1) & 1) ^ 1));
            tc_fence_after();
            const uint32_t s = sbase + p.ring_off + slot * p.stage, a = sbase + p.a_off;
            const uint32_t ka = FEW ? s : a, qa = FEW ? a : s;
#pragma unroll
            for (int c = 0; c < CHUNKS; c++) {
                const uint64_t da = make_smem_desc(ka + c * ATT_CHUNK), db = make_smem_desc(qa + c * p.cols * 128);
#pragma unroll
                for (int k = 0; k < 4; k++)
                    tc_mma_f16_by<false>(leader && ok, tmem + p.cols * (i & 1), da + 2 * k, db + 2 * k, idesc, c + k > 0);
            }
            tc_commit_by<false>(leader && ok, bar_s + (i & 1) * 8);
            tc_commit_by<false>(leader && ok, bar_empty + slot * 8);
            if (++slot == p.ring) {
                slot = 0;
                phase ^= 1;
            }
        }
        if (!ok) {   // let the MMAs in flight retire before tensor memory goes away
            const long long t0 = clock64();
            while (clock64() - t0 < 200000LL) {
            }
        }
    } else if (warp < 4) {
        // ------------------------------ log-sums of the streamed query rows
        if (!FEW) {
            for (int i = 0; i < n; i++) {
                const int x = i % MASS_STATS;
                if (!__all_sync(0xffffffffu, wait(bar_used + x * 8, ((i / MASS_STATS) & 1) ^ 1))) break;
#pragma unroll
                for (int s = 0; s < MASS_SLOTS; s += 64)
                    slot_stat(p, b, kvh, len, (int)first + i, threadIdx.x - 64 + s, stat_lse + x * MASS_SLOTS, stat_end + x * MASS_SLOTS);
                __syncwarp();
                mbar_arrive_if(lane == 0, bar_stat + x * 8);
            }
        }
    } else {
        const int wg = (warp - 4) >> 2, ew = warp & 3;
        const float c = p.scale * kLog2e;
        float sum = 0.f;
        bool ok = true;
        for (int i = wg; i < n; i += 2) {
            ok = wait(bar_s + wg * 8, (i >> 1) & 1);
            if (!FEW) ok = ok && wait(bar_stat + (i % MASS_STATS) * 8, (i / MASS_STATS) & 1);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const int64_t key = (FEW ? first + i : (int64_t)blk) * 128 + ew * 32 + lane;
            const uint32_t ts = tmem + p.cols * wg + ((uint32_t)(ew * 32) << 16);
            const uint32_t lse = sbase + p.stat_off + (FEW ? 0 : i % MASS_STATS * MASS_SLOTS * 4), ends = lse + MASS_STATS * MASS_SLOTS * 4;
            // causal: some query of the tile does not see some key of this warp
            bool masked = false;
            if (p.len.causal) {
                const int64_t tmin = FEW ? 0 : (first + i) / p.rt.gchunks * p.rt.bt;
                masked = key - lane + 32 > p.len.seen(len, tmin);
            }
            // in groups of eight, each step for the whole group (see weigh32)
            float2 part[4] = {};
            for (int c0 = 0; c0 < p.cols; c0 += 16) {
                uint32_t s[16];
                tc_ld16_wait(ts + c0, s);
#pragma unroll
                for (int h = 0; h < 16; h += 8) {
                    float2 y[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const uint4 l = lds128(lse + (c0 + h + 2 * e) * 4);   // the negated log-sums
                        y[e] = fma2(make_float2(__uint_as_float(s[h + 2 * e]), __uint_as_float(s[h + 2 * e + 1])), make_float2(c, c),
                                    make_float2(__uint_as_float(l.x), __uint_as_float(l.y)));
                        y[e + 1] = fma2(make_float2(__uint_as_float(s[h + 2 * e + 2]), __uint_as_float(s[h + 2 * e + 3])),
                                        make_float2(c, c), make_float2(__uint_as_float(l.z), __uint_as_float(l.w)));
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        y[e].x = ex2(y[e].x);
                        y[e].y = ex2(y[e].y);
                    }
                    if (masked) {
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const uint4 z = lds128(ends + (c0 + h + 2 * e) * 4);
                            if (key >= (int)z.x) y[e].x = 0.f;
                            if (key >= (int)z.y) y[e].y = 0.f;
                            if (key >= (int)z.z) y[e + 1].x = 0.f;
                            if (key >= (int)z.w) y[e + 1].y = 0.f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) part[e] = add2(part[e], y[e]);
                }
            }
            const float2 both = add2(add2(part[0], part[1]), add2(part[2], part[3]));
            sum += both.x + both.y;
            tc_fence_before();
            __syncwarp();
            mbar_arrive_if(lane == 0, bar_free + wg * 8);
            if (!FEW) mbar_arrive_if(lane == 0, bar_used + (i % MASS_STATS) * 8);
            if (FEW) {
                if (key < len) p.mass_out[unit * p.len.n + key] = (p.mass_in ? p.mass_in[unit * p.len.n + key] : 0.f) + sum;
                sum = 0.f;
            }
        }
        if (!FEW) {
            // the two groups hold the same keys
            if (wg == 1) other[ew * 32 + lane] = sum;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            if (wg == 0) {
                const int64_t key = (int64_t)blk * 128 + ew * 32 + lane;
                sum = key < len ? sum + other[ew * 32 + lane] : 0.f;
                if (key < p.len.n) {
                    if (p.part) p.part[(sp * p.units + unit) * p.len.n + key] = sum;
                    else p.mass_out[unit * p.len.n + key] = (p.mass_in ? p.mass_in[unit * p.len.n + key] : 0.f) + sum;
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
}

// mass_out = mass_in + the ranges' sums, in order.  splits = 0: no queries.
__global__ void __launch_bounds__(256) mass_join_kernel(const float* part, int splits, int64_t total, const float* mass_in, float* mass_out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    float s = 0.f;
    for (int k = 0; k < splits; k++) s += part[k * total + i];
    mass_out[i] = (mass_in ? mass_in[i] : 0.f) + s;
}

// ---- host ---------------------------------------------------------------------------------------

struct MassPlan {
    RowTiles rt;
    bool few;
    int cols, blocks, chunk, splits;
    size_t scratch;
};
MassPlan plan_mass(const B200FAttentionMassArgs& a) {
    MassPlan pl{};
    const int64_t units = a.batch * a.kv_heads, sm = cached_sm_count(), tiles = ceil_div64(a.n, 128);
    pl.rt = row_tiles(MASS_SLOTS, a.queries, a.heads / a.kv_heads);
    pl.few = pl.rt.tiles == 1;
    pl.cols = (int)round_up64(pl.rt.gb * pl.rt.bt, 16);
    pl.splits = 1;
    if (pl.few) {
        // chunks of keys: about four CTAs' turns an SM slot
        const int64_t chunk = ceil_div64(units * tiles, 8 * sm);
        pl.chunk = (int)(chunk < 1 ? 1 : chunk < tiles ? chunk : (tiles > 0 ? tiles : 1));
        pl.blocks = (int)ceil_div64(tiles, pl.chunk);
    } else {
        pl.blocks = (int)tiles;
        int64_t s = units * tiles > 0 ? 4 * sm / (units * tiles) : 1;
        // at least four row tiles a range: joining costs 3 us, as much as four take (8 heads of 4 x 512 queries and keys, d = 64: 8.8 us in one
        // range, 10.2 in two; 12 heads of 3 x 700 over 300: 10.2 and 13.2 in three; 4 key heads, 4,444 rows over 2,049: 40 and 22 in eight)
        if (s > pl.rt.tiles / 4) s = pl.rt.tiles / 4;
        pl.splits = (int)(s < 1 ? 1 : s);
    }
    pl.scratch = 256 + (pl.splits > 1 ? (size_t)pl.splits * units * a.n * 4 : 0);
    return pl;
}

int check_mass(const B200FAttentionMassArgs* a) {
    if (!a) return B200F_ERR_BAD_ARG;
    return att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale);
}

template <typename T, int DP, bool FEW>
int launch_mass(const CUtensorMap* maps, MassParams p, int64_t items, cudaStream_t st) {
    const int key_bytes = DP / 64 * ATT_CHUNK, query_bytes = DP / 64 * p.cols * 128;   // multiples of 1024
    // two CTAs an SM: with more than 48 query rows of d > 64 a third key tile would leave room for one (16 x 8,192 keys of 8 heads, 52 / 64 /
    // 128 rows: 71.3 / 72.1 / 87.4 us with three, 54.4 / 54.7 / 65.4 us with two)
    p.ring = DP == 64 ? 5 : FEW && p.cols <= 48 ? 3 : 2;
    p.a_off = 0;
    p.ring_off = FEW ? query_bytes : key_bytes;
    p.stage = FEW ? key_bytes : query_bytes;
    p.stat_off = p.ring_off + p.ring * p.stage;
    p.bar_off = p.stat_off + MASS_STAT;
    p.tmem_cols = 32;
    while (p.tmem_cols < 2 * p.cols) p.tmem_cols *= 2;
    const int smem = p.bar_off + (2 * MASS_RING + 5 + 2 * MASS_STATS) * 8 + 16;
    static bool attr_set[kMaxDevices] = {false};
    const int slot = device_slot();
    if (!attr_set[slot]) {
        // the largest layout: the ring of key tiles and a query tile of 128 rows
        B200F_CUDA_TRY(cudaFuncSetAttribute(mass_kernel<T, DP, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                            (DP == 64 ? 6 : 4) * DP / 64 * ATT_CHUNK + MASS_STAT + 256));
        attr_set[slot] = true;
    }
    mass_kernel<T, DP, FEW><<<(unsigned)items, MASS_THREADS, smem, st>>>(maps[0], maps[1], p);
    count_launch();
    B200F_LAUNCH_CHECK();
    return B200F_OK;
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" size_t b200f_attention_mass_scratch_bytes(const B200FAttentionMassArgs* a) {
    return check_mass(a) == B200F_OK ? plan_mass(*a).scratch : 0;
}

extern "C" int b200f_attention_mass(const B200FAttentionMassArgs* a) {
    int rc = check_mass(a);
    if (rc != B200F_OK) return rc;
    if (a->batch == 0 || a->n == 0) return B200F_OK;
    const AttView q = att_view(a->q, a->q_stride), k = att_view(a->k, a->k_stride);
    const int group = a->heads / a->kv_heads;
    if (!a->status || !a->mass_out || !att_view_ok(k, a->batch, a->n, a->kv_heads) ||
        (a->queries > 0 && (!att_view_ok(q, a->batch, a->queries, a->heads) || (group > 1 && q.sh == 0) || !a->lse)))
        return B200F_ERR_BAD_ARG;
    const MassPlan pl = plan_mass(*a);
    if (pl.splits > 1 && (!a->scratch || (reinterpret_cast<uintptr_t>(a->scratch) & 255) != 0 || a->scratch_bytes < pl.scratch))
        return B200F_ERR_SCRATCH;
    const cudaStream_t st = (cudaStream_t)a->stream;
    const int64_t units = a->batch * a->kv_heads, total = units * a->n, items = units * pl.blocks * pl.splits;
    if (items > 0x7fffffff || ceil_div64(total, 256) > 0x7fffffff) return B200F_ERR_UNSUPPORTED;
    if (a->queries > 0) {
        CUtensorMap maps[2] = {};
        MassParams p{};
        rc = make_rows_map(&maps[0], &p.km, k, a->storage, a->d, a->n, a->kv_heads, a->batch);
        if (rc == B200F_OK) rc = make_queries_map(&maps[1], &p.qm, q, a->storage, a->d, pl.rt, a->kv_heads, a->batch);
        if (rc != B200F_OK) return rc;
        p.len = AttLengths{a->key_lengths, a->n, a->queries, a->causal};
        p.rt = pl.rt;
        p.lse = a->lse;
        p.mass_in = a->mass_in;
        p.mass_out = a->mass_out;
        p.part = pl.splits > 1 ? static_cast<float*>(a->scratch) : nullptr;
        p.queries = a->queries;
        p.units = units;
        p.heads = a->heads;
        p.kv_heads = a->kv_heads;
        p.group = group;
        p.scale = a->scale;
        p.cols = pl.cols;
        p.blocks = pl.blocks;
        p.chunk = pl.chunk;
        p.splits = pl.splits;
        p.status = a->status;
        const bool half = a->storage == B200F_STORAGE_F16, wide = a->d > 64;
        if (pl.few)
            rc = half ? (wide ? launch_mass<__half, 128, true>(maps, p, items, st) : launch_mass<__half, 64, true>(maps, p, items, st))
                      : (wide ? launch_mass<__nv_bfloat16, 128, true>(maps, p, items, st)
                              : launch_mass<__nv_bfloat16, 64, true>(maps, p, items, st));
        else
            rc = half ? (wide ? launch_mass<__half, 128, false>(maps, p, items, st) : launch_mass<__half, 64, false>(maps, p, items, st))
                      : (wide ? launch_mass<__nv_bfloat16, 128, false>(maps, p, items, st)
                              : launch_mass<__nv_bfloat16, 64, false>(maps, p, items, st));
        if (rc != B200F_OK || pl.splits == 1) return rc;
    }
    mass_join_kernel<<<(unsigned)ceil_div64(total, 256), 256, 0, st>>>(static_cast<const float*>(a->scratch), a->queries > 0 ? pl.splits : 0,
                                                                      total, a->mass_in, a->mass_out);
    count_launch();
    B200F_LAUNCH_CHECK();
    return B200F_OK;
}
