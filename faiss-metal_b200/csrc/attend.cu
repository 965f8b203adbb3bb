// Attention: softmax(scale * q k^T) v over keys that all sequences share and keys of each sequence.
//
// The query rows of a key head (queries x heads of its group; for shared keys those of all sequences) are packed into
// tiles of 128, so that a tensor-core tile is full whatever the head layout, and keys are read once for all rows that see them.
#include "attention_mma.cuh"

#include <math.h>

namespace b200f {

namespace {

// ---- attend_tile_kernel ------------------------------------------------------------------
// One CTA takes two streams of score tiles [128 rows][128 keys], each with its own four softmax warps (a row a thread) and its own half
// of tensor memory; one warp issues the products of both: S (128 columns, whose first half then holds the weights P) and O.  PAIR: two row tiles
// over the same keys, each key tile fetched once for both.  SPLIT (no more than 128 rows): one row tile, the streams have
// different keys.  While one stream exponentiates, the tensor cores work for the other.
// Weights are exp2(c (s - m)), times a constant, for a reference m that is taken from a row's first tile and moves, with O rescaled, only when a tile's
// weights add up to 2^15 or more: no maximum is looked for before the exponentials.  Sums stay in fp32.  The weights of the first 96
// keys go to the tensor cores while those of the others are computed.
// d <= 64 leaves tensor memory for P beside S (APART): the next scores are computed as soon as these are in registers, and the way
// round is the softmax alone.
// Measured (bf16, d = 128, 8 x 2,048 queries of 16 heads on 4 key heads, 4,096 keys): 513 us, 1,070 TFLOP/s, at the 1.48 GHz that
// the power limit leaves; 2,850 cycles for both streams' tiles, 2,048 of them of the tensor cores.  Slower when measured
// against the kernel of that time: tiles of 64 keys in two buffers a stream (789 us against 620), two threads a row (3,640 cycles
// against 3,360), an issuing warp a stream (647 us against 588).
constexpr int TILE_THREADS = 384;          // TMA, MMA, two spare warps (setmaxnreg is by four); 2 x 4 softmax warps
constexpr int TILE_REGS_FEW = 80, TILE_REGS_MANY = 208;   // 128 and 256 threads of the 384 x 168 at launch
static_assert(128 * TILE_REGS_FEW + 256 * TILE_REGS_MANY <= 384 * 168, "registers of a CTA");
constexpr int PART_KEYS = 96;             // keys whose weights are handed on first
constexpr float WEIGHTS_MAX = 32768.f;     // fp16 weights end at 65504
// The reference's own weight is 2^(this): fp16 weights down to 2^-22 of it are normal numbers and 2^-33 still counts, where a weight of 1 lost
// what lies below 2^-25, with 1,000,000 such keys 1.5 % of a row.  96 weights of 2^8 add up to less than WEIGHTS_MAX.
template <typename T>
constexpr int TILE_WEIGHT_BITS = std::is_same<T, __half>::value ? 8 : 0;
// Up to this scaled reference c m the weights are exp2(c s - c m), one operation before the exponential; c m is rounded, by 2^-12 at most here.  Beyond, where
// it would be off by whole powers of two, a row has c (s - m), and a new look at its maximum in every tile.
constexpr float NEAR_REFERENCE = 4096.f;
// ends of sequences are weighed with the reference as it is up to this power of two
template <typename T>
constexpr float TILE_MASKED_BITS = std::is_same<T, __half>::value ? 12.f : 8.f;
constexpr int TILE_KEYS = 128;
// A product is added to the sum in tensor memory with some two bits below that sum's last place, the rest cut off: a term loses 2^-26 of the sum
// on average, and 1,000,000 keys behind one that outweighs them lost 30 % of their share.  After so many tiles (2^15 keys, 2^-11 of the sum)
// a row's sums go to memory, where they are added up in fp32, and start from 0 again; so does the sum of its weights, whose small terms round the same way
// one after the other.
constexpr int SUM_TILES = 256;
constexpr int TILE_MAX_STAGES = 10;
template <int DP>
constexpr int TILE_Q_BYTES = DP / 64 * ATT_CHUNK;
template <int DP>
constexpr int TILE_STAGE_BYTES = DP / 64 * TILE_KEYS * 128;
template <int DP>
constexpr int TILE_STAGES = DP == 128 ? 5 : 10;
template <int DP>
constexpr int TILE_SM_BAR = 2 * TILE_Q_BYTES<DP> + TILE_STAGES<DP>*TILE_STAGE_BYTES<DP>;
template <int DP>
constexpr int TILE_SMEM = TILE_SM_BAR<DP> + (2 * TILE_MAX_STAGES + 14) * 8 + 16;
static_assert(TILE_SMEM<128> <= 232448 && TILE_SMEM<64> <= 232448, "shared memory of a CTA");
constexpr uint32_t TM_S = 0, TM_O = 256;   // stream t: S at 128 t, O at 256 + 128 t; P: see APART
template <int DP>
constexpr bool TILE_APART = DP == 64;
template <int DP>
constexpr uint32_t TM_P = TILE_APART<DP> ? TM_O + 64 : TM_S;

// A set of keys and the query rows that read them.  Work items: (unit, block of rows, range of keys).
struct Segment {
    int64_t n;             // keys of a unit
    AttMap km, vm;
    int rows;              // packed query rows of a unit
    int row_blocks;        // of 256 rows, or 128 (split)
    int splits;            // ranges of keys
    int split;             // SPLIT: streams take different keys
    int few;               // attend_few_kernel takes it
    int part0;             // first partial result
    int64_t items;         // CTAs
};

struct TileParams {
    Segment seg[2];        // shared, own
    AttView q;
    AttLengths len;        // own keys
    int64_t queries, rows_total;
    int heads, kv_heads, group, d;
    float scale;
    uint16_t* out;
    float* lse;
    float* part_o;         // [parts][rows_total][d], null: the one part is the result
    float2* part_sum;      // [parts][rows_total]: the reference, as a score before scaling, and the sum of the weights against it
    float* sums;           // [rows_total][d]: of streams of more than SUM_TILES tiles, where there is one part (others have part_o's rows)
    int32_t* status;
};

struct RowAt {
    int64_t b, t;
    int h;
};
// packed row r of a unit
__device__ __forceinline__ RowAt row_at(const TileParams& p, int shared, int64_t unit, int64_t r) {
    // below 2^31: batch * queries * heads
    const uint32_t tt = (uint32_t)r / (uint32_t)p.group, ub = (uint32_t)unit / (uint32_t)p.kv_heads;
    RowAt a;
    a.h = (int)(((uint32_t)unit - ub * p.kv_heads) * p.group + ((uint32_t)r - tt * p.group));
    a.b = shared ? tt / (uint32_t)p.queries : ub;
    a.t = shared ? tt % (uint32_t)p.queries : tt;
    return a;
}

template <typename T, int DP>
__global__ void __launch_bounds__(TILE_THREADS, 1)
attend_tile_kernel(const __grid_constant__ CUtensorMap map_sk, const __grid_constant__ CUtensorMap map_sv,
                   const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TileParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int STAGES = TILE_STAGES<DP>, STAGE = TILE_STAGE_BYTES<DP>, QBYTES = TILE_Q_BYTES<DP>, CHUNKS = DP / 64;
    constexpr int HALF_RING = (STAGES + 1) / 2;
    constexpr bool APART = TILE_APART<DP>;
    const uint32_t sbase = smem_u32(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar_full = sbase + TILE_SM_BAR<DP>, bar_empty = bar_full + TILE_MAX_STAGES * 8;
    const uint32_t bar_s = bar_empty + TILE_MAX_STAGES * 8, bar_p = bar_s + 16, bar_part = bar_p + 32, bar_done = bar_part + 16;   // [stream]; P: [stream][part]
    const uint32_t bar_free = bar_done + 16, bar_o = bar_free + 16;   // APART: scores read; P V done
    volatile uint32_t* tmem_ptr = reinterpret_cast<volatile uint32_t*>(smem + TILE_SMEM<DP> - 16);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);

    pdl_wait();
    pdl_trigger();
    if ((sbase & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(p.status, kDevErrSmemAlign);
        return;
    }
    // ---- this CTA's item
    const int64_t before = p.seg[0].few ? 0 : p.seg[0].items;   // CTAs of the shared keys
    const int shared = (int64_t)blockIdx.x < before ? 1 : 0;
    const Segment& sg = p.seg[shared ? 0 : 1];
    int64_t item = (int64_t)blockIdx.x - (shared ? 0 : before);
    const int rb = (int)(item % sg.row_blocks);
    item /= sg.row_blocks;
    const int sp = (int)(item % sg.splits);
    const int64_t unit = item / sg.splits;
    const int64_t row0 = (int64_t)rb * (sg.split ? 128 : 256);
    const int kvh = (int)(unit % p.kv_heads);
    const int64_t ub = shared ? 0 : unit / p.kv_heads;
    const int64_t seq_len = shared ? sg.n : p.len.of(ub);
    // keys that any row of this block sees
    int64_t seen_max = seq_len;
    if (!shared && p.len.causal) {
        const int64_t last = min((int64_t)sg.rows, row0 + (sg.split ? 128 : 256)) - 1;
        seen_max = p.len.seen(seq_len, last / p.group);
    }
    const int64_t ntiles = (seen_max + TILE_KEYS - 1) / TILE_KEYS;
    const int pieces = sg.split ? 2 * sg.splits : sg.splits;
    const int64_t per = (ntiles + pieces - 1) / pieces;
    const int64_t ka = min(ntiles, per * (sg.split ? 2 * sp : sp)), kb = min(ntiles, ka + per);
    const int64_t kb2 = min(ntiles, kb + per);
    // stream t: tiles first[t] .. first[t] + n[t]
    const int first0 = (int)ka, n0 = (int)(kb - ka);
    const int first1 = sg.split ? (int)kb : (int)ka;
    const int n1 = sg.split ? (int)(kb2 - kb) : (row0 + 128 < sg.rows ? n0 : 0);

    if (warp != 0) {
        // query rows to shared memory, swizzled as TMA would: 16-byte piece c of row r goes to piece c ^ (r & 7).  DP / 8 threads a row;
        // asynchronous, so that all rows are on their way at once, and without a division a row
        constexpr int PER_ROW = DP / 8, AT_ONCE = (TILE_THREADS - 32) / PER_ROW;
        const int nrows = sg.split ? 128 : 256, c = (threadIdx.x - 32) % PER_ROW;
        int r = (threadIdx.x - 32) / PER_ROW;
        uint32_t tt = (uint32_t)(row0 + r) / (uint32_t)p.group, g = (uint32_t)(row0 + r) - tt * p.group;
        const uint32_t dt = AT_ONCE / (uint32_t)p.group, dg = AT_ONCE - dt * p.group;
        const uint16_t* const base = p.q.at(ub, 0, (int64_t)kvh * p.group) + c * 8;
        for (; r < nrows; r += AT_ONCE) {
            const bool there = row0 + r < sg.rows && c * 8 < p.d;
            const uint32_t b = shared ? tt / (uint32_t)p.queries : 0, t = shared ? tt - b * (uint32_t)p.queries : tt;
            const uint16_t* const src = there ? base + b * p.q.sb + t * p.q.sr + g * p.q.sh : p.q.p;
            cp_async16(sbase + (r >> 7) * QBYTES + (c >> 3) * ATT_CHUNK + (r & 127) * 128 + (((c & 7) ^ (r & 7)) << 4), src, there);
            tt += dt;
            g += dg;
            if (g >= (uint32_t)p.group) {
                g -= p.group;
                tt++;
            }
        }
    }
    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(bar_s + i * 8, 1);
            mbar_init(bar_part + i * 8, 1);
            mbar_init(bar_done + i * 8, 1);
            mbar_init(bar_free + i * 8, 4);
            mbar_init(bar_o + i * 8, 1);
        }
        for (int i = 0; i < 4; i++) mbar_init(bar_p + i * 8, 4);
        mbar_fence_init();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_ptr)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_ptr;
    const uint32_t ring = sbase + 2 * QBYTES;
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status); };

    if (warp != 0) {
        asm volatile("cp.async.wait_all;" ::: "memory");
        fence_proxy_async_shared();
        asm volatile("bar.sync 1, %0;" ::"n"(TILE_THREADS - 32) : "memory");
    }
    if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TILE_REGS_FEW));
    if (warp == 0) {
        // ------------------------------ keys and values in the order of their use ------------------------------
        if (elect_one()) {
            int slot[2] = {0, HALF_RING};   // SPLIT: a half of the ring a stream
            uint32_t phase[2] = {0, 0};
            bool ok = true;
            auto load = [&](int t, const CUtensorMap* m, const AttMap& am, int tile) {
                const int s = slot[t];
                if (!ok || !(ok = wait(bar_empty + s * 8, phase[t] ^ 1))) return;
                mbar_arrive_expect_tx(bar_full + s * 8, STAGE);
                for (int c = 0; c < CHUNKS; c++)
                    tma_load_4d(ring + s * STAGE + c * TILE_KEYS * 128, m, bar_full + s * 8, c * 64, tile * TILE_KEYS,
                                kvh * am.head_step, (int)ub * am.batch_step);
                const int end = sg.split && t == 0 ? HALF_RING : STAGES;
                if (++slot[t] == end) {
                    slot[t] = t == 0 ? 0 : HALF_RING;
                    phase[t] ^= 1;
                }
            };
            const CUtensorMap* mk = shared ? &map_sk : &map_k;
            const CUtensorMap* mv = shared ? &map_sv : &map_v;
            if (n0 > 0) load(0, mk, sg.km, first0);
            if (sg.split && n1 > 0) load(1, mk, sg.km, first1);
            for (int j = 0; j < n0 && ok; j++) {
                if (APART && j + 1 < n0) load(0, mk, sg.km, first0 + j + 1);
                load(0, mv, sg.vm, first0 + j);
                if (!APART && j + 1 < n0) load(0, mk, sg.km, first0 + j + 1);
                if (sg.split && j < n1) {
                    if (APART && j + 1 < n1) load(1, mk, sg.km, first1 + j + 1);
                    load(1, mv, sg.vm, first1 + j);
                    if (!APART && j + 1 < n1) load(1, mk, sg.km, first1 + j + 1);
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
        // ------------------------------ MMA issuer ------------------------------
        // Lean, and in control flow that the compiler knows to be uniform (every wait is voted on): what this warp does between a barrier and
        // the product behind it is time the tensor cores stand still.
        const bool leader = elect_one();
        bool ok = true;
        const int tail = (int)(seq_len & (TILE_KEYS - 1));
        const int boundary = seq_len < sg.n && tail ? (int)(seq_len / TILE_KEYS) : -1;
        auto issue = [&](auto split_c) __attribute__((always_inline)) {
            constexpr bool SPLIT = decltype(split_c)::value;
            const uint64_t dq = make_smem_desc(sbase), dk = make_smem_desc(ring), dv = make_smem_desc_mn(ring, TILE_KEYS * 128);
            constexpr uint64_t QCHUNK = ATT_CHUNK >> 4, KCHUNK = (TILE_KEYS * 128) >> 4;
            const bool gives[2] = {SPLIT || n1 == 0, true};   // PAIR: the stream that uses a stage last gives it back
            int slot[2] = {0, SPLIT ? HALF_RING : 0};
            uint32_t phase[2] = {0, 0};
            auto waits = [&](uint32_t bar, uint32_t parity) __attribute__((always_inline)) {
                return (bool)__all_sync(0xffffffffu, wait(bar, parity));
            };
            auto next = [&](int t) __attribute__((always_inline)) {
                if (++slot[t] == (SPLIT && t == 0 ? HALF_RING : STAGES)) {
                    slot[t] = SPLIT && t == 1 ? HALF_RING : 0;
                    phase[t] ^= 1;
                }
            };
            auto keys_there = [&](int t) __attribute__((always_inline)) {
                return !(t == 0 || SPLIT) || waits(bar_full + slot[t] * 8, phase[t]);
            };
            auto scores = [&](int t) __attribute__((always_inline)) {   // from the next stage, which is there
                const uint64_t da = dq + (SPLIT ? 0 : t * (uint64_t)(QBYTES >> 4)), db = dk + (uint64_t)(slot[t] * (STAGE >> 4));
#pragma unroll
                for (int c = 0; c < CHUNKS; c++)
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        tc_mma_f16_by<false>(leader, tmem + TM_S + 128 * t, da + c * QCHUNK + 2 * k, db + c * KCHUNK + 2 * k,
                                             att_idesc<T>(TILE_KEYS, false), c + k > 0);
                tc_commit_by<false>(leader, bar_s + t * 8);
                if (gives[t]) tc_commit_by<false>(leader, bar_empty + slot[t] * 8);
                next(t);
            };
            // P V of tile j and, more, the scores of the next: behind it, or APART in front
            auto turn = [&](int t, int j, bool more) __attribute__((always_inline)) {
                if (APART && more) {
                    if (!keys_there(t) || !waits(bar_free + t * 8, j & 1)) return false;
                    tc_fence_after();
                    scores(t);
                }
                if (t == 0 || SPLIT) {
                    if (!waits(bar_full + slot[t] * 8, phase[t])) return false;
                    // rows behind the sequence's end, within the tensor: whatever they hold, 0 * it must be 0
                    if ((t ? first1 : first0) + j == boundary)
                        zero_tile_rows(smem + 2 * QBYTES + slot[t] * STAGE, CHUNKS, tail, TILE_KEYS);
                }
                const int s = slot[t];
                const uint64_t db = dv + (uint64_t)(s * (STAGE >> 4));
                auto product = [&](int k) __attribute__((always_inline)) {   // 16 keys
                    tc_mma_ts_by(leader, tmem + TM_O + 128 * t, tmem + TM_P<DP> + 128 * t + 8 * k, db + 128 * k, att_idesc<T>(DP, true),
                                 k > 0 ? 1u : (uint32_t)(j % SUM_TILES != 0));
                };
                if (!waits(bar_p + 2 * t * 8, j & 1)) return false;
                tc_fence_after();
#pragma unroll
                for (int k = 0; k < PART_KEYS / 16; k++) product(k);
                tc_commit_by<false>(leader, bar_part + t * 8);
                next(t);
                if (!APART && more && !keys_there(t)) return false;
                if (!waits(bar_p + (2 * t + 1) * 8, j & 1)) return false;
                tc_fence_after();
#pragma unroll
                for (int k = PART_KEYS / 16; k < TILE_KEYS / 16; k++) product(k);
                if (!more) tc_commit_by<false>(leader, bar_done + t * 8);
                else if (APART) tc_commit_by<false>(leader, bar_o + t * 8);
                else scores(t);
                if (gives[t]) tc_commit_by<false>(leader, bar_empty + s * 8);
                return true;
            };
            if (n0 > 0) {
                if (!keys_there(0)) return false;
                scores(0);
            }
            if (n1 > 0) {
                if (!keys_there(1)) return false;
                scores(1);
            }
            for (int j = 0; j < n0; j++) {
                if (!turn(0, j, j + 1 < n0)) return false;
                if (j < n1 && !turn(1, j, j + 1 < n1)) return false;
            }
            return true;
        };
        ok = sg.split ? issue(std::true_type()) : issue(std::false_type());
        if (!ok) {   // let the MMAs in flight retire before tensor memory goes away
            const long long t0 = clock64();
            while (clock64() - t0 < 200000LL) {
            }
        }
    }
    } else {
        // ------------------------------ softmax, a row a thread ------------------------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TILE_REGS_MANY));
        const int t = (warp - 4) >> 2, ew = warp & 3;
        const int nt = t ? n1 : n0, kt0 = t ? first1 : first0;
        const int64_t r = row0 + (sg.split ? 0 : t * 128) + ew * 32 + lane;
        const bool live = r < sg.rows;
        const bool warp_live = row0 + (sg.split ? 0 : t * 128) + ew * 32 < sg.rows;
        RowAt at{0, 0, 0};
        if (live) at = row_at(p, shared, unit, r);
        // keys this row sees; rows that do not exist are not masked
        const int end = !live ? 0x7ffffff0 : (int)(shared ? seq_len : p.len.seen(seq_len, at.t));
        const uint32_t ts = tmem + TM_S + 128 * t + ((uint32_t)(ew * 32) << 16);
        const uint32_t to = tmem + TM_O + 128 * t + ((uint32_t)(ew * 32) << 16), tp = tmem + TM_P<DP> + 128 * t + ((uint32_t)(ew * 32) << 16);
        const float c = p.scale * kLog2e;
        float m = -CUDART_INF_F, l = 0.f;
        float mc = CUDART_NAN_F;   // TILE_WEIGHT_BITS - c m; no reference yet: the first tile's sum fails the test below
        bool ok = true;
        const bool whole = p.part_o == nullptr;
        const int part = sg.part0 + (sg.split ? 2 * sp + t : sp);
        auto row_index = [&] { return (at.b * p.queries + at.t) * p.heads + at.h; };
        // where this row's sums are kept, in units of the reference m_kept
        auto kept_row = [&] { return whole ? p.sums + row_index() * p.d : p.part_o + (part * p.rows_total + row_index()) * p.d; };
        float m_kept = -CUDART_INF_F, l_kept = 0.f;
        auto keep_sums = [&](bool first) __attribute__((always_inline)) {
            float* const kept = kept_row();
            const float f = m_kept == m ? 1.f : ex2((m_kept - m) * c);
            m_kept = m;
            l_kept = fmaf(l_kept, f, l);
            l = 0.f;
#pragma unroll 1
            for (int i = 0; i < DP / 16; i++) {
                uint32_t o[16];
                tc_ld16_wait(to + 16 * i, o);
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                    if (live && 16 * i + e < p.d) {
                        float4* const x = reinterpret_cast<float4*>(kept + 16 * i + e);
                        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (!first) y = *x;
                        *x = make_float4(fmaf(y.x, f, __uint_as_float(o[e])), fmaf(y.y, f, __uint_as_float(o[e + 1])),
                                         fmaf(y.z, f, __uint_as_float(o[e + 2])), fmaf(y.w, f, __uint_as_float(o[e + 3])));
                    }
            }
        };
        uint32_t s[4][32];
        // weights of 32 keys to tensor memory; returns their sum
        auto weigh = [&](auto mix, uint32_t (&x)[32], float mc_now, float from, int i) __attribute__((always_inline)) {
            uint32_t w[16];
            const float2 z = weigh32<T, decltype(mix)::value>(x, c, mc_now, from, w);
            tc_st16(tp + 16 * i, w);
            return z.x + z.y;
        };
        for (int j = 0; j < nt; j++) {
            ok = __all_sync(0xffffffffu, wait(bar_s + t * 8, j & 1));
            if (!ok) break;
            tc_fence_after();
            const int lim = end - (kt0 + j) * TILE_KEYS;
            const bool masked = __any_sync(0xffffffffu, lim < TILE_KEYS);
            tc_ld32(ts, s[0]);
            if (APART && j > 0) {   // P and O may be written when the previous product is done
                ok = __all_sync(0xffffffffu, wait(bar_o + t * 8, (j - 1) & 1));
                if (!ok) break;
                tc_fence_after();
            }
            if (j > 0 && j % SUM_TILES == 0) keep_sums(j == SUM_TILES);   // the previous product is done (APART: waited for, else since the scores are there)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                constexpr int PART = PART_KEYS / 32;
                float sum = 0.f;
#pragma unroll
                for (int i = h ? PART : 0; i < (h ? 4 : PART); i++) {
                    tc_wait_ld32(s[i]);
                    if (i < 3) tc_ld32(ts + 32 * (i + 1), s[i + 1]);   // under the exponentials of this chunk
                    if (APART && i == 3) {
                        tc_fence_before();
                        __syncwarp();
                        mbar_arrive_if(lane == 0, bar_free + t * 8);
                    }
                    if (!masked) {
                        sum += weigh(std::true_type(), s[i], mc, 0.f, i);
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; e++)
                            if (32 * i + e >= lim) s[i][e] = 0xff800000u;   // -INF
                    }
                }
                if (masked || __any_sync(0xffffffffu, !(sum < WEIGHTS_MAX))) {
                    // perhaps a new reference, from the maximum of these keys, which are then weighed (once more)
                    float top = -CUDART_INF_F;
#pragma unroll
                    for (int i = h ? PART : 0; i < (h ? 4 : PART); i++)
#pragma unroll
                        for (int e = 0; e < 32; e += 2) top = max3(top, __uint_as_float(s[i][e]), __uint_as_float(s[i][e + 1]));
                    const bool grown = masked ? !(fmaf(top, c, mc) <= TILE_MASKED_BITS<T>) : !(sum < WEIGHTS_MAX);
                    const float now = grown ? fmaxf(top, m) : m;
                    const bool moved = __any_sync(0xffffffffu, now != m);
                    const float f = now == m ? 1.f : ex2((m - now) * c);   // 0 where nothing was seen before
                    m = now;
                    l *= f;
                    // scaled scores beyond fp32's range count as infinite: +INF makes the row NaN, -INF weighs nothing
                    const float m2 = m * c;
                    const bool far = !(fabsf(m2) <= NEAR_REFERENCE);
                    mc = far ? CUDART_NAN_F : (float)TILE_WEIGHT_BITS<T> - m2;   // far: the next sum is NaN and comes here
                    const float from = !far || m2 == -CUDART_INF_F ? 0.f : m2 == CUDART_INF_F ? CUDART_NAN_F : m;
                    const float add = !far ? mc : m2 == -CUDART_INF_F ? 0.f : (float)TILE_WEIGHT_BITS<T>;
                    // O holds what came before: the previous tile's product is done (APART: waited for, else since the scores are there); the first part's
                    // may be under way
                    if (moved && h == 1) {
                        ok = __all_sync(0xffffffffu, wait(bar_part + t * 8, j & 1));
                        tc_fence_after();
                    }
                    if (moved && (h == 1 || j > 0)) {
#pragma unroll 1
                        for (int i = 0; i < DP / 16; i++) {
                            uint32_t o[16];
                            tc_ld16_wait(to + 16 * i, o);
#pragma unroll
                            for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                            tc_st16(to + 16 * i, o);
                        }
                    }
                    sum = 0.f;
#pragma unroll
                    for (int i = h ? PART : 0; i < (h ? 4 : PART); i++)
                        sum += weigh(std::false_type(), s[i], add, from, i);
                }
                l += sum;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_if(lane == 0, bar_p + (2 * t + h) * 8);
            }
        }
        // ------------------------------ this row's output ------------------------------
        if (ok && nt > 0) ok = wait(bar_done + t * 8, 0);
        ok = __all_sync(0xffffffffu, ok);
        if (ok && warp_live) {
            tc_fence_after();
            const bool none = nt == 0;
            float* const kept = kept_row();
            if (nt > SUM_TILES) {
                keep_sums(false);
                l = l_kept;
            }
            const int64_t grow = row_index();
            const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
            const float lse2 = l > 0.f || l != l ? log2f(l) - (float)TILE_WEIGHT_BITS<T> + (m == -CUDART_INF_F ? 0.f : m * c) : -CUDART_INF_F;
            if (live) {
                if (whole) {
                    if (p.lse) p.lse[grow] = lse2 * kLn2;
                } else {
                    p.part_sum[part * p.rows_total + grow] = make_float2(m, l * (1.f / (float)(1 << TILE_WEIGHT_BITS<T>)));
                }
            }
            // results: through shared memory (the stream's query tile is done with), so that whole rows are written
            uint8_t* const stage = smem + t * QBYTES + ew * 32 * (DP * 2);
#pragma unroll 1
            for (int i = 0; i < DP / 32; i++) {
                uint32_t o[32];
                if (nt > SUM_TILES) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) {
                        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (live && 32 * i + e < p.d) y = *reinterpret_cast<const float4*>(kept + 32 * i + e);
                        o[e] = __float_as_uint(y.x);
                        o[e + 1] = __float_as_uint(y.y);
                        o[e + 2] = __float_as_uint(y.z);
                        o[e + 3] = __float_as_uint(y.w);
                    }
                } else if (!none) {
                    tc_ld32(to + 32 * i, o);
                    tc_wait_ld32(o);
                }
#pragma unroll
                for (int e = 0; e < 32; e++) o[e] = inv == 0.f ? 0u : __float_as_uint(__uint_as_float(o[e]) * inv);
                if (whole) {
                    stage_columns32<T, DP>(stage, o, 4 * i);
                } else if (live && !none) {
                    float* const po = kept;
#pragma unroll
                    for (int e = 0; e < 32; e += 8)
                        if (32 * i + e < p.d) {
                            const float v[8] = {__uint_as_float(o[e]),     __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                                __uint_as_float(o[e + 3]), __uint_as_float(o[e + 4]), __uint_as_float(o[e + 5]),
                                                __uint_as_float(o[e + 6]), __uint_as_float(o[e + 7])};
                            st_global_v8(po + 32 * i + e, v);
                        }
                }
            }
            if (whole) store_rows<DP>(stage, p.out, live ? grow * p.d : -1, 0, p.d);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
}

// ---- attend_few_kernel ---------------------------------------------------------------------------------
// Blocks of 16 packed query rows, at most one a unit as a rule, as when decoding: reading keys and values once is the bound, 3 us of HBM time for every
// us of tensor work even on mma.sync, whose 16-row tile wastes nothing here (a tcgen05 tile has 128).  Four warps share tiles of
// 64 keys that TMA streams in, 16 keys a warp, each with a softmax of its own; they are joined once at the end.  Two
// CTAs an SM, so that one streams while the other starts or ends.
// Measured (bf16, d = 128, 32 sequences of one query, 32 heads on 8 key heads, up to 4,096 keys, the join included): 59 us, 5.2 TB/s;
// by 128-row tiles 76 us.
constexpr int FEW_ROWS = 16;
constexpr int FEW_KEYS = 64;            // keys of a tile
constexpr int FEW_THREADS = 160;        // four warps, TMA
// The reference's own weight is 2^(this), as in the tiles; a row's largest may be 2^FEW_SLACK_BITS above it: 2^15, below fp16's end.
template <typename T>
constexpr int FEW_WEIGHT_BITS = std::is_same<T, __half>::value ? 7 : 0;
constexpr int FEW_SLACK_BITS = 8;
constexpr int FEW_SUM_TILES = 2048;     // longest range: a warp's share of it is 2^15 keys (see SUM_TILES)
template <int DP>
constexpr int FEW_TILE = DP / 64 * FEW_KEYS * 128;
template <int DP>
constexpr int FEW_STAGES = DP == 128 ? 3 : 6;
template <int DP>
constexpr int FEW_SM_BAR = FEW_STAGES<DP> * 2 * FEW_TILE<DP>;
template <int DP>
constexpr int FEW_SMEM = FEW_SM_BAR<DP> + 2 * FEW_STAGES<DP> * 8 + 16;
static_assert(4 * FEW_ROWS * (128 + 2) * 4 <= FEW_SM_BAR<128> && 4 * FEW_ROWS * (64 + 2) * 4 <= FEW_SM_BAR<64>, "the warps' results fit the ring");

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int DP>
__global__ void __launch_bounds__(FEW_THREADS, 2)
attend_few_kernel(const __grid_constant__ CUtensorMap map_sk, const __grid_constant__ CUtensorMap map_sv,
                  const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TileParams p) {
    extern __shared__ __align__(1024) uint8_t smem[];
    constexpr int STAGES = FEW_STAGES<DP>, TILE = FEW_TILE<DP>, CHUNK = FEW_KEYS * 128;
    const uint32_t sbase = smem_u32(smem);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar_full = sbase + FEW_SM_BAR<DP>, bar_empty = bar_full + STAGES * 8;
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + FEW_SM_BAR<DP> + 2 * STAGES * 8);

    // Launched behind the tile kernel of the same call, whose inputs are complete and whose results it does not read: it runs on the SMs
    // that this one leaves free, and its last CTA waits for it at its end, so that whoever waits for this grid has both.  (All CTAs
    // waiting would keep those SMs from taking the next.)
    pdl_trigger();
    if ((sbase & 1023u) != 0) {
        if (threadIdx.x == 0) atomicOr(p.status, kDevErrSmemAlign);
        return;
    }
    const int shared = p.seg[0].few && (int64_t)blockIdx.x < p.seg[0].items ? 1 : 0;
    const Segment& sg = p.seg[shared ? 0 : 1];
    const int64_t item = (int64_t)blockIdx.x - (shared || !p.seg[0].few ? 0 : p.seg[0].items);
    const uint32_t x_rb = (uint32_t)item / (uint32_t)sg.row_blocks, row0 = ((uint32_t)item - x_rb * sg.row_blocks) * FEW_ROWS;
    const uint32_t unit = x_rb / (uint32_t)sg.splits;
    const int sp = (int)(x_rb - unit * sg.splits);
    const int64_t ub = shared ? 0 : unit / (uint32_t)p.kv_heads;
    const int kvh = (int)(shared ? unit : unit - (uint32_t)ub * p.kv_heads);
    const int64_t seq_len = shared ? sg.n : p.len.of(ub);
    const int64_t ntiles = (seq_len + FEW_KEYS - 1) / FEW_KEYS;   // causal ends lie in the last tiles
    const int64_t per = (ntiles + sg.splits - 1) / sg.splits;
    const int64_t first = min(ntiles, per * sp);
    const int n = (int)(min(ntiles, first + per) - first);

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(bar_full + s * 8, 1);
            mbar_init(bar_empty + s * 8, 4);
        }
        mbar_fence_init();
    }
    __syncthreads();
    auto wait = [&](uint32_t bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.status); };
    bool ok = true;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};   // rows lane / 4 and 8 more
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[i][e] = 0.f;

    if (warp == 4) {
        if (elect_one()) {
            const CUtensorMap* mk = shared ? &map_sk : &map_k;
            const CUtensorMap* mv = shared ? &map_sv : &map_v;
            int slot = 0;
            uint32_t phase = 0;
            for (int i = 0; i < n && ok; i++) {
                ok = wait(bar_empty + slot * 8, phase ^ 1);
                if (!ok) break;
                const uint32_t dst = sbase + slot * 2 * TILE, full = bar_full + slot * 8;
                mbar_arrive_expect_tx(full, 2 * TILE);
                for (int c = 0; c < DP / 64; c++)
                    tma_load_4d(dst + c * CHUNK, mk, full, c * 64, (int)(first + i) * FEW_KEYS, kvh * sg.km.head_step,
                                (int)ub * sg.km.batch_step);
                for (int c = 0; c < DP / 64; c++)
                    tma_load_4d(dst + TILE + c * CHUNK, mv, full, c * 64, (int)(first + i) * FEW_KEYS, kvh * sg.vm.head_step,
                                (int)ub * sg.vm.batch_step);
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
    } else {
        // query fragments: rows lane / 4 and 8 more, columns 16 i + 2 (lane % 4) and 8 more
        uint32_t q[DP / 16][4];
        int64_t end[2];
        const int col = (lane & 3) * 2;
#pragma unroll
        for (int i = 0; i < DP / 16; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) q[i][e] = 0;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int r = (int)row0 + (lane >> 2) + 8 * e;
            end[e] = (int64_t)1 << 40;   // rows that do not exist are not masked
            if (r < sg.rows) {
                const RowAt at = row_at(p, shared, unit, r);
                end[e] = shared ? seq_len : p.len.seen(seq_len, at.t);
                const uint16_t* const src = p.q.at(at.b, at.t, at.h);
#pragma unroll
                for (int i = 0; i < DP / 16; i++) {
                    if (16 * i < p.d) q[i][e] = *reinterpret_cast<const uint32_t*>(src + 16 * i + col);
                    if (16 * i + 8 < p.d) q[i][2 + e] = *reinterpret_cast<const uint32_t*>(src + 16 * i + 8 + col);
                }
            }
        }
        const float c = p.scale * kLog2e;
        float from[2] = {0.f, 0.f};   // the reference, where there is one
        // this lane's row address in ldmatrix: matrix lane / 8, row lane % 8 of the warp's 16 keys
        const int mi = lane >> 3, mr = lane & 7;
        const int krow = warp * 16 + (mi >> 1) * 8 + mr, kpiece = mi & 1;   // keys: (0-7, d 0-7), (0-7, d 8-15), (8-15, ..)
        const int vrow = warp * 16 + (mi & 1) * 8 + mr, vpiece = mi >> 1;   // values: (keys 0-7, d 0-7), (8-15, d 0-7), ..
        int slot = 0;
        uint32_t phase = 0;
        for (int i = 0; i < n; i++) {
            ok = __all_sync(0xffffffffu, wait(bar_full + slot * 8, phase));
            if (!ok) break;
            const uint32_t kt = sbase + slot * 2 * TILE, vt = kt + TILE;
            const int64_t key0 = (first + i) * FEW_KEYS + warp * 16;
            float s[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < DP / 16; ks++) {
                uint32_t b[4];
                ldmatrix4(kt + (ks >> 2) * CHUNK + krow * 128 + ((((ks & 3) * 2 + kpiece) ^ mr) << 4), b);
                mma16816<T>(s[0], q[ks], b[0], b[1]);
                mma16816<T>(s[1], q[ks], b[2], b[3]);
            }
            if (key0 + 16 > seq_len && seq_len < sg.n) {
                // rows behind the sequence's end, within the tensor: whatever they hold, 0 * it must be 0
                const int dead = (int)max(seq_len - key0, (int64_t)0);
                for (int x = lane; x < (16 - dead) * (DP / 8); x += 32) {
                    const int rr = warp * 16 + dead + x / (DP / 8), pc = x % (DP / 8);
                    *reinterpret_cast<uint4*>(smem + slot * 2 * TILE + TILE + (pc >> 3) * CHUNK + rr * 128 + (pc & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
            // s[h][2 e + x]: row lane / 4 + 8 e, key key0 + 8 h + col + x
            if (__any_sync(0xffffffffu, key0 + 16 > end[0] || key0 + 16 > end[1])) {
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (key0 + 8 * h + col + (x & 1) >= end[x >> 1]) s[h][x] = -CUDART_INF_F;
            }
            float top[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                top[e] = fmaxf(fmaxf(s[0][2 * e], s[0][2 * e + 1]), fmaxf(s[1][2 * e], s[1][2 * e + 1]));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 1));
                top[e] = fmaxf(top[e], __shfl_xor_sync(0xffffffffu, top[e], 2));
            }
            const bool g0 = (top[0] - m[0]) * c > (float)FEW_SLACK_BITS, g1 = (top[1] - m[1]) * c > (float)FEW_SLACK_BITS;
            if (__any_sync(0xffffffffu, g0 || g1)) {
                const float f0 = g0 ? ex2((m[0] - top[0]) * c) : 1.f, f1 = g1 ? ex2((m[1] - top[1]) * c) : 1.f;
                if (g0) m[0] = top[0];
                if (g1) m[1] = top[1];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    // scaled scores beyond fp32's range count as infinite, as in the tiles
                    const float m2 = m[e] * c;
                    from[e] = m2 == -CUDART_INF_F ? 0.f : m2 == CUDART_INF_F ? CUDART_NAN_F : m[e];
                }
                l[0] *= f0;
                l[1] *= f1;
#pragma unroll
                for (int t = 0; t < DP / 8; t++) {
                    o[t][0] *= f0;
                    o[t][1] *= f0;
                    o[t][2] *= f1;
                    o[t][3] *= f1;
                }
            }
            uint32_t w[4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const float x = ex2(fmaf(s[h][2 * e] - from[e], c, (float)FEW_WEIGHT_BITS<T>));
                    const float y = ex2(fmaf(s[h][2 * e + 1] - from[e], c, (float)FEW_WEIGHT_BITS<T>));
                    l[e] += x + y;
                    w[2 * h + e] = pack2<T>(x, y);
                }
#pragma unroll
            for (int t = 0; t < DP / 16; t++) {
                uint32_t b[4];
                ldmatrix4_trans(vt + (t >> 2) * CHUNK + vrow * 128 + ((((t & 3) * 2 + vpiece) ^ mr) << 4), b);
                mma16816<T>(o[2 * t], w, b[0], b[1]);
                mma16816<T>(o[2 * t + 1], w, b[2], b[3]);
            }
            // The values may still be on their way to registers (the products that take them are under way): the stage is not given to TMA
            // before they are there.
            fence_proxy_async_shared();
            __syncwarp();
            mbar_arrive_if(lane == 0, bar_empty + slot * 8);
            if (++slot == STAGES) {
                slot = 0;
                phase ^= 1;
            }
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
            l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        }
    }
    // ---- the four warps' results become one, through the ring, which nobody uses any more
    __syncthreads();
    if (!*abort_flag) {
        float* const po = reinterpret_cast<float*>(smem);                       // [4][FEW_ROWS][DP]
        float* const pm = po + 4 * FEW_ROWS * DP, * const pl = pm + 4 * FEW_ROWS;   // reference, sum
        const float c = p.scale * kLog2e;
        if (warp < 4) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int r = (lane >> 2) + 8 * e;
                if ((lane & 3) == 0) {
                    pm[warp * FEW_ROWS + r] = m[e];
                    pl[warp * FEW_ROWS + r] = l[e];
                }
#pragma unroll
                for (int t = 0; t < DP / 8; t++)
                    *reinterpret_cast<float2*>(po + (warp * FEW_ROWS + r) * DP + 8 * t + (lane & 3) * 2) = make_float2(o[t][2 * e], o[t][2 * e + 1]);
            }
        }
        __syncthreads();
        const int part = sg.part0 + sp;
        const int live_rows = min(sg.rows - (int)row0, FEW_ROWS);
        for (int i = threadIdx.x; i < live_rows * (DP / 8); i += FEW_THREADS) {
            const int r = i / (DP / 8), c0 = i % (DP / 8) * 8;
            if (c0 >= p.d) continue;
            float top = -CUDART_INF_F, total = 0.f, acc[8] = {};
            for (int x = 0; x < 4; x++) top = fmaxf(top, pm[x * FEW_ROWS + r]);
            for (int x = 0; x < 4; x++) {
                const float lx = pl[x * FEW_ROWS + r];
                if (lx == 0.f) continue;   // saw nothing
                // a sum that is not 0 with maximum -INF: NaN came in
                const float mx = pm[x * FEW_ROWS + r], f = mx == top ? 1.f : ex2((mx - top) * c);
                total = fmaf(f, lx, total);
                const float* const src = po + (x * FEW_ROWS + r) * DP + c0;
#pragma unroll
                for (int e = 0; e < 8; e++) acc[e] = fmaf(f, src[e], acc[e]);
            }
            const bool none = total == 0.f;
            const float inv = none ? 0.f : 1.f / total;
            const RowAt at = row_at(p, shared, unit, row0 + r);
            const int64_t grow = (at.b * p.queries + at.t) * p.heads + at.h;
            const float lse2 = none ? -CUDART_INF_F : log2f(total) - (float)FEW_WEIGHT_BITS<T> + (top == -CUDART_INF_F ? 0.f : top * c);
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = none ? 0.f : acc[e] * inv;
            if (!p.part_o) {
                *reinterpret_cast<uint4*>(p.out + grow * p.d + c0) = make_uint4(pack2<T>(acc[0], acc[1]), pack2<T>(acc[2], acc[3]),
                                                                              pack2<T>(acc[4], acc[5]), pack2<T>(acc[6], acc[7]));
                if (c0 == 0 && p.lse) p.lse[grow] = lse2 * kLn2;
            } else {
                float4* const dst = reinterpret_cast<float4*>(p.part_o + (part * p.rows_total + grow) * p.d + c0);
                dst[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                dst[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                if (c0 == 0) p.part_sum[part * p.rows_total + grow] = make_float2(top, total * (1.f / (float)(1 << FEW_WEIGHT_BITS<T>)));
            }
        }
    }
    if (blockIdx.x == gridDim.x - 1) pdl_wait();
}

// ---- attend_join_kernel: partial results of a row become its result ------------------
// W warps a row, each W-th part, so that many parts are on their way at once (1,000 rows of 37 parts: 31 us with a warp a row).
// 8 warps a CTA, or W = 32.  Parts bring references and sums, not their log-sums: where scores are large, these differ by less than
// their rounding.
template <typename T>
__global__ void __launch_bounds__(1024) attend_join_kernel(const float* part_o, const float2* part_sum, int parts, int64_t rows, int d, int W,
                                                          float c, uint16_t* out, float* lse) {
    __shared__ float4 acc_s[32][32];
    __shared__ float total_s[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * ((blockDim.x >> 5) / W) + warp / W;
    pdl_wait();
    pdl_trigger();
    const bool in = row < rows;
    float top = -CUDART_INF_F;
    bool some = false;
    if (in) {
        for (int i = lane; i < parts; i += 32) {
            const float2 x = __ldcg(part_sum + i * rows + row);
            if (x.y == 0.f) continue;   // saw nothing
            top = fmaxf(top, x.x);
            some = true;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    some = __any_sync(0xffffffffu, some);
    float total = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    const bool mine = lane * 4 < d;
    if (in && some) {
#pragma unroll 4
        for (int i = warp % W; i < parts; i += W) {
            const float2 x = __ldcg(part_sum + i * rows + row);
            if (x.y == 0.f) continue;   // nothing was written there
            const float w = x.y * (x.x == top ? 1.f : ex2((x.x - top) * c));
            total += w;
            if (mine) {
                const float4 o = __ldcg(reinterpret_cast<const float4*>(part_o + (i * rows + row) * d) + lane);
                acc.x = fmaf(w, o.x, acc.x);
                acc.y = fmaf(w, o.y, acc.y);
                acc.z = fmaf(w, o.z, acc.z);
                acc.w = fmaf(w, o.w, acc.w);
            }
        }
    }
    if (W > 1) {
        acc_s[warp][lane] = acc;
        if (lane == 0) total_s[warp] = total;
        __syncthreads();
        if (warp % W != 0) return;
        for (int x = 1; x < W; x++) {
            const float4 o = acc_s[warp + x][lane];
            acc.x += o.x;
            acc.y += o.y;
            acc.z += o.z;
            acc.w += o.w;
            total += total_s[warp + x];
        }
    }
    if (!in) return;
    const float inv = some ? 1.f / total : 0.f;
    if (mine)
        *reinterpret_cast<uint2*>(out + row * d + lane * 4) =
                make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    if (lane == 0 && lse) lse[row] = some ? ((top == -CUDART_INF_F ? 0.f : top * c) + log2f(total)) * kLn2 : -CUDART_INF_F;
}

// ---- host ---------------------------------------------------------------------------------------

struct AttendPlan {
    Segment seg[2];
    int64_t items[2];   // CTAs of the tile kernel, of the few-rows kernel
    int parts;
    bool sums;          // TileParams::sums is wanted
    size_t scratch;
};

// How a segment's work is cut: ranges of keys that fill the SMs, of at least MIN_TILES tiles; and by which kernel.  Blocks of more than
// 16 rows may go to either: the few-rows kernel starts and ends sooner, but reads the keys again for every block.  What is measured
// (us, bf16, d = 128): a tile CTA 7 and 1.7 a tile of 128 keys, one an SM; a few-rows CTA 3.5 and 0.5 a tile of 64, two an SM; joining parts
// 4.5.  Few-rows / tiles at d = 128, then at d = 64: 2 units of 64 rows over 4,096 keys 10.6 / 15.7, 9.2 / 13.9; 2 of 48 over 16,384 16.7 / 18.4,
// 14.1 / 16.9; 8 of 512 over 256 8.3 / 12.9, 6.0 / 10.8; 8 of 512 over 512 19.2 / 16.0, 14.7 / 13.5; 64 of 48 over 512 17.8 / 13.8, 13.6 /
// 11.9; 148 of 64 over 1,024 43.8 / 20.9, 30.6 / 18.8.  Both cost less at d = 64, in much the same measure: of twelve such pairs at d = 128, 64 and 32
// each the faster side was taken every time.
constexpr int MIN_TILES = 2;
constexpr int FEW_MIN_TILES = 4;
constexpr double TILE_START_US = 7, TILE_US = 1.7, FEW_START_US = 3.5, FEW_US = 0.5, JOIN_US = 4.5;

// share: CTAs that the segment may fill.  Returns its time.
double cut_tiles(Segment& s, int64_t units, int64_t rows, double share, bool joined) {
    const int64_t tiles = ceil_div64(s.n, TILE_KEYS);
    // a join costs what three or four tiles take, one after the other
    const int64_t alone = joined ? 1 : 4;
    s.few = 0;
    s.split = rows <= 128 && tiles > alone;
    s.row_blocks = (int)ceil_div64(rows, s.split ? 128 : 256);
    const int64_t base = units * s.row_blocks, most = tiles <= alone ? 1 : tiles / (s.split ? 2 * MIN_TILES : MIN_TILES);
    int64_t splits = (int64_t)(share / base);
    if (splits > most) splits = most;
    s.splits = (int)(splits < 1 ? 1 : splits);
    s.items = base * s.splits;
    const int streams = s.split ? 2 * s.splits : s.splits;
    const int64_t sm = cached_sm_count();
    return (double)ceil_div64(s.items, sm) * (TILE_START_US + TILE_US * (double)ceil_div64(tiles, streams)) +
           (!joined && streams > 1 ? JOIN_US : 0);
}
double cut_few(Segment& s, int64_t units, int64_t rows, bool joined) {
    const int64_t tiles = ceil_div64(s.n, FEW_KEYS), sm = cached_sm_count();
    s.few = 1;
    s.split = 0;
    s.row_blocks = (int)ceil_div64(rows, FEW_ROWS);
    const int64_t base = units * s.row_blocks;
    // one turn of the two CTAs an SM takes; with more blocks than SMs about four, since sequences differ in length
    int64_t want = (base >= sm ? 8 : 2) * sm / base;
    if (want > tiles / FEW_MIN_TILES) want = tiles / FEW_MIN_TILES;
    if (want < ceil_div64(tiles, FEW_SUM_TILES)) want = ceil_div64(tiles, FEW_SUM_TILES);
    s.splits = (int)(want < 1 ? 1 : want);
    s.items = base * s.splits;
    return (double)ceil_div64(s.items, 2 * sm) * (FEW_START_US + FEW_US * (double)ceil_div64(tiles, s.splits)) +
           (!joined && s.splits > 1 ? JOIN_US : 0);
}

// Tiles beside blocks of 16 rows, which take few_us on all SMs: as many SMs for the tiles as make both end soonest.  64 tokens, 32 heads on 8, behind
// 32,768 shared and up to 1,024 own rows: 80 us with 0.6 - 0.7 of the SMs, 90 us with all, one kernel after the other; 128 tokens, 16
// heads on 2, behind 4,096 and up to 512: 33 - 36 us against 43; with all but 5 us the tiles' work all is best (32 x 2 tokens behind 65,536 rows: 73 us
// against 78 with 0.8).
void leave_sms(Segment& s, int64_t units, int64_t rows, double few_us) {
    const double sm = (double)cached_sm_count();
    const int64_t base = units * s.row_blocks;
    Segment best = s;
    double least = 1e30;
    for (int64_t splits = s.splits; splits >= 1; splits--) {
        Segment t = s;
        const double us = cut_tiles(t, units, rows, (double)(base * splits), true), left = sm - (double)t.items;
        if (left < 0) continue;
        const double total = left * us >= few_us * sm ? us : (us * (double)t.items + few_us * sm) / sm;
        if (total < least) {
            least = total;
            best = t;
        }
    }
    s = best;
}

AttendPlan plan_attend(const B200FAttendArgs& a) {
    AttendPlan pl{};
    const int group = a.heads / a.kv_heads;
    const double sm = (double)cached_sm_count();
    const bool joined = a.shared_n > 0 && a.n > 0;
    int64_t units[2], rows_of[2];
    bool on[2];
    double weight[2] = {0, 0}, few_us[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        Segment& s = pl.seg[i];
        units[i] = i == 0 ? a.kv_heads : a.batch * a.kv_heads;
        s.n = i == 0 ? a.shared_n : a.n;
        rows_of[i] = (i == 0 ? a.batch : 1) * a.queries * group;
        s.rows = (int)rows_of[i];
        s.splits = s.row_blocks = 1;
        // without any keys rows of zeros are written by the own segment
        on[i] = s.n > 0 || (i == 1 && a.shared_n == 0);
        if (!on[i]) {
            s.few = 1;   // no CTAs of either kernel
            continue;
        }
        Segment tile = s;
        few_us[i] = cut_few(s, units[i], rows_of[i], joined);
        if (rows_of[i] <= FEW_ROWS) continue;
        if (cut_tiles(tile, units[i], rows_of[i], sm, joined) < few_us[i]) {
            s = tile;
            weight[i] = (double)units[i] * s.row_blocks * (double)ceil_div64(s.n, TILE_KEYS);
        }
    }
    // both by tiles: each gets the SMs that its tiles ask for; one: it leaves some to the other kernel
    if (weight[0] > 0 && weight[1] > 0)
        for (int i = 0; i < 2; i++) (void)cut_tiles(pl.seg[i], units[i], rows_of[i], sm * weight[i] / (weight[0] + weight[1]), joined);
    for (int i = 0; i < 2; i++)
        if (weight[i] > 0 && on[1 - i] && pl.seg[1 - i].few) leave_sms(pl.seg[i], units[i], rows_of[i], few_us[1 - i]);
    for (int i = 0; i < 2; i++) {
        Segment& s = pl.seg[i];
        s.part0 = pl.parts;
        pl.items[s.few] += s.items;
        const int streams = s.split ? 2 * s.splits : s.splits;
        if (s.items > 0) pl.parts += streams;
        if (!s.few && ceil_div64(ceil_div64(s.n, TILE_KEYS), streams) > SUM_TILES) pl.sums = true;
    }
    if (pl.parts > 1) pl.sums = false;
    const int64_t rows = a.batch * a.queries * a.heads;
    pl.scratch = 256;
    if (pl.sums) pl.scratch = (size_t)(256 + rows * a.d * 4);
    if (pl.parts > 1) pl.scratch = (size_t)(round_up64(pl.parts * rows * 8, 256) + pl.parts * rows * a.d * 4);
    return pl;
}

int check_attend(const B200FAttendArgs* a) {
    if (!a) return B200F_ERR_BAD_ARG;
    const int rc = att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale);
    if (rc != B200F_OK) return rc;
    if (a->shared_n < 0) return B200F_ERR_BAD_ARG;
    return a->shared_n > ((int64_t)1 << 31) - 1025 ? B200F_ERR_UNSUPPORTED : B200F_OK;
}

template <typename T, int DP>
int launch_attend(const CUtensorMap* maps, const TileParams& p, const AttendPlan& pl, cudaStream_t st) {
    static bool attr_set[kMaxDevices] = {false};
    const int slot = device_slot();
    if (!attr_set[slot]) {
        B200F_CUDA_TRY(cudaFuncSetAttribute(attend_tile_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, TILE_SMEM<DP>));
        B200F_CUDA_TRY(cudaFuncSetAttribute(attend_few_kernel<T, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM<DP>));
        attr_set[slot] = true;
    }
    cudaError_t e = cudaSuccess;
    if (pl.items[0] > 0) {
        e = launch_kernel(attend_tile_kernel<T, DP>, dim3((unsigned)pl.items[0]), TILE_THREADS, TILE_SMEM<DP>, Launch(st), maps[0], maps[1],
                          maps[2], maps[3], p);
        count_launch();
    }
    if (e == cudaSuccess && pl.items[1] > 0) {
        e = launch_kernel(attend_few_kernel<T, DP>, dim3((unsigned)pl.items[1]), FEW_THREADS, FEW_SMEM<DP>, Launch(st, pl.items[0] > 0),
                          maps[0], maps[1], maps[2], maps[3], p);
        count_launch();
    }
    if (e == cudaSuccess && pl.parts > 1) {
        const int W = pl.parts > 64 ? 32 : pl.parts > 16 ? 8 : pl.parts > 8 ? 4 : pl.parts > 4 ? 2 : 1, warps = W > 8 ? W : 8;
        e = launch_kernel(attend_join_kernel<T>, dim3((unsigned)ceil_div64(p.rows_total, warps / W)), 32 * warps, 0, Launch(st, true),
                          static_cast<const float*>(p.part_o), static_cast<const float2*>(p.part_sum), pl.parts, p.rows_total, p.d, W,
                          p.scale * kLog2e, p.out, p.lse);
        count_launch();
    }
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return B200F_ERR_CUDA;
    }
    return B200F_OK;
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" size_t b200f_attend_scratch_bytes(const B200FAttendArgs* a) {
    if (check_attend(a) != B200F_OK) return 0;
    return a->batch == 0 || a->queries == 0 ? 256 : plan_attend(*a).scratch;
}

extern "C" int b200f_attend(const B200FAttendArgs* a) {
    int rc = check_attend(a);
    if (rc != B200F_OK) return rc;
    if (a->batch == 0 || a->queries == 0) return B200F_OK;
    const AttView q = att_view(a->q, a->q_stride), k = att_view(a->k, a->k_stride), v = att_view(a->v, a->v_stride);
    const AttView sk{static_cast<const uint16_t*>(a->shared_k), 0, a->shared_k_stride[0], a->shared_k_stride[1]};
    const AttView sv{static_cast<const uint16_t*>(a->shared_v), 0, a->shared_v_stride[0], a->shared_v_stride[1]};
    if (!att_view_ok(q, a->batch, a->queries, a->heads) || !a->out || (reinterpret_cast<uintptr_t>(a->out) & 15) != 0 || !a->status ||
        (a->n > 0 && (!att_view_ok(k, a->batch, a->n, a->kv_heads) || !att_view_ok(v, a->batch, a->n, a->kv_heads))) ||
        (a->shared_n > 0 && (!att_view_ok(sk, 1, a->shared_n, a->kv_heads) || !att_view_ok(sv, 1, a->shared_n, a->kv_heads))))
        return B200F_ERR_BAD_ARG;
    AttendPlan pl = plan_attend(*a);
    if ((pl.parts > 1 || pl.sums) && (!a->scratch || (reinterpret_cast<uintptr_t>(a->scratch) & 255) != 0 || a->scratch_bytes < pl.scratch))
        return B200F_ERR_SCRATCH;
    if (pl.items[0] > 0x7fffffff || pl.items[1] > 0x7fffffff) return B200F_ERR_UNSUPPORTED;
    CUtensorMap maps[4] = {};
    if (a->shared_n > 0) {
        rc = make_rows_map(&maps[0], &pl.seg[0].km, sk, a->storage, a->d, a->shared_n, a->kv_heads, 1, pl.seg[0].few ? FEW_KEYS : TILE_KEYS);
        if (rc == B200F_OK) rc = make_rows_map(&maps[1], &pl.seg[0].vm, sv, a->storage, a->d, a->shared_n, a->kv_heads, 1, pl.seg[0].few ? FEW_KEYS : TILE_KEYS);
    }
    if (a->n > 0 && rc == B200F_OK) {
        rc = make_rows_map(&maps[2], &pl.seg[1].km, k, a->storage, a->d, a->n, a->kv_heads, a->batch, pl.seg[1].few ? FEW_KEYS : TILE_KEYS);
        if (rc == B200F_OK) rc = make_rows_map(&maps[3], &pl.seg[1].vm, v, a->storage, a->d, a->n, a->kv_heads, a->batch, pl.seg[1].few ? FEW_KEYS : TILE_KEYS);
    }
    if (rc != B200F_OK) return rc;
    TileParams p{};
    p.seg[0] = pl.seg[0];
    p.seg[1] = pl.seg[1];
    p.q = q;
    p.len = AttLengths{a->key_lengths, a->n, a->queries, a->causal};
    p.queries = a->queries;
    p.rows_total = a->batch * a->queries * a->heads;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.group = a->heads / a->kv_heads;
    p.d = a->d;
    p.scale = a->scale;
    p.out = static_cast<uint16_t*>(a->out);
    p.lse = a->lse;
    p.status = a->status;
    if (pl.parts > 1) {
        p.part_sum = static_cast<float2*>(a->scratch);
        p.part_o = static_cast<float*>(a->scratch) + round_up64(pl.parts * p.rows_total * 2, 64);
    }
    if (pl.sums) p.sums = static_cast<float*>(a->scratch);
    const cudaStream_t st = (cudaStream_t)a->stream;
    if (a->storage == B200F_STORAGE_F16)
        return a->d > 64 ? launch_attend<__half, 128>(maps, p, pl, st) : launch_attend<__half, 64>(maps, p, pl, st);
    return a->d > 64 ? launch_attend<__nv_bfloat16, 128>(maps, p, pl, st) : launch_attend<__nv_bfloat16, 64>(maps, p, pl, st);
}

extern "C" int32_t* b200f_attention_status(void) {
    static int32_t* const word = []() -> int32_t* {
        // allowed while a stream of this thread is being captured: nothing of the capture depends on it
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        if (cudaThreadExchangeStreamCaptureMode(&mode) != cudaSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, 4 * sizeof(int32_t), cudaHostAllocPortable | cudaHostAllocMapped);
        (void)cudaThreadExchangeStreamCaptureMode(&mode);
        if (e != cudaSuccess) {
            (void)cudaGetLastError();
            return nullptr;
        }
        for (int i = 0; i < 4; i++) static_cast<int32_t*>(p)[i] = 0;
        return static_cast<int32_t*>(p);
    }();
    return word;
}
