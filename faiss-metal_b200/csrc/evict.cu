// Eviction from a cache by accumulated attention weight: which rows stay (evict_select_kernel), and their move
// (evict_move_kernel).
#include "attention.cuh"
#include "ptx.cuh"

namespace b200f {

namespace {

// Weights order as in a sort from the largest: NaN first, -0 as 0.
__device__ __forceinline__ uint32_t mass_key(float f) { return f != f ? 0xffffffffu : float_to_ordered(f + 0.f); }

constexpr int SEL_THREADS = 1024;
constexpr int SEL_SMEM_KEYS = 45 * 1024;   // weights of a row held in shared memory; longer rows are read again (L2)
constexpr int SEL_BINS = 2048;             // a digit: 11, 11 and 10 bits from the top
constexpr int SEL_COPIES = 2;              // histograms, for every second warp one: weights crowd into few of the first digit's bins

// Exclusive prefix sums of (a, b) over the CTA.  All threads call it; warps is free again after the next barrier.
__device__ __forceinline__ void block_scan2(uint32_t& a, uint32_t& b, uint2* warps) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t a0 = a, b0 = b;
    auto scan = [&](uint32_t& x, uint32_t& y) {   // inclusive, over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t ux = __shfl_up_sync(0xffffffffu, x, o), uy = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) {
                x += ux;
                y += uy;
            }
        }
    };
    scan(a, b);
    if (lane == 31) warps[warp] = make_uint2(a, b);
    __syncthreads();
    uint2 w = warps[lane];   // SEL_THREADS / 32 == 32 warps
    const uint2 own = w;
    scan(w.x, w.y);
    a += __shfl_sync(0xffffffffu, w.x - own.x, warp) - a0;
    b += __shfl_sync(0xffffffffu, w.y - own.y, warp) - b0;
}

// One CTA a (sequence, key head).  The keep - recent largest of the first n - recent weights are those above a threshold, which three
// histograms of digits find from the top, and of those equal to it the lowest rows; a scan in row order gives the kept rows
// their slots.
__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const float* mass, AttLengths len, int kv_heads, int64_t keep,
                                                                   int64_t recent, float* out_mass, int32_t* out_rows,
                                                                   int32_t* out_lengths) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[SEL_COPIES][SEL_BINS], pick[2];
    __shared__ uint2 warps[32];
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x, b = bh / kv_heads;
    const int64_t n = len.of(b);
    const float* const m = mass + bh * len.n;
    int32_t* const rows = out_rows + bh * keep;
    float* const om = out_mass + bh * keep;
    const int64_t kept = min(n, keep);
    if (tid == 0 && bh % kv_heads == 0) out_lengths[b] = (int32_t)kept;
    for (int64_t i = kept + tid; i < keep; i += SEL_THREADS) {
        rows[i] = -1;
        om[i] = 0.f;
    }
    if (n <= keep) {
        for (int64_t i = tid; i < n; i += SEL_THREADS) {
            rows[i] = (int32_t)i;
            om[i] = m[i];
        }
        return;
    }
    const int64_t old = n - recent;          // rows that compete, for keep - recent slots
    const uint32_t want = (uint32_t)(keep - recent);
    for (int64_t i = tid; i < recent; i += SEL_THREADS) {
        rows[want + i] = (int32_t)(old + i);
        om[want + i] = m[old + i];
    }
    if (want == 0) return;
    const bool staged = old <= SEL_SMEM_KEYS;
    if (staged) {
#pragma unroll 8
        for (int i = tid; i < (int)old; i += SEL_THREADS) keys[i] = mass_key(m[i]);
    }
    auto key = [&](int64_t i) { return staged ? keys[i] : mass_key(m[i]); };
    uint32_t prefix = 0, need = want;   // the threshold's digits so far; slots left for keys that share them
#pragma unroll 1
    for (int digit = 0; digit < 3; digit++) {
        const int shift = digit == 0 ? 21 : digit == 1 ? 10 : 0, bits = digit == 2 ? 10 : 11;
        for (int i = tid; i < SEL_COPIES * SEL_BINS; i += SEL_THREADS) hist[0][i] = 0;
        __syncthreads();
        uint32_t* const mine = hist[(tid >> 5) % SEL_COPIES];
#pragma unroll 4
        for (int64_t i = tid; i < old; i += SEL_THREADS) {
            const uint32_t k = key(i);
            if (digit == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&mine[(k >> shift) & ((1u << bits) - 1u)], 1u);
        }
        __syncthreads();
        // two bins a thread, from the largest
        uint32_t own[2], sum = 0, none = 0;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int bin = SEL_BINS - 1 - (2 * tid + i);
            own[i] = 0;
#pragma unroll
            for (int x = 0; x < SEL_COPIES; x++) own[i] += hist[x][bin];
            sum += own[i];
        }
        uint32_t before = sum;
        block_scan2(before, none, warps);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (before < need && need <= before + own[i]) {
                pick[0] = SEL_BINS - 1 - (2 * tid + i);
                pick[1] = need - before;
            }
            before += own[i];
        }
        __syncthreads();
        prefix = (prefix << bits) | pick[0];
        need = pick[1];
    }
    // kept: key > prefix, and the first `need` equal to it.  A thread takes consecutive rows.
    const int64_t per = (old + SEL_THREADS - 1) / SEL_THREADS;
    const int64_t i0 = min(old, tid * per), i1 = min(old, i0 + per);
    uint32_t above = 0, equal = 0;
    for (int64_t i = i0; i < i1; i++) {
        const uint32_t k = key(i);
        above += k > prefix;
        equal += k == prefix;
    }
    block_scan2(above, equal, warps);
    for (int64_t i = i0; i < i1; i++) {
        const uint32_t k = key(i);
        if (k > prefix || (k == prefix && equal < need)) {
            const uint32_t at = above + min(equal, need);
            rows[at] = (int32_t)i;
            om[at] = staged ? ordered_to_float(k) : m[i];   // -0 as 0
        }
        above += k > prefix;
        equal += k == prefix;
    }
}

// Slot s of (b, h) receives row rows[b][h][s] of keys and values, zero where that is -1: 16 bytes of each a thread, two slots at once.
// Bound by HBM (bf16, d = 128, 16 sequences of 8 key heads to 2,048 rows: 41 us, as long as a copy of these bytes).
constexpr int MOVE_THREADS = 256;
__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(AttView k, AttView v, const int32_t* rows, int kv_heads, int keep, int vecs,
                                                                  int64_t slots, uint4* out_k, uint4* out_v) {
    pdl_wait();
    pdl_trigger();
    const int at_once = MOVE_THREADS / vecs, sub = threadIdx.x / vecs, c = threadIdx.x - sub * vecs;
    if (sub >= at_once) return;
    const int64_t step = (int64_t)gridDim.x * at_once;
    for (int64_t s0 = (int64_t)blockIdx.x * at_once + sub; s0 < slots; s0 += 2 * step) {
        uint4 x[2], y[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int64_t s = s0 + i * step;
            x[i] = y[i] = make_uint4(0, 0, 0, 0);
            if (s < slots) {
                int64_t bs, b;
                if (slots < (int64_t)1 << 31) {
                    bs = (uint32_t)s / (uint32_t)kv_heads;
                    b = (uint32_t)bs / (uint32_t)keep;
                } else {
                    bs = s / kv_heads;
                    b = bs / keep;
                }
                const int h = (int)(s - bs * kv_heads);
                const int32_t row = __ldcg(rows + (b * kv_heads + h) * keep + (bs - b * keep));
                if (row >= 0) {
                    x[i] = __ldg(reinterpret_cast<const uint4*>(k.at(b, row, h)) + c);
                    y[i] = __ldg(reinterpret_cast<const uint4*>(v.at(b, row, h)) + c);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
            if (s0 + i * step < slots) {
                out_k[(s0 + i * step) * vecs + c] = x[i];
                out_v[(s0 + i * step) * vecs + c] = y[i];
            }
    }
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" int b200f_evict(const B200FEvictArgs* a) {
    if (!a || (a->storage != B200F_STORAGE_F16 && a->storage != B200F_STORAGE_BF16) || a->batch < 0 || a->n < 0 || a->kv_heads <= 0 ||
        a->d <= 0 || a->d % 8 != 0 || a->d > 8 * 128 || a->keep < 1 || a->recent < 0 || a->recent > a->keep)
        return B200F_ERR_BAD_ARG;
    const int64_t lim = ((int64_t)1 << 31) - 1;
    if (a->n > lim || a->keep > lim || a->batch > lim / a->kv_heads) return B200F_ERR_UNSUPPORTED;
    if (a->batch == 0) return B200F_OK;
    const AttView k = att_view(a->k, a->k_stride), v = att_view(a->v, a->v_stride);
    if (!a->out_k || !a->out_v || !a->out_mass || !a->out_rows || !a->out_lengths || (reinterpret_cast<uintptr_t>(a->out_k) & 15) != 0 ||
        (reinterpret_cast<uintptr_t>(a->out_v) & 15) != 0 ||
        (a->n > 0 && (!a->mass || !att_view_ok(k, a->batch, a->n, a->kv_heads) || !att_view_ok(v, a->batch, a->n, a->kv_heads))))
        return B200F_ERR_BAD_ARG;
    const cudaStream_t st = (cudaStream_t)a->stream;
    const AttLengths len{a->key_lengths, a->n, 0, 0};
    static bool attr_set[kMaxDevices] = {false};
    const int slot = device_slot();
    if (!attr_set[slot]) {
        B200F_CUDA_TRY(cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SEL_SMEM_KEYS * 4));
        attr_set[slot] = true;
    }
    const size_t smem = (size_t)(a->n < SEL_SMEM_KEYS ? a->n : SEL_SMEM_KEYS) * 4;
    evict_select_kernel<<<(unsigned)(a->batch * a->kv_heads), SEL_THREADS, smem, st>>>(a->mass, len, a->kv_heads, a->keep, a->recent,
                                                                                      a->out_mass, a->out_rows, a->out_lengths);
    count_launch();
    B200F_LAUNCH_CHECK();
    const int64_t slots = a->batch * a->keep * a->kv_heads;
    const int vecs = a->d / 8, at_once = MOVE_THREADS / vecs;
    const int64_t want = ceil_div64(slots, (int64_t)at_once * 2), most = (int64_t)cached_sm_count() * 16;
    const cudaError_t e = launch_kernel(evict_move_kernel, dim3((unsigned)(want < most ? want : most)), MOVE_THREADS, 0, Launch(st, true), k, v,
                                        static_cast<const int32_t*>(a->out_rows), a->kv_heads, (int)a->keep, vecs, slots,
                                        static_cast<uint4*>(a->out_k), static_cast<uint4*>(a->out_v));
    if (e != cudaSuccess) {
        (void)cudaGetLastError();
        return B200F_ERR_CUDA;
    }
    count_launch();
    return B200F_OK;
}
