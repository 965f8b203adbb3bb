// Eviction from a cache by accumulated attention weight: which rows stay (evict_select_kernel), and their move
// (evict_move_kernel).
#include "attention.cuh"

namespace b200f {

namespace {

// Weights order as in a sort from the largest: NaN first, -0 as 0.
__device__ __forceinline__ uint32_t mass_key(float f) { return f != f ? 0xffffffffu : float_to_ordered(f + 0.f); }

constexpr int SEL_THREADS = 1024;
constexpr int SEL_SMEM_KEYS = 48 * 1024;   // weights of a row held in shared memory; longer rows are read again (L2)

// Exclusive prefix sums of (a, b) over the CTA; *ta receives the sum of a.  All threads call it.
__device__ __forceinline__ void block_scan2(uint32_t& a, uint32_t& b, uint32_t* warps, uint32_t* ta) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t ua = __shfl_up_sync(0xffffffffu, a, o), ub = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) {
            a += ua;
            b += ub;
        }
    }
    if (lane == 31) {
        warps[warp] = a;
        warps[32 + warp] = b;
    }
    __syncthreads();
    uint32_t pa = 0, pb = 0, total = 0;
    for (int w = 0; w < SEL_THREADS / 32; w++) {
        if (w < warp) {
            pa += warps[w];
            pb += warps[32 + w];
        }
        total += warps[w];
    }
    __syncthreads();
    a += pa - a0;
    b += pb - b0;
    *ta = total;
}

// One CTA a (sequence, key head).  The keep - recent largest of the first n - recent weights are those above the T-th
// digit string, found by four 8-bit digits from the top, and of those equal to it the lowest rows; a scan in
// row order gives the kept rows their slots.
__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const float* mass, AttLengths len, int kv_heads, int64_t keep,
                                                                   int64_t recent, float* out_mass, int32_t* out_rows,
                                                                   int32_t* out_lengths) {
    extern __shared__ uint32_t keys[];
    __shared__ uint32_t hist[256], warps[64], pick[2];
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
    if (staged)
        for (int64_t i = tid; i < old; i += SEL_THREADS) keys[i] = mass_key(m[i]);
    auto key = [&](int64_t i) { return staged ? keys[i] : mass_key(m[i]); };
    uint32_t prefix = 0, need = want;   // the threshold's digits so far; slots left for keys that share them
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int64_t i = tid; i < old; i += SEL_THREADS) {
            const uint32_t k = key(i);
            if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1u);
        }
        __syncthreads();
        if (tid < 32) {   // eight digits a lane, from the largest
            uint32_t own[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; i++) sum += own[i] = hist[255 - (tid * 8 + i)];
            uint32_t incl = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t u = __shfl_up_sync(0xffffffffu, incl, o);
                if (tid >= o) incl += u;
            }
            uint32_t before = incl - sum;
            if (before < need && need <= incl) {
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    if (before < need && need <= before + own[i]) {
                        pick[0] = 255 - (tid * 8 + i);
                        pick[1] = need - before;
                    }
                    before += own[i];
                }
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | pick[0];
        need = pick[1];
    }
    // kept: key > prefix, and the first `need` equal to it.  A thread takes consecutive rows.
    const int64_t per = (old + SEL_THREADS - 1) / SEL_THREADS;
    const int64_t i0 = min(old, tid * per), i1 = min(old, i0 + per);
    uint32_t above = 0, equal = 0, total;
    for (int64_t i = i0; i < i1; i++) {
        const uint32_t k = key(i);
        above += k > prefix;
        equal += k == prefix;
    }
    block_scan2(above, equal, warps, &total);
    for (int64_t i = i0; i < i1; i++) {
        const uint32_t k = key(i);
        if (k > prefix || (k == prefix && equal < need)) {
            const uint32_t at = above + min(equal, need);
            rows[at] = (int32_t)i;
            om[at] = m[i];
        }
        above += k > prefix;
        equal += k == prefix;
    }
}

// 16 bytes a thread and array: slot i of (b, h) receives row rows[b][h][i], zero where that is -1.
__global__ void __launch_bounds__(256) evict_move_kernel(AttView k, AttView v, const int32_t* rows, int kv_heads, int64_t keep, int vecs,
                                                         int64_t total, uint4* out_k, uint4* out_v) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
        const int c = (int)(i % vecs);
        const int64_t slot = i / vecs;
        const int h = (int)(slot % kv_heads);
        const int64_t s = slot / kv_heads % keep, b = slot / kv_heads / keep;
        const int32_t row = rows[(b * kv_heads + h) * keep + s];
        uint4 x = make_uint4(0, 0, 0, 0), y = x;
        if (row >= 0) {
            x = *reinterpret_cast<const uint4*>(k.at(b, row, h) + c * 8);
            y = *reinterpret_cast<const uint4*>(v.at(b, row, h) + c * 8);
        }
        out_k[i] = x;
        out_v[i] = y;
    }
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" int b200f_evict(const B200FEvictArgs* a) {
    if (!a || (a->storage != B200F_STORAGE_F16 && a->storage != B200F_STORAGE_BF16) || a->batch < 0 || a->n < 0 || a->kv_heads <= 0 ||
        a->d <= 0 || a->d % 8 != 0 || a->keep < 1 || a->recent < 0 || a->recent > a->keep)
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
    const int vecs = a->d / 8;
    const int64_t total = a->batch * a->keep * a->kv_heads * vecs;
    const int64_t want = ceil_div64(total, 256), most = (int64_t)cached_sm_count() * 8;
    evict_move_kernel<<<(unsigned)(want < most ? want : most), 256, 0, st>>>(k, v, a->out_rows, a->kv_heads, a->keep, vecs, total,
                                                                           static_cast<uint4*>(a->out_k), static_cast<uint4*>(a->out_v));
    count_launch();
    B200F_LAUNCH_CHECK();
    return B200F_OK;
}
