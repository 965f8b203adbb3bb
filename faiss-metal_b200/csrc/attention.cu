// Accumulated weights: a CTA a key, dot products by warp shuffles.
#include "attention.cuh"

#include <math.h>

namespace b200f {

namespace {

constexpr int WARPS = 4;
constexpr int LD = ATT_MAX_D / 32;   // elements a lane holds: lane + 32 i

template <typename T>
__device__ __forceinline__ void load_row(const uint16_t* p, int d, int lane, float (&x)[LD]) {
#pragma unroll
    for (int i = 0; i < LD; i++) x[i] = lane + 32 * i < d ? to_f32<T>(p[lane + 32 * i]) : 0.f;
}
__device__ __forceinline__ float dot(const float (&a)[LD], const float (&b)[LD]) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < LD; i++) s = fmaf(a[i], b[i], s);
    return warp_sum(s);
}

struct Dims {
    int64_t batch, queries;
    int heads, group, d;
    float scale;
};

// The accumulated weight of one key.
template <typename T>
__global__ void mass_kernel(AttView q, AttView k, AttLengths len, Dims dm, const float* lse, const float* mass_in, float* mass_out) {
    __shared__ float part[WARPS];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = dm.heads / dm.group;
    const int64_t j = blockIdx.x % len.n, bh = blockIdx.x / len.n;
    const int hk = (int)(bh % kvh);
    const int64_t b = bh / kvh, n = len.of(b);
    float y[LD], x[LD], w = 0.f;
    load_row<T>(k.at(b, j, hk), dm.d, lane, y);
    for (int64_t r = warp; r < dm.queries * dm.group; r += WARPS) {
        const int64_t t = r / dm.group;
        const int h = hk * dm.group + (int)(r % dm.group);
        if (j >= len.seen(n, t)) continue;
        load_row<T>(q.at(b, t, h), dm.d, lane, x);
        const float ls = lse[(b * dm.queries + t) * dm.heads + h];
        w += ls == -CUDART_INF_F ? 0.f : expf(dot(x, y) * dm.scale - ls);
    }
    if (lane == 0) part[warp] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
        float s = mass_in ? mass_in[bh * len.n + j] : 0.f;
        for (int i = 0; i < WARPS; i++) s += part[i];
        mass_out[bh * len.n + j] = s;
    }
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" size_t b200f_attention_mass_scratch_bytes(const B200FAttentionMassArgs* a) {
    if (!a || att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale) != B200F_OK) return 0;
    return 256;
}

extern "C" int b200f_attention_mass(const B200FAttentionMassArgs* a) {
    if (!a) return B200F_ERR_BAD_ARG;
    const int rc = att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale);
    if (rc != B200F_OK) return rc;
    if (a->batch == 0 || a->n == 0) return B200F_OK;
    const AttView q = att_view(a->q, a->q_stride), k = att_view(a->k, a->k_stride);
    if (!a->status || !a->mass_out || !att_view_ok(k, a->batch, a->n, a->kv_heads) ||
        (a->queries > 0 && (!att_view_ok(q, a->batch, a->queries, a->heads) || !a->lse)))
        return B200F_ERR_BAD_ARG;
    const Dims dm{a->batch, a->queries, a->heads, a->heads / a->kv_heads, a->d, a->scale};
    const AttLengths len{a->key_lengths, a->n, a->queries, a->causal};
    (a->storage == B200F_STORAGE_F16 ? mass_kernel<__half> : mass_kernel<__nv_bfloat16>)
            <<<(unsigned)(a->batch * a->n * a->kv_heads), 32 * WARPS, 0, (cudaStream_t)a->stream>>>(q, k, len, dm, a->lse, a->mass_in,
                                                                                                   a->mass_out);
    count_launch();
    B200F_LAUNCH_CHECK();
    return B200F_OK;
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
