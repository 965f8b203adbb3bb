// Gradient of attention and accumulated weights: a CTA a row or a key, dot products by warp shuffles.
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

template <typename T>
__global__ void grad_q_kernel(AttView g, AttView q, AttView k, AttView v, AttLengths len, Dims dm, const uint16_t* out,
                              const float* lse, float* delta, uint16_t* grad_q) {
    __shared__ float part[WARPS][ATT_MAX_D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = blockIdx.x;
    const int h = (int)(row % dm.heads);
    const int64_t t = row / dm.heads % dm.queries, b = row / dm.heads / dm.queries;
    float x[LD], go[LD], y[LD], z[LD], acc[LD] = {};
    load_row<T>(q.at(b, t, h), dm.d, lane, x);
    load_row<T>(g.at(b, t, h), dm.d, lane, go);
    load_row<T>(out + row * dm.d, dm.d, lane, y);
    const float dl = dot(go, y), ls = lse[row];
    if (threadIdx.x == 0) delta[row] = dl;
    const int64_t end = len.n ? len.of(b) : 0;
    for (int64_t j = warp; j < end; j += WARPS) {
        load_row<T>(k.at(b, j, h / dm.group), dm.d, lane, y);
        load_row<T>(v.at(b, j, h / dm.group), dm.d, lane, z);
        const float p = expf(dot(x, y) * dm.scale - ls), ds = p * (dot(go, z) - dl) * dm.scale;
#pragma unroll
        for (int i = 0; i < LD; i++) acc[i] = fmaf(ds, y[i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < LD; i++) part[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float s = 0.f;
    for (int w = 0; w < WARPS; w++) s += part[w][threadIdx.x];
    if ((int)threadIdx.x < dm.d) grad_q[row * dm.d + threadIdx.x] = from_f32<T>(s);
}

// GRADS: grad_k and grad_v of one key; else its accumulated weight.
template <typename T, bool GRADS>
__global__ void key_kernel(AttView g, AttView q, AttView k, AttView v, AttLengths len, Dims dm, const float* lse,
                           const float* delta, uint16_t* grad_k, uint16_t* grad_v, const float* mass_in, float* mass_out) {
    __shared__ float part[WARPS][2 * ATT_MAX_D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = dm.heads / dm.group;
    const int64_t j = blockIdx.x % len.n, bh = blockIdx.x / len.n;
    const int hk = (int)(bh % kvh);
    const int64_t b = bh / kvh, n = len.of(b);
    float y[LD], z[LD], x[LD], go[LD], dk[LD] = {}, dv[LD] = {}, w = 0.f;
    load_row<T>(k.at(b, j, hk), dm.d, lane, y);
    if (GRADS) load_row<T>(v.at(b, j, hk), dm.d, lane, z);
    for (int64_t r = warp; r < dm.queries * dm.group; r += WARPS) {
        const int64_t t = r / dm.group;
        const int h = hk * dm.group + (int)(r % dm.group);
        if (j >= len.seen(n, t)) continue;
        const int64_t row = (b * dm.queries + t) * dm.heads + h;
        load_row<T>(q.at(b, t, h), dm.d, lane, x);
        const float ls = lse[row];
        const float p = ls == -CUDART_INF_F ? 0.f : expf(dot(x, y) * dm.scale - ls);
        w += p;
        if (!GRADS) continue;
        load_row<T>(g.at(b, t, h), dm.d, lane, go);
        const float ds = p * (dot(go, z) - delta[row]) * dm.scale;
#pragma unroll
        for (int i = 0; i < LD; i++) {
            dk[i] = fmaf(ds, x[i], dk[i]);
            dv[i] = fmaf(p, go[i], dv[i]);
        }
    }
    if constexpr (!GRADS) {
        if (lane == 0) part[warp][0] = w;
        __syncthreads();
        if (threadIdx.x == 0) {
            float s = mass_in ? mass_in[bh * len.n + j] : 0.f;
            for (int i = 0; i < WARPS; i++) s += part[i][0];
            mass_out[bh * len.n + j] = s;
        }
    } else {
#pragma unroll
    for (int i = 0; i < LD; i++) {
        part[warp][lane + 32 * i] = dk[i];
        part[warp][ATT_MAX_D + lane + 32 * i] = dv[i];
    }
    __syncthreads();
    float sk = 0.f, sv = 0.f;
    for (int i = 0; i < WARPS; i++) {
        sk += part[i][threadIdx.x];
        sv += part[i][ATT_MAX_D + threadIdx.x];
    }
    if ((int)threadIdx.x < dm.d) {
        const int64_t o = ((b * len.n + j) * kvh + hk) * dm.d + threadIdx.x;
        grad_k[o] = from_f32<T>(sk);
        grad_v[o] = from_f32<T>(sv);
    }
    }
}

}  // namespace

}  // namespace b200f

using namespace b200f;

extern "C" size_t b200f_attend_backward_scratch_bytes(const B200FAttendBackwardArgs* a) {
    if (!a || att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale) != B200F_OK) return 0;
    return (size_t)round_up64(a->batch * a->queries * a->heads * 4 + 1, 256);
}

extern "C" int b200f_attend_backward(const B200FAttendBackwardArgs* a) {
    if (!a) return B200F_ERR_BAD_ARG;
    const int rc = att_sizes_ok(a->batch, a->queries, a->n, a->heads, a->kv_heads, a->d, a->storage, a->scale);
    if (rc != B200F_OK) return rc;
    if (a->batch == 0) return B200F_OK;
    const AttView g = att_view(a->grad_out, a->grad_out_stride), q = att_view(a->q, a->q_stride);
    const AttView k = att_view(a->k, a->k_stride), v = att_view(a->v, a->v_stride);
    if (!a->status || (a->queries > 0 && (!att_view_ok(g, a->batch, a->queries, a->heads) || !att_view_ok(q, a->batch, a->queries, a->heads) ||
                                          !a->out || !a->lse || !a->grad_q)) ||
        (a->n > 0 && (!att_view_ok(k, a->batch, a->n, a->kv_heads) || !att_view_ok(v, a->batch, a->n, a->kv_heads) || !a->grad_k || !a->grad_v)))
        return B200F_ERR_BAD_ARG;
    if (!a->scratch || a->scratch_bytes < b200f_attend_backward_scratch_bytes(a)) return B200F_ERR_SCRATCH;
    const Dims dm{a->batch, a->queries, a->heads, a->heads / a->kv_heads, a->d, a->scale};
    const AttLengths len{a->key_lengths, a->n, a->queries, 0};
    float* const delta = static_cast<float*>(a->scratch);
    const bool half = a->storage == B200F_STORAGE_F16;
    if (a->queries > 0) {
        (half ? grad_q_kernel<__half> : grad_q_kernel<__nv_bfloat16>)<<<(unsigned)(a->batch * a->queries * a->heads), 32 * WARPS, 0,
                                                                        (cudaStream_t)a->stream>>>(
                g, q, k, v, len, dm, static_cast<const uint16_t*>(a->out), a->lse, delta, static_cast<uint16_t*>(a->grad_q));
        count_launch();
        B200F_LAUNCH_CHECK();
    }
    if (a->n > 0) {
        (half ? key_kernel<__half, true> : key_kernel<__nv_bfloat16, true>)<<<(unsigned)(a->batch * a->n * a->kv_heads), 32 * WARPS, 0,
                                                                              (cudaStream_t)a->stream>>>(
                g, q, k, v, len, dm, a->lse, delta, static_cast<uint16_t*>(a->grad_k), static_cast<uint16_t*>(a->grad_v), nullptr,
                nullptr);
        count_launch();
        B200F_LAUNCH_CHECK();
    }
    return B200F_OK;
}

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
    (a->storage == B200F_STORAGE_F16 ? key_kernel<__half, false> : key_kernel<__nv_bfloat16, false>)
            <<<(unsigned)(a->batch * a->n * a->kv_heads), 32 * WARPS, 0, (cudaStream_t)a->stream>>>(
                    AttView{}, q, k, AttView{}, len, dm, a->lse, nullptr, nullptr, nullptr, a->mass_in, a->mass_out);
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
