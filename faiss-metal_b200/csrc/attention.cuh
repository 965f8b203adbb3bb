// What the soft reads share: operand views, argument checks.
#pragma once

#include "common.cuh"

namespace b200f {

constexpr int ATT_MAX_D = 128;
constexpr int ATT_MAX_GROUP = 128;   // query heads a key head
constexpr float ATT_MAX_SCALE = 2e38f;   // scale * log2(e) is finite
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// [batch][row][head][d] with strides in elements; the last dimension is dense.
struct AttView {
    const uint16_t* p;
    int64_t sb, sr, sh;
    __host__ __device__ const uint16_t* at(int64_t b, int64_t r, int64_t h) const { return p + b * sb + r * sr + h * sh; }
};

inline AttView att_view(const void* p, const int64_t (&s)[3]) {
    return AttView{static_cast<const uint16_t*>(p), s[0], s[1], s[2]};
}

// 16-byte vectors and tensor maps want aligned bases and strides.  Strides of dimensions of one element do not matter.
inline bool att_view_ok(const AttView& v, int64_t batch, int64_t rows, int64_t heads) {
    if (!v.p || (reinterpret_cast<uintptr_t>(v.p) & 15) != 0) return false;
    auto bad = [](int64_t s, int64_t n) { return n > 1 && (s < 0 || s % 8 != 0 || s >= (int64_t)1 << 38); };
    return !bad(v.sb, batch) && !bad(v.sr, rows) && !bad(v.sh, heads) && !(rows > 1 && v.sr == 0);
}

// What all soft reads want of their sizes.
inline int att_sizes_ok(int64_t batch, int64_t queries, int64_t n, int heads, int kv_heads, int d, int storage, float scale) {
    if (storage != B200F_STORAGE_F16 && storage != B200F_STORAGE_BF16) return B200F_ERR_BAD_ARG;
    if (batch < 0 || queries < 0 || n < 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 ||
        heads / kv_heads > ATT_MAX_GROUP || d < 8 || d > ATT_MAX_D || d % 8 != 0 || !(scale > 0.f) || scale > ATT_MAX_SCALE)
        return B200F_ERR_BAD_ARG;
    const int64_t lim = ((int64_t)1 << 31) - 1;
    if (n > lim - 1024 || batch > lim || queries > lim || kv_heads > 65535 || (batch > 0 && queries > lim / batch) ||
        (batch * queries > 0 && heads > lim / (batch * queries)) || (n > 0 && batch * kv_heads > lim))
        return B200F_ERR_UNSUPPORTED;
    return B200F_OK;
}

template <typename T>
__device__ __forceinline__ float to_f32(uint16_t u);
template <>
__device__ __forceinline__ float to_f32<__half>(uint16_t u) { return __half2float(__ushort_as_half(u)); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(uint16_t u) { return __bfloat162float(__ushort_as_bfloat16(u)); }
// Keys that query t of sequence b sees: its length, clamped, and the causal end.
struct AttLengths {
    const int32_t* lengths;   // null: all n
    int64_t n, queries;
    int causal;
    __device__ __forceinline__ int64_t of(int64_t b) const {
        return lengths ? min(max((int64_t)__ldg(lengths + b), (int64_t)0), n) : n;
    }
    __device__ __forceinline__ int64_t seen(int64_t len, int64_t t) const {
        return causal ? max(len - queries + 1 + t, (int64_t)0) : len;
    }
};

}  // namespace b200f
