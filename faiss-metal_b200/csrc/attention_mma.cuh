// tcgen05 pieces of the soft reads: operand tiles of 128 rows, products with an operand in tensor memory, masks.
#pragma once

#include "attention.cuh"
#include "gemm_common.cuh"

namespace b200f {

constexpr int ATT_TILE = 128;              // keys, or packed query rows, of a tile
constexpr int ATT_CHUNK = ATT_TILE * 128;  // bytes of 64 columns of a tile: a swizzled box of 128-byte rows

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3) {
    asm volatile(
            "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5, %6}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
            : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3,
                                            int c4) {
    asm volatile(
            "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
            " [%0], [%1, {%3, %4, %5, %6, %7}], [%2];"
            ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
            : "memory");
}

// 16 bytes global -> shared, zeros where not `there` (src is not read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

// Shared-memory writes of this thread become visible to TMA and tcgen05.
__device__ __forceinline__ void fence_proxy_async_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void mbar_arrive_if(bool on, uint32_t bar) {
    asm volatile(
            "{\n\t"
            ".reg .pred p;\n\t"
            "setp.ne.b32 p, %1, 0;\n\t"
            "@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t"
            "}\n" ::"r"(bar),
            "r"((uint32_t)on)
            : "memory");
}

// The A operand in tensor memory: 16-bit elements, two a column, row i in lane i.
__device__ __forceinline__ void tc_mma_ts_by(bool leader, uint32_t d_tmem, uint32_t a_tmem, uint64_t desc_b, uint32_t idesc,
                                             uint32_t accumulate) {
    asm volatile(
            "{\n\t"
            ".reg .pred p, q;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "setp.ne.b32 q, %5, 0;\n\t"
            "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
            "}\n" ::"r"(d_tmem),
            "r"(a_tmem), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"((uint32_t)leader)
            : "memory");
}

// 32 registers a thread -> 32 lanes x 32 consecutive columns
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
            "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
            ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
              "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
              "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
              "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
            : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
            "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
            "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
            ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
              "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
            : "memory");
}
// 32 lanes x 16 consecutive columns, complete on return
__device__ __forceinline__ void tc_ld16_wait(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
            "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
            "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
            "tcgen05.wait::ld.sync.aligned;"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
              "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
            : "r"(taddr)
            : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t"
        ".reg .b64 a, b, c, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\t"
        "mov.b64 {%0, %1}, d;\n\t"
        "}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t"
        ".reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "add.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t"
        "}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t"
        ".reg .b64 a, b, d;\n\t"
        "mov.b64 a, {%2, %3};\n\t"
        "mov.b64 b, {%4, %5};\n\t"
        "mul.rn.f32x2 d, a, b;\n\t"
        "mov.b64 {%0, %1}, d;\n\t"
        "}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// 2^y of two values on the FMA pipe: y = n + f with n the nearest integer (Cody and Waite's range reduction, the rounding by adding
// 1.5 * 2^23), 2^f by a polynomial of degree 4 (fitted here to the relative error on [-1/2, 1/2], 2.7e-6 in fp32), n added to the
// exponent.  2^-126 below that, 2^126 above, and something above 2^126 or NaN for NaN.
__device__ __forceinline__ float clamp126(float y) {
    float z;
    asm("{\n\t"
        ".reg .f32 t;\n\t"
        "max.NaN.f32 t, %1, 0fC2FC0000;\n\t"
        "min.NaN.f32 %0, t, 0f42FC0000;\n\t"
        "}\n"
        : "=f"(z)
        : "f"(y));
    return z;
}
__device__ __forceinline__ float2 ex2_fma(float2 y) {
    constexpr float ROUND = 12582912.f;
    y.x = clamp126(y.x);
    y.y = clamp126(y.y);
    const float2 r = add2(y, make_float2(ROUND, ROUND));
    const float2 f = add2(y, fma2(r, make_float2(-1.f, -1.f), make_float2(ROUND, ROUND)));
    float2 z = fma2(f, make_float2(0.009570104735915316f, 0.009570104735915316f), make_float2(0.05591786050289549f, 0.05591786050289549f));
    z = fma2(z, f, make_float2(0.2402474475630491f, 0.2402474475630491f));
    z = fma2(z, f, make_float2(0.6931218146697293f, 0.6931218146697293f));
    z = fma2(z, f, make_float2(0.9999992614616359f, 0.9999992614616359f));
    // the low bits of r are n
    return make_float2(__uint_as_float(__float_as_uint(r.x) * 8388608u + __float_as_uint(z.x)),
                       __uint_as_float(__float_as_uint(r.y) * 8388608u + __float_as_uint(z.y)));
}

// w = exp2((x - from) c + mc) of 32 values, packed; returns their sums.  MIX: from is 0.  In groups of eight, and each step for the whole group before the next:
// the compiler keeps this order, and an exponential's result takes some 40 cycles (a warp alone on its scheduler: 1,090
// cycles for 64 values step by step, 600 this way; the exponential unit takes 512).
// MIX: two of eight by ex2_fma, which takes the load off that unit; -INF gives 2^-126, +INF and NaN a large sum.
template <typename T, bool MIX>
__device__ __forceinline__ float2 weigh32(const uint32_t (&x)[32], float c, float mc, float from, uint32_t* w) {
    const float2 c2 = make_float2(c, c), mc2 = make_float2(mc, mc);
    float2 add[4];
#pragma unroll
    for (int g = 0; g < 16; g += 4) {
        float2 y[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            y[e] = make_float2(__uint_as_float(x[2 * (g + e)]), __uint_as_float(x[2 * (g + e) + 1]));
            if (!MIX) y[e] = add2(y[e], make_float2(-from, -from));
            y[e] = fma2(y[e], c2, mc2);
        }
#pragma unroll
        for (int e = 0; e < (MIX ? 3 : 4); e++) {
            y[e].x = ex2(y[e].x);
            y[e].y = ex2(y[e].y);
        }
        if (MIX) y[3] = ex2_fma(y[3]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            add[e] = g == 0 ? y[e] : add2(add[e], y[e]);
            w[g + e] = pack2<T>(y[e].x, y[e].y);
        }
    }
    return add2(add2(add[0], add[1]), add2(add[2], add[3]));
}

// Descriptor of an operand tile whose rows (128 bytes, swizzled) run along K: 64 elements of M or N a row, 8-row
// groups 1024 bytes apart, the next 64 elements `chunk` bytes further on.  A K step of 16 rows is 2048 bytes.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t saddr, uint32_t chunk) {
    uint64_t desc = 0;
    desc |= (uint64_t)((saddr & 0x3FFFFu) >> 4);
    desc |= (uint64_t)(chunk >> 4) << 16;
    desc |= (uint64_t)(1024 >> 4) << 32;
    desc |= (uint64_t)1 << 46;
    desc |= (uint64_t)2 << 61;
    return desc;
}

// fp32 accumulate, M = 128
template <typename T>
__host__ __device__ constexpr uint32_t att_idesc(int n, bool b_mn_major) {
    const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// D[128][N] = A B^T over DP columns, both operands tiles (of 128 and N rows) in shared memory with K along their rows.
template <typename T, int DP, int N>
__device__ __forceinline__ void mma_rows(bool leader, uint32_t d_tmem, uint32_t a_smem, uint32_t b_smem) {
#pragma unroll
    for (int c = 0; c < DP / 64; c++) {
        const uint64_t da = make_smem_desc(a_smem + c * ATT_CHUNK), db = make_smem_desc(b_smem + c * (N * 128));
#pragma unroll
        for (int k = 0; k < 4; k++)
            tc_mma_f16_by<false>(leader, d_tmem, da + 2 * k, db + 2 * k, att_idesc<T>(N, false), c + k > 0);
    }
}
// The same with A [128][DP] in tensor memory.
template <typename T, int DP, int N>
__device__ __forceinline__ void mma_rows_ts(bool leader, uint32_t d_tmem, uint32_t a_tmem, uint32_t b_smem) {
#pragma unroll
    for (int c = 0; c < DP / 64; c++) {
        const uint64_t db = make_smem_desc(b_smem + c * (N * 128));
#pragma unroll
        for (int k = 0; k < 4; k++)
            tc_mma_ts_by(leader, d_tmem, a_tmem + 32 * c + 8 * k, db + 2 * k, att_idesc<T>(N, false), c + k > 0);
    }
}
// D[128][DP] (+)= P B over the K rows of the tile B; P [128][K] in tensor memory.
template <typename T, int DP, int K>
__device__ __forceinline__ void mma_weights(bool leader, uint32_t d_tmem, uint32_t p_tmem, uint32_t b_smem, bool accumulate) {
    const uint64_t db = make_smem_desc_mn(b_smem, K * 128);
#pragma unroll
    for (int k = 0; k < K / 16; k++)
        tc_mma_ts_by(leader, d_tmem, p_tmem + 8 * k, db + 128 * k, att_idesc<T>(DP, true), accumulate || k > 0);
}

// 32 rows of COLS 16-bit elements that a warp has put into `stage` (row r's 16-byte piece c at piece c ^ (r & 7)) go to global memory
// as whole rows: row r to dst + at, its lane r's `at` (negative: nowhere), d elements of it from column col on.
template <int COLS>
__device__ __forceinline__ void store_rows(const uint8_t* stage, uint16_t* dst, int64_t at, int col, int d) {
    constexpr int PER_ROW = COLS / 8;
    const int lane = threadIdx.x & 31, piece = lane % PER_ROW;
    __syncwarp();
#pragma unroll 4
    for (int r = lane / PER_ROW; r < 32; r += 32 / PER_ROW) {
        const int64_t to = __shfl_sync(0xffffffffu, at, r);
        if (to >= 0 && col + piece * 8 < d)
            *reinterpret_cast<uint4*>(dst + to + col + piece * 8) =
                    *reinterpret_cast<const uint4*>(stage + r * (COLS * 2) + ((piece ^ (r & (PER_ROW < 8 ? PER_ROW - 1 : 7))) << 4));
    }
    __syncwarp();
}
// 32 of a lane's columns, from piece c0 on, to that stage
template <typename T, int COLS>
__device__ __forceinline__ void stage_columns32(uint8_t* stage, const uint32_t (&o)[32], int c0) {
    constexpr int PER_ROW = COLS / 8;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < 4; e++)
        *reinterpret_cast<uint4*>(stage + lane * (COLS * 2) + (((c0 + e) ^ (lane & (PER_ROW < 8 ? PER_ROW - 1 : 7))) << 4)) =
                make_uint4(pack2<T>(__uint_as_float(o[8 * e]), __uint_as_float(o[8 * e + 1])),
                           pack2<T>(__uint_as_float(o[8 * e + 2]), __uint_as_float(o[8 * e + 3])),
                           pack2<T>(__uint_as_float(o[8 * e + 4]), __uint_as_float(o[8 * e + 5])),
                           pack2<T>(__uint_as_float(o[8 * e + 6]), __uint_as_float(o[8 * e + 7])));
}

// Rows [first, rows) of a tile in shared memory become zero; a warp calls it.
__device__ __forceinline__ void zero_tile_rows(uint8_t* tile, int chunks, int first, int rows) {
    const int lane = threadIdx.x & 31;
    for (int c = 0; c < chunks; c++)
        for (int i = first * 8 + lane; i < rows * 8; i += 32)
            *reinterpret_cast<uint4*>(tile + c * rows * 128 + i * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_shared();
    __syncwarp();
}

// ---- host side -------------------------------------------------------------------------

// Coordinates of a repeated sequence or head stay 0.
struct AttMap {
    int batch_step, head_step;
};

// 4-D map {column, row, head, sequence} of keys or values, box {64, box_rows, 1, 1}; columns and rows beyond the end read 0.
inline int make_rows_map(CUtensorMap* map, AttMap* am, const AttView& v, int storage, int d, int64_t rows, int64_t heads, int64_t batch,
                         int box_rows = ATT_TILE) {
    EncodeTiledFn fn = get_encode_fn();
    if (!fn) return B200F_ERR_CUDA;
    am->batch_step = batch > 1 && v.sb == 0 ? 0 : 1;
    am->head_step = heads > 1 && v.sh == 0 ? 0 : 1;
    const int64_t nh = am->head_step ? heads : 1, nb = am->batch_step ? batch : 1;
    cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)rows, (cuuint64_t)nh, (cuuint64_t)nb};
    // strides of dimensions of one element are not used, but checked
    cuuint64_t strides[3] = {(cuuint64_t)(rows > 1 ? v.sr * 2 : 256), (cuuint64_t)(nh > 1 ? v.sh * 2 : 256),
                             (cuuint64_t)(nb > 1 ? v.sb * 2 : 256)};
    cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, storage == B200F_STORAGE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                          const_cast<uint16_t*>(v.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? B200F_OK : B200F_ERR_CUDA;
}

// How the query rows of a key head are packed into tiles that TMA fetches: `bt` queries of `gb` heads a tile, the group in
// `gchunks` pieces.  Slot s of tile i is query (i / gchunks) * bt + s / gb, head (i % gchunks) * gb + s % gb of the group.
struct RowTiles {
    int slots, gb, bt, gchunks, group;
    int queries, tiles;   // batch * queries * heads is below 2^31
    __host__ __device__ bool at(int tile, int slot, int* t, int* g) const {
        const int q = (int)((unsigned)slot / (unsigned)gb), block = (int)((unsigned)tile / (unsigned)gchunks);
        *t = block * bt + q;
        *g = (tile - block * gchunks) * gb + (slot - q * gb);
        return q < bt && *t < queries && *g < group;
    }
    __host__ __device__ int64_t place(int t, int g) const {   // tile * slots + slot
        return ((int64_t)(t / bt) * gchunks + g / gb) * slots + t % bt * gb + g % gb;
    }
};
inline RowTiles row_tiles(int slots, int64_t queries, int group) {
    RowTiles r;
    r.slots = slots;
    r.group = group;
    r.queries = (int)queries;
    r.gb = group < slots ? group : slots;
    r.bt = slots / r.gb;
    if (r.bt > queries) r.bt = queries > 0 ? (int)queries : 1;
    r.gchunks = (group + r.gb - 1) / r.gb;
    r.tiles = (int)(ceil_div64(queries, r.bt) * r.gchunks);
    return r;
}
// 5-D map {column, head of the group, query, key head, sequence} of queries, box {64, gb, bt, 1, 1}.  Heads of a group do not repeat.
inline int make_queries_map(CUtensorMap* map, AttMap* am, const AttView& v, int storage, int d, const RowTiles& rt, int kv_heads,
                            int64_t batch) {
    EncodeTiledFn fn = get_encode_fn();
    if (!fn) return B200F_ERR_CUDA;
    if (rt.group > 1 && v.sh == 0) return B200F_ERR_BAD_ARG;
    am->batch_step = batch > 1 && v.sb == 0 ? 0 : 1;
    am->head_step = kv_heads > 1 && v.sh == 0 ? 0 : 1;
    const int64_t nh = am->head_step ? kv_heads : 1, nb = am->batch_step ? batch : 1;
    cuuint64_t dims[5] = {(cuuint64_t)d, (cuuint64_t)rt.group, (cuuint64_t)rt.queries, (cuuint64_t)nh, (cuuint64_t)nb};
    cuuint64_t strides[4] = {(cuuint64_t)(rt.group > 1 ? v.sh * 2 : 256), (cuuint64_t)(rt.queries > 1 ? v.sr * 2 : 256),
                             (cuuint64_t)(nh > 1 ? v.sh * rt.group * 2 : 256), (cuuint64_t)(nb > 1 ? v.sb * 2 : 256)};
    cuuint32_t box[5] = {64, (cuuint32_t)rt.gb, (cuuint32_t)rt.bt, 1, 1};
    cuuint32_t estr[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, storage == B200F_STORAGE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                          const_cast<uint16_t*>(v.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? B200F_OK : B200F_ERR_CUDA;
}

}  // namespace b200f
