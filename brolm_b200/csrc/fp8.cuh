// Rows of 8-bit floating point numbers with a scale for every 128 numbers of a row, as the fp8 kernels keep them.
//
// A number is e4m3 (largest 448) times 2^(s - 127), s being the byte of its block: the least from 0 on under which none of
// the block's numbers is beyond 448 * 2^(s - 127).  A power of two because x * 2^(127 - s) is then exact, so that a number is
// rounded once and the same wherever it is rounded, and because tcgen05.mma takes such scales itself (kind::mxf8f6f4: an
// exponent for every 32 numbers along K; a block of 128 is four of them with one exponent).  A block with a number that is
// not finite has the byte 255 and NaN for every number: all that is computed from it is NaN.
//
// Scales lie as the tensor core wants them in tensor memory: a tile of 512 bytes holds 128 rows times four blocks; row r,
// block b of the tile at byte (r % 32) * 16 + (r / 32) * 4 + b, so that tcgen05.cp with the shape 32x128b makes of it four columns of
// tensor memory, row r in lane r % 32 of column r / 32, its four blocks in the four bytes of that word.  Tiles are ordered
// [128 rows][512 columns].
#pragma once

#include "tcgen05.cuh"

namespace fp8 {

constexpr int BLOCK = 128;                 // numbers that share a scale
constexpr int SF_TILE = 512;               // bytes of scales for 128 rows x 4 blocks

__host__ __device__ __forceinline__ int blocks_of(int cols) { return (cols + BLOCK - 1) / BLOCK; }
__host__ __device__ __forceinline__ int quads_of(int cols) { return (cols + 4 * BLOCK - 1) / (4 * BLOCK); }

// where the four scales of row r (of the matrix, or r of the tile's rows with `tile0` its first tile) and blocks 4 q .. lie
__device__ __forceinline__ size_t scale_at(long row, int q, int quads) {
    return ((size_t)(row >> 7) * quads + q) * SF_TILE + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// the scale's byte for a block whose largest magnitude has these bits
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
    const int e = (int)(bits >> 23);
    if (e >= 255) return 255u;
    // 448 = 1.75 * 2^8: an exponent of eight less, one more where the mantissa is beyond 0.75
    return (uint32_t)max(e - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}
__device__ __forceinline__ float scale_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }      // byte <= 247
__device__ __forceinline__ float scale_value(uint32_t byte) {
    return byte == 255u ? __uint_as_float(0x7fc00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
// four numbers, scaled by `inv` (exact), rounded to nearest even
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, float inv) {
    uint32_t r;
    asm("{\n.reg .b16 lo, hi;\ncvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\ncvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\nmov.b32 %0, {lo, hi};\n}"
        : "=r"(r) : "f"(a * inv), "f"(b * inv), "f"(c * inv), "f"(d * inv));
    return r;
}
constexpr uint32_t NAN4 = 0x7f7f7f7fu;

// One lane of a warp that is there as a whole.  The compiler knows of this one that it is alone and keeps what the products are
// given in uniform registers.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}

// Activations that leave what is not a number so (a block that is NaN makes NaN of all that is computed from it; fminf and fmaxf
// would take the other number).
enum : int { ACT_NONE = 0, ACT_RELU2 = 1 };
__device__ __forceinline__ float act_of(float v, int act) {
    if (act == ACT_RELU2) {
        v = v < 0.0f ? 0.0f : v;
        return v * v;
    }
    return v;
}
__device__ __forceinline__ float gate_of(float z, float u, int act, float limit) {
    if (act == 2) {
        z = z > limit ? limit : z;
        u = (u > limit ? limit : u < -limit ? -limit : u) + 1.0f;
        return z * tc::fast_rcp(1.0f + tc::fast_exp2(-1.4426950408889634f * 1.702f * z)) * u;
    }
    // z * sigmoid(k): k = z for silu (act 1), k = 2 sqrt(2/pi) (z + 0.044715 z^3) for the tanh form of gelu (act 0); one code for
    // both, which the epilogues are shorter and faster with
    constexpr float LOG2E = 1.4426950408889634f, A = 1.5957691216057308f;
    const float c = act == 0 ? -LOG2E * A : -LOG2E;
    const float f = act == 0 ? fmaf(-LOG2E * A * 0.044715f * z, z, c) : c;
    return z * tc::fast_rcp(1.0f + tc::fast_exp2(z * f)) * u;
}

// ---- tensor core, operands e4m3, scales ue8m0
// Instruction descriptor of kind::mxf8f6f4 without the scales' byte numbers (a: bits 29-30, b: bits 4-5).
__device__ __forceinline__ uint32_t idesc_mx(int m, int n) {
    return (1u << 23) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t with_block(uint32_t id, int a_byte, int b_byte) {
    return id | ((uint32_t)a_byte << 29) | ((uint32_t)b_byte << 4);
}
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\n"
                 "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// A scale tile in shared memory: 32 rows of 16 bytes, eight rows (128 bytes) to the next group, no swizzle.
__device__ __forceinline__ uint64_t desc_scales(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fffu) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint64_t desc) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// an untiled copy; both addresses and the size multiples of 16 bytes
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// ---- host: what the launchers take, packed by the host as C lays it out
struct RowsCall {                // brolm_fp8_quantize, brolm_fp8_read
    void *x, *values, *scales;
    cudaStream_t stream;
    long long ldx, ldv, rows;
    int dtype, cols, group, group_pad, early;
};
struct ProductCall {             // brolm_fp8_stream, brolm_fp8_gemm and, with the second half, their forms for experts
    const void *x, *x_scales, *w, *w_scales;
    void *y, *y_scales;
    cudaStream_t stream;
    long long ldx, ldw, ldy;
    int M, N, K, epilogue, act, out, fused, cut;       // cut: slices (stream), blocks of a piece (gemm)
    float limit;
    int experts;
    const void *tile_group, *tile_row0, *offsets, *perm, *scale;
    int group_rows, down, top, tokens, rows, max_tiles;
    int listed;                  // the list is older than the kernel before, which has waited for its own predecessor before it let this one begin
    // rows that are still to be rounded into x and x_scales, by brolm_fp8_quantize ahead of the product (null: they are there)
    int (*quantize)(const RowsCall*);
    const void* raw;
    long long ld_raw;
    int raw_dtype;
    int piece;                   // (stream) blocks of K that a float result is summed over before the sum goes to registers; 0: all
    int fresh;                   // (dense) W may be what the kernel before writes: it is not read before that has ended
};
static inline int round_first(const ProductCall* c) {
    if (!c->quantize) return BROLM_OK;
    const RowsCall r = {const_cast<void*>(c->raw), const_cast<void*>(c->x), const_cast<void*>(c->x_scales), c->stream, c->ld_raw, c->ldx, c->M,
                        c->raw_dtype, c->K, c->M, c->M, 1};
    return c->quantize(&r);
}

// ---- host: rows x cols bytes, row-major with `ld` bytes between rows; box = box_rows x 128 columns, 128-byte swizzle
static inline int make_map_u8(CUtensorMap* map, const void* ptr, long long rows, long long cols, long long ld, int box_rows) {
    tc::EncodeTiled enc = tc::encoder();
    if (!enc) return BROLM_ERR_BAD_SIZE;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, elem,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? BROLM_OK : BROLM_ERR_ALIGNMENT;
}

}  // namespace fp8
