// Rows to 8 bits and back (the format is in fp8.cuh).
//
//   fp8_quantize   rows of float or bfloat16 numbers -> e4m3 numbers and a scale byte for every 128 of them
//   fp8_read       the values that they stand for
//
// Both are one pass over the data: a warp takes four blocks of a row at a time (512 numbers, one word of scales), eight
// lanes a block and sixteen numbers a lane; the block's largest magnitude goes round its eight lanes in three shuffles.
#include "fp8.cuh"

namespace {

using namespace fp8;

constexpr int THREADS = 256, WARPS = THREADS / 32;

struct RowsArgs {
    const void* x; long ldx;        // elements
    uint8_t* values; long ldv;      // bytes
    uint8_t* scales;
    long rows;                      // of all groups
    int cols, quads;
    // rows come in groups of `group` rows; in the matrix a group takes `group_pad` rows (the same for a plain matrix)
    int group, group_pad;
    int early;                      // the next kernel may begin before this one's results are there
};

// Sixteen numbers of a row from column c on; zeros from `cols` on.
template <bool WIDE>
__device__ __forceinline__ void load16(const bf16* row, int c, int cols, float (&v)[16]) {
    if (WIDE && c + 16 <= cols) {
        float a[8], b[8];
        load8(row + c, a);
        load8(row + c + 8, b);
#pragma unroll
        for (int i = 0; i < 8; ++i) { v[i] = a[i]; v[8 + i] = b[i]; }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < cols ? __bfloat162float(row[c + i]) : 0.0f;
}
template <bool WIDE>
__device__ __forceinline__ void load16(const float* row, int c, int cols, float (&v)[16]) {
    if (WIDE && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const float4 f = *reinterpret_cast<const float4*>(row + c + i);
            v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = c + i < cols ? row[c + i] : 0.0f;
}

// The warp's 512 numbers to 8 bits: this lane's sixteen, and (in every lane) the word of the four blocks' scales.
__device__ __forceinline__ uint4 round16(const float (&v)[16], uint32_t& word) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) most = max(most, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
    const uint32_t byte = scale_byte(most);
    uint4 q = make_uint4(NAN4, NAN4, NAN4, NAN4);
    if (byte != 255u) {
        const float inv = scale_inverse(byte);
        q.x = pack4(v[0], v[1], v[2], v[3], inv);
        q.y = pack4(v[4], v[5], v[6], v[7], inv);
        q.z = pack4(v[8], v[9], v[10], v[11], inv);
        q.w = pack4(v[12], v[13], v[14], v[15], inv);
    }
    word = byte << (8 * ((threadIdx.x & 31) >> 3));
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    word |= __shfl_xor_sync(0xffffffffu, word, 16);
    return q;
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) quantize_kernel(RowsArgs g) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long row = item / g.quads;
        const int quad = (int)(item - row * g.quads), c = quad * 512 + lane * 16;
        const long at = g.group == g.group_pad ? row : row / g.group * g.group_pad + row % g.group;
        float v[16];
        load16<WIDE>((const T*)g.x + row * g.ldx, c, g.cols, v);
        uint32_t word;
        const uint4 q = round16(v, word);
        if (c < g.ldv) *reinterpret_cast<uint4*>(g.values + at * g.ldv + c) = q;     // ldv is a multiple of 16
        if (lane == 0) *reinterpret_cast<uint32_t*>(g.scales + scale_at(at, quad, g.quads)) = word;
    }
    // The products read their matrix before they wait for the kernel before them, so a kernel that writes a matrix lets
    // nothing begin before it has ended; one that writes rows that a product waits for may.
    if (g.early) pdl_trigger();
}

template <typename T> __device__ __forceinline__ void store16(T* row, int c, int cols, const float (&v)[16], bool wide);
template <> __device__ __forceinline__ void store16<float>(float* row, int c, int cols, const float (&v)[16], bool wide) {
    if (wide && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(row + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) if (c + i < cols) row[c + i] = v[i];
}
template <> __device__ __forceinline__ void store16<bf16>(bf16* row, int c, int cols, const float (&v)[16], bool wide) {
    if (wide && c + 16 <= cols) {
#pragma unroll
        for (int i = 0; i < 16; i += 8) {
            uint4 p;
            __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&p);
#pragma unroll
            for (int e = 0; e < 4; ++e) h[e] = __floats2bfloat162_rn(v[i + 2 * e], v[i + 2 * e + 1]);
            *reinterpret_cast<uint4*>(row + c + i) = p;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) if (c + i < cols) row[c + i] = __float2bfloat16_rn(v[i]);
}

template <typename T>
__global__ void __launch_bounds__(THREADS) read_kernel(RowsArgs g, T* __restrict__ y, long ldy, bool wide) {
    const int lane = threadIdx.x & 31;
    const long items = g.rows * g.quads;
    pdl_wait();
    for (long item = (long)blockIdx.x * WARPS + (threadIdx.x >> 5); item < items; item += (long)gridDim.x * WARPS) {
        const long row = item / g.quads;
        const int quad = (int)(item - row * g.quads), c = quad * 512 + lane * 16;
        const long at = g.group == g.group_pad ? row : row / g.group * g.group_pad + row % g.group;
        if (c >= g.cols) continue;
        const uint4 q = *reinterpret_cast<const uint4*>(g.values + at * g.ldv + c);
        const float s = scale_value(g.scales[scale_at(at, quad, g.quads) + (lane >> 3)]);
        const uint32_t words[4] = {q.x, q.y, q.z, q.w};
        float v[16];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t lo, hi;                     // e4m3 numbers are f16 numbers
            asm("{\n.reg .b16 a, b;\nmov.b32 {a, b}, %2;\ncvt.rn.f16x2.e4m3x2 %0, a;\ncvt.rn.f16x2.e4m3x2 %1, b;\n}" : "=r"(lo), "=r"(hi) : "r"(words[i]));
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&lo)), h = __half22float2(*reinterpret_cast<const __half2*>(&hi));
            v[4 * i] = f.x * s; v[4 * i + 1] = f.y * s; v[4 * i + 2] = h.x * s; v[4 * i + 3] = h.y * s;
        }
        store16<T>(y + row * ldy, c, g.cols, v, wide);
    }
    pdl_trigger();
}

int grid_for(long items) {
    const long blocks = (items + WARPS - 1) / WARPS, most = 16L * tc::device_sms();
    return (int)(blocks < most ? blocks : most);
}

}  // namespace

// x [rows, cols] (float or bfloat16, ldx elements between rows) -> values (ldv bytes between rows, a multiple of 16, at least
// cols) and scales.  Rows come in groups of `group`, which lie `group_pad` rows (a multiple of 128 if not `group`) apart.
BROLM_API int brolm_fp8_quantize(int dtype, const void* x, long long ldx, void* values, long long ldv, void* scales, long long rows,
                                 int cols, int group, int group_pad, int early, cudaStream_t stream) {
    if (rows <= 0 || cols <= 0) return BROLM_OK;
    if (ldv % 16 != 0 || ldv < cols || ((uintptr_t)values & 15) || ((uintptr_t)scales & 15)) return BROLM_ERR_ALIGNMENT;
    if (group <= 0 || group_pad < group) return BROLM_ERR_BAD_SIZE;
    RowsArgs g = {x, (long)ldx, (uint8_t*)values, (long)ldv, (uint8_t*)scales, (long)rows, cols, fp8::quads_of(cols), group, group_pad, early};
    const dim3 grid(grid_for(rows * g.quads)), block(THREADS);
    if (dtype == BROLM_BF16) {
        if (((uintptr_t)x & 15) == 0 && ldx % 8 == 0) return launch_pdl(quantize_kernel<bf16, true>, grid, block, 0, stream, g);
        return launch_pdl(quantize_kernel<bf16, false>, grid, block, 0, stream, g);
    }
    if (dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    if (((uintptr_t)x & 15) == 0 && ldx % 4 == 0) return launch_pdl(quantize_kernel<float, true>, grid, block, 0, stream, g);
    return launch_pdl(quantize_kernel<float, false>, grid, block, 0, stream, g);
}

BROLM_API int brolm_fp8_read(int dtype, const void* values, long long ldv, const void* scales, void* y, long long ldy, long long rows,
                             int cols, int group, int group_pad, cudaStream_t stream) {
    if (rows <= 0 || cols <= 0) return BROLM_OK;
    if (ldv % 16 != 0 || ldv < cols || ((uintptr_t)values & 15)) return BROLM_ERR_ALIGNMENT;
    if (group <= 0 || group_pad < group) return BROLM_ERR_BAD_SIZE;
    RowsArgs g = {nullptr, 0, (uint8_t*)const_cast<void*>(values), (long)ldv, (uint8_t*)const_cast<void*>(scales), (long)rows, cols,
                  fp8::quads_of(cols), group, group_pad, 1};
    const dim3 grid(grid_for(rows * g.quads)), block(THREADS);
    const bool base = ((uintptr_t)y & 15) == 0;
    if (dtype == BROLM_BF16) return launch_pdl(read_kernel<bf16>, grid, block, 0, stream, g, (bf16*)y, (long)ldy, base && ldy % 8 == 0);
    if (dtype != BROLM_F32) return BROLM_ERR_BAD_DTYPE;
    return launch_pdl(read_kernel<float>, grid, block, 0, stream, g, (float*)y, (long)ldy, base && ldy % 4 == 0);
}
