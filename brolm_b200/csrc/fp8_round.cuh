// Numbers of a row on their way to 8 bits: a warp takes four blocks of 128 at a time, eight lanes a block, sixteen numbers a lane.
#pragma once

#include "fp8.cuh"

namespace fp8 {

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

}  // namespace fp8
