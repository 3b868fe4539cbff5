// Numbers of a row on their way to 8 bits: a warp takes four blocks of 128 at a time, eight lanes a block, sixteen numbers a
// lane, so that the block's largest magnitude goes round in three shuffles.  (With the lanes' words side by side, as they are
// best loaded, it takes eight: 8,192 x 4,608 bfloat16 numbers 32.9 us where this took 24.8.)
#pragma once

#include "fp8.cuh"

namespace fp8 {

// The same sixteen numbers on their way: where all of them are there and lie on a border of sixteen bytes they are asked for
// without being looked at, so that several pieces can be under way.
template <typename T, bool WIDE>
struct Piece {
    static constexpr int WORDS = (int)sizeof(T);               // sixteen numbers are 2 or 4 sixteen-byte words
    uint4 raw[WORDS];
    __device__ __forceinline__ void ask(const T* row, int c, int cols, bool wanted) {
        const uint4* src = reinterpret_cast<const uint4*>(row + c);
#pragma unroll
        for (int i = 0; i < WORDS; ++i) raw[i] = WIDE && wanted && c + 16 <= cols ? src[i] : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(const T* row, int c, int cols, float (&v)[16]) const {
        if (WIDE && c + 16 <= cols) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) {
                const uint32_t u[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if constexpr (WORDS == 2) {
                        v[8 * i + 2 * j] = __uint_as_float(u[j] << 16);
                        v[8 * i + 2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                    } else {
                        v[4 * i + j] = __uint_as_float(u[j]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = c + i < cols ? to_float(row[c + i]) : 0.0f;
        }
    }
};

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
