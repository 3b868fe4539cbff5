// The cache in 8 bits, as its kernels see it.
//
// Keys and values lie in blocks [block][kv head][P tokens][D entries] of int8; a number q of block b and head g stands for
// q * scale[b][g], and the scale is a power of two:
//
//     2^e,  e the least integer >= -126 with  max |x| <= 127 * 2^e  over all that the block of that head has been given.
//
// Why a power of two and not max / 127: x * 2^-e and q * 2^e are exact, so the same numbers give the same bits wherever
// they are rounded; and a block that fills token by token is rounded anew whenever its scale grows, by half a step of the
// new scale each time, which adds up to less than one step if the steps at least double (1/2 + 1/4 + ...) and to much
// more if they creep.  It costs up to a factor of two (1.44 on average) in the step of a block that is filled at once.
//
// A block that is given a number that is not finite has the scale NaN until it is begun anew: all that it holds for that
// head reads as NaN, and a query that sees any of its keys gets NaN.
#pragma once

#include "common.cuh"

namespace kv8 {

constexpr int MAX_DIM = 256;           // entries of a head
constexpr int MAX_BLOCK = 256;         // tokens of a block

// Exponent of the scale that `amax` (finite, >= 0) needs: amax = 1.m 2^x fits 127 2^(x - 6) unless 1.m > 127/64.
__device__ __forceinline__ int scale_exponent(float amax) {
    const unsigned bits = __float_as_uint(amax);
    const int e = (int)(bits >> 23) - 127 - 6 + ((bits & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return max(e, -126);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }   // -126 <= e <= 127

}  // namespace kv8
