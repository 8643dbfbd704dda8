// The rounding to 8 bits (e4m3) with a power of two as a block's scale, shared by the kernels that do it.
#pragma once

#include "common.cuh"

namespace block_scaled {

constexpr int kBlock = 128;              // numbers along a row that share a scale
constexpr int kMostAlong = 0x7fffff00;   // rows or columns: places are counted in 32 bits, up to the end of a tile

// The scale of a block whose largest magnitude has the bits `largest`, and its inverse: the exponent of the magnitude, one more where the
// mantissa is above 448's (0x600000), less 8; not below 2^-126.  NaN where the block holds an infinity or a NaN.
struct Rounding {
    float scale, inverse;
};
__device__ __forceinline__ Rounding rounding_of(uint32_t largest) {
    const bool finite = largest < 0x7f800000u;
    const uint32_t bits = finite ? (uint32_t)max((int)((largest + 0x1fffffu) >> 23) - 8, 1) << 23 : 0x7fffffffu;
    Rounding r;
    r.scale = __uint_as_float(bits);
    r.inverse = __uint_as_float(finite ? (254u << 23) - bits : 0x7fffffffu);
    return r;
}

// Four numbers as e4m3, the first in the lowest byte.
__device__ __forceinline__ uint32_t four_of(float a, float b, float c, float d, float inverse) {
    uint16_t low, high;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(low) : "f"(b * inverse), "f"(a * inverse));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(high) : "f"(d * inverse), "f"(c * inverse));
    return (uint32_t)low | (uint32_t)high << 16;
}

}  // namespace block_scaled
