// e4m3 values with scales of blocks of 128 columns: what their writers and readers share.
#pragma once

#include "common.cuh"

namespace b200q {

constexpr int DT_E4M3 = 3;                // beside the C ABI's dtype codes, where a call says so
constexpr int kF8Block = 128;

int f8_status_read_clear(int* v);         // f8_linear.cu

// The scale of a block whose largest magnitude is `top`: that becomes 448. Blocks of zeros have a scale whose reciprocal is a number.
__device__ __forceinline__ float f8_scale(float top) { return fmaxf(top, 1e-30f) * (1.f / 448.f); }

// Four values, the first in the lowest byte; nearest even, beyond the type's range its largest number, NaN stays
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t)hi << 16 | lo;
}
__device__ __forceinline__ void e4m3x4_values(uint32_t w, float* v) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t h;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)(w >> 16 * i)));
        const float2 f = __half22float2(*reinterpret_cast<const half2*>(&h));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
    }
}

}  // namespace b200q
