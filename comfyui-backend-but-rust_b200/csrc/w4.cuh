// What the kernels of the 4-bit linear share: its arguments, codes as matrix operands, f32 rows as bf16 terms, the way out.
#pragma once

#include "common.cuh"
#include "mma.cuh"

namespace b200q {

__device__ __forceinline__ float scale_at(const void* s, int dt, int64_t i) {
    return dt == DT_F16 ? __half2float(gload(reinterpret_cast<const half*>(s) + i)) : __bfloat162float(gload(reinterpret_cast<const bf16*>(s) + i));
}

// What a CTA of the kernel for few columns has in shared memory.
struct RowsShare {
    int kw, kw_log, rows, rows_log, splits_log;      // warps along K, rows, CTAs along K: powers of two
    int blocks, stages, x_pitch;                     // blocks of 128 of K to a CTA, stages of a warp, bytes to a column of x
    int scale_words, zero_words, scales, smem;       // words to a row of scales and of zero points, where they begin, all of it
};
struct W4Params {
    const void* x;
    int64_t x_stride;
    const uint8_t* W;
    const void* scales;
    const uint8_t* zeros;
    const void* bias;
    void* out;
    int64_t out_stride;
    int M, N, K, G, scale_dt, out_dt, groups;
    float beta;
    int group_shift; // log2(G / 32)
    int splits;      // CTAs that share a tile's K
    RowsShare share;
};

// Codes in registers: a word holds columns 8t..8t+7 of a row, a pair of neighbours in each byte. The pair's byte goes to both halves of a
// register, the exponent of 1024 (f16) or 1/32 (bf16) around its nibble, and one instruction takes away the offset and the zero point: the
// code minus its zero point is a small integer (bf16: times 2^-12), exact in either type, and so are its products with x in the f32 sums.
// The 2^-12 keeps a group's sum, up to 256 terms of 15 |x|, in f32's range for every x that bf16 and f32 have; kUp takes it out of the
// finished row's value. (|x| below 2^-100 may lose bits to it.)
// `expand` gives neighbouring columns (2i, 2i + 1); `expand4` columns (i, i + 4), which takes fewer instructions but needs x in that order.
template <typename T> struct Nibbles;
template <> struct Nibbles<half> {
    static constexpr float kUp = 1.f;
    uint32_t sub;       // (-1024 - z, -64 - z): the high half's nibble sits four bits up, its scale of 1/16 is in the same instruction
    uint32_t lo, hi;    // the same for both halves of a register alike
    __device__ __forceinline__ explicit Nibbles(uint32_t z)
        : sub((0xE400u + z) | (0xD400u + (z << 4)) << 16), lo((0xE400u + z) * 0x00010001u), hi((0xD400u + (z << 4)) * 0x00010001u) {}
    static constexpr uint32_t kBits = 0x64006400u;
    __device__ __forceinline__ void expand4(uint32_t w, uint32_t (&r)[4], uint32_t bits) const {      // bits: kBits, held
        const uint32_t one_16th = 0x2C002C00u;
#pragma unroll
        for (int i = 0; i < 2; ++i, w >>= 8) {
            const uint32_t a = and_or<0x000F000Fu>(w, bits), b = and_or<0x00F000F0u>(w, bits);
            const half2 x = __hadd2(*reinterpret_cast<const half2*>(&a), *reinterpret_cast<const half2*>(&lo));
            const half2 y = __hfma2(*reinterpret_cast<const half2*>(&b), *reinterpret_cast<const half2*>(&one_16th), *reinterpret_cast<const half2*>(&hi));
            r[2 * i] = *reinterpret_cast<const uint32_t*>(&x), r[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&y);
        }
    }
    __device__ __forceinline__ void expand(uint32_t w, uint32_t (&r)[4]) const {
        const uint32_t one_16th = 0x2C003C00u;      // (1, 1/16)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (__byte_perm(w, 0, 0x4040 + 0x0101 * i) & 0x00F0000Fu) | 0x64006400u;
            const half2 v = __hfma2(*reinterpret_cast<const half2*>(&b), *reinterpret_cast<const half2*>(&one_16th), *reinterpret_cast<const half2*>(&sub));
            r[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};
template <> struct Nibbles<bf16> {
    static constexpr float kUp = 4096.f;
    uint32_t sub;       // 2^-5 + 2^-12 z in both halves
    __device__ __forceinline__ explicit Nibbles(uint32_t z) : sub((0x3D00u + z) * 0x00010001u) {}
    static constexpr uint32_t kBits = 0x3D003D00u;
    __device__ __forceinline__ void expand4(uint32_t w, uint32_t (&r)[4], uint32_t bits) const {      // bits: kBits, held
#pragma unroll
        for (int i = 0; i < 4; ++i, w >>= 4) {
            const uint32_t b = and_or<0x000F000Fu>(w, bits);
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&sub));
            r[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    __device__ __forceinline__ void expand(uint32_t w, uint32_t (&r)[4]) const {
        const uint32_t up = w >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (__byte_perm(w, up, 0x4040 + 0x0101 * i + 0x0400) & 0x000F000Fu) | kBits;
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&sub));
            r[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};

// Two f32 values as three bf16 numbers each, whose sum they are: eight leading bits each, cut off, so that every remainder is exact.
// Infinities and NaN stay in the first.
__device__ __forceinline__ void split3(float v, uint32_t (&part)[3]) {
    if (!(fabsf(v) <= FLT_MAX)) {
        part[0] = (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) << 16, part[1] = part[2] = 0u;
        return;
    }
    part[0] = __float_as_uint(v) & 0xFFFF0000u;
    v -= __uint_as_float(part[0]), part[1] = __float_as_uint(v) & 0xFFFF0000u;
    v -= __uint_as_float(part[1]), part[2] = __float_as_uint(v);
}
template <int P> __device__ __forceinline__ void split2(float a, float b, uint4 (&r)[P], int at) {
    uint32_t pa[3], pb[3];
    split3(a, pa), split3(b, pb);
#pragma unroll
    for (int q = 0; q < P; ++q) reinterpret_cast<uint32_t*>(&r[q])[at] = __byte_perm(pa[q], pb[q], 0x7632);
}

template <int XT> struct XType { using Mma = bf16; };
template <> struct XType<DT_F16> { using Mma = half; };

// Columns of the product: a token's values, or the three parts of an f32 token's.
template <int XT> __host__ __device__ constexpr int parts_of() { return XT == DT_F32 ? 3 : 1; }

// Eight values of token m from k on, for each of its columns the four registers that two steps of the product take; zeros outside.
template <int XT> __device__ __forceinline__ void x_words(const W4Params& p, int m, int k, uint4 (&r)[parts_of<XT>()]) {
    if (m >= p.M || k >= p.K) {
#pragma unroll
        for (int q = 0; q < parts_of<XT>(); ++q) r[q] = make_uint4(0, 0, 0, 0);
    } else if (XT != DT_F32) {
        r[0] = gload(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + m * p.x_stride + k));
    } else {
        const float* src = reinterpret_cast<const float*>(p.x) + m * p.x_stride + k;
        const float4 a = gload(reinterpret_cast<const float4*>(src)), b = gload(reinterpret_cast<const float4*>(src) + 1);
        split2(a.x, a.y, r, 0), split2(a.z, a.w, r, 1), split2(b.x, b.y, r, 2), split2(b.z, b.w, r, 3);
    }
}

template <typename T> __device__ __forceinline__ float out_value(const W4Params& p, float y, int n, T* o) {
    if (p.bias) y += to_f<T>(gload(reinterpret_cast<const T*>(p.bias) + n));
    if (p.beta != 0.f) y = __fmaf_rn(p.beta, to_f<T>(gload(o)), y);
    return y;
}
__device__ __forceinline__ void store_out(const W4Params& p, float y, int m, int n) {
    const int64_t at = m * p.out_stride + n;
    if (p.out_dt == DT_F32) {
        float* o = reinterpret_cast<float*>(p.out) + at;
        *o = out_value<float>(p, y, n, o);
    } else if (p.out_dt == DT_F16) {
        half* o = reinterpret_cast<half*>(p.out) + at;
        *o = __float2half_rn(out_value<half>(p, y, n, o));
    } else {
        bf16* o = reinterpret_cast<bf16*>(p.out) + at;
        *o = __float2bfloat16_rn(out_value<bf16>(p, y, n, o));
    }
}

// What a kernel may have of shared memory is one setting for all threads of the program: always the most a CTA can have, never a call's own need,
// which another thread's smaller one could replace before the launch.
constexpr int kMostSmem = 227 * 1024;

// The kernel for many tokens (w4_tile.cu)
int w4_tile(int dtype, const W4Params& p, cudaStream_t st);
int w4_status_read_clear(int* out);

}  // namespace b200q
