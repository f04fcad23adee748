// What the attention kernels share.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "mma.cuh"

namespace b200q {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kTiny = 1e-30f;          // the smallest scale of a page that the cache's writer gives; attention takes smaller ones for it

struct AttnParams {
    const void *q, *k, *v;
    void* out;
    int64_t qs[3], ks[3], vs[3], os[3];      // strides of batch, row, head in elements (k and v: 16-bit rows only)
    const float *k_scale, *v_scale;          // pages: [pages, Hkv]
    const int32_t* table;                    // [B, max_pages]
    int64_t table_stride, pages;
    const int32_t* kv_len;                   // keys of each sequence, or null: Lkv
    const int32_t* q_len;                    // query rows of each sequence, or null: Lq
    const uint8_t* mask;                     // [B, Lkv], 0 = not seen, or null
    int64_t mask_stride;
    int B, Lq, Lkv, H, Hkv, D, T, causal, splits, row_tiles;
    float scale;
    // packed sequences: rows offsets[b] to offsets[b + 1] of `rows` are sequence b; a tile has tile_tokens of its tokens and `pack` heads of each,
    // which read one head of k and v
    const int32_t* offsets;
    int rows, pack, tile_tokens;
};

// ---- packed sequences
// Their tiles are numbered without a table: sequence b has those from offsets[b] / tile_tokens + b on, at least as many as it fills and at most one
// more than it needs. Offsets outside the rows, or falling ones, give tiles inside the rows all the same.
struct PackedTile {
    int64_t start;             // row of the sequence's first token
    int len, token0, tokens;   // its tokens, and those of the tile; none: a tile that nobody needs
};
__device__ __forceinline__ int offset_at(const AttnParams& p, int b) { return min(max(gload(p.offsets + b), 0), p.rows); }
// A whole warp finds the tile, 32 sequences at a look; up to 31 with one load for all that it has to know
__device__ __forceinline__ PackedTile packed_tile(const AttnParams& p, int tile) {
    const int lane = threadIdx.x & 31;
    int lo = 0, start, end;
    if (p.B < 32) {
        const int mine = offset_at(p, min(lane, p.B));
        lo = max(0, __popc(__ballot_sync(0xffffffffu, lane < p.B && mine / p.tile_tokens + lane <= tile)) - 1);
        start = __shfl_sync(0xffffffffu, mine, lo), end = __shfl_sync(0xffffffffu, mine, lo + 1);
    } else {
        int hi = p.B;
        while (hi - lo > 1) {
            const int step = (hi - lo + 31) / 32, b = lo + (lane + 1) * step;
            const bool before = b < hi && offset_at(p, b) / p.tile_tokens + b <= tile;
            lo += __popc(__ballot_sync(0xffffffffu, before)) * step;
            hi = min(hi, lo + step);
        }
        start = offset_at(p, lo), end = offset_at(p, lo + 1);
    }
    PackedTile x;
    const int ahead = tile - (start / p.tile_tokens + lo);
    x.start = start;
    x.len = ahead < 0 ? 0 : max(0, end - start);
    x.token0 = ahead < 0 || ahead > x.len / p.tile_tokens ? x.len : ahead * p.tile_tokens;
    x.tokens = min(p.tile_tokens, x.len - x.token0);
    return x;
}
// Numbers beyond the type's range, and what is none, among eight neighbouring values
template <typename T> __device__ __forceinline__ bool any_infinite(uint4 w) {
    const uint32_t top = std::is_same<T, half>::value ? 0x7C007C00u : 0x7F807F80u;
    return (__vcmpeq2(w.x & top, top) | __vcmpeq2(w.y & top, top) | __vcmpeq2(w.z & top, top) | __vcmpeq2(w.w & top, top)) != 0;
}
// sum += 0 * x in both halves: NaN once one of them is
template <typename T> __device__ __forceinline__ void add_zero_times(uint32_t& sum, uint32_t x) {
    if (std::is_same<T, half>::value) asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0));
    else asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(x), "r"(0));
}
// Takes them out of values of V that some rows of a tile see and others do not (a weight of 0 does not hide them in a product) and notes for each
// of the eight columns the first key that had one: rows from that token on get NaN there.
template <typename T> __device__ __forceinline__ uint4 without_infinite(uint4 w, int key, int* from) {
    T* v = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        if (!(fabsf(to_f<T>(v[e])) <= FLT_MAX)) {
            v[e] = from_f<T>(0.f);
            atomicMin(from + e, key);
        }
    return w;
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Four int8 codes as four halves, exact: each byte, its sign bit turned, becomes the low byte of 1024 + (code + 128), and 1152 is taken away.
__device__ __forceinline__ uint2 halves_of4(uint32_t w) {
    const uint32_t off = 0x64806480u, a = w ^ 0x80808080u;
    const uint32_t lo = __byte_perm(a, 0x64646464u, 0x4140), hi = __byte_perm(a, 0x64646464u, 0x4342);
    const half2 x = __hsub2(*reinterpret_cast<const half2*>(&lo), *reinterpret_cast<const half2*>(&off));
    const half2 y = __hsub2(*reinterpret_cast<const half2*>(&hi), *reinterpret_cast<const half2*>(&off));
    return make_uint2(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y));
}

// bf16 queries over int8 keys are taken as halves times a power of two: 2^e brings a row's largest magnitude to [2^14, 2^15). e is -113 for the
// type's largest numbers and at most 126, so that 2^e and 2^-e are normal f32 numbers; rows below 2^-112 stay smaller, but times 2^126 every
// bf16 number of at most that size is a half exactly (the smallest, 2^-133, is 2^-7).
__device__ __forceinline__ int row_exponent(float top) {
    return top > 0.f && top <= FLT_MAX ? min(126, 14 - ((int)(__float_as_uint(top) >> 23) - 127)) : 0;
}

// A page's scale of V in the logits (its power of two, which p then carries) and out of the sum of p again. A scale below kTiny is taken for it. NaN
// makes p NaN where a key is seen; its weight is a number, so that a key which is not seen adds nothing.
__device__ __forceinline__ float v_scale_log2(float s) { return log2f(s < kTiny ? kTiny : s); }
__device__ __forceinline__ float v_scale_weight(float s) { return s != s ? 1.f : 1.f / fmaxf(s, kTiny); }

// Eight columns of a finished row; one that saw no key is zeros, NaN stays.
template <typename QT> __device__ __forceinline__ void store_piece(QT* dst, const float (&y)[8], float total) {
    const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
    uint4 w;
    uint32_t* ow = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) ow[e] = pack2<QT>(y[2 * e] * inv, y[2 * e + 1] * inv);
    *reinterpret_cast<uint4*>(dst) = w;
}
template <typename QT> __device__ __forceinline__ void store_row(const AttnParams& p, const float (&y)[8], float total, int b, int row, int kvh, int ratio, int d, QT) {
    store_piece(reinterpret_cast<QT*>(p.out) + b * p.os[0] + (int64_t)(row / ratio) * p.os[1] + (kvh * ratio + row % ratio) * p.os[2] + d, y, total);
}

// The kernel for many query rows (attention_tc.cu): takes rows of at most 128 values and positive scales.
bool attention_tc_takes(const AttnParams& p, bool kv8);
int attention_tc(int dtype, bool kv8, AttnParams& p, cudaStream_t st);
bool attention_tc_takes_packed(const AttnParams& p);
int attention_tc_packed(int dtype, AttnParams& p, cudaStream_t st);
int attention_status_read_clear(int* v);

}  // namespace b200q
