// Linears with 4-bit weights and group scales (no counterpart in the reference, whose smallest weight has 6 bits and int8 activations;
// its text encoders keep their activations in floating point beside weight-only int8, src/te.rs:493-511, which is the use here).
//
//   gpu_w4_requant   f32 / f16 / bf16 weight -> codes, group scales, zero points
//   gpu_w4_dequant   the way back
//   gpu_w4_linear    out = beta * out + x . W^T + bias straight from the codes
//
// W[n, k] = (c[n, k] - z[n, k/G]) * s[n, k/G] with c and z in 0..15 (z = 8 without zero points). Codes [N, K/2]: column 2i in the low
// nibble of byte i, 2i + 1 in the high one (the order of the W6 format's nibble plane).
#include "common.cuh"
#include "mma.cuh"

namespace {

__device__ __forceinline__ float scale_at(const void* s, int dt, int64_t i) {
    return dt == DT_F16 ? __half2float(gload(reinterpret_cast<const half*>(s) + i)) : __bfloat162float(gload(reinterpret_cast<const bf16*>(s) + i));
}

// ---- the linear -------------------------------------------------------------------------------------------------------------------

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
    int splits;      // warps that share a tile's K
};

// Codes in registers: a word holds columns 8t..8t+7 of a row, a pair of neighbours in each byte. The pair's byte goes to both halves of a
// register, the exponent of 1024 (f16) or 128 (bf16) around its nibble, and one instruction takes away the offset and the zero point: the
// code minus its zero point is a small integer, exact in either type, and so are its products with x in the f32 sums.
template <typename T> struct Nibbles;
template <> struct Nibbles<half> {
    uint32_t sub;       // (-1024 - z, -64 - z): the high half's nibble sits four bits up, its scale of 1/16 is in the same instruction
    __device__ __forceinline__ explicit Nibbles(uint32_t z) : sub((0xE400u + z) | (0xD400u + (z << 4)) << 16) {}
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
    uint32_t sub;       // 128 + z in both halves
    __device__ __forceinline__ explicit Nibbles(uint32_t z) : sub((0x4300u + z) * 0x00010001u) {}
    __device__ __forceinline__ void expand(uint32_t w, uint32_t (&r)[4]) const {
        const uint32_t up = w >> 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = (__byte_perm(w, up, 0x4040 + 0x0101 * i + 0x0400) & 0x000F000Fu) | 0x43004300u;
            const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), *reinterpret_cast<const __nv_bfloat162*>(&sub));
            r[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
    }
};

// One row's f32 value as three bf16 numbers whose sum it is: eight leading bits each, cut off, so that every remainder is exact.
// Infinities and NaN stay in the first.
__device__ __forceinline__ uint32_t bf16_part(float v, int part) {
    if (!(fabsf(v) <= FLT_MAX)) return part == 0 ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v)) : 0u;
    uint32_t hi = __float_as_uint(v) & 0xFFFF0000u;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i < part) v -= __uint_as_float(hi), hi = __float_as_uint(v) & 0xFFFF0000u;
    return hi >> 16;
}

template <int XT> struct XType { using Mma = bf16; };
template <> struct XType<DT_F16> { using Mma = half; };

// Columns of the product: a token's values, or the three parts of an f32 token's.
template <int XT> __host__ __device__ constexpr int parts_of() { return XT == DT_F32 ? 3 : 1; }

// Eight values of column `col` from k on, as the four registers that two steps of the product take; zeros outside.
template <int XT> __device__ __forceinline__ uint4 x_words(const W4Params& p, int col, int k) {
    constexpr int P = parts_of<XT>();
    const int m = col / P;
    if (m >= p.M || k >= p.K) return make_uint4(0, 0, 0, 0);
    if (XT != DT_F32) return gload(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p.x) + m * p.x_stride + k));
    const float* src = reinterpret_cast<const float*>(p.x) + m * p.x_stride + k;
    const float4 a = gload(reinterpret_cast<const float4*>(src)), b = gload(reinterpret_cast<const float4*>(src) + 1);
    const int part = col % P;
    uint4 r;
    r.x = bf16_part(a.x, part) | bf16_part(a.y, part) << 16, r.y = bf16_part(a.z, part) | bf16_part(a.w, part) << 16;
    r.z = bf16_part(b.x, part) | bf16_part(b.y, part) << 16, r.w = bf16_part(b.z, part) | bf16_part(b.w, part) << 16;
    return r;
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

// A stage: 128 columns of 16 rows, 64 bytes a row. Eight rows read at the same column have to lie in eight different 16-byte banks: two
// rows fill a line of 128 bytes, and the pair's number turns the column's.
constexpr int kStageBytes = 16 * 64;
__device__ __forceinline__ uint32_t stage_at(int row, int c) { return (uint32_t)(row * 64 + ((c ^ (row >> 1)) & 3) * 16); }

// One warp's copy of columns 128 * block .. of rows n0..n0+15.
__device__ __forceinline__ void load_stage(const W4Params& p, uint32_t dst, int n0, int block, int lane) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = i * 8 + (lane >> 2), c = lane & 3, k = block * 128 + c * 32;
        const bool valid = n0 + row < p.N && k < p.K;
        cp_async16(dst + stage_at(row, c), valid ? p.W + (int64_t)(n0 + row) * (p.K >> 1) + (k >> 1) : p.W, valid);
    }
}

// Group scales and zero points of the rows that a lane's sums belong to (g and g + 8 of the tile), for one block of 128 columns.
template <int GB> struct Groups {        // GB groups a block: 4, 2 or 1
    float s[GB][2];
    uint32_t z[GB][2];
    __device__ __forceinline__ void load(const W4Params& p, int n0, int block, int lane) {
#pragma unroll
        for (int j = 0; j < GB; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int n = n0 + (lane >> 2) + 8 * h;
                const int grp = (block * 128 + j * (128 / GB)) / p.G;
                const bool valid = n < p.N && grp < p.groups;
                const int64_t at = (int64_t)n * p.groups + grp;
                s[j][h] = valid ? scale_at(p.scales, p.scale_dt, at) : 0.f;
                z[j][h] = valid && p.zeros ? gload(p.zeros + at) & 15u : 8u;
            }
    }
};

// Few columns (at most 8 NT): bound by the weight's bytes. A warp owns 16 rows and a share of K, keeps ST - 1 stages of its own in flight
// (nothing is shared, so nothing waits for another warp) and multiplies in f32 sums of a group, which its scale then adds to the total.
// The warps of a tile meet once, at its end, in shared memory, in a fixed order.
constexpr int kRowsStages = 8;
constexpr int kRowsWarps = 8;

template <int XT, int NT, int GB> __global__ void __launch_bounds__(kRowsWarps * 32) w4_rows_kernel(const W4Params p) {
    using T = typename XType<XT>::Mma;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int S = p.splits, tile = blockIdx.x * (kRowsWarps / S) + warp / S, split = warp % S;
    const int n0 = tile * 16, blocks = (p.K + 127) / 128;
    const int first = (int)((int64_t)split * blocks / S), last = n0 < p.N ? (int)((int64_t)(split + 1) * blocks / S) : first;
    const uint32_t ring = smem_u32(smem) + warp * kRowsStages * kStageBytes;
    pdl_wait();
#pragma unroll
    for (int i = 0; i < kRowsStages - 1; ++i) {
        if (first + i < last) load_stage(p, ring + i * kStageBytes, n0, first + i, lane);
        cp_async_commit();
    }
    float total[NT][4] = {};
    Groups<GB> gr;
    uint4 xw[4][NT];
    auto fetch = [&](int b) {
        gr.load(p, n0, b, lane);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int j = 0; j < NT; ++j) xw[c][j] = x_words<XT>(p, j * 8 + g, b * 128 + c * 32 + t * 8);
    };
    if (first < last) fetch(first);
    int slot = 0;
    for (int b = first; b < last; ++b) {
        cp_async_wait<kRowsStages - 2>();
        __syncwarp();
        const uint32_t at = ring + slot * kStageBytes;
        uint32_t w[2][4];      // [columns 0..63, 64..127][row half, column quarter]
#pragma unroll
        for (int c = 0; c < 2; ++c) ldmatrix4(w[c], at + stage_at((lane & 7) + (lane & 8), 2 * c + (lane >> 4)));
        float sum[NT][4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int grp = c * GB / 4;
            uint32_t lo[4], hi[4];
            Nibbles<T>(gr.z[grp][0]).expand(w[c >> 1][(c & 1) * 2], lo);
            Nibbles<T>(gr.z[grp][1]).expand(w[c >> 1][(c & 1) * 2 + 1], hi);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                mma16816<T>(sum[j], lo[0], hi[0], lo[1], hi[1], xw[c][j].x, xw[c][j].y);
                mma16816<T>(sum[j], lo[2], hi[2], lo[3], hi[3], xw[c][j].z, xw[c][j].w);
            }
            if ((c + 1) * GB % 4 == 0) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) total[j][i] = __fmaf_rn(gr.s[grp][i >> 1], sum[j][i], total[j][i]), sum[j][i] = 0.f;
            }
        }
        if (b + 1 < last) fetch(b + 1);
        __syncwarp();
        const int ahead = b + kRowsStages - 1;
        if (ahead < last) load_stage(p, ring + (slot == 0 ? kRowsStages - 1 : slot - 1) * kStageBytes, n0, ahead, lane);
        cp_async_commit();
        slot = slot + 1 == kRowsStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    // sums of the tile's warps: [warp][column][row], behind the rings
    float* red = reinterpret_cast<float*>(smem + kRowsWarps * kRowsStages * kStageBytes);
    constexpr int kCols = NT * 8;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[(warp * kCols + j * 8 + t * 2 + (i & 1)) * 16 + g + (i >> 1) * 8] = total[j][i];
    __syncthreads();
    constexpr int P = parts_of<XT>();
    const int tiles = kRowsWarps / S;
    for (int i = threadIdx.x; i < tiles * 16 * p.M; i += kRowsWarps * 32) {
        const int r = i & 15, tl = (i >> 4) % tiles, m = (i >> 4) / tiles, n = (blockIdx.x * tiles + tl) * 16 + r;
        if (n >= p.N) continue;
        float y = 0.f;
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int q = 0; q < P; ++q) y += red[((tl * S + s) * kCols + m * P + q) * 16 + r];
        store_out(p, y, m, n);
    }
}

// Many columns: 128 rows of the weight by 64 columns a CTA. Each warp has 16 rows, expanded once for all 64 columns; the columns come in
// blocks of 128 of K that the CTA shares.
constexpr int kTileCols = 64;
constexpr int kTileStages = 3;
constexpr int kTileXBytes = kTileCols * 256;

template <int XT, int GB> __global__ void __launch_bounds__(256) w4_tile_kernel(const W4Params p) {
    using T = typename XType<XT>::Mma;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int P = parts_of<XT>(), kTokens = kTileCols / P;
    const int ntiles = (p.N + 127) / 128, nt = blockIdx.x % ntiles;
    const int n0 = nt * 128 + warp * 16, m0 = blockIdx.x / ntiles * kTokens;
    const int blocks = (p.K + 127) / 128;
    const uint32_t xs = smem_u32(smem), ring = xs + kTileStages * kTileXBytes + warp * kTileStages * kStageBytes;
    uint8_t* xs_ptr = smem;
    pdl_wait();
    // 16 bytes of a column (8 values): column `col`, piece `c` of 16
    auto x_at = [](int col, int c) { return (uint32_t)(col * 256 + (c ^ ((col & 1) << 2)) * 16); };
    auto load = [&](int b, int slot) {
        for (int i = threadIdx.x; i < kTileCols * 16; i += 256) {
            const int col = i >> 4, c = i & 15, k = b * 128 + c * 8, m = m0 + col / P;
            if (XT == DT_F32)
                *reinterpret_cast<uint4*>(xs_ptr + slot * kTileXBytes + x_at(col, c)) = col < kTokens * P ? x_words<XT>(p, m0 * P + col, k) : make_uint4(0, 0, 0, 0);
            else {
                const bool valid = m < p.M && k < p.K;
                cp_async16(xs + slot * kTileXBytes + x_at(col, c), valid ? reinterpret_cast<const uint16_t*>(p.x) + m * p.x_stride + k : p.x, valid);
            }
        }
        load_stage(p, ring + slot * kStageBytes, n0, b, lane);
    };
#pragma unroll
    for (int i = 0; i < kTileStages - 1; ++i) {
        if (i < blocks) load(i, i);
        cp_async_commit();
    }
    float total[8][4] = {};
    Groups<GB> gr;
    gr.load(p, n0, 0, lane);
    int slot = 0;
    for (int b = 0; b < blocks; ++b) {
        cp_async_wait<kTileStages - 2>();
        __syncthreads();
        if (b + kTileStages - 1 < blocks) load(b + kTileStages - 1, slot == 0 ? kTileStages - 1 : slot - 1);
        cp_async_commit();
        const uint32_t at = ring + slot * kStageBytes;
        uint32_t w[2][4];
#pragma unroll
        for (int c = 0; c < 2; ++c) ldmatrix4(w[c], at + stage_at((lane & 7) + (lane & 8), 2 * c + (lane >> 4)));
        float sum[8][4] = {};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int grp = c * GB / 4;
            uint32_t lo[4], hi[4];
            Nibbles<T>(gr.z[grp][0]).expand(w[c >> 1][(c & 1) * 2], lo);
            Nibbles<T>(gr.z[grp][1]).expand(w[c >> 1][(c & 1) * 2 + 1], hi);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint4 x = *reinterpret_cast<const uint4*>(xs_ptr + slot * kTileXBytes + x_at(j * 8 + g, c * 4 + t));
                mma16816<T>(sum[j], lo[0], hi[0], lo[1], hi[1], x.x, x.y);
                mma16816<T>(sum[j], lo[2], hi[2], lo[3], hi[3], x.z, x.w);
            }
            if ((c + 1) * GB % 4 == 0) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < 4; ++i) total[j][i] = __fmaf_rn(gr.s[grp][i >> 1], sum[j][i], total[j][i]), sum[j][i] = 0.f;
            }
        }
        if (b + 1 < blocks) gr.load(p, n0, b + 1, lane);
        slot = slot + 1 == kTileStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncthreads();
    // [column][row] of the tile, a row of 132 floats
    float* red = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[(j * 8 + t * 2 + (i & 1)) * 132 + warp * 16 + g + (i >> 1) * 8] = total[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < kTokens * 128; i += 256) {
        const int r = i & 127, m = i >> 7, n = nt * 128 + r;
        if (n >= p.N || m0 + m >= p.M) continue;
        float y = 0.f;
#pragma unroll
        for (int q = 0; q < P; ++q) y += red[(m * P + q) * 132 + r];
        store_out(p, y, m0 + m, n);
    }
}

template <int XT, int GB> int launch_w4(W4Params& p, cudaStream_t st) {
    const int cols = p.M * parts_of<XT>();
    if (cols > 16) {
        const size_t smem = kTileStages * (kTileXBytes + 8 * kStageBytes);
        auto kern = w4_tile_kernel<XT, GB>;
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return (int)e;
        const int tokens = kTileCols / parts_of<XT>();
        const int64_t grid = (int64_t)((p.N + 127) / 128) * ((p.M + tokens - 1) / tokens);
        if (grid > INT32_MAX) return -1;
        return launch_pdl(kern, dim3((unsigned)grid), 256, smem, st, p);
    }
    // the fewest warps to a tile that still give the device eight warps an SM
    const int tiles = (p.N + 15) / 16;
    p.splits = 1;
    while (p.splits < kRowsWarps && tiles * p.splits < 148 * 8) p.splits *= 2;
    const int per = kRowsWarps / p.splits;
    const int NT = cols > 8 ? 2 : 1;
    const size_t smem = kRowsWarps * (kRowsStages * kStageBytes + NT * 8 * 16 * 4);
    auto kern = NT == 1 ? w4_rows_kernel<XT, 1, GB> : w4_rows_kernel<XT, 2, GB>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) return (int)e;
    return launch_pdl(kern, dim3((tiles + per - 1) / per), kRowsWarps * 32, smem, st, p);
}
template <int XT> int launch_w4_groups(W4Params& p, cudaStream_t st) {
    return p.G == 32 ? launch_w4<XT, 4>(p, st) : p.G == 64 ? launch_w4<XT, 2>(p, st) : launch_w4<XT, 1>(p, st);
}

// ---- the packer and its inverse -----------------------------------------------------------------------------------------------------

// Eight neighbouring values in f32
template <typename T> __device__ __forceinline__ void load8(const T* src, float (&v)[8]) {
    const uint4 r = gload(reinterpret_cast<const uint4*>(src));
    const T* h = reinterpret_cast<const T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f<T>(h[i]);
}
template <> __device__ __forceinline__ void load8<float>(const float* src, float (&v)[8]) {
    const float4 a = gload(reinterpret_cast<const float4*>(src)), b = gload(reinterpret_cast<const float4*>(src) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}

// A thread packs 16 values (8 bytes of codes); a group's 2 to 16 threads are neighbours in a warp. Bound by the weight's bytes: one read,
// a quarter (bf16) written.
template <typename T> __global__ void __launch_bounds__(256) w4_requant_kernel(const T* w, int64_t w_stride, uint8_t* packed, int scale_dt, void* scales,
                                                                                uint8_t* zeros, int64_t N, int K, int G) {
    pdl_wait();
    const int per_row = K / 16, per_group = G / 16, groups = K / G;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool live = i < N * per_row;             // K % G == 0 and 256 % per_group == 0: a group's threads are live together
    const int64_t n = live ? i / per_row : 0;
    const int at = live ? (int)(i % per_row) : 0;
    float v[2][8];
    load8(w + n * w_stride + at * 16, v[0]);
    load8(w + n * w_stride + at * 16 + 8, v[1]);
    float lo = 0.f, hi = 0.f;                      // NaN is passed over
#pragma unroll
    for (int j = 0; j < 16; ++j) lo = fminf(lo, v[j >> 3][j & 7]), hi = fmaxf(hi, v[j >> 3][j & 7]);
    for (int o = 1; o < per_group; o <<= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    float s = zeros ? __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f) : __fmul_rn(fmaxf(-lo, hi), 1.f / 7.f);
    // the scale as it is stored, at most the type's largest number; the codes are fitted to that
    s = scale_dt == DT_F16 ? rnd<half>(fminf(s, 65504.f)) : rnd<bf16>(fminf(s, 3.3895313892515355e38f));
    const float z = zeros ? (s > 0.f ? fminf(15.f, fmaxf(0.f, rintf(__fdiv_rn(-lo, s)))) : 0.f) : 8.f;
    uint32_t word[2] = {};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float c = __fadd_rn(s > 0.f ? rintf(__fdiv_rn(v[j >> 3][j & 7], s)) : 0.f, z);
        word[j >> 3] |= (uint32_t)fminf(15.f, fmaxf(0.f, c)) << 4 * (j & 7);
    }
    if (!live) return;
    reinterpret_cast<uint2*>(packed)[i] = make_uint2(word[0], word[1]);
    if (at % per_group == 0) {
        const int64_t gi = n * groups + at / per_group;
        if (scale_dt == DT_F16) reinterpret_cast<half*>(scales)[gi] = __float2half_rn(s);
        else reinterpret_cast<bf16*>(scales)[gi] = __float2bfloat16_rn(s);
        if (zeros) zeros[gi] = (uint8_t)z;
    }
}

template <typename T> __global__ void __launch_bounds__(256) w4_dequant_kernel(const uint8_t* packed, int scale_dt, const void* scales, const uint8_t* zeros,
                                                                                T* out, int64_t N, int K, int G) {
    pdl_wait();
    const int per_row = K / 8, groups = K / G;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= N * per_row) return;
    const int64_t gi = i / per_row * groups + (i % per_row) * 8 / G;
    const uint32_t w = gload(reinterpret_cast<const uint32_t*>(packed) + i);
    const float s = scale_at(scales, scale_dt, gi);
    const int z = zeros ? gload(zeros + gi) & 15 : 8;
    __align__(16) T v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = from_f<T>(__fmul_rn((float)((int)(w >> 4 * j & 15u) - z), s));
#pragma unroll
    for (int j = 0; j < (int)sizeof(T) / 2; ++j) reinterpret_cast<uint4*>(out + i * 8)[j] = reinterpret_cast<const uint4*>(v)[j];
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool bad_groups(int64_t N, int K, int G) { return N < 0 || K <= 0 || (G != 32 && G != 64 && G != 128 && G != 256) || K % G != 0; }
bool bad_scales(int dt) { return dt != DT_F16 && dt != DT_BF16; }

}  // namespace

GPU_API int gpu_w4_requant(int dtype, const void* w, int64_t w_stride, void* packed, int scale_dt, void* scales, void* zeros, int64_t N, int K, int G,
                           void* stream) {
    if (bad_groups(N, K, G)) return -1;
    if (bad_scales(scale_dt) || dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N == 0) return 0;
    const int item = dtype == DT_F32 ? 4 : 2;
    if (!w || !packed || !scales || !aligned16(w) || w_stride * item % 16 != 0 || w_stride < K || (reinterpret_cast<uintptr_t>(packed) & 7)) return -5;
    const int64_t grid = (N * (K / 16) + 255) / 256;
    if (grid > INT32_MAX) return -1;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32)
        return launch_pdl(w4_requant_kernel<float>, dim3((unsigned)grid), 256, 0, st, (const float*)w, w_stride, (uint8_t*)packed, scale_dt, scales, (uint8_t*)zeros, N, K, G);
    if (dtype == DT_F16)
        return launch_pdl(w4_requant_kernel<half>, dim3((unsigned)grid), 256, 0, st, (const half*)w, w_stride, (uint8_t*)packed, scale_dt, scales, (uint8_t*)zeros, N, K, G);
    return launch_pdl(w4_requant_kernel<bf16>, dim3((unsigned)grid), 256, 0, st, (const bf16*)w, w_stride, (uint8_t*)packed, scale_dt, scales, (uint8_t*)zeros, N, K, G);
}

GPU_API int gpu_w4_dequant(int dtype, const void* packed, int scale_dt, const void* scales, const void* zeros, void* out, int64_t N, int K, int G,
                           void* stream) {
    if (bad_groups(N, K, G)) return -1;
    if (bad_scales(scale_dt) || dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N == 0) return 0;
    if (!packed || !scales || !out || !aligned16(out) || (reinterpret_cast<uintptr_t>(packed) & 3)) return -5;
    const int64_t grid = (N * (K / 8) + 255) / 256;
    if (grid > INT32_MAX) return -1;
    cudaStream_t st = (cudaStream_t)stream;
    const uint8_t *q = (const uint8_t*)packed, *z = (const uint8_t*)zeros;
    if (dtype == DT_F32) return launch_pdl(w4_dequant_kernel<float>, dim3((unsigned)grid), 256, 0, st, q, scale_dt, scales, z, (float*)out, N, K, G);
    if (dtype == DT_F16) return launch_pdl(w4_dequant_kernel<half>, dim3((unsigned)grid), 256, 0, st, q, scale_dt, scales, z, (half*)out, N, K, G);
    return launch_pdl(w4_dequant_kernel<bf16>, dim3((unsigned)grid), 256, 0, st, q, scale_dt, scales, z, (bf16*)out, N, K, G);
}

GPU_API int gpu_w4_linear(int dtype, const void* x, int64_t x_stride, const void* Wq4, int scale_dt, const void* scales, const void* zeros, const void* bias,
                          int out_dt, void* out, int64_t out_stride, float beta, int M, int N, int K, int G, void* stream) {
    if (bad_groups(N, K, G) || M < 0) return -1;
    if (bad_scales(scale_dt) || dtype < DT_F32 || dtype > DT_BF16 || (out_dt != dtype && out_dt != DT_F32)) return -4;
    if (beta != 0.f && beta != 1.f) return -207;
    if (M == 0 || N == 0) return 0;
    const int item = dtype == DT_F32 ? 4 : 2;
    if (!x || !Wq4 || !scales || !out || !aligned16(x) || !aligned16(Wq4) || x_stride * item % 16 != 0 || (M > 1 && (x_stride < K || out_stride < N))) return -5;
    W4Params p{x, x_stride, (const uint8_t*)Wq4, scales, (const uint8_t*)zeros, bias, out, out_stride, M, N, K, G, scale_dt, out_dt, K / G, beta, 1};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return launch_w4_groups<DT_F32>(p, st);
    if (dtype == DT_F16) return launch_w4_groups<DT_F16>(p, st);
    return launch_w4_groups<DT_BF16>(p, st);
}
