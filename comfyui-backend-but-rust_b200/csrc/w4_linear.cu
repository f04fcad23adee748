// Linears with 4-bit weights and group scales (no counterpart in the reference, whose smallest weight has 6 bits and int8 activations;
// its text encoders keep their activations in floating point beside weight-only int8, src/te.rs:493-511, which is the use here).
//
//   gpu_w4_requant   f32 / f16 / bf16 weight -> codes, group scales, zero points
//   gpu_w4_dequant   the way back
//   gpu_w4_linear    out = beta * out + x . W^T + bias straight from the codes
//
// W[n, k] = (c[n, k] - z[n, k/G]) * s[n, k/G] with c and z in 0..15 (z = 8 without zero points). Codes [N, K/2]: column 2i in the low
// nibble of byte i, 2i + 1 in the high one (the order of the W6 format's nibble plane).
#include "w4.cuh"

namespace {

using namespace b200q;

// ---- the linear -------------------------------------------------------------------------------------------------------------------

// A stage: 128 columns of 16 rows, 64 bytes a row. Eight rows read at the same column have to lie in eight different 16-byte banks: two
// rows fill a line of 128 bytes, and the pair's number turns the column's.
constexpr int kStageBytes = 16 * 64;
__device__ __forceinline__ uint32_t stage_at(int row, int c) { return (uint32_t)(row * 64 + ((c ^ (row >> 1)) & 3) * 16); }

// The 4-byte words that `bytes` bytes at src lie in, every step-th from word j on. (A word with one byte of an array in it is in memory.)
__device__ __forceinline__ void copy_words(uint32_t dst, const uint8_t* src, int bytes, int j, int step) {
    const int before = (int)(reinterpret_cast<uintptr_t>(src) & 3);
    for (; j * 4 < before + bytes; j += step) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst + j * 4), "l"(src - before + j * 4) : "memory");
}
// cp.async.wait_group for a number known at run time (0 to 3)
__device__ __forceinline__ void cp_async_wait_all_but(int n) {
    if (n >= 3) cp_async_wait<3>();
    else if (n == 2) cp_async_wait<2>();
    else if (n == 1) cp_async_wait<1>();
    else cp_async_wait<0>();
}

// Few columns (at most 8 NT): bound by the weight's bytes. A CTA of eight warps has 256 / kw rows, 32 to a warp, and a share of K, which kw
// warps divide among them; the CTAs of a cluster share a row tile, and all sums of a row meet at the end in one another's shared memory, in a
// fixed order. A warp keeps ST - 1 stages of its own rows in flight (nothing is shared, so nothing waits for another warp). x, the scales
// and the zero points of the CTA's share of K are brought into shared memory once, x in the order in which codes come out of a word. Each
// group's sum is in f32 and added to the total times its scale. Measured: 1 x 2560 -> 19456 bf16 10.8 us (25.7 MB: 3.9 at the DRAM's rate; some 4
// are the loop, the rest its beginning and end), 8 x 9728 -> 2560 13.5, 16 x 5120 -> 13824 fp16 27, 5 x 9728 -> 2563 f32 18.
constexpr int kRowsStages = 4, kRowsWarps = 8, kRowsStage = 2 * kStageBytes;

inline int log2_of(int v) { return v <= 1 ? 0 : 1 + log2_of(v >> 1); }
inline RowsShare rows_share(int K, int G, int splits, int kw, int cols, bool zeros) {
    RowsShare r;
    r.kw = kw, r.kw_log = log2_of(kw), r.rows = kRowsWarps * 32 / kw, r.rows_log = 8 - r.kw_log, r.splits_log = log2_of(splits);
    static_assert(kRowsWarps * 32 == 256, "rows_log");
    r.blocks = ((K + 127) / 128 + splits - 1) / splits;
    const int per_warp = (r.blocks + kw - 1) / kw;
    r.stages = per_warp < 2 ? 2 : per_warp < kRowsStages ? per_warp : kRowsStages;
    r.x_pitch = r.blocks * 256 + 64;         // two columns side by side lie in different halves of the banks
    const int groups = (r.blocks * 128 + G - 1) / G + 1;
    r.scale_words = (groups * 2 + 5) / 4 | 1, r.zero_words = (groups + 6) / 4 | 1;      // odd: rows start in different banks
    r.scales = kRowsWarps * r.stages * kRowsStage + cols * r.x_pitch;
    r.smem = r.scales + r.rows * (r.scale_words + (zeros ? r.zero_words : 0)) * 4;
    const int sums = kRowsWarps * 32 * cols * 4;
    if (r.smem < sums) r.smem = sums;
    return r;
}

template <int XT, int NT, int GB, bool ZP> __global__ void __launch_bounds__(kRowsWarps * 32, NT == 1 ? 4 : 2) w4_rows_kernel(const W4Params p) {
    using T = typename XType<XT>::Mma;
    constexpr int P = parts_of<XT>(), kThreads = kRowsWarps * 32;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const RowsShare sh = p.share;
    const int kw = sh.kw, wk = warp & (kw - 1), row0 = (warp >> sh.kw_log) * 32;
    const int S = p.splits, split = blockIdx.x & (S - 1), tile0 = (int)(blockIdx.x >> sh.splits_log) << sh.rows_log, n0 = tile0 + row0;
    const int used = p.M * P;
    const int all_blocks = (p.K + 127) >> 7, cta_first = min(split * sh.blocks, all_blocks), cta_n = min(sh.blocks, all_blocks - cta_first);
    const int per = (cta_n + kw - 1) >> sh.kw_log, mine = min(wk * per, cta_n), first = cta_first + mine, n = min(per, cta_n - mine);
    const uint32_t ring = smem_u32(smem) + warp * sh.stages * kRowsStage;
    uint8_t* xs = smem + kRowsWarps * sh.stages * kRowsStage;
    const int shift = p.group_shift, group0 = cta_first * 4 >> shift, here = min((cta_n * 4 >> shift) + 1, p.groups - group0);
    const uint8_t* scales = smem + sh.scales;
    const uint8_t* zeros = scales + sh.rows * sh.scale_words * 4;
    // This lane's pieces of a stage: 16 bytes (32 columns) of rows lane / 4 + 8 i. Rows that there are not repeat the last one; nothing of
    // them is stored. Columns behind K are zeros.
    const uint8_t* src[4];
    uint32_t dst[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = i * 8 + (lane >> 2);
        src[i] = p.W + (int64_t)min(n0 + row, p.N - 1) * (p.K >> 1) + first * 64 + (lane & 3) * 16;
        dst[i] = ring + (row >> 4) * kStageBytes + stage_at(row & 15, lane & 3);
    }
    const int tail = p.K - first * 128 - (lane & 3) * 32;      // columns from this lane's piece of block 0 on
    auto load = [&](int b, int slot) {
        const bool valid = b * 128 < tail;
#pragma unroll
        for (int i = 0; i < 4; ++i) cp_async16(dst[i] + slot * kRowsStage, valid ? src[i] + b * 64 : p.W, valid);
    };
    pdl_wait();
    {   // scales and zero points of a row as the words that they lie in; kw threads to a row
        const int row = threadIdx.x >> sh.kw_log, j0 = threadIdx.x & (kw - 1);
        const int64_t at = (int64_t)min(tile0 + row, p.N - 1) * p.groups + group0;
        copy_words(smem_u32(scales) + row * sh.scale_words * 4, reinterpret_cast<const uint8_t*>(p.scales) + at * 2, here * 2, j0, kw);
        if (ZP) copy_words(smem_u32(zeros) + row * sh.zero_words * 4, p.zeros + at, here, j0, kw);
    }
    const int pieces = cta_n * 16, all_pieces = p.M * pieces;      // eight columns of a token each
    const float per_piece = 1.f / (float)max(pieces, 1);
    if (XT != DT_F32)
        for (int i = threadIdx.x; i < all_pieces; i += kThreads) {
            const int m = (int)(((float)i + 0.5f) * per_piece), c = i - m * pieces, k = cta_first * 128 + c * 8;      // exact: i < 2^22
            const bool valid = k < p.K;
            cp_async16(smem_u32(xs) + m * sh.x_pitch + c * 16, valid ? reinterpret_cast<const uint16_t*>(p.x) + m * p.x_stride + k : p.x, valid);
        }
    cp_async_commit();
    const int stages = sh.stages;
    for (int i = 0; i < stages - 1; ++i) {
        if (i < n) load(i, i);
        cp_async_commit();
    }
    if (XT == DT_F32) {      // three terms each, four pieces requested at a time
        constexpr int kBatch = 4;
        for (int i0 = threadIdx.x; i0 < all_pieces; i0 += kBatch * kThreads) {
            uint4 v[kBatch][P];
            int m[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kThreads;
                m[u] = i < all_pieces ? (int)(((float)i + 0.5f) * per_piece) : p.M;
                x_words<XT>(p, m[u], cta_first * 128 + (i - m[u] * pieces) * 8, v[u]);
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u)
                if (m[u] < p.M)
#pragma unroll
                    for (int q = 0; q < P; ++q) *reinterpret_cast<uint4*>(xs + (m[u] * P + q) * sh.x_pitch + (i0 + u * kThreads - m[u] * pieces) * 16) = v[u][q];
        }
    }
    cp_async_wait_all_but(stages - 1);
    __syncthreads();
    float total[2][NT][4] = {};
    const uint8_t* x_col[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) x_col[j] = xs + min(j * 8 + g, used - 1) * sh.x_pitch + mine * 256 + t * 16;
    // where the scales (and zero points) of this lane's four rows begin; a group of a row is so many values on
    const uint8_t *s_row[4], *z_row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row0 + i * 8 + g;
        const int64_t at = (int64_t)min(tile0 + row, p.N - 1) * p.groups + group0;
        s_row[i] = scales + row * sh.scale_words * 4 + ((int)reinterpret_cast<uintptr_t>(reinterpret_cast<const uint8_t*>(p.scales) + at * 2) & 3);
        if (ZP) z_row[i] = zeros + row * sh.zero_words * 4 + ((int)reinterpret_cast<uintptr_t>(p.zeros + at) & 3);
    }
    auto scale = [&](int i, int grp) {
        const uint16_t b = *reinterpret_cast<const uint16_t*>(s_row[i] + grp * 2);
        return p.scale_dt == DT_F16 ? __half2float(__ushort_as_half(b)) : __uint_as_float((uint32_t)b << 16);
    };
    const uint32_t frag = stage_at(lane & 15, lane >> 4), frag2 = stage_at(lane & 15, 2 + (lane >> 4));
    const uint32_t bits = held<Nibbles<T>::kBits>();
    int slot = 0;
    for (int b = 0; b < n; ++b) {
        cp_async_wait_all_but(stages - 2);
        __syncwarp();
        const uint32_t at = ring + slot * kRowsStage;
        constexpr int kChains = NT <= 2 && GB < 4 ? 2 : 1;      // sums of a group side by side: a product waits for the one before it
        float sum[2][NT][kChains][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {      // 64 columns
            uint32_t w[2][4];              // [16 rows][row half, column quarter]
#pragma unroll
            for (int r = 0; r < 2; ++r) ldmatrix4(w[r], at + r * kStageBytes + (h ? frag2 : frag));
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int grp = min(((first + b) * 4 + h * 2 + c >> shift) - group0, here - 1);      // columns behind K: x is zeros
                uint4 x[NT];
#pragma unroll
                for (int j = 0; j < NT; ++j) {      // columns 0..7 -> 0, 4, 1, 5, 2, 6, 3, 7
                    const uint4 v = *reinterpret_cast<const uint4*>(x_col[j] + b * 256 + (h * 2 + c) * 64);
                    x[j] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
                }
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    uint32_t lo[4], hi[4];
                    Nibbles<T>(ZP ? z_row[r * 2][grp] & 15u : 8u).expand4(w[r][c * 2], lo, bits);
                    Nibbles<T>(ZP ? z_row[r * 2 + 1][grp] & 15u : 8u).expand4(w[r][c * 2 + 1], hi, bits);
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const bool begins = (h * 2 + c) * GB % 4 == 0;
                        if (begins) mma16816_first<T>(sum[r][j][0], lo[0], hi[0], lo[1], hi[1], x[j].x, x[j].y);
                        else mma16816<T>(sum[r][j][0], lo[0], hi[0], lo[1], hi[1], x[j].x, x[j].y);
                        if (begins && kChains > 1) mma16816_first<T>(sum[r][j][kChains - 1], lo[2], hi[2], lo[3], hi[3], x[j].z, x[j].w);
                        else mma16816<T>(sum[r][j][kChains - 1], lo[2], hi[2], lo[3], hi[3], x[j].z, x[j].w);
                    }
                    if ((h * 2 + c + 1) * GB % 4 == 0) {
                        const float s[2] = {scale(r * 2, grp), scale(r * 2 + 1, grp)};
#pragma unroll
                        for (int j = 0; j < NT; ++j)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                total[r][j][i] = __fmaf_rn(s[i >> 1], kChains > 1 ? sum[r][j][0][i] + sum[r][j][kChains - 1][i] : sum[r][j][0][i], total[r][j][i]);
                    }
                }
            }
        }
        __syncwarp();
        if (b + stages - 1 < n) load(b + stages - 1, slot == 0 ? stages - 1 : slot - 1);
        cp_async_commit();
        slot = slot + 1 == stages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
    __syncthreads();
    float* red = reinterpret_cast<float*>(smem);       // [warp along K][column][row], over the rings
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (j * 8 + t * 2 + (i & 1) < used) red[(wk * used + j * 8 + t * 2 + (i & 1)) * sh.rows + row0 + r * 16 + g + (i >> 1) * 8] = total[r][j][i];
    if (S > 1) cluster_sync_all();
    else __syncthreads();
    const uint32_t red_at = smem_u32(red);
    const int rows = sh.rows >> sh.splits_log, rows_log = sh.rows_log - sh.splits_log;      // each CTA of the cluster finishes its share of the rows
    for (int i = threadIdx.x; i < rows * p.M; i += kThreads) {
        const int r = split * rows + (i & (rows - 1)), m = i >> rows_log;
        float y = 0.f;
        if (S == 1) {
#pragma unroll 4
            for (int w = 0; w < kw; ++w)
#pragma unroll
                for (int q = 0; q < P; ++q) y += red[((w * used + m * P + q) << sh.rows_log) + r];
        } else
            for (int s = 0; s < S; ++s)
#pragma unroll 4
                for (int w = 0; w < kw; ++w)
#pragma unroll
                    for (int q = 0; q < P; ++q) y += dsmem_f32(red_at + (((w * used + m * P + q) << sh.rows_log) + r) * 4, s);
        if (tile0 + r < p.N) store_out(p, y * Nibbles<T>::kUp, m, tile0 + r);
    }
    if (S > 1) cluster_sync_all();                     // nobody leaves while its sums are read
}

template <int XT, int GB> int launch_w4(W4Params& p, cudaStream_t st) {
    if (p.M > 32 / parts_of<XT>()) return w4_tile(XT, p, st);      // before what is counted in 32 bits for few columns
    const int cols = p.M * parts_of<XT>();
    // CTAs along K (a cluster): as few as leave a CTA's share of x and its rings in shared memory. Warps along K in all: four to an SM as long
    // as each has two blocks of K, and up to 32 where each keeps as many blocks as there are columns, so that bringing x in costs less than
    // the weight. Warps along K in a CTA x CTAs, us:
    //   1 x 2560 -> 19456 bf16      1x4 14.4   2x2 13.8   4x1 13.0   8x1 12.0
    //   8 x 9728 -> 2560 bf16       1x4 25.3   1x8 16.1   2x4 14.9   4x2 14.2   8x2 18.7   4x4 19.0
    //   5 x 9728 -> 2563 f32        1x8 21.8   2x4 20.7   4x4 30.5
    //   16 x 5120 -> 13824 f16      1x2 25.8   2x2 31.3   1x4 33.0   2x4 30.6
    const int all = (p.K + 127) / 128, slices = (p.N + 31) / 32;
    auto smem_of = [&](int splits, int kw) { return rows_share(p.K, p.G, splits, kw, cols, p.zeros != nullptr).smem; };
    int ksplit = 1;
    while (ksplit < 64 && ((slices * ksplit < 148 * 4 && all >= ksplit * 4) || (slices * ksplit < 148 * 32 && all >= ksplit * 2 * max(2, cols)))) ksplit *= 2;
    p.splits = 1;
    while (p.splits < 8 && (ksplit > p.splits * 8 || smem_of(p.splits, max(1, ksplit / p.splits)) > 200 * 1024)) p.splits *= 2;
    const int kw = max(1, ksplit / p.splits);
    const int tiles = (p.N + 256 / kw - 1) / (256 / kw);
    const RowsShare sh = p.share = rows_share(p.K, p.G, p.splits, kw, cols, p.zeros != nullptr);
    if (sh.smem <= 224 * 1024) {
        auto kern = p.zeros ? (cols <= 8 ? w4_rows_kernel<XT, 1, GB, true> : cols <= 16 ? w4_rows_kernel<XT, 2, GB, true> : cols <= 24 ? w4_rows_kernel<XT, 3, GB, true>
                                                                                                                         : w4_rows_kernel<XT, 4, GB, true>)
                            : (cols <= 8 ? w4_rows_kernel<XT, 1, GB, false> : cols <= 16 ? w4_rows_kernel<XT, 2, GB, false> : cols <= 24 ? w4_rows_kernel<XT, 3, GB, false>
                                                                                                                           : w4_rows_kernel<XT, 4, GB, false>);
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) return (int)e;
        return launch_pdl_cluster(kern, dim3((unsigned)(tiles * p.splits)), kRowsWarps * 32, sh.smem, st, p.splits, p);
    }
    return w4_tile(XT, p, st);
}
template <int XT> int launch_w4_groups(W4Params& p, cudaStream_t st) {
    return p.G == 32 ? launch_w4<XT, 4>(p, st) : p.G == 64 ? launch_w4<XT, 2>(p, st) : launch_w4<XT, 1>(p, st);
}

// ---- the packer and its inverse -----------------------------------------------------------------------------------------------------

// Word e of values side by side
__device__ __forceinline__ uint32_t bits32(const float* v, int e) { return __float_as_uint(v[e]); }
__device__ __forceinline__ uint32_t bits32(const half* v, int e) { return (uint32_t)__half_as_ushort(v[2 * e]) | (uint32_t)__half_as_ushort(v[2 * e + 1]) << 16; }
__device__ __forceinline__ uint32_t bits32(const bf16* v, int e) { return (uint32_t)__bfloat16_as_ushort(v[2 * e]) | (uint32_t)__bfloat16_as_ushort(v[2 * e + 1]) << 16; }

// A thread packs 16 values (8 bytes of codes); a group's 2 to 16 threads are neighbours in a warp. Bound by the weight's bytes (one read, a
// quarter of bf16 written) once the codes are not sixteen divisions: those took 533 instructions a warp and 141 us at 13824 x 5120 bf16.
template <typename T> __global__ void __launch_bounds__(256) w4_requant_kernel(const T* w, int64_t w_stride, uint8_t* packed, int scale_dt, void* scales,
                                                                                uint8_t* zeros, uint32_t threads, int K, int group_log) {
    pdl_wait();
    const uint32_t per_row = K / 16, i = blockIdx.x * 256u + threadIdx.x;
    const int per_group = 1 << (group_log - 4);
    const bool live = i < threads;                 // K % G == 0 and 256 % per_group == 0: a group's threads are live together
    const uint32_t n = live ? i / per_row : 0, at = live ? i - n * per_row : 0;
    float v[16];
    load8(w + n * w_stride + at * 16, reinterpret_cast<float(&)[8]>(v[0]));
    load8(w + n * w_stride + at * 16 + 8, reinterpret_cast<float(&)[8]>(v[8]));
    float lo = 0.f, hi = 0.f;                      // NaN is passed over
#pragma unroll
    for (int j = 0; j < 16; ++j) lo = fminf(lo, v[j]), hi = fmaxf(hi, v[j]);
    for (int o = 1; o < per_group; o <<= 1) lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    float s = zeros ? __fmul_rn(__fsub_rn(hi, lo), 1.f / 15.f) : __fmul_rn(fmaxf(-lo, hi), 1.f / 7.f);
    // the scale as it is stored, at most the type's largest number; the codes are fitted to that
    s = scale_dt == DT_F16 ? rnd<half>(fminf(s, 65504.f)) : rnd<bf16>(fminf(s, 3.3895313892515355e38f));
    const float z = zeros ? (s > 0.f ? fminf(15.f, fmaxf(0.f, rintf(__fdiv_rn(-lo, s)))) : 0.f) : 8.f;
    float q[16];
    rint_quotients<16>(v, s, q);
    uint32_t word[2] = {};
#pragma unroll
    for (int j = 0; j < 16; ++j) {                 // 2^23 + code: the code in the low bits
        const float c = __fadd_rn(fminf(15.f, fmaxf(0.f, __fadd_rn(q[j], z))), 8388608.f);
        word[j >> 3] |= (__float_as_uint(c) & 15u) << 4 * (j & 7);
    }
    if (!live) return;
    reinterpret_cast<uint2*>(packed)[i] = make_uint2(word[0], word[1]);
    if ((i & (per_group - 1)) == 0) {              // rows are whole groups: the i-th thread's group, counted through
        const uint32_t gi = i >> (group_log - 4);
        if (scale_dt == DT_F16) reinterpret_cast<half*>(scales)[gi] = __float2half_rn(s);
        else reinterpret_cast<bf16*>(scales)[gi] = __float2bfloat16_rn(s);
        if (zeros) zeros[gi] = (uint8_t)z;
    }
}

// 32 bytes of the result a thread and store, four times a CTA's width apart. Rows are whole groups: the index counts through them.
template <typename T> __global__ void __launch_bounds__(256) w4_dequant_kernel(const uint8_t* packed, int scale_dt, const void* scales, const uint8_t* zeros,
                                                                                T* out, int64_t values, int group_log) {
    constexpr int kCodes = 32 / sizeof(T), kTimes = 4;
    pdl_wait();
    const int64_t first = ((int64_t)blockIdx.x * (256 * kTimes) + threadIdx.x) * kCodes;
    uint32_t w[kTimes][kCodes / 8];
    float s[kTimes];
    int z[kTimes];
#pragma unroll
    for (int u = 0; u < kTimes; ++u) {
        const int64_t k = first + u * 256 * kCodes;
        if (k < values) {
#pragma unroll
            for (int e = 0; e < kCodes / 8; ++e) w[u][e] = gload(reinterpret_cast<const uint32_t*>(packed + (k >> 1)) + e);
            s[u] = scale_at(scales, scale_dt, k >> group_log);
            z[u] = zeros ? gload(zeros + (k >> group_log)) & 15 : 8;
        }
    }
#pragma unroll
    for (int u = 0; u < kTimes; ++u) {
        const int64_t k = first + u * 256 * kCodes;
        if (k >= values) break;
        T v[kCodes];
#pragma unroll
        for (int j = 0; j < kCodes; ++j) v[j] = from_f<T>(__fmul_rn((float)((int)(w[u][j >> 3] >> 4 * (j & 7) & 15u) - z[u]), s[u]));
        uint32_t r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = bits32(v, e);
        store32(out + k, r);
    }
}
template <typename T> int launch_requant(const void* w, int64_t w_stride, void* packed, int scale_dt, void* scales, void* zeros, int64_t N, int K, int G, cudaStream_t st) {
    const int64_t threads = N * (K / 16);
    if (N > INT32_MAX / (K / 16)) return -1;
    auto kern = w4_requant_kernel<T>;
    return launch_pdl(kern, dim3((unsigned)((threads + 255) / 256)), 256, 0, st, (const T*)w, w_stride, (uint8_t*)packed, scale_dt, scales, (uint8_t*)zeros,
                      (uint32_t)threads, K, 5 + log2_of(G / 32));
}
template <typename T> int launch_dequant(const void* packed, int scale_dt, const void* scales, const void* zeros, void* out, int64_t N, int K, int G, cudaStream_t st) {
    const int64_t per_cta = 1024 * (32 / (int)sizeof(T));
    if (N > (int64_t)INT32_MAX * 16 / K) return -1;
    auto kern = w4_dequant_kernel<T>;
    return launch_pdl(kern, dim3((unsigned)((N * K + per_cta - 1) / per_cta)), 256, 0, st, (const uint8_t*)packed, scale_dt, scales, (const uint8_t*)zeros, (T*)out,
                      N * K, 5 + log2_of(G / 32));
}

constexpr int kMostRows = INT32_MAX - 1024;      // of x and of the weight: a tile's number and its last row fit 32 bits
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
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return launch_requant<float>(w, w_stride, packed, scale_dt, scales, zeros, N, K, G, st);
    if (dtype == DT_F16) return launch_requant<half>(w, w_stride, packed, scale_dt, scales, zeros, N, K, G, st);
    return launch_requant<bf16>(w, w_stride, packed, scale_dt, scales, zeros, N, K, G, st);
}

GPU_API int gpu_w4_dequant(int dtype, const void* packed, int scale_dt, const void* scales, const void* zeros, void* out, int64_t N, int K, int G,
                           void* stream) {
    if (bad_groups(N, K, G)) return -1;
    if (bad_scales(scale_dt) || dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N == 0) return 0;
    if (!packed || !scales || !out || (reinterpret_cast<uintptr_t>(out) & 31) || (reinterpret_cast<uintptr_t>(packed) & 3)) return -5;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return launch_dequant<float>(packed, scale_dt, scales, zeros, out, N, K, G, st);
    if (dtype == DT_F16) return launch_dequant<half>(packed, scale_dt, scales, zeros, out, N, K, G, st);
    return launch_dequant<bf16>(packed, scale_dt, scales, zeros, out, N, K, G, st);
}

GPU_API int gpu_w4_linear(int dtype, const void* x, int64_t x_stride, const void* Wq4, int scale_dt, const void* scales, const void* zeros, const void* bias,
                          int out_dt, void* out, int64_t out_stride, float beta, int M, int N, int K, int G, void* stream) {
    if (bad_groups(N, K, G) || M < 0 || M > kMostRows || N > kMostRows) return -1;
    if (bad_scales(scale_dt) || dtype < DT_F32 || dtype > DT_BF16 || (out_dt != dtype && out_dt != DT_F32)) return -4;
    if (beta != 0.f && beta != 1.f) return -207;
    if (M == 0 || N == 0) return 0;
    const int item = dtype == DT_F32 ? 4 : 2;
    if (!x || !Wq4 || !scales || !out || !aligned16(x) || !aligned16(Wq4) || x_stride * item % 16 != 0 || (M > 1 && (x_stride < K || out_stride < N))) return -5;
    W4Params p{x, x_stride, (const uint8_t*)Wq4, scales, (const uint8_t*)zeros, bias, out, out_stride, M, N, K, G, scale_dt, out_dt, K / G, beta, G == 32 ? 0 : G == 64 ? 1 : G == 128 ? 2 : 3, 1, {}};
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return launch_w4_groups<DT_F32>(p, st);
    if (dtype == DT_F16) return launch_w4_groups<DT_F16>(p, st);
    return launch_w4_groups<DT_BF16>(p, st);
}
