// Attention next to the quantized linears: cross attention to an encoder's states, and attention over a cache of int8 keys and values.
//
//   gpu_cross_attention   q rows of one sequence, k and v rows of another, 16-bit
//   gpu_kv8_attention     q rows over pages of int8 keys and values, one f32 scale for each page and head
//   gpu_packed_attention  rows of several sequences one after the other, each over its own, 16-bit
//
// o[i] = sum_t p[i, t] v[t] / sum_t p[i, t],  p[i, t] = exp(scale q[i] . k[t] - m[i]), m[i] the largest exponent seen so far; a row that sees
// no key is zeros. One pass over the keys: the sums are scaled when m grows. Exponents, m and both sums are f32; p is rounded to the type
// of the matrix product (as its operands have to be: q's for 16-bit keys, fp16 over the cache) after it entered the sum of p. That is at most
// half a step of each term, and below fp16's normal numbers at most 2^-25 of the largest p: keys far below the maximum may count in the sum of
// p and not in the result.
#include "attention.cuh"

namespace {

using namespace b200q;

// 64 query rows (a kv head's queries: row r is query r / ratio, head r % ratio of its group), 64 keys a step, four warps of 16 rows.
constexpr int kRows = 64, kKeys = 64, kThreads = 128;

template <int DP> struct Tile {
    static constexpr int kRowBytes = DP * 2, kBytes = kKeys * DP * 2;
    // Q | K, V x 2 | 0 or -inf per key x 2 | m, l of every row; the sums of the rows, f32, over K and V at the end
    static constexpr int kLoaded = kRows * kRowBytes, kKeyInfo = kLoaded + 4 * kBytes, kStats = kKeyInfo + 2 * kKeys * 4, kSmem = kStats + 2 * kRows * 4;
    static constexpr int kFrom = kSmem, kSmemPacked = kFrom + DP * 4;      // packed: for each column the first token whose row is NaN there
    static __device__ __forceinline__ uint32_t at(int row, int c) { return (uint32_t)(row * kRowBytes + ((c ^ (row & 7)) * 16)); }
};

template <typename T, int DP, bool PACKED> __global__ void __launch_bounds__(kThreads) attention_tile_kernel(const AttnParams p) {
    using L = Tile<DP>;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % p.splits, rt = blockIdx.x / p.splits % p.row_tiles, bh = blockIdx.x / p.splits / p.row_tiles;
    const int D = p.D, chunks = DP / 8;
    pdl_wait();
    // packed: the last tiles of a sequence, which have most keys, first
    const PackedTile x = PACKED ? packed_tile(p, p.row_tiles - 1 - rt) : PackedTile();
    if (PACKED && x.tokens == 0) return;
    const int b = PACKED ? 0 : bh / p.Hkv, ratio = PACKED ? p.pack : p.H / p.Hkv, group = PACKED ? bh : bh % p.Hkv;      // group: of `ratio` heads
    const int kvh = PACKED ? group * ratio / (p.H / p.Hkv) : group;
    const int len = PACKED ? (p.causal ? x.token0 + x.tokens : x.len) : p.kv_len ? min(max(gload(p.kv_len + b), 0), p.Lkv) : p.Lkv;
    const int r0 = PACKED ? x.token0 * ratio : rt * kRows, live = PACKED ? x.tokens * ratio : min(kRows, p.Lq * ratio - r0);    // rows of this tile that exist
    const int64_t q_at = PACKED ? x.start * p.qs[1] : b * p.qs[0], k_at = PACKED ? x.start * p.ks[1] : b * p.ks[0], v_at = PACKED ? x.start * p.vs[1] : b * p.vs[0];
    const int steps = (len + kKeys - 1) / kKeys, per = (steps + p.splits - 1) / p.splits;
    const int first = min(split * per, steps), last = min(first + per, steps);

    const uint32_t base = smem_u32(smem);
    float* key_info = reinterpret_cast<float*>(smem + L::kKeyInfo);     // [stage][key]
    // ---- queries into shared memory
    {
        const int row = tid >> 1, i = (r0 + row) / ratio, h = group * ratio + (r0 + row) % ratio;
        const T* src = reinterpret_cast<const T*>(p.q) + q_at + (int64_t)i * p.qs[1] + h * p.qs[2];
        for (int c = tid & 1; c < chunks; c += 2)
            *reinterpret_cast<uint4*>(smem + L::at(row, c)) =
                row < live && c * 8 < D ? gload(reinterpret_cast<const uint4*>(src) + c) : make_uint4(0, 0, 0, 0);
    }
    // ---- one step's keys and values on their way; what is not seen is zeros, whatever lies there
    auto load = [&](int step, int stage) {
        const uint32_t ks = base + L::kLoaded + stage * 2 * L::kBytes, vs = ks + L::kBytes;
        for (int i = tid; i < kKeys * chunks; i += kThreads) {
            const int key = i / chunks, c = i % chunks, at = step * kKeys + key;
            const bool valid = at < len && c * 8 < D && (!p.mask || gload(p.mask + b * p.mask_stride + at));
            const T* k = reinterpret_cast<const T*>(p.k) + (valid ? k_at + at * p.ks[1] + kvh * p.ks[2] + c * 8 : 0);
            const T* v = reinterpret_cast<const T*>(p.v) + (valid ? v_at + at * p.vs[1] + kvh * p.vs[2] + c * 8 : 0);
            cp_async16(ks + L::at(key, c), k, valid);
            cp_async16(vs + L::at(key, c), v, valid);
        }
        if (tid < kKeys) {
            const int at = step * kKeys + tid;
            key_info[stage * kKeys + tid] = at < len && (!p.mask || gload(p.mask + b * p.mask_stride + at)) ? 0.f : -INFINITY;
        }
    };
    float o[DP / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
    const float to_log2 = p.scale * kLog2e;
    int* from = reinterpret_cast<int*>(smem + L::kFrom);
    int bound[2] = {};          // keys that this thread's rows see
    if constexpr (PACKED) {
        for (int i = tid; i < DP; i += kThreads) from[i] = INT32_MAX;
#pragma unroll
        for (int h = 0; h < 2; ++h) bound[h] = p.causal ? (r0 + warp * 16 + g + 8 * h) / ratio + 1 : len;
    }
    if (first < last) load(first, 0);
    cp_async_commit();
    for (int step = first; step < last; ++step) {
        const int stage = (step - first) & 1;
        if (step + 1 < last) load(step + 1, stage ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        const uint32_t ks = base + L::kLoaded + stage * 2 * L::kBytes, vs = ks + L::kBytes;
        const bool mixed = PACKED && p.causal && step * kKeys + kKeys > x.token0 + 1;      // some rows see keys here that others do not
        if (mixed) {
            for (int i = tid; i < kKeys * (DP / 8); i += kThreads) {
                const int key = i / (DP / 8), c = i % (DP / 8);
                uint4* at = reinterpret_cast<uint4*>(smem + (vs - base) + L::at(key, c));
                if (any_infinite<T>(*at)) *at = without_infinite<T>(*at, step * kKeys + key, from + c * 8);
            }
            __syncthreads();
        }
        float s[8][4] = {};
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            uint32_t a[4];
            ldmatrix4(a, base + L::at(warp * 16 + (lane & 15), 2 * kk + (lane >> 4)));
#pragma unroll
            for (int n = 0; n < 8; n += 2) {
                uint32_t k4[4];
                ldmatrix4(k4, ks + L::at(n * 8 + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
                mma16816<T>(s[n], a[0], a[1], a[2], a[3], k4[0], k4[1]);
                mma16816<T>(s[n + 1], a[0], a[1], a[2], a[3], k4[2], k4[3]);
            }
        }
        const float* info = key_info + stage * kKeys;
        float top[2] = {m[0], m[1]};
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[n][i] = info[n * 8 + 2 * t + (i & 1)] == 0.f ? s[n][i] * to_log2 : -INFINITY;
                if (mixed && step * kKeys + n * 8 + 2 * t + (i & 1) >= bound[i >> 1]) s[n][i] = -INFINITY;
                top[i >> 1] = fmaxf(top[i >> 1], s[n][i]);
            }
        float keep[2], shift[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
            top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            shift[h] = top[h] == -INFINITY ? 0.f : top[h];
            keep[h] = exp2_fast(m[h] - shift[h]);
            m[h] = top[h], l[h] *= keep[h];
        }
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][i] *= keep[i >> 1];
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk) {
            uint32_t a[4];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int n = 2 * kk + j;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[n][i] = exp2_fast(s[n][i] - shift[i >> 1]);
                    l[i >> 1] += s[n][i];
                }
                a[2 * j] = pack2<T>(s[n][0], s[n][1]), a[2 * j + 1] = pack2<T>(s[n][2], s[n][3]);
            }
#pragma unroll
            for (int n = 0; n < DP / 8; n += 2) {
                uint32_t v4[4];
                ldmatrix4_t(v4, vs + L::at(kk * 16 + (lane & 15), n + (lane >> 4)));
                mma16816<T>(o[n], a[0], a[1], a[2], a[3], v4[0], v4[1]);
                mma16816<T>(o[n + 1], a[0], a[1], a[2], a[3], v4[2], v4[3]);
            }
        }
        __syncthreads();
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1), l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    // ---- rows out, by way of shared memory; with several CTAs to a row tile each finishes its share of the rows from all of them
    constexpr int kPitch = DP;
    float* part = reinterpret_cast<float*>(smem + L::kLoaded);          // [64][DP], over the loaded tiles
    float* stats = reinterpret_cast<float*>(smem + L::kStats);
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = warp * 16 + g + 8 * h;
        if (t == 0) stats[row] = m[h], stats[kRows + row] = l[h];
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2*>(part + row * kPitch + ((n ^ (g & 3)) * 8 + 2 * t)) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    const uint32_t part_at = smem_u32(part), stats_at = smem_u32(stats);
    const int pieces = (D + 7) / 8;
    for (int i = tid + split * kThreads; i < live * pieces; i += kThreads * p.splits) {
        const int row = i / pieces, n = i % pieces;
        float y[8] = {}, total = 0.f;
        if (p.splits == 1) {
            total = stats[kRows + row];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = part[row * kPitch + (n ^ (row & 3)) * 8 + e];
        } else {
            float top = -INFINITY;
            for (int s = 0; s < p.splits; ++s) top = fmaxf(top, dsmem_f32(stats_at + row * 4, s));
            for (int s = 0; s < p.splits; ++s) {
                const float w = top == -INFINITY ? 0.f : exp2_fast(dsmem_f32(stats_at + row * 4, s) - top);
                total = __fmaf_rn(dsmem_f32(stats_at + (kRows + row) * 4, s), w, total);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = __fmaf_rn(dsmem_f32(part_at + (row * kPitch + (n ^ (row & 3)) * 8 + e) * 4, s), w, y[e]);
            }
        }
        if constexpr (PACKED) {
            const int token = (r0 + row) / ratio;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (token >= from[n * 8 + e]) y[e] = NAN;
            store_piece(reinterpret_cast<T*>(p.out) + (x.start + token) * p.os[1] + (group * ratio + (r0 + row) % ratio) * p.os[2] + n * 8, y, total);
        } else store_row(p, y, total, b, r0 + row, kvh, ratio, n * 8, T());
    }
    if (p.splits > 1) cluster_sync_all();      // nobody leaves while its shared memory is read
}

template <typename T, int DP> int launch_tile(AttnParams& p, cudaStream_t st) {
    using L = Tile<DP>;
    auto kern = attention_tile_kernel<T, DP, false>;
    const int64_t rows = (int64_t)p.Lq * (p.H / p.Hkv), tiles = (rows + kRows - 1) / kRows;
    if (rows > INT32_MAX - kRows || tiles > INT32_MAX / p.B / p.Hkv) return -1;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem)) return (int)e;
    const int64_t base = tiles * p.B * p.Hkv;
    p.row_tiles = (int)tiles;
    // CTAs to a row tile: as long as the device has room for twice as many and each keeps 256 keys
    p.splits = 1;
    while (p.splits < 8 && base * p.splits * 2 <= 296 && (int64_t)p.Lkv >= (int64_t)p.splits * 2 * 256) p.splits *= 2;
    return launch_pdl_cluster(kern, dim3((unsigned)(base * p.splits)), kThreads, L::kSmem, st, p.splits, p);
}
template <typename T, int DP> int launch_packed(AttnParams& p, cudaStream_t st) {
    using L = Tile<DP>;
    auto kern = attention_tile_kernel<T, DP, true>;
    p.tile_tokens = kRows / p.pack, p.splits = 1;
    const int64_t tiles = (int64_t)p.rows / p.tile_tokens + p.B;
    if (tiles > INT32_MAX / (p.H / p.pack) || p.rows > (INT32_MAX - kRows) / p.pack) return -1;      // (rows of a tile are counted from the sequence's first)
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemPacked)) return (int)e;
    p.row_tiles = (int)tiles;
    return launch_pdl(kern, dim3((unsigned)(tiles * (p.H / p.pack))), kThreads, L::kSmemPacked, st, p);
}
// ---- rows over the cache ---------------------------------------------------------------------------------------------------------
// Tiles of 16 rows of a kv head (a token's query heads, or a few tokens'): bound by the cache's bytes. A CTA's eight warps take 16 keys each
// in turn, and every warp is on its own until the end: its ring of stages, its m, l and sums. The operands of the products come out of the
// codes as they lie in memory, because the order of a product's inner index is free as long as both operands have it: a lane multiplies 16
// neighbouring values of a key with the same 16 of its query row, and in p . v its column 16 g + j of every key stands for column g of the
// product's j-th tile. So codes are read from shared memory in 16-byte pieces and nothing is transposed. Measured (32 heads over 8 of 128): a
// token over 1999 keys 8.6 us; 16 tokens over up to 32768 keys 121 us on the same buffers again and again, 124 to 131 on new ones (4.1 to 4.3
// TB/s). 475 warp instructions to 4 KB of codes take half of the issue slots: with four warps to a scheduler 6.9 cycles pass between two of a
// warp's instructions, 2.0 of them fixed latencies, 0.8 the integer pipe (44 % busy), 0.8 the other warps' turns.
constexpr int kRowsWarps = 8, kRowsStages = 3;
constexpr float kSlack = 8.f;

template <int DP> struct RowsTile {
    static constexpr int kHalf = 16 * DP, kStage = 2 * kHalf, kRing = kRowsWarps * kRowsStages * kStage;
    static constexpr int kPitch = DP + 8;                              // floats to a row of sums
    static constexpr int kParts = kRowsWarps * 16 * kPitch * 4, kSmem0 = kParts + 16 * kPitch * 4 > kRing ? kParts + 16 * kPitch * 4 : kRing;
    static constexpr int kStats = kSmem0, kInfo = kStats + (kRowsWarps + 1) * 32 * 4, kSmem = kInfo + kRowsWarps * 64 * 16;
};

// Four int8 codes (sign bits turned) of each of two rows as four registers of halves (row a's value, row b's value)
__device__ __forceinline__ void half_pairs(uint32_t a, uint32_t b, uint32_t (&r)[4]) {
    const uint32_t off = 0x64806480u, lo = __byte_perm(a, b, 0x5140), hi = __byte_perm(a, b, 0x7362);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t v = __byte_perm(i < 2 ? lo : hi, 0x64646464u, i & 1 ? 0x4342 : 0x4140);
        const half2 h = __hsub2(*reinterpret_cast<const half2*>(&v), *reinterpret_cast<const half2*>(&off));
        r[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

template <typename QT, int DP> __global__ void __launch_bounds__(kRowsWarps * 32, DP <= 128 ? 2 : 1) kv8_rows_kernel(const AttnParams p) {
    using R = RowsTile<DP>;
    constexpr bool kBf16 = std::is_same<QT, bf16>::value;
    extern __shared__ __align__(128) uint8_t smem[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % p.splits, rt = blockIdx.x / p.splits % p.row_tiles, bh = blockIdx.x / p.splits / p.row_tiles;
    const int kvh = bh % p.Hkv, ratio = p.H / p.Hkv, D = p.D;
    int b = bh / p.Hkv;
    pdl_wait();
    if (p.B > 1 && p.B <= 32) {      // the longest sequences first: the last CTAs to run then have little to do. Every warp finds the b-th longest.
        const int mine = lane < p.B ? gload(p.kv_len + lane) : INT32_MIN;
        int rank = 0;
        for (int j = 0; j < p.B; ++j) {
            const int other = __shfl_sync(0xffffffffu, mine, j);
            rank += other > mine || (other == mine && j < lane);
        }
        b = __ffs((int)__ballot_sync(0xffffffffu, lane < p.B && rank == b)) - 1;
    }
    const int len = min(max(gload(p.kv_len + b), 0), p.Lkv);
    const int ql = p.q_len ? min(max(gload(p.q_len + b), 0), p.Lq) : p.Lq;
    const int r0 = rt * 16, live = min(16, ql * ratio - r0);
    if (live <= 0) return;                                              // the same for every CTA of the cluster
    const int seen = p.causal ? max(0, min(len, len - ql + (r0 + live - 1) / ratio + 1)) : len;
    // blocks of 16 keys: a CTA's share is at least one for each of its warps
    const int blocks = (seen + 15) / 16, per = max((blocks + p.splits - 1) / p.splits, kRowsWarps);
    const int first = min(split * per, blocks), last = min(first + per, blocks);
    const int mine = (last - first - warp + kRowsWarps - 1) / kRowsWarps;      // blocks first + warp + 8 i, i < mine
    const uint32_t ring = smem_u32(smem) + warp * kRowsStages * R::kStage;
    float4* info = reinterpret_cast<float4*>(smem + R::kInfo) + warp * 64;      // [block % 64]: factor, offset, weight of its page, and whether there is one

    // Pages of the next 32 blocks, one to a lane. Their scales are requested with the blocks and worked out behind them (note_scales).
    int64_t page_off = -1;
    float k_scale = 0.f, v_scale = 1.f;
    auto look_up = [&](int i0) {
        page_off = -1;
        const int key = (first + warp + (i0 + lane) * kRowsWarps) * 16;
        if (i0 + lane < mine) {
            const int64_t page = gload(p.table + b * p.table_stride + key / p.T);
            if (page >= 0 && page < p.pages) {
                page_off = ((page * p.Hkv + kvh) * p.T + key % p.T) * D;
                k_scale = gload(p.k_scale + page * p.Hkv + kvh), v_scale = gload(p.v_scale + page * p.Hkv + kvh);
            }
        }
    };
    auto note_scales = [&](int i0) {
        info[(i0 + lane) & 63] =
            page_off >= 0 ? make_float4(k_scale * (p.scale * kLog2e), v_scale_log2(v_scale), v_scale_weight(v_scale), 1.f) : make_float4(0.f, 0.f, 0.f, 0.f);
    };
    // 16 rows of K, then of V. K's 16-byte pieces are read four to a row by two rows at a time, V's two to a row by four pairs of rows: the
    // piece's number is turned so that either lies in all 32 banks. A lane has the same piece of every kStep-th row.
    constexpr int kPieces = DP / 16, kStep = 32 / kPieces;
    const int piece = lane % kPieces, row0 = lane / kPieces, from = row0 * D + piece * 16;
    const uint32_t to = ring + row0 * DP;
    const bool wide = piece * 16 < D;
    auto load = [&](int i, int slot) {
        const int64_t off = __shfl_sync(0xffffffffu, page_off, i & 31);
        const int left = seen - (first + warp + i * kRowsWarps) * 16;      // rows that are seen
        const uint32_t dst = to + slot * R::kStage;
        const int8_t *k = reinterpret_cast<const int8_t*>(p.k) + (off < 0 ? 0 : off + from), *v = reinterpret_cast<const int8_t*>(p.v) + (off < 0 ? 0 : off + from);
        if (left >= 16 && off >= 0 && D == DP) {
#pragma unroll
            for (int j = 0; j < 16 / kStep; ++j) {
                const int row = j * kStep;
                cp_async16(dst + row * DP + ((piece ^ (row0 & 1) << 2) & (kPieces - 1)) * 16, k + row * D, true);
                cp_async16(dst + R::kHalf + row * DP + ((piece ^ ((row + row0) & 6)) & (kPieces - 1)) * 16, v + row * D, true);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16 / kStep; ++j) {
                const int row = j * kStep;
                const bool valid = off >= 0 && wide && row + row0 < left;
                cp_async16(dst + row * DP + ((piece ^ ((row + row0) & 1) << 2) & (kPieces - 1)) * 16, valid ? k + row * D : reinterpret_cast<const int8_t*>(p.k), valid);
                cp_async16(dst + R::kHalf + row * DP + ((piece ^ ((row + row0) & 6)) & (kPieces - 1)) * 16, valid ? v + row * D : reinterpret_cast<const int8_t*>(p.v), valid);
            }
        }
    };
    float o[DP / 8][4] = {}, m[2] = {-INFINITY, -INFINITY}, l[2] = {};
    uint32_t q[DP / 16][4];
    float factor[2] = {1.f, 1.f};
    look_up(0);
#pragma unroll
    for (int i = 0; i < kRowsStages - 1; ++i) {
        if (i < mine) load(i, i);
        cp_async_commit();
    }
    note_scales(0);
    int bound[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = g + 8 * h;
        bound[h] = p.causal ? len - ql + (r0 + row) / ratio + 1 : len;
        const QT* src = reinterpret_cast<const QT*>(p.q) + b * p.qs[0] + (int64_t)((r0 + row) / ratio) * p.qs[1] + (kvh * ratio + (r0 + row) % ratio) * p.qs[2];
        uint4 w[DP / 64][2];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int d = c * 64 + t * 16 + e * 8;
                w[c][e] = row < live && d < D ? gload(reinterpret_cast<const uint4*>(src + d)) : make_uint4(0, 0, 0, 0);
                if (kBf16)
#pragma unroll
                    for (int x = 0; x < 8; ++x) top = fmaxf(top, fabsf(to_f<QT>(reinterpret_cast<const QT*>(&w[c][e])[x])));
            }
        float mult = 1.f;
        if (kBf16) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = row_exponent(top);
            mult = __uint_as_float((uint32_t)(127 + e) << 23), factor[h] = __uint_as_float((uint32_t)(127 - e) << 23);
        }
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t v = reinterpret_cast<const uint32_t*>(&w[c][j >> 1])[(j & 1) * 2 + e];
                    const QT* x = reinterpret_cast<const QT*>(&v);
                    q[c * 4 + j][2 * e + h] = kBf16 ? pack2<half>(to_f<QT>(x[0]) * mult, to_f<QT>(x[1]) * mult) : v;
                }
    }
    const int lowest = p.causal ? len - ql + r0 / ratio + 1 : len;      // keys that every row sees
    int slot = 0;
    for (int i = 0; i < mine; ++i) {
        cp_async_wait<kRowsStages - 2>();
        __syncwarp();
        const uint32_t ks = ring + slot * R::kStage, vs = ks + R::kHalf;
        const float4 in = info[i & 63];
        const int key0 = (first + warp + i * kRowsWarps) * 16;
        if (in.w != 0.f) {      // the page exists
            float s[2][4] = {};
#pragma unroll
            for (int c = 0; c < DP / 64; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int row = n * 8 + g;
                    const uint4 w = lds128(ks + row * DP + (((4 * c + t) ^ ((row & 1) << 2)) & (DP / 16 - 1)) * 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint2 k2 = halves_of4(reinterpret_cast<const uint32_t*>(&w)[j]);
                        mma16816<half>(s[n], q[c * 4 + j][0], q[c * 4 + j][1], q[c * 4 + j][2], q[c * 4 + j][3], k2.x, k2.y);
                    }
                }
            float top[2] = {m[0], m[1]};
            const bool all = key0 + 16 <= lowest;
            // the row's power with the page's factor: with the product, of up to 2^30, it may leave f32's range where the logit does not
            const float times[2] = {in.x * factor[0], in.x * factor[1]};
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int h = x >> 1;
                    s[n][x] = __fmaf_rn(s[n][x], times[h], in.y);
                    if (!all && key0 + n * 8 + 2 * t + (x & 1) >= bound[h]) s[n][x] = -INFINITY;
                    top[h] = fmaxf(top[h], s[n][x]);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
                top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
            }
            // m follows the largest exponent only when that has grown by 2^8: until then p is at most 256, and the sums stay as they are
            const bool grew[2] = {top[0] > m[0] + kSlack, top[1] > m[1] + kSlack};
            if (__any_sync(0xffffffffu, grew[0] || grew[1])) {
                float keep[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    keep[h] = grew[h] ? exp2_fast(m[h] - top[h]) : 1.f;
                    if (grew[h]) m[h] = top[h];
                    l[h] *= keep[h];
                }
#pragma unroll
                for (int n = 0; n < DP / 8; ++n)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[n][x] *= keep[x >> 1];
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    s[n][x] = exp2_fast(s[n][x] - (m[x >> 1] == -INFINITY ? 0.f : m[x >> 1]));
                    l[x >> 1] = __fmaf_rn(s[n][x], in.z, l[x >> 1]);
                }
            const uint32_t a0 = pack2<half>(s[0][0], s[0][1]), a1 = pack2<half>(s[0][2], s[0][3]), a2 = pack2<half>(s[1][0], s[1][1]), a3 = pack2<half>(s[1][2], s[1][3]);
            constexpr int kWide = DP >= 128 ? 16 : 8;      // neighbouring columns of a lane: 16 g + j, or 8 g + j
#pragma unroll
            for (int u = 0; u < DP / 8 / kWide; ++u) {
                uint32_t w[4][kWide / 4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 2 * t + (r & 1) + (r >> 1) * 8;
                    if (kWide == 16) {
                        const uint4 v = lds128(vs + row * DP + (((8 * u + g) ^ (row & 6)) & (DP / 16 - 1)) * 16);
                        w[r][0] = v.x, w[r][1] = v.y, w[r][kWide / 4 - 2] = v.z, w[r][kWide / 4 - 1] = v.w;
                    } else {
                        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[r][0]), "=r"(w[r][1])
                                     : "r"(vs + row * DP + (((g >> 1) ^ (row & 6)) & (DP / 16 - 1)) * 16 + (g & 1) * 8) : "memory");
                    }
#pragma unroll
                    for (int j = 0; j < kWide / 4; ++j) w[r][j] ^= 0x80808080u;
                }
#pragma unroll
                for (int j = 0; j < kWide / 4; ++j) {
                    uint32_t b0[4], b1[4];
                    half_pairs(w[0][j], w[1][j], b0);
                    half_pairs(w[2][j], w[3][j], b1);
#pragma unroll
                    for (int e = 0; e < 4; ++e) mma16816<half>(o[u * kWide + j * 4 + e], a0, a1, a2, a3, b0[e], b1[e]);
                }
            }
        }
        __syncwarp();
        const int ahead = i + kRowsStages - 1;
        if (ahead < mine) {
            if ((ahead & 31) == 0) look_up(ahead), note_scales(ahead);
            load(ahead, slot == 0 ? kRowsStages - 1 : slot - 1);
        }
        cp_async_commit();
        slot = slot + 1 == kRowsStages ? 0 : slot + 1;
    }
    cp_async_wait<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1), l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    // ---- the warps' sums into the CTA's, the CTAs' into the row: m, l and o of each, in this order
    __syncthreads();                                                  // every ring is done with
    float* part = reinterpret_cast<float*>(smem);                     // [warp][16][pitch] in the products' order of columns, then the CTA's
    float* stats = reinterpret_cast<float*>(smem + R::kStats);        // [warp][m, l][16], then the CTA's
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int row = g + 8 * h;
        if (t == 0) stats[warp * 32 + row] = m[h], stats[warp * 32 + 16 + row] = l[h];
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2*>(part + (warp * 16 + row) * R::kPitch + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
    }
    __syncthreads();
    float* all = part + kRowsWarps * 16 * R::kPitch;
    float* all_stats = stats + kRowsWarps * 32;
    for (int x = tid; x < live * (DP / 4); x += kRowsWarps * 32) {
        const int row = x / (DP / 4), c = x % (DP / 4) * 4;
        float top = -INFINITY, total = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, stats[w * 32 + row]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) {
            const float k = top == -INFINITY ? 0.f : exp2_fast(stats[w * 32 + row] - top);
            const float4 v = *reinterpret_cast<const float4*>(part + (w * 16 + row) * R::kPitch + c);
            total = __fmaf_rn(stats[w * 32 + 16 + row], k, total);
            y.x = __fmaf_rn(v.x, k, y.x), y.y = __fmaf_rn(v.y, k, y.y), y.z = __fmaf_rn(v.z, k, y.z), y.w = __fmaf_rn(v.w, k, y.w);
        }
        *reinterpret_cast<float4*>(all + row * R::kPitch + c) = y;
        if (c == 0) all_stats[row] = top, all_stats[16 + row] = total;
    }
    if (p.splits > 1) cluster_sync_all();
    else __syncthreads();
    constexpr int kWide = DP >= 128 ? 16 : 8;
    const uint32_t part_at = smem_u32(all), stats_at = smem_u32(all_stats);
    const int pieces = D / 8;
    for (int x = tid + split * kRowsWarps * 32; x < live * pieces; x += kRowsWarps * 32 * p.splits) {
        const int row = x / pieces, d = x % pieces * 8;
        // column d + e = kWide g + j of unit u lies at (kWide u + j) * 8 + g
        const int col = (d / (8 * kWide) * kWide + d % kWide) * 8 + d % (8 * kWide) / kWide;
        float y[8] = {}, total = 0.f;
        if (p.splits == 1) {
            total = all_stats[16 + row];
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = all[row * R::kPitch + col + e * 8];
        } else {
            float top = -INFINITY;
            for (int s = 0; s < p.splits; ++s) top = fmaxf(top, dsmem_f32(stats_at + row * 4, s));
            for (int s = 0; s < p.splits; ++s) {
                const float k = top == -INFINITY ? 0.f : exp2_fast(dsmem_f32(stats_at + row * 4, s) - top);
                total = __fmaf_rn(dsmem_f32(stats_at + (16 + row) * 4, s), k, total);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] = __fmaf_rn(dsmem_f32(part_at + (row * R::kPitch + col + e * 8) * 4, s), k, y[e]);
            }
        }
        store_row(p, y, total, b, r0 + row, kvh, ratio, d, QT());
    }
    if (p.splits > 1) cluster_sync_all();      // nobody leaves while its shared memory is read
}

template <typename QT, int DP> int launch_rows(AttnParams& p, cudaStream_t st) {
    using R = RowsTile<DP>;
    auto kern = kv8_rows_kernel<QT, DP>;
    const int64_t rows = (int64_t)p.Lq * (p.H / p.Hkv), tiles = (rows + 15) / 16;
    if (rows > INT32_MAX - 16 || tiles > INT32_MAX / p.B / p.Hkv) return -1;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kSmem)) return (int)e;
    const int64_t base = tiles * p.B * p.Hkv;
    p.row_tiles = (int)tiles;
    // CTAs along the keys: as long as there are fewer than one to an SM (two where sequences of different lengths leave some idle) and each has
    // a block for each warp. CTAs begin and end slowly: 16 sequences of up to 32768 tokens, 8 kv heads, 2 | 4 | 8 CTAs 182 | 120 | 156 us; 8 of up to
    // 8000 with 64 rows a head 94 | 73 | 148; one of 8000 with 120 rows a head 37 | 48 | 53.
    p.splits = 1;
    while (p.splits < 8 && base * p.splits < (p.B > 1 ? 296 : 148) && (int64_t)p.Lkv > (int64_t)p.splits * 16 * kRowsWarps) p.splits *= 2;
    return launch_pdl_cluster(kern, dim3((unsigned)(base * p.splits)), kRowsWarps * 32, R::kSmem, st, p.splits, p);
}

template <typename T> int launch_cross(AttnParams& p, cudaStream_t st) {
    if (attention_tc_takes(p, false)) return attention_tc(std::is_same<T, half>::value ? DT_F16 : DT_BF16, false, p, st);
    if (p.D <= 64) return launch_tile<T, 64>(p, st);
    if (p.D <= 128) return launch_tile<T, 128>(p, st);
    return p.D <= 192 ? launch_tile<T, 192>(p, st) : launch_tile<T, 256>(p, st);
}
template <typename T> int launch_packed(AttnParams& p, cudaStream_t st) {
    if (attention_tc_takes_packed(p)) return attention_tc_packed(std::is_same<T, half>::value ? DT_F16 : DT_BF16, p, st);
    if (p.D <= 64) return launch_packed<T, 64>(p, st);
    if (p.D <= 128) return launch_packed<T, 128>(p, st);
    return p.D <= 192 ? launch_packed<T, 192>(p, st) : launch_packed<T, 256>(p, st);
}
template <typename QT> int launch_kv8(AttnParams& p, cudaStream_t st) {
    if (attention_tc_takes(p, true)) return attention_tc(std::is_same<QT, half>::value ? DT_F16 : DT_BF16, true, p, st);
    return p.D <= 64 ? launch_rows<QT, 64>(p, st) : p.D <= 128 ? launch_rows<QT, 128>(p, st) : launch_rows<QT, 256>(p, st);
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
// Strides in elements of 16 bits: whole 16-byte pieces
bool ragged(const int64_t* s, int n) {
    for (int i = 0; i < n; ++i)
        if (s[i] % 8 != 0) return true;
    return false;
}

// Rows of the result in the same place
bool shared_rows(const int64_t* s, int B, int Lq, int H) { return (B > 1 && s[0] == 0) || (Lq > 1 && s[1] == 0) || (H > 1 && s[2] == 0); }

}  // namespace

GPU_API int gpu_cross_attention(int dtype, const void* q, const void* k, const void* v, void* out, const int64_t* strides, const int32_t* kv_len,
                                const uint8_t* key_mask, int64_t mask_stride, int B, int Lq, int Lkv, int H, int Hkv, int D, float scale, void* stream) {
    if (B < 0 || Lq < 0 || Lkv < 0 || Lkv > INT32_MAX - 256 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || D % 8 != 0 || D > 256) return -1;
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (B == 0 || Lq == 0) return 0;
    if (!q || !out || !strides || (Lkv > 0 && (!k || !v)) || off16(q) || off16(k) || off16(v) || off16(out) || ragged(strides, 12) || shared_rows(strides + 9, B, Lq, H))
        return -5;
    AttnParams p = {};
    p.q = q, p.k = k, p.v = v, p.out = out, p.kv_len = kv_len, p.mask = key_mask, p.mask_stride = mask_stride;
    for (int i = 0; i < 3; ++i) p.qs[i] = strides[i], p.ks[i] = strides[3 + i], p.vs[i] = strides[6 + i], p.os[i] = strides[9 + i];
    p.B = B, p.Lq = Lq, p.Lkv = Lkv, p.H = H, p.Hkv = Hkv, p.D = D, p.T = 1, p.scale = scale;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F16 ? launch_cross<half>(p, st) : launch_cross<bf16>(p, st);
}

GPU_API int gpu_kv8_attention(int dtype, const void* q, void* out, const int64_t* strides, const int8_t* k8, const int8_t* v8, const float* k_scale,
                              const float* v_scale, const int32_t* table, int64_t table_stride, const int32_t* lengths, const int32_t* q_len, int causal, int B,
                              int Lq, int H, int Hkv, int D, int T, int64_t pages, int max_pages, float scale, void* stream) {
    if (B < 0 || Lq < 0 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || D % 16 != 0 || D > 256 || pages < 0 || max_pages < 0) return -1;
    if (T != 16 && T != 32 && T != 64 && T != 128) return -206;
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if ((int64_t)max_pages * T > INT32_MAX - 256) return -1;
    if (B == 0 || Lq == 0) return 0;
    if (!q || !out || !strides || !lengths || off16(q) || off16(out) || off16(k8) || off16(v8) || ragged(strides, 6) || shared_rows(strides + 3, B, Lq, H)) return -5;
    if (max_pages > 0 && pages > 0 && (!k8 || !v8 || !k_scale || !v_scale || !table)) return -5;
    AttnParams p = {};
    p.q = q, p.k = k8, p.v = v8, p.out = out, p.k_scale = k_scale, p.v_scale = v_scale, p.table = table, p.table_stride = table_stride, p.pages = pages;
    for (int i = 0; i < 3; ++i) p.qs[i] = strides[i], p.os[i] = strides[3 + i];
    p.kv_len = lengths, p.q_len = q_len, p.causal = causal;
    p.B = B, p.Lq = Lq, p.Lkv = pages > 0 ? max_pages * T : 0, p.H = H, p.Hkv = Hkv, p.D = D, p.T = T, p.scale = scale;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F16 ? launch_kv8<half>(p, st) : launch_kv8<bf16>(p, st);
}

GPU_API int gpu_packed_attention(int dtype, const void* q, const void* k, const void* v, void* out, const int64_t* strides, const int32_t* offsets, int causal, int B,
                                 int rows, int H, int Hkv, int D, float scale, void* stream) {
    if (B < 0 || rows < 0 || rows > INT32_MAX - 512 || H <= 0 || Hkv <= 0 || H % Hkv != 0 || D <= 0 || D % 8 != 0 || D > 256) return -1;
    if (dtype != DT_F16 && dtype != DT_BF16) return -4;
    if (B == 0 || rows == 0) return 0;
    if (!q || !k || !v || !out || !strides || !offsets || off16(q) || off16(k) || off16(v) || off16(out) || ragged(strides, 8)) return -5;
    if ((rows > 1 && strides[6] == 0) || (H > 1 && strides[7] == 0)) return -5;      // rows of the result in the same place
    AttnParams p = {};
    p.q = q, p.k = k, p.v = v, p.out = out, p.offsets = offsets, p.rows = rows, p.causal = causal != 0;
    for (int i = 0; i < 2; ++i) p.qs[1 + i] = strides[i], p.ks[1 + i] = strides[2 + i], p.vs[1 + i] = strides[4 + i], p.os[1 + i] = strides[6 + i];
    p.B = B, p.H = H, p.Hkv = Hkv, p.D = D, p.scale = scale;
    // Heads of a token that share a tile: all that read one head of k and v, or as many as divide them and leave a tile several tokens
    const int ratio = H / Hkv;
    for (p.pack = ratio < 16 ? ratio : 16; ratio % p.pack != 0;) --p.pack;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F16 ? launch_packed<half>(p, st) : launch_packed<bf16>(p, st);
}
