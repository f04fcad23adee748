// The 4-bit linear of many tokens, on tcgen05: tiles of 128 rows of the weight by up to 192 columns (tokens; an f32 token is three).
//
// Codes become 16-bit operands in shared memory as they are (code minus zero point: a small integer), so nothing is rounded; the products of
// one group of K land in tensor memory, and the group's scale, one number to a row and so to a thread, takes them from there into sums in
// registers. Two to four accumulators take turns: while a group is multiplied, the one before is read. One thread an output row and half the
// columns: 96 sums of f32 at most. A CTA an SM, persistent over its tiles; where there are few tiles a cluster shares one along K and adds up in
// shared memory, in a fixed order.
//
// Warps 0-3 and 4-7: sums, for the first and second half of the columns. Warps 8-11: codes from global memory (each its 32 rows, a ring of its
// own) to operands, K-major with the 128-byte swizzle, a row to a lane; for f32 x also its three terms. Warp 12 issues the products, warp 13
// loads 16-bit x by TMA.
// Measured, 5120 -> 13824 fp16, us for groups of 32 | 64 | 128 | 256: 112 tokens 99 | 58 | 38 | 36 (a tile an SM), 333 tokens 231 | 143 | 86 | 81 (two tiles of 176
// columns; 330 and 545 TFLOP/s at 64 and 128). So there are two bounds. A block of 64 of K takes 0.45 us with 112 columns and 0.5 with 176 where groups are long:
// its codes' way through four warps. A group takes 0.6 to 0.7 us with 112 columns and 0.7 to 0.9 with 176: its way from tensor memory into the sums, which
// spill there (384 bytes a thread with fp16, 224 with bf16, 530 with f32 x). Issue slots 42 %, tensor pipe 14 % at 333 tokens, groups of 64.
// f32 x: 32 | 77 | 512 x 2560 -> 19456, groups of 128, 80 | 126 | 382 us: x's three terms are made again by every row tile, codes by every 64 tokens.
// Every wait is bounded; one that runs out is recorded in g_w4_status and the CTA unwinds.
#include "umma16.cuh"
#include "w4.cuh"

#include <type_traits>

namespace {

using namespace b200q;

__device__ int g_w4_status = 0;

constexpr int kRows = 128, kBlock = 64, kStages = 4, kBuffers = 4, kABytes = kRows * 128, kRing = 8, kRingBytes = 32 * 32;

struct TileParams {
    W4Params w;
    int tokens, columns, token_tiles, tiles, splits, blocks;      // of a tile; tiles in all; CTAs along K and blocks of 64 of each
    int buffers;                                                  // accumulators: as many as fit, at most four
};
__host__ __device__ inline int stage_bytes(int columns) { return kABytes + columns * 128; }
__host__ __device__ inline int tail_at(int columns) { return kStages * stage_bytes(columns) + 4 * kRing * kRingBytes; }

// Sums, operands, issue: their threads' shares of the launch's 512 x 128. What has more than 128 takes them (setmaxnreg.inc), the others give
// theirs up (setmaxnreg.dec takes no larger number than the launch's).
template <int XT> struct Regs {
    static constexpr int kSums = XT == DT_F32 ? 160 : 184, kCodes = XT == DT_F32 ? 136 : 88, kIssue = 56;
    static_assert(2 * kSums + kCodes + kIssue == 4 * 128, "register split");
};

template <int N> __device__ __forceinline__ float sum_at(const uint64_t (&acc)[N], int c) {
    float v[2];
    unpack_f32(acc[c >> 1], v[0], v[1]);
    return v[c & 1];
}
// One output row's sums (P to a token) from `token` on: bias once, and where the result is added to, sixteen of its values before the first
// is written.
template <typename T, int P, int N> __device__ __forceinline__ void store_column(const W4Params& w, const uint64_t (&acc)[N], float up, int token, int tokens, int n) {
    T* out = reinterpret_cast<T*>(w.out) + token * w.out_stride + n;
    const float bias = w.bias ? to_f<T>(gload(reinterpret_cast<const T*>(w.bias) + n)) : 0.f;
    constexpr int kTokens = 2 * N / P, kBatch = 8;
#pragma unroll
    for (int t0 = 0; t0 < kTokens; t0 += kBatch) {
        if (t0 >= tokens) break;
        float old[kBatch];
        if (w.beta != 0.f) {
#pragma unroll
            for (int t = 0; t < kBatch; ++t) old[t] = t0 + t < tokens ? to_f<T>(gload(out + t * w.out_stride)) : 0.f;
        }
#pragma unroll
        for (int t = 0; t < kBatch; ++t) {
            const int c = (t0 + t) * P;
            float y = sum_at(acc, c);
#pragma unroll
            for (int q = 1; q < P; ++q) y += sum_at(acc, c + q);
            y *= up;
            if (w.bias) y += bias;
            if (w.beta != 0.f) y = __fmaf_rn(w.beta, old[t], y);
            if (t0 + t < tokens) *out = from_f<T>(y);
            out += w.out_stride;
        }
    }
}

template <int XT, bool G32, bool WIDE> __global__ void __launch_bounds__(512, 1) w4_tile_kernel(const __grid_constant__ CUtensorMap tmap_x, const TileParams p) {
    using T = typename XType<XT>::Mma;
    constexpr int P = parts_of<XT>(), kMine = WIDE ? 96 : 64;      // columns of a sums thread
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const W4Params& w = p.w;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, stage_size = stage_bytes(p.columns);
    const uint32_t bars = base + tail_at(p.columns), full = bars, empty = bars + 8 * kStages, d_full = empty + 8 * kStages, d_empty = d_full + 8 * kBuffers;
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(sm + tail_at(p.columns) + 16 * kStages + 16 * kBuffers);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(full + 8 * i, XT == DT_F32 ? 4 : 5), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < kBuffers; ++i) mbar_init(d_full + 8 * i, 1), mbar_init(d_empty + 8 * i, 8);
        *abort_s = 0;
        fence_mbar_init();
        if (XT != DT_F32) prefetch_tmap(&tmap_x);
    }
    if (warp == 12) {
        tmem_alloc(smem_u32(tmem_s), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_s;
    pdl_wait();
    const int split = p.splits > 1 ? (int)cluster_ctarank() : 0;
    const int tile_first = blockIdx.x / p.splits, tile_step = gridDim.x / p.splits;
    const int all_blocks = (w.K + kBlock - 1) / kBlock, first = min(split * p.blocks, all_blocks), last = min(first + p.blocks, all_blocks);
    // groups of this CTA's share of K (which begins with one)
    const int block_shift = w.group_shift - 1, group0 = first * 64 / w.G, group_n = min((last * 64 + w.G - 1) / w.G, w.groups) - group0;

    if (warp < 8) {
        // ---- sums
        more_registers<Regs<XT>::kSums>();
        const int side = warp >> 2, quarter = warp & 3;
        // chunks of 16 columns; all columns of a token (16 of them fill P chunks) on one side
        const int front = (p.tokens / 16 - p.tokens / 32) * P, mine = side ? p.columns / 16 - front : front, col0 = side ? front * 16 : 0;
        const uint32_t at = tmem + ((uint32_t)(quarter * 32) << 16) + col0;
        uint32_t phase = 0;      // flips when the accumulators have been gone through
        int buf = 0;
        bool ok = true;
        for (int tile = tile_first; tile < p.tiles && ok; tile += tile_step) {
            const int n = tile / p.token_tiles * kRows + quarter * 32 + lane, m0 = tile % p.token_tiles * p.tokens;
            const int64_t scale_row = (int64_t)min(n, w.N - 1) * w.groups + group0;
            uint64_t acc[kMine / 2];      // two columns each
#pragma unroll
            for (int c = 0; c < kMine / 2; ++c) acc[c] = 0;
            // a group's scale is requested a group ahead, as the bits it is: a conversion here would wait for it
            const uint16_t* scales = reinterpret_cast<const uint16_t*>(w.scales) + scale_row;
            uint16_t next = group_n > 0 ? gload(scales) : (uint16_t)0;
            for (int g = 0; g < group_n; ++g) {
                const uint16_t bits = next;
                if (g + 1 < group_n) next = gload(scales + g + 1);
                if (!__all_sync(0xffffffffu, mbar_wait(d_full + 8 * buf, phase, abort_s, ST_TIMEOUT_TMEM_FULL))) { ok = false; break; }
                tc_fence_after();
                const float scale = w.scale_dt == DT_F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((uint32_t)bits << 16);
                const uint64_t s = pack_f32(scale, scale);
                constexpr int kAtOnce = WIDE ? 3 : 4;      // chunks requested together: as many as there are registers for
#pragma unroll
                for (int c0 = 0; c0 < kMine / 16; c0 += kAtOnce) {
                    uint32_t r[kAtOnce][16];
                    if (c0 < mine) {
#pragma unroll
                        for (int c = 0; c < kAtOnce; ++c)
                            if (c0 + c < mine) tmem_ld16(at + buf * p.columns + (c0 + c) * 16, r[c]);
                        tmem_ld_wait();
                    }
                    if (c0 + kAtOnce >= kMine / 16) {      // all are in registers
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(d_empty + 8 * buf);
                    }
#pragma unroll
                    for (int c = 0; c < kAtOnce; ++c)
                        if (c0 + c < mine)
#pragma unroll
                            for (int e = 0; e < 16; e += 2) acc[(c0 + c) * 8 + e / 2] = fma_f32x2(pack_f32(__uint_as_float(r[c][e]), __uint_as_float(r[c][e + 1])), s, acc[(c0 + c) * 8 + e / 2]);
                }
                if (++buf == p.buffers) buf = 0, phase ^= 1;
            }
            if (!ok) break;
            if (p.splits > 1) {      // [column][row], over the stages: every product of this CTA's only tile is done
                float* red = reinterpret_cast<float*>(sm);
#pragma unroll
                for (int c = 0; c < kMine; ++c)
                    if (c / 16 < mine) red[(col0 + c) * kRows + quarter * 32 + lane] = sum_at(acc, c);
            } else if (n < w.N) {
                const int first_token = m0 + col0 / P, tokens = min(mine * 16 / P, w.M - first_token);
                if (w.out_dt == DT_F32) store_column<float, P>(w, acc, Nibbles<T>::kUp, first_token, tokens, n);
                else if (w.out_dt == DT_F16) store_column<half, P>(w, acc, Nibbles<T>::kUp, first_token, tokens, n);
                else store_column<bf16, P>(w, acc, Nibbles<T>::kUp, first_token, tokens, n);
            }
        }
    } else if (warp < 12) {
        // ---- operands
        if constexpr (Regs<XT>::kCodes > 128) more_registers<Regs<XT>::kCodes>();
        else fewer_registers<Regs<XT>::kCodes>();
        const int mw = warp - 8, row = mw * 32 + lane;
        const uint32_t ring = base + kStages * stage_size + mw * kRing * kRingBytes;
        uint32_t step = 0;      // stages filled so far
        bool ok = true;
        for (int tile = tile_first; tile < p.tiles && ok; tile += tile_step) {
            const int n0 = tile / p.token_tiles * kRows, m0 = tile % p.token_tiles * p.tokens, n = min(n0 + row, w.N - 1);
            const int count = last - first;
            // 32 bytes of each of the warp's rows: two lanes to a row, sixteen rows at a time
            const uint8_t* src[2];
            uint32_t dst[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = i * 16 + (lane >> 1), c = lane & 1;
                src[i] = w.W + (int64_t)min(n0 + mw * 32 + r, w.N - 1) * (w.K >> 1) + first * 32 + c * 16;
                dst[i] = ring + r * 32 + ((c ^ (r >> 2)) & 1) * 16;
            }
            const int tail = w.K - first * kBlock - (lane & 1) * 32;      // columns from this lane's piece of block 0 on
            auto request = [&](int b) {
                const bool valid = b < count && b * kBlock < tail;
#pragma unroll
                for (int i = 0; i < 2; ++i) cp_async16(dst[i] + (b % kRing) * kRingBytes, valid ? src[i] + b * 32 : w.W, valid);
                cp_async_commit();
            };
#pragma unroll
            for (int b = 0; b < kRing; ++b) request(b);
            const int64_t zero_row = (int64_t)n * w.groups;
            // f32: a piece of eight columns of every sixteen tokens a lane, requested a block ahead
            float4 raw[XT == DT_F32 ? 8 : 1];
            auto request_x = [&](int b) {
                if constexpr (XT == DT_F32) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (u * 16 >= p.tokens) break;      // tokens of a tile come in sixteens
                        const int t = u * 16 + mw * 4 + (lane >> 3), k = (first + b) * kBlock + (lane & 7) * 8;
                        const bool valid = b < count && m0 + t < w.M && k < w.K;
                        const float* x = reinterpret_cast<const float*>(w.x) + (int64_t)(m0 + t) * w.x_stride + k;
                        raw[2 * u] = valid ? gload(reinterpret_cast<const float4*>(x)) : make_float4(0.f, 0.f, 0.f, 0.f);
                        raw[2 * u + 1] = valid ? gload(reinterpret_cast<const float4*>(x) + 1) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
                }
            };
            request_x(0);
            // codes and zero points are in registers a block ahead of their use
            uint4 code[2], code_next[2];
            uint32_t z[2] = {8u, 8u}, z_next[2] = {8u, 8u};
            auto fetch = [&](int b) {
                cp_async_wait<kRing - 1>();
                __syncwarp();
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(code_next[c].x), "=r"(code_next[c].y), "=r"(code_next[c].z), "=r"(code_next[c].w)
                                 : "r"(ring + (b % kRing) * kRingBytes + lane * 32 + ((c ^ (lane >> 2)) & 1) * 16) : "memory");
                if (w.zeros) {
                    const int k = (first + b) * 2;      // in halves of a block
                    z_next[0] = gload(w.zeros + zero_row + min(k >> w.group_shift, w.groups - 1));
                    z_next[1] = G32 ? gload(w.zeros + zero_row + min(k + 1, w.groups - 1)) : z_next[0];
                }
            };
            fetch(0);
            for (int b = 0; b < count; ++b, ++step) {
                const uint32_t stage = step % kStages;
#pragma unroll
                for (int c = 0; c < 2; ++c) code[c] = code_next[c], z[c] = z_next[c] & 15u;
                __syncwarp();                       // everybody has read block b's slot before it is written again
                request(b + kRing);
                fetch(b + 1);
                if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * stage, (step / kStages & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY))) { ok = false; break; }
                uint8_t* a = sm + stage * stage_size + row * 128;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Nibbles<T> nib(z[c]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        uint32_t v[4];
                        nib.expand(reinterpret_cast<const uint32_t*>(&code[c])[e], v);
                        *reinterpret_cast<uint4*>(a + (((c * 4 + e) ^ row) & 7) * 16) = make_uint4(v[0], v[1], v[2], v[3]);
                    }
                }
                if constexpr (XT == DT_F32) {
                    uint8_t* xs = sm + stage * stage_size + kABytes;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        if (u * 16 >= p.tokens) break;
                        const int t = u * 16 + mw * 4 + (lane >> 3);
                        uint4 v[3];
                        split2(raw[2 * u].x, raw[2 * u].y, v, 0), split2(raw[2 * u].z, raw[2 * u].w, v, 1);
                        split2(raw[2 * u + 1].x, raw[2 * u + 1].y, v, 2), split2(raw[2 * u + 1].z, raw[2 * u + 1].w, v, 3);
#pragma unroll
                        for (int q = 0; q < 3; ++q) *reinterpret_cast<uint4*>(xs + (t * 3 + q) * 128 + ((lane ^ (t * 3 + q)) & 7) * 16) = v[q];
                    }
                    request_x(b + 1);
                }
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(full + 8 * stage);
            }
            cp_async_wait<0>();      // the next tile's ring begins anew
            __syncwarp();
        }
    } else {
      fewer_registers<Regs<XT>::kIssue>();
      if (warp == 12) {
        // ---- products
        const uint32_t idesc = umma_idesc_16(std::is_same<T, bf16>::value, false, kRows, p.columns);
        const bool one = elect_one();
        uint32_t step = 0, phase = 1;
        int buf = 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity, int code) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, code)); };
        for (int tile = tile_first; tile < p.tiles && ok; tile += tile_step) {
            for (int b = first; b < last; ++b, ++step) {
                const uint32_t stage = step % kStages, a = umma_desc_lo(base + stage * stage_size), x = umma_desc_lo(base + stage * stage_size + kABytes);
                if (!wait(full + 8 * stage, step / kStages & 1, ST_TIMEOUT_FULL)) break;
#pragma unroll
                for (int part = 0; part < (G32 ? 2 : 1); ++part) {
                    if (G32 && b * 2 + part >= w.groups) break;
                    const bool begins = G32 || (b & ((1 << block_shift) - 1)) == 0, ends = G32 || b + 1 == last || ((b + 1) & ((1 << block_shift) - 1)) == 0;
                    if (begins) {
                        if (!wait(d_empty + 8 * buf, phase, ST_TIMEOUT_TMEM_EMPTY)) break;
                    }
                    tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < (G32 ? 2 : 4); ++kk) {
                            const uint32_t k = (part * 2 + kk) * 2;
                            umma_16_ss(tmem + buf * p.columns, a + k, x + k, idesc, !(begins && kk == 0));
                        }
                        if (ends) umma_commit(d_full + 8 * buf);
                    }
                    __syncwarp();
                    if (ends && ++buf == p.buffers) buf = 0, phase ^= 1;
                }
                if (!ok) break;
                if (one) umma_commit(empty + 8 * stage);
                __syncwarp();
            }
        }
      } else if (warp == 13 && XT != DT_F32) {
        // ---- 16-bit x
        uint32_t step = 0;
        bool ok = true;
        for (int tile = tile_first; tile < p.tiles && ok; tile += tile_step) {
            const int m0 = tile % p.token_tiles * p.tokens;
            for (int b = first; b < last; ++b, ++step) {
                const uint32_t stage = step % kStages;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * stage, (step / kStages & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY)))) break;
                if (lane == 0) {
                    mbar_arrive_expect_tx(full + 8 * stage, p.columns * 128);
                    tma_load_2d(base + stage * stage_size + kABytes, &tmap_x, b * kBlock, m0, full + 8 * stage);
                }
                __syncwarp();
            }
        }
      }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_s != 0) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // leave time for copies and products still in flight, then report
        if (threadIdx.x == 0) atomicCAS(&g_w4_status, 0, *abort_s);
        __syncthreads();
    }
    if (warp == 12) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
    if (p.splits > 1) {
        cluster_sync_all();
        const int n0 = tile_first / p.token_tiles * kRows, m0 = tile_first % p.token_tiles * p.tokens, tokens = min(p.tokens, w.M - m0);
        for (int i = threadIdx.x + split * 512; i < tokens * kRows; i += 512 * p.splits) {
            const int m = i >> 7, r = i & (kRows - 1);
            float y = 0.f;
            for (int s = 0; s < p.splits; ++s)
#pragma unroll
                for (int q = 0; q < P; ++q) y += dsmem_f32(base + ((m * P + q) * kRows + r) * 4, s);
            if (n0 + r < w.N) store_out(w, y * Nibbles<T>::kUp, m0 + m, n0 + r);
        }
        cluster_sync_all();      // nobody leaves while its sums are read
    }
}

template <int XT, bool G32, bool WIDE> int launch_tile(const CUtensorMap& tm, const TileParams& p, int grid, cudaStream_t st) {
    const int smem = tail_at(p.columns) + 256 + 1024;
    auto kern = w4_tile_kernel<XT, G32, WIDE>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem)) return (int)e;
    return launch_pdl_cluster(kern, dim3((unsigned)grid), 512, smem, st, p.splits, tm, p);
}

template <int XT> int launch(const W4Params& w, cudaStream_t st) {
    TileParams p = {};
    p.w = w;
    constexpr int P = parts_of<XT>(), kMost = XT == DT_F32 ? 64 : 192, kStep = 16;      // tokens of a tile
    const int sms = sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    const int64_t row_tiles = (w.N + kRows - 1) / kRows;
    // The number of token tiles that costs least: rounds of tiles over the SMs times what a tile takes, which grows with its columns from a
    // start of some 300 (a block takes 0.73 us with 112 columns and 0.91 with 176 at groups of 64, 0.48 and 0.56 at 128).
    int64_t best = INT64_MAX;
    const int fewest = (w.M + kMost - 1) / kMost;
    for (int t = fewest; t <= fewest + 3; ++t) {
        const int tokens = (int)(((int64_t)w.M + t - 1) / t + kStep - 1) / kStep * kStep;
        const int64_t rounds = (row_tiles * t + sms - 1) / sms, cost = rounds * (300 + tokens * P);
        if (cost < best) best = cost, p.token_tiles = t, p.tokens = tokens;
    }
    p.columns = p.tokens * P;
    p.buffers = 512 / p.columns < kBuffers ? 512 / p.columns : kBuffers;
    const int64_t tiles = row_tiles * p.token_tiles;
    if (tiles > INT32_MAX / 2) return -1;      // and so does a tile a round further on
    p.tiles = (int)tiles;
    // few tiles: a cluster of CTAs to each, every one with whole groups and at least four blocks
    const int all = (w.K + kBlock - 1) / kBlock, unit = w.G > kBlock ? w.G / kBlock : 1;
    p.splits = 1;
    while (p.splits < 8 && tiles * p.splits * 2 <= sms && all >= p.splits * 8) p.splits *= 2;
    p.blocks = ((all + p.splits - 1) / p.splits + unit - 1) / unit * unit;
    CUtensorMap tm = {};
    if (XT != DT_F32) {
        EncodeTiledFn enc = encode_fn();
        const cuuint64_t dims[2] = {(cuuint64_t)w.K, (cuuint64_t)w.M}, strides[1] = {(cuuint64_t)(w.M > 1 ? w.x_stride * 2 : (int64_t)w.K * 2)};
        const cuuint32_t box[2] = {kBlock, (cuuint32_t)p.columns}, estr[2] = {1, 1};
        if (!enc || enc(&tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(w.x), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return -203;
    }
    const int grid = p.splits > 1 ? p.tiles * p.splits : (int)(tiles < sms ? tiles : sms);
    if (p.columns <= 128) return w.G == 32 ? launch_tile<XT, true, false>(tm, p, grid, st) : launch_tile<XT, false, false>(tm, p, grid, st);
    return w.G == 32 ? launch_tile<XT, true, true>(tm, p, grid, st) : launch_tile<XT, false, true>(tm, p, grid, st);
}

}  // namespace

int b200q::w4_tile(int dtype, const W4Params& p, cudaStream_t st) {
    return dtype == DT_F32 ? launch<DT_F32>(p, st) : dtype == DT_F16 ? launch<DT_F16>(p, st) : launch<DT_BF16>(p, st);
}

int b200q::w4_status_read_clear(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_w4_status, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_w4_status, &zero, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    *out = v;
    return 0;
}
