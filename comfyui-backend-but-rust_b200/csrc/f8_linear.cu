// gpu_f8_linear: out = beta out + sum over blocks g of 128 columns of xs[m, g] ws[n / 128, g] (sum over k in g of x8[m, k] W8[n, k]) + bias,
// x8 and W8 e4m3. Products on tcgen05 kind::f8f6f4, a block's sum in tensor memory, from there times its scale into f32 sums in registers: the
// scales of two blocks of one output differ, so the tensor cores cannot go on adding. One rounding, to out's type.
//
// Few tokens, f8_few_kernel: the weight's bytes are the bound. 128 rows of the weight are the product's M, the tokens its N, so that both operands
// come straight from TMA; a cluster of CTAs shares a tile's K where there are few tiles and adds up in shared memory, in a fixed order.
// Many tokens, f8_tile_kernel: 128 tokens by up to 256 outputs, a persistent CTA an SM. While the tensor cores multiply one block, two warpgroups
// take the block before out of the other accumulator; an output row to a thread, whose scale is one number a block then.
// Every wait is bounded; one that runs out is recorded in g_f8_status and the CTA unwinds.
#include "f8.cuh"
#include "mma.cuh"
#include "umma16.cuh"

namespace {

using namespace b200q;

__device__ int g_f8_status = 0;

constexpr int kBlock = kF8Block, kBox = 128 * kBlock;      // bytes of 128 rows of a block

struct F8Params {
    const float *xs, *ws;
    const void* bias;
    void* out;
    int64_t out_stride;
    int M, N, K, groups, out_dt, add;      // add: onto out
    int m_tiles, tiles, splits, per;       // per: blocks to a CTA of a cluster
};

// kind::f8f6f4: D f32 (bits 4-5 = 1), A and B e4m3 (0), both K-major; 32 values of K an instruction
__host__ __device__ constexpr uint32_t umma_idesc_f8(int m, int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void umma_f8(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128) : "memory");
}

__device__ __forceinline__ float value_at(const void* p, int dt, int64_t i) {
    return dt == DT_F32 ? gload(reinterpret_cast<const float*>(p) + i) : dt == DT_F16 ? __half2float(gload(reinterpret_cast<const half*>(p) + i))
                                                                                      : __bfloat162float(gload(reinterpret_cast<const bf16*>(p) + i));
}
__device__ __forceinline__ void put_value(void* p, int dt, int64_t i, float v) {
    if (dt == DT_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (dt == DT_F16) reinterpret_cast<half*>(p)[i] = __float2half_rn(v);
    else reinterpret_cast<bf16*>(p)[i] = __float2bfloat16_rn(v);
}

// The end of a CTA: tensor memory back, a wait that ran out recorded
__device__ __forceinline__ void leave(volatile int* abort_s, bool allocated, uint32_t tmem, uint32_t columns) {
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_s != 0) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // leave time for copies and products still in flight, then report
        if (threadIdx.x == 0) atomicCAS(&g_f8_status, 0, *abort_s);
        __syncthreads();
    }
    if (allocated) {
        tc_fence_after();
        tmem_dealloc(tmem, columns);
    }
}

// ---- few tokens -----------------------------------------------------------------------------------------------------------------------
// Warps 0-3: sums, a row of the weight to a thread; warp 4 loads; warp 5 issues the products.
template <int NT> struct Few {
    static constexpr int kStage = kBox + NT * kBlock, kStages = NT <= 32 ? 5 : 4, kBuffers = 4, kColumns = kBuffers * NT;
    static constexpr int kTail = kStages * kStage, kScales = kTail + 256, kThreads = 192;
    static constexpr int smem(int per) { return kScales + per * NT * 4 + 1024; }
};

template <int NT> __global__ void __launch_bounds__(Few<NT>::kThreads) f8_few_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                                                                                  const F8Params p) {
    using L = Few<NT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = base + L::kTail, empty = full + 8 * L::kStages, t_full = empty + 8 * L::kStages, t_empty = t_full + 8 * L::kBuffers;
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(sm + L::kTail + 240);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
    float* sc = reinterpret_cast<float*>(sm + L::kScales);      // [block][token]
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < L::kBuffers; ++i) mbar_init(t_full + 8 * i, 1), mbar_init(t_empty + 8 * i, 4);
        *abort_s = 0;
        fence_mbar_init();
        prefetch_tmap(&tmap_x), prefetch_tmap(&tmap_w);
    }
    if (warp == 5) {
        tmem_alloc(smem_u32(tmem_s), L::kColumns);
        tmem_relinquish();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_s;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits;
    const int first = min(split * p.per, p.groups), blocks = min(p.per, p.groups - first);
    pdl_wait();
    float sum[NT] = {};
    if (warp < 4) {
        const float* ws = p.ws + (int64_t)tile * p.groups + first;
        for (int i = threadIdx.x; i < blocks * NT; i += 128) {
            const int m = i / blocks, g = i - m * blocks;
            sc[g * NT + m] = m < p.M ? gload(p.xs + (int64_t)m * p.groups + first + g) * gload(ws + g) : 0.f;
        }
        named_bar_sync(1, 128);
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        for (int g = 0; g < blocks; ++g) {
            const int buf = g % L::kBuffers;
            if (!__all_sync(0xffffffffu, mbar_wait(t_full + 8 * buf, g / L::kBuffers & 1, abort_s, ST_TIMEOUT_TMEM_FULL))) break;
            tc_fence_after();
            float t[NT];
            if constexpr (NT == 16) tmem_ld16(lanes + buf * NT, reinterpret_cast<uint32_t(&)[16]>(t));
            else
#pragma unroll
                for (int c = 0; c < NT; c += 32) tmem_ld32(lanes + buf * NT + c, reinterpret_cast<uint32_t(&)[32]>(t[c]));
            tmem_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(t_empty + 8 * buf);
#pragma unroll
            for (int c = 0; c < NT; c += 4) {
                const float4 s = *reinterpret_cast<const float4*>(sc + g * NT + c);
                sum[c] = __fmaf_rn(t[c], s.x, sum[c]), sum[c + 1] = __fmaf_rn(t[c + 1], s.y, sum[c + 1]);
                sum[c + 2] = __fmaf_rn(t[c + 2], s.z, sum[c + 2]), sum[c + 3] = __fmaf_rn(t[c + 3], s.w, sum[c + 3]);
            }
        }
    } else if (warp == 4) {
        for (int g = 0; g < blocks; ++g) {
            const int stage = g % L::kStages;
            if (!__all_sync(0xffffffffu, mbar_wait(empty + 8 * stage, (g / L::kStages & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY))) break;
            if (lane == 0) {
                const uint32_t at = base + stage * L::kStage;
                mbar_arrive_expect_tx(full + 8 * stage, L::kStage);
                tma_load_2d(at, &tmap_w, (first + g) * kBlock, tile * 128, full + 8 * stage);
                tma_load_2d(at + kBox, &tmap_x, (first + g) * kBlock, 0, full + 8 * stage);
            }
            __syncwarp();
        }
    } else {
        const bool one = elect_one();
        for (int g = 0; g < blocks; ++g) {
            const int stage = g % L::kStages, buf = g % L::kBuffers;
            if (!__all_sync(0xffffffffu, mbar_wait(full + 8 * stage, g / L::kStages & 1, abort_s, ST_TIMEOUT_FULL))) break;
            if (!__all_sync(0xffffffffu, mbar_wait(t_empty + 8 * buf, (g / L::kBuffers & 1) ^ 1, abort_s, ST_TIMEOUT_TMEM_EMPTY))) break;
            tc_fence_after();
            if (one) {
                const uint32_t w = umma_desc_lo(base + stage * L::kStage), x = umma_desc_lo(base + stage * L::kStage + kBox);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_f8(tmem + buf * NT, w + 2 * k, x + 2 * k, umma_idesc_f8(128, NT), k > 0);
                umma_commit(empty + 8 * stage);
                umma_commit(t_full + 8 * buf);
            }
            __syncwarp();
        }
    }
    // ---- out: the CTAs of a cluster take turns over the tokens, each adding up its tokens' sums of all
    const int n = tile * 128 + (int)threadIdx.x;
    if (p.splits > 1) {
        float* part = reinterpret_cast<float*>(sm);      // [token][row], over the stages: every product is done
        if (warp < 4)
#pragma unroll
            for (int c = 0; c < NT; ++c) part[c * 128 + threadIdx.x] = sum[c];
        __syncwarp();
        cluster_sync_all();
        if (warp < 4 && n < p.N)
            for (int m = split; m < p.M; m += p.splits) {
                float y = 0.f;
                for (int s = 0; s < p.splits; ++s) y += dsmem_f32(smem_u32(part + m * 128 + threadIdx.x), s);
                if (p.bias) y += value_at(p.bias, p.out_dt, n);
                const int64_t at = m * p.out_stride + n;
                if (p.add) y += value_at(p.out, p.out_dt, at);
                put_value(p.out, p.out_dt, at, y);
            }
        __syncwarp();
        cluster_sync_all();      // nobody leaves while its shared memory is read
    } else if (warp < 4 && n < p.N) {
        const float b = p.bias ? value_at(p.bias, p.out_dt, n) : 0.f;
#pragma unroll
        for (int m = 0; m < NT; ++m)
            if (m < p.M) {
                const int64_t at = m * p.out_stride + n;
                float y = sum[m] + b;
                if (p.add) y += value_at(p.out, p.out_dt, at);
                put_value(p.out, p.out_dt, at, y);
            }
    }
    leave(abort_s, warp == 5, tmem, L::kColumns);
}

// ---- many tokens ------------------------------------------------------------------------------------------------------------------------
// Warps 0-3 and 4-7: sums of the left and the right half of a tile's columns, an output row to a thread; warp 8 loads, warp 9 issues.
template <int BN> struct Tile {
    static constexpr int kStage = kBox + BN * kBlock, kStages = BN == 256 ? 4 : 5, kBuffers = 512 / BN, kHalf = BN / 2;
    static constexpr int kStaging = kStages * kStage, kTail = kStaging + 8 * 4096, kSmem = kTail + 256 + 1024, kThreads = 384;
    // registers: 384 threads x 168 at launch; a sums' thread holds a row of kHalf sums and 64 columns on their way
    static constexpr int kSumRegs = 224, kRestRegs = 56;
};

template <int BN> __global__ void __launch_bounds__(Tile<BN>::kThreads, 1) f8_tile_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                                                                                       const F8Params p) {
    using L = Tile<BN>;
    constexpr int kHalf = L::kHalf;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t full = base + L::kTail, empty = full + 8 * L::kStages, t_full = empty + 8 * L::kStages, t_empty = t_full + 8 * L::kBuffers;
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(sm + L::kTail + 240);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < L::kBuffers; ++i) mbar_init(t_full + 8 * i, 1), mbar_init(t_empty + 8 * i, 8);
        *abort_s = 0;
        fence_mbar_init();
        prefetch_tmap(&tmap_x), prefetch_tmap(&tmap_w);
    }
    if (warp == 9) {
        tmem_alloc(smem_u32(tmem_s), 512);
        tmem_relinquish();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_s;
    pdl_wait();
    if (warp < 8) {
        more_registers<L::kSumRegs>();
        const int side = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + side * kHalf;
        uint8_t* stage = sm + L::kStaging + warp * 4096;
        uint32_t no = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x) {
            const int m0 = tile % p.m_tiles * 128 + quarter * 32, n0 = tile / p.m_tiles * BN + side * kHalf;
            const float* xs = p.xs + (int64_t)min(m0 + lane, p.M - 1) * p.groups;
            const float* ws = p.ws + (int64_t)(min(n0, p.N - 1) / 128) * p.groups;
            uint64_t sum[kHalf / 2] = {};
            float now[4], next[4];      // scales of four blocks, requested four blocks ahead
            auto request = [&](int g0) {
#pragma unroll
                for (int i = 0; i < 4; ++i) next[i] = g0 + i < p.groups ? gload(xs + g0 + i) * gload(ws + g0 + i) : 0.f;
            };
            request(0);
            for (int g = 0; g < p.groups; ++g, ++no) {
                if ((g & 3) == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) now[i] = next[i];
                    request(g + 4);
                }
                const uint64_t s = pack_f32(now[0], now[0]);
                now[0] = now[1], now[1] = now[2], now[2] = now[3];
                const uint32_t buf = no % L::kBuffers;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(t_full + 8 * buf, no / L::kBuffers & 1, abort_s, ST_TIMEOUT_TMEM_FULL)))) break;
                tc_fence_after();
                uint32_t t[2][32];
                tmem_ld32(lanes + buf * BN, t[0]);
#pragma unroll
                for (int c = 0; c < kHalf; c += 32) {
                    tmem_ld_wait();
                    if (c + 32 < kHalf) tmem_ld32(lanes + buf * BN + c + 32, t[(c >> 5) + 1 & 1]);
                    else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(t_empty + 8 * buf);
                    }
                    const uint32_t(&r)[32] = t[c >> 5 & 1];
#pragma unroll
                    for (int e = 0; e < 32; e += 2)
                        sum[(c + e) / 2] = fma_f32x2(pack_f32(__uint_as_float(r[e]), __uint_as_float(r[e + 1])), s, sum[(c + e) / 2]);
                }
            }
            if (!ok) break;
            // ---- rows out: 32 columns of f32 at a time through this warp's staging, so that a row's pieces are stored together
            const int esize = p.out_dt == DT_F32 ? 4 : 2;
            const bool whole = n0 + kHalf <= p.N && (p.out_stride * esize) % (4 * esize) == 0 && (reinterpret_cast<uintptr_t>(p.out) % (4 * esize)) == 0;
#pragma unroll
            for (int c = 0; c < kHalf; c += 32) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float4 v;
                    unpack_f32(sum[c / 2 + 2 * e], v.x, v.y), unpack_f32(sum[c / 2 + 2 * e + 1], v.z, v.w);
                    *reinterpret_cast<float4*>(stage + lane * 128 + ((e ^ lane) & 7) * 16) = v;
                }
                __syncwarp();
                const int e = lane & 7, col = n0 + c + e * 4;
                float b[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) b[i] = p.bias && col + i < p.N ? value_at(p.bias, p.out_dt, col + i) : 0.f;
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int r = k * 4 + (lane >> 3), row = m0 + r;
                    if (row >= p.M) continue;
                    const float4 v4 = *reinterpret_cast<const float4*>(stage + r * 128 + ((e ^ r) & 7) * 16);
                    float y[4] = {v4.x + b[0], v4.y + b[1], v4.z + b[2], v4.w + b[3]};
                    const int64_t at = (int64_t)row * p.out_stride + col;
                    if (whole) {
                        if (p.out_dt == DT_F32) {
                            float4* dst = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at);
                            float4 o = make_float4(y[0], y[1], y[2], y[3]);
                            if (p.add) {
                                const float4 old = gload(dst);
                                o.x += old.x, o.y += old.y, o.z += old.z, o.w += old.w;
                            }
                            *dst = o;
                        } else {
                            uint2* dst = reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at);
                            if (p.add)
#pragma unroll
                                for (int i = 0; i < 4; ++i) y[i] += value_at(p.out, p.out_dt, at + i);
                            *dst = p.out_dt == DT_F16 ? make_uint2(pack2<half>(y[0], y[1]), pack2<half>(y[2], y[3]))
                                                      : make_uint2(pack2<bf16>(y[0], y[1]), pack2<bf16>(y[2], y[3]));
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (col + i < p.N) put_value(p.out, p.out_dt, at + i, y[i] + (p.add ? value_at(p.out, p.out_dt, at + i) : 0.f));
                    }
                }
                __syncwarp();
            }
        }
    } else {
        fewer_registers<L::kRestRegs>();
        if (warp == 8) {
            uint32_t no = 0;
            bool ok = true;
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
                for (int g = 0; g < p.groups; ++g, ++no) {
                    const uint32_t stage = no % L::kStages;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * stage, (no / L::kStages & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY)))) break;
                    if (lane == 0) {
                        const uint32_t at = base + stage * L::kStage;
                        mbar_arrive_expect_tx(full + 8 * stage, L::kStage);
                        tma_load_2d(at, &tmap_x, g * kBlock, tile % p.m_tiles * 128, full + 8 * stage);
                        tma_load_2d(at + kBox, &tmap_w, g * kBlock, tile / p.m_tiles * BN, full + 8 * stage);
                    }
                    __syncwarp();
                }
        } else if (warp == 9) {
            const bool one = elect_one();
            uint32_t no = 0;
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, int code) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, code)); };
            for (int tile = blockIdx.x; tile < p.tiles && ok; tile += gridDim.x)
                for (int g = 0; g < p.groups; ++g, ++no) {
                    const uint32_t stage = no % L::kStages, buf = no % L::kBuffers;
                    if (!wait(t_empty + 8 * buf, (no / L::kBuffers & 1) ^ 1, ST_TIMEOUT_TMEM_EMPTY) || !wait(full + 8 * stage, no / L::kStages & 1, ST_TIMEOUT_FULL)) break;
                    tc_fence_after();
                    if (one) {
                        const uint32_t x = umma_desc_lo(base + stage * L::kStage), w = umma_desc_lo(base + stage * L::kStage + kBox);
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_f8(tmem + buf * BN, x + 2 * k, w + 2 * k, umma_idesc_f8(128, BN), k > 0);
                        umma_commit(empty + 8 * stage);
                        umma_commit(t_full + 8 * buf);
                    }
                    __syncwarp();
                }
        }
    }
    leave(abort_s, warp == 9, tmem, 512);
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------

bool codes_map(CUtensorMap* tm, const void* ptr, int64_t stride, int rows, int K, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(rows > 1 ? stride : (K + 15) / 16 * 16)};
    const cuuint32_t box[2] = {kBlock, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc && enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT> int launch_few(const void* x, int64_t x_stride, const void* W, F8Params& p, cudaStream_t st) {
    using L = Few<NT>;
    CUtensorMap tx, tw;
    if (!codes_map(&tx, x, x_stride, p.M, p.K, NT) || !codes_map(&tw, W, p.K, p.N, p.K, 128)) return -203;
    p.tiles = (p.N + 127) / 128;
    p.splits = 1;
    while (p.splits < 8 && p.tiles * p.splits * 2 <= 296 && p.groups >= p.splits * 4) p.splits *= 2;
    p.per = (p.groups + p.splits - 1) / p.splits;
    const int smem = L::smem(p.per);
    auto kern = f8_few_kernel<NT>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem(256))) return (int)e;
    return launch_pdl_cluster(kern, dim3((unsigned)(p.tiles * p.splits)), L::kThreads, smem, st, p.splits, tx, tw, p);
}
template <int BN> int launch_tile(const void* x, int64_t x_stride, const void* W, F8Params& p, int sms, cudaStream_t st) {
    using L = Tile<BN>;
    CUtensorMap tx, tw;
    if (!codes_map(&tx, x, x_stride, p.M, p.K, 128) || !codes_map(&tw, W, p.K, p.N, p.K, BN)) return -203;
    p.m_tiles = (p.M + 127) / 128;
    const int64_t tiles = (int64_t)p.m_tiles * ((p.N + BN - 1) / BN);
    if (tiles > INT32_MAX / 2) return -1;      // and so does a tile a round further on
    p.tiles = (int)tiles;
    auto kern = f8_tile_kernel<BN>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem)) return (int)e;
    return launch_pdl(kern, dim3((unsigned)(p.tiles < sms ? p.tiles : sms)), L::kThreads, L::kSmem, st, tx, tw, p);
}

}  // namespace

int b200q::f8_status_read_clear(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_f8_status, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_f8_status, &zero, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    *out = v;
    return 0;
}

GPU_API int gpu_f8_linear(const void* x, int64_t x_stride, const float* xs, const void* W, const float* ws, const void* bias, int out_dt, void* out,
                          int64_t out_stride, float beta, int M, int N, int K, void* stream) {
    if (out_dt < DT_F32 || out_dt > DT_BF16) return -4;
    if (M < 0 || N < 0 || K <= 0 || K % 16 != 0 || M > INT32_MAX - 256 || N > INT32_MAX - 256) return -1;
    if (K > 32768) return -2;
    if (beta != 0.f && beta != 1.f) return -207;
    if (M == 0 || N == 0) return 0;
    auto off16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) != 0; };
    if (!x || !xs || !W || !ws || !out || off16(x) || off16(W) || (M > 1 && (x_stride % 16 != 0 || x_stride < K || out_stride < N))) return -5;
    F8Params p = {};
    p.xs = xs, p.ws = ws, p.bias = bias, p.out = out, p.out_stride = out_stride, p.M = M, p.N = N, p.K = K, p.groups = (K + kBlock - 1) / kBlock;
    p.out_dt = out_dt, p.add = beta != 0.f;
    cudaStream_t st = (cudaStream_t)stream;
    if (M <= 16) return launch_few<16>(x, x_stride, W, p, st);
    if (M <= 32) return launch_few<32>(x, x_stride, W, p, st);
    if (M <= 64) return launch_few<64>(x, x_stride, W, p, st);
    const int sms = sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    // tiles of 256 outputs where they fill the device
    const int64_t wide = (int64_t)((M + 127) / 128) * ((N + 255) / 256);
    return wide >= 2 * sms ? launch_tile<256>(x, x_stride, W, p, sms, st) : launch_tile<128>(x, x_stride, W, p, sms, st);
}
