// gpu_f8_linear: out = beta out + sum over blocks g of 128 columns of xs[m, g] ws[n / 128, g] (sum over k in g of x8[m, k] W8[n, k]) + bias,
// x8 and W8 e4m3. Products on tcgen05 kind::f8f6f4, a block's sum in tensor memory, from there times its scale into f32 sums in registers: the
// scales of two blocks of one output differ, so the tensor cores cannot go on adding. One rounding, to out's type.
//
// Few tokens, f8_few_kernel: the weight's bytes are the bound. 128 rows of the weight are the product's M, the tokens its N, so that both operands
// come straight from TMA; a cluster of CTAs shares a tile's K where there are few tiles and adds up in shared memory, in a fixed order.
// Many tokens, f8_tile_kernel: 256 tokens by 256 outputs, a persistent pair of CTAs. While the tensor cores multiply one block, two warpgroups
// take the block before out of the other accumulator; an output row to a thread, whose scale is one number a block then.
// Every wait is bounded; one that runs out is recorded in g_f8_status and the CTA unwinds.
#include "cluster_room.h"
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

__device__ __forceinline__ float4 dsmem_f32x4(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mapa_shared(addr, rank)) : "memory");
    return v;
}
// Four columns of sums that the CTAs `from`, from + by, ... of the cluster (kMost at most, p.splits in all) have at `addr`, in this order. All are on their way
// at once: one after the other a row of 64 waits for each
template <int kMost> __device__ __forceinline__ void add_up(const F8Params& p, uint32_t addr, uint32_t from, uint32_t by, float (&y)[4]) {
    float4 v[kMost];
#pragma unroll
    for (int s = 0; s < kMost; ++s) v[s] = s < p.splits ? dsmem_f32x4(addr, from + s * by) : make_float4(0.f, 0.f, 0.f, 0.f);
    y[0] = v[0].x, y[1] = v[0].y, y[2] = v[0].z, y[3] = v[0].w;
#pragma unroll
    for (int s = 1; s < kMost; ++s)
        if (s < p.splits) y[0] += v[s].x, y[1] += v[s].y, y[2] += v[s].z, y[3] += v[s].w;
}
// Four columns of a row from `col` on: bias and what was there, and out; whole: rows of out begin on the four columns' bytes
__device__ __forceinline__ bool whole_rows(const F8Params& p) { return p.out_stride % 4 == 0 && (reinterpret_cast<uintptr_t>(p.out) & (p.out_dt == DT_F32 ? 15 : 7)) == 0; }
__device__ __forceinline__ void finish4(const F8Params& p, int row, int col, bool whole, bool add, float (&y)[4]) {
    const int64_t at = (int64_t)row * p.out_stride + col;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (col + e >= p.N) continue;
        if (p.bias) y[e] += value_at(p.bias, p.out_dt, col + e);
        if (add) y[e] += value_at(p.out, p.out_dt, at + e);
    }
    if (whole && col + 4 <= p.N) {
        if (p.out_dt == DT_F32) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
        else
            *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = p.out_dt == DT_F16 ? make_uint2(pack2<half>(y[0], y[1]), pack2<half>(y[2], y[3]))
                                                                                                    : make_uint2(pack2<bf16>(y[0], y[1]), pack2<bf16>(y[2], y[3]));
    } else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (col + e < p.N) put_value(p.out, p.out_dt, at + e, y[e]);
}

// Four columns of a row as they lie in memory: loaded in one place, made numbers in another, so that nobody waits between the loads
struct Four {
    uint4 w;
    __device__ __forceinline__ void load(const void* base, int dt, int64_t at) {
        if (dt == DT_F32) w = gload(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(base) + at));
        else {
            const uint2 v = gload(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(base) + at));
            w = make_uint4(v.x, v.x >> 16, v.y, v.y >> 16);
        }
    }
    __device__ __forceinline__ float value(int dt, uint32_t x) const {
        return dt == DT_F32 ? __uint_as_float(x) : dt == DT_F16 ? __half2float(__ushort_as_half((uint16_t)x)) : __bfloat162float(__ushort_as_bfloat16((uint16_t)x));
    }
};

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
        pdl_trigger();      // the last blocks are on their way: the next kernel's CTAs find room beside this one's and can set up
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
        const int col = tile * 128 + lane * 4;
        const bool whole = whole_rows(p);
        if (warp < 4 && col < p.N)      // a token to a warp
            for (int m = split + warp * p.splits; m < p.M; m += 4 * p.splits) {
                float y[4];
                add_up<6>(p, smem_u32(part + m * 128 + lane * 4), 0, 1, y);
                finish4(p, m, col, whole, p.add, y);
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
// A pair of CTAs on a tile of 256 tokens by 256 outputs: each has its 128 tokens' sums and loads its tokens' block and half of the weight's, which
// the tensor cores read from both. (A CTA alone on 128 x 256 needs 48 KB a block instead of 32: from L2 the device has some 14 TB/s, which bound
// that form to 0.5 us a block, the products' own 0.27.) Warps 0-3 and 4-7: sums of the left and the right half of a tile's columns, an output row to a
// thread; warp 8 loads, warp 9 of the first CTA issues the products of both, warps 10 and 11 bring in the scales.
struct Tile {
    static constexpr int kStage = 2 * kBox, kStages = 5, kBuffers = 2, kColumns = 256, kHalf = 128, kChunk = 8;
    // kChunk blocks' scales, twice: of 128 rows of x, of two blocks of the weight
    static constexpr int kStaging = kStages * kStage, kXScales = kStaging + 8 * 4096, kWScales = kXScales + 2 * kChunk * 512, kTail = kWScales + 2 * kChunk * 8;
    static constexpr int kSmem = kTail + 256 + 1024, kThreads = 384;
    // registers: 384 threads x 168 at launch; a sums' thread holds a row of kHalf sums and 64 columns on their way
    static constexpr int kSumRegs = 224, kRestRegs = 56;
    static_assert(2 * kSumRegs + kRestRegs == 3 * 168, "register split");
};
__device__ __forceinline__ void umma_f8_pair(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 da, {%1, %5};\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], da, db, %3, p;\n\t}"
        ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128) : "memory");
}

// The mbarrier at this offset in both CTAs of the pair gets an arrival once the products that this thread issued are done; `mask`: the pair's ranks
__device__ __forceinline__ void commit_pair(uint32_t bar, uint16_t mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask) : "memory");
}

// A warp's 32 rows of sums out, by way of its staging, so that a row's pieces are stored together
__device__ __forceinline__ void rows_out(const F8Params& p, const float (&sum)[Tile::kHalf], uint8_t* stage, int m0, int n0, int lane) {
    constexpr int kCols = Tile::kHalf;
    const int left = min(32, p.M - m0), esize = p.out_dt == DT_F32 ? 4 : 2;
    if (left <= 0 || n0 >= p.N) return;
    const bool whole = n0 + kCols <= p.N && p.out_stride * esize % 16 == 0 && (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 &&
                       (!p.bias || (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0);
    if (whole && esize == 2 && !p.add) {
#pragma unroll
        for (int c = 0; c < kCols; c += 64) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) y[i] = sum[c + e * 8 + i];
                if (p.bias) {
                    float b[8];
                    if (p.out_dt == DT_F16) load8<half>(reinterpret_cast<const half*>(p.bias) + n0 + c + e * 8, b);
                    else load8<bf16>(reinterpret_cast<const bf16*>(p.bias) + n0 + c + e * 8, b);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] += b[i];
                }
                *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ lane) & 7) * 16) =
                    p.out_dt == DT_F16 ? make_uint4(pack2<half>(y[0], y[1]), pack2<half>(y[2], y[3]), pack2<half>(y[4], y[5]), pack2<half>(y[6], y[7]))
                                       : make_uint4(pack2<bf16>(y[0], y[1]), pack2<bf16>(y[2], y[3]), pack2<bf16>(y[4], y[5]), pack2<bf16>(y[6], y[7]));
            }
            __syncwarp();
            const int e = lane & 7;
            uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (int64_t)(m0 + (lane >> 3)) * p.out_stride + n0 + c + e * 8;
            uint4 v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const uint4*>(stage + (k * 4 + (lane >> 3)) * 128 + ((e ^ (k * 4 + (lane >> 3))) & 7) * 16);
#pragma unroll
            for (int k = 0; k < 8; ++k, out += 4 * p.out_stride)
                if (k * 4 + (lane >> 3) < left) *reinterpret_cast<uint4*>(out) = v[k];
            __syncwarp();
        }
        return;
    }
    // f32 rows, rows that are added to, ragged ones: 32 columns of f32 at a time
#pragma unroll
    for (int c = 0; c < kCols; c += 32) {
        Four was[8] = {};      // what is added to: eight rows on their way at once (one after the other 4352 x 2560 -> 2560 in bf16 takes 88 us instead of 66)
        if (whole && p.add)
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (k * 4 + (lane >> 3) < left) was[k].load(p.out, p.out_dt, (int64_t)(m0 + k * 4 + (lane >> 3)) * p.out_stride + n0 + c + (lane & 7) * 4);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            *reinterpret_cast<float4*>(stage + lane * 128 + ((e ^ lane) & 7) * 16) = make_float4(sum[c + 4 * e], sum[c + 4 * e + 1], sum[c + 4 * e + 2], sum[c + 4 * e + 3]);
        __syncwarp();
        if (whole) {
            const int e = lane & 7, col = n0 + c + e * 4;
            float b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) b[i] = p.bias ? value_at(p.bias, p.out_dt, col + i) : 0.f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = k * 4 + (lane >> 3);
                if (r >= left) continue;
                const float4 v = *reinterpret_cast<const float4*>(stage + r * 128 + ((e ^ r) & 7) * 16);
                const uint4 w = was[k].w;
                const float y[4] = {v.x + b[0] + was[k].value(p.out_dt, w.x), v.y + b[1] + was[k].value(p.out_dt, w.y), v.z + b[2] + was[k].value(p.out_dt, w.z),
                                    v.w + b[3] + was[k].value(p.out_dt, w.w)};
                const int64_t at = (int64_t)(m0 + r) * p.out_stride + col;
                if (esize == 4) *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.out) + at) = make_float4(y[0], y[1], y[2], y[3]);
                else
                    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.out) + at) = p.out_dt == DT_F16 ? make_uint2(pack2<half>(y[0], y[1]), pack2<half>(y[2], y[3]))
                                                                                                            : make_uint2(pack2<bf16>(y[0], y[1]), pack2<bf16>(y[2], y[3]));
            }
        } else if (n0 + c + lane < p.N) {
            const int col = n0 + c + lane;
            const float b = p.bias ? value_at(p.bias, p.out_dt, col) : 0.f;
#pragma unroll 2
            for (int r = 0; r < left; ++r) {
                float y = *reinterpret_cast<const float*>(stage + r * 128 + (((lane >> 2) ^ r) & 7) * 16 + (lane & 3) * 4) + b;
                const int64_t at = (int64_t)(m0 + r) * p.out_stride + col;
                if (p.add) y += value_at(p.out, p.out_dt, at);
                put_value(p.out, p.out_dt, at, y);
            }
        }
        __syncwarp();
    }
}

// Few tiles: a cluster of `splits` pairs on each, which share its K and add up in shared memory, in a fixed order.
template <bool SPLIT> __global__ void __launch_bounds__(Tile::kThreads, 1) f8_tile_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w, const F8Params p) {
    using L = Tile;
    constexpr int kHalf = L::kHalf;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;      // the same in both CTAs
    uint8_t* sm = smem_raw + (base - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // full and t_empty: the first CTA's are used
    const uint32_t full = base + L::kTail, empty = full + 8 * L::kStages, t_full = empty + 8 * L::kStages, t_empty = t_full + 8 * L::kBuffers;
    const uint32_t s_full = t_empty + 8 * L::kBuffers, s_empty = s_full + 16;
    float *x_scales = reinterpret_cast<float*>(sm + L::kXScales), *w_scales = reinterpret_cast<float*>(sm + L::kWScales);      // [chunk % 2][block][row], [block][side]
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(sm + L::kTail + 240);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
    const uint32_t in_cluster = cluster_ctarank(), rank = SPLIT ? in_cluster & 1 : in_cluster, leader = SPLIT ? in_cluster & ~1u : 0;
    if (threadIdx.x == 0) {
        for (int i = 0; i < L::kStages; ++i) mbar_init(full + 8 * i, 1), mbar_init(empty + 8 * i, 1);
        for (int i = 0; i < L::kBuffers; ++i) mbar_init(t_full + 8 * i, 1), mbar_init(t_empty + 8 * i, 16);
        for (int i = 0; i < 2; ++i) mbar_init(s_full + 8 * i, 2), mbar_init(s_empty + 8 * i, 8);
        *abort_s = 0;
        fence_mbar_init();
        prefetch_tmap(&tmap_x), prefetch_tmap(&tmap_w);
    }
    if (warp == 9) {
        tmem_alloc_pair(smem_u32(tmem_s), 512);
        tmem_relinquish_pair();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();      // the other CTA's barriers exist before anything signals them
    tc_fence_after();
    const uint32_t tmem = *tmem_s;
    pdl_wait();
    const int pair = blockIdx.x / (SPLIT ? 2 * p.splits : 2), pairs = gridDim.x / (SPLIT ? 2 * p.splits : 2);      // (clusters; one tile each if they have several pairs)
    const int g_first = SPLIT ? (int)(in_cluster >> 1) * p.per : 0, g_last = SPLIT ? min(g_first + p.per, p.groups) : p.groups;
    if (warp < 8) {
        more_registers<L::kSumRegs>();
        const int side = warp >> 2, quarter = warp & 3;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + side * kHalf;
        uint8_t* stage = sm + L::kStaging + warp * 4096;
        uint32_t no = 0, chunk = 0;
        bool ok = true;
        for (int tile = pair; tile < p.tiles && ok; tile += pairs) {
            const int m0 = tile % p.m_tiles * 256 + (int)rank * 128 + quarter * 32, n0 = tile / p.m_tiles * L::kColumns + side * kHalf;
            float sum[kHalf] = {};
            for (int g = g_first; g < g_last; ++g, ++no) {
                const int part = (g - g_first) % L::kChunk, at = (int)(chunk & 1) * L::kChunk + part;
                if (part == 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * (chunk & 1), chunk >> 1 & 1, abort_s, ST_TIMEOUT_UNPACK)))) break;
                const float scale = x_scales[at * 128 + quarter * 32 + lane] * w_scales[at * 2 + side];
                if (part == L::kChunk - 1 || g == g_last - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty + 8 * (chunk & 1));
                    ++chunk;
                }
                const uint32_t buf = no % L::kBuffers;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(t_full + 8 * buf, no / L::kBuffers & 1, abort_s, ST_TIMEOUT_TMEM_FULL)))) break;
                if (warp == 0 && lane == 0) mbar_arrive(empty + 8 * (no % L::kStages));      // the products have read the stage as well: one commit a block
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < kHalf; c += 64) {
                    uint32_t t[64];
                    tmem_ld32(lanes + buf * L::kColumns + c, reinterpret_cast<uint32_t(&)[32]>(t[0]));
                    tmem_ld32(lanes + buf * L::kColumns + c + 32, reinterpret_cast<uint32_t(&)[32]>(t[32]));
                    tmem_ld_wait();
                    if (c + 64 == kHalf) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_remote(mapa_shared(t_empty + 8 * buf, leader));
                    }
#pragma unroll
                    for (int e = 0; e < 64; e += 2) {      // two sums an instruction (single ones: 288 us instead of 282, 4352 x 5120 -> 13824)
                        const float2 y = __ffma2_rn(make_float2(__uint_as_float(t[e]), __uint_as_float(t[e + 1])), make_float2(scale, scale), make_float2(sum[c + e], sum[c + e + 1]));
                        sum[c + e] = y.x, sum[c + e + 1] = y.y;
                    }
                }
            }
            if (!ok) break;
            if (!SPLIT) rows_out(p, sum, stage, m0, n0, lane);
            else {      // [row][256 columns] in pieces of four, over the stages: every product of the pair is done
                const int row = quarter * 32 + lane;
#pragma unroll
                for (int e = 0; e < kHalf / 4; ++e)
                    *reinterpret_cast<float4*>(sm + row * 1024 + ((side * (kHalf / 4) + e) ^ (row & 7)) * 16) = make_float4(sum[4 * e], sum[4 * e + 1], sum[4 * e + 2], sum[4 * e + 3]);
            }
        }
    } else {
        fewer_registers<L::kRestRegs>();
        if (warp == 8) {
            uint32_t no = 0;
            bool ok = true;
            for (int tile = pair; tile < p.tiles && ok; tile += pairs) {
                const int row_x = tile % p.m_tiles * 256 + (int)rank * 128, row_w = tile / p.m_tiles * L::kColumns + (int)rank * 128;
                for (int g = g_first; g < g_last; ++g, ++no) {
                    const uint32_t stage = no % L::kStages;
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(empty + 8 * stage, (no / L::kStages & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY)))) break;
                    if (lane == 0) {
                        const uint32_t at = base + stage * L::kStage, bar = mapa_shared(full + 8 * stage, leader);
                        if (rank == 0) mbar_arrive_expect_tx(full + 8 * stage, 2 * L::kStage);
                        tma_load_2d_pair(at, &tmap_x, g * kBlock, row_x, bar);
                        tma_load_2d_pair(at + kBox, &tmap_w, g * kBlock, row_w, bar);
                    }
                    __syncwarp();
                }
            }
        } else if (warp >= 10) {
            // ---- scales, kChunk blocks at a time, 64 rows a warp: rows of x lie groups * 4 bytes apart, 32 sectors to a load, which the sums' warps would
            // wait for block by block (4352 x 5120 -> 13824: 291 us with their loads two blocks ahead)
            uint32_t chunk = 0;
            bool ok = true;
            for (int tile = pair; tile < p.tiles && ok; tile += pairs) {
                const int m0 = tile % p.m_tiles * 256 + (int)rank * 128 + (warp - 10) * 64, n0 = tile / p.m_tiles * L::kColumns;
                for (int g0 = g_first; g0 < g_last; g0 += L::kChunk, ++chunk) {
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait(s_empty + 8 * (chunk & 1), (chunk >> 1 & 1) ^ 1, abort_s, ST_TIMEOUT_EMPTY)))) break;
                    float v[2][L::kChunk], w = 0.f;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < L::kChunk; ++e)
                            v[i][e] = m0 + i * 32 + lane < p.M && g0 + e < p.groups ? gload(p.xs + (int64_t)(m0 + i * 32 + lane) * p.groups + g0 + e) : 0.f;
                    if (warp == 10 && lane < 2 * L::kChunk && g0 + lane / 2 < p.groups && n0 + lane % 2 * kHalf < p.N)
                        w = gload(p.ws + (int64_t)((n0 + lane % 2 * kHalf) / kBlock) * p.groups + g0 + lane / 2);
                    const int at = (int)(chunk & 1) * L::kChunk;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int e = 0; e < L::kChunk; ++e) x_scales[(at + e) * 128 + (warp - 10) * 64 + i * 32 + lane] = v[i][e];
                    if (warp == 10 && lane < 2 * L::kChunk) w_scales[at * 2 + lane] = w;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_full + 8 * (chunk & 1));
                }
            }
        } else if (warp == 9 && rank == 0) {
            const bool one = elect_one();
            uint32_t no = 0;
            bool ok = true;
            auto wait = [&](uint32_t bar, uint32_t parity, int code) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, code)); };
            for (int tile = pair; tile < p.tiles && ok; tile += pairs)
                for (int g = g_first; g < g_last; ++g, ++no) {
                    const uint32_t stage = no % L::kStages, buf = no % L::kBuffers;
                    if (!wait(full + 8 * stage, no / L::kStages & 1, ST_TIMEOUT_FULL) || !wait(t_empty + 8 * buf, (no / L::kBuffers & 1) ^ 1, ST_TIMEOUT_TMEM_EMPTY)) break;
                    tc_fence_after();
                    if (one) {
                        const uint32_t x = umma_desc_lo(base + stage * L::kStage), w = umma_desc_lo(base + stage * L::kStage + kBox);
#pragma unroll
                        for (int k = 0; k < 4; ++k) umma_f8_pair(tmem + buf * L::kColumns, x + 2 * k, w + 2 * k, umma_idesc_f8(256, L::kColumns), k > 0);
                        commit_pair(t_full + 8 * buf, (uint16_t)(3u << leader));
                    }
                    __syncwarp();
                }
        }
    }
    if (SPLIT) {
        __syncwarp();
        cluster_sync_all();
        // the CTAs of a tile's 128 rows take turns over them, each adding up all of a row
        const int m0 = pair % p.m_tiles * 256 + (int)rank * 128, n0 = pair / p.m_tiles * L::kColumns, left = min(128, p.M - m0);
        const bool whole = whole_rows(p);
        const int first = threadIdx.x + (int)(in_cluster >> 1) * 256, by = 256 * p.splits, last = warp < 8 && pair < p.tiles ? left * 64 : 0;
        if (p.add && whole && p.N % 4 == 0) {      // what is added to: four rows on their way at once (700 x 9728 -> 2560 onto bf16 42 us without, 34)
            const int col = n0 + (first & 63) * 4;
            for (int i = first; i < last && col < p.N; i += 4 * by) {
                Four was[4] = {};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (i + k * by < last) was[k].load(p.out, p.out_dt, (int64_t)(m0 + (i + k * by >> 6)) * p.out_stride + col);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (i + k * by >= last) continue;
                    const int row = i + k * by >> 6;
                    const uint4 w = was[k].w;
                    float y[4];
                    add_up<4>(p, base + row * 1024 + ((i & 63) ^ (row & 7)) * 16, rank, 2, y);
                    y[0] += was[k].value(p.out_dt, w.x), y[1] += was[k].value(p.out_dt, w.y), y[2] += was[k].value(p.out_dt, w.z), y[3] += was[k].value(p.out_dt, w.w);
                    finish4(p, m0 + row, col, whole, false, y);
                }
            }
        } else
#pragma unroll 2
            for (int i = first; i < last; i += by) {
                const int row = i >> 6, piece = i & 63, col = n0 + piece * 4;
                if (col >= p.N) continue;
                float y[4];
                add_up<4>(p, base + row * 1024 + (piece ^ (row & 7)) * 16, rank, 2, y);
                finish4(p, m0 + row, col, whole, p.add, y);
            }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync_all();      // nobody leaves while the other may still signal its barriers or read its tiles
    if (*abort_s != 0) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // leave time for copies and products still in flight, then report
        if (threadIdx.x == 0) atomicCAS(&g_f8_status, 0, *abort_s);
        __syncthreads();
    }
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// ---- host -------------------------------------------------------------------------------------------------------------------------------

bool codes_map(CUtensorMap* tm, const void* ptr, int64_t stride, int rows, int K, int box_rows) {
    EncodeTiledFn enc = encode_fn();
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(rows > 1 ? stride : (K + 15) / 16 * 16)};
    const cuuint32_t box[2] = {kBlock, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc && enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                      CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Clusters of 2 .. 8 CTAs, one to an SM, that the current device holds at once, for few and many tokens. A cluster lies in one group of SMs, so that there
// is room for fewer than the SMs' number says.
template <bool MANY, typename... P> int clusters_at_once(void (*kern)(P...), int threads, const int** room) {
    constexpr int smem = 227 * 1024;      // an SM has one such CTA
    static ClusterRoom rooms;
    int dev = 0;
    if (cudaError_t e = cudaGetDevice(&dev)) return (int)e;
    const int rc = rooms.get(dev, [&](int ctas, int& n) {
        if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) return (int)e;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute at;
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = (unsigned)ctas, at.val.clusterDim.y = 1, at.val.clusterDim.z = 1;
        cfg.attrs = &at, cfg.numAttrs = 1;
        return (int)cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
    }, room);
    if (rc != 0) (void)cudaGetLastError();      // the call returns it; no later launch is to find it
    return rc;
}

template <int NT> int launch_few(const void* x, int64_t x_stride, const void* W, F8Params& p, cudaStream_t st) {
    using L = Few<NT>;
    CUtensorMap tx, tw;
    if (!codes_map(&tx, x, x_stride, p.M, p.K, NT) || !codes_map(&tw, W, p.K, p.N, p.K, 128)) return -203;
    p.tiles = (p.N + 127) / 128;
    auto kern = f8_few_kernel<NT>;
    // CTAs to a tile: as many as find room at once, with four blocks each; six at most (us with 4 | 5 | 6 | 7 | 8: 16 x 9728 -> 2560 8.7 | 8.4 | 8.0 | 8.9 | 8.5,
    // 1 x 13824 -> 5120 14.3 | 14.0 | 13.9 | 19.4 | 18.1). 16 x 4096, 4 | 5 | 6: 44 tiles 7.9 | 8.0 | 8.0, 46 8.0 | 8.1 | 12.0, 58 8.9 | 13.0. More stages where
    // an SM has one CTA: nothing.
    constexpr int kTwo = 113 * 1024;      // shared memory of a CTA, up to which an SM holds two
    const int* room = nullptr;
    if (int rc = clusters_at_once<false>(kern, L::kThreads, &room)) return rc;
    for (p.splits = 6; p.splits > 1; --p.splits) {
        if (p.groups < p.splits * 4) continue;
        const int to_sm = L::smem((p.groups + p.splits - 1) / p.splits) <= kTwo ? 2 : 1;
        if (p.tiles <= to_sm * room[p.splits]) break;
    }
    p.per = (p.groups + p.splits - 1) / p.splits;
    const int smem = L::smem(p.per);
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024)) return (int)e;
    return launch_pdl_cluster(kern, dim3((unsigned)(p.tiles * p.splits)), L::kThreads, smem, st, p.splits, tx, tw, p);
}
int launch_tile(const void* x, int64_t x_stride, const void* W, F8Params& p, int sms, cudaStream_t st) {
    using L = Tile;
    CUtensorMap tx, tw;
    if (!codes_map(&tx, x, x_stride, p.M, p.K, 128) || !codes_map(&tw, W, p.K, p.N, p.K, 128)) return -203;
    p.m_tiles = (p.M + 255) / 256;
    const int64_t tiles = (int64_t)p.m_tiles * ((p.N + L::kColumns - 1) / L::kColumns);
    if (tiles > INT32_MAX / 2) return -1;      // and so does a tile a round further on
    p.tiles = (int)tiles;
    // pairs to a tile: as many as find room at once, four at most, with four blocks each (128 x 4096, us with 2 | 3 | 4: 15 tiles 18.0 | 15.0 | 13.6, 16 tiles
    // 18.1 | 15.3 | 25.0, 23 tiles 18.4 | 28.6)
    const int* room = nullptr;
    if (int rc = clusters_at_once<true>(f8_tile_kernel<true>, L::kThreads, &room)) return rc;
    for (p.splits = 4; p.splits > 1 && (p.groups < p.splits * 4 || p.tiles > room[2 * p.splits]);) --p.splits;
    p.per = (p.groups + p.splits - 1) / p.splits;
    p.splits = (p.groups + p.per - 1) / p.per;
    const int pairs = p.splits > 1 ? p.tiles * p.splits : p.tiles < sms / 2 ? p.tiles : sms / 2;
    auto kern = p.splits > 1 ? f8_tile_kernel<true> : f8_tile_kernel<false>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem)) return (int)e;
    return launch_pdl_cluster(kern, dim3((unsigned)(2 * pairs)), L::kThreads, L::kSmem, st, 2 * p.splits, tx, tw, p);
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
    // Tokens as the products' N up to 64, in the smallest of three widths, or as their M. us, 16 | 32 | 64 wide | as M: 17 x 2560 -> 19456 - | 11.5 | 15.1 | 26.8, 32 x 5120 ->
    // 13824 - | 15.7 | 16.2 | 25.0, 64 x 5120 -> 13824 - | - | 18.5 | 25.1, 64 x 9728 -> 2560 - | - | 10.2 | 16.7, 64 x 2560 -> 2560 - | - | 6.6 | 10.2.
    if (M <= 16) return launch_few<16>(x, x_stride, W, p, st);
    if (M <= 32) return launch_few<32>(x, x_stride, W, p, st);
    if (M <= 64) return launch_few<64>(x, x_stride, W, p, st);
    const int sms = sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    return launch_tile(x, x_stride, W, p, sms, st);
}
