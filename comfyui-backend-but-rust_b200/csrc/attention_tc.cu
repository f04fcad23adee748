// Attention with many query rows, on tcgen05: the kernel behind gpu_cross_attention and gpu_kv8_attention where tiles of 128 rows fill.
//
// A CTA an SM, persistent, two tiles of 128 query rows at a time over tiles of 128 keys. Per key tile and query tile: S = Q K^T into tensor
// memory (128 columns of f32), p = exp2(S c - m) by one thread a row, p back into the same columns as 16-bit values, O += p V with p as the
// operand from tensor memory. While the softmax warps of one query tile work, the tensor cores multiply for the other. Tensor memory: S of
// both tiles in columns 0..255, O in 256..511.
//
// Warps 0-3 and 4-7: softmax of the two tiles, over the cache also their rows' way out. Warp 8 issues the products (one thread), in the order
// S0 S1 | O0 S0' O1 S1' | ..., in which the tensor cores execute them: S' of the next key tile overwrites p only behind the product that read
// it; the product of the first three quarters of the keys (half, with 64 columns) starts when their p is there. 16-bit keys: warp 9 loads Q, K and V by TMA, warps 10 and 11
// clear hidden rows of V, warps 12-15 carry the rows out (by the softmax warps that took 181 us instead of 131 at 16384 x 512 x 24 heads of
// 128). Cache: warps 12-15 load codes, turn them into halves and write them as TMA would; what they request they take up a step later.
// m follows the running maximum only when that has grown by 2^8: until then p is at most 256 and the sums need no rescaling; O is then scaled
// in tensor memory by the row's own thread, which nothing else touches between the two products of its tile.
// Keys that are not seen get p = 0; what V holds there (16-bit V comes as it lies in memory, NaN perhaps) is overwritten with zeros in shared
// memory before the product.
// Waits are by parity, so no barrier may complete twice before everybody who waits for the first completion has seen it, nor get an arrival meant
// for the next. s_full is the tight one: an item's first logits are issued without a wait for the softmax warps, so "O is done" has a barrier of
// its own (o_full). Between two completions of s_full there is the p_full that answers the first, between two of o_full an item's p_full.
// tests/test_attention_order.py goes through the roles' orders.
// Measured: 1.83 us a step of 256 rows, 128 keys and 128 columns (the products 1.1 at the tensor rate, the exponentials as much: 16 a cycle);
// 16384 rows, 24 heads of 128: 2048 keys 1214 TFLOP/s, 512 keys 924, 785 with a mask (720 one call at a time on new inputs). At most 128 keys:
// a chain of two products, softmax and the rows' way for each item. Over the cache, chunks of 1024 tokens 470 TFLOP/s: a step of 128 keys waits
// for the softmax, whose exponentials and products each take a quarter of the time, issue slots 31 %.
// Every wait is bounded; one that runs out is recorded in g_attention_status and the CTA unwinds. Two kinds of wait can be as long as whole items:
// for sums, and for the logits of a second row tile behind items that have none. Their limit counts from the last key tile that was multiplied.
#include "attention.cuh"
#include "umma16.cuh"

namespace {

using namespace b200q;

__device__ int g_attention_status = 0;

constexpr int kTileKeys = 128, kSlots = 4, kBox = 128 * 128;       // a box: 128 rows of 128 bytes, 128-byte swizzle
constexpr float kSlack = 8.f;                                      // by how much (a power of two) p may exceed 1

template <int DP, bool KV8> struct Tc {
    static constexpr int kTile = DP / 64 * kBox;                   // 128 rows of Q, K or V
    static constexpr int kRing = 2 * kTile, kStaging = kRing + kSlots * kTile, kTail = kStaging + (KV8 ? 8 * 2048 : 4 * 4096);
    // barriers and three words | key tile % 4: bits of the keys that are seen | the same as limits of logits (16-bit), or factors of the pages |
    // item of the tile % 2: l of every row (16-bit), or bf16 queries' powers of two
    static constexpr int kWords = kTail + 208, kInfo = kWords + kSlots * 16, kRowInfo = kInfo + kSlots * (KV8 ? 96 : 512);
    static constexpr int kOrder = kRowInfo + 2048, kEnd = kOrder + 128, kSmem = kEnd + 1024;
    static constexpr int kThreads = 512;
    // Quarters of a key tile whose products with V start before the softmax has the rest: what is left of them stands between it and the next
    // logits, which take p's place. 16384 rows, 2048 keys, 128 columns, two | three: 357 | 349 us; 4096 x 4096, 64 columns: 165 | 166.
    static constexpr int kEarly = DP > 64 ? 3 : 2;
    // Registers of the warpgroups (softmax twice, products and loads, codes or rows out): a softmax thread holds a row of 128 logits. Their
    // sum over the threads is what the launch has, 512 x 128.
    static constexpr int kSoftmaxRegs = 184, kIssueRegs = KV8 ? 40 : 56, kLastRegs = KV8 ? 104 : 88;
    static_assert(2 * kSoftmaxRegs + kIssueRegs + kLastRegs == 4 * 128, "register split");
};

__device__ __forceinline__ void tma_prefetch_4d(const void* tmap, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void* tmap, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// A from tensor memory, B from shared memory
__device__ __forceinline__ void umma_16_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "mov.b64 db, {%2, %5};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}"
        ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "r"(accumulate), "r"(kDescHiSw128) : "memory");
}
// V lies with its columns side by side: rows of 64 columns, 8 keys to a swizzle atom (1024 bytes apart, the stride offset); the next 64
// columns are a box further on (the leading offset).
__device__ __forceinline__ uint32_t umma_desc_lo_n_major(uint32_t addr) { return ((addr & 0x3FFFFu) >> 4) | ((uint32_t)(kBox >> 4) << 16); }

// mbar_wait whose limit begins anew whenever *moving has changed
__device__ __forceinline__ bool mbar_wait_moving(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code, const volatile uint32_t* moving) {
    if (mbar_try_wait(bar, parity)) return true;
    uint64_t t0 = 0;
    uint32_t last = 0;
    for (uint32_t it = 1;; ++it) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((it & 63u) == 0u) {
            if (*abort_flag) return false;
            const uint64_t now = globaltimer_ns();
            const uint32_t at = *moving;
            if (t0 == 0 || at != last) t0 = now, last = at;
            else if (now - t0 > kWaitLimitNs) {
                *abort_flag = code;
                return false;
            }
        }
    }
}

struct TcParams {
    AttnParams a;
    int q_tiles;             // pairs of tiles: 256 rows
    uint32_t items;
    int kv_batch, kv_head;   // 0: the batch's (the heads') keys and values are one
    int q_batch, q_head;
};
struct Item {
    int b, h, row0, rows, len, ql, seen, n;      // h: query head, or kv head of packed rows; rows from row0 on; n key tiles
};
// The item of a CTA's r-th round: the rounds run through the CTAs forwards and backwards in turn, so that where the items get smaller, as the
// cache's do, the sums of a CTA's items come out alike.
__device__ __forceinline__ uint32_t item_of(uint32_t r) { return r * gridDim.x + (r & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x); }
template <bool KV8> __device__ __forceinline__ Item item_at(const TcParams& p, uint32_t i, const int* order) {
    Item x;
    const uint32_t heads = KV8 ? p.a.Hkv : p.a.H;
    // Heads next to one another: together they read and write whole rows of Q and of the result. Cache: long sequences first, of each the
    // tiles with most keys.
    const uint32_t rest = i / heads, b = rest / (uint32_t)p.q_tiles, qt = rest - b * p.q_tiles;
    x.h = (int)(i - rest * heads);
    x.b = KV8 && p.a.B <= 32 ? order[b] : (int)b, x.row0 = (int)(KV8 ? p.q_tiles - 1 - qt : qt) * 256;
    x.len = p.a.kv_len ? min(max(gload(p.a.kv_len + x.b), 0), p.a.Lkv) : p.a.Lkv;
    x.ql = p.a.Lq;
    x.seen = x.len;
    if (KV8) {
        const int ratio = p.a.H / p.a.Hkv;
        if (p.a.q_len) x.ql = min(max(gload(p.a.q_len + x.b), 0), p.a.Lq);
        x.rows = min(256, x.ql * ratio - x.row0);
        if (p.a.causal) x.seen = max(0, min(x.len, x.len - x.ql + (x.row0 + x.rows - 1) / ratio + 1));
    } else x.rows = min(256, p.a.Lq - x.row0);
    x.n = x.rows > 0 ? (x.seen + kTileKeys - 1) / kTileKeys : 0;
    return x;
}

template <typename QT, int DP, bool KV8> __global__ void __launch_bounds__(Tc<DP, KV8>::kThreads, 1)
attention_tc_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                    const TcParams p) {
    using L = Tc<DP, KV8>;
    constexpr bool kBf16 = std::is_same<QT, bf16>::value, kBf16Mma = kBf16 && !KV8;
    using T = typename std::conditional<KV8, half, QT>::type;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
    uint8_t* sm = smem_raw + (base - raw);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t bars = base + L::kTail;
    const uint32_t kv_full = bars, kv_empty = bars + 32, q_full = bars + 64, q_empty = bars + 80, s_full = bars + 96, p_full = bars + 112,
                   o_full = bars + 128, o_empty = bars + 144, p_early = bars + 160, v_ready = bars + 176;
    uint32_t* tmem_s = reinterpret_cast<uint32_t*>(sm + L::kTail + 192);
    volatile int* abort_s = reinterpret_cast<volatile int*>(tmem_s + 1);
    volatile uint32_t* moving = tmem_s + 2;                                   // key tiles multiplied
    uint32_t* words = reinterpret_cast<uint32_t*>(sm + L::kWords);            // [key tile % 4][4]: bit = key is seen
    // [key tile % 4]: 16-bit: [key] +inf, or -inf where a key is not seen; cache: [factor, offset, weight][16 keys]
    float* info = reinterpret_cast<float*>(sm + L::kInfo);
    // [n % 2][tile][row]: of a tile's n-th item, counted by each tile for itself, since an item of at most 128 rows has no second tile. Written again
    // for item n + 2 only behind what waited for item n's reader: l behind the logits of n + 2, which are issued behind the sums of n + 1, and those
    // wait for o_empty of n, which the rows' way out gives when it has read; powers behind q_empty of n + 1, whose logits are issued behind p of n.
    float* row_info = reinterpret_cast<float*>(sm + L::kRowInfo);
    if (threadIdx.x == 0) {
        for (int i = 0; i < kSlots; ++i) mbar_init(kv_full + 8 * i, KV8 ? 4 : 1), mbar_init(kv_empty + 8 * i, 1);
        for (int t = 0; t < 2; ++t) mbar_init(q_full + 8 * t, KV8 ? 4 : 1), mbar_init(q_empty + 8 * t, 1), mbar_init(s_full + 8 * t, 2), mbar_init(p_full + 8 * t, 4),
            mbar_init(o_full + 8 * t, 2), mbar_init(o_empty + 8 * t, 4), mbar_init(p_early + 8 * t, 4), mbar_init(v_ready + 8 * t, 2);
        *abort_s = 0, *moving = 0;
        fence_mbar_init();
        if (!KV8) prefetch_tmap(&tmap_q), prefetch_tmap(&tmap_k), prefetch_tmap(&tmap_v);
    }
    if (warp == 8) {
        tmem_alloc(smem_u32(tmem_s), 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_s;
    pdl_wait();
    const int D = p.a.D;
    int* order = reinterpret_cast<int*>(sm + L::kOrder);      // sequences by length, the longest first
    if (KV8 && p.a.B <= 32) {
        if (warp == 0) {
            const int mine = lane < p.a.B ? gload(p.a.kv_len + lane) : INT32_MIN;
            int rank = 0;
            for (int j = 0; j < p.a.B; ++j) {
                const int other = __shfl_sync(0xffffffffu, mine, j);
                rank += other > mine || (other == mine && j < lane);
            }
            if (lane < p.a.B) order[rank] = lane;
        }
        __syncthreads();
    }

    if (warp < 8) {
        more_registers<L::kSoftmaxRegs>();
        // ---- softmax of tile t, one row a thread
        const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, ratio = KV8 ? p.a.H / p.a.Hkv : 1;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16, s_at = tmem + lanes + t * 128, o_at = tmem + lanes + 256 + t * 128;
        const float c = p.a.scale * kLog2e;
        uint8_t* stage = sm + L::kStaging + warp * 2048;
        uint32_t s_phase = 0, tile_no = 0, item_no = 0;
        bool ok = true;
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            if (x.n > 0 && t * 128 >= x.rows) {
                tile_no += x.n;
                continue;
            }
            if (x.rows <= 0 || (!KV8 && x.n == 0)) continue;
            float m = -INFINITY, l = 0.f, factor = 1.f;
            // keys that this row sees
            const int bound = KV8 && p.a.causal ? x.len - x.ql + (x.row0 + t * 128 + row) / ratio + 1 : x.seen;
            for (int j = 0; j < x.n; ++j, ++tile_no) {
                if (!__all_sync(0xffffffffu, mbar_wait_moving(s_full + 8 * t, s_phase, abort_s, ST_TIMEOUT_TMEM_FULL, moving))) { ok = false; break; }
                s_phase ^= 1;
                tc_fence_after();
                const uint32_t* w = words + (tile_no & 3) * 4;
                const float* in = info + (tile_no & 3) * (KV8 ? 24 : 128);
                if (KV8 && kBf16 && j == 0) factor = row_info[(item_no & 1) * 256 + t * 128 + row];
                const int limit = bound - j * kTileKeys;
                const bool all = (w[0] & w[1] & w[2] & w[3]) == 0xffffffffu && (!KV8 || __all_sync(0xffffffffu, limit >= kTileKeys));
                // logits: in powers of two for the cache, without the factor c for 16-bit keys (the exponent's product applies it)
                float v[128];
#pragma unroll
                for (int q = 0; q < 4; ++q) tmem_ld32(s_at + q * 32, reinterpret_cast<uint32_t(&)[32]>(v[q * 32]));
                tmem_ld_wait();
                if (KV8) {
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        const uint64_t mul = pack_f32(in[q] * factor, in[q] * factor), add = pack_f32(in[8 + q], in[8 + q]);
#pragma unroll
                        for (int e = 0; e < 16; e += 2)
                            unpack_f32(fma_f32x2(pack_f32(v[q * 16 + e], v[q * 16 + e + 1]), mul, add), v[q * 16 + e], v[q * 16 + e + 1]);
                    }
                }
                if (!all) {
                    if (KV8) {      // pages that there are not: groups of 16 keys; then the row's own bound
#pragma unroll
                        for (int q = 0; q < 8; ++q) {
                            const int end = w[q >> 1] >> (q & 1) * 16 & 1 ? limit - q * 16 : 0;
#pragma unroll
                            for (int e = 0; e < 16; ++e) v[q * 16 + e] = e < end ? v[q * 16 + e] : -INFINITY;
                        }
                    } else {        // the smaller of logit and limit: -inf also for what is no number
#pragma unroll
                        for (int q = 0; q < 32; ++q) {
                            const float4 f = reinterpret_cast<const float4*>(in)[q];
                            v[q * 4] = fminf(v[q * 4], f.x), v[q * 4 + 1] = fminf(v[q * 4 + 1], f.y);
                            v[q * 4 + 2] = fminf(v[q * 4 + 2], f.z), v[q * 4 + 3] = fminf(v[q * 4 + 3], f.w);
                        }
                    }
                }
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 128; e += 8)
#pragma unroll
                    for (int f = 0; f < 4; ++f) tops[f] = fmaxf(tops[f], fmaxf(v[e + 2 * f], v[e + 2 * f + 1]));
                float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                if (!KV8) top *= c;
                const bool grew = top > m + kSlack;
                if (__any_sync(0xffffffffu, grew)) {
                    const float keep = grew ? exp2_fast(m - top) : 1.f;
                    if (grew) m = top;
                    l *= keep;
                    if (j > 0) {
#pragma unroll 1
                        for (int q = 0; q < DP / 32; ++q) {
                            uint32_t r[32];
                            tmem_ld32(o_at + q * 32, r);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * keep);
                            tmem_st32(o_at + q * 32, r);
                        }
                    }
                }
                const float shift = m == -INFINITY ? 0.f : m;
                const uint64_t minus = pack_f32(-shift, -shift), by = pack_f32(c, c);
                uint64_t sum[2] = {};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t out[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        float a, b;
                        const uint64_t x = pack_f32(v[q * 32 + e], v[q * 32 + e + 1]);
                        unpack_f32(KV8 ? add_f32x2(x, minus) : fma_f32x2(x, by, minus), a, b);
                        a = exp2_fast(a), b = exp2_fast(b);
                        const float wt = KV8 ? in[16 + q * 2 + (e >> 4)] : 0.f;
                        sum[e >> 1 & 1] = KV8 ? fma_f32x2(pack_f32(a, b), pack_f32(wt, wt), sum[e >> 1 & 1]) : add_f32x2(pack_f32(a, b), sum[e >> 1 & 1]);
                        out[e >> 1] = pack2<T>(a, b);
                    }
                    tmem_st16(s_at + q * 16, out);
                    if (q == 3) {
                        float even, odd;
                        unpack_f32(add_f32x2(sum[0], sum[1]), even, odd);
                        l += even + odd;
                        // l for the rows' way out, announced with p: an arrival of its own behind p could be that of a warp which is an item ahead, in
                        // place of one that is late (2 x 4096 x 77 15.5 us instead of 15.2, 16384 x 512 130.6 instead of 130.1)
                        if (!KV8 && j + 1 == x.n) row_info[(item_no++ & 1) * 256 + t * 128 + row] = l;
                    }
                    if (q == L::kEarly - 1 || q == 3) {
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive((q < 3 ? p_early : p_full) + 8 * t);
                    }
                }
            }
            if (!ok) break;
            if (!KV8) continue;
            // ---- the rows out: 32 columns at a time through this warp's staging, so that a row's pieces are stored together
            if (x.n > 0) {
                if (!__all_sync(0xffffffffu, mbar_wait(o_full + 8 * t, item_no & 1, abort_s, ST_TIMEOUT_TMEM_FULL))) break;
                ++item_no;
                tc_fence_after();
            }
            const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
            for (int q = 0; q * 32 < D; ++q) {
                uint32_t r[32] = {};
                if (x.n > 0) {
                    tmem_ld32(o_at + q * 32, r);
                    tmem_ld_wait();
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint4 v;
                    uint32_t* o = reinterpret_cast<uint32_t*>(&v);
                    // (l = 0: the columns may hold anything, an earlier row's infinity among it)
#pragma unroll
                    for (int f = 0; f < 4; ++f)
                        o[f] = inv == 0.f && l == 0.f ? 0u : pack2<QT>(__uint_as_float(r[e * 8 + 2 * f]) * inv, __uint_as_float(r[e * 8 + 2 * f + 1]) * inv);
                    *reinterpret_cast<uint4*>(stage + lane * 64 + ((e ^ (lane >> 1)) & 3) * 16) = v;
                }
                __syncwarp();
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int rr = k * 8 + (lane >> 2), e = lane & 3, at = t * 128 + quarter * 32 + rr, d = q * 32 + e * 8;
                    if (at < x.rows && d < D) {
                        const int gr = x.row0 + at, query = KV8 ? gr / ratio : gr, head = KV8 ? x.h * ratio + gr % ratio : x.h;
                        QT* dst = reinterpret_cast<QT*>(p.a.out) + x.b * p.a.os[0] + query * p.a.os[1] + head * p.a.os[2] + d;
                        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(stage + rr * 64 + ((e ^ (rr >> 1)) & 3) * 16);
                    }
                }
                __syncwarp();
            }
            tc_fence_before();
        }
    } else if (warp < 12) {
      fewer_registers<L::kIssueRegs>();
      if (warp == 8) {
        // ---- products
        const uint32_t idesc_s = umma_idesc_16(kBf16Mma, false, 128, kTileKeys), idesc_o = umma_idesc_16(kBf16Mma, true, 128, DP);
        const bool one = elect_one();
        uint32_t kv_no = 0, q_no[2] = {}, p_phase[2] = {}, o_phase[2] = {1, 1};
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity, int code) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, code)); };
        auto issue_s = [&](int t, uint32_t slot) {
            const uint32_t q = umma_desc_lo(base + t * L::kTile), k = umma_desc_lo(base + L::kRing + slot * L::kTile);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
                const uint32_t step = (kk & 3) * 2 + (kk >> 2) * (kBox >> 4);
                umma_16_ss(tmem + t * 128, q + step, k + step, idesc_s, kk > 0);
            }
        };
        auto announce = [&](uint32_t bar) {      // one arrival when the products are done, one that orders what this warp has seen in shared memory
            umma_commit(bar);
            mbar_arrive(bar);
        };
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            if (x.n == 0) continue;
            const int tiles = x.rows > 128 ? 2 : 1;
            uint32_t ks = kv_no & 3, k_phase = kv_no >> 2 & 1;
            if (!wait(kv_full + 8 * ks, k_phase, ST_TIMEOUT_FULL)) break;
            for (int t = 0; t < tiles; ++t) {
                if (!wait(q_full + 8 * t, q_no[t] & 1, ST_TIMEOUT_FULL)) break;
                ++q_no[t];
                tc_fence_after();
                if (one) {
                    issue_s(t, ks);
                    if (x.n == 1) umma_commit(q_empty + 8 * t);
                    announce(s_full + 8 * t);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (one) umma_commit(kv_empty + 8 * ks);
            for (int j = 0; j < x.n; ++j) {
                const uint32_t v_no = kv_no + 1, vs = v_no & 3;
                const bool more = j + 1 < x.n;
                if (!wait(kv_full + 8 * vs, v_no >> 2 & 1, ST_TIMEOUT_FULL)) break;
                if (!KV8 && !wait(v_ready + 8 * (vs >> 1), v_no >> 2 & 1, ST_TIMEOUT_UNPACK)) break;
                ks = (kv_no + 2) & 3, k_phase = (kv_no + 2) >> 2 & 1;
                for (int t = 0; t < tiles; ++t) {
                    if (!wait(p_early + 8 * t, p_phase[t], ST_TIMEOUT_TMEM_EMPTY)) break;
                    if (!KV8 && j == 0) {      // the rows before have left O
                        if (!wait(o_empty + 8 * t, o_phase[t], ST_TIMEOUT_TMEM_EMPTY)) break;
                        o_phase[t] ^= 1;
                    }
                    const uint32_t v = umma_desc_lo_n_major(base + L::kRing + vs * L::kTile);
                    tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int kk = 0; kk < 2 * L::kEarly; ++kk)      // 16 keys: 8 columns of p, two swizzle atoms of V
                            umma_16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v + kk * (2048 >> 4), idesc_o, j > 0 || kk > 0);
                    }
                    __syncwarp();
                    if (!wait(p_full + 8 * t, p_phase[t], ST_TIMEOUT_TMEM_EMPTY)) break;
                    p_phase[t] ^= 1;
                    if (more && t == 0 && !wait(kv_full + 8 * ks, k_phase, ST_TIMEOUT_FULL)) break;
                    tc_fence_after();
                    if (one) {
#pragma unroll
                        for (int kk = 2 * L::kEarly; kk < 8; ++kk) umma_16_ts(tmem + 256 + t * 128, tmem + t * 128 + kk * 8, v + kk * (2048 >> 4), idesc_o, 1);
                        if (more) {
                            issue_s(t, ks);
                            if (j + 2 == x.n) umma_commit(q_empty + 8 * t);
                        }
                        announce((more ? s_full : o_full) + 8 * t);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                if (one) {
                    umma_commit(kv_empty + 8 * vs);
                    if (more) umma_commit(kv_empty + 8 * ks);
                }
                kv_no += 2;
                if (one) *moving = kv_no;
            }
        }
      } else if (!KV8 && warp == 9) {
        // ---- loads
        uint32_t kv_no = 0, q_no[2] = {}, tile_no = 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, ST_TIMEOUT_EMPTY)); };
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            if (x.n == 0) continue;
            const int tiles = x.rows > 128 ? 2 : 1, kvh = x.h / (p.a.H / p.a.Hkv);
            auto load_kv = [&](int j, int which) {
                const uint32_t slot = kv_no & 3;
                if (!wait(kv_empty + 8 * slot, (kv_no >> 2 & 1) ^ 1)) return;
                if (which == 0) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int key = j * kTileKeys + q * 32 + lane;
                        const bool seen = key < x.seen && (!p.a.mask || gload(p.a.mask + x.b * p.a.mask_stride + key) != 0);
                        const uint32_t w = __ballot_sync(0xffffffffu, seen);
                        if (lane == 0) words[(tile_no & 3) * 4 + q] = w;
                        info[(tile_no & 3) * 128 + q * 32 + lane] = seen ? INFINITY : -INFINITY;
                    }
                    __syncwarp();
                }
                if (lane == 0) {
                    mbar_arrive_expect_tx(kv_full + 8 * slot, L::kTile);
#pragma unroll
                    for (int box = 0; box < DP / 64; ++box)
                        tma_load_4d(base + L::kRing + slot * L::kTile + box * kBox, which ? &tmap_v : &tmap_k, box * 64, j * kTileKeys, kvh * p.kv_head, x.b * p.kv_batch,
                                    kv_full + 8 * slot);
                }
                __syncwarp();
                ++kv_no;
            };
            load_kv(0, 0);      // before Q, whose place is free only when the last product of the item before has read it
            for (int t = 0; t < tiles && ok; ++t) {
                if (!wait(q_empty + 8 * t, (q_no[t] & 1) ^ 1)) break;
                ++q_no[t];
                if (lane == 0) {
                    mbar_arrive_expect_tx(q_full + 8 * t, L::kTile);
#pragma unroll
                    for (int box = 0; box < DP / 64; ++box)
                        tma_load_4d(base + t * L::kTile + box * kBox, &tmap_q, box * 64, x.row0 + t * 128, x.h * p.q_head, x.b * p.q_batch, q_full + 8 * t);
                }
                __syncwarp();
            }
            if (ok) load_kv(0, 1);
            ++tile_no;
            if (lane == 0 && item_of(r + 1) < p.items) {      // the next item's queries to L2
                const Item y = item_at<KV8>(p, item_of(r + 1), order);
                for (int t = 0; t < 2 && t * 128 < y.rows; ++t)
#pragma unroll
                    for (int box = 0; box < DP / 64; ++box) tma_prefetch_4d(&tmap_q, box * 64, y.row0 + t * 128, y.h * p.q_head, y.b * p.q_batch);
            }
            __syncwarp();
            for (int j = 1; j < x.n && ok; ++j, ++tile_no) {
                load_kv(j, 0);
                if (ok) load_kv(j, 1);
            }
        }
      } else if (!KV8) {
        // ---- rows of V behind keys that are not seen: zeros. Two warps, 16 lanes (8 with 64 columns) to a row.
        uint32_t kv_no = 1, tile_no = 0;
        bool ok = true;
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            for (int j = 0; j < x.n; ++j, ++tile_no, kv_no += 2) {
                const uint32_t slot = kv_no & 3;
                if (!(ok = __all_sync(0xffffffffu, mbar_wait(kv_full + 8 * slot, kv_no >> 2 & 1, abort_s, ST_TIMEOUT_FULL)))) break;
                const uint32_t* w = words + (tile_no & 3) * 4;
                if ((w[0] & w[1] & w[2] & w[3]) != 0xffffffffu) {
                    constexpr int kLanes = DP / 8;
                    const int piece = lane % kLanes, there = min(kTileKeys, p.a.Lkv - j * kTileKeys);      // the rest is zeros already
                    uint8_t* tile = sm + L::kRing + slot * L::kTile + (piece >> 3) * kBox + (piece & 7) * 16;
                    for (int key = ((warp - 10) * 32 + lane) / kLanes; key < there; key += 64 / kLanes)
                        if (!(w[key >> 5] >> (key & 31) & 1)) *reinterpret_cast<uint4*>(tile + key * 128) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(v_ready + 8 * (slot >> 1));
            }
        }
      }
    } else if (!KV8) {
        // ---- the rows' way out: 64 columns at a time through this warp's staging, so that a row's pieces are stored together
        fewer_registers<L::kLastRegs>();
        const int quarter = warp & 3;
        uint8_t* stage = sm + L::kStaging + quarter * 4096;
        uint32_t phase[2] = {}, item_no[2] = {};
        bool ok = true;
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            for (int t = 0; t < 2 && t * 128 < x.rows; ++t) {
                float inv = 0.f;
                if (x.n > 0) {
                    if (!(ok = __all_sync(0xffffffffu, mbar_wait_moving(o_full + 8 * t, phase[t], abort_s, ST_TIMEOUT_TMEM_FULL, moving)))) break;
                    phase[t] ^= 1;
                    tc_fence_after();
                    const float l = row_info[(item_no[t]++ & 1) * 256 + t * 128 + quarter * 32 + lane];
                    inv = l > 0.f || l != l ? 1.f / l : 0.f;      // 0: zeros, whatever the sums hold
                }
                const int left = min(32, x.rows - t * 128 - quarter * 32);      // rows of this warp; none: nothing is stored
                QT* dst = reinterpret_cast<QT*>(p.a.out) + x.b * p.a.os[0] + (x.row0 + t * 128 + quarter * 32) * p.a.os[1] + x.h * p.a.os[2];
#pragma unroll
                for (int q = 0; q < DP / 64; ++q) {
                    uint32_t r[2][32];
                    if (x.n > 0) {
                        tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + 256 + t * 128 + q * 64, r[0]);
                        tmem_ld32(tmem + ((uint32_t)(quarter * 32) << 16) + 256 + t * 128 + q * 64 + 32, r[1]);
                        tmem_ld_wait();
                        if (q == DP / 64 - 1) {      // the next item's products may have O
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(o_empty + 8 * t);
                        }
                    }
                    if (__any_sync(0xffffffffu, inv == 0.f)) {      // no key seen: the columns may hold anything
#pragma unroll
                        for (int e = 0; e < 64; ++e) r[e >> 5][e & 31] = inv == 0.f ? 0u : r[e >> 5][e & 31];
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint4 v;
                        uint32_t* o = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            o[f] = pack2<QT>(__uint_as_float(r[e >> 2][(e & 3) * 8 + 2 * f]) * inv, __uint_as_float(r[e >> 2][(e & 3) * 8 + 2 * f + 1]) * inv);
                        *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ lane) & 7) * 16) = v;
                    }
                    __syncwarp();
                    const int e = lane & 7, d = q * 64 + e * 8;
                    uint4 row[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) row[k] = *reinterpret_cast<const uint4*>(stage + (k * 4 + (lane >> 3)) * 128 + ((e ^ (k * 4 + (lane >> 3))) & 7) * 16);
                    QT* out = dst + (lane >> 3) * p.a.os[1] + d;
#pragma unroll
                    for (int k = 0; k < 8; ++k, out += 4 * p.a.os[1])
                        if (k * 4 + (lane >> 3) < left && d < D) *reinterpret_cast<uint4*>(out) = row[k];
                    __syncwarp();
                }
            }
        }
    } else {
        fewer_registers<L::kLastRegs>();
        // ---- codes to halves: four warps of 32 keys (or query rows) each
        const int w = warp - 12;
        uint32_t kv_no = 0, q_no[2] = {}, tile_no = 0;
        bool ok = true;
        auto wait = [&](uint32_t bar, uint32_t parity) { return ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_s, ST_TIMEOUT_EMPTY)); };
        auto done = [&](uint32_t bar) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        auto put = [&](uint8_t* tile, int row, int piece, uint4 v) {      // 8 values: piece `piece` of a row of 16-bit values
            *reinterpret_cast<uint4*>(tile + (piece >> 3) * kBox + row * 128 + ((piece ^ row) & 7) * 16) = v;
        };
        const int ratio = p.a.H / p.a.Hkv;
        for (uint32_t r = 0; item_of(r) < p.items && ok; ++r) {
            const Item x = item_at<KV8>(p, item_of(r), order);
            if (x.n == 0) continue;
            const int tiles = x.rows > 128 ? 2 : 1;
            for (int t = 0; t < tiles; ++t) {
                if (!wait(q_empty + 8 * t, (q_no[t] & 1) ^ 1)) break;
                const uint32_t item_no = q_no[t]++;
                constexpr int kLanes = DP / 8, kAtOnce = 32 / kLanes;        // lanes to a row, rows to an instruction
#pragma unroll 4
                for (int k = 0; k < 32 / kAtOnce; ++k) {
                    const int row = w * 32 + k * kAtOnce + lane / kLanes, piece = lane % kLanes, at = t * 128 + row, gr = x.row0 + at;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (at < x.rows && piece * 8 < D)
                        v = gload(reinterpret_cast<const uint4*>(reinterpret_cast<const QT*>(p.a.q) + x.b * p.a.qs[0] + (gr / ratio) * p.a.qs[1] +
                                                                 (x.h * ratio + gr % ratio) * p.a.qs[2]) + piece);
                    if (kBf16) {
                        const QT* y = reinterpret_cast<const QT*>(&v);
                        float top = 0.f;
#pragma unroll
                        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(to_f<QT>(y[e])));
#pragma unroll
                        for (int o = 1; o < kLanes; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                        const int e2 = row_exponent(top);
                        const float mult = __uint_as_float((uint32_t)(127 + e2) << 23);
                        if (piece == 0) row_info[(item_no & 1) * 256 + t * 128 + row] = __uint_as_float((uint32_t)(127 - e2) << 23);
                        uint4 z;
                        uint32_t* o = reinterpret_cast<uint32_t*>(&z);
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[e] = pack2<half>(to_f<QT>(y[2 * e]) * mult, to_f<QT>(y[2 * e + 1]) * mult);
                        v = z;
                    }
                    put(sm + t * L::kTile, row, piece, v);
                }
                done(q_full + 8 * t);
            }
            // Nothing is waited for when it is requested: a tile's page indices two tiles ahead, its scales one, its codes (K and V) as soon as the
            // tile before has been converted.
            constexpr int kLanes = DP / 16, kAtOnce = 32 / kLanes;
            auto page_of = [&](int j) {      // this warp's 32 keys of a tile: one to a lane
                const int key = j * kTileKeys + w * 32 + lane;
                return key < x.seen ? gload(p.a.table + x.b * p.a.table_stride + key / p.a.T) : -1;
            };
            auto offset_of = [&](int j, int page) {
                const int key = j * kTileKeys + w * 32 + lane;
                return page >= 0 && page < p.a.pages ? (((int64_t)page * p.a.Hkv + x.h) * p.a.T + key % p.a.T) * D : (int64_t)-1;
            };
            auto scales_of = [&](int page, float& k, float& v) {
                const bool there = page >= 0 && page < p.a.pages;
                k = there ? gload(p.a.k_scale + (int64_t)page * p.a.Hkv + x.h) : 0.f, v = there ? gload(p.a.v_scale + (int64_t)page * p.a.Hkv + x.h) : 1.f;
            };
            auto request = [&](uint4 (&code)[32 / kAtOnce], int64_t offs, int which) {
                const int8_t* src = reinterpret_cast<const int8_t*>(which ? p.a.v : p.a.k);
                const int piece = lane % kLanes;
#pragma unroll
                for (int k = 0; k < 32 / kAtOnce; ++k) {
                    const int64_t o = __shfl_sync(0xffffffffu, offs, k * kAtOnce + lane / kLanes);
                    code[k] = o >= 0 && piece * 16 < D ? gload(reinterpret_cast<const uint4*>(src + o) + piece) : make_uint4(0, 0, 0, 0);
                }
            };
            auto convert = [&](const uint4 (&code)[32 / kAtOnce], uint32_t slot) {
                uint8_t* tile = sm + L::kRing + slot * L::kTile;
                const int piece = lane % kLanes;
#pragma unroll
                for (int k = 0; k < 32 / kAtOnce; ++k) {
                    const int row = w * 32 + k * kAtOnce + lane / kLanes;
                    const uint2 a = halves_of4(code[k].x), b = halves_of4(code[k].y), e = halves_of4(code[k].z), f = halves_of4(code[k].w);
                    put(tile, row, 2 * piece, make_uint4(a.x, a.y, b.x, b.y));
                    put(tile, row, 2 * piece + 1, make_uint4(e.x, e.y, f.x, f.y));
                }
                done(kv_full + 8 * slot);
            };
            uint4 kc[32 / kAtOnce], vc[32 / kAtOnce];
            float k_scale, v_scale;
            int page = page_of(0), page_next = page_of(1);
            int64_t off = offset_of(0, page);
            request(kc, off, 0);
            request(vc, off, 1);
            scales_of(page, k_scale, v_scale);
            for (int j = 0; j < x.n && ok; ++j, ++tile_no) {
                uint32_t slot = kv_no & 3;
                if (!wait(kv_empty + 8 * slot, (kv_no >> 2 & 1) ^ 1)) break;
                ++kv_no;
                const uint32_t seen = __ballot_sync(0xffffffffu, off >= 0);
                if (lane == 0) words[(tile_no & 3) * 4 + w] = seen;
                if ((lane & 15) == 0) {
                    float* in = info + (tile_no & 3) * 24 + w * 2 + (lane >> 4);
                    in[0] = k_scale * (p.a.scale * kLog2e), in[8] = v_scale_log2(v_scale), in[16] = v_scale_weight(v_scale);
                }
                convert(kc, slot);
                page = page_next, off = offset_of(j + 1, page);      // past the last tile: no key is seen, nothing is requested
                request(kc, off, 0);
                scales_of(page, k_scale, v_scale);
                page_next = page_of(j + 2);
                slot = kv_no & 3;
                if (!wait(kv_empty + 8 * slot, (kv_no >> 2 & 1) ^ 1)) break;
                ++kv_no;
                convert(vc, slot);
                request(vc, off, 1);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (*abort_s != 0) {
        for (int i = 0; i < 2000; ++i) __nanosleep(1000);      // leave time for copies and products still in flight, then report
        if (threadIdx.x == 0) atomicCAS(&g_attention_status, 0, *abort_s);
        __syncthreads();
    }
    if (warp == 8) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------------------

// Rows [B, L, H, D] of 16-bit values as boxes of 64 columns by 128 rows; columns and rows outside read as zeros. A dimension without a
// stride is one entry.
bool make_rows_map(CUtensorMap* tm, const void* ptr, const int64_t (&s)[3], int B, int L, int H, int D) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return false;
    auto dim = [](int64_t stride, int n) { return (cuuint64_t)(stride ? n : 1); };
    auto pitch = [](int64_t stride) { return (cuuint64_t)(stride ? stride * 2 : 16); };
    const cuuint64_t dims[4] = {(cuuint64_t)D, dim(s[1], L), dim(s[2], H), dim(s[0], B)}, strides[3] = {pitch(s[1]), pitch(s[2]), pitch(s[0])};
    const cuuint32_t box[4] = {64, 128, 1, 1}, estr[4] = {1, 1, 1, 1};
    return enc(tm, CU_TENSOR_MAP_DATA_TYPE_UINT16, 4, const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename QT, int DP, bool KV8> int launch_tc(const CUtensorMap (&tm)[3], const TcParams& p, cudaStream_t st) {
    using L = Tc<DP, KV8>;
    auto kern = attention_tc_kernel<QT, DP, KV8>;
    if (cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem)) return (int)e;
    const int sms = sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    return launch_pdl(kern, dim3(p.items < (uint32_t)sms ? p.items : (uint32_t)sms), L::kThreads, L::kSmem, st, tm[0], tm[1], tm[2], p);
}

}  // namespace

bool b200q::attention_tc_takes(const AttnParams& p, bool kv8) {
    if (p.D > 128 || !(p.scale > 0.f) || p.Lkv <= 0 || p.Lkv > 1 << 26) return false;
    // Half an item's rows at least, and enough tiles of 64 rows: with fewer the other kernels, which share a row tile's keys among CTAs, are
    // done sooner. Over the cache, 8 sequences of 1000 to 8000 tokens and 128 rows for each of 8 kv heads (128 tiles): 219 us here, 124 with 16 rows at
    // a time; one sequence of 8000 and 256 rows: 232 and 63; two of up to 4133 and 4096 rows (1024 tiles): 148 here.
    const int64_t rows = kv8 ? (int64_t)p.Lq * (p.H / p.Hkv) : p.Lq;
    const int64_t few = (kv8 ? 160 : 64) - 1;
    if (rows < 128 || (rows + 63) / 64 <= few / p.B / (kv8 ? p.Hkv : p.H)) return false;
    // rows without a stride between them have no tensor map
    return kv8 || ((p.Lq == 1 || p.qs[1] > 0) && (p.Lkv == 1 || (p.ks[1] > 0 && p.vs[1] > 0)) && p.qs[0] >= 0 && p.qs[2] >= 0 && p.ks[0] >= 0 &&
                   p.ks[2] >= 0 && p.vs[0] >= 0 && p.vs[2] >= 0 && (p.ks[0] == 0) == (p.vs[0] == 0) && (p.ks[2] == 0) == (p.vs[2] == 0));
}

int b200q::attention_tc(int dtype, bool kv8, AttnParams& a, cudaStream_t st) {
    TcParams p = {};
    p.a = a;
    const int64_t rows = kv8 ? (int64_t)a.Lq * (a.H / a.Hkv) : a.Lq, tiles = (rows + 255) / 256;
    const int heads = kv8 ? a.Hkv : a.H;
    if (rows > INT32_MAX - 512 || tiles > INT32_MAX / 2 / a.B / heads) return -1;
    p.q_tiles = (int)tiles, p.items = (uint32_t)(tiles * a.B * heads);
    p.q_batch = a.qs[0] != 0, p.q_head = a.qs[2] != 0, p.kv_batch = a.ks[0] != 0, p.kv_head = a.ks[2] != 0;
    CUtensorMap tm[3] = {};
    if (!kv8 && (!make_rows_map(&tm[0], a.q, a.qs, a.B, a.Lq, a.H, a.D) || !make_rows_map(&tm[1], a.k, a.ks, a.B, a.Lkv, a.Hkv, a.D) ||
                 !make_rows_map(&tm[2], a.v, a.vs, a.B, a.Lkv, a.Hkv, a.D)))
        return -203;
    const bool h = dtype == DT_F16, wide = a.D > 64;
    if (kv8) return h ? (wide ? launch_tc<half, 128, true>(tm, p, st) : launch_tc<half, 64, true>(tm, p, st))
                      : (wide ? launch_tc<bf16, 128, true>(tm, p, st) : launch_tc<bf16, 64, true>(tm, p, st));
    return h ? (wide ? launch_tc<half, 128, false>(tm, p, st) : launch_tc<half, 64, false>(tm, p, st))
             : (wide ? launch_tc<bf16, 128, false>(tm, p, st) : launch_tc<bf16, 64, false>(tm, p, st));
}

int b200q::attention_status_read_clear(int* out) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_attention_status, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_attention_status, &zero, sizeof(int));
    if (e != cudaSuccess) return (int)e;
    *out = v;
    return 0;
}
