// A cache of keys and values in 8 bits (no counterpart in the reference's path; it keeps such a cache inside one video model's kernels).
//
//   gpu_kv8_append    new rows of each sequence onto its pages
//   gpu_kv8_dequant   a sequence's rows back in floating point
//
// k8, v8 int8 [pages, Hkv, T, D], one f32 scale for each page and head: a value is code * scale. Sequence b's token i is row i % T of page
// table[b, i / T]. The T rows of a page and head are contiguous: what attention reads for one head is whole runs of T * D bytes.
#include "attention.cuh"

namespace {

using namespace b200q;

struct AppendParams {
    const void *k, *v;
    int64_t ks[3], vs[3];            // strides of batch, row, head in elements
    int8_t *k8, *v8;
    float *k_scale, *v_scale;
    const int32_t *table, *start, *count;
    int64_t table_stride, pages;
    int B, L, Hkv, D, T, max_pages, touched;      // touched: pages that L rows can reach
};

__device__ __forceinline__ uint32_t pack4(const float* c) {
    return ((uint32_t)(int)c[0] & 255u) | ((uint32_t)(int)c[1] & 255u) << 8 | ((uint32_t)(int)c[2] & 255u) << 16 | (uint32_t)(int)c[3] << 24;
}
// codes rint(value / scale), NaN -> 0
__device__ __forceinline__ uint2 codes_of(const float (&v)[8], float s) {
    float c[8];
    rint_quotients<8>(v, s, c);
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = fminf(127.f, fmaxf(-127.f, c[e]));
    return make_uint2(pack4(c), pack4(c + 4));
}

// One CTA for each of K and V, page and head. Twice over the new rows (at most T * D values, so the second time from L1 or L2): their
// largest magnitude, then their codes. A page that was begun before keeps its scale unless the new rows need a larger one; then its old
// codes are rounded to the new one, each time by at most half a step. Latency: a token of 8 sequences 5 us.
template <typename XT> __global__ void __launch_bounds__(256) kv8_append_kernel(const AppendParams p) {
    __shared__ float tops[8];
    pdl_wait();
    const int which = blockIdx.x & 1, h = (blockIdx.x >> 1) % p.Hkv, rest = (blockIdx.x >> 1) / p.Hkv, j = rest % p.touched, b = rest / p.touched;
    const int64_t start = gload(p.start + b);
    const int count = p.count ? min(gload(p.count + b), p.L) : p.L;
    if (start < 0 || count <= 0) return;
    const int64_t slot = start / p.T + j;
    // rows of this page that are new: from..to, the sequence's new row number `from` is src_row
    const int64_t page_at = slot * p.T;
    const int from = (int)max((int64_t)0, start - page_at), to = (int)min((int64_t)p.T, start + count - page_at);
    if (from >= to || slot >= p.max_pages) return;
    const int64_t page = gload(p.table + b * p.table_stride + slot);
    if (page < 0 || page >= p.pages) return;
    const int64_t* xs = which ? p.vs : p.ks;
    const XT* src = reinterpret_cast<const XT*>(which ? p.v : p.k) + b * xs[0] + (page_at + from - start) * xs[1] + h * xs[2];
    int8_t* dst = (which ? p.v8 : p.k8) + (page * p.Hkv + h) * p.T * p.D;
    float* scale = (which ? p.v_scale : p.k_scale) + page * p.Hkv + h;
    const int pieces = p.D / 8, n = (to - from) * pieces;
    float top = 0.f;
    for (int i = threadIdx.x; i < n; i += 256) {
        float v[8];
        load8(src + (int64_t)(i / pieces) * xs[1] + i % pieces * 8, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, tops[w]);
    float s = fmaxf(__fmul_rn(fminf(top, FLT_MAX), 1.f / 127.f), kTiny);
    if (from > 0) {
        const float old = gload(scale);
        s = fmaxf(s, old);
        if (s != old) {      // also for an old scale that is NaN: its codes become zeros
            const float r = __fdiv_rn(old, s);
            for (int i = threadIdx.x; i < from * p.D / 8; i += 256) {
                const uint2 w = gload(reinterpret_cast<const uint2*>(dst) + i);
                float c[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) c[e] = __fmul_rn((float)(int8_t)((e < 4 ? w.x : w.y) >> 8 * (e & 3)), r);
                reinterpret_cast<uint2*>(dst)[i] = codes_of(c, 1.f);
            }
        }
    }
    for (int i = threadIdx.x; i < n; i += 256) {
        float v[8];
        load8(src + (int64_t)(i / pieces) * xs[1] + i % pieces * 8, v);
        reinterpret_cast<uint2*>(dst)[from * pieces + i] = codes_of(v, s);
    }
    __syncthreads();             // everybody has read the old scale
    if (threadIdx.x == 0) *scale = s;
}

struct DequantParams {
    const int8_t *k8, *v8;
    const float *k_scale, *v_scale;
    const int32_t *table, *lengths;
    void *k, *v;
    int64_t table_stride, pages, rows;      // rows to a sequence of the result
    int B, Hkv, D, T, max_pages, page_log, seq_blocks;
};

// A thread has the same 32 bytes of the result in eight rows, which lie on one page; rows behind a sequence's last token, or on a page that
// there is not, are zeros. Threads side by side have neighbouring pieces of a row, of K or of V.
template <typename XT> __global__ void __launch_bounds__(256) kv8_dequant_kernel(const DequantParams p) {
    constexpr int kCodes = 32 / sizeof(XT), kRows = 8;
    pdl_wait();
    const int which = blockIdx.x & 1, b = (int)(blockIdx.x >> 1) / p.seq_blocks;
    const int i = ((int)(blockIdx.x >> 1) - b * p.seq_blocks) * 256 + threadIdx.x, pieces = p.D / kCodes, across = pieces * p.Hkv;
    const int row0 = i / across * kRows, at = i % across, h = at / pieces, c = at % pieces;
    if (row0 >= p.rows) return;
    const int length = gload(p.lengths + b), slot = row0 >> p.page_log;
    int64_t page = -1;
    if (row0 < length && slot < p.max_pages) page = gload(p.table + b * p.table_stride + slot);
    const bool there = page >= 0 && page < p.pages;
    uint32_t w[kRows][kCodes / 4];
    float s = 0.f;
    if (there) {
        const int8_t* src = (which ? p.v8 : p.k8) + ((page * p.Hkv + h) * p.T + (row0 & (p.T - 1))) * p.D + c * kCodes;
        s = gload((which ? p.v_scale : p.k_scale) + page * p.Hkv + h);
#pragma unroll
        for (int r = 0; r < kRows; ++r)
#pragma unroll
            for (int e = 0; e < kCodes / 4; e += 2) {
                const uint2 x = gload(reinterpret_cast<const uint2*>(src + r * p.D) + e / 2);
                w[r][e] = x.x, w[r][e + 1] = x.y;
            }
    }
    XT* out = reinterpret_cast<XT*>(which ? p.v : p.k) + (((int64_t)b * p.rows + row0) * p.Hkv + h) * p.D + c * kCodes;
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (row0 + r >= p.rows) return;
        const bool seen = there && row0 + r < length;
        uint32_t o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if constexpr (sizeof(XT) == 4) o[e] = seen ? __float_as_uint(__fmul_rn((float)(int8_t)(w[r][e >> 2] >> 8 * (e & 3)), s)) : 0u;
            else o[e] = seen ? pack2<XT>(__fmul_rn((float)(int8_t)(w[r][e >> 1] >> 16 * (e & 1)), s), __fmul_rn((float)(int8_t)(w[r][e >> 1] >> (16 * (e & 1) + 8)), s)) : 0u;
        }
        store32(out + (int64_t)r * p.Hkv * p.D, o);
    }
}
template <typename XT> int launch_dequant(DequantParams& p, cudaStream_t st) {
    const int64_t threads = (p.rows + 7) / 8 * p.Hkv * (p.D / (32 / (int)sizeof(XT)));
    if (threads > INT32_MAX - 256) return -1;
    p.seq_blocks = (int)((threads + 255) / 256);
    const int64_t grid = (int64_t)2 * p.B * p.seq_blocks;
    if (grid > INT32_MAX) return -1;
    auto kern = kv8_dequant_kernel<XT>;
    return launch_pdl(kern, dim3((unsigned)grid), 256, 0, st, p);
}

bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
int bad_cache(int Hkv, int D, int T, int64_t pages, int max_pages) {
    if (Hkv <= 0 || D <= 0 || D % 16 != 0 || D > 256 || pages < 0 || max_pages < 0 || (int64_t)max_pages * 128 > INT32_MAX - 256) return -1;
    return T == 16 || T == 32 || T == 64 || T == 128 ? 0 : -206;
}

}  // namespace

GPU_API int gpu_kv8_append(int dtype, const void* k, const void* v, const int64_t* strides, int8_t* k8, int8_t* v8, float* k_scale, float* v_scale,
                           const int32_t* table, int64_t table_stride, const int32_t* start, const int32_t* count, int B, int L, int Hkv, int D, int T,
                           int64_t pages, int max_pages, void* stream) {
    if (int e = bad_cache(Hkv, D, T, pages, max_pages)) return e;
    if (B < 0 || L < 0) return -1;
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (B == 0 || L == 0 || pages == 0 || max_pages == 0) return 0;
    if (!k || !v || !strides || !k8 || !v8 || !k_scale || !v_scale || !table || !start || off16(k) || off16(v) || off16(k8) || off16(v8)) return -5;
    for (int i = 0; i < 6; ++i)
        if (strides[i] % (dtype == DT_F32 ? 4 : 8) != 0) return -5;
    AppendParams p = {k, v, {strides[0], strides[1], strides[2]}, {strides[3], strides[4], strides[5]}, k8, v8, k_scale, v_scale, table, start, count,
                      table_stride, pages, B, L, Hkv, D, T, max_pages, (L - 1) / T + 2};
    if (p.touched > INT32_MAX / 2 / Hkv / B) return -1;
    const int64_t grid = (int64_t)2 * Hkv * p.touched * B;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == DT_F32) return launch_pdl(kv8_append_kernel<float>, dim3((unsigned)grid), 256, 0, st, p);
    if (dtype == DT_F16) return launch_pdl(kv8_append_kernel<half>, dim3((unsigned)grid), 256, 0, st, p);
    return launch_pdl(kv8_append_kernel<bf16>, dim3((unsigned)grid), 256, 0, st, p);
}

GPU_API int gpu_kv8_dequant(int dtype, const int8_t* k8, const int8_t* v8, const float* k_scale, const float* v_scale, const int32_t* table,
                            int64_t table_stride, const int32_t* lengths, void* k, void* v, int B, int64_t rows, int Hkv, int D, int T, int64_t pages,
                            int max_pages, void* stream) {
    if (int e = bad_cache(Hkv, D, T, pages, max_pages)) return e;
    if (B < 0 || rows < 0) return -1;
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (B == 0 || rows == 0) return 0;
    if (!k || !v || !lengths || ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 31) || off16(k8) || off16(v8)) return -5;
    if (max_pages > 0 && pages > 0 && (!k8 || !v8 || !k_scale || !v_scale || !table)) return -5;
    DequantParams p = {k8, v8, k_scale, v_scale, table, lengths, k, v, table_stride, pages, rows, B, Hkv, D, T, pages > 0 ? max_pages : 0, 0, 0};
    while (1 << p.page_log < T) ++p.page_log;
    if (rows > INT32_MAX / Hkv) return -1;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F32 ? launch_dequant<float>(p, st) : dtype == DT_F16 ? launch_dequant<half>(p, st) : launch_dequant<bf16>(p, st);
}
