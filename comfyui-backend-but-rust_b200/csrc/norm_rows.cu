// Rows between the linears of a text encoder's layer, and blocks of e4m3:
//
//   gpu_norm_rows    s = T(x + resid) back to the residual stream, y = s / sqrt(mean(s^2) + eps) w (RMS), or y = x, or y = silu(x) up;
//                    y as rows of floating point, or as e4m3 with one scale for each 128 columns of a row
//   gpu_f8_requant   a weight as e4m3 with one scale for each block of 128 x 128
//   gpu_f8_dequant   either of them back
//
// s = max(amax, 1e-30) (1 / 448), code = e4m3(y (1 / s)), both products f32: a multiplication with the reciprocal, so that a code is within
// half a step and 2^-23 of y / s; the largest value of a block is 448 then, the type's largest number. Sums and y are f32.
#include <type_traits>

#include "common.cuh"
#include "f8.cuh"
#include "mma.cuh"

namespace {

using namespace b200q;

enum { PRO_PLAIN = 0, PRO_RMS = 1, PRO_SWIGLU = 3 };

struct NormParams {
    const void *x, *resid;
    void *resid_out, *out;
    const float* norm_w;
    float* scales;
    int64_t x_stride, up_offset, resid_stride, resid_out_stride, out_stride;
    float eps;
    int M, K, out_dt, warps;      // warps to a row
};

template <typename T> __device__ __forceinline__ void store8(void* base, int64_t at, const float (&v)[8]) {
    T* p = reinterpret_cast<T*>(base) + at;
    if (sizeof(T) == 4) {
        reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        uint4 w;
        T* e = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = from_f<T>(v[i]);
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// A thread has V pieces of eight columns, `warps` * 32 pieces apart; sixteen lanes have a group of 128 columns.
template <typename T, int PRO, int V> __global__ void __launch_bounds__(1024) norm_rows_kernel(const NormParams p) {
    __shared__ float part[32];
    const int threads = p.warps * 32, in_row = threadIdx.x % threads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = blockIdx.x * (blockDim.x / threads) + threadIdx.x / threads, pieces = p.K / 8;
    const bool there = row < p.M;
    pdl_wait();
    float y[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int piece = in_row + i * threads;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[i][e] = 0.f;
        if (there && piece < pieces) load8<T>(reinterpret_cast<const T*>(p.x) + row * p.x_stride + piece * 8, y[i]);
    }
    if (PRO == PRO_SWIGLU) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int piece = in_row + i * threads;
            float up[8] = {};
            if (there && piece < pieces) load8<T>(reinterpret_cast<const T*>(p.x) + row * p.x_stride + p.up_offset + piece * 8, up);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = silu_f(y[i][e]) * up[e];
        }
    }
    if (PRO == PRO_RMS) {
        if (p.resid) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int piece = in_row + i * threads;
                float s[8];
                if (there && piece < pieces) {
                    load8<T>(reinterpret_cast<const T*>(p.resid) + row * p.resid_stride + piece * 8, s);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[i][e] = rnd<T>(y[i][e] + s[e]);
                    store8<T>(p.resid_out, row * p.resid_out_stride + piece * 8, y[i]);
                }
            }
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = __fmaf_rn(y[i][e], y[i][e], sum);
        sum = warp_sum(sum);
        if (p.warps > 1) {
            if (lane == 0) part[warp] = sum;
            __syncthreads();
            const int first = warp / p.warps * p.warps;
            sum = 0.f;
            for (int w = 0; w < p.warps; ++w) sum += part[first + w];
        }
        const float r = rsqrtf(sum / (float)p.K + p.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int piece = in_row + i * threads;
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = 1.f;
            if (p.norm_w && piece < pieces) load8<float>(p.norm_w + piece * 8, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * r * w[e];
        }
    }
    pdl_trigger();
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int piece = in_row + i * threads;
        const bool mine = there && piece < pieces;
        const int64_t at = row * p.out_stride + piece * 8;
        if (p.out_dt == DT_E4M3) {
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[i][e]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float s = f8_scale(top), inv = __frcp_rn(s);
            if (mine) {
                *reinterpret_cast<uint2*>(reinterpret_cast<uint8_t*>(p.out) + at) =
                    make_uint2(e4m3x4(y[i][0] * inv, y[i][1] * inv, y[i][2] * inv, y[i][3] * inv), e4m3x4(y[i][4] * inv, y[i][5] * inv, y[i][6] * inv, y[i][7] * inv));
                if ((piece & 15) == 0) p.scales[(int64_t)row * ((p.K + 127) / 128) + piece / 16] = s;
            }
        } else if (mine) {
            if (p.out_dt == DT_F32) store8<float>(p.out, at, y[i]);
            else if (p.out_dt == DT_F16) store8<half>(p.out, at, y[i]);
            else store8<bf16>(p.out, at, y[i]);
        }
    }
}

template <typename T, int PRO, int V> int launch_norm(NormParams& p, cudaStream_t st) {
    const int pieces = p.K / 8;
    p.warps = (pieces + 32 * V - 1) / (32 * V);
    const int rows = p.warps >= 8 ? 1 : 8 / p.warps;      // to a CTA
    return launch_pdl(norm_rows_kernel<T, PRO, V>, dim3((p.M + rows - 1) / rows), rows * p.warps * 32, 0, st, p);
}
template <typename T, int PRO> int launch_norm(NormParams& p, cudaStream_t st) {
    return p.K <= 4096 ? launch_norm<T, PRO, 1>(p, st) : p.K <= 16384 ? launch_norm<T, PRO, 2>(p, st) : launch_norm<T, PRO, 4>(p, st);
}
template <typename T> int launch_norm(int prologue, NormParams& p, cudaStream_t st) {
    return prologue == PRO_PLAIN ? launch_norm<T, PRO_PLAIN>(p, st) : prologue == PRO_RMS ? launch_norm<T, PRO_RMS>(p, st) : launch_norm<T, PRO_SWIGLU>(p, st);
}

// ---- weights ------------------------------------------------------------------------------------------------------------------------
// A CTA a block of 128 x 128: 256 threads, 16 to a row, eight rows each.
template <typename T> __global__ void __launch_bounds__(256) f8_requant_kernel(const void* w, int64_t w_stride, uint8_t* codes, float* scales, int64_t N, int K, int groups) {
    __shared__ float part[8];
    const int64_t block = blockIdx.x, bn = block / groups;
    const int g = (int)(block - bn * groups), col = g * 128 + (threadIdx.x & 15) * 8;
    pdl_wait();
    float v[8][8];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = bn * 128 + i * 16 + threadIdx.x / 16;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
        if (row < N && col < K) load8<T>(reinterpret_cast<const T*>(w) + row * w_stride + col, v[i]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[i][e]));
    }
    top = warp_max(top);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, part[i]);
    const float s = f8_scale(top), inv = __frcp_rn(s);
    if (threadIdx.x == 0) scales[block] = s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t row = bn * 128 + i * 16 + threadIdx.x / 16;
        if (row < N && col < K)
            *reinterpret_cast<uint2*>(codes + row * K + col) =
                make_uint2(e4m3x4(v[i][0] * inv, v[i][1] * inv, v[i][2] * inv, v[i][3] * inv), e4m3x4(v[i][4] * inv, v[i][5] * inv, v[i][6] * inv, v[i][7] * inv));
    }
}
// Eight codes a thread; a block of 256 threads takes 2048 codes of the matrix as it lies
template <typename T> __global__ void __launch_bounds__(256) f8_dequant_kernel(const uint8_t* codes, const float* scales, int block_rows, void* out, int64_t total, int K, int groups) {
    pdl_wait();
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
    if (at >= total) return;
    const int64_t row = at / K;
    const float s = gload(scales + row / block_rows * groups + (at - row * K) / 128);
    const uint2 c = gload(reinterpret_cast<const uint2*>(codes + at));
    float v[8];
    e4m3x4_values(c.x, v), e4m3x4_values(c.y, v + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] *= s;
    store8<T>(out, at, v);
}

bool off(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace

GPU_API int gpu_norm_rows(int dtype, int prologue, const void* x, int64_t x_stride, int64_t up_offset, const void* resid, int64_t resid_stride, void* resid_out,
                          int64_t resid_out_stride, const float* norm_w, float eps, int out_dt, void* out, int64_t out_stride, float* scales, int M, int K,
                          void* stream) {
    if (dtype < DT_F32 || dtype > DT_BF16 || out_dt < DT_F32 || out_dt > DT_E4M3) return -4;
    const bool f8 = out_dt == DT_E4M3;
    if (M < 0 || K <= 0 || K % (f8 ? 16 : 8) != 0) return -1;
    if (K > 32768) return -2;
    if ((prologue != PRO_PLAIN && prologue != PRO_RMS && prologue != PRO_SWIGLU) || (prologue != PRO_RMS && (resid || norm_w))) return -3;
    if (M == 0) return 0;
    const int e = dtype == DT_F32 ? 4 : 2, oe = f8 ? 1 : out_dt == DT_F32 ? 4 : 2;
    auto rows_off = [&](const void* ptr, int64_t stride, int size) { return !ptr || off(ptr, 16) || (M > 1 && (stride * size % 16 != 0 || stride < K)); };
    if (rows_off(x, x_stride, e) || rows_off(out, out_stride, oe) || (f8 && !scales) || (norm_w && off(norm_w, 16))) return -5;
    if (resid && (rows_off(resid, resid_stride, e) || rows_off(resid_out, resid_out_stride, e))) return -5;
    if (prologue == PRO_SWIGLU && up_offset * e % 16 != 0) return -5;
    NormParams p = {};
    p.x = x, p.x_stride = x_stride, p.up_offset = up_offset, p.resid = resid, p.resid_stride = resid_stride, p.resid_out = resid_out;
    p.resid_out_stride = resid_out_stride, p.norm_w = norm_w, p.eps = eps, p.out_dt = out_dt, p.out = out, p.out_stride = out_stride, p.scales = scales;
    p.M = M, p.K = K;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F32 ? launch_norm<float>(prologue, p, st) : dtype == DT_F16 ? launch_norm<half>(prologue, p, st) : launch_norm<bf16>(prologue, p, st);
}

GPU_API int gpu_f8_requant(int dtype, const void* w, int64_t w_stride, void* codes, float* scales, int64_t N, int K, void* stream) {
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N < 0 || K <= 0 || K % 16 != 0) return -1;
    const int64_t groups = ((int64_t)K + 127) / 128, blocks = (N / 128 + (N % 128 != 0)) * groups;
    if (N > (int64_t)1 << 40 || blocks > INT32_MAX) return -1;
    if (N == 0) return 0;
    if (!w || !codes || !scales || off(w, 16) || off(codes, 16) || (N > 1 && (w_stride * (dtype == DT_F32 ? 4 : 2) % 16 != 0 || w_stride < K))) return -5;
    auto kern = dtype == DT_F32 ? f8_requant_kernel<float> : dtype == DT_F16 ? f8_requant_kernel<half> : f8_requant_kernel<bf16>;
    return launch_pdl(kern, dim3((unsigned)blocks), 256, 0, (cudaStream_t)stream, w, w_stride, (uint8_t*)codes, scales, N, K, (int)groups);
}

GPU_API int gpu_f8_dequant(int dtype, const void* codes, const float* scales, int block_rows, void* out, int64_t N, int K, void* stream) {
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N < 0 || K <= 0 || K % 16 != 0 || (block_rows != 1 && block_rows != 128)) return -1;
    if (N > (int64_t)1 << 40 || N * K / 2048 > INT32_MAX - 1) return -1;
    if (N == 0) return 0;
    if (!codes || !scales || !out || off(codes, 16) || off(out, 16)) return -5;
    const int64_t total = N * K;
    auto kern = dtype == DT_F32 ? f8_dequant_kernel<float> : dtype == DT_F16 ? f8_dequant_kernel<half> : f8_dequant_kernel<bf16>;
    return launch_pdl(kern, dim3((unsigned)((total + 2047) / 2048)), 256, 0, (cudaStream_t)stream, (const uint8_t*)codes, scales, block_rows, out, total, K,
                      (K + 127) / 128);
}
