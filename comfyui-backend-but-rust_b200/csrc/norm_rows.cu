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

// Eight values as they lie in memory
template <typename T> struct Raw {
    static constexpr int kWords = sizeof(T) / 2;      // of 16 bytes
    uint4 w[kWords];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = to_f<T>(e[i]);
    }
    // Whether one of them may be below `bound`, a negative number that T has. 16-bit values as whole numbers: what is more negative is larger
    __device__ __forceinline__ bool below(float bound) const {
        if constexpr (std::is_same<T, float>::value) {
            float v[8];
            values(v);
            return fminf(fminf(fminf(v[0], v[1]), fminf(v[2], v[3])), fminf(fminf(v[4], v[5]), fminf(v[6], v[7]))) < bound;
        } else {
            const T b = from_f<T>(bound);
            const uint32_t most = __vmaxu2(__vmaxu2(w[0].x, w[0].y), __vmaxu2(w[0].z, w[0].w)), end = *reinterpret_cast<const uint16_t*>(&b);
            return (most >> 16) > end || (most & 0xffffu) > end;
        }
    }
    // The sum in T. Of 16-bit values directly: their f32 sum is exact, or the smaller one below half a step of the larger, which is the result either way
    __device__ __forceinline__ void add(const Raw& o) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            uint32_t *x = &w[i].x, y[4] = {o.w[i].x, o.w[i].y, o.w[i].z, o.w[i].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (std::is_same<T, float>::value) x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(y[e]));
                else if (std::is_same<T, half>::value) asm("add.rn.f16x2 %0, %0, %1;" : "+r"(x[e]) : "r"(y[e]));
                else asm("add.rn.bf16x2 %0, %0, %1;" : "+r"(x[e]) : "r"(y[e]));
            }
        }
    }
    __device__ __forceinline__ void store(void* base, int64_t at) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<uint4*>(reinterpret_cast<T*>(base) + at)[i] = w[i];
    }
};

// Eight columns of a row on their way out: to `at`, of out's type; sixteen lanes have a group of 128 columns and all call this. `scale`: where the first
// of them writes the group's, null for the others.
__device__ __forceinline__ void emit(int out_dt, const float (&y)[8], uint8_t* at, float* scale, bool mine) {
    if (out_dt == DT_E4M3) {
        float top = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(y[e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float s = f8_scale(top), inv = __frcp_rn(s);
        if (mine) {
            *reinterpret_cast<uint2*>(at) =
                make_uint2(e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv), e4m3x4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv));
            if (scale) *scale = s;
        }
    } else if (mine) {
        if (out_dt == DT_F32) store8<float>(at, 0, y);
        else if (out_dt == DT_F16) store8<half>(at, 0, y);
        else store8<bf16>(at, 0, y);
    }
}
__device__ __forceinline__ int out_size(int out_dt) { return out_dt == DT_E4M3 ? 1 : out_dt == DT_F32 ? 4 : 2; }

// x / (1 + e^-x): e^-x as 2^h, h = -x log2 e, the power and the reciprocal from the special function unit, 2^-22.5 and 2^-23. Infinities and NaN as the
// formula has them.
//   16-bit rows to 16-bit rows or codes: h as it is rounded, with log2 e in f32, is 2^-23.7 of itself off, 2^-17.2 of the power where x is -87, far below half
//   a step of either. Below -87.3 the reciprocal is no normal number and the value 0.
//   f32 rows, or to f32 rows: what is left of the exponent is -x - h ln 2 (ln 2 in f32: 2^-22 of the power where x is -80) and is multiplied on: 2^-20 in all.
//   Below kSiluFar the value is x e^x, by two halves that are normal numbers; seldom, so that eight values together are asked for one. 4096 x 9728 bf16 to e4m3:
//   38.7 us the first way, 43.1 this way; 512 x 9728 f32, which wait for HBM, 8.7 and 9.0.
constexpr float kSiluFar = -80.f;
template <bool FINE> __device__ __forceinline__ float silu_near(float x) {
    float e, r;
    const float t = FINE ? fmaxf(-x, kSiluFar) : -x, h = __fmul_rn(t, 1.4426950408889634f);      // (beyond 80 the power is nothing beside 1; infinity has no rest)
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(h));
    if (FINE) e = __fmaf_rn(e, __fmaf_rn(h, -0.6931471805599453f, t), e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return x * r;
}
template <typename T, bool FINE> __device__ __forceinline__ void silu8(const Raw<T>& a, float (&y)[8]) {
    a.values(y);
    const bool far = FINE && a.below(kSiluFar);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = silu_near<FINE>(y[e]);
    if (far) {
        float x[8];
        a.values(x);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float half = expf(0.5f * x[e]);
            if (x[e] < kSiluFar) y[e] = x[e] * half * half;
        }
    }
}

// Rows without a norm: sixteen lanes take a group of 128 columns, of every `step`-th row, whose values are on their way a row ahead; a CTA has
// `wide` neighbouring groups of as many rows as fit. 4096 x 9728 bf16, SWIGLU: 107 us with expf and a division, 57 with rows and groups counted by one
// number (41 instructions a value, the issue slots' limit).
template <typename T, int PRO, bool FINE> __global__ void __launch_bounds__(256) group_rows_kernel(const NormParams p, const int wide, const int step) {
    const int slot = threadIdx.x / 16, group = blockIdx.x * wide + slot % wide, piece = group * 16 + (threadIdx.x & 15), rows = blockDim.x / (16 * wide);
    const bool in_row = piece < p.K / 8;
    int row = slot < rows * wide ? blockIdx.y * rows + slot / wide : p.M;      // (whole warps: half of one may have nothing to do)
    const T* x = reinterpret_cast<const T*>(p.x) + (int64_t)row * p.x_stride + piece * 8;
    const int64_t next = (int64_t)step * p.x_stride, out_next = (int64_t)step * p.out_stride * out_size(p.out_dt);
    const int groups = (p.K + 127) / 128;
    uint8_t* out = reinterpret_cast<uint8_t*>(p.out) + ((int64_t)row * p.out_stride + piece * 8) * out_size(p.out_dt);
    float* scale = (threadIdx.x & 15) == 0 && p.scales ? p.scales + (int64_t)row * groups + group : nullptr;
    pdl_wait();
    Raw<T> a, b;
    a.clear(), b.clear();
    auto take = [](Raw<T>& r, const T* from) {
#pragma unroll
        for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = gload(reinterpret_cast<const uint4*>(from) + i);
    };
    auto request = [&] {
        if (in_row && row < p.M) {
            take(a, x);
            if (PRO == PRO_SWIGLU) take(b, x + p.up_offset);
        }
    };
    request();
    while (__any_sync(0xffffffffu, row < p.M)) {
        const bool mine = in_row && row < p.M;
        float y[8];
        if (PRO == PRO_SWIGLU) {
            float up[8];
            silu8<T, FINE>(a, y);
            b.values(up);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] *= up[e];
        } else a.values(y);
        row += step, x += next;
        request();
        if (!__any_sync(0xffffffffu, row < p.M)) pdl_trigger();
        emit(p.out_dt, y, out, scale, mine);
        out += out_next;
        if (scale) scale += (int64_t)step * groups;
    }
}

template <typename T, int V> constexpr bool ahead() { return sizeof(T) == 2 && V <= 2; }
// RMS: a thread has V pieces of eight columns, `warps` * 32 pieces apart. A CTA takes rows in turn: weights stay in registers (read anew for every
// row they are as many bytes as 16-bit rows and their stream), the next row's values are on their way while this one's sum goes round. With more than
// two pieces a thread has no room for either, nor with f32 rows: those CTAs have one turn, or several with more than kMostStep rows.
template <typename T, int V> __global__ void __launch_bounds__(V <= 2 ? 512 : 1024, V > 2 ? 1 : ahead<T, V>() ? 2 : 3) rms_rows_kernel(const NormParams p) {
    constexpr bool kAhead = ahead<T, V>();
    __shared__ __align__(16) float part[2][32];
    const int threads = p.warps * 32, in_row = threadIdx.x % threads, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rows = blockDim.x / threads, pieces = p.K / 8, step = gridDim.x * rows, groups = (p.K + 127) / 128;
    if (threadIdx.x < 64) part[threadIdx.x >> 5][threadIdx.x & 31] = 0.f;
    if (p.warps > 1) __syncthreads();
    const float by_k = 1.f / (float)p.K;
    pdl_wait();
    float w[kAhead ? V : 1][8];
    auto weights = [&](float (&v)[8], int piece) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = 1.f;
        if (p.norm_w && piece < pieces) load8<float>(p.norm_w + piece * 8, v);
    };
    if (kAhead)
#pragma unroll
        for (int i = 0; i < V; ++i) weights(w[i], in_row + i * threads);
    Raw<T> a[V], b[V];
    auto take = [](Raw<T>& r, const T* from) {
#pragma unroll
        for (int i = 0; i < Raw<T>::kWords; ++i) r.w[i] = gload(reinterpret_cast<const uint4*>(from) + i);
    };
    auto request = [&](int row) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int piece = in_row + i * threads;
            if (row < p.M && piece < pieces) {
                take(a[i], reinterpret_cast<const T*>(p.x) + row * p.x_stride + piece * 8);
                if (p.resid) take(b[i], reinterpret_cast<const T*>(p.resid) + row * p.resid_stride + piece * 8);
            } else a[i].clear(), b[i].clear();
        }
    };
    int row = blockIdx.x * rows + threadIdx.x / threads, turn = 0;
    if (kAhead) request(row);
    for (int first = blockIdx.x * rows; first < p.M; first += step, row += step, turn ^= 1) {
        const bool there = row < p.M;
        if (!kAhead) request(row);
        float y[V][8], sum = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int piece = in_row + i * threads;
            if (p.resid) {
                a[i].add(b[i]);
                if (there && piece < pieces) a[i].store(p.resid_out, row * p.resid_out_stride + piece * 8);
            }
            a[i].values(y[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum = __fmaf_rn(y[i][e], y[i][e], sum);
        }
        if (kAhead) request(row + step);      // (rows of this CTA alone: what another one writes is not read here)
        sum = warp_sum(sum);
        if (p.warps > 1) {
            if (lane == 0) part[turn][warp] = sum;
            __syncthreads();
            // (a row of its own CTA has all parts, zeros behind the last; several rows to a CTA have at most four warps each)
            sum = 0.f;
            if (rows == 1) {
                const float4* all = reinterpret_cast<const float4*>(part[turn]);
                for (int i = 0; i * 4 < p.warps; ++i) {
                    const float4 v = all[i];
                    sum += (v.x + v.y) + (v.z + v.w);
                }
            } else {
                const int w0 = warp / p.warps * p.warps;
                for (int i = 0; i < p.warps; ++i) sum += part[turn][w0 + i];
            }
        }
        if (first + step >= p.M) pdl_trigger();
        const float r = rsqrtf(__fmaf_rn(sum, by_k, p.eps));
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int piece = in_row + i * threads;
            float v[8];
            if (!kAhead) weights(v, piece);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[i][e] = y[i][e] * r * (kAhead ? w[kAhead ? i : 0][e] : v[e]);
            emit(p.out_dt, y[i], reinterpret_cast<uint8_t*>(p.out) + (row * p.out_stride + piece * 8) * out_size(p.out_dt),
                 (piece & 15) == 0 ? p.scales + (int64_t)row * groups + piece / 16 : nullptr, there && piece < pieces);
        }
    }
}

constexpr int kThreadsAhead = 1024;      // to an SM
constexpr int kMostStep = 1 << 19;       // rows from a CTA's turn to its next: the last row's number and this one fit 32 bits (gpu_norm_rows leaves twice as much)
template <typename T, int PRO, bool FINE = false> int launch_groups(NormParams& p, cudaStream_t st) {
    const int groups = (p.K + 127) / 128, columns = (groups + 15) / 16, wide = (groups + columns - 1) / columns;
    const int rows = 16 / wide, sms = sm_count();      // rows to a CTA
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    const int threads = (rows * wide * 16 + 31) / 32 * 32;
    const int64_t all = ((int64_t)p.M + rows - 1) / rows, some = (int64_t)sms * (2048 / threads) / columns, most = some < 1 ? 1 : some;
    const int down = (int)(all < most ? all : most);
    return launch_pdl(group_rows_kernel<T, PRO, FINE>, dim3(columns, down), threads, 0, st, p, wide, down * rows);
}
template <typename T, int V> int launch_rms(NormParams& p, cudaStream_t st) {
    const int pieces = p.K / 8, sms = sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    p.warps = (pieces + 32 * V - 1) / (32 * V);
    const int rows = p.warps >= 8 ? 1 : 8 / p.warps, ctas = (p.M + rows - 1) / rows;      // rows to a CTA
    const int most = ahead<T, V>() ? sms * (kThreadsAhead / (rows * p.warps * 32)) : kMostStep / rows;
    return launch_pdl(rms_rows_kernel<T, V>, dim3(ctas < most ? ctas : most), rows * p.warps * 32, 0, st, p);
}
template <typename T> int launch_norm(int prologue, NormParams& p, cudaStream_t st) {
    if (prologue == PRO_PLAIN) return launch_groups<T, PRO_PLAIN>(p, st);
    if (prologue == PRO_SWIGLU) return sizeof(T) == 4 || p.out_dt == DT_F32 ? launch_groups<T, PRO_SWIGLU, true>(p, st) : launch_groups<T, PRO_SWIGLU, sizeof(T) == 4>(p, st);
    // Pieces to a thread, 1 | 2 | 4 (more would not fit its CTA's threads beyond 4096 and 8192 columns), us, onto the stream. 4096 rows, bf16 to e4m3: 1280
    // columns 7.7 | 8.9 | 9.7, 1536 9.0 | 9.3 | 10.9, 2048 11.7 | 11.4 | 13.0, 4096 22.5 | 21.2 | 24.5, 8192 - | 40.0 | 43.5; f32 rows, nothing ahead: 2560 27.2 | 29.8 |
    // 35.0, 4096 42.9 | 46.6 | 55.1, 8192 - | 90 | 103. 64 rows, 2560 columns, bf16: 1.8 | 2.4 | 3.6.
    if (p.K <= (sizeof(T) == 4 ? 4096 : 1536)) return launch_rms<T, 1>(p, st);
    return p.K <= 8192 ? launch_rms<T, 2>(p, st) : launch_rms<T, 4>(p, st);
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
    if (M < 0 || M > INT32_MAX - (1 << 20) || K <= 0 || K % (f8 ? 16 : 8) != 0) return -1;
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
    if (N < 0 || N > (int64_t)1 << 38 || K <= 0 || K % 16 != 0) return -1;
    const int64_t groups = ((int64_t)K + 127) / 128, blocks = (N / 128 + (N % 128 != 0)) * groups;
    if (blocks > INT32_MAX) return -1;
    if (N == 0) return 0;
    if (!w || !codes || !scales || off(w, 16) || off(codes, 16) || (N > 1 && (w_stride * (dtype == DT_F32 ? 4 : 2) % 16 != 0 || w_stride < K))) return -5;
    auto kern = dtype == DT_F32 ? f8_requant_kernel<float> : dtype == DT_F16 ? f8_requant_kernel<half> : f8_requant_kernel<bf16>;
    return launch_pdl(kern, dim3((unsigned)blocks), 256, 0, (cudaStream_t)stream, w, w_stride, (uint8_t*)codes, scales, N, K, (int)groups);
}

GPU_API int gpu_f8_dequant(int dtype, const void* codes, const float* scales, int block_rows, void* out, int64_t N, int K, void* stream) {
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (N < 0 || K <= 0 || K % 16 != 0 || (block_rows != 1 && block_rows != 128)) return -1;
    if (N > (int64_t)(INT32_MAX - 1) * 2048 / K) return -1;
    if (N == 0) return 0;
    if (!codes || !scales || !out || off(codes, 16) || off(out, 16)) return -5;
    const int64_t total = N * K;
    auto kern = dtype == DT_F32 ? f8_dequant_kernel<float> : dtype == DT_F16 ? f8_dequant_kernel<half> : f8_dequant_kernel<bf16>;
    return launch_pdl(kern, dim3((unsigned)((total + 2047) / 2048)), 256, 0, (cudaStream_t)stream, (const uint8_t*)codes, scales, block_rows, out, total, K,
                      (K + 127) / 128);
}
