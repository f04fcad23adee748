// gpu_rotary: queries and keys turned by their positions, one launch for both, the norm of each head before it where the model has one.
//
//   y = x, or x / sqrt(mean(x^2) + eps) w over a head's D values
//   (a, b) -> scale (a cos t - b sin t, a sin t + b cos t) for the pairs of the first rot values, t = pos freq; the others stay as y
//   pairs: (i, i + rot / 2), or neighbours (2 i, 2 i + 1)
//
// Angles: freq and pos freq in 64 bits (position 10^6 times 1 radian leaves an f32 angle 0.06 off), as turns, of which the whole ones are
// dropped; the rest's sine and cosine in f32. A token's angles are worked out once, by as many threads, and serve all of its heads from shared
// memory; the rotation is f32, one rounding to the rows' type. Bound by the rows' bytes.
#include "common.cuh"

namespace {

struct RotaryParams {
    const void* x[2];            // q, k
    void* y[2];
    const float* norm[2];
    int64_t xs[2][3], ys[2][3];  // strides of batch, row, head
    const int32_t* pos;          // [axes, B, L]
    const uint8_t* axis;         // [rot / 2], or null: 0
    const double* freq;          // [rot / 2]
    int64_t pos_axis, pos_batch;
    float scale, eps;
    int B, L, H, heads, D, half, interleaved, axes, tokens;      // heads: of q and k together; tokens: to a CTA
};

// V neighbouring values as they lie in memory
template <typename T, int V> struct Vec {
    static constexpr int kBytes = V * sizeof(T);
    T e[V];
    __device__ __forceinline__ void load(const T* p) {
        if (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(e)[i] = gload(reinterpret_cast<const uint4*>(p) + i);
        } else if (kBytes == 8) *reinterpret_cast<uint2*>(e) = gload(reinterpret_cast<const uint2*>(p));
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = gload(p + i);
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if (kBytes % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kBytes / 16; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
        } else if (kBytes == 8) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
        else {
#pragma unroll
            for (int i = 0; i < V; ++i) p[i] = e[i];
        }
    }
    __device__ __forceinline__ void values(float (&v)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f<T>(e[i]);
    }
    __device__ __forceinline__ void round(const float (&v)[V]) {
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] = from_f<T>(v[i]);
    }
};

constexpr int kThreads = 256, kMaxHalf = 128, kMaxTokens = 4;

// Two vectors of a head, slot `s`: those that are paired with one another, or next to each other
template <int V> __device__ __forceinline__ void places(const RotaryParams& p, int s, int& a, int& b) {
    if (p.interleaved || s >= p.half / V) a = 2 * V * s, b = a + V;
    else a = V * s, b = a + p.half;
}
template <int V> __device__ __forceinline__ void scaled(float (&u)[V], const float* w, float r) {
    Vec<float, V> x;
    x.load(w);
#pragma unroll
    for (int e = 0; e < V; ++e) u[e] = u[e] * r * x.e[e];
}
// A token's cosines and sines: two pairs of a slot next to each other, then the same two of the next slot, so that neighbouring threads read neighbouring
// 16 bytes (in the pairs' order a thread's 64 bytes meet its fourth neighbour's in the same banks)
template <int V> __device__ __forceinline__ int turn_at(int f, int rotated) { return V == 1 ? f : (f % V / 2 * rotated + f / V) * 2 + f % 2; }
template <int V> __device__ __forceinline__ void turned(const RotaryParams& p, float (&u)[V], float (&v)[V], const float2* at, int rotated) {
    float2 cs[V];
    if (V == 1) cs[0] = at[0];
    else {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float4 two = reinterpret_cast<const float4*>(at)[e / 2 * rotated];
            cs[e] = make_float2(two.x, two.y), cs[e + 1] = make_float2(two.z, two.w);
        }
    }
    if (p.interleaved && V > 1) {
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const float2 c = cs[e / 2], d = cs[(V + e) / 2];
            const float u0 = u[e], u1 = u[(e + 1) % V], v0 = v[e], v1 = v[(e + 1) % V];
            u[e] = u0 * c.x - u1 * c.y, u[(e + 1) % V] = u0 * c.y + u1 * c.x;
            v[e] = v0 * d.x - v1 * d.y, v[(e + 1) % V] = v0 * d.y + v1 * d.x;
        }
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float2 c = cs[e];
            const float u0 = u[e], v0 = v[e];
            u[e] = u0 * c.x - v0 * c.y, v[e] = u0 * c.y + v0 * c.x;
        }
    }
}

// A group of `lanes` threads has a head, a thread of it one slot of 2 V values (several with V = 1); the next head's values are on their way. Measured
// (us, floor at the copy's rate): 2 x 4179 tokens, 24 / 24 heads of 128, fp16, 38.7 (31.3; before the table's order above 40.4, before that 50.3 with
// 64-bit divisions for every head and nothing ahead; 47.5 with a token's angles in registers, which leave room for fewer threads); 4096 tokens, 32 / 8 heads
// of 128, bf16, 18.3 (12.8; 19.5), heads normalised 19.7 (26.3); 8192 tokens, 32 / 8 heads of 96, the first 40 values turned, normalised 53 (19.2): four
// values at a time and 12 threads of 16.
template <typename T, int V> __global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams p, const int lanes) {
    extern __shared__ __align__(16) float2 turn[];      // [token][half]: cos, sin
    __shared__ int64_t row[4][kMaxTokens];      // of q, k and the results, where a token's row begins
    const int64_t tokens = (int64_t)p.B * p.L, first = (int64_t)blockIdx.x * p.tokens;
    const int here = (int)min((int64_t)p.tokens, tokens - first);
    pdl_wait();
    if (threadIdx.x >= kThreads - 4 * kMaxTokens) {
        const int i = threadIdx.x - (kThreads - 4 * kMaxTokens), t = i / 4, which = i & 1;
        const int64_t at = first + min(t, here - 1), b = at / p.L, l = at - b * p.L;
        row[i & 3][t] = i & 2 ? b * p.ys[which][0] + l * p.ys[which][1] : b * p.xs[which][0] + l * p.xs[which][1];
    }
    for (int i = threadIdx.x; i < here * p.half; i += kThreads) {
        const int t = i / p.half, f = i - t * p.half;
        const int64_t at = first + t, b = at / p.L;
        const int axis = p.axis ? min((int)gload(p.axis + f), p.axes - 1) : 0;
        const int pos = gload(p.pos + axis * p.pos_axis + b * p.pos_batch + (at - b * p.L));
        // turns: two products of 64 bits; less than half a turn is left, which f32 holds to 2^-25
        const double turns = (double)pos * gload(p.freq + f) * 0.15915494309189533577;
        float s, c;
        sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
        turn[t * p.half + turn_at<V>(f, p.half / V)] = make_float2(c * p.scale, s * p.scale);
    }
    __syncthreads();
    const int lane = threadIdx.x % lanes, slots = p.D / (2 * V), rotated = p.half / V, step = kThreads / lanes;
    const unsigned mask = lanes == 32 ? 0xffffffffu : ((1u << lanes) - 1) << (threadIdx.x & 31 & ~(lanes - 1));
    const float by_d = 1.f / (float)p.D;
    struct Head {
        int t, h;
        __device__ __forceinline__ void wrap(int heads) {
            while (h >= heads) h -= heads, ++t;
        }
    };
    auto x_of = [&](const Head& n) { return reinterpret_cast<const T*>(p.x[n.h >= p.H]) + row[n.h >= p.H][n.t] + (n.h >= p.H ? (n.h - p.H) * p.xs[1][2] : n.h * p.xs[0][2]); };
    auto y_of = [&](const Head& n) { return reinterpret_cast<T*>(p.y[n.h >= p.H]) + row[2 + (n.h >= p.H)][n.t] + (n.h >= p.H ? (n.h - p.H) * p.ys[1][2] : n.h * p.ys[0][2]); };
    auto factor = [&](float sum) {
        for (int o = lanes >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(mask, sum, o);
        return rsqrtf(__fmaf_rn(sum, by_d, p.eps));
    };
    Head n = {0, (int)threadIdx.x / lanes};
    n.wrap(p.heads);
    if constexpr (V > 1) {
        int a, b;
        places<V>(p, lane, a, b);
        const bool mine = lane < slots;
        Vec<T, V> x, y;
        auto request = [&] {
            if (mine && n.t < here) {
                const T* src = x_of(n);
                x.load(src + a), y.load(src + b);
            }
        };
        request();
        while (n.t < here) {
            float u[V] = {}, v[V] = {};
            if (mine) x.values(u), y.values(v);
            T* dst = y_of(n);
            const float* w = p.norm[n.h >= p.H];
            const float2* cs = turn + n.t * p.half + lane * 2;
            n.h += step;
            n.wrap(p.heads);
            request();
            if (n.t >= here) pdl_trigger();
            if (w) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) sum = __fmaf_rn(u[e], u[e], __fmaf_rn(v[e], v[e], sum));
                const float r = factor(sum);
                if (mine) scaled<V>(u, w + a, r), scaled<V>(v, w + b, r);
            }
            if (lane < rotated) turned<V>(p, u, v, cs, rotated);
            if (mine) {
                Vec<T, V> o;
                o.round(u), o.store(dst + a);
                o.round(v), o.store(dst + b);
            }
        }
    } else {
        for (; n.t < here; n.h += step, n.wrap(p.heads)) {
            const T* src = x_of(n);
            T* dst = y_of(n);
            const float* w = p.norm[n.h >= p.H];
            float r = 1.f, u[V], v[V];
            Vec<T, V> x, y;
            auto read = [&](int s, int& a, int& b) {
                places<V>(p, s, a, b);
                x.load(src + a), y.load(src + b);
                x.values(u), y.values(v);
            };
            int a, b;
            if (w) {
                float sum = 0.f;
                for (int s = lane; s < slots; s += lanes) read(s, a, b), sum = __fmaf_rn(u[0], u[0], __fmaf_rn(v[0], v[0], sum));
                r = factor(sum);
            }
            for (int s = lane; s < slots; s += lanes) {
                read(s, a, b);
                if (w) scaled<V>(u, w + a, r), scaled<V>(v, w + b, r);
                if (s < rotated) turned<V>(p, u, v, turn + n.t * p.half + s, rotated);
                x.round(u), x.store(dst + a);
                y.round(v), y.store(dst + b);
            }
        }
    }
}

template <typename T> int launch_rotary(RotaryParams& p, cudaStream_t st) {
    // Values side by side to a thread: what pairs, the rest and whole vectors allow
    const int rest = (p.D - 2 * p.half) / 2;
    const int V = p.half % 8 == 0 && rest % 8 == 0 ? 8 : p.half % 4 == 0 && rest % 4 == 0 ? 4 : 1;
    const int slots = p.D / (2 * V);
    int lanes = 1;
    while (lanes < 32 && lanes < slots) lanes *= 2;
    const int64_t tokens = (int64_t)p.B * p.L;
    if (tokens / kMaxTokens >= INT32_MAX) return -1;
    const int sms = b200q::sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    // Tokens to a CTA: as many as leave four CTAs an SM. us with 1 | 2 | 4, 32 / 8 normalised heads of 128: 592 tokens 4.9 | 4.9 | 5.9, 1184 8.6 | 6.8 | 8.5, 2368
    // 16.5 | 13.1 | 11.5, 8192 52.6 | 40.8 | 35.8; of 96, 40 values turned: 1184 10.5 | 10.3 | 12.8, 2368 19.1 | 17.2 | 18.6, 8192 64 | 56 | 53.
    p.tokens = 1;
    while (p.tokens < kMaxTokens && tokens >= (int64_t)p.tokens * 2 * 4 * sms) p.tokens *= 2;
    const int64_t ctas = (tokens + p.tokens - 1) / p.tokens;
    auto kern = V == 8 ? rotary_kernel<T, 8> : V == 4 ? rotary_kernel<T, 4> : rotary_kernel<T, 1>;
    return launch_pdl(kern, dim3((unsigned)ctas), kThreads, p.tokens * p.half * sizeof(float2), st, p, lanes);
}

bool off(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

}  // namespace

GPU_API int gpu_rotary(int dtype, const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, const int32_t* pos, int64_t pos_axis,
                       int64_t pos_batch, int axes, const uint8_t* axis, const double* freq, int rot, int interleaved, float scale, const float* q_norm,
                       const float* k_norm, float eps, int B, int L, int H, int Hkv, int D, void* stream) {
    if (dtype < DT_F32 || dtype > DT_BF16) return -4;
    if (B < 0 || L < 0 || H < 0 || Hkv < 0 || H > 65536 || Hkv > 65536 || D <= 0 || D % 8 != 0 || D > 2 * kMaxHalf || rot < 0 || rot % 2 != 0 || rot > D || axes < 1) return -1;
    if (B == 0 || L == 0 || H + Hkv == 0) return 0;
    if (!strides || (H > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !k_out)) || (rot > 0 && (!pos || !freq || (axes > 1 && !axis)))) return -5;
    const int e = dtype == DT_F32 ? 4 : 2;
    if (off(q, 16) || off(k, 16) || off(q_out, 16) || off(k_out, 16) || (q_norm && off(q_norm, 16)) || (k_norm && off(k_norm, 16))) return -5;
    RotaryParams p = {};
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < 4; ++j)
            if (strides[3 * j + i] * e % 16 != 0) return -5;
        p.xs[0][i] = strides[i], p.xs[1][i] = strides[3 + i], p.ys[0][i] = strides[6 + i], p.ys[1][i] = strides[9 + i];
    }
    const int sizes[3] = {B, L, 0};
    for (int w = 0; w < 2; ++w)
        for (int i = 0; i < 3; ++i)
            if ((i < 2 ? sizes[i] : w ? Hkv : H) > 1 && (w ? Hkv : H) > 0 && p.ys[w][i] == 0) return -5;
    p.x[0] = q, p.x[1] = k, p.y[0] = q_out, p.y[1] = k_out, p.norm[0] = q_norm, p.norm[1] = k_norm;
    p.pos = pos, p.pos_axis = pos_axis, p.pos_batch = pos_batch, p.axis = axis, p.axes = axes, p.freq = freq, p.scale = scale, p.eps = eps;
    p.B = B, p.L = L, p.H = H, p.heads = H + Hkv, p.D = D, p.half = rot / 2, p.interleaved = interleaved != 0;
    cudaStream_t st = (cudaStream_t)stream;
    return dtype == DT_F32 ? launch_rotary<float>(p, st) : dtype == DT_F16 ? launch_rotary<half>(p, st) : launch_rotary<bf16>(p, st);
}
