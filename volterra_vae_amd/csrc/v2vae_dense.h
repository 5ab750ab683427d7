// Shared pieces of the dense-layer kernels (linear, gated block, distillation): element types, activations, argument blocks.
#ifndef V2VAE_DENSE_H
#define V2VAE_DENSE_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "v2vae_dense_plan.h"

namespace v2vae {

using bf16_t = __bf16;
using f16_t = _Float16;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;

// Elements of one 16-byte piece of T, to and from float.  A 16-bit result is rounded once, to nearest even.
template <typename T> struct Vec16 {
    static constexpr int N = 16 / sizeof(T);
    union { u32x4 raw; T e[N]; };
};

template <typename T> struct Elem;
// bf16 pieces of an element, operand of a matrix instruction
template <> struct Elem<float> { static constexpr int NP = 3; typedef bf16x8 frag; };
template <> struct Elem<bf16_t> { static constexpr int NP = 1; typedef bf16x8 frag; };
template <> struct Elem<f16_t> { static constexpr int NP = 1; typedef f16x8 frag; };

__device__ __forceinline__ f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma32(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// two floats -> their three bf16 pieces, each pair packed in a word
__device__ __forceinline__ void split_pair(float x0, float x1, unsigned p[3]) {
    typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const bf16x2 h = {(__bf16)x0, (__bf16)x1};
        unsigned u = __builtin_bit_cast(unsigned, h);
        asm("" : "+v"(u));  // no instruction: keeps the compiler from converting each float again to get at its half of the pair
        p[i] = u;
        x0 -= __uint_as_float(u << 16);
        x1 -= __uint_as_float(u & 0xFFFF0000u);
    }
}

// exp(x + lo) for |lo| far below |x|, x <= 88: x log2(e) is carried as a float and its remainder, so the result is off by about
// two units however large |x| is; below exp(-87) it is 0.
__device__ __forceinline__ float exp_with_rest(float x, float lo) {
    constexpr float L = 1.44269502f, L_LO = 1.92596299e-8f, LN2 = 0.693147181f;
    const float t = x * L;
    const float r = fmaf(lo, L, fmaf(x, L_LO, fmaf(x, L, -t)));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * LN2, e);
}
// 1 / d to half a unit or so: the hardware's reciprocal and one Newton step (0 where it is subnormal)
__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(r, fmaf(-d, r, 1.f), r);
}
// Phi(z) and exp(-z^2 / 2), |z| <= 80.  With x = |z| / sqrt 2 and t = 1 / (1 + 0.42 x), erfc(x) = exp(-x^2) t P(t); P is a
// least-squares fit of erfc(x) exp(x^2) / t in relative error (2.3e-9 at its worst over all x >= 0).  Both halves of the tail keep
// their relative accuracy: nothing is subtracted for z < 0.
__device__ __forceinline__ float normal_cdf(float z, float* gauss) {
    const float q = z * z, rest = fmaf(z, z, -q);
    const float e = exp_with_rest(-0.5f * q, -0.5f * rest);
    const float t = reciprocal(fmaf(0.42f * 0.70710678118654752f, fabsf(z), 1.f));
    float p = -0.04113757392246231f;
    p = fmaf(p, t, 0.23070600708015587f);
    p = fmaf(p, t, -0.4866447164102488f);
    p = fmaf(p, t, 0.43715272615373146f);
    p = fmaf(p, t, -0.19733165247973258f);
    p = fmaf(p, t, 0.21373484799346232f);
    p = fmaf(p, t, 0.15004025649345917f);
    p = fmaf(p, t, 0.21989457161457882f);
    p = fmaf(p, t, 0.23661220944910594f);
    p = fmaf(p, t, 0.2369733217454039f);
    const float half = 0.5f * (e * (t * p));
    *gauss = e;
    return z < 0.f ? half : 1.f - half;
}

// tanh z: below 0.55 an odd polynomial (least-squares fit of tanh(z) / z - 1 in z^2, 1e-9 at its worst), else from e = exp(-2 |z|), and
// so its slope 4 e / (1 + e)^2 there, which keeps its relative accuracy down to e = 2^-126 (beyond |z| = 43.6 it is 0), where
// 1 - tanh(z)^2 has none left from |z| = 9 on
template <bool SLOPE> __device__ __forceinline__ float tanh_of(float z, float* slope) {
    const float u = z * z, y = fabsf(z);
    float p = -0.006282466723832369f;
    p = fmaf(p, u, 0.02107775339065489f);
    p = fmaf(p, u, -0.053853856641005726f);
    p = fmaf(p, u, 0.13332601672040642f);
    p = fmaf(p, u, -0.33333318045245297f);
    const float e = exp_with_rest(-2.f * fminf(y, 60.f), 0.f), r = reciprocal(1.f + e);
    const float small = fmaf(z * u, p, z), large = copysignf((1.f - e) * r, z);
    if constexpr (SLOPE) *slope = y < 0.55f ? fmaf(-small, small, 1.f) : (z != z ? z : 4.f * e * r * r);
    return y < 0.55f ? small : (z != z ? z : large);
}

// act(z) and act'(z); the kinds are V2VAE_ACT_*.  For |z| beyond 80 the soft activations are their asymptotes to the last bit of
// a float; the clamp keeps z (1 - s) and z exp(-z^2 / 2) from becoming inf * 0 there.  A NaN stays one.
template <bool SLOPE> __device__ __forceinline__ float act_both(int kind, float z, float* slope) {
    switch (kind) {
        case V2VAE_ACT_RELU:
            if constexpr (SLOPE) *slope = z > 0.f ? 1.f : (z != z ? z : 0.f);
            return z > 0.f ? z : (z != z ? z : 0.f);
        case V2VAE_ACT_SILU: {
            const float zc = fminf(fmaxf(z, -80.f), 80.f), e = exp_with_rest(-zc, 0.f), s = reciprocal(1.f + e);
            if constexpr (SLOPE) *slope = z != z ? z : s * fmaf(zc, e * s, 1.f);
            return z != z ? z : (z < -80.f ? 0.f : z * s);
        }
        case V2VAE_ACT_GELU: {
            const float zc = fminf(fmaxf(z, -80.f), 80.f);
            float gauss;
            const float phi = normal_cdf(zc, &gauss);
            if constexpr (SLOPE) *slope = z != z ? z : fmaf(zc, 0.39894228040143268f * gauss, phi);
            return z != z ? z : (z < -80.f ? 0.f : z * phi);
        }
        case V2VAE_ACT_TANH:
            return tanh_of<SLOPE>(z, slope);
        default:
            if constexpr (SLOPE) *slope = 1.f;
            return z;
    }
}
__device__ __forceinline__ float act_value(int kind, float z) { return act_both<false>(kind, z, nullptr); }
__device__ __forceinline__ float act_slope(int kind, float z, float* value) {
    float slope;
    *value = act_both<true>(kind, z, &slope);
    return slope;
}

// One product D[m][n] = sum over segments and k of A(m, k) B(n, k), with what happens to D afterwards.
struct GemmArgs {
    const void* a[2];       // operand A of segment s (contraction cut in two segments), or of batch entry b
    const void* b[2];       // operand B likewise; gated forward: gate and up weights
    void* c[2];             // output of batch entry b
    float* partial;         // split contraction: [batch][split][M][N] sums
    int64_t lda, ldb[2], ldc;  // elements between rows (k contiguous) or between k (rows contiguous)
    int M, N, K;            // rows of A, rows of B (output columns; gated forward: features), contraction length of a segment
    int segs, batch, splits, steps_per_split;
    int pad_a, pad_b;       // rows of A, B are padded with zeros to a multiple of 16 bytes
    const void* bias[2];
    const void* residual;
    int64_t ldr;
    float* z[2];            // pre-activations kept for the backward pass, [M][N]; may be NULL
    int act;
    // float32: the weights as three planes [plane_rows][plane_ld] of bf16 pieces (NULL: split on the way into LDS)
    const void* planes;
    int64_t plane_bytes;
    int plane_rows, plane_ld;
};

// What happens to the finished sums of row m, columns n ... n + C - 1 (batch entry 1 has an output of its own, nothing else).
// `whole`: all C columns exist; they are moved together at any address (11816 x 464 -> 2 x 572 bf16, whose rows start at odd
// multiples of 8 bytes: 44 us with element by element moves there, 32 this way).
template <typename T, int C> struct __attribute__((packed, aligned(sizeof(T)))) Columns { T e[C]; };
template <typename T, int C> __device__ __forceinline__ void load_columns(const void* p, int64_t at, int count, bool whole, float v[C]) {
    if (whole) {
        const Columns<T, C> t = *reinterpret_cast<const Columns<T, C>*>((const T*)p + at);
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = (float)t.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = e < count ? (float)((const T*)p)[at + e] : 0.f;
    }
}
template <typename T, int C> __device__ __forceinline__ void store_columns(void* p, int64_t at, int count, bool whole, const float v[C]) {
    if (whole) {
        Columns<T, C> t;
#pragma unroll
        for (int e = 0; e < C; ++e) t.e[e] = (T)v[e];
        *reinterpret_cast<Columns<T, C>*>((T*)p + at) = t;
    } else {
#pragma unroll
        for (int e = 0; e < C; ++e)
            if (e < count) ((T*)p)[at + e] = (T)v[e];
    }
}
template <int C> __device__ __forceinline__ void act_columns(int kind, float v[C]) {
    if (kind == V2VAE_ACT_NONE) return;
    // one switch for all columns
    auto all = [&](auto k) {
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = act_value(decltype(k)::value, v[e]);
    };
    switch (kind) {
        case V2VAE_ACT_RELU: all(std::integral_constant<int, V2VAE_ACT_RELU>()); break;
        case V2VAE_ACT_SILU: all(std::integral_constant<int, V2VAE_ACT_SILU>()); break;
        case V2VAE_ACT_GELU: all(std::integral_constant<int, V2VAE_ACT_GELU>()); break;
        case V2VAE_ACT_TANH: all(std::integral_constant<int, V2VAE_ACT_TANH>()); break;
    }
}
template <typename T, int C> __device__ __forceinline__ void finish_value(const GemmArgs& g, int64_t m, int n, float s[C], int bat, bool whole,
                                                                                       const T* res = nullptr) {
    const int count = g.N - n;
    float v[C];
    if (g.bias[0]) {
        load_columns<T, C>(g.bias[0], n, count, whole, v);
#pragma unroll
        for (int e = 0; e < C; ++e) s[e] += v[e];
    }
    if (g.z[0]) store_columns<float, C>(g.z[0], m * g.N + n, count, whole, s);
    act_columns<C>(g.act, s);
    if (g.residual) {
        if (whole && res) {  // already here
#pragma unroll
            for (int e = 0; e < C; ++e) v[e] = (float)res[e];
        } else {
            load_columns<T, C>(g.residual, m * g.ldr + n, count, whole, v);
        }
#pragma unroll
        for (int e = 0; e < C; ++e) s[e] += v[e];
    }
    store_columns<T, C>(g.c[bat], m * g.ldc + n, count, whole, s);
}
template <typename T, int C>
__device__ __forceinline__ void finish_gated(const GemmArgs& g, int64_t m, int n, float gate[C], float up[C], bool whole) {
    const int count = g.N - n;
    float v[C];
    if (g.bias[0]) {
        load_columns<T, C>(g.bias[0], n, count, whole, v);
#pragma unroll
        for (int e = 0; e < C; ++e) gate[e] += v[e];
    }
    if (g.bias[1]) {
        load_columns<T, C>(g.bias[1], n, count, whole, v);
#pragma unroll
        for (int e = 0; e < C; ++e) up[e] += v[e];
    }
    if (g.z[0]) {
        store_columns<float, C>(g.z[0], m * g.N + n, count, whole, gate);
        store_columns<float, C>(g.z[1], m * g.N + n, count, whole, up);
    }
    act_columns<C>(g.act, gate);
#pragma unroll
    for (int e = 0; e < C; ++e) gate[e] *= up[e];
    store_columns<T, C>(g.c[0], m * g.ldc + n, count, whole, gate);
}
// launchers; 0 or a V2VAE_E* code
enum { LAYOUT_KK = 0, LAYOUT_KM = 1, LAYOUT_MM = 2 };  // A / B with the contraction (K) or the row index (M) contiguous
int gemm_direct_bf16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_direct_f16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int split_planes(const GemmArgs&, bool transposed, bool gated, int N, int K, hipStream_t);  // b[], ldb[]: N x K weights
int gemm_split(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);  // float32
int gemm_staged_bf16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_staged_f16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);

int dense_rows(const GemmArgs& g, int dtype, bool gated, hipStream_t st);

int dense_launch_error(const char* where);  // V2VAE_OK, or V2VAE_ELAUNCH with the text kept for v2vae_last_error

}  // namespace v2vae
#endif
