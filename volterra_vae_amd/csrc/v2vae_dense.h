// Shared pieces of the dense-layer kernels (linear, gated block, distillation): element types, activations, argument blocks.
#ifndef V2VAE_DENSE_H
#define V2VAE_DENSE_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/v2vae_hip.h"

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

// act(z); the kinds are V2VAE_ACT_*.  exp, erfc and tanh are the device library's float functions
// (erfc rather than 1 + erf: no cancellation where z is far below zero).
__device__ __forceinline__ float act_value(int kind, float z) {
    switch (kind) {
        case V2VAE_ACT_RELU: return z > 0.f ? z : (z != z ? z : 0.f);
        case V2VAE_ACT_SILU: return z / (1.f + expf(-z));
        case V2VAE_ACT_GELU: return 0.5f * z * erfcf(z * -0.70710678118654752f);
        case V2VAE_ACT_TANH: return tanhf(z);
        default: return z;
    }
}
// act(z) and act'(z).  For |z| beyond 80 both soft activations are their asymptotes to the last bit of a float; the clamp keeps
// z (1 - s) and z exp(-z^2 / 2) from becoming inf * 0 there.
__device__ __forceinline__ float act_slope(int kind, float z, float* value) {
    const float zc = fminf(fmaxf(z, -80.f), 80.f);
    switch (kind) {
        case V2VAE_ACT_RELU: *value = z > 0.f ? z : (z != z ? z : 0.f); return z > 0.f ? 1.f : (z != z ? z : 0.f);
        case V2VAE_ACT_SILU: {
            const float s = 1.f / (1.f + expf(-zc));
            *value = z != z ? z : (z < -80.f ? 0.f : z * s);
            return z != z ? z : s * (1.f + zc * (1.f - s));
        }
        case V2VAE_ACT_GELU: {
            const float phi = 0.5f * erfcf(zc * -0.70710678118654752f);
            *value = z != z ? z : (z < -80.f ? 0.f : z * phi);
            return z != z ? z : phi + zc * (0.39894228040143268f * expf(-0.5f * zc * zc));
        }
        case V2VAE_ACT_TANH: { const float t = tanhf(z); *value = t; return 1.f - t * t; }
        default: *value = z; return 1.f;
    }
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
    int vec_a, vec_b;       // 16-byte loads allowed
    int vec_c;              // eight columns at a time in the epilogue: N, strides and pointers allow it
    const void* bias[2];
    const void* residual;
    int64_t ldr;
    float* z[2];            // pre-activations kept for the backward pass, [M][N]; may be NULL
    int act;
};

// What happens to the finished sums of row m, columns n ... n + C - 1 (batch entry 1 has an output of its own, nothing else).
// `whole`: all C columns exist and every pointer is aligned for them.
template <typename T, int C> __device__ __forceinline__ void load_columns(const void* p, int64_t at, int count, bool whole, float v[C]) {
    struct alignas(C * sizeof(T) > 16 ? 16 : C * sizeof(T)) TC { T e[C]; };
    if (whole) {
        const TC t = *reinterpret_cast<const TC*>((const T*)p + at);
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = (float)t.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] = e < count ? (float)((const T*)p)[at + e] : 0.f;
    }
}
template <typename T, int C> __device__ __forceinline__ void store_columns(void* p, int64_t at, int count, bool whole, const float v[C]) {
    struct alignas(C * sizeof(T) > 16 ? 16 : C * sizeof(T)) TC { T e[C]; };
    if (whole) {
        TC t;
#pragma unroll
        for (int e = 0; e < C; ++e) t.e[e] = (T)v[e];
        *reinterpret_cast<TC*>((T*)p + at) = t;
    } else {
#pragma unroll
        for (int e = 0; e < C; ++e)
            if (e < count) ((T*)p)[at + e] = (T)v[e];
    }
}
template <int C> __device__ __forceinline__ void act_columns(int kind, float v[C]) {
    if (kind == V2VAE_ACT_NONE) return;
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = act_value(kind, v[e]);
}
template <typename T, int C> __device__ __forceinline__ void finish_value(const GemmArgs& g, int64_t m, int n, float s[C], int bat, bool whole) {
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
        load_columns<T, C>(g.residual, m * g.ldr + n, count, whole, v);
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
// launchers, one object file per element type; 0 or a V2VAE_E* code
enum { LAYOUT_KK = 0, LAYOUT_KM = 1, LAYOUT_MM = 2 };  // A / B with the contraction (K) or the row index (M) contiguous
enum { TILE_128 = 0, TILE_64 = 1, TILE_256 = 2 };
int gemm_direct_bf16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_direct_f16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_staged_f32(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_staged_bf16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);
int gemm_staged_f16(const GemmArgs&, int layout, bool gated, int tile, hipStream_t);

// one to sixteen rows (v2vae_dense_rows.hip)
constexpr int ROWS_MAX = 16;
int dense_rows(const GemmArgs& g, int dtype, bool gated, hipStream_t st);

int dense_launch_error(const char* where);  // V2VAE_OK, or V2VAE_ELAUNCH with the text kept for v2vae_last_error

}  // namespace v2vae
#endif
