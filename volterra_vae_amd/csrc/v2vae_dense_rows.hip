// One to sixteen rows through a dense layer or a gated block: the form that answers single symbols.
//
// The weights are read once and nothing else counts, so the kernel is a stream over them: a workgroup owns NR weight rows, its
// 256 threads run along the contraction in 16-byte pieces (all NR pieces of a step in flight together), every piece is multiplied
// with the MR input rows (held by the caches) into MR x NR float sums per thread, and the sums are joined over the lanes by
// shuffles and over the four waves through LDS, in a fixed order.
#include "v2vae_dense.h"

namespace v2vae {

template <typename T, int MR, int NR, bool GATED> __global__ __launch_bounds__(256) void k_dense_rows(GemmArgs g) {
    constexpr int E = Vec16<T>::N, FT = GATED ? NR / 2 : NR;  // features of the workgroup
    __shared__ float s_sum[4][MR * NR];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n0 = blockIdx.x * FT;
    const T* w[NR];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
        const int n = n0 + (GATED ? r >> 1 : r), nc = n < g.N ? n : g.N - 1, which = GATED ? r & 1 : 0;
        w[r] = (const T*)g.b[which] + (int64_t)nc * g.ldb[which];
    }
    const T* const x = (const T*)g.a[0];
    float acc[MR][NR];
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int r = 0; r < NR; ++r) acc[m][r] = 0.f;
    if (g.vec_a && g.vec_b) {
        for (int k = tid * E; k < g.K; k += 256 * E) {
            Vec16<T> wv[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) wv[r].raw = *reinterpret_cast<const u32x4*>(w[r] + k);
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                Vec16<T> xv;
                xv.raw = *reinterpret_cast<const u32x4*>(x + (int64_t)(m < g.M ? m : g.M - 1) * g.lda + k);
#pragma unroll
                for (int r = 0; r < NR; ++r)
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[m][r] = fmaf((float)wv[r].e[e], (float)xv.e[e], acc[m][r]);
            }
        }
    } else {
        for (int k = tid; k < g.K; k += 256) {
            float wv[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) wv[r] = (float)w[r][k];
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const float xv = (float)x[(int64_t)(m < g.M ? m : g.M - 1) * g.lda + k];
#pragma unroll
                for (int r = 0; r < NR; ++r) acc[m][r] = fmaf(wv[r], xv, acc[m][r]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float s = acc[m][r];
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) s += __shfl_xor(s, d);
            if (lane == 0) s_sum[wave][m * NR + r] = s;
        }
    __syncthreads();
    for (int i = tid; i < MR * FT; i += 256) {
        const int m = i / FT, f = i % FT, n = n0 + f;
        if (m >= g.M || n >= g.N) continue;
        auto total = [&](int r) { return (s_sum[0][m * NR + r] + s_sum[1][m * NR + r]) + (s_sum[2][m * NR + r] + s_sum[3][m * NR + r]); };
        float s0 = total(GATED ? 2 * f : f);
        if constexpr (GATED) {
            float s1 = total(2 * f + 1);
            finish_gated<T, 1>(g, m, n, &s0, &s1, true);
        } else {
            finish_value<T, 1>(g, m, n, &s0, 0, true);
        }
    }
}

template <typename T, int MR, bool GATED> static void launch_rows(const GemmArgs& g, hipStream_t st) {
    constexpr int NR = 4, FT = GATED ? NR / 2 : NR;
    hipLaunchKernelGGL((k_dense_rows<T, MR, NR, GATED>), dim3((g.N + FT - 1) / FT), dim3(256), 0, st, g);
}
template <typename T, bool GATED> static void pick_rows(const GemmArgs& g, hipStream_t st) {
    if (g.M <= 1) launch_rows<T, 1, GATED>(g, st);
    else if (g.M <= 2) launch_rows<T, 2, GATED>(g, st);
    else if (g.M <= 4) launch_rows<T, 4, GATED>(g, st);
    else if (g.M <= 8) launch_rows<T, 8, GATED>(g, st);
    else launch_rows<T, 16, GATED>(g, st);
}

int dense_rows(const GemmArgs& g, int dtype, bool gated, hipStream_t st) {
    if (dtype == V2VAE_F32) gated ? pick_rows<float, true>(g, st) : pick_rows<float, false>(g, st);
    else if (dtype == V2VAE_BF16) gated ? pick_rows<bf16_t, true>(g, st) : pick_rows<bf16_t, false>(g, st);
    else gated ? pick_rows<f16_t, true>(g, st) : pick_rows<f16_t, false>(g, st);
    return dense_launch_error("dense layer, few rows");
}

}  // namespace v2vae
