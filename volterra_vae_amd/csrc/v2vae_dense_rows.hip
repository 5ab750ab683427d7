// One to sixteen rows through a dense layer or a gated block: the form that answers single symbols.
//
// The weights are read once and nothing else counts, so the kernel is a stream over them.  A workgroup owns 16 weight rows (gated
// block: 8 gate and 8 up rows of the same features); its waves (8, or 16) take turns along the contraction, 128 elements
// each, and multiply on v_mfma_f32_16x16x32 with the input rows as the other operand (rows beyond the last repeat it): the matrix
// instruction sums over lanes, which costs a vector kernel six shuffles per output and wave.  The fragments come straight from
// memory (16 bytes a lane, any alignment); float operands are split into three bf16 pieces in registers (six products).  The
// waves' sums are joined through LDS in a fixed order.
#include "v2vae_dense.h"

namespace v2vae {

typedef __attribute__((ext_vector_type(4))) float acc4;
__device__ __forceinline__ acc4 mma16(bf16x8 a, bf16x8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ acc4 mma16(f16x8 a, f16x8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// eight consecutive elements of a row, at any alignment; TAIL: some may lie beyond K, zeros there
template <typename T> struct Eight { T e[8]; };
template <typename T, bool TAIL> __device__ __forceinline__ Eight<T> load_eight(const T* p, int k, int K) {
    struct __attribute__((packed, aligned(sizeof(T)))) Loose { T e[8]; };
    Eight<T> v;
    if constexpr (!TAIL) {
        const Loose t = *reinterpret_cast<const Loose*>(p + k);
#pragma unroll
        for (int e = 0; e < 8; ++e) v.e[e] = t.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v.e[e] = k + e < K ? p[k + e] : (T)0.f;
    }
    return v;
}
template <typename T> __device__ __forceinline__ void pieces_of(const Eight<T>& v, typename Elem<T>::frag f[Elem<T>::NP]) {
    if constexpr (sizeof(T) == 4) {
        union { unsigned u[4]; bf16x8 f; } w[3];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            unsigned p[3];
            split_pair(v.e[2 * i], v.e[2 * i + 1], p);
#pragma unroll
            for (int q = 0; q < 3; ++q) w[q].u[i] = p[q];
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) f[q] = w[q].f;
    } else {
        f[0] = __builtin_bit_cast(typename Elem<T>::frag, v);
    }
}

template <typename T, int W, bool GATED> __global__ __launch_bounds__(64 * W) void k_dense_rows(GemmArgs g) {
    constexpr int NP = Elem<T>::NP, FT = GATED ? 8 : 16;  // features of the workgroup
    typedef typename Elem<T>::frag frag;
    __shared__ float s_sum[W][16][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, kl = (lane >> 4) * 8, n0 = blockIdx.x * FT;
    const int n = n0 + r % FT, nc = n < g.N ? n : g.N - 1, mc = r < g.M ? r : g.M - 1, which = GATED ? r >> 3 : 0;
    const T* const w = (const T*)g.b[which] + (int64_t)nc * g.ldb[which];
    const T* const x = (const T*)g.a[0] + (int64_t)mc * g.lda;
    acc4 acc = acc4{0.f, 0.f, 0.f, 0.f};
    constexpr int CH = 4, CE = CH * 32;  // loads and elements of a wave's turn
    struct Turn { Eight<T> v[CH]; };
    auto load = [&](const T* from, int k0, auto tail) {
        Turn t;
#pragma unroll
        for (int i = 0; i < CH; ++i) t.v[i] = load_eight<T, decltype(tail)::value>(from, k0 + i * 32 + kl, g.K);
        return t;
    };
    auto multiply = [&](const Turn& wt, const Turn& xt) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
            frag xf[NP], wf[NP];
            pieces_of<T>(xt.v[i], xf);
            pieces_of<T>(wt.v[i], wf);
#pragma unroll
            for (int sum = NP - 1; sum >= 0; --sum)
#pragma unroll
                for (int p = 0; p <= sum; ++p) acc = mma16(wf[p], xf[sum - p], acc);
        }
    };
    const int whole = g.K / CE * CE;
    // The weights of the next turn are asked for before this one's are multiplied.  The last turn asks for its own again (out of the
    // caches): without a branch the compiler knows what is in flight and waits for no more than it needs.
    int k = wave * CE;
    if (k < whole) {
        auto after = [&](int at) { return at + W * CE < whole ? at + W * CE : at; };
        Turn w0 = load(w, k, std::false_type()), w1;
        for (;;) {
            const Turn x0 = load(x, k, std::false_type());
            w1 = load(w, after(k), std::false_type());
            multiply(w0, x0);
            k += W * CE;
            if (k >= whole) break;
            const Turn x1 = load(x, k, std::false_type());
            w0 = load(w, after(k), std::false_type());
            multiply(w1, x1);
            k += W * CE;
            if (k >= whole) break;
        }
    }
    if (whole < g.K && (whole / CE) % W == wave) multiply(load(w, whole, std::true_type()), load(x, whole, std::true_type()));
    // lane: input row lane % 16, weight rows 4 (lane / 16) ... + 3
#pragma unroll
    for (int e = 0; e < 4; ++e) s_sum[wave][r][4 * (lane >> 4) + e] = acc[e];
    __syncthreads();
    if (tid >= 16 * FT) return;
    const int m = tid / FT, f = tid % FT;
    if (m >= g.M || n0 + f >= g.N) return;
    auto total = [&](int at) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < W; ++q) s += s_sum[q][m][at];
        return s;
    };
    float s0 = total(f);
    if constexpr (GATED) {
        float s1 = total(f + 8);
        finish_gated<T, 1>(g, m, n0 + f, &s0, &s1, true);
    } else {
        finish_value<T, 1>(g, m, n0 + f, &s0, 0, true);
    }
}

template <typename T, int W> static void launch_waves(const GemmArgs& g, bool gated, hipStream_t st) {
    if (gated) hipLaunchKernelGGL((k_dense_rows<T, W, true>), dim3((g.N + 7) / 8), dim3(64 * W), 0, st, g);
    else hipLaunchKernelGGL((k_dense_rows<T, W, false>), dim3((g.N + 15) / 16), dim3(64 * W), 0, st, g);
}
template <typename T> static void launch_rows(const GemmArgs& g, bool gated, hipStream_t st) {
    // float needs twice the registers a turn: eight waves; 16 bit from 1025 columns on sixteen
    if (sizeof(T) == 2 && g.K > 1024) launch_waves<T, sizeof(T) == 2 ? 16 : 8>(g, gated, st); else launch_waves<T, 8>(g, gated, st);
}

int dense_rows(const GemmArgs& g, int dtype, bool gated, hipStream_t st) {
    if (dtype == V2VAE_F32) launch_rows<float>(g, gated, st);
    else if (dtype == V2VAE_BF16) launch_rows<bf16_t>(g, gated, st);
    else launch_rows<f16_t>(g, gated, st);
    return dense_launch_error("dense layer, few rows");
}

}  // namespace v2vae
