// Few rows through a dense layer or a gated block: the form that answers single symbols (16 bit up to 16 rows, float up to 32).
//
// The weights are read once and nothing else counts, so the kernel is a stream over them.  A workgroup owns 16 weight rows (gated
// block: 8 gate and 8 up rows of the same features); its waves (8, or 16) take turns along the contraction, 128 elements each, and
// multiply on v_mfma_f32_16x16x32 with the input rows as the other operand (rows beyond the last repeat it): the matrix
// instruction sums over lanes, which costs a vector kernel six shuffles per output and wave.  The fragments come straight from
// memory (16 bytes a lane, any alignment); float operands are split into three bf16 pieces in registers (six products).  The
// waves' sums are joined through LDS in a fixed order.
//
// Bound by the weights' bytes and the time until the first of them arrive: bf16 one row of 4096 x 4096 8.6 ... 9.5 us (3.9 TB/s at best; two turns
// a wave), f16 five rows of 2048 -> 2 x 5632 12.1 ... 13.1 us (3.5 TB/s; one turn a wave, so nothing is asked for ahead), float one row of
// 8192 x 8192 57 us (4.7 TB/s; a large copy: 5.2).  Measured and not kept: lanes
// in pairs of 128 bytes (no change), turns of 256 elements (spills), multiply-adds instead of the matrix unit for one row (5.4 us at
// 4096 x 4096, but a call takes the host 9 either way).
#include "v2vae_dense_gemm.h"

namespace v2vae {

typedef __attribute__((ext_vector_type(4))) float acc4;
__device__ __forceinline__ acc4 mma16(bf16x8 a, bf16x8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ acc4 mma16(f16x8 a, f16x8 b, acc4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// eight consecutive elements of a row, from whole words; TAIL: some may lie beyond K, zeros there
template <typename T> struct Eight { T e[8]; };
// ODD: 16-bit rows that may start in the middle of a word.  Loads at 2-byte addresses are slow (one row of 8191 x 8192: 70 us), so the
// words that hold the elements are read and shifted into place; the word at either end holds one neighbour that is not used.
template <typename T, bool TAIL, bool ODD> __device__ __forceinline__ Eight<T> load_eight(const T* p, int k, int K) {
    struct __attribute__((packed, aligned(4))) Loose { T e[8]; };
    struct __attribute__((packed, aligned(4))) Words { unsigned w[4]; };
    Eight<T> v;
    if constexpr (!TAIL && ODD) {
        const uintptr_t at = (uintptr_t)(p + k);
        const unsigned* const q = reinterpret_cast<const unsigned*>(at & ~(uintptr_t)3);
        const unsigned shift = (at & 2) * 8;
        const Words t = *reinterpret_cast<const Words*>(q);
        const unsigned last = q[at & 2 ? 4 : 3];
        union { unsigned w[4]; Eight<T> v; } u;
        u.w[0] = __builtin_amdgcn_alignbit(t.w[1], t.w[0], shift);
        u.w[1] = __builtin_amdgcn_alignbit(t.w[2], t.w[1], shift);
        u.w[2] = __builtin_amdgcn_alignbit(t.w[3], t.w[2], shift);
        u.w[3] = __builtin_amdgcn_alignbit(last, t.w[3], shift);
        v = u.v;
    } else if constexpr (!TAIL) {
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

template <typename T, int W, int MT, bool ODD, bool GATED> __global__ __launch_bounds__(64 * W) void k_dense_rows(GemmArgs g) {
    constexpr int NP = Elem<T>::NP, FT = GATED ? 8 : 16;  // features of the workgroup
    typedef typename Elem<T>::frag frag;
    __shared__ float s_sum[W][16 * MT][17];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, kl = (lane >> 4) * 8, n0 = blockIdx.x * FT;
    const int n = n0 + r % FT, nc = n < g.N ? n : g.N - 1, which = GATED ? r >> 3 : 0;
    const T* const w = (const T*)g.b[which] + (int64_t)nc * g.ldb[which];
    const T* x[MT];  // 16 input rows each
    acc4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int m = 16 * t + r;
        x[t] = (const T*)g.a[0] + (int64_t)(m < g.M ? m : g.M - 1) * g.lda;
        acc[t] = acc4{0.f, 0.f, 0.f, 0.f};
    }
    constexpr int CH = 4, CE = CH * 32;  // loads and elements of a wave's turn
    struct Turn { Eight<T> v[CH]; };
    auto load = [&](const T* from, int k0, auto tail) {
        Turn t;
#pragma unroll
        for (int i = 0; i < CH; ++i) t.v[i] = load_eight<T, decltype(tail)::value, ODD>(from, k0 + i * 32 + kl, g.K);
        return t;
    };
    auto multiply = [&](const Turn& wt, const Turn& first, int k0, auto tail) {
        frag wf[CH][NP];
#pragma unroll
        for (int i = 0; i < CH; ++i) pieces_of<T>(wt.v[i], wf[i]);
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const Turn xt = t == 0 ? first : load(x[t], k0, tail);
#pragma unroll
            for (int i = 0; i < CH; ++i) {
                frag xf[NP];
                pieces_of<T>(xt.v[i], xf);
#pragma unroll
                for (int sum = NP - 1; sum >= 0; --sum)
#pragma unroll
                    for (int p = 0; p <= sum; ++p) acc[t] = mma16(wf[i][p], xf[sum - p], acc[t]);
            }
        }
    };
    constexpr std::false_type inside{};
    constexpr std::true_type tail{};
    const int whole = g.K / CE * CE, lo = blockIdx.y * g.steps_per_split * CE;
    const bool last = blockIdx.y + 1 == gridDim.y;
    const int hi = last || lo + g.steps_per_split * CE > whole ? whole : lo + g.steps_per_split * CE;
    // The weights of the next turn are asked for before this one's are multiplied.  The last turn asks for its own again (out of the
    // caches): without a branch the compiler knows what is in flight and waits for no more than it needs.
    int k = lo + wave * CE;
    if (k < hi) {
        auto after = [&](int at) { return at + W * CE < hi ? at + W * CE : at; };
        Turn w0 = load(w, k, inside), w1;
        for (;;) {
            const Turn x0 = load(x[0], k, inside);
            w1 = load(w, after(k), inside);
            multiply(w0, x0, k, inside);
            k += W * CE;
            if (k >= hi) break;
            const Turn x1 = load(x[0], k, inside);
            w0 = load(w, after(k), inside);
            multiply(w1, x1, k, inside);
            k += W * CE;
            if (k >= hi) break;
        }
    }
    if (last && whole < g.K && ((whole - lo) / CE) % W == wave) multiply(load(w, whole, tail), load(x[0], whole, tail), whole, tail);
    // lane: input row lane % 16, weight rows 4 (lane / 16) ... + 3
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) s_sum[wave][16 * t + r][4 * (lane >> 4) + e] = acc[t][e];
    __syncthreads();
    float* const part = g.partial ? g.partial + (int64_t)blockIdx.y * g.M * g.N * (GATED ? 2 : 1) : nullptr;
    for (int i = tid; i < 16 * MT * FT; i += 64 * W) {
        const int m = i / FT, f = i % FT;
        if (m >= g.M || n0 + f >= g.N) continue;
        auto total = [&](int at) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < W; ++q) s += s_sum[q][m][at];
            return s;
        };
        float s0 = total(f);
        if constexpr (GATED) {
            float s1 = total(f + 8);
            if (part) {
                part[(int64_t)m * 2 * g.N + n0 + f] = s0;
                part[((int64_t)m * 2 + 1) * g.N + n0 + f] = s1;
                continue;
            }
            finish_gated<T, 1>(g, m, n0 + f, &s0, &s1, true);
        } else {
            if (part) {
                part[(int64_t)m * g.N + n0 + f] = s0;
                continue;
            }
            finish_value<T, 1>(g, m, n0 + f, &s0, 0, true);
        }
    }
}

template <typename T, int W, int MT, bool ODD> static void launch_waves(const GemmArgs& g, bool gated, hipStream_t st) {
    if (gated) hipLaunchKernelGGL((k_dense_rows<T, W, MT, ODD, true>), dim3((g.N + 7) / 8, g.splits), dim3(64 * W), 0, st, g);
    else hipLaunchKernelGGL((k_dense_rows<T, W, MT, ODD, false>), dim3((g.N + 15) / 16, g.splits), dim3(64 * W), 0, st, g);
}
template <typename T> static void launch_rows(const GemmArgs& g, bool gated, hipStream_t st) {
    // sixteen waves on a long contraction; float, which needs twice the registers a turn, eight
    if constexpr (sizeof(T) == 4) {
        if (g.M > 16) launch_waves<T, 8, 2, false>(g, gated, st); else launch_waves<T, 8, 1, false>(g, gated, st);
    } else {
        auto words = [&](const void* p, int64_t ld) { return (uintptr_t)p % 4 == 0 && ld % 2 == 0; };
        if (words(g.a[0], g.lda) && words(g.b[0], g.ldb[0]) && (!gated || words(g.b[1], g.ldb[1]))) {
            if (g.K > 1024) launch_waves<T, 16, 1, false>(g, gated, st); else launch_waves<T, 8, 1, false>(g, gated, st);
        } else {
            if (g.K > 1024) launch_waves<T, 16, 1, true>(g, gated, st); else launch_waves<T, 8, 1, true>(g, gated, st);
        }
    }
}

int dense_rows(const GemmArgs& args, int dtype, bool gated, hipStream_t st) {
    GemmArgs g = args;
    g.steps_per_split = (g.K / 128 + g.splits - 1) / g.splits;
    if (dtype == V2VAE_F32) launch_rows<float>(g, gated, st);
    else if (dtype == V2VAE_BF16) launch_rows<bf16_t>(g, gated, st);
    else launch_rows<f16_t>(g, gated, st);
    if (g.partial) {
        if (gated) launch_join<float, true>(g, st); else launch_join<float, false>(g, st);
    }
    return dense_launch_error("dense layer, few rows");
}

}  // namespace v2vae
