// The staged matrix product of the dense layers for 16-bit operands, and what all their products share: the order of tiles, the
// epilogue, the join of a split contraction.  D[m][n] = sum_k A(m, k) B(n, k), any strides, any alignment, any size.
//
// A workgroup of four waves owns a (64 TM) x (64 TN) tile of D, each wave 32 TM x 32 TN of it in accumulators of
// v_mfma_f32_32x32x16.  A contraction step of 64 elements of every row goes global -> registers -> LDS: the next step's loads are
// in flight while the current one is multiplied, and the step through registers is what makes the rest general:
//  * an operand whose rows, not whose contraction, are contiguous (both operands of a weight gradient) is read with lanes along
//    the rows and transposed by the store into LDS;
//  * rows and contraction ends that do not fill a tile are loaded element by element, and rows may start at any element.
// LDS rows are 128 bytes plus 16: the row stride is an odd multiple of 16 bytes, so the 16-byte reads of 16 consecutive rows touch
// every bank once.
//
// Bound by the loads, which are many and small for rows that are not 16-byte aligned: 65537 x 131 -> 257 bf16 forward 55 us (80 TF);
// from PACK_FORWARD and PACK_BACKWARD on such operands are copied for the direct kernel instead (both sides there).
#ifndef V2VAE_DENSE_GEMM_H
#define V2VAE_DENSE_GEMM_H
#include "v2vae_dense.h"

namespace v2vae {

// One operand's tile of one contraction step: ROWS rows x BK, held by 256 threads between the global load and the LDS store.
template <typename T, int ROWS, bool KC> struct Stage;

// contraction contiguous: eight lanes along a row (16 bytes each), 32 rows a pass
template <typename T, int ROWS> struct Stage<T, ROWS, true> {
    static constexpr int E = 8, PASS = ROWS / 32, BK = 64, ROWB = BK * 2 + 16;
    Vec16<T> v[PASS];
    // row_of(r): pointer of tile row r at k = 0, or NULL beyond the matrix
    template <typename F> __device__ __forceinline__ void load(int tid, int k0, int K, F row_of) {
        const int k = k0 + (tid & 7) * E;
#pragma unroll
        for (int j = 0; j < PASS; ++j) {
            const T* p = row_of((tid >> 3) + 32 * j);
            v[j].raw = u32x4{0, 0, 0, 0};
            if (p == nullptr) continue;
            struct __attribute__((packed, aligned(sizeof(T)))) Loose { u32x4 raw; };
            if (k + E <= K) {
                v[j].raw = reinterpret_cast<const Loose*>(p + k)->raw;
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (k + e < K) v[j].e[e] = p[k + e];
            }
        }
    }
    __device__ __forceinline__ void store(int tid, char* lds) const {
#pragma unroll
        for (int j = 0; j < PASS; ++j) *reinterpret_cast<u32x4*>(lds + ((tid >> 3) + 32 * j) * ROWB + (tid & 7) * 16) = v[j].raw;
    }
};

// rows contiguous: lanes along the rows (element loads, coalesced at any alignment), every thread KT consecutive k of its row
template <typename T, int ROWS> struct Stage<T, ROWS, false> {
    static constexpr int BK = 64, ROWB = BK * 2 + 16, KT = BK * ROWS / 256;
    T v[KT];
    template <typename F> __device__ __forceinline__ void load(int tid, int k0, int K, int64_t ld, F row_of) {
        const int k = k0 + (tid / ROWS) * KT;
        const T* p = row_of(tid % ROWS);
        if (p != nullptr) p += (int64_t)k * ld;
#pragma unroll
        for (int e = 0; e < KT; ++e) v[e] = (p != nullptr && k + e < K) ? p[e * ld] : (T)0.f;
    }
    __device__ __forceinline__ void store(int tid, char* lds) const {
        char* d = lds + (tid % ROWS) * ROWB + (tid / ROWS) * KT * 2;
#pragma unroll
        for (int e = 0; e < KT; e += 8) {
            Vec16<T> w;
#pragma unroll
            for (int i = 0; i < 8; ++i) w.e[i] = v[e + i];
            *reinterpret_cast<u32x4*>(d + e * 2) = w.raw;
        }
    }
};

// Block number -> tile: consecutive blocks go to the eight XCDs in turn, so every XCD gets a contiguous run of tiles (its own
// L2), walked in groups of eight tile rows.
__device__ __forceinline__ void tile_of(int id, int tiles_m, int tiles_n, int* tm, int* tn) {
    const int total = tiles_m * tiles_n, q = total / 8, r = total % 8, x = id & 7, i = id >> 3;
    const int t = x * q + (x < r ? x : r) + i;
    const int group = 8 * tiles_n, g = t / group, first = g * 8, rows = tiles_m - first < 8 ? tiles_m - first : 8;
    const int in = t - g * group;
    *tm = first + in % rows;
    *tn = in / rows;
}

// The sums of one 32-row block of a wave, 32 TN columns, from matrix registers to memory.  The operands enter the matrix
// instruction swapped, so a lane holds row lane % 32 and columns 32 j + 8 q + 4 (lane / 32) ... + 3.  They go through the wave's
// own piece of LDS to become rows again: eight consecutive columns a lane, whole cache lines per row for every load and store of
// the epilogue, and its code (bias, activation, residual) exists once per block instead of once per register.
template <int TN> constexpr int EPI_ROWB = 32 * TN * 4 + 16;
template <int TN> constexpr int EPI_BYTES = 32 * EPI_ROWB<TN>;
template <typename T, int TN, bool GATED>
__device__ __forceinline__ void finish_block(const GemmArgs& g, const f32x16 (&acc)[TN], char* lds, int lane, int m0, int n0, float* part, int bat) {
    constexpr int ROWB = EPI_ROWB<TN>, COLS = GATED ? 32 : 32 * TN, PER = COLS / 8, ROWS = 64 / PER;
    const int c = (lane % PER) * 8, n = n0 + c;
    const bool whole = n + 8 <= g.N;
    // the residual's rows are asked for before anything else
    typedef Columns<T, 8> T8;
    const bool fetched = !GATED && !part && g.residual && whole;
    auto residual_at = [&](int r) {
        const int64_t m = m0 + r < g.M ? m0 + r : g.M - 1;
        return *reinterpret_cast<const T8*>((const T*)g.residual + m * g.ldr + n);
    };
    T8 next[32 / ROWS];
    if (fetched) {
#pragma unroll
        for (int q = 0; q < 32 / ROWS; ++q) next[q] = residual_at(lane / PER + q * ROWS);
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            *reinterpret_cast<f32x4*>(lds + (lane & 31) * ROWB + (32 * j + 8 * q + 4 * (lane >> 5)) * 4) =
                f32x4{acc[j][4 * q], acc[j][4 * q + 1], acc[j][4 * q + 2], acc[j][4 * q + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int r = lane / PER; r < 32; r += ROWS) {
        const int64_t m = m0 + r;
        const T8 res = next[0];
#pragma unroll
        for (int q = 1; q < 32 / ROWS; ++q) next[q - 1] = next[q];
        if (m >= g.M || n >= g.N) continue;
        float s[8], u[8];
        const f32x4* p = reinterpret_cast<const f32x4*>(lds + r * ROWB + c * 4);
        *reinterpret_cast<f32x4*>(s) = p[0];
        *reinterpret_cast<f32x4*>(s + 4) = p[1];
        if constexpr (GATED) {
            const f32x4* p2 = reinterpret_cast<const f32x4*>(lds + r * ROWB + (c + 32) * 4);
            *reinterpret_cast<f32x4*>(u) = p2[0];
            *reinterpret_cast<f32x4*>(u + 4) = p2[1];
        }
        if (part) {
            if constexpr (GATED) {
                store_columns<float, 8>(part, m * 2 * g.N + n, g.N - n, whole, s);
                store_columns<float, 8>(part, m * 2 * g.N + g.N + n, g.N - n, whole, u);
            } else {
                store_columns<float, 8>(part, m * g.N + n, g.N - n, whole, s);
            }
        } else if constexpr (GATED) {
            finish_gated<T, 8>(g, m, n, s, u, whole);
        } else {
            finish_value<T, 8>(g, m, n, s, bat, whole, res.e);
        }
    }
}

template <typename T, int TM, int TN, bool AKC, bool BKC, bool GATED>
__global__ __launch_bounds__(256, 2) void k_gemm_staged(GemmArgs g) {
    constexpr int BK = 64, ROWB = BK * 2 + 16, BM = 64 * TM, BN = 64 * TN;
    static_assert(!GATED || TN == 2, "a gated wave holds one gate and one up block");
    typedef typename Elem<T>::frag frag;
    constexpr int TILES = (BM + BN) * ROWB, EPI = 4 * EPI_BYTES<TN>;
    __shared__ __align__(16) char lds[TILES > EPI ? TILES : EPI];
    char* const lds_a = lds;
    char* const lds_b = lds + BM * ROWB;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
    const int out_bn = GATED ? BN / 2 : BN;
    const int tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.N + out_bn - 1) / out_bn;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const int split = blockIdx.y, bat = blockIdx.z;
    const int m0 = tm * BM, n0 = tn * out_bn;
    const int steps_seg = (g.K + BK - 1) / BK, steps = steps_seg * g.segs;
    const int s_lo = split * g.steps_per_split, s_hi = s_lo + g.steps_per_split < steps ? s_lo + g.steps_per_split : steps;

    Stage<T, BM, AKC> sa;
    Stage<T, BN, BKC> sb;
    auto fetch = [&](int s) {
        const int seg = s >= steps_seg ? 1 : 0, k0 = (s - seg * steps_seg) * BK, sel = seg | bat;
        const T* a = (const T*)g.a[sel];
        const T* b = (const T*)g.b[sel];
        auto row_a = [&](int r) -> const T* {
            const int m = m0 + r;
            return m < g.M ? a + (AKC ? (int64_t)m * g.lda : (int64_t)m) : nullptr;
        };
        auto row_b = [&](int r) -> const T* {
            if constexpr (GATED) {  // blocks of 32 rows: gate and up of the same features in turn, so that a wave holds both
                const int n = n0 + (r >> 6) * 32 + (r & 31);
                const T* w = (const T*)((r & 32) ? g.b[1] : g.b[0]);
                return n < g.N ? w + (int64_t)n * g.ldb[(r >> 5) & 1] : nullptr;
            } else {
                const int n = n0 + r;
                return n < g.N ? b + (BKC ? (int64_t)n * g.ldb[sel] : (int64_t)n) : nullptr;
            }
        };
        if constexpr (AKC) sa.load(tid, k0, g.K, row_a); else sa.load(tid, k0, g.K, g.lda, row_a);
        if constexpr (BKC) sb.load(tid, k0, g.K, row_b); else sb.load(tid, k0, g.K, g.ldb[sel], row_b);
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    if (s_lo < s_hi) {
        fetch(s_lo);
        sa.store(tid, lds_a);
        sb.store(tid, lds_b);
    }
    __syncthreads();
    const char* const fa = lds_a + (wm * 32 * TM + (lane & 31)) * ROWB + (lane >> 5) * 16;
    const char* const fb = lds_b + (wn * 32 * TN + (lane & 31)) * ROWB + (lane >> 5) * 16;
    for (int s = s_lo; s < s_hi; ++s) {
        if (s + 1 < s_hi) fetch(s + 1);
#pragma unroll
        for (int kk = 0; kk < BK / 16; ++kk) {
            frag a[TM], b[TN];
#pragma unroll
            for (int i = 0; i < TM; ++i) a[i] = *reinterpret_cast<const frag*>(fa + i * 32 * ROWB + kk * 32);
#pragma unroll
            for (int j = 0; j < TN; ++j) b[j] = *reinterpret_cast<const frag*>(fb + j * 32 * ROWB + kk * 32);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = mma32(b[j], a[i], acc[i][j]);
        }
        __syncthreads();
        if (s + 1 < s_hi) {
            sa.store(tid, lds_a);
            sb.store(tid, lds_b);
        }
        __syncthreads();
    }

    float* const part = g.partial ? g.partial + ((int64_t)bat * g.splits + split) * ((int64_t)g.M * (GATED ? 2 : 1) * g.N) : nullptr;
#pragma unroll
    for (int i = 0; i < TM; ++i)
        finish_block<T, TN, GATED>(g, acc[i], lds + wave * EPI_BYTES<TN>, lane, m0 + (wm * TM + i) * 32, n0 + wn * (GATED ? 32 : 32 * TN), part, bat);
}

// Sums of a split contraction and the rest of the epilogue; C columns a thread.  Y threads share an output's parts, thread y those
// from y on in steps of Y, and their sums are added in order.  One pass over the parts, 4 ... 10 us, most of it the launch.
template <typename T, int C, int Y, bool GATED> __global__ __launch_bounds__(256) void k_gemm_join(GemmArgs g) {
    constexpr int X = 256 / Y, W = GATED ? 2 : 1;
    __shared__ float s_part[Y > 1 ? Y : 1][Y > 1 ? X : 1][Y > 1 ? W * C : 1];
    const int64_t per = (int64_t)g.M * g.N * W, count = (int64_t)g.M * (g.N / C);
    const int bat = blockIdx.y, x = threadIdx.x % X, y = threadIdx.x / X;
    const float* base = g.partial + bat * (int64_t)g.splits * per;
    for (int64_t i0 = (int64_t)blockIdx.x * X; i0 < count; i0 += (int64_t)gridDim.x * X) {
        const int64_t i = i0 + x < count ? i0 + x : count - 1, m = i / (g.N / C);
        const int n = (int)(i - m * (g.N / C)) * C;
        float s[C], u[C], v[C];
#pragma unroll
        for (int e = 0; e < C; ++e) s[e] = u[e] = 0.f;
#pragma unroll 4
        for (int p = y; p < g.splits; p += Y) {
            load_columns<float, C>(base, p * per + m * W * g.N + n, C, true, v);
#pragma unroll
            for (int e = 0; e < C; ++e) s[e] += v[e];
            if constexpr (GATED) {
                load_columns<float, C>(base, p * per + m * W * g.N + g.N + n, C, true, v);
#pragma unroll
                for (int e = 0; e < C; ++e) u[e] += v[e];
            }
        }
        if constexpr (Y > 1) {
            __syncthreads();
#pragma unroll
            for (int e = 0; e < C; ++e) {
                s_part[y][x][e] = s[e];
                if constexpr (GATED) s_part[y][x][C + e] = u[e];
            }
            __syncthreads();
            if (y > 0) continue;
            for (int q = 1; q < Y; ++q)
#pragma unroll
                for (int e = 0; e < C; ++e) {
                    s[e] += s_part[q][x][e];
                    if constexpr (GATED) u[e] += s_part[q][x][C + e];
                }
        }
        if (i0 + x >= count) continue;
        if constexpr (GATED) finish_gated<T, C>(g, m, n, s, u, true); else finish_value<T, C>(g, m, n, s, bat, true);
    }
}

template <typename T, bool GATED> void launch_join(const GemmArgs& g, hipStream_t st) {
    const int c = g.N % 4 == 0 ? 4 : 1;
    const int64_t count = (int64_t)g.M * (g.N / c);
    // many parts of few outputs (96 x 28 of 431 parts: 40 us with one thread an output, 6 with sixteen; 512 x 256 of 32 parts: 6 and 9)
    const bool shared = g.splits >= 32 && (int64_t)g.M * g.N < 65536;
    int64_t blocks = shared ? (count + 15) / 16 : (count + 255) / 256;
    if (blocks > 4096) blocks = 4096;
    const dim3 grid((unsigned)blocks, g.batch);
    if (shared && c == 4) hipLaunchKernelGGL((k_gemm_join<T, 4, 16, GATED>), grid, dim3(256), 0, st, g);
    else if (shared) hipLaunchKernelGGL((k_gemm_join<T, 1, 16, GATED>), grid, dim3(256), 0, st, g);
    else if (c == 4) hipLaunchKernelGGL((k_gemm_join<T, 4, 1, GATED>), grid, dim3(256), 0, st, g);
    else hipLaunchKernelGGL((k_gemm_join<T, 1, 1, GATED>), grid, dim3(256), 0, st, g);
}

template <typename T, int TM, int TN, bool AKC, bool BKC, bool GATED> void launch_staged(const GemmArgs& g, hipStream_t st) {
    const int bn = GATED ? 32 * TN : 64 * TN;
    const int64_t tiles = (int64_t)((g.M + 64 * TM - 1) / (64 * TM)) * ((g.N + bn - 1) / bn);
    hipLaunchKernelGGL((k_gemm_staged<T, TM, TN, AKC, BKC, GATED>), dim3((unsigned)tiles, g.splits, g.batch), dim3(256), 0, st, g);
    if (g.partial) launch_join<T, GATED>(g, st);
}

// tile: TILE_128, or TILE_64 (gated: 64 rows x 64 features)
template <typename T> int gemm_staged(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    if (gated) {
        if (tile == TILE_128) launch_staged<T, 2, 2, true, true, true>(g, st); else launch_staged<T, 1, 2, true, true, true>(g, st);
    } else if (layout == LAYOUT_KK) {
        if (tile == TILE_128) launch_staged<T, 2, 2, true, true, false>(g, st); else launch_staged<T, 1, 1, true, true, false>(g, st);
    } else if (layout == LAYOUT_KM) {
        if (tile == TILE_128) launch_staged<T, 2, 2, true, false, false>(g, st); else launch_staged<T, 1, 1, true, false, false>(g, st);
    } else {
        if (tile == TILE_128) launch_staged<T, 2, 2, false, false, false>(g, st); else launch_staged<T, 1, 1, false, false, false>(g, st);
    }
    return dense_launch_error("dense matrix product");
}

}  // namespace v2vae
#endif
