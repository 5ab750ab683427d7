// Matrix product of the dense layers for float32 operands on the bf16 matrix pipe: D[m][n] = sum_k A(m, k) B(n, k).
//
// Every float is the exact sum of three bf16 pieces (v2vae_bf16_split.h; here the gfx950 conversion instruction rounds two at a
// time) and the six piece products down to 2^-24 of the whole are accumulated in float, the smallest first: float32 results at
// six bf16 instructions, bf16 rate / 6 = 417 TF at the peak where the f32 matrix instructions give 157 TF.
//
// A workgroup of four waves owns 128 rows x 32 TN columns, every wave 32 whole rows of it.  A's rows belong to one wave alone, so
// they go from memory to registers in the layout of the matrix operand (8 consecutive k a lane; any alignment: gfx950 loads 16
// bytes at 4-byte addresses) and are split there, once, without LDS or a barrier.  B's tile (the weights, or the narrow side of a
// weight gradient) is shared through LDS as three planes of 32-element rows 80 bytes apart (16 rows touch every bank once), two
// steps' tiles so that there is one barrier a step.  Splitting costs 5.5 vector instructions an element, so
//  * B_PLANES: weights that many row blocks use are split once per call, into planes in the workspace (k_split_planes) whose
//    tiles then go to LDS directly (global_load_lds), 64 bytes a row, pieces of 16 bytes permuted so that 16 rows touch every
//    bank once; A's loads run one step ahead;
//  * B_ROWS, B_COLUMNS: otherwise the workgroup splits its tile on the way into LDS (contraction or rows contiguous in memory).
//    Both operands then come from far away and run two steps ahead, in two register sets each; the last two steps are written out
//    so that the loop's loads are unconditional and the compiler can count what is in flight.
// Bound by issue and latency: splitting A (44 vector instructions a step and 32 x 32 block of it) and the matrix instructions share a
// SIMD's cycles, which is why planes pay and why wider tiles do, up to the registers: 32768 x 256 -> 2 x 512 gated forward 121 us (142 TF,
// or 850 TF of bf16 products; 39 us of it are its bytes; a SIMD issues vector instructions for 41 us and is busy with matrix ones for 43),
// its dx 95, dw 107; 65536 x 256 -> 130 38 us.  Contractions of a step or two wait more than they issue: 262144 x 50 -> 64 37 us, of which
// 23 are its bytes, 22 vector and 5 matrix instructions, because a workgroup's epilogue has no load in flight.  Measured and not kept: blocks of zeros at the edge skipped by a branch (training pass 420 us against 405), planes
// through registers two steps ahead (fewer waves, slower).
// One scalar base and 32-bit lane offsets per load: strides are at most 2^22 elements.
// Rows beyond the matrix repeat its last one (their products are not stored); contraction ends take zeros, element by element.
#ifndef V2VAE_DENSE_SPLIT_H
#define V2VAE_DENSE_SPLIT_H
#include "v2vae_dense_direct.h"

namespace v2vae {

enum { B_ROWS, B_COLUMNS, B_PLANES };

__device__ __forceinline__ float at(const char* base, unsigned off) { return *reinterpret_cast<const float*>(base + off); }
// element `e` steps after base + off, which is element k of the contraction; beyond its end 0 (and the last one is read instead)
__device__ __forceinline__ float tail_at(const char* base, unsigned off, int k, int left, int64_t step, int e) {
    const int back = k < left ? 0 : k - left + 1;
    const float v = *reinterpret_cast<const float*>(base + off + (e - back) * step);
    return back ? 0.f : v;
}

template <int TN, bool AKC, int FROM, bool GATED>
__global__ __launch_bounds__(256, FROM == B_PLANES ? (TN <= 2 ? 4 : TN <= 4 ? 3 : 2) : 2) void k_gemm_split(GemmArgs g) {
    constexpr int BK = 32, BM = 128, BN = 32 * TN, EPI = 4 * EPI_BYTES<2>;
    constexpr bool PLANES = FROM == B_PLANES, BKC = FROM == B_ROWS;
    constexpr int ROWB = PLANES ? 64 : 80, PLANE = BN * ROWB, TILE = 3 * PLANE;
    static_assert(TN % 2 == 0 || (PLANES && !GATED), "tiles of an odd number of blocks: weights from planes, one matrix");
    __shared__ __align__(1024) char lds[2 * TILE > EPI ? 2 * TILE : EPI];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int out_bn = GATED ? BN / 2 : BN;
    const int tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.N + out_bn - 1) / out_bn;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const int split = blockIdx.y, bat = blockIdx.z, mt = tm * BM, m0 = mt + wave * 32, n0 = tn * out_bn;
    const int steps_seg = (g.K + BK - 1) / BK, steps = steps_seg * g.segs;
    const int s_lo = split * g.steps_per_split, s_hi = s_lo + g.steps_per_split < steps ? s_lo + g.steps_per_split : steps;
    // operands of the two segments (a batch entry has one)
    const void *const a_0 = g.a[bat], *const a_1 = g.a[1], *const b_0 = g.b[bat], *const b_1 = g.b[1];
    const int64_t ldb_0 = g.ldb[bat], ldb_1 = g.ldb[1], lda = g.lda;

    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

    // lane offsets (bytes) from the tile's corner
    const int row_a = m0 + (lane & 31) < g.M ? m0 + (lane & 31) - mt : g.M - 1 - mt;
    const unsigned off_a = AKC ? (unsigned)(row_a * lda + half * 8) * 4u : (unsigned)(row_a + half * 8 * lda) * 4u;
    // The last step of a row reads on into the rows that follow, zeroed when it is split, where there is that much behind the tile.
    const bool over = AKC && (int64_t)(g.M - mt - BM) * lda >= BK;
    typedef struct __attribute__((packed, aligned(4))) { float e[4]; } Loose4;
    constexpr int PASS = BN / 32, KT = BK * BN / 256;  // B_ROWS: 16-byte loads, B_COLUMNS: elements, per thread
    constexpr int LOADS = 3 * BN / 16, NB = PLANES ? (LOADS + 3) / 4 : BKC ? PASS : 1;
    struct SetA { float v[2][8]; };
    struct SetB { float v[PLANES ? 1 : KT]; };
    unsigned off_b[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        if constexpr (PLANES) {  // 16 rows of one plane an instruction
            const int i = j * 4 + wave < LOADS ? j * 4 + wave : LOADS - 1, plane = i / (BN / 16);
            const int r = i % (BN / 16) * 16 + (lane >> 2), piece = (lane & 3) ^ ((r >> 2) & 3);
            const int last = g.plane_rows - 1, row = tn * BN + r < last ? tn * BN + r : last;
            off_b[j] = (unsigned)((int64_t)plane * g.plane_bytes + (int64_t)(row - tn * BN) * g.plane_ld * 2 + piece * 16);
        } else if constexpr (BKC) {
            const int r = (tid >> 3) + 32 * j;
            int row = GATED ? (r >> 6) * 32 + (r & 31) : r;  // blocks of 32 rows: gate and up of the same features in turn
            row = n0 + row < g.N ? row : g.N - 1 - n0;
            off_b[j] = (unsigned)(row * g.ldb[GATED ? j & 1 : 0] + (tid & 7) * 4) * 4u;
        } else {
            const int r = tid % BN, row = n0 + r < g.N ? r : g.N - 1 - n0;
            off_b[j] = (unsigned)row * 4u;
        }
    }
    auto fetch_b = [&](int s, SetB& rb) {
        const int seg = s >= steps_seg ? 1 : 0, k0 = (s - seg * steps_seg) * BK, left = g.K - k0;
        const int64_t ldb = seg ? ldb_1 : ldb_0;
        if constexpr (BKC) {
#pragma unroll
            for (int j = 0; j < PASS; ++j) {
                const bool second = GATED ? j & 1 : seg;
                const char* const b = (const char*)(second ? b_1 : b_0) + ((int64_t)n0 * (second ? ldb_1 : ldb_0) + k0) * 4;
                if (left >= BK) {
                    const Loose4 t = *reinterpret_cast<const Loose4*>(b + off_b[j]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) rb.v[4 * j + e] = t.e[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) rb.v[4 * j + e] = tail_at(b, off_b[j], (tid & 7) * 4 + e, left, 4, e);
                }
            }
        } else {
            const char* const b = (const char*)(seg ? b_1 : b_0) + ((int64_t)k0 * ldb + n0) * 4;
            const int kt = (tid / BN) * KT;
            const unsigned off = off_b[0] + (unsigned)(kt * ldb) * 4u;
            if (left >= BK) {
#pragma unroll
                for (int e = 0; e < KT; ++e) rb.v[e] = at(b + e * ldb * 4, off);
            } else {
#pragma unroll
                for (int e = 0; e < KT; ++e) rb.v[e] = tail_at(b, off, kt + e, left, ldb * 4, e);
            }
        }
    };
    auto planes_to_lds = [&](int s, int buf) {
        const char* const b = uniform64((const char*)g.planes + ((int64_t)tn * BN * g.plane_ld + (int64_t)s * BK) * 2);
#pragma unroll
        for (int j = 0; j < NB; ++j)
            if (LOADS % 4 == 0 || j * 4 + wave < LOADS) load_to_lds(b, off_b[j], lds0 + buf + (j * 4 + wave) * 1024);
    };
    auto fetch_a = [&](int s, SetA& ra) {
        const int seg = s >= steps_seg ? 1 : 0, k0 = (s - seg * steps_seg) * BK, left = g.K - k0;
        const char* const a = (const char*)(seg ? a_1 : a_0) + (AKC ? (int64_t)mt * lda + k0 : (int64_t)k0 * lda + mt) * 4;
        if (left >= BK || over) {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                if constexpr (AKC) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const Loose4 t = *reinterpret_cast<const Loose4*>(a + q * 64 + h * 16 + off_a);
#pragma unroll
                        for (int e = 0; e < 4; ++e) ra.v[q][4 * h + e] = t.e[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) ra.v[q][e] = at(a + (q * 16 + e) * lda * 4, off_a);
                }
            }
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) ra.v[q][e] = tail_at(a, off_a, q * 16 + e + half * 8, left, AKC ? 4 : lda * 4, q * 16 + e);
        }
    };
    auto store_b = [&](char* tile, const SetB& rb) {
        if constexpr (BKC) {
#pragma unroll
            for (int j = 0; j < PASS; ++j) {
                unsigned lo[3], hi[3];
                split_pair(rb.v[4 * j], rb.v[4 * j + 1], lo);
                split_pair(rb.v[4 * j + 2], rb.v[4 * j + 3], hi);
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x2*>(tile + p * PLANE + ((tid >> 3) + 32 * j) * ROWB + (tid & 7) * 8) = u32x2{lo[p], hi[p]};
            }
        } else {
#pragma unroll
            for (int e = 0; e < KT; e += 8) {
                unsigned q[4][3];
#pragma unroll
                for (int i = 0; i < 4; ++i) split_pair(rb.v[e + 2 * i], rb.v[e + 2 * i + 1], q[i]);
#pragma unroll
                for (int p = 0; p < 3; ++p)
                    *reinterpret_cast<u32x4*>(tile + p * PLANE + (tid % BN) * ROWB + (tid / BN) * KT * 2 + e * 2) =
                        u32x4{q[0][p], q[1][p], q[2][p], q[3][p]};
            }
        }
    };

    f32x16 acc[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[j][e] = 0.f;

    // fragments of B: row lane % 32 of a block, 8 k from 16 q + 8 half
    unsigned fb[2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
        fb[q] = (lane & 31) * ROWB + (PLANES ? ((q * 2 + half) ^ ((lane >> 2) & 3)) * 16 : q * 32 + half * 16);
    auto split_a = [&](int s, SetA& ra, bf16x8 (&a)[2][3]) {
        const int left = g.K - (s >= steps_seg ? s - steps_seg : s) * BK;
        if (over && left < BK) {
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int e = 0; e < 8; ++e) ra.v[q][e] = q * 16 + half * 8 + e < left ? ra.v[q][e] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            union { unsigned u[4]; bf16x8 f; } w[3];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                unsigned p[3];
                split_pair(ra.v[q][2 * e], ra.v[q][2 * e + 1], p);
#pragma unroll
                for (int c = 0; c < 3; ++c) w[c].u[e] = p[c];
            }
#pragma unroll
            for (int c = 0; c < 3; ++c) a[q][c] = w[c].f;
        }
    };
    auto multiply = [&](const bf16x8 (&a)[2][3], int buf) {
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                bf16x8 b[3];
#pragma unroll
                for (int c = 0; c < 3; ++c) b[c] = *reinterpret_cast<const bf16x8*>(lds + (fb[q] + buf) + c * PLANE + j * 32 * ROWB);
#pragma unroll
                for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                    for (int c = 0; c <= sum; ++c) acc[j] = mma32(b[sum - c], a[q][c], acc[j]);
            }
    };
    SetA ra[2];
    if constexpr (PLANES) {
        if (s_lo < s_hi) {
            planes_to_lds(s_lo, 0);
            fetch_a(s_lo, ra[0]);
        }
        for (int s = s_lo; s < s_hi; ++s) {
            const int buf = ((s - s_lo) & 1) * TILE;
            wait_tile();
            if (s + 1 < s_hi) {
                planes_to_lds(s + 1, TILE - buf);
                fetch_a(s + 1, ra[1]);
            }
            bf16x8 a[2][3];
            split_a(s, ra[0], a);
            multiply(a, buf);
            ra[0] = ra[1];
        }
    } else {
        SetB rb[2];
        // one step: U = parity of its tile and sets; load: two steps later exist; store: a next step exists
        auto step = [&](int s, auto U, auto load, auto store) {
            constexpr int u = decltype(U)::value;
            __syncthreads();  // this step's tile is written, the other one read
            if constexpr (decltype(store)::value) store_b(lds + (u ^ 1) * TILE, rb[u ^ 1]);
            bf16x8 a[2][3];
            split_a(s, ra[u], a);
            if constexpr (decltype(load)::value) {
                fetch_b(s + 2, rb[u]);
                fetch_a(s + 2, ra[u]);
            }
            multiply(a, u * TILE);
        };
        constexpr std::integral_constant<int, 0> even{};
        constexpr std::integral_constant<int, 1> odd{};
        constexpr std::true_type yes{};
        constexpr std::false_type no{};
        int s = s_lo;
        if (s < s_hi) {
            fetch_b(s, rb[0]);
            fetch_a(s, ra[0]);
            if (s + 1 < s_hi) {
                fetch_b(s + 1, rb[1]);
                fetch_a(s + 1, ra[1]);
            }
            store_b(lds, rb[0]);
            for (; s + 3 < s_hi; s += 2) {
                step(s, even, yes, yes);
                step(s + 1, odd, yes, yes);
            }
            if (s_hi - s == 3) {
                step(s, even, yes, yes);
                step(s + 1, odd, no, yes);
                step(s + 2, even, no, no);
            } else if (s_hi - s == 2) {
                step(s, even, no, yes);
                step(s + 1, odd, no, no);
            } else {
                step(s, even, no, no);
            }
        }
    }
    __syncthreads();

    float* const part = g.partial ? g.partial + ((int64_t)bat * g.splits + split) * ((int64_t)g.M * (GATED ? 2 : 1) * g.N) : nullptr;
#pragma unroll
    for (int j = 0; j + 1 < TN; j += 2) {
        const f32x16 pair[2] = {acc[j], acc[j + 1]};
        finish_block<float, 2, GATED>(g, pair, lds + wave * EPI_BYTES<2>, lane, m0, n0 + (GATED ? 16 : 32) * j, part, bat);
    }
    if constexpr (TN % 2 != 0) {
        const f32x16 last[1] = {acc[TN - 1]};
        finish_block<float, 1, false>(g, last, lds + wave * EPI_BYTES<2>, lane, m0, n0 + 32 * (TN - 1), part, bat);
    }
}

// One pass over the weights, 2 x 512 rows of 256: 4 us, transposed 6.5; most of it is the launch.
// Weights -> three planes [rows][ld] of bf16 pieces, contraction contiguous, zeros beyond its end (ld is a multiple of 32).
//  forward: plane row r is weight row r; gated: blocks of 32 rows, gate and up of the same features in turn.
//  backward (TRANSPOSED): plane row r is weight column r, the contraction runs over the weights' rows (gated: gate's, padded to a
//  multiple of 32, then up's).
struct PlaneArgs {
    const float* w[2];
    int64_t ld_w[2];
    char* out;
    int64_t plane_bytes;
    int rows, ld, N, K, gated;  // planes; weights N x K
};
template <bool TRANSPOSED> __global__ __launch_bounds__(256) void k_split_planes(PlaneArgs a) {
    __shared__ float s_t[TRANSPOSED ? 32 : 1][TRANSPOSED ? 65 : 1];
    const int tid = threadIdx.x;
    float v[8];
    int r, k;
    const int across = TRANSPOSED ? a.ld / 32 : (a.ld + 127) / 128, bx = blockIdx.x % across, by = blockIdx.x / across;
    if constexpr (TRANSPOSED) {  // 32 k x 64 rows a block
        const int k0 = bx * 32, r0 = by * 64, pad = a.ld / (a.gated ? 2 : 1), which = k0 >= pad ? 1 : 0;
        for (int i = tid; i < 32 * 64; i += 256) {
            const int kk = k0 - which * pad + (i >> 6), c = r0 + (i & 63);
            s_t[i >> 6][i & 63] = kk < a.N && c < a.K ? a.w[which][kk * a.ld_w[which] + c] : 0.f;
        }
        __syncthreads();
        r = r0 + (tid >> 2);
        k = k0 + (tid & 3) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s_t[(tid & 3) * 8 + e][tid >> 2];
    } else {                     // 16 rows x 128 k a block
        r = by * 16 + (tid >> 4);
        k = bx * 128 + (tid & 15) * 8;
        const int which = a.gated ? (r >> 5) & 1 : 0, f = a.gated ? (r >> 6) * 32 + (r & 31) : r;
        const float* const p = a.w[which] + f * a.ld_w[which];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = f < a.N && k + e < a.K ? p[k + e] : 0.f;
    }
    if (r >= a.rows || k >= a.ld) return;
    unsigned q[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_pair(v[2 * i], v[2 * i + 1], q[i]);
#pragma unroll
    for (int p = 0; p < 3; ++p)
        *reinterpret_cast<u32x4*>(a.out + p * a.plane_bytes + ((int64_t)r * a.ld + k) * 2) = u32x4{q[0][p], q[1][p], q[2][p], q[3][p]};
}

template <int TN, bool AKC, int FROM, bool GATED> void launch_split(const GemmArgs& g, hipStream_t st) {
    constexpr int BN = 32 * TN / (GATED ? 2 : 1);
    const int64_t tiles = (int64_t)((g.M + 127) / 128) * ((g.N + BN - 1) / BN);
    hipLaunchKernelGGL((k_gemm_split<TN, AKC, FROM, GATED>), dim3((unsigned)tiles, g.splits, g.batch), dim3(256), 0, st, g);
    if (g.partial) launch_join<float, GATED>(g, st);
}
template <bool AKC, int FROM, bool GATED> void pick_split(const GemmArgs& g, int tile, hipStream_t st) {
    if constexpr (FROM == B_PLANES && !GATED) {
        if (tile == TILE_96) return launch_split<3, AKC, FROM, GATED>(g, st);
        if (tile == TILE_160) return launch_split<5, AKC, FROM, GATED>(g, st);
    }
    if (tile == TILE_128) launch_split<4, AKC, FROM, GATED>(g, st); else launch_split<2, AKC, FROM, GATED>(g, st);
}

}  // namespace v2vae
#endif
