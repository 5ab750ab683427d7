// Matrix product of the dense layers for 16-bit operands whose rows are 16-byte aligned: tiles go from memory to LDS directly.
//
// Mathematics and arguments as in v2vae_dense_gemm.h.  WM x WN waves own a tile of 32 TM WM x 32 TN WN outputs; a contraction step
// is 64 elements, two steps' tiles live in LDS, and while one is multiplied the loads of the next (global_load_lds, 16 bytes a
// lane, no registers) are in flight: one barrier a step.  Such a load writes its 64 pieces in lane order, so the order of pieces
// in LDS is chosen by which piece a lane fetches:
//  * contraction contiguous: a row is 8 pieces; row r holds piece p at position p ^ (r / 2 % 8), and the 16-byte reads of a
//    fragment (32 rows, one piece each) spread over all banks;
//  * rows contiguous: a contraction index is a line of 32 TM WM (or TN WN) elements, read as a transposed fragment by
//    ds_read_b64_tr_b16 (16 lanes read 4 k x 16 rows and receive 4 k of one row each).  Line k holds its 64-byte blocks at
//    position b ^ (k % 4 + 4 (k / 8 % 2)): the eight lines that one instruction reads then fall on different banks.
// Rows beyond the matrix repeat its last row (or last 16 bytes): their products are not stored.  The last step of a contraction
// that is not a multiple of 64 takes the 16-byte pieces (or lines) beyond it from a page of zeros.  Operands whose rows are not whole
// pieces come as copies that are padded with zeros (pad_a, pad_b; v2vae_dense.hip).
//
// Three tiles (the rule is cut_product's): 256 x 256 on eight waves of 128 x 64, which asks memory for half as much as 128 x 128 on
// four waves of 64 x 64; 128 x 64 for outputs of one column of tiles (60992 x 88 -> 16: 10 us, 28 with 256 x 256).  The loads of a
// step have one step of products to arrive in, so the larger tile, with twice the products a step, waits less: bound by that
// latency and by the clock, which the chip's power holds at 1.9 ... 2.0 GHz under it; the matrix unit is busy 40 ... 56 % of the cycles.
// bf16, 8192 x 4096 -> 4096: forward with residual 252 us (1090 TF), dx 234 (1170 TF), dw 220 (1250 TF); 4999 x 2048 -> 2 x 5632 gated
// forward 241 (957 TF).  Measured and not kept: 256 x 256 on four waves of 128 x 128 (training pass 841 us against 750), loads spread
// over the step's products (gated forward 272 against 253), raised wave priority around the products (no change).
#ifndef V2VAE_DENSE_DIRECT_H
#define V2VAE_DENSE_DIRECT_H
#include "v2vae_dense_gemm.h"

namespace v2vae {

__device__ __align__(16) const unsigned g_zero_piece[4] = {0, 0, 0, 0};

// 64 lanes' pieces of 16 bytes from base + off to LDS at lds + 16 lane.  Not tracked by the compiler: wait_tile() waits for them and
// is what LDS reads may not cross; between two of its calls reads and loads concern different tiles and may change places.
__device__ __forceinline__ void load_to_lds(const void* base, unsigned off, unsigned lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0");
}
__device__ __forceinline__ void load_to_lds(const void* at, unsigned lds) {
    lds = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(at), "s"(lds) : "m0");
}
// this wave's loads have landed and its LDS reads are done, then all waves' (the builtin, so that the compiler knows that its own
// loads have arrived as well and asks for no wait of its own after the next ones are under way)
__device__ __forceinline__ void wait_tile() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

template <typename V> __device__ __forceinline__ V uniform64(V p) {
    const uint64_t u = (uint64_t)p;
    const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)u), hi = __builtin_amdgcn_readfirstlane((unsigned)(u >> 32));
    return (V)(((uint64_t)hi << 32) | lo);
}

// One operand: ROWS rows of the tile, loaded by NW waves.
template <typename T, int ROWS, int NW, bool KC, bool GATED> struct Tile {
    static constexpr int LOADS = ROWS / 8 / NW, BYTES = ROWS * 128;
    unsigned off[LOADS];  // byte offset of this lane's piece from the tile's corner
    // corner: first row of the tile; R rows (features) in all
    __device__ __forceinline__ void init(int lane, int wave, int64_t ld, int first, int R, const int64_t* ld2) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const int i = j * NW + wave;
            if constexpr (KC) {
                const int r = i * 8 + (lane >> 3), piece = (lane & 7) ^ ((r >> 1) & 7);
                int row = GATED ? (r >> 6) * 32 + (r & 31) : r;
                row = first + row < R ? row : R - 1 - first;
                off[j] = (unsigned)(row * (GATED ? ld2[(r >> 5) & 1] : ld) + piece * 8) * 2u;
            } else {
                const int k = (i * 64 + lane) / (ROWS / 8), p = (i * 64 + lane) % (ROWS / 8);
                const int piece = p ^ (4 * ((k & 3) | (((k >> 3) & 1) << 2)) % (ROWS / 8));
                const int row = first + piece * 8 < R ? piece * 8 : (R - 1) / 8 * 8 - first;
                off[j] = (unsigned)(k * ld + row) * 2u;
            }
        }
    }
    // loads lo ... hi - 1 of this wave; base0 (base1): corner at contraction index k0, left = contraction elements from k0 on
    template <bool TAIL> __device__ __forceinline__ void fetch(const char* base0, const char* base1, int left, int lane, int wave, unsigned lds,
                                                               int lo, int hi) const {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            if (j < lo || j >= hi) continue;
            const int i = j * NW + wave;
            const char* b = GATED && (((i * 8) >> 5) & 1) ? base1 : base0;
            if constexpr (TAIL) {
                int k;
                if constexpr (KC) k = ((lane & 7) ^ (((i * 8 + (lane >> 3)) >> 1) & 7)) * 8; else k = (i * 64 + lane) / (ROWS / 8);
                load_to_lds(k < left ? (const void*)(b + off[j]) : (const void*)g_zero_piece, lds + i * 1024);
            } else {
                load_to_lds(b, off[j], lds + i * 1024);
            }
        }
    }
};

template <typename T, int WM, int WN, int TM, int TN, bool AKC, bool BKC, bool GATED>
__global__ __launch_bounds__(64 * WM * WN, (WM * WN) / 4) void k_gemm_direct(GemmArgs g) {
    typedef typename Elem<T>::frag frag;
    typedef __attribute__((ext_vector_type(4))) short s16x4;
    constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, STAGE = (BM + BN) * 128;
    static_assert(TN % 2 == 0, "the epilogue takes blocks in pairs (gated: gate and up)");
    static_assert(NW * EPI_BYTES<2> <= 2 * STAGE, "the epilogue's rows fit the tiles' memory");
    __shared__ __align__(1024) char lds[2 * STAGE];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    const int out_bn = GATED ? BN / 2 : BN;
    const int tiles_m = (g.M + BM - 1) / BM, tiles_n = (g.N + out_bn - 1) / out_bn;
    int tm, tn;
    tile_of(blockIdx.x, tiles_m, tiles_n, &tm, &tn);
    const int split = blockIdx.y, bat = blockIdx.z, m0 = tm * BM, n0 = tn * out_bn;
    const int steps_seg = (g.K + 63) / 64, steps = steps_seg * g.segs;
    const int s_lo = split * g.steps_per_split, s_hi = s_lo + g.steps_per_split < steps ? s_lo + g.steps_per_split : steps;
    // operands of the two segments (a batch entry has one)
    const void *const a_0 = g.a[bat], *const a_1 = g.a[1], *const b_0 = g.b[bat], *const b_1 = g.b[1];
    const int64_t ldb_0 = g.ldb[bat], ldb_1 = g.ldb[1];
    const unsigned lds0 = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds;

    Tile<T, BM, NW, AKC, false> ta;
    Tile<T, BN, NW, BKC, GATED> tb;
    ta.init(lane, wave, g.lda, m0, g.M, nullptr);
    tb.init(lane, wave, g.ldb[bat], n0, g.N, g.ldb);
    // where the next tile comes from: corners of both operands at its contraction index, what is left of its segment
    const int64_t step_a = (AKC ? 64 : 64 * g.lda) * 2;
    const char *pa, *pb, *pb1 = nullptr;
    int left, seg;
    int64_t step_b;
    auto enter = [&](int sg, int k0) {
        seg = sg;
        left = g.K - k0;
        const int64_t ldb = sg ? ldb_1 : ldb_0;
        step_b = (BKC ? 64 : 64 * ldb) * 2;
        pa = uniform64((const char*)(sg ? a_1 : a_0) + (AKC ? (int64_t)m0 * g.lda + k0 : (int64_t)k0 * g.lda + m0) * 2);
        pb = uniform64((const char*)(sg ? b_1 : b_0) + (BKC ? (int64_t)n0 * ldb + k0 : (int64_t)k0 * ldb + n0) * 2);
        if constexpr (GATED) pb1 = uniform64((const char*)b_1 + ((int64_t)n0 * ldb_1 + k0) * 2);
    };
    int at_step = 0;  // step that the corners stand at
    auto go_to = [&](int s) {
        at_step = s;
        enter(s >= steps_seg ? 1 : 0, (s >= steps_seg ? s - steps_seg : s) * 64);
    };
    auto advance = [&]() {
        ++at_step;
        if (at_step < s_hi && left > 64) {
            left -= 64;
            pa += step_a;
            pb += step_b;
            if constexpr (GATED) pb1 += step_b;
        } else {
            go_to(at_step < s_hi ? at_step : s_lo);
        }
    };
    constexpr int LA = Tile<T, BM, NW, AKC, false>::LOADS, LB = Tile<T, BN, NW, BKC, GATED>::LOADS;
    auto fetch = [&](int buf, int lo, int hi) {  // loads lo ... hi - 1 of the next tile, A's first
        if (left >= 64) {
            ta.template fetch<false>(pa, nullptr, left, lane, wave, lds0 + buf * STAGE, lo, hi);
            tb.template fetch<false>(pb, pb1, left, lane, wave, lds0 + buf * STAGE + BM * 128, lo - LA, hi - LA);
        } else {
            ta.template fetch<true>(pa, nullptr, left, lane, wave, lds0 + buf * STAGE, lo, hi);
            tb.template fetch<true>(pb, pb1, left, lane, wave, lds0 + buf * STAGE + BM * 128, lo - LA, hi - LA);
        }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    // LDS byte offsets of this lane's fragments.  Contraction contiguous: row base + piece kk * 2 + lane / 32, one offset per kk.
    // Rows contiguous: 4 k x 16 rows per 16 lanes; one offset per 32-row block, kk and the two halves as constants.
    constexpr int OA = AKC ? 4 : TM, OB = BKC ? 4 : TN;
    unsigned oa[OA], ob[OB];
    const int g16 = lane >> 4, i16 = lane & 15, ks = (i16 >> 2) | ((g16 >> 1) << 2);
    auto mn_offset = [&](int block, int rows) {
        const int k = (g16 >> 1) * 8 + (i16 >> 2);
        return (unsigned)(k * rows * 2 + (((block ^ ks) % (rows / 32)) * 64) + (g16 & 1) * 32 + (i16 & 3) * 8);
    };
#pragma unroll
    for (int q = 0; q < OA; ++q) {
        if constexpr (AKC) oa[q] = (unsigned)((wm * 32 * TM + (lane & 31)) * 128 + (((q * 2 + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16));
        else oa[q] = mn_offset(wm * TM + q, BM);
    }
#pragma unroll
    for (int q = 0; q < OB; ++q) {
        if constexpr (BKC) ob[q] = (unsigned)((wn * 32 * TN + (lane & 31)) * 128 + (((q * 2 + (lane >> 5)) ^ ((lane >> 1) & 7)) * 16));
        else ob[q] = mn_offset(wn * TN + q, BN);
    }
    auto frag_mn = [&](unsigned at, int rows, int kk) {
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + kk * 32 * rows));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)(at + kk * 32 * rows + 8 * rows));
        union { s16x4 h[2]; frag f; } u;
        u.h[0] = lo;
        u.h[1] = hi;
        return u.f;
    };
    typedef __attribute__((address_space(3))) frag lds_frag;

    auto read = [&](unsigned la, int kk, frag (&a)[TM], frag (&b)[TN]) {
        const unsigned lb = la + BM * 128;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if constexpr (BKC) b[j] = *(const lds_frag*)(uintptr_t)(lb + ob[kk] + j * 4096);
            else b[j] = frag_mn(lb + ob[j], BN, kk);
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            if constexpr (AKC) a[i] = *(const lds_frag*)(uintptr_t)(la + oa[kk] + i * 4096);
            else a[i] = frag_mn(la + oa[i], BM, kk);
        }
    };
    // Neighbouring tiles start up to seven steps apart in the contraction and wrap round: rows a power of two apart would otherwise
    // have every workgroup ask the same few cache channels for the same 128-byte column of the operands at a time.
    const int n_steps = s_hi - s_lo;
    frag a[2][TM], b[2][TN];
    auto products = [&](int q) {
        // reads that were just written down are issued before these products, not where their fragments are used
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) acc[i][j] = mma32(b[q][j], a[q][i], acc[i][j]);
        __builtin_amdgcn_sched_barrier(0);
    };
    if (n_steps > 0) {
        go_to(s_lo + (n_steps >= 16 ? (int)((blockIdx.x >> 3) & 7) : 0));
        fetch(0, 0, LA + LB);
        wait_tile();
        if (n_steps > 1) {
            advance();
            fetch(1, 0, LA + LB);
        }
        read(lds0, 0, a[0], b[0]);
    }
    for (int i = 0; i < n_steps; ++i) {
        const int buf = i & 1;
        const unsigned here = lds0 + buf * STAGE;
        read(here, 1, a[1], b[1]);
        products(0);
        read(here, 2, a[0], b[0]);
        products(1);
        read(here, 3, a[1], b[1]);
        products(0);
        // The tile is read; while its last products run, the next one's first fragments come in and the one after it is asked for.
        if (i + 1 < n_steps) {
            wait_tile();
            read(lds0 + (buf ^ 1) * STAGE, 0, a[0], b[0]);
            if (i + 2 < n_steps) {
                advance();
                fetch(buf, 0, LA + LB);
            }
        }
        products(1);
    }

    wait_tile();  // LDS is free
    float* const part = g.partial ? g.partial + ((int64_t)bat * g.splits + split) * ((int64_t)g.M * (GATED ? 2 : 1) * g.N) : nullptr;
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; j += 2) {
            const f32x16 pair[2] = {acc[i][j], acc[i][j + 1]};
            finish_block<T, 2, GATED>(g, pair, lds + wave * EPI_BYTES<2>, lane, m0 + (wm * TM + i) * 32,
                                      n0 + (wn * TN + j) * (GATED ? 16 : 32), part, bat);
        }
}

template <typename T, int WM, int WN, int TM, int TN, bool AKC, bool BKC, bool GATED> void launch_direct(const GemmArgs& g, hipStream_t st) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN / (GATED ? 2 : 1);
    const int64_t tiles = (int64_t)((g.M + BM - 1) / BM) * ((g.N + BN - 1) / BN);
    hipLaunchKernelGGL((k_gemm_direct<T, WM, WN, TM, TN, AKC, BKC, GATED>), dim3((unsigned)tiles, g.splits, g.batch), dim3(64 * WM * WN), 0,
                       st, g);
    if (g.partial) launch_join<T, GATED>(g, st);
}
template <typename T, bool AKC, bool BKC, bool GATED> void pick_direct(const GemmArgs& g, int tile, hipStream_t st) {
    if (tile == TILE_256) launch_direct<T, 2, 4, 4, 2, AKC, BKC, GATED>(g, st);
    else if (tile == TILE_64) launch_direct<T, 4, 1, 1, 2, AKC, BKC, GATED>(g, st);
    else launch_direct<T, 2, 2, 2, 2, AKC, BKC, GATED>(g, st);
}
template <typename T> int gemm_direct(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    if (gated) pick_direct<T, true, true, true>(g, tile, st);
    else if (layout == LAYOUT_KK) pick_direct<T, true, true, false>(g, tile, st);
    else if (layout == LAYOUT_KM) pick_direct<T, true, false, false>(g, tile, st);
    else pick_direct<T, false, false, false>(g, tile, st);
    return dense_launch_error("dense matrix product");
}

}  // namespace v2vae
#endif
