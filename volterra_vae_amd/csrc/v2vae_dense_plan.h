// How the calls of the dense layers are cut and what workspace they take: host arithmetic alone, no HIP, so that a program without a
// GPU can go through it over as many sizes as it likes.
#ifndef V2VAE_DENSE_PLAN_H
#define V2VAE_DENSE_PLAN_H
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/v2vae_hip.h"

namespace v2vae {

enum { TILE_128, TILE_64, TILE_256, TILE_96, TILE_160 };  // float32: columns of a tile of 128 rows; else both sides

// few rows (v2vae_dense_rows.hip); beyond, the tiled products read the weights as fast
inline int64_t few_rows(int dtype) { return dtype == V2VAE_F32 ? 32 : 16; }
// Parts of the contraction there.  Float on few, long weight rows: the contraction in parts, to a workgroup a compute unit (9 x 8165 -> 2 x 504: 25 us in one part,
// 16.7 in four and their join, kernels of 11.4 and 4.8).  16-bit rows, of half the bytes, end before a second launch would pay.
inline int rows_splits(int dtype, int64_t in, int64_t out, bool gated) {
    if (dtype != V2VAE_F32) return 1;
    const int64_t groups = gated ? (out + 7) / 8 : (out + 15) / 16;
    int64_t s = 256 / groups;
    if (s > in / 1024) s = in / 1024;
    if (s < 3) return 1;
    const int64_t turns = in / 128, per = (turns + s - 1) / s;
    return (int)((turns + per - 1) / per);  // none without a turn
}

inline int elem_bytes(int dtype) { return dtype == V2VAE_F32 ? 4 : 2; }
inline size_t round_up(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr int64_t ROWS_LIMIT = (int64_t)1 << 30, WIDTH_LIMIT = (int64_t)1 << 22;  // columns and strides: 32-bit offsets inside a tile

inline int check_dense(const v2vae_dense* d, bool gated, bool backward, bool residual) {
    if (!d || d->dtype < V2VAE_F32 || d->dtype > V2VAE_F16) return V2VAE_EINVAL;
    if (d->activation < V2VAE_ACT_NONE || d->activation > V2VAE_ACT_TANH) return V2VAE_EINVAL;
    if (d->rows < 0 || d->in < 1 || d->out < 1) return V2VAE_EINVAL;
    if (d->rows > ROWS_LIMIT || d->in > WIDTH_LIMIT || d->out > WIDTH_LIMIT) return V2VAE_ESIZE;
    if (d->ld_x < 0 || d->ld_w < 0 || (gated && d->ld_w2 < 0)) return V2VAE_EINVAL;
    if ((residual && d->ld_res < 0) || (backward && d->ld_dy < 0)) return V2VAE_EINVAL;
    if (d->ld_x > WIDTH_LIMIT || d->ld_w > WIDTH_LIMIT || (gated && d->ld_w2 > WIDTH_LIMIT) || (residual && d->ld_res > WIDTH_LIMIT) ||
        (backward && d->ld_dy > WIDTH_LIMIT))
        return V2VAE_ESIZE;
    // a launch holds fewer than 2^32 threads: 256 for every tile of 64 x 64 (gated forward: 64 x 32 features)
    const int64_t m = (d->rows + 63) / 64, n = (d->out + 63) / 64 * (gated ? 2 : 1), k = (d->in + 63) / 64, most = (int64_t)1 << 24;
    if (m * n >= most || m * k >= most || n * k >= most) return V2VAE_ESIZE;
    return V2VAE_OK;
}

constexpr double PACK_FORWARD = 4e9, PACK_BACKWARD = 3e8;  // rows x in x out from which copies pay

// float32: planes of split weights, for a forward (plane rows = weight rows) or a dx product (plane rows = weight columns).
// From 1024 rows on: then at least eight row blocks share every weight, and splitting it once saves more vector work in the
// product than the pass over the weights costs.
struct Planes { int rows, ld; size_t plane, bytes; };
inline Planes planes_of(const v2vae_dense* d, bool gated, bool transposed) {
    Planes p = {};
    if (d->dtype != V2VAE_F32 || d->rows < 1024) return p;
    auto pad = [](int64_t n) { return (n + 31) / 32 * 32; };
    p.rows = (int)(transposed ? d->in : gated ? 2 * pad(d->out) : d->out);
    p.ld = (int)(transposed ? pad(d->out) * (gated ? 2 : 1) : pad(d->in));
    p.plane = (size_t)p.rows * p.ld * 2;
    // a tile's lane offsets span all three planes in 32 bits, and its columns are counted in 31
    if (2 * p.plane + (size_t)160 * p.ld * 2 >= (size_t)0xFFFF0000u) return Planes{};
    p.bytes = round_up(3 * p.plane);
    return p;
}

// How a product M x N x K is cut: tile size and the number of parts of the contraction.  `direct`: 16-bit operands, aligned.
// The workspace does not know the alignment, so it is laid out for the larger of the two cuts.
struct Product { int64_t M, N, K; int segs, batch; bool gated, planes; };
struct Cut { int tile, splits, per; };
inline Cut cut_product(const Product& p, int dtype, bool direct) {
    const int64_t M = p.M, N = p.N, K = p.K, batch = p.batch;
    const bool gated = p.gated;
    const int64_t bk = dtype == V2VAE_F32 ? 32 : 64, steps = ((K + bk - 1) / bk) * p.segs;
    auto tiles_of = [&](int64_t t) { return ((M + t - 1) / t) * ((N * (gated ? 2 : 1) + t - 1) / t) * batch; };
    // A compute unit holds one 256 x 256 tile or two of 128 x 128.  The larger tile runs 1.12 times as fast (8192 x 4096 x 4096
    // training pass 755 against 861 us) where the tiles fill the matrix and the chip's last round as well: rounds() is the work of
    // all rounds (179673 x 331 -> 104 forward: 130 us with 256, 91 with 128).
    auto rounds = [&](int64_t t, int64_t slots) { return (double)((tiles_of(t) + slots - 1) / slots * slots) * t * t; };
    Cut c;
    int64_t tiles, s = 1;
    if (dtype == V2VAE_F32) {
        const int64_t rows = (M + 127) / 128, wide = rows * ((N * (gated ? 2 : 1) + 127) / 128) * batch;
        const int64_t narrow = rows * ((N * (gated ? 2 : 1) + 63) / 64) * batch;
        // 128 columns a tile where that leaves two workgroups a compute unit, of at least 16 steps if the contraction is cut (300 x
        // 2000 x 2000 forward: 39 us with 128 columns, 31 with 64) and no half-empty last column of tiles (130 columns, 65536 rows:
        // the weight gradient takes 55 us with 64 columns a tile, 76 with 128); 32768 x 256 x 512 the other way round: gated forward
        // 135 us with 128, 150 with 64
        c.tile = (wide >= 512 || wide * (steps / 16) >= 512) && wide * 2 == narrow ? TILE_128 : TILE_64;
        tiles = c.tile == TILE_128 ? wide : narrow;
        if (p.planes && !gated) {
            // One matrix of split weights: of the widths that leave two workgroups a compute unit, the one of least work.  A step
            // of a tile costs 12 cycles a column in matrix instructions and about 500 for A's splitting and the loads, whatever
            // the width (65536 x 256 -> 130: 60 us with 64 columns, 51 with 160).
            const struct { int tile, width; } widths[] = {{TILE_64, 64}, {TILE_96, 96}, {TILE_128, 128}, {TILE_160, 160}};
            int64_t best = 0;
            for (const auto& w : widths) {
                const int64_t across = (N + w.width - 1) / w.width, cost = across * (12 * w.width + 500);
                if (w.tile != TILE_64 && (rows * across < 512 || cost >= best)) continue;
                best = cost;
                c.tile = w.tile;
                tiles = rows * across;
            }
        }
    } else if (direct && N * (gated ? 2 : 1) <= 64) {  // 128 x 64: one column of tiles, more of them on a compute unit
        c.tile = TILE_64;
        tiles = ((M + 127) / 128) * batch;
    } else if (direct && tiles_of(256) >= 128 && 0.88 * rounds(256, 256) <= rounds(128, 512)) {
        c.tile = TILE_256;
        tiles = tiles_of(256);
    } else if (tiles_of(128) >= 256 || tiles_of(128) * (steps / 8) >= 256 || direct) {
        c.tile = TILE_128;
        tiles = tiles_of(128);
    } else {
        c.tile = TILE_64;
        tiles = ((M + 63) / 64) * ((N + 63) / 64) * batch;
    }
    if (tiles < 256) {
        // The contraction in parts, to two workgroups a compute unit; a part is eight steps at least (1000 x 1000 x 1000 float32
        // forward: 29 us, 38 with four), four where there are few tiles (100 x 500 x 700: 19 us with eight, 15 with four).
        const int64_t least = tiles < 32 ? 4 : 8;
        s = 512 / (tiles < 1 ? 1 : tiles);
        if (s > steps / least) s = steps / least;
        if (s < 1) s = 1;
    }
    c.per = (int)((steps + s - 1) / s);
    if (c.per < 1) c.per = 1;
    c.splits = (int)((steps + c.per - 1) / c.per);
    if (c.splits < 1) c.splits = 1;
    return c;
}
// the sums of its parts: bytes that `batch` products cut this way write, and room for either alignment
inline size_t cut_bytes(const Product& p, const Cut& c, int batch) {
    return c.splits > 1 ? (size_t)c.splits * batch * p.M * p.N * (p.gated ? 2 : 1) * 4 : 0;
}
inline size_t partial_bytes(const Product& p, int dtype) {
    size_t most = 0;
    for (int direct = 0; direct < (dtype == V2VAE_F32 ? 1 : 2); ++direct) {
        const size_t n = cut_bytes(p, cut_product(p, dtype, direct), p.batch);
        if (n > most) most = n;
    }
    return round_up(most);
}

// The three products of a layer.  A gated block's weight gradients are one product of two batch entries and are cut as such
// also where a call wants one of them alone: the sums are then the same to the bit, and the workspace has room for them.
inline Product forward_product(const v2vae_dense* d, bool gated) {
    return Product{d->rows, d->out, d->in, 1, 1, gated, planes_of(d, gated, false).bytes > 0};
}
inline Product input_product(const v2vae_dense* d, bool gated) {
    return Product{d->rows, d->in, d->out, gated ? 2 : 1, 1, false, planes_of(d, gated, true).bytes > 0};
}
inline Product weight_product(const v2vae_dense* d, bool gated) {
    return Product{d->out, d->in, d->rows, 1, gated ? 2 : 1, false, false};
}

inline size_t rows_bytes(const v2vae_dense* d, bool gated) {
    const int s = rows_splits(d->dtype, d->in, d->out, gated);
    return s > 1 ? round_up((size_t)s * d->rows * d->out * (gated ? 2 : 1) * 4) : 0;
}

inline void slope_shape(int64_t M, int64_t N, int* cx, int* gx, int* chunks) {
    const int64_t cols = (N + 3) / 4;
    int c = 1;
    while (c < cols && c < 64) c *= 2;
    // Narrower strips, down to 256 bytes of float, where they leave fewer threads without a column (gated 166354 x 302, 76 threads'
    // columns: 325 us in strips of 64, 286 in strips of 16).
    auto padded = [&](int s) { return (cols + s - 1) / s * s; };
    *cx = c;
    for (int s = c / 2; s >= 16; s /= 2)
        if (padded(s) * 4 <= padded(c) * 3 && padded(s) < padded(*cx)) *cx = s;
    c = *cx;
    *gx = (int)((cols + c - 1) / c);
    int64_t n = 2048 / *gx;
    const int64_t most = M / ((256 / c) * 4);
    if (n > most) n = most;
    if (n > 1024) n = 1024;
    *chunks = (int)(n < 1 ? 1 : n);
}

// 16-bit operands whose rows are not whole 16-byte pieces: copied when the products are large enough to win the copies back.
// Measured in bf16, forward and gradients, us without / with copies: 4001 x 2047 x 2043 86 / 63 and 518 / 138, 2000 x 101 x 3999 80 / 65 backward,
// 65537 x 131 x 257 55 / 67 forward (therefore without) and 186 / 129 backward, 1001 x 515 x 1027 60 / 57 backward.  Rows of a few
// elements: 165488 x 28 x 96 36 / 70 forward (therefore without) and 97 / 66 backward, 141724 x 25 -> 2 x 161 287 / 178 backward.
struct Packs { bool x, w, dz; size_t x_bytes, w_bytes; int ld_in, ld_out; };
inline Packs packs_of(const v2vae_dense* d, bool gated, bool backward) {
    Packs p = {};
    p.ld_in = (int)((d->in + 7) / 8 * 8);
    p.ld_out = (int)d->out;
    const int64_t least = backward ? 8 : 32;  // at most twice the bytes of the original
    if (d->dtype == V2VAE_F32 || d->rows <= few_rows(d->dtype) || d->in < least || d->out < least) return p;
    if ((double)d->rows * d->in * d->out * (gated ? 2 : 1) < (backward ? PACK_BACKWARD : PACK_FORWARD)) return p;
    const bool odd = d->in % 8 != 0;
    p.x = odd || d->ld_x % 8 != 0;
    p.w = odd || d->ld_w % 8 != 0 || (gated && d->ld_w2 % 8 != 0);
    p.x_bytes = p.x ? round_up((size_t)d->rows * p.ld_in * 2) : 0;
    p.w_bytes = p.w ? round_up((size_t)d->out * p.ld_in * 2) * (gated ? 2 : 1) : 0;
    if (backward) {
        p.ld_out = (int)((d->out + 7) / 8 * 8);
        p.dz = d->out % 8 != 0 || d->ld_dy % 8 != 0;  // without an activation dy itself is copied
    }
    return p;
}

// workspace of the forward pass: planes or copies, the partials of the product (few rows: partials alone)
struct FwdLayout { size_t planes, x, w, prod, total; };
inline FwdLayout fwd_layout(const v2vae_dense* d, bool gated) {
    FwdLayout l = {};
    if (d->rows <= few_rows(d->dtype)) {
        l.total = rows_bytes(d, gated);
        return l;
    }
    const Packs p = packs_of(d, gated, false);
    l.x = planes_of(d, gated, false).bytes;
    l.w = l.x + p.x_bytes;
    l.prod = l.w + p.w_bytes;
    l.total = l.prod + partial_bytes(forward_product(d, gated), d->dtype);
    return l;
}

// workspace of the backward pass: dz (two for the gated block), the column partials, planes or copies, the partials of a product
struct BwdLayout { size_t dz[2], part[2], planes, x, w, prod, total; };
inline BwdLayout bwd_layout(const v2vae_dense* d, bool gated) {
    BwdLayout l;
    const Packs p = packs_of(d, gated, true);
    const int n = gated ? 2 : 1;
    size_t o = 0;
    for (int i = 0; i < 2; ++i) {
        l.dz[i] = o;
        if (i < n && (gated || d->activation != V2VAE_ACT_NONE || p.dz)) o += round_up((size_t)d->rows * p.ld_out * elem_bytes(d->dtype));
    }
    int cx, gx, chunks;
    size_t most = 1;
    for (int64_t width : {d->out, (int64_t)p.ld_out}) {
        slope_shape(d->rows, width, &cx, &gx, &chunks);
        if ((size_t)chunks > most) most = chunks;
    }
    for (int i = 0; i < 2; ++i) {
        l.part[i] = o;
        if (i < n) o += round_up(most * d->out * 4);
    }
    l.planes = o;
    o += planes_of(d, gated, true).bytes;
    l.x = o;
    o += p.x_bytes;
    l.w = o;
    o += p.w_bytes;
    l.prod = o;
    const size_t a = partial_bytes(input_product(d, gated), d->dtype), b = partial_bytes(weight_product(d, gated), d->dtype);
    l.total = o + (a > b ? a : b);
    return l;
}

}  // namespace v2vae
#endif
