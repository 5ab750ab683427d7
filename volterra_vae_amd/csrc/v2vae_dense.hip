// Dense layers behind the C ABI: argument checks, workspace, choice of product kernel, and the elementwise half of the backward.
#include <math.h>

#include "v2vae_dense.h"

namespace v2vae {

// ---- dz = dy act'(z) and its column sums -------------------------------------------------------------------------------------
// One pass over dy and the float pre-activations; memory bound.  A block owns a strip of columns and every so many rows (a chunk): all
// blocks move through memory together (65536 x 256 float 37 us, 43 with rows that follow one another; gated 173475 x 1320 1180 and
// 1300).  It sums its columns in float in a fixed order (per thread along the rows, then over the block's row threads) and leaves one
// partial per chunk; k_column_join adds the chunks (4 ... 5 us).  dz is rounded to T here, once, after its contribution to the column
// sum.  Float 65536 x 256: 5.5 TB/s; bf16 gated 4096 x 5632: 61 us (5.3 TB/s).
struct SlopeArgs {
    const void* dy;
    int64_t ld_dy;
    const float* z[2];  // pre-activations [M][N] (NULL: no activation), gated: gate and up
    void* d[2];         // dz [M][ld_d], zeros in columns N ... ld_d - 1 (NULL: only the sums)
    int64_t ld_d;
    float* part[2];     // [chunks][N] (NULL: no sums)
    int64_t M;
    int N, cx;          // cx threads along the columns, four each, 256 / cx along the rows
};

template <typename T, int ACT, bool GATED> __global__ __launch_bounds__(256) void k_dense_slopes(SlopeArgs a) {
    constexpr int V = 4;  // columns a thread
    __shared__ float s_sum[GATED ? 2 : 1][256 * V];
    const int tid = threadIdx.x, cx = a.cx, ry = 256 / cx, tx = tid % cx, ty = tid / cx;
    const int64_t n = ((int64_t)blockIdx.x * cx + tx) * V;
    float s0[V], s1[V];
#pragma unroll
    for (int v = 0; v < V; ++v) s0[v] = s1[v] = 0.f;
    // The last columns, fewer than V, are taken together with the ones before them, which their own thread has as well (and writes the
    // same): a wave goes through its rows once, without a branch.  Not WHOLE: fewer than V columns in all.
    const int beyond = n < a.N && n + V > a.N && a.N >= V ? (int)(n + V - a.N) : 0;
    auto rows = [&](auto all) {
        constexpr bool WHOLE = decltype(all)::value;
        const int64_t n1 = n - beyond;
        const int count = (int)(a.N - n1);
#pragma unroll 2
        for (int64_t m = (int64_t)blockIdx.y * ry + ty; m < a.M; m += (int64_t)gridDim.y * ry) {
            float dy[V], z0[V], z1[V];
            load_columns<T, V>(a.dy, m * a.ld_dy + n1, count, WHOLE, dy);
            if (a.z[0]) load_columns<float, V>(a.z[0], m * a.N + n1, count, WHOLE, z0);
            if constexpr (GATED) load_columns<float, V>(a.z[1], m * a.N + n1, count, WHOLE, z1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float val;
                if constexpr (GATED) {
                    const float slope = act_slope(ACT, z0[v], &val), d = dy[v];
                    dy[v] = d * z1[v] * slope;
                    z1[v] = d * val;
                    s1[v] += z1[v];
                } else {
                    if (a.z[0]) dy[v] *= act_slope(ACT, z0[v], &val);
                }
                s0[v] += dy[v];
            }
            if (a.d[0]) store_columns<T, V>(a.d[0], m * a.ld_d + n1, count, WHOLE, dy);
            if constexpr (GATED)
                if (a.d[1]) store_columns<T, V>(a.d[1], m * a.ld_d + n1, count, WHOLE, z1);
        }
    };
    if (n < a.N) {
        if (a.N >= V) rows(std::true_type()); else rows(std::false_type());
    }
    if (a.d[0] && n + V > a.N && n < a.ld_d) {  // zeros in the columns that dz is padded with
        for (int64_t m = (int64_t)blockIdx.y * ry + ty; m < a.M; m += (int64_t)gridDim.y * ry)
            for (int64_t i = n > a.N ? n : a.N; i < n + V && i < a.ld_d; ++i) {
                ((T*)a.d[0])[m * a.ld_d + i] = (T)0.f;
                if constexpr (GATED) ((T*)a.d[1])[m * a.ld_d + i] = (T)0.f;
            }
    }
    for (int q = 0; q < beyond; ++q) {  // this thread's own columns to the front
#pragma unroll
        for (int v = 0; v + 1 < V; ++v) {
            s0[v] = s0[v + 1];
            s1[v] = s1[v + 1];
        }
    }
    if (a.part[0] == nullptr) return;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        s_sum[0][tid * V + v] = s0[v];
        if constexpr (GATED) s_sum[1][tid * V + v] = s1[v];
    }
    __syncthreads();
    for (int i = tid; i < cx * V; i += 256) {
        const int64_t col = (int64_t)blockIdx.x * cx * V + i;
        if (col >= a.N) continue;
#pragma unroll
        for (int q = 0; q < (GATED ? 2 : 1); ++q) {
            float s = 0.f;
            for (int y = 0; y < ry; ++y) s += s_sum[q][y * cx * V + i];
            a.part[q][(int64_t)blockIdx.y * a.N + col] = s;
        }
    }
}

// out[n] = sum of the chunks' partials, in a fixed order; 32 columns x 32 lanes a block
template <typename T> __global__ __launch_bounds__(1024) void k_column_join(const float* part0, const float* part1, void* out0, void* out1,
                                                                           int chunks, int N) {
    __shared__ float s_sum[32][33];
    const float* part = blockIdx.y ? part1 : part0;
    T* out = (T*)(blockIdx.y ? out1 : out0);
    const int c = threadIdx.x & 31, y = threadIdx.x >> 5, n = blockIdx.x * 32 + c;
    float s = 0.f;
    if (out && n < N)
#pragma unroll 4
        for (int i = y; i < chunks; i += 32) s += part[(int64_t)i * N + n];
    s_sum[y][c] = s;
    __syncthreads();
    if (y == 0 && out && n < N) {
        float t = 0.f;
        for (int i = 0; i < 32; ++i) t += s_sum[i][c];
        out[n] = (T)t;
    }
}

// ---- rows of whole 16-byte pieces --------------------------------------------------------------------------------------------
// 16-bit matrices whose rows are not: copied once, padded with zeros, for the product kernel that loads tiles straight into LDS.
// One pass over the operand, eight columns a thread (the loads may be unaligned, the stores are not); bound by bytes: 9416 x 3231 18 us
// (6.6 TB/s, part of it in the last-level cache).
struct PackArgs { const void* src[2]; void* dst[2]; int64_t ld_src[2], R; int C, ld; };
__global__ __launch_bounds__(256) void k_pack_rows(PackArgs a) {
    struct __attribute__((packed, aligned(2))) Loose { u32x4 raw; };
    const int per = a.ld / 8, which = blockIdx.y;
    const uint16_t* const src = (const uint16_t*)a.src[which];
    uint16_t* const dst = (uint16_t*)a.dst[which];
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.R * per; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per;
        const int c = (int)(i - r * per) * 8;
        const uint16_t* const p = src + r * a.ld_src[which] + c;
        union { u32x4 raw; uint16_t e[8]; } v;
        if (c + 8 <= a.C) {
            v.raw = reinterpret_cast<const Loose*>(p)->raw;
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v.e[e] = c + e < a.C ? p[e] : (uint16_t)0;
        }
        *reinterpret_cast<u32x4*>(dst + r * a.ld + c) = v.raw;
    }
}

// ---- host side ---------------------------------------------------------------------------------------------------------------
static bool aligned_to(const void* p, int n) { return ((uintptr_t)p % n) == 0; }
static void pack_rows(const void* s0, const void* s1, int64_t ld0, int64_t ld1, void* d0, void* d1, int64_t R, int C, int ld, hipStream_t st) {
    PackArgs a = {{s0, s1}, {d0, d1}, {ld0, ld1}, R, C, ld};
    int64_t blocks = (R * (ld / 8) + 255) / 256;
    if (blocks > 8192) blocks = 8192;
    if (blocks > 0) hipLaunchKernelGGL(k_pack_rows, dim3((unsigned)blocks, s1 ? 2 : 1), dim3(256), 0, st, a);
}

// g as `p` describes it, of whose batch entries g.batch are formed; `room` bytes at `partial`
static int run_product(GemmArgs& g, const Product& p, int dtype, int layout, bool gated, float* partial, size_t room, hipStream_t st) {
    if (g.M == 0 || g.N == 0) return V2VAE_OK;
    const int e = 16 / elem_bytes(dtype);
    auto aligned_rows = [&](const void* const p[2], int64_t ld0, int64_t ld1) {
        return aligned_to(p[0], 16) && (p[1] == nullptr || aligned_to(p[1], 16)) && ld0 % e == 0 && ld1 % e == 0;
    };
    const bool a_kc = layout != LAYOUT_MM, b_kc = layout == LAYOUT_KK;
    // every row whole 16-byte pieces, in memory and in the part of it that counts (or zeros behind that)
    const bool whole_a = aligned_rows(g.a, g.lda, g.lda) && (g.pad_a || (a_kc ? g.K : g.M) % e == 0);
    const bool whole_b = aligned_rows(g.b, g.ldb[0], g.ldb[1]) && (g.pad_b || (b_kc ? g.K : g.N) % e == 0);
    // straight to LDS: 16-bit, whole pieces, offsets inside a tile below 2^31, one stride
    const int64_t ld_max = g.lda > g.ldb[0] ? (g.lda > g.ldb[1] ? g.lda : g.ldb[1]) : (g.ldb[0] > g.ldb[1] ? g.ldb[0] : g.ldb[1]);
    const bool direct = dtype != V2VAE_F32 && whole_a && whole_b && ld_max <= (1 << 21) && (gated || g.ldb[0] == g.ldb[1]);
    const Cut c = cut_product(p, dtype, direct);
    if (cut_bytes(p, c, g.batch) > room) return V2VAE_ESIZE;  // the layout of the workspace has room for every cut
    g.splits = c.splits;
    g.steps_per_split = c.per;
    g.partial = c.splits > 1 ? partial : nullptr;
    if (direct) return dtype == V2VAE_BF16 ? gemm_direct_bf16(g, layout, gated, c.tile, st) : gemm_direct_f16(g, layout, gated, c.tile, st);
    if (dtype == V2VAE_F32) return gemm_split(g, layout, gated, c.tile, st);
    if (dtype == V2VAE_BF16) return gemm_staged_bf16(g, layout, gated, c.tile, st);
    return gemm_staged_f16(g, layout, gated, c.tile, st);
}

static int use_planes(GemmArgs& g, const Planes& p, bool transposed, bool gated, char* at, hipStream_t st) {
    g.planes = at;
    g.plane_bytes = (int64_t)p.plane;
    g.plane_rows = p.rows;
    g.plane_ld = p.ld;
    return split_planes(g, transposed, gated, transposed ? g.K : g.N, transposed ? g.N : g.K, st);
}

static int forward(const v2vae_dense* d, const void* x, const void* w0, const void* w1, const void* b0, const void* b1,
                   const void* res, void* y, float* z, void* ws, hipStream_t st) {
    const bool gated = w1 != nullptr;
    GemmArgs g = {};
    g.a[0] = x;
    g.b[0] = w0;
    g.b[1] = w1;
    g.c[0] = y;
    g.lda = d->ld_x;
    g.ldb[0] = d->ld_w;
    g.ldb[1] = gated ? d->ld_w2 : d->ld_w;
    g.ldc = d->out;
    g.M = (int)d->rows;
    g.N = (int)d->out;
    g.K = (int)d->in;
    g.segs = g.batch = g.splits = 1;
    g.bias[0] = b0;
    g.bias[1] = b1;
    g.residual = res;
    g.ldr = d->ld_res;
    g.z[0] = z;
    g.z[1] = z ? z + (int64_t)d->rows * d->out : nullptr;
    g.act = d->activation;
    const FwdLayout l = fwd_layout(d, gated);
    char* const base = (char*)ws;
    const Planes p = planes_of(d, gated, false);
    if (p.bytes) {
        const int rc = use_planes(g, p, false, gated, base + l.planes, st);
        if (rc != V2VAE_OK) return rc;
    }
    if (d->rows <= few_rows(d->dtype)) {
        g.splits = rows_splits(d->dtype, d->in, d->out, gated);
        g.partial = g.splits > 1 ? (float*)ws : nullptr;
        return dense_rows(g, d->dtype, gated, st);
    }
    const Packs k = packs_of(d, gated, false);
    if (k.x) {
        pack_rows(x, nullptr, d->ld_x, 0, base + l.x, nullptr, d->rows, g.K, k.ld_in, st);
        g.a[0] = base + l.x;
        g.lda = k.ld_in;
        g.pad_a = 1;
    }
    if (k.w) {
        char* const up = gated ? base + l.w + k.w_bytes / 2 : nullptr;
        pack_rows(w0, w1, d->ld_w, d->ld_w2, base + l.w, up, d->out, g.K, k.ld_in, st);
        g.b[0] = base + l.w;
        g.b[1] = up;
        g.ldb[0] = g.ldb[1] = k.ld_in;
        g.pad_b = 1;
    }
    return run_product(g, forward_product(d, gated), d->dtype, LAYOUT_KK, gated, (float*)(base + l.prod), l.total - l.prod, st);
}

static int backward(const v2vae_dense* d, const void* x, const void* w0, const void* w1, const float* z, const void* dy, void* dx,
                    void* dw0, void* dw1, void* db0, void* db1, void* ws, hipStream_t st) {
    const Packs k = packs_of(d, w1 != nullptr, true);
    const bool gated = w1 != nullptr, act = gated || d->activation != V2VAE_ACT_NONE, copy = act || k.dz;
    const BwdLayout l = bwd_layout(d, gated);
    char* const base = (char*)ws;
    const int64_t M = d->rows;
    const void* dz[2] = {dy, nullptr};
    int64_t ld_dz = d->ld_dy;
    const bool want_b = db0 || db1, want_dz = dx || dw0 || dw1;
    if ((copy && want_dz) || want_b) {
        SlopeArgs s = {};
        s.dy = dy;
        s.ld_dy = d->ld_dy;
        s.M = M;
        s.N = (int)d->out;
        s.z[0] = act ? z : nullptr;
        s.z[1] = gated ? z + M * d->out : nullptr;
        s.ld_d = d->out;
        if (copy && want_dz) {
            s.ld_d = k.ld_out;
            s.d[0] = base + l.dz[0];
            s.d[1] = gated ? base + l.dz[1] : nullptr;
            dz[0] = s.d[0];
            dz[1] = s.d[1];
            ld_dz = k.ld_out;
        }
        if (want_b) {
            s.part[0] = (float*)(base + l.part[0]);
            s.part[1] = gated ? (float*)(base + l.part[1]) : nullptr;
        }
        int gx, chunks;
        slope_shape(M, s.ld_d, &s.cx, &gx, &chunks);
        const dim3 grid(gx, chunks);
        auto slopes = [&](auto t, auto kind) {
            typedef decltype(t) T;
            constexpr int ACT = decltype(kind)::value;
            if (gated) hipLaunchKernelGGL((k_dense_slopes<T, ACT, true>), grid, dim3(256), 0, st, s);
            else hipLaunchKernelGGL((k_dense_slopes<T, ACT, false>), grid, dim3(256), 0, st, s);
        };
        auto go = [&](auto t) {
            typedef decltype(t) T;
            switch (d->activation) {
                case V2VAE_ACT_RELU: slopes(t, std::integral_constant<int, V2VAE_ACT_RELU>()); break;
                case V2VAE_ACT_SILU: slopes(t, std::integral_constant<int, V2VAE_ACT_SILU>()); break;
                case V2VAE_ACT_GELU: slopes(t, std::integral_constant<int, V2VAE_ACT_GELU>()); break;
                case V2VAE_ACT_TANH: slopes(t, std::integral_constant<int, V2VAE_ACT_TANH>()); break;
                default: slopes(t, std::integral_constant<int, V2VAE_ACT_NONE>()); break;
            }
            if (want_b)
                hipLaunchKernelGGL((k_column_join<T>), dim3((unsigned)((d->out + 31) / 32), gated ? 2 : 1), dim3(1024), 0, st, s.part[0],
                                   s.part[1], db0, db1, chunks, (int)d->out);
        };
        if (d->dtype == V2VAE_F32) go(float());
        else if (d->dtype == V2VAE_BF16) go(bf16_t());
        else go(f16_t());
        const int rc = dense_launch_error("dense layer, backward");
        if (rc != V2VAE_OK) return rc;
    }
    float* const prod = (float*)(base + l.prod);
    const size_t room = l.total - l.prod;
    const bool padded = k.dz;
    if (dx && k.w && M > 0) {
        char* const up = gated ? base + l.w + k.w_bytes / 2 : nullptr;
        pack_rows(w0, w1, d->ld_w, d->ld_w2, base + l.w, up, d->out, (int)d->in, k.ld_in, st);
    }
    if ((dw0 || dw1) && k.x) pack_rows(x, nullptr, d->ld_x, 0, base + l.x, nullptr, M, (int)d->in, k.ld_in, st);
    if (dx) {
        GemmArgs g = {};
        g.a[0] = dz[0];
        g.a[1] = dz[1];
        g.b[0] = w0;
        g.b[1] = w1;
        g.c[0] = dx;
        g.lda = ld_dz;
        g.ldb[0] = d->ld_w;
        g.ldb[1] = gated ? d->ld_w2 : d->ld_w;
        g.pad_a = padded;
        if (k.w) {
            g.b[0] = base + l.w;
            g.b[1] = gated ? base + l.w + k.w_bytes / 2 : nullptr;
            g.ldb[0] = g.ldb[1] = k.ld_in;
            g.pad_b = 1;
        }
        g.ldc = d->in;
        g.M = (int)M;
        g.N = (int)d->in;
        g.K = (int)d->out;
        g.segs = gated ? 2 : 1;
        g.batch = 1;
        const Planes p = planes_of(d, gated, true);
        if (p.bytes && M > 0) {
            const int rc = use_planes(g, p, true, gated, base + l.planes, st);
            if (rc != V2VAE_OK) return rc;
        }
        const int rc = run_product(g, input_product(d, gated), d->dtype, LAYOUT_KM, false, prod, room, st);
        if (rc != V2VAE_OK) return rc;
    }
    if (dw0 || dw1) {
        GemmArgs g = {};
        g.a[0] = dw0 ? dz[0] : dz[1];
        g.a[1] = dz[1];
        g.b[0] = g.b[1] = x;
        g.c[0] = dw0 ? dw0 : dw1;
        g.c[1] = dw1;
        g.lda = ld_dz;
        g.ldb[0] = g.ldb[1] = d->ld_x;
        g.pad_a = padded;
        if (k.x) {
            g.b[0] = g.b[1] = base + l.x;
            g.ldb[0] = g.ldb[1] = k.ld_in;
            g.pad_b = 1;
        }
        g.ldc = d->in;
        g.M = (int)d->out;
        g.N = (int)d->in;
        g.K = (int)M;
        g.segs = 1;
        g.batch = dw0 && dw1 ? 2 : 1;
        return run_product(g, weight_product(d, gated), d->dtype, LAYOUT_MM, false, prod, room, st);
    }
    return V2VAE_OK;
}

}  // namespace v2vae

using namespace v2vae;

extern "C" {

size_t v2vae_linear_workspace_bytes(const v2vae_dense* d, int backward) {
    if (check_dense(d, false, backward != 0, false) != V2VAE_OK) return 0;
    return backward ? bwd_layout(d, false).total : fwd_layout(d, false).total;
}

size_t v2vae_gated_workspace_bytes(const v2vae_dense* d, int backward) {
    if (check_dense(d, true, backward != 0, false) != V2VAE_OK) return 0;
    return backward ? bwd_layout(d, true).total : fwd_layout(d, true).total;
}

int v2vae_linear_fwd(const v2vae_dense* d, const void* x, const void* w, const void* bias, const void* residual, void* y, float* z,
                     void* ws, void* stream) {
    const int rc = check_dense(d, false, false, residual != nullptr);
    if (rc != V2VAE_OK) return rc;
    if (d->rows == 0) return V2VAE_OK;
    const int b = elem_bytes(d->dtype);
    if (!x || !w || !y || !aligned_to(x, b) || !aligned_to(w, b) || !aligned_to(y, b) || !aligned_to(z, 4) || !aligned_to(ws, 256) ||
        !aligned_to(bias, b) || !aligned_to(residual, b))
        return V2VAE_EINVAL;
    if (!ws && v2vae_linear_workspace_bytes(d, 0) > 0) return V2VAE_EINVAL;
    return forward(d, x, w, nullptr, bias, nullptr, residual, y, z, ws, (hipStream_t)stream);
}

int v2vae_linear_bwd(const v2vae_dense* d, const void* x, const void* w, const float* z, const void* dy, void* dx, void* dw,
                     void* dbias, void* ws, void* stream) {
    const int rc = check_dense(d, false, true, false);
    if (rc != V2VAE_OK) return rc;
    const int b = elem_bytes(d->dtype);
    if (d->rows > 0 && (!dy || (dw && !x) || (dx && !w) || (d->activation != V2VAE_ACT_NONE && !z))) return V2VAE_EINVAL;
    if (!aligned_to(x, b) || !aligned_to(w, b) || !aligned_to(z, 4) || !aligned_to(dy, b) || !aligned_to(dx, b) || !aligned_to(dw, b) ||
        !aligned_to(dbias, b) || !aligned_to(ws, 256) || !ws)
        return V2VAE_EINVAL;
    return backward(d, x, w, nullptr, z, dy, dx, dw, nullptr, dbias, nullptr, ws, (hipStream_t)stream);
}

int v2vae_gated_fwd(const v2vae_dense* d, const void* x, const void* wg, const void* wu, const void* bg, const void* bu, void* h,
                    float* gu, void* ws, void* stream) {
    const int rc = check_dense(d, true, false, false);
    if (rc != V2VAE_OK) return rc;
    if (d->rows == 0) return V2VAE_OK;
    const int b = elem_bytes(d->dtype);
    if (!x || !wg || !wu || !h || !aligned_to(x, b) || !aligned_to(wg, b) || !aligned_to(wu, b) || !aligned_to(h, b) ||
        !aligned_to(gu, 4) || !aligned_to(ws, 256) || !aligned_to(bg, b) || !aligned_to(bu, b))
        return V2VAE_EINVAL;
    if (!ws && v2vae_gated_workspace_bytes(d, 0) > 0) return V2VAE_EINVAL;
    return forward(d, x, wg, wu, bg, bu, nullptr, h, gu, ws, (hipStream_t)stream);
}

int v2vae_gated_bwd(const v2vae_dense* d, const void* x, const void* wg, const void* wu, const float* gu, const void* dh, void* dx,
                    void* dwg, void* dwu, void* dbg, void* dbu, void* ws, void* stream) {
    const int rc = check_dense(d, true, true, false);
    if (rc != V2VAE_OK) return rc;
    const int b = elem_bytes(d->dtype);
    if (!wg || !wu || !ws || (d->rows > 0 && (!dh || !gu || ((dwg || dwu) && !x)))) return V2VAE_EINVAL;
    if (!aligned_to(x, b) || !aligned_to(wg, b) || !aligned_to(wu, b) || !aligned_to(gu, 4) || !aligned_to(dh, b) || !aligned_to(dx, b) ||
        !aligned_to(dwg, b) || !aligned_to(dwu, b) || !aligned_to(dbg, b) || !aligned_to(dbu, b) || !aligned_to(ws, 256))
        return V2VAE_EINVAL;
    return backward(d, x, wg, wu, gu, dh, dx, dwg, dwu, dbg, dbu, ws, (hipStream_t)stream);
}

}  // extern "C"
