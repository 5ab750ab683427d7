// Matrix product of the dense layers, float32 operands.
#include "v2vae_dense_split.h"

namespace v2vae {

int split_planes(const GemmArgs& g, bool transposed, bool gated, int N, int K, hipStream_t st) {
    PlaneArgs a = {};
    for (int i = 0; i < 2; ++i) {
        a.w[i] = (const float*)g.b[i];
        a.ld_w[i] = g.ldb[i];
    }
    a.out = (char*)g.planes;
    a.plane_bytes = g.plane_bytes;
    a.rows = g.plane_rows;
    a.ld = g.plane_ld;
    a.N = N;
    a.K = K;
    a.gated = gated;
    if (transposed) hipLaunchKernelGGL(k_split_planes<true>, dim3((unsigned)(a.ld / 32) * ((a.rows + 63) / 64)), dim3(256), 0, st, a);
    else hipLaunchKernelGGL(k_split_planes<false>, dim3((unsigned)((a.ld + 127) / 128) * ((a.rows + 15) / 16)), dim3(256), 0, st, a);
    return dense_launch_error("dense layer, weights");
}

int gemm_split(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    if (g.planes) {
        if (gated) pick_split<true, B_PLANES, true>(g, tile, st); else pick_split<true, B_PLANES, false>(g, tile, st);
    } else if (gated) {
        pick_split<true, B_ROWS, true>(g, tile, st);
    } else if (layout == LAYOUT_KK) {
        pick_split<true, B_ROWS, false>(g, tile, st);
    } else if (layout == LAYOUT_KM) {
        pick_split<true, B_COLUMNS, false>(g, tile, st);
    } else {
        pick_split<false, B_COLUMNS, false>(g, tile, st);
    }
    return dense_launch_error("dense matrix product");
}

}  // namespace v2vae
