// Staged matrix product of the dense layers, f16 operands.
#include "v2vae_dense_gemm.h"

namespace v2vae {
int gemm_staged_f16(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    return gemm_staged<f16_t>(g, layout, gated, tile, st);
}
}  // namespace v2vae
