// Staged matrix product of the dense layers, bf16 operands.
#include "v2vae_dense_gemm.h"

namespace v2vae {
int gemm_staged_bf16(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    return gemm_staged<bf16_t>(g, layout, gated, tile, st);
}
}  // namespace v2vae
