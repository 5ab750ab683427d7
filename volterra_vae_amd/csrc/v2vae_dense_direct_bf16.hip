// Matrix product of the dense layers straight from memory to LDS, bf16 operands.
#include "v2vae_dense_direct.h"

namespace v2vae {
int gemm_direct_bf16(const GemmArgs& g, int layout, bool gated, int tile, hipStream_t st) {
    return gemm_direct<bf16_t>(g, layout, gated, tile, st);
}
}  // namespace v2vae
