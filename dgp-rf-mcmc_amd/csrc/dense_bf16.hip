// dense_bf16.hip — the bf16 instances of the dense operators' tiled product.
#include "dense_gemm_impl.h"

hipError_t dense::launch_gemm_bf16(int layout, int tile, const GemmArgs& a, const EpiDev& e,
                                 hipStream_t s) {
  return launch_gemm<bf16_t>(layout, tile, a, e, s);
}
