// dense_f16.hip — the f16 instances of the dense operators' tiled product.
#include "dense_gemm_impl.h"

hipError_t dense::launch_gemm_f16(int layout, int tile, const GemmArgs& a, const EpiDev& e,
                                 hipStream_t s) {
  return launch_gemm<f16_t>(layout, tile, a, e, s);
}
