// dense_f32.hip — the f32 instances of the dense operators' tiled product.
#include "dense_gemm_impl.h"

hipError_t dense::launch_gemm_f32(int layout, int tile, const GemmArgs& a, const EpiDev& e,
                                 hipStream_t s) {
  return launch_gemm<float>(layout, tile, a, e, s);
}
