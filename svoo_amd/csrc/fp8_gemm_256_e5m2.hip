// The product on 256 x 256 tiles, a in e5m2 (gradients: without activation).
#include "fp8_gemm.h"

namespace svoo {

template <int C>
static void launch(const GemmArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_tile_kernel<kFp8E5m2, C, kActNone, 256>), dim3(gemm_blocks(256)), dim3(256), 0, s, g);
}

void launch_gemm_256_e5m2(const GemmArgs& g, int c, hipStream_t s) {
  if (c == kShare) launch<kShare>(g, s);
  else if (c == kRowBf16) launch<kRowBf16>(g, s);
  else launch<kRowF16>(g, s);
}

}  // namespace svoo
