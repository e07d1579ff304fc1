// The product on 256 x 256 tiles, a in e4m3.
#include "fp8_gemm.h"

namespace svoo {

template <int C, int ACT>
static void launch(const GemmArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_tile_kernel<kFp8E4m3, C, ACT, 256>), dim3(gemm_blocks(256)), dim3(256), 0, s, g);
}

void launch_gemm_256(const GemmArgs& g, int a_type, int c, hipStream_t s) {
  if (a_type == kFp8E5m2) return launch_gemm_256_e5m2(g, c, s);
  if (c == kShare) launch<kShare, kActNone>(g, s);
  else if (c == kRowBf16) g.act == kActNone ? launch<kRowBf16, kActNone>(g, s) : launch<kRowBf16, kActGeluTanh>(g, s);
  else g.act == kActNone ? launch<kRowF16, kActNone>(g, s) : launch<kRowF16, kActGeluTanh>(g, s);
}

}  // namespace svoo
