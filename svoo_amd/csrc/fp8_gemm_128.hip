// The product on 128 x 128 tiles: every type of a and c.
#include "fp8_gemm.h"

namespace svoo {

template <int A, int C>
static void launch(const GemmArgs& g, hipStream_t s) {
  hipLaunchKernelGGL((fp8_gemm_tile_kernel<A, C, kActAny, 128>), dim3(gemm_blocks(128)), dim3(256), 0, s, g);
}

template <int A>
static void launch_a(const GemmArgs& g, int c, hipStream_t s) {
  if (c == kShare) launch<A, kShare>(g, s);
  else if (c == kShareWide) launch<A, kShareWide>(g, s);
  else if (c == kRowBf16) launch<A, kRowBf16>(g, s);
  else if (c == kRowF16) launch<A, kRowF16>(g, s);
  else launch<A, kRowF32>(g, s);
}

void launch_gemm_128(const GemmArgs& g, int a_type, int c, hipStream_t s) {
  if (a_type == kFp8E4m3) launch_a<kFp8E4m3>(g, c, s);
  else launch_a<kFp8E5m2>(g, c, s);
}

}  // namespace svoo
