// The scales of MXFP4 blocks: what the quantization (sage_mxfp4.hip) and the norms that
// quantize their output (sage_norm.hip) share.
#pragma once
#include <type_traits>

#include "sage_common.h"

namespace sage {

namespace {

// The scale 2^(e - 127) as a float (0: the subnormal 2^-127).
__device__ __forceinline__ float scale_of(int e) { return __int_as_float(e ? e << 23 : 0x00400000); }

// The largest of the four lanes' values of a block (lanes 4 i .. + 3), in all of them.
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  v = max(v, dpp(v, std::integral_constant<int, 0xb1>{}));     // quad_perm [1,0,3,2]
  return max(v, dpp(v, std::integral_constant<int, 0x4e>{}));  // quad_perm [2,3,0,1]
}

// The biased exponent of a block's scale from the bits of its largest magnitude as fp32.
__device__ __forceinline__ int block_exponent(uint32_t bits) {
  const int e = (int)(bits >> 23);
  return e == 255 ? 255 : max(e - 2, 0);
}

}  // namespace

}  // namespace sage
