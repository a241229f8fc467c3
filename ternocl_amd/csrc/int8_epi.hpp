// int8_epi.hpp -- what the engines of ternocl_int8_gemm do to a sum of products.
#pragma once

#include "common.hpp"

namespace tcl {
namespace {

// The whole sum (exact in 32 bits: K below 2^17), rounded to fp32 where it passes 2^24,
// times the channel's scale, then the token's: a token's scale may be as large as its
// activations (2^120 at bf16), and the channel's has brought the sum down before it.
__device__ __forceinline__ float i8_scaled(int acc, float sb, float sa) { return ((float)acc * sb) * sa; }

}  // namespace
}  // namespace tcl
