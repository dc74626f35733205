// Layout of attention against a key / value cache of 8 bits (attention_q8.cu, attention_q8_tcgen05.cu).
//
//   k codes (B, G, blocks, 64, dim) int8, v codes (B, G, blocks, 64, vdim) int8, scales (B, G, blocks) fp32:
//     value = code * scale, scale = max |x| / 127 over the block, code = x / scale rounded to the nearest whole number
//   tails (B, G, 64, dim | vdim): the block in progress, as it was computed
//
// A position reads its own block as it was computed and earlier blocks from the codes. For a portion of T tokens the rows of the
// blocks that it touches are laid out as `raw` (B, G, T + 64, dim | vdim): row i of a sequence is position pos / 64 * 64 + i.
#pragma once
#include "attention_window.cuh"

constexpr int Q8_BLOCK = 64;

// exponent e with 2^e above every factor, so that normalised rows divided by 2^e are at most sqrt(features) and fit 16-bit floats
__device__ __forceinline__ float q8_norm_unit(const float* w, int dim, int lane) {
  float top = 0.f;
  for (int d = lane; d < dim; d += 32) top = fmaxf(top, fabsf(w[d]));
  top = xl_warp_max(top);
  return top > 0.f && top < 1e30f ? exp2f((float)(ilogbf(top) + 1)) : 1.f;
}

__device__ __forceinline__ int q8_code(float x, float scale) {
  return scale > 0.f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale)))) : 0;
}
