// Layout of attention against a key / value cache of 8 bits (attention_q8.cu, attention_q8_tcgen05.cu).
//
//   k codes (B, G, blocks, 64, dim) int8, v codes (B, G, blocks, 64, vdim) int8, scales (B, G, blocks) fp32:
//     value = code * scale, scale = max |x| / 127 over the block, code = x / scale rounded to the nearest whole number;
//     a block that holds a number that is not finite: scale NaN, codes 0
//   tails (B, G, 64, dim | vdim): the block in progress, as it was computed
//
// A position reads its own block as it was computed and earlier blocks from the codes. For a portion of T tokens the rows of the
// blocks that it touches are laid out as `raw` (B, G, T + 64, dim | vdim): row i of a sequence is position pos / 64 * 64 + i.
#pragma once
#include "attention_window.cuh"

constexpr int Q8_BLOCK = 64;
// blocks that a portion of T tokens can touch, wherever it begins
__host__ __device__ constexpr int q8_touched(int T) { return (T + 2 * Q8_BLOCK - 2) / Q8_BLOCK; }

// Where the codes of a block are held as 16-bit numbers while a portion from position `pos` on is worked on: those of the kept first tokens,
// then those from the first block that a window of the portion reaches, side by side. Blocks in between are not held.
struct Q8Slots {
  int kept, from;
  __device__ __forceinline__ int of(int blk) const { return blk < kept ? blk : kept + blk - from; }
};
__device__ __forceinline__ Q8Slots q8_slots(int pos, int window, int keep_first) {
  if (!window) return {0, 0};
  const int kept = (int)(((long long)keep_first + Q8_BLOCK - 1) / Q8_BLOCK);
  return {kept, max(kept, max(0, pos - window + 1) / Q8_BLOCK)};
}
// How many there are at most, for a portion of T tokens: its last complete block is less than (T + window - 1) / 64 + 1 behind `from`.
inline long long q8_held(int T, int blocks, int window, int keep_first) {
  const long long n = ((long long)keep_first + Q8_BLOCK - 1) / Q8_BLOCK + ((long long)T + window - 1) / Q8_BLOCK + 1;
  return window && n < blocks ? n : blocks;
}

// A power of two above every factor of a norm: normalised rows divided by it are at most sqrt(features) and fit 16-bit floats. `top`: the
// largest absolute factor that the lane has seen; the result is that of the warp.
__device__ __forceinline__ float q8_norm_unit(float top) {
  const uint32_t e = __reduce_max_sync(0xffffffffu, __float_as_uint(top)) >> 23;  // floats above zero are ordered like their bits
  return e > 0 && e < 250 ? __uint_as_float((e + 1) << 23) : 1.f;
}
__device__ __forceinline__ float q8_norm_unit(const float* w, int dim, int lane) {
  float top = 0.f;
  for (int d = lane; d < dim; d += 32) top = fmaxf(top, fabsf(w[d]));
  return q8_norm_unit(top);
}

// The larger of two numbers, NaN where either is one (fmaxf drops a NaN); of a warp; and the scale of a block from its largest absolute value.
__device__ __forceinline__ float q8_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float q8_warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = q8_max(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float q8_scale_of(float top) { return top < INFINITY ? __fdiv_rn(top, 127.f) : __uint_as_float(0x7fc00000u); }
// Whether positions that read a block of such scales (of its keys, of its values) become NaN
__device__ __forceinline__ bool q8_spoiled(float k_scale, float v_scale) { return !(k_scale + v_scale < INFINITY); }

// Codes of a block: x / scale rounded to the nearest whole number. A product with the reciprocal is off by less than 2^-15 (three roundings of
// numbers below 128), so
// only next to the middle between two codes does it take the division to know. Added to 1.5 * 2^23, a number of at most 127 leaves its
// nearest whole number in the low bits of the sum. A scale that is NaN makes every code zero.
struct Q8Step {
  float scale, inv;
  __device__ __forceinline__ explicit Q8Step(float s) : scale(s), inv(s > 1e-30f ? 1.f / s : 0.f) {}
  __device__ __forceinline__ int exact(float x) const {
    return scale > 0.f ? max(-127, min(127, __float2int_rn(__fdiv_rn(x, scale)))) : 0;
  }
  // N codes, four to a word
  template <int N> __device__ __forceinline__ void codes(const float (&x)[N], uint32_t (&w)[(N + 3) / 4]) const {
    float far = inv == 0.f ? 1.f : 0.f;
    uint32_t c[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float y = x[e] * inv, r = __fadd_rn(y, 12582912.f);
      far = fmaxf(far, fabsf(y - __fsub_rn(r, 12582912.f)));
      c[e] = __float_as_uint(r) & 0xffu;
    }
    if (!(far < 0.49996f)) {
#pragma unroll
      for (int e = 0; e < N; ++e) c[e] = (uint32_t)exact(x[e]) & 0xffu;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) w[e >> 2] = (e & 3 ? w[e >> 2] : 0u) | c[e] << (8 * (e & 3));
  }
};
