// Sliding-window attention against a key / value cache of 8 bits: normalised queries and keys, kept first tokens, a sink, a gate
// (the mathematics of attention_window.cu; layouts in attention_q8.cuh). Keys are normalised in 64 bits and rounded once to the
// model's type, so that every kernel and every division into portions comes to the same codes. Queries are not rounded to it.
//
//   xl_q8_append          queries to their buffer, keys and values to `raw`; complete blocks to codes, the rest to the tails
//   xl_q8_attn_general    any sizes and types, scores and weights in fp32 on the CUDA cores: one warp per row and head
//   xl_q8_append_expand   the same, laid out for the tensor cores (xl_q8_attn_tcgen05 in attention_q8_tcgen05.cu)
//   xl_q8_attn_few        few rows per sequence, bf16, on mma.sync; of a single token norms, append and codes in the same launch
#include "attention_decode.cuh"
#include "attention_q8.cuh"
#include "tcgen05.cuh"

#include <math.h>

#include <type_traits>

namespace {

constexpr int Q8_MAX_DIM = 512;

struct Q8AppendParams {
  const void* proj;
  long long ld;
  const float *wq, *wk;
  void* q;          // (B, G, T, H/G, dim) fp32
  void *raw_k, *raw_v;
  int8_t *kc, *vc;
  float *ks, *vs;
  void *kt, *vt;
  const int *pos, *count;
  int T, H, G, dim, vdim, blocks;
  double eps;
};

template <typename T, int V> struct alignas(V * sizeof(T)) Q8Piece { T v[V]; };

// Grid (blocks a portion can touch, G, B): a CTA has the rows of one block of one key / value head; a warp takes a row's heads in
// turn: the query heads of the group, the key, the value. Accesses of V elements.
// The tail is read by the CTA of the portion's first block (its earlier tokens) and written once that has been done, by the same
// CTA: the rows of the last block, if that is another one, are computed again there, which gives the same bits.
template <typename T, int V>
__global__ void __launch_bounds__(256) q8_append_kernel(const Q8AppendParams p) {
  constexpr int NP = Q8_MAX_DIM / (32 * V);
  constexpr int WARPS = 8;
  __shared__ float tops[2][WARPS];
  __shared__ float scales[2];
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int blk = blockIdx.x, g = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int pos = p.pos[b], n = min(p.count[b], p.T), R = p.H / p.G;
  if (n <= 0 || pos < 0 || (long long)pos + n > (long long)p.blocks * Q8_BLOCK) return;
  const int fill = pos % Q8_BLOCK, end = fill + n;  // rows of the block in progress, rows after the portion
  const int r0 = blk * Q8_BLOCK, r1 = min(r0 + Q8_BLOCK, end);
  if (r0 >= end) return;
  const long long head = (long long)b * p.G + g;
  const T* proj = (const T*)p.proj + (long long)b * p.T * p.ld;
  T* raw[2] = {(T*)p.raw_k + head * (p.T + Q8_BLOCK) * p.dim, (T*)p.raw_v + head * (p.T + Q8_BLOCK) * p.vdim};
  T* tail[2] = {(T*)p.kt + head * Q8_BLOCK * p.dim, (T*)p.vt + head * Q8_BLOCK * p.vdim};
  const int width[2] = {p.dim, p.vdim};
  auto load = [&](const T* src, int w, float (&x)[NP][V]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (lane + 32 * i) * V;
      if (c < w) {
        const Q8Piece<T, V> piece = *reinterpret_cast<const Q8Piece<T, V>*>(src + c);
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = xl_to_float(piece.v[e]);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = 0.f;
      }
    }
  };
  auto store = [&](T* dst, int w, const float (&x)[NP][V]) {  // the values have the precision of T
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (lane + 32 * i) * V;
      if (c < w) {
        Q8Piece<T, V> piece;
#pragma unroll
        for (int e = 0; e < V; ++e) piece.v[e] = xl_from_float<T>(x[i][e]);
        *reinterpret_cast<Q8Piece<T, V>*>(dst + c) = piece;
      }
    }
  };
  // key (kind 0) or value (1) of a new token, rounded to T
  auto fresh = [&](int kind, int t, float (&x)[NP][V]) {
    const T* row = proj + (long long)t * p.ld;
    if (kind) {
      load(row + (long long)(p.H + p.G) * p.dim + (long long)g * p.vdim, p.vdim, x);
      return;
    }
    load(row + (long long)(p.H + g) * p.dim, p.dim, x);
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += (double)x[i][e] * (double)x[i][e];
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const double f = 1.0 / sqrt(sum / p.dim + p.eps);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (lane + 32 * i) * V;
      if (c < p.dim) {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i][e] = xl_to_float(xl_from_float<T>((float)((double)x[i][e] * f * (double)p.wk[c + e])));
      }
    }
  };
  const bool complete = r1 == r0 + Q8_BLOCK;
  float top[2] = {0.f, 0.f};
  const int first = max(r0, fill), items = R + 2;
  // tokens that were there before (of the first block: rows of the tail and of `raw` are consecutive)
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
#pragma unroll 4
    for (int i = threadIdx.x * V; i < (first - r0) * width[kind]; i += 256 * V) {
      const Q8Piece<T, V> piece = *reinterpret_cast<const Q8Piece<T, V>*>(tail[kind] + i);
      *reinterpret_cast<Q8Piece<T, V>*>(raw[kind] + i) = piece;
#pragma unroll
      for (int e = 0; e < V; ++e) top[kind] = q8_max(top[kind], fabsf(xl_to_float(piece.v[e])));
    }
  }
  for (int i = warp; i < (r1 - first) * items; i += WARPS) {
    float x[NP][V];
    const int r = first + i / items, item = i % items, t = r - fill;
    if (item < R) {  // a query head
      load(proj + (long long)t * p.ld + (long long)(g * R + item) * p.dim, p.dim, x);
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < NP; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) sum += x[u][e] * x[u][e];
      const float f = 1.f / sqrtf(xl_warp_sum(sum) / p.dim + (float)p.eps);
      float* dst = (float*)p.q + ((head * p.T + t) * R + item) * p.dim;
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        const int c = (lane + 32 * u) * V;
        if (c < p.dim) {
#pragma unroll
          for (int e = 0; e < V; ++e) dst[c + e] = x[u][e] * f * p.wq[c + e];
        }
      }
      continue;
    }
    const int kind = item - R;
    fresh(kind, t, x);
    store(raw[kind] + (long long)r * width[kind], width[kind], x);
    if (blk == 0 && end < Q8_BLOCK) store(tail[kind] + (long long)r * width[kind], width[kind], x);
#pragma unroll
    for (int u = 0; u < NP; ++u)
#pragma unroll
      for (int e = 0; e < V; ++e) top[kind] = q8_max(top[kind], fabsf(x[u][e]));
  }
  if (complete) {
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const float m = q8_warp_max(top[kind]);
      if (lane == 0) tops[kind][warp] = m;
    }
    __syncthreads();  // the raw rows of this block are written
    const long long at = head * p.blocks + pos / Q8_BLOCK + blk;
    if (threadIdx.x < 2) {
      const int kind = threadIdx.x;
      float m = 0.f;
      for (int w = 0; w < WARPS; ++w) m = q8_max(m, tops[kind][w]);
      scales[kind] = q8_scale_of(m);
      (kind ? p.vs : p.ks)[at] = scales[kind];
    }
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const T* src = raw[kind] + (long long)r0 * width[kind];
      int8_t* dst = (kind ? p.vc : p.kc) + at * Q8_BLOCK * width[kind];
      const Q8Step step(scales[kind]);
      for (int i = threadIdx.x * V; i < Q8_BLOCK * width[kind]; i += 256 * V) {
        const Q8Piece<T, V> piece = *reinterpret_cast<const Q8Piece<T, V>*>(src + i);
        float x[V];
        uint32_t word[1];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = xl_to_float(piece.v[e]);
        step.codes(x, word);
        Q8Piece<int8_t, V> code;
#pragma unroll
        for (int e = 0; e < V; ++e) code.v[e] = (int8_t)(word[0] >> (8 * e));
        *reinterpret_cast<Q8Piece<int8_t, V>*>(dst + i) = code;
      }
    }
  }
  if (blk == 0 && end >= Q8_BLOCK) {  // the tail is the start of a later block
    __syncthreads();                  // its old rows have been read
    const int last = end / Q8_BLOCK * Q8_BLOCK;
    for (int i = warp; i < 2 * (end - last); i += WARPS) {
      float x[NP][V];
      fresh(i & 1, last + (i >> 1) - fill, x);
      store(tail[i & 1] + (long long)(i >> 1) * width[i & 1], width[i & 1], x);
    }
  }
}

__device__ __forceinline__ uint32_t q8_pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// two codes of a word (selected bytes, biased by 128) -> fp16 pair
template <int SEL> __device__ __forceinline__ uint32_t q8_pair(uint32_t biased) {
  const uint32_t w = __byte_perm(biased, 0x64646464u, SEL);
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xe480e480u));  // - 1152
  return r;
}

// ---- append for the tensor cores ----------------------------------------------------------------------------------------------
// What attention_q8_tcgen05.cu reads: queries and raw keys as fp16 in units of a power of two, raw values, and the codes of
// complete blocks as fp16 (keys) and bf16 (values). bf16 projections, dim and vdim multiples of 8 up to 128. Sixteen lanes share a row, 16 bytes
// each; a CTA has the rows of one block of one key / value head. 2 x 4096 tokens of 32 heads on 8 of 128: 65 us; the fp64 sums of the keys' norms
// and five layouts of results bound it. Raw value rows that the last block's keys do not fill are zeros: a weight of
// zero times what memory happened to hold could be NaN. For the same reason a raw value that is not finite becomes zero, and its block's
// `raw_unit` NaN instead of 1: the rows that read the block become NaN by that, and no other row of their tile.
struct Q8ExpandParams {
  const __nv_bfloat16* proj;
  long long ld;
  const float *wq, *wk;
  __half* q;                        // (B, G, T, H/G, dim)
  __half* raw_k;                    // (B, G, raw_rows, dim)
  __nv_bfloat16* raw_v;             // (B, G, raw_rows, vdim)
  float* raw_unit;                  // (B, G, q8_touched(T))
  __half* kx;                       // (B, G, held * 64, dim)
  __nv_bfloat16* vx;                // (B, G, held * 64, vdim)
  int8_t *kc, *vc;
  float *ks, *vs;
  __nv_bfloat16 *kt, *vt;
  const int *pos, *count;
  int T, H, G, dim, vdim, blocks, held, raw_rows, window, keep_first;
  double eps, inv_dim;
};

__device__ __forceinline__ void q8_unpack(const uint4& w, float (&x)[8]) {
  x[0] = dd_lo(w.x); x[1] = dd_hi(w.x); x[2] = dd_lo(w.y); x[3] = dd_hi(w.y);
  x[4] = dd_lo(w.z); x[5] = dd_hi(w.z); x[6] = dd_lo(w.w); x[7] = dd_hi(w.w);
}
__device__ __forceinline__ uint4 q8_halves(const float (&x)[8]) {
  return make_uint4(q8_pack_f16(x[0], x[1]), q8_pack_f16(x[2], x[3]), q8_pack_f16(x[4], x[5]), q8_pack_f16(x[6], x[7]));
}
// two bf16 numbers, zero in the place of one that is not finite
__device__ __forceinline__ uint32_t q8_finite_pair(uint32_t w) {
  return ((w & 0x7f80u) == 0x7f80u ? 0u : w & 0xffffu) | ((w & 0x7f800000u) == 0x7f800000u ? 0u : w & 0xffff0000u);
}
// eight codes as fp16, and as bf16
__device__ __forceinline__ uint4 q8_code_halves(const uint2& c) {
  const uint32_t a = c.x ^ 0x80808080u, b = c.y ^ 0x80808080u;
  return make_uint4(q8_pair<0x4140>(a), q8_pair<0x4342>(a), q8_pair<0x4140>(b), q8_pair<0x4342>(b));
}
__device__ __forceinline__ uint4 q8_code_values(const uint2& c) {
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = (float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3)));
  return make_uint4(dd_pack(x[0], x[1]), dd_pack(x[2], x[3]), dd_pack(x[4], x[5]), dd_pack(x[6], x[7]));
}

__global__ void __launch_bounds__(256, 4) q8_append_expand_kernel(const Q8ExpandParams p) {
  constexpr int HALVES = 16;  // half warps
  __shared__ __align__(16) uint4 tile[2][Q8_BLOCK][16];
  __shared__ float tops[2][HALVES / 2], scales[2];
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int blk = blockIdx.x, g = blockIdx.y, b = blockIdx.z, half = threadIdx.x >> 4, l = threadIdx.x & 15, lane = threadIdx.x & 31;
  const int pos = p.pos[b], n = min(p.count[b], p.T), R = p.H / p.G;
  if (n <= 0 || pos < 0 || (long long)pos + n > (long long)p.blocks * Q8_BLOCK) return;
  const int fill = pos % Q8_BLOCK, end = fill + n, r0 = blk * Q8_BLOCK, r1 = min(r0 + Q8_BLOCK, end);
  if (r0 >= end) return;
  const long long head = (long long)b * p.G + g, at = head * p.blocks + pos / Q8_BLOCK + blk;
  const long long x_at = head * p.held + q8_slots(pos, p.window, p.keep_first).of(pos / Q8_BLOCK + blk);  // if it is complete
  const __nv_bfloat16* proj = p.proj + (long long)b * p.T * p.ld;
  const bool on_k = l * 8 < p.dim, on_v = l * 8 < p.vdim;
  float wq[8], wk[8], top_q = 0.f, top_w = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = on_k ? p.wq[l * 8 + e] : 0.f;
    wk[e] = on_k ? p.wk[l * 8 + e] : 0.f;
    top_q = fmaxf(top_q, fabsf(wq[e]));
    top_w = fmaxf(top_w, fabsf(wk[e]));
  }
  const float unit_q = q8_norm_unit(top_q), inv_k = 1.f / q8_norm_unit(top_w);
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  auto key_of = [&](const uint4& w) {  // the normalised key, rounded to bf16; all lanes of the warp together
    float x[8];
    q8_unpack(w, x);
    double sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += (double)x[e] * x[e];
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const double f = rsqrt(sum * p.inv_dim + p.eps);
    uint32_t y[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = dd_pack((float)((double)x[2 * e] * f * wk[2 * e]), (float)((double)x[2 * e + 1] * f * wk[2 * e + 1]));
    return make_uint4(y[0], y[1], y[2], y[3]);
  };
  float top[2] = {0.f, 0.f};
  auto largest = [&](const uint4& w) {
    float x[8];
    q8_unpack(w, x);
    float m = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) m = q8_max(m, fabsf(x[e]));
    return m;
  };
  auto put_key = [&](int r, const uint4& w) {
    float x[8];
    q8_unpack(w, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= inv_k;
    tile[0][r - r0][l] = w;
    top[0] = q8_max(top[0], largest(w));
    if (on_k) *reinterpret_cast<uint4*>(p.raw_k + (head * p.raw_rows + r) * p.dim + l * 8) = q8_halves(x);
  };
  auto put_value = [&](int r, uint4 w) {
    tile[1][r - r0][l] = w;
    const float m = largest(w);
    top[1] = q8_max(top[1], m);
    if (!(m < INFINITY)) w = make_uint4(q8_finite_pair(w.x), q8_finite_pair(w.y), q8_finite_pair(w.z), q8_finite_pair(w.w));
    if (on_v) *reinterpret_cast<uint4*>(p.raw_v + (head * p.raw_rows + r) * p.vdim + l * 8) = w;
  };
  // tokens that were there before
  for (int r = r0 + half; r < min(r1, fill); r += HALVES) {
    put_key(r, on_k ? *reinterpret_cast<const uint4*>(p.kt + (head * Q8_BLOCK + r) * p.dim + l * 8) : zero);
    put_value(r, on_v ? *reinterpret_cast<const uint4*>(p.vt + (head * Q8_BLOCK + r) * p.vdim + l * 8) : zero);
  }
  // new tokens: whole warps go through the rows, for the sums' shuffles
  const bool to_tail = end < Q8_BLOCK;
  const int first = max(r0, fill);
  {
    constexpr int ROWS = Q8_BLOCK / HALVES;
    uint4 w[ROWS], v[ROWS];  // every load of this block before the first use
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = first + i * HALVES + half;
      const __nv_bfloat16* row = proj + (long long)(r - fill) * p.ld;
      w[i] = r < r1 && on_k ? *reinterpret_cast<const uint4*>(row + (long long)(p.H + g) * p.dim + l * 8) : zero;
      v[i] = r < r1 && on_v ? *reinterpret_cast<const uint4*>(row + (long long)(p.H + p.G) * p.dim + (long long)g * p.vdim + l * 8) : zero;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = first + i * HALVES + half;
      if (first + i * HALVES >= r1) break;
      const uint4 y = key_of(w[i]);
      if (r < r1) {
        put_key(r, y);
        put_value(r, v[i]);
        if (to_tail && on_k) *reinterpret_cast<uint4*>(p.kt + (head * Q8_BLOCK + r) * p.dim + l * 8) = y;
        if (to_tail && on_v) *reinterpret_cast<uint4*>(p.vt + (head * Q8_BLOCK + r) * p.vdim + l * 8) = v[i];
      }
    }
  }
  const int queries = (r1 - first) * R;  // consecutive in `q`, heads of a token side by side in a row of the projections
  __half* q = p.q + (head * p.T + (first - fill)) * R * p.dim;
  constexpr int BATCH = 4;
  for (int i0 = 0; i0 < queries; i0 += HALVES * BATCH) {
    uint4 w[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * HALVES + half, t = i / R, hh = i - t * R;
      w[k] = i < queries && on_k ? *reinterpret_cast<const uint4*>(proj + (long long)(first - fill + t) * p.ld + (long long)(g * R + hh) * p.dim + l * 8)
                                 : zero;
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * HALVES + half;
      float x[8], sum = 0.f;
      q8_unpack(w[k], x);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += x[e] * x[e];
#pragma unroll
      for (int d = 8; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float f = 1.f / (sqrtf(sum / p.dim + (float)p.eps) * unit_q);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= f * wq[e];
      if (i < queries && on_k) *reinterpret_cast<uint4*>(q + (long long)i * p.dim + l * 8) = q8_halves(x);
    }
  }
  for (int r = r1 + half; r < r0 + Q8_BLOCK; r += HALVES)
    if (on_v) *reinterpret_cast<uint4*>(p.raw_v + (head * p.raw_rows + r) * p.vdim + l * 8) = zero;
#pragma unroll
  for (int kind = 0; kind < 2; ++kind) {
    const float m = q8_warp_max(top[kind]);
    if (lane == 0) tops[kind][threadIdx.x >> 5] = m;
  }
  __syncthreads();
  const bool complete = r1 == r0 + Q8_BLOCK;
  if (threadIdx.x < 2) {
    float m = 0.f;
    for (int w = 0; w < HALVES / 2; ++w) m = q8_max(m, tops[threadIdx.x][w]);
    scales[threadIdx.x] = q8_scale_of(m);
    if (complete) (threadIdx.x ? p.vs : p.ks)[at] = scales[threadIdx.x];
    if (threadIdx.x == 1) p.raw_unit[head * gridDim.x + blk] = m < INFINITY ? 1.f : scales[1];
  }
  if (complete) {
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const Q8Step step(scales[kind]);
      for (int r = half; r < Q8_BLOCK; r += HALVES) {
        float x[8];
        uint32_t c[2];
        q8_unpack(tile[kind][r][l], x);
        step.codes(x, c);
        const uint2 word = make_uint2(c[0], c[1]);
        const long long row = at * Q8_BLOCK + r, x_row = x_at * Q8_BLOCK + r;
        if (kind == 0 && on_k) {
          *reinterpret_cast<uint2*>(p.kc + row * p.dim + l * 8) = word;
          *reinterpret_cast<uint4*>(p.kx + x_row * p.dim + l * 8) = q8_code_halves(word);
        } else if (kind == 1 && on_v) {
          *reinterpret_cast<uint2*>(p.vc + row * p.vdim + l * 8) = word;
          *reinterpret_cast<uint4*>(p.vx + x_row * p.vdim + l * 8) = q8_code_values(word);
        }
      }
    }
  }
  if (blk == 0 && end >= Q8_BLOCK) {  // the tail is the start of a later block
    __syncthreads();                  // its old rows have been read
    const int last = end / Q8_BLOCK * Q8_BLOCK;
    for (int rr = last; rr < end; rr += HALVES) {
      const int r = rr + half, t = r - fill;
      const bool on = r < end;
      const __nv_bfloat16* row = proj + (long long)(on ? t : 0) * p.ld;
      const uint4 w = key_of(on && on_k ? *reinterpret_cast<const uint4*>(row + (long long)(p.H + g) * p.dim + l * 8) : zero);
      if (on && on_k) *reinterpret_cast<uint4*>(p.kt + (head * Q8_BLOCK + r - last) * p.dim + l * 8) = w;
      if (on && on_v)
        *reinterpret_cast<uint4*>(p.vt + (head * Q8_BLOCK + r - last) * p.vdim + l * 8) =
            *reinterpret_cast<const uint4*>(row + (long long)(p.H + p.G) * p.dim + (long long)g * p.vdim + l * 8);
    }
  }
}

// Blocks that were complete before the portion and that its queries see: those of the kept first tokens and those from the first window
// on. Grid (groups of blocks, G, B).
constexpr int Q8_EXPAND_GROUP = 8;
__global__ void __launch_bounds__(256) q8_expand_kernel(const Q8ExpandParams p) {
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int g = blockIdx.y, b = blockIdx.z, half = threadIdx.x >> 4, l = threadIdx.x & 15;
  const int pos = p.pos[b], n = min(p.count[b], p.T);
  if (n <= 0 || pos < 0 || (long long)pos + n > (long long)p.blocks * Q8_BLOCK) return;
  const int done = pos / Q8_BLOCK, from = p.window ? max(0, pos - p.window + 1) / Q8_BLOCK : 0;
  const int kept = (int)(((long long)p.keep_first + Q8_BLOCK - 1) / Q8_BLOCK);
  const Q8Slots slots = q8_slots(pos, p.window, p.keep_first);
  const long long head = (long long)b * p.G + g;
  const bool on_k = l * 8 < p.dim, on_v = l * 8 < p.vdim;
  for (int j = blockIdx.x * Q8_EXPAND_GROUP; j < min(done, (int)(blockIdx.x + 1) * Q8_EXPAND_GROUP); ++j) {
    if (j < from && j >= kept) continue;
    const long long at = head * p.blocks + j, x_at = head * p.held + slots.of(j);
    uint2 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = at * Q8_BLOCK + half + 16 * i;
      if (on_k) k[i] = *reinterpret_cast<const uint2*>(p.kc + row * p.dim + l * 8);
      if (on_v) v[i] = *reinterpret_cast<const uint2*>(p.vc + row * p.vdim + l * 8);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long row = x_at * Q8_BLOCK + half + 16 * i;
      if (on_k) *reinterpret_cast<uint4*>(p.kx + row * p.dim + l * 8) = q8_code_halves(k[i]);
      if (on_v) *reinterpret_cast<uint4*>(p.vx + row * p.vdim + l * 8) = q8_code_values(v[i]);
    }
  }
}

// Keys of one query position: earlier blocks from the codes, its own block from `raw`; in both a kept range and a window.
struct Q8Ranges { int kept, first, own; };  // [0, kept) and [first, p]; positions from `own` on are raw
__device__ __forceinline__ Q8Ranges q8_ranges(int p, int window, int keep_first) {
  const WindowRange seen = window_range(p, window, keep_first);
  return {seen.kept, seen.first, p / Q8_BLOCK * Q8_BLOCK};
}

// four codes of a word as fp32: the byte c + 128 under 2^23, less 2^23 + 128 (a conversion instruction runs at a quarter of this rate)
__device__ __forceinline__ void q8_floats(uint32_t w, float (&x)[4]) {
  w ^= 0x80808080u;
  x[0] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540)) - 8388736.f;
  x[1] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7541)) - 8388736.f;
  x[2] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7542)) - 8388736.f;
  x[3] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7543)) - 8388736.f;
}
// dot product of n values in shared memory with a row of codes
__device__ __forceinline__ float q8_row_dot(const float* a, const int8_t* row, int n) {
  float s = 0.f;
  if ((n & 3) == 0 && (((uintptr_t)row) & 3) == 0) {
    float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int d = 0; d < n; d += 4) {
      float x[4];
      q8_floats(*reinterpret_cast<const uint32_t*>(row + d), x);
      const float4 q = *reinterpret_cast<const float4*>(a + d);
      t[0] = fmaf(q.x, x[0], t[0]);
      t[1] = fmaf(q.y, x[1], t[1]);
      t[2] = fmaf(q.z, x[2], t[2]);
      t[3] = fmaf(q.w, x[3], t[3]);
    }
    s = (t[0] + t[1]) + (t[2] + t[3]);
  } else {
    for (int d = 0; d < n; ++d) s = fmaf(a[d], (float)row[d], s);
  }
  return s;
}

struct Q8AttnParams {
  const float* q;
  const void *raw_k, *raw_v;
  const int8_t *kc, *vc;
  const float *ks, *vs;
  const void* gate;
  long long ldg;
  void* out;
  long long ldo;
  const int *pos, *count;
  int T, H, G, dim, vdim, blocks, window, keep_first;
  float scale, sink;
};

// SPLIT 1: a warp per query row, four of them per CTA. SPLIT 8: a CTA per query row whose warps take its blocks of 32 keys in turn
// and merge their parts of the softmax in shared memory, for the few rows of a decoding step (4 sequences of 216 keys, 8 heads on 2 of 128, fp32: 10 us
// after 10 of the append; codes become floats by byte selection, since conversions run at a quarter of its rate).
// VPL: value features per lane. WIDE: four neighbours at a time, for value rows of whole words; else one of each 32.
template <typename T, int VPL, int SPLIT, bool WIDE>
__global__ void __launch_bounds__(SPLIT == 1 ? 128 : SPLIT * 32) q8_attn_general_kernel(const Q8AttnParams p) {
  constexpr int ROWS = SPLIT == 1 ? 4 : 1;
  __shared__ __align__(16) float sq[ROWS][Q8_MAX_DIM];
  __shared__ float so[SPLIT == 1 ? 1 : SPLIT][SPLIT == 1 ? 1 : 32 * VPL], sm[SPLIT], sl[SPLIT];
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int slot = SPLIT == 1 ? warp : 0, part = SPLIT == 1 ? 0 : warp;
  const int h = blockIdx.y, b = blockIdx.z, R = p.H / p.G, g = h / R;
  const int t = blockIdx.x * ROWS + slot, n = min(p.count[b], p.T), pos0 = p.pos[b];
  if (t >= n || pos0 < 0 || (long long)pos0 + n > (long long)p.blocks * Q8_BLOCK) return;  // whole warps, with SPLIT > 1 whole CTAs
  const int pos = pos0 + t, base = pos0 / Q8_BLOCK * Q8_BLOCK;
  const long long head = (long long)b * p.G + g;
  const float* q = p.q + ((head * p.T + t) * R + h % R) * p.dim;
  for (int d = part * 32 + lane; d < p.dim; d += 32 * SPLIT) sq[slot][d] = q[d];
  if (SPLIT == 1) __syncwarp();
  else __syncthreads();
  const Q8Ranges seen = q8_ranges(pos, p.window, p.keep_first);
  const int8_t* kc = p.kc + head * p.blocks * Q8_BLOCK * p.dim;
  const int8_t* vc = p.vc + head * p.blocks * Q8_BLOCK * p.vdim;
  const float *ks = p.ks + head * p.blocks, *vs = p.vs + head * p.blocks;
  const T* kr = (const T*)p.raw_k + head * (p.T + Q8_BLOCK) * p.dim;
  const T* vr = (const T*)p.raw_v + head * (p.T + Q8_BLOCK) * p.vdim;
  auto feature = [&](int e) { return WIDE ? (e / 4 * 32 + lane) * 4 + (e & 3) : lane + 32 * e; };
  float o[VPL], mx = part ? -INFINITY : p.sink, l = part || p.sink == -INFINITY ? 0.f : 1.f;  // the sink is the first part's
#pragma unroll
  for (int e = 0; e < VPL; ++e) o[e] = 0.f;
  int groups = 0;
  auto walk = [&](int begin, int end, auto is_raw) {
    constexpr bool RAW = decltype(is_raw)::value;
    const int mine = (part - groups % SPLIT + SPLIT) % SPLIT;  // the warps take the groups of all ranges in turn
    groups += max(0, (end - begin + 31) / 32);
    for (int j0 = begin + mine * 32; j0 < end; j0 += 32 * SPLIT) {
      const int j = j0 + lane;
      float s = -INFINITY;
      if (j < end) {
        if (RAW) s = xl_row_dot(sq[slot], kr + (long long)(j - base) * p.dim, p.dim) * p.scale;
        else s = q8_row_dot(sq[slot], kc + (long long)j * p.dim, p.dim) * ks[j / Q8_BLOCK] * p.scale;
      }
      const float m_new = fmaxf(mx, xl_warp_max(s));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;  // scores may be infinite
      const float corr = expf(mx - m_use), w = expf(s - m_use);
      l = l * corr + xl_warp_sum(w);
      mx = m_new;
#pragma unroll
      for (int e = 0; e < VPL; ++e) o[e] *= corr;
      const float wv = RAW ? w : w * (j < end ? vs[j / Q8_BLOCK] : 0.f);
      const int m = min(32, end - j0);
#pragma unroll 8
      for (int k = 0; k < m; ++k) {
        const float wk = __shfl_sync(0xffffffffu, wv, k);
        const T* row_r = vr + (long long)(j0 + k - base) * p.vdim;
        const int8_t* row_c = vc + (long long)(j0 + k) * p.vdim;
        if (WIDE) {
#pragma unroll
          for (int e = 0; e < VPL; e += 4) {
            const int c = feature(e);
            if (c < p.vdim) {
              float x[4];
              if (RAW) {
                const Q8Piece<T, 4> piece = *reinterpret_cast<const Q8Piece<T, 4>*>(row_r + c);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = xl_to_float(piece.v[i]);
              } else {
                q8_floats(*reinterpret_cast<const uint32_t*>(row_c + c), x);
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) o[e + i] = fmaf(wk, x[i], o[e + i]);
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < VPL; ++e) {
            const int c = feature(e);
            if (c < p.vdim) o[e] = fmaf(wk, RAW ? xl_to_float(row_r[c]) : (float)row_c[c], o[e]);
          }
        }
      }
    }
  };
  using Codes = std::false_type;
  using Raw = std::true_type;
  walk(0, min(seen.kept, seen.own), Codes{});
  walk(seen.first, seen.own, Codes{});
  walk(seen.own, seen.kept, Raw{});
  walk(max(seen.first, seen.own), pos + 1, Raw{});
  if (SPLIT > 1) {
    if (lane == 0) { sm[warp] = mx; sl[warp] = l; }
#pragma unroll
    for (int e = 0; e < VPL; ++e) so[warp][lane + 32 * e] = o[e];
    __syncthreads();
    if (warp != 0) return;
    mx = sm[0];
    for (int i = 1; i < SPLIT; ++i) mx = fmaxf(mx, sm[i]);
    l = 0.f;
#pragma unroll
    for (int e = 0; e < VPL; ++e) o[e] = 0.f;
    for (int i = 0; i < SPLIT; ++i) {
      const float f = sm[i] == -INFINITY ? 0.f : expf(sm[i] - mx);  // 0 for a warp without keys
      l += sl[i] * f;
#pragma unroll
      for (int e = 0; e < VPL; ++e) o[e] += so[i][lane + 32 * e] * f;
    }
  }
  const long long row = (long long)b * p.T + t;
  const T* gr = p.gate ? (const T*)p.gate + row * p.ldg + (long long)h * p.vdim : nullptr;
#pragma unroll
  for (int e = 0; e < VPL; ++e) {
    const int c = feature(e);
    if (c < p.vdim) {
      float v = o[e] / l;
      if (gr) v *= 1.f / (1.f + expf(-xl_to_float(gr[c])));
      ((T*)p.out)[row * p.ldo + (long long)h * p.vdim + c] = xl_from_float<T>(v);
    }
  }
}

// ---- few query rows per key / value head: mma.sync -----------------------------------------------------------------------
// Grid (splits, G * row chunks, B). A CTA takes up to 8 RT rows (token-major, the query heads of one key / value head) and a share of
// the keys that any of them sees: codes in items of 32 keys, then (the last split) its raw rows in tiles of 16. Its four warps walk
// their items independently, each through a ring of its own (the codes by TMA, swizzled so that 16-byte reads by rows and ldmatrix
// by columns meet few bank conflicts), with online softmax state in registers.
//
// The products are taken transposed, so that the few query rows are the eight columns of the instruction and its sixteen rows are
// keys and features (with queries as rows, eight heads fill half of every instruction and every accumulator):
//   S^T = K Q^T   A: codes as fp16, which is exact; B: queries as fp16, divided by a power of two above the norm's factors. The
//                 scale of the block multiplies the fp32 result.
//   O^T = V^T P^T A: codes as fp16; B: weights times value scale over a 2^15th of the largest of the CTA's, as fp16 (2^-11 relative),
//                 transposed between the lanes by movmatrix
//   raw rows      keys as fp16 likewise, values in bf16 with weights as sums of two bf16 numbers
//
// A code c becomes fp16 by two instructions for two of them: the byte c + 128 is the low byte of 1024 + (c + 128) under the high byte
// 0x64, from which 1152 is taken. The value product needs keys in pairs: ldmatrix transposes pairs of bytes, that is two features of
// two keys, and the same byte selection takes even and odd features apart, whose results go to tiles of their own.
//
// FUSED (T = 1): norms, the new key and value, and a block that they complete in the same launch.
//
// Heads of 128: 16 sequences of up to 8000 keys, 32 heads on 8, 51.6 us (222 MB, read once: 4.3 TB/s; the loads alone 43.8, the rest is the
// start and the merge of the slices); one sequence of 33 keys, 16 heads on 4, 8.2; 40 sequences in a window of 256 whose token completes a
// block, 20.5: a chain of loads, norms, products and merges.
constexpr int QD_WARPS = 4;
constexpr int QD_KEYS = 32, QD_RAW = 16;
constexpr int QD_MAX_SPLITS = 64;
constexpr int QD_TABLE = 128;  // items of a CTA whose scales wait in shared memory; those of more are read when they are needed
enum { ERR_Q8_CODES = 91 };

struct Q8FewParams {
  const __nv_bfloat16* proj;
  long long ld;
  const float *wq, *wk;
  const float* q;                       // not FUSED: (B, G, T, H/G, dim), and raw rows
  const __nv_bfloat16 *raw_k, *raw_v;
  int8_t *kc, *vc;
  float *ks, *vs;
  __nv_bfloat16 *kt, *vt, *out;
  long long ldo;
  const int *pos, *count;
  int T, H, G, dim, vdim, blocks, window, keep_first, gated;
  float scale, sink;
  double eps, inv_dim;
  float* part;             // [B * G * chunks][splits][rows per CTA][vdim], then the same with [2]: maximum, sum
  unsigned int* counters;  // [B * G * chunks], zero between launches
  int stages, read_ahead, R, chunks;
  int* err;
};

__device__ __forceinline__ void q8_mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void q8_mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// transpose of an 8 x 8 matrix of 16-bit values: lane 4 r + c holds elements (r, 2 c), (r, 2 c + 1) before and (2 c, r), (2 c + 1, r) after
__device__ __forceinline__ uint32_t q8_transpose(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
template <int DK, int DV> __host__ __device__ constexpr int q8_stage_bytes() { return QD_KEYS * (DK + DV); }

// DK, DV: 64 or 128, features of a key and of a value rounded up
template <int DK, int DV, int RT, bool FUSED>
__global__ void __launch_bounds__(QD_WARPS * 32, RT == 1 ? 3 : 2)
    q8_few_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const Q8FewParams p) {
  using namespace xl_tc;
  constexpr int ROWS = 8 * RT, STAGE = q8_stage_bytes<DK, DV>(), KG = DK / 64, VT = DV / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  __shared__ __align__(16) __half sq[ROWS][DK];
  __shared__ __align__(16) __nv_bfloat16 new_k[DK], new_v[DV];
  __shared__ uint64_t bars[QD_WARPS][4];
  __shared__ float tops[3][QD_WARPS];  // value scales of the items; the block that the token completes
  __shared__ float2 table[QD_TABLE];
  __shared__ float sm[QD_WARPS][ROWS], sl[QD_WARPS][ROWS], fw[QD_WARPS][ROWS], fl[ROWS];
  __shared__ float wt[QD_MAX_SPLITS * ROWS], wl[QD_MAX_SPLITS * ROWS];
  __shared__ unsigned int is_last;
  __shared__ volatile int abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, j = lane & 3;
  const int R = p.R, chunks = p.chunks;
  const int split = blockIdx.x, splits = gridDim.x, g = chunks == 1 ? blockIdx.y : blockIdx.y / chunks, chunk = blockIdx.y - g * chunks, b = blockIdx.z;
  if (threadIdx.x == 0) {
    for (int w = 0; w < QD_WARPS; ++w)
      for (int i = 0; i < 4; ++i) mbar_init(&bars[w][i], 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (!p.read_ahead) xl_grid_dependency_wait();
  const int pos = p.pos[b], n_tok = min(p.count[b], p.T), nh = min(ROWS, n_tok * R - chunk * ROWS);
  if (nh <= 0 || pos < 0 || (long long)pos + n_tok > (long long)p.blocks * Q8_BLOCK) {
    xl_grid_dependency_wait();  // no kernel of a chain ends before its predecessor
    return;
  }
  const int p_lo = FUSED ? pos : pos + chunk * ROWS / R, p_hi = FUSED ? pos : pos + (chunk * ROWS + nh - 1) / R;
  const int base = pos / Q8_BLOCK * Q8_BLOCK, own_lo = p_lo / Q8_BLOCK * Q8_BLOCK, own_hi = p_hi / Q8_BLOCK * Q8_BLOCK;
  const long long head = (long long)b * p.G + g;
  // ---- this CTA's items -----------------------------------------------------------------------------------------------------
  const int w0 = p.window ? max(0, p_lo - p.window + 1) / QD_KEYS * QD_KEYS : 0;
  const int kept = min(min(p.keep_first, w0), own_hi), kept_items = (kept + QD_KEYS - 1) / QD_KEYS;
  const int items = kept_items + max(0, own_hi - w0) / QD_KEYS;
  const int raw0 = own_lo - base, raw_end = p_hi - base + 1, raw_tiles = (raw_end - raw0 + QD_RAW - 1) / QD_RAW;
  const unsigned all = items + raw_tiles;  // at most 2^25 items, 2^6 splits
  const int it0 = splits == 1 ? 0 : min(items, (int)(split * all / splits));
  const int it1 = splits == 1 ? items : min(items, (int)((split + 1) * all / splits));
  const bool has_raw = split == splits - 1;
  auto first_key = [&](int it) { return it < kept_items ? it * QD_KEYS : w0 + (it - kept_items) * QD_KEYS; };
  const int n_raw = has_raw ? max(0, (raw_tiles - warp + QD_WARPS - 1) / QD_WARPS) : 0;
  const int n_code = max(0, (it1 - it0 - warp + QD_WARPS - 1) / QD_WARPS), n_all = n_raw + n_code;
  const int fill = pos - base;  // FUSED: the new token's row
  uint8_t* ring = smem + warp * p.stages * STAGE;
  const int row_base = (int)(head * p.blocks) * Q8_BLOCK;
  const __nv_bfloat16* raw_k = FUSED ? p.kt + head * Q8_BLOCK * p.dim : p.raw_k + head * (p.T + Q8_BLOCK) * p.dim;
  const __nv_bfloat16* raw_v = FUSED ? p.vt + head * Q8_BLOCK * p.vdim : p.raw_v + head * (p.T + Q8_BLOCK) * p.vdim;
  auto prefetch = [&](int n) {
    if (n >= n_all) return;
    const int slot = n % p.stages;
    uint8_t* st = ring + slot * STAGE;
    if (n < n_raw) {
      const int r0 = raw0 + (warp + n * QD_WARPS) * QD_RAW, valid = FUSED ? fill : raw_end;
      for (int i = lane; i < QD_RAW * (DK / 8); i += 32) {
        const int r = i / (DK / 8), c = i % (DK / 8);
        const bool on = r0 + r < valid && c * 8 < p.dim;
        dd_cp16_zfill(st + r * (DK * 2) + ((c ^ (r & 7)) * 16), on ? raw_k + (long long)(r0 + r) * p.dim + c * 8 : raw_k, on);
      }
      for (int i = lane; i < QD_RAW * (DV / 8); i += 32) {
        const int r = i / (DV / 8), c = i % (DV / 8);
        const bool on = r0 + r < valid && c * 8 < p.vdim;
        dd_cp16_zfill(st + QD_RAW * DK * 2 + r * (DV * 2) + ((c ^ (r & 6)) * 16), on ? raw_v + (long long)(r0 + r) * p.vdim + c * 8 : raw_v, on);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    } else if (lane == 0) {
      const int row = row_base + first_key(it0 + warp + (n - n_raw) * QD_WARPS);
      mbar_expect_tx(&bars[warp][slot], STAGE);
      tma_load_2d(st, &map_k, &bars[warp][slot], 0, row);
      tma_load_2d(st + QD_KEYS * DK, &map_v, &bars[warp][slot], 0, row);
    }
  };
  for (int n = p.stages - 1; n >= 0; --n) prefetch(n);  // codes come from further away than the raw rows
  // ---- scales of the items (read once, by all threads), factors of the norms, and the largest value scale: the unit of the output --
  auto item_block = [&](int it) { return head * p.blocks + first_key(it) / Q8_BLOCK; };
  // scales of a block; where either is NaN, that of the keys is: the scores that a row sees become NaN, and its weights by them
  auto factors = [&](long long blk) {
    const float k = p.ks[blk], v = p.vs[blk];
    return make_float2(fmaf(v, 0.f, k), fmaxf(v, 0.f));
  };
  const int tabled = min(it1 - it0, QD_TABLE);
  float top_v = 0.f;
  for (int i = threadIdx.x; i < it1 - it0; i += QD_WARPS * 32) {
    const long long blk = item_block(it0 + i);
    const float2 x = factors(blk);
    if (i < QD_TABLE) table[i] = x;
    top_v = fmaxf(top_v, x.y);
  }
  float2 wq[DK / 64], wk[DK / 64];
  float top_q = 0.f, top_k = 0.f;
#pragma unroll
  for (int u = 0; u < DK / 64; ++u) {
    const int e = 2 * lane + 64 * u;
    const bool on = e < p.dim;
    wq[u] = on ? *reinterpret_cast<const float2*>(p.wq + e) : make_float2(0.f, 0.f);
    wk[u] = on ? *reinterpret_cast<const float2*>(p.wk + e) : make_float2(0.f, 0.f);
    top_q = fmaxf(top_q, fmaxf(fabsf(wq[u].x), fabsf(wq[u].y)));
    top_k = fmaxf(top_k, fmaxf(fabsf(wk[u].x), fabsf(wk[u].y)));
  }
  if (p.read_ahead) xl_grid_dependency_wait();  // the new projections
  xl_grid_launch_dependents();
  // ---- queries (fp16, in units) to shared memory; the new key and value (the last warp) --------------------------------------------
  const int plain = (p.H + p.G) * p.dim + p.G * p.vdim;
  constexpr int Q_WARPS = FUSED ? QD_WARPS - 1 : QD_WARPS, MINE_Q = (ROWS + Q_WARPS - 1) / Q_WARPS;
  float unit_q;
  if (!FUSED || warp < Q_WARPS) {
    float2 x[MINE_Q][DK / 64];
#pragma unroll
    for (int i = 0; i < MINE_Q; ++i)
#pragma unroll
      for (int u = 0; u < DK / 64; ++u) {
        const int r = warp + i * Q_WARPS, at = chunk * ROWS + r, e = 2 * lane + 64 * u;
        x[i][u] = make_float2(0.f, 0.f);
        if (r < nh && e < p.dim) {
          if (FUSED) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(p.proj + (long long)b * p.ld + (long long)(g * R + at) * p.dim + e);
            x[i][u] = make_float2(dd_lo(w), dd_hi(w));
          } else {
            x[i][u] = *reinterpret_cast<const float2*>(p.q + ((head * p.T + at / R) * R + at % R) * p.dim + e);
          }
        }
      }
    unit_q = q8_norm_unit(top_q);
    float f[MINE_Q];
#pragma unroll
    for (int i = 0; i < MINE_Q; ++i) {
      f[i] = 0.f;
#pragma unroll
      for (int u = 0; u < DK / 64; ++u) f[i] += x[i][u].x * x[i][u].x + x[i][u].y * x[i][u].y;
    }
    if (FUSED) {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1)  // the rows' sums side by side
#pragma unroll
        for (int i = 0; i < MINE_Q; ++i) f[i] += __shfl_xor_sync(0xffffffffu, f[i], d);
    }
#pragma unroll
    for (int i = 0; i < MINE_Q; ++i) {
      const int r = warp + i * Q_WARPS;
      f[i] = FUSED ? 1.f / (sqrtf(f[i] / p.dim + (float)p.eps) * unit_q) : 1.f / unit_q;
      if (r < ROWS) {
#pragma unroll
        for (int u = 0; u < DK / 64; ++u)
          *reinterpret_cast<uint32_t*>(&sq[r][2 * lane + 64 * u]) =
              FUSED ? q8_pack_f16(x[i][u].x * f[i] * wq[u].x, x[i][u].y * f[i] * wq[u].y) : q8_pack_f16(x[i][u].x * f[i], x[i][u].y * f[i]);
      }
    }
  } else {
    unit_q = q8_norm_unit(top_q);
  }
  const float unit_k = q8_norm_unit(top_k);
  {
    const float m = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)));
    if (lane == 0) tops[0][warp] = m;
  }
  const bool writes = FUSED && has_raw && chunk == 0, completes = writes && fill == Q8_BLOCK - 1;
  if (FUSED && has_raw && warp == QD_WARPS - 1) {
    const __nv_bfloat16* src = p.proj + (long long)b * p.ld + (long long)(p.H + g) * p.dim;
    const __nv_bfloat16* vsrc = p.proj + (long long)b * p.ld + (long long)(p.H + p.G) * p.dim + (long long)g * p.vdim;
    uint32_t w[DK / 64], vw[DV / 64];
    double sum = 0.0;
#pragma unroll
    for (int u = 0; u < DK / 64; ++u) w[u] = 2 * lane + 64 * u < p.dim ? *reinterpret_cast<const uint32_t*>(src + 2 * lane + 64 * u) : 0u;
#pragma unroll
    for (int u = 0; u < DV / 64; ++u) vw[u] = 2 * lane + 64 * u < p.vdim ? *reinterpret_cast<const uint32_t*>(vsrc + 2 * lane + 64 * u) : 0u;
#pragma unroll
    for (int u = 0; u < DK / 64; ++u) sum += (double)dd_lo(w[u]) * dd_lo(w[u]) + (double)dd_hi(w[u]) * dd_hi(w[u]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const double f = rsqrt(sum * p.inv_dim + p.eps);
#pragma unroll
    for (int u = 0; u < DK / 64; ++u) {
      const int e = 2 * lane + 64 * u;
      const uint32_t y = dd_pack((float)(dd_lo(w[u]) * f * (double)wk[u].x), (float)(dd_hi(w[u]) * f * (double)wk[u].y));
      *reinterpret_cast<uint32_t*>(new_k + e) = y;
      if (e < p.dim && writes && !completes) *reinterpret_cast<uint32_t*>(p.kt + (head * Q8_BLOCK + fill) * p.dim + e) = y;
    }
#pragma unroll
    for (int u = 0; u < DV / 64; ++u) {
      const int e = 2 * lane + 64 * u;
      *reinterpret_cast<uint32_t*>(new_v + e) = vw[u];
      if (e < p.vdim && writes && !completes) *reinterpret_cast<uint32_t*>(p.vt + (head * Q8_BLOCK + fill) * p.vdim + e) = vw[u];
    }
  }
  __syncthreads();
  // weights of 1 under the largest scale are 2^15, so that those under a scale a million times smaller are still normal numbers of fp16
  const float ref = it1 > it0 ? fmaxf(fmaxf(fmaxf(tops[0][0], tops[0][1]), fmaxf(tops[0][2], tops[0][3])), 1e-20f) * (1.f / 32768.f) : 1.f;
  uint32_t q[RT][KG][8];  // rows quad + 8 m, features 64 i + 16 j .. + 15
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int i = 0; i < KG; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 w = *reinterpret_cast<const uint4*>(&sq[quad + 8 * m][64 * i + 16 * j + 8 * u]);
        q[m][i][4 * u] = w.x; q[m][i][4 * u + 1] = w.y; q[m][i][4 * u + 2] = w.z; q[m][i][4 * u + 3] = w.w;
      }
  int qpos[RT][2];  // positions of this lane's rows of the scores: 8 m + 2 j + e
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) qpos[m][e] = FUSED ? pos : min(p_hi, pos + (chunk * ROWS + 8 * m + 2 * j + e) / R);
  const int lo_max = p.window ? p_hi - p.window + 1 : 0;
  auto sees = [&](int at, int key, bool raw) {
    const int own = at / Q8_BLOCK * Q8_BLOCK;
    return (raw ? key >= own && key <= at : key < own) && (!p.window || key > at - p.window || key < p.keep_first);
  };
  float o[VT][RT][4];  // features 16 t + 2 quad + (e >> 1), rows 8 m + 2 j + (e & 1)
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[t][m][e] = 0.f;
  float mx[RT][2], l[RT][2];
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      mx[m][e] = -INFINITY;
      l[m][e] = 0.f;
    }
  const float c_unit = p.scale * 1.4426950408889634f * unit_q, inv_ref = 1.f / ref;
  // scores of NT tiles of 16 keys (keys 16 t + quad + 8 (e >> 1)) -> weights (in place); rescales the output where a maximum moved
  auto softmax = [&](auto& s) {
    constexpr int NT = sizeof(s) / sizeof(s[0]);
    bool moved = false;
    float alpha[RT][2];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = -INFINITY;
#pragma unroll
        for (int t = 0; t < NT; ++t) v = fmaxf(v, fmaxf(s[t][m][e], s[t][m][e + 2]));
#pragma unroll
        for (int d = 4; d < 32; d *= 2) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, d));
        const float m_new = fmaxf(mx[m][e], v), m_use = m_new == -INFINITY ? 0.f : m_new;  // a row may see none of these keys
        alpha[m][e] = xl_tc::fast_exp2(mx[m][e] - m_use);
        moved |= m_new != mx[m][e];
        mx[m][e] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int u = 0; u < 4; u += 2) {
            s[t][m][e + u] = xl_tc::fast_exp2(s[t][m][e + u] - m_use);
            sum += s[t][m][e + u];
          }
        l[m][e] = l[m][e] * alpha[m][e] + sum;  // this lane's share of the row sum
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[t][m][e] *= alpha[m][e & 1];
    }
  };
  bool ok = true;
  int given_up = 0;
  // ---- raw tiles -------------------------------------------------------------------------------------------------------------
  for (int n = 0; n < n_raw; ++n) {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();
    uint8_t* st = ring + (n % p.stages) * STAGE;
    uint8_t* sv = st + QD_RAW * DK * 2;
    const int r0 = raw0 + (warp + n * QD_WARPS) * QD_RAW, key0 = base + r0;
    if (FUSED && fill >= r0 && fill < r0 + QD_RAW) {  // the new key and value take their place
      const int r = fill - r0;
      if (lane < DK / 8) *reinterpret_cast<uint4*>(st + r * (DK * 2) + ((lane ^ (r & 7)) * 16)) = *reinterpret_cast<const uint4*>(new_k + lane * 8);
      if (lane < DV / 8) *reinterpret_cast<uint4*>(sv + r * (DV * 2) + ((lane ^ (r & 6)) * 16)) = *reinterpret_cast<const uint4*>(new_v + lane * 8);
      __syncwarp();
    }
    if (completes) {  // every warp of the CTA has one tile: together the whole block
      float top[2] = {0.f, 0.f};
      auto largest = [&](const uint4& w, float& m) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) m = q8_max(m, q8_max(fabsf(dd_lo(u[e])), fabsf(dd_hi(u[e]))));
      };
      for (int i = lane; i < QD_RAW * (DK / 8); i += 32) largest(*reinterpret_cast<const uint4*>(st + i * 16), top[0]);
      for (int i = lane; i < QD_RAW * (DV / 8); i += 32) largest(*reinterpret_cast<const uint4*>(sv + i * 16), top[1]);
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        const float m = q8_warp_max(top[kind]);
        if (lane == 0) tops[1 + kind][warp] = m;
      }
      __syncthreads();
      const long long blk = head * p.blocks + pos / Q8_BLOCK;
      float scale[2];
#pragma unroll
      for (int kind = 0; kind < 2; ++kind) {
        float m = tops[1 + kind][0];
        for (int w = 1; w < QD_WARPS; ++w) m = q8_max(m, tops[1 + kind][w]);
        scale[kind] = q8_scale_of(m);
        if (threadIdx.x == 0) (kind ? p.vs : p.ks)[blk] = scale[kind];
      }
      const Q8Step step_k(scale[0]), step_v(scale[1]);
      auto write = [&](const uint4& w, int8_t* dst, const Q8Step& step) {
        const float x[8] = {dd_lo(w.x), dd_hi(w.x), dd_lo(w.y), dd_hi(w.y), dd_lo(w.z), dd_hi(w.z), dd_lo(w.w), dd_hi(w.w)};
        uint32_t c[2];
        step.codes(x, c);
        *reinterpret_cast<uint2*>(dst) = make_uint2(c[0], c[1]);
      };
#pragma unroll
      for (int i = lane; i < QD_RAW * (DK / 8); i += 32) {
        const int r = i / (DK / 8), c = i % (DK / 8);
        if (c * 8 < p.dim)
          write(*reinterpret_cast<const uint4*>(st + r * (DK * 2) + ((c ^ (r & 7)) * 16)), p.kc + (blk * Q8_BLOCK + r0 + r) * p.dim + c * 8, step_k);
      }
      for (int i = lane; i < QD_RAW * (DV / 8); i += 32) {
        const int r = i / (DV / 8), c = i % (DV / 8);
        if (c * 8 < p.vdim)
          write(*reinterpret_cast<const uint4*>(sv + r * (DV * 2) + ((c ^ (r & 6)) * 16)), p.vc + (blk * Q8_BLOCK + r0 + r) * p.vdim + c * 8, step_v);
      }
    }
    // Rows of different positions share a product, where a weight of zero times a value that is not finite would reach positions that do
    // not see it: such a key's values become zero, its scores NaN. (Of a single token every row sees the same keys.)
    uint32_t bad = 0u;  // bits 2 r, 2 r + 1: row r of the tile
    if (!FUSED) {
      bool any = false;
      const int r = lane >> 1;
#pragma unroll
      for (int c8 = lane & 1; c8 < DV / 8; c8 += 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(sv + r * (DV * 2) + ((c8 ^ (r & 6)) * 16));
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) any |= q8_finite_pair(x[e]) != x[e];
      }
      bad = __ballot_sync(0xffffffffu, any);
    }
    auto is_bad = [&](int r) { return (bad >> (2 * r) & 3u) != 0u; };
    float s[1][RT][4];
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[0][m][e] = 0.f;
    const float inv = 1.f / unit_k;
#pragma unroll
    for (int i = 0; i < KG; ++i)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        uint32_t k[2][4];  // keys quad, quad + 8
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 w = *reinterpret_cast<const uint4*>(st + (quad + 8 * h) * (DK * 2) + (((8 * i + 2 * j + u) ^ quad) * 16));
          const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) k[h][e] = q8_pack_f16(dd_lo(x[e]) * inv, dd_hi(x[e]) * inv);
        }
#pragma unroll
        for (int e = 0; e < 4; e += 2)
#pragma unroll
          for (int m = 0; m < RT; ++m)
            q8_mma_f16(s[0][m], k[0][e], k[1][e], k[0][e + 1], k[1][e + 1], q[m][i][4 * u + e], q[m][i][4 * u + e + 1]);
      }
    const float c = c_unit * unit_k;
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (!FUSED && bad && is_bad(quad + 8 * (e >> 1))) s[0][m][e] = __uint_as_float(0x7fc00000u);
        s[0][m][e] = sees(qpos[m][e & 1], key0 + quad + 8 * (e >> 1), true) ? s[0][m][e] * c : -INFINITY;
      }
    softmax(s);
    uint32_t ph[RT][2], pl[RT][2];  // weights in units of `ref` as operands of the second product, and their rounding errors
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float x = s[0][m][2 * u] * inv_ref, y = s[0][m][2 * u + 1] * inv_ref;
        const uint32_t w = dd_pack(x, y);
        ph[m][u] = q8_transpose(w);
        pl[m][u] = q8_transpose(dd_pack(x - dd_lo(w), y - dd_hi(w)));
      }
    bool seen[4];  // rows 2 j, 2 j + 1, 2 j + 8, 2 j + 9 of the tile: one that no row sees may hold anything
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = 2 * j + (e & 1) + 8 * (e >> 1), key = key0 + r;
      seen[e] = key <= p_hi && (!p.window || key >= p_lo - p.window + 1 || key < p.keep_first) && (FUSED || !is_bad(r));
    }
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 2 * j + (e & 1) + 8 * (e >> 1), c2 = 2 * t + (quad >> 2);
        w[e] = seen[e] ? *reinterpret_cast<const uint32_t*>(sv + r * (DV * 2) + ((c2 ^ (r & 6)) * 16) + (quad & 3) * 4) : 0u;
      }
      const uint32_t a0 = __byte_perm(w[0], w[1], 0x5410), a1 = __byte_perm(w[0], w[1], 0x7632), a2 = __byte_perm(w[2], w[3], 0x5410),
                     a3 = __byte_perm(w[2], w[3], 0x7632);
#pragma unroll
      for (int m = 0; m < RT; ++m) {
        q8_mma_bf16(o[t][m], a0, a1, a2, a3, ph[m][0], ph[m][1]);
        q8_mma_bf16(o[t][m], a0, a1, a2, a3, pl[m][0], pl[m][1]);
      }
    }
    fence_proxy_async_smem();  // ordinary accesses to the stage before TMA fills it
    __threadfence_block();
    __syncwarp();
    prefetch(n + p.stages);
  }
  // ---- codes -----------------------------------------------------------------------------------------------------------------
  for (int i = 0; i < n_code; ++i) {
    const int n = n_raw + i, slot = n % p.stages, key0 = first_key(it0 + warp + i * QD_WARPS);
    const int it = warp + i * QD_WARPS;
    float2 scale = it < tabled ? table[it] : make_float2(0.f, 0.f);
    if (it >= tabled) scale = factors(item_block(it0 + it));
    const float c = c_unit * scale.x, rel = scale.y * inv_ref;
    ok = mbar_wait_warp(&bars[warp][slot], (uint32_t)(i / p.stages) & 1u, &abort_flag, p.err, ERR_Q8_CODES);
    if (!ok) {
      given_up = i;
      break;
    }
    const uint8_t* st = ring + slot * STAGE;
    constexpr int NT = QD_KEYS / 16;
    float s[NT][RT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][m][e] = 0.f;
#pragma unroll
    for (int i2 = 0; i2 < KG; ++i2) {
      uint32_t k[NT][2][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = 16 * t + 8 * h + quad, ch = DK == 128 ? (4 * i2 + j) ^ quad : j ^ ((r >> 1) & 3);
          const uint4 w = *reinterpret_cast<const uint4*>(st + r * DK + ch * 16);
          k[t][h][0] = w.x ^ 0x80808080u; k[t][h][1] = w.y ^ 0x80808080u; k[t][h][2] = w.z ^ 0x80808080u; k[t][h][3] = w.w ^ 0x80808080u;
        }
#pragma unroll
      for (int e = 0; e < 4; ++e)  // the tiles' products side by side
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const uint32_t a0 = q8_pair<0x4140>(k[t][0][e]), a1 = q8_pair<0x4140>(k[t][1][e]), a2 = q8_pair<0x4342>(k[t][0][e]),
                         a3 = q8_pair<0x4342>(k[t][1][e]);
#pragma unroll
          for (int m = 0; m < RT; ++m) q8_mma_f16(s[t][m], a0, a1, a2, a3, q[m][i2][2 * e], q[m][i2][2 * e + 1]);
        }
    }
    const bool full = key0 + QD_KEYS <= own_lo && (key0 >= lo_max || key0 + QD_KEYS <= p.keep_first);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][m][e] *= c;
    if (!full) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int m = 0; m < RT; ++m)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (!sees(qpos[m][e & 1], key0 + 16 * t + quad + 8 * (e >> 1), false)) s[t][m][e] = -INFINITY;
    }
    softmax(s);
    uint32_t ph[NT][RT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u) ph[t][m][u] = q8_transpose(q8_pack_f16(s[t][m][2 * u] * rel, s[t][m][2 * u + 1] * rel));
    const uint32_t sv = smem_u32(st + QD_KEYS * DK) + lane * DV;
#pragma unroll
    for (int t = 0; t < VT; ++t) {
      if (t * 16 < p.vdim) {
        uint32_t w[4];  // keys 8 e + 2 j, + 1: features 16 t + 2 quad, + 1 of each
        const int ch = DV == 128 ? t ^ (lane & 7) : t ^ ((lane >> 1) & 3);
        asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                     : "r"(sv + ch * 16));
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] ^= 0x80808080u;
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          const uint32_t a0 = q8_pair<0x4240>(w[2 * k]), a1 = q8_pair<0x4341>(w[2 * k]), a2 = q8_pair<0x4240>(w[2 * k + 1]),
                         a3 = q8_pair<0x4341>(w[2 * k + 1]);
#pragma unroll
          for (int m = 0; m < RT; ++m) q8_mma_f16(o[t][m], a0, a1, a2, a3, ph[k][m][0], ph[k][m][1]);
        }
      }
    }
    __threadfence_block();  // the reads of all lanes have taken place before the stage is filled again
    __syncwarp();
    prefetch(n + p.stages);
  }
  if (!ok) {  // loads in flight target this CTA's shared memory: give them a bounded time to land before the CTA ends
    for (int i = given_up; i < min(n_code, given_up + p.stages); ++i)
      for (uint32_t w = 0; w < MBAR_SPIN_LIMIT && !mbar_try_wait(&bars[warp][(n_raw + i) % p.stages], (uint32_t)(i / p.stages) & 1u); ++w) {}
  }
  // From here on one warp per row; features c of a lane: (lane + 32 u) * 4 .. The gates are asked for before they are needed.
  constexpr int CH = (DV + 127) / 128, MINE = ROWS / QD_WARPS;
  uint2 gates[MINE][CH];
#pragma unroll
  for (int i = 0; i < MINE; ++i)
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int r = warp + i * QD_WARPS, at = chunk * ROWS + r, c = (lane + 32 * u) * 4;
      gates[i][u] = make_uint2(0u, 0u);
      if (p.gated && r < nh && c < p.vdim)
        gates[i][u] = *reinterpret_cast<const uint2*>(p.proj + ((long long)b * p.T + (FUSED ? 0 : at / R)) * p.ld + plain + (long long)(g * R + (FUSED ? at : at % R)) * p.vdim + c);
    }
#pragma unroll
  for (int m = 0; m < RT; ++m)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int d = 4; d < 32; d *= 2) l[m][e] += __shfl_xor_sync(0xffffffffu, l[m][e], d);
      if (quad == 0) {
        sm[warp][8 * m + 2 * j + e] = mx[m][e];
        sl[warp][8 * m + 2 * j + e] = l[m][e];
      }
    }
  __syncthreads();  // all rings are idle: their memory holds the warps' outputs from here on
  float* so = reinterpret_cast<float*>(smem);  // [QD_WARPS][ROWS][vdim + 8]
  const int old = p.vdim + 8;                  // the padding keeps the stores of different rows in different banks
#pragma unroll
  for (int t = 0; t < VT; ++t) {
    if (t * 16 < p.vdim) {
#pragma unroll
      for (int m = 0; m < RT; ++m)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<float2*>(so + (warp * ROWS + 8 * m + 2 * j + e) * old + t * 16 + 2 * quad) =
              make_float2(o[t][m][e] * ref, o[t][m][e + 2] * ref);
    }
  }
  // ---- merge of the warps: their weights, and the sums of the weights --------------------------------------------------------
  const long long units = (long long)gridDim.z * gridDim.y, unit = (long long)b * gridDim.y + blockIdx.y;
  const float sink = p.sink * 1.4426950408889634f;
  float2* stats = reinterpret_cast<float2*>(p.part + units * splits * ROWS * p.vdim);
  if (threadIdx.x < ROWS) {
    const int r = threadIdx.x;
    float m = splits > 1 ? -INFINITY : sink;
#pragma unroll
    for (int w = 0; w < QD_WARPS; ++w) m = fmaxf(m, sm[w][r]);
    float ll = splits > 1 || sink == -INFINITY ? 0.f : xl_tc::fast_exp2(sink - m);
#pragma unroll
    for (int w = 0; w < QD_WARPS; ++w) {
      const float f = sm[w][r] == -INFINITY ? 0.f : xl_tc::fast_exp2(sm[w][r] - m);
      fw[w][r] = f;
      ll += sl[w][r] * f;  // NaN where the warp's only visible keys were no numbers, and its maximum says nothing of them
    }
    fl[r] = ll;
    if (splits > 1) __stcg(stats + (unit * splits + split) * ROWS + r, make_float2(m, ll));
  }
  __syncthreads();
  auto merged = [&](int r, int c) {  // row r, features c .. c + 3, over this CTA's warps
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < QD_WARPS; ++w) {
      const float f = fw[w][r];
      const float4 x = *reinterpret_cast<const float4*>(so + (w * ROWS + r) * old + c);
      if (sm[w][r] != -INFINITY) a = make_float4(a.x + x.x * f, a.y + x.y * f, a.z + x.z * f, a.w + x.w * f);
    }
    return a;
  };
  if (splits > 1) {
    for (int r = warp; r < nh; r += QD_WARPS)
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const int c = (lane + 32 * u) * 4;
        if (c < p.vdim) __stcg(reinterpret_cast<float4*>(p.part + ((unit * splits + split) * ROWS + r) * p.vdim + c), merged(r, c));
      }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) is_last = atomicAdd(p.counters + unit, 1u) == (unsigned int)splits - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    for (int i = threadIdx.x; i < splits * ROWS; i += blockDim.x) {
      const float2 v = __ldcg(stats + unit * splits * ROWS + i);
      wt[i] = v.x;
      wl[i] = v.y;
    }
    __syncthreads();
    if (threadIdx.x < ROWS) {
      float m = sink;
      for (int k = 0; k < splits; ++k) m = fmaxf(m, wt[k * ROWS + threadIdx.x]);
      float ll = sink == -INFINITY ? 0.f : xl_tc::fast_exp2(sink - m);
      for (int k = 0; k < splits; ++k) {
        float& w = wt[k * ROWS + threadIdx.x];
        w = w == -INFINITY ? 0.f : xl_tc::fast_exp2(w - m);
        ll += w * wl[k * ROWS + threadIdx.x];
      }
      fl[threadIdx.x] = ll;
    }
    if (threadIdx.x == 0) p.counters[unit] = 0;
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int r = warp + i * QD_WARPS;
    if (r >= nh) break;
    const int at = chunk * ROWS + r;
    const float sum = fl[r];
    __nv_bfloat16* out = p.out + ((long long)b * p.T + (FUSED ? 0 : at / R)) * p.ldo + (long long)(g * R + (FUSED ? at : at % R)) * p.vdim;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int c = (lane + 32 * u) * 4;
      if (c >= p.vdim) continue;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
      if (splits > 1) {
        const float* src = p.part + (unit * splits * ROWS + r) * p.vdim + c;
#pragma unroll 4
        for (int k = 0; k < splits; ++k) {
          const float f = wt[k * ROWS + r];
          const float4 x = __ldcg(reinterpret_cast<const float4*>(src + (long long)k * ROWS * p.vdim));
          a = make_float4(a.x + x.x * f, a.y + x.y * f, a.z + x.z * f, a.w + x.w * f);
        }
      } else {
        a = merged(r, c);
      }
      float v[4] = {a.x / sum, a.y / sum, a.z / sum, a.w / sum};
      if (p.gated) {
        const uint2 gt = gates[i][u];
        v[0] *= 1.f / (1.f + expf(-dd_lo(gt.x)));
        v[1] *= 1.f / (1.f + expf(-dd_hi(gt.x)));
        v[2] *= 1.f / (1.f + expf(-dd_lo(gt.y)));
        v[3] *= 1.f / (1.f + expf(-dd_hi(gt.y)));
      }
      dd_store4(out + c, v[0], v[1], v[2], v[3], ((uintptr_t)out & 3) == 0);
    }
  }
}

// 2-D map over rows of `cols` codes, boxes of {width, QD_KEYS}: columns past the row are filled with zeros
int q8_make_map(CUtensorMap* map, const void* ptr, long long rows, int cols, int width) {
  xl_tc::EncodeTiledFn fn = xl_tc::get_encode_fn();
  if (!fn) return -2;
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)cols};
  cuuint32_t box[2] = {(cuuint32_t)width, QD_KEYS};
  cuuint32_t estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, (void*)ptr, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        width == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : -3;
}

constexpr int q8_ring_limit(int rt) { return (rt == 1 ? 65 : 100) * 1024; }  // three CTAs per SM, two

template <int DK, int DV, int RT, bool FUSED> int q8_few_launch(Q8FewParams p, int B, int splits, cudaStream_t s) {
  constexpr int STAGE = q8_stage_bytes<DK, DV>() * QD_WARPS;
  p.stages = 4 * STAGE <= q8_ring_limit(RT) ? 4 : (3 * STAGE <= q8_ring_limit(RT) ? 3 : 2);
  static_assert(2 * STAGE <= q8_ring_limit(RT), "ring");
  constexpr int merge = QD_WARPS * 8 * RT * (DV + 8) * 4;
  const int ring = p.stages * STAGE, bytes = (ring > merge ? ring : merge) + 1024;
  CUtensorMap mk, mv;
  const long long rows = (long long)B * p.G * p.blocks * Q8_BLOCK;
  int r = q8_make_map(&mk, p.kc, rows, p.dim, DK);
  if (!r) r = q8_make_map(&mv, p.vc, rows, p.vdim, DV);
  if (r) return r;
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(q8_few_rows_kernel<DK, DV, RT, FUSED>, bytes, smem));
  p.R = p.H / p.G;
  p.chunks = (p.T * p.R + 8 * RT - 1) / (8 * RT);
  const cudaError_t e = xl_launch_overlapped(q8_few_rows_kernel<DK, DV, RT, FUSED>, dim3(splits, p.G * p.chunks, B), dim3(QD_WARPS * 32),
                                             (size_t)bytes, s, mk, mv, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <int DK, int DV> int q8_few_sizes(const Q8FewParams& p, int B, int splits, cudaStream_t s) {
  const bool one = p.T * (p.H / p.G) <= 8;
  if (p.T == 1) return one ? q8_few_launch<DK, DV, 1, true>(p, B, splits, s) : q8_few_launch<DK, DV, 2, true>(p, B, splits, s);
  return one ? q8_few_launch<DK, DV, 1, false>(p, B, splits, s) : q8_few_launch<DK, DV, 2, false>(p, B, splits, s);
}

bool q8_sizes_ok(int B, int T, int H, int G, int dim, int vdim, int blocks) {
  return B >= 1 && B <= 65535 && T >= 1 && T <= (1 << 24) && G >= 1 && G <= 65535 && H >= 1 && H <= 65535 && H % G == 0 && dim >= 1 &&
         dim <= Q8_MAX_DIM && vdim >= 1 && vdim <= Q8_MAX_DIM && blocks >= 1 && blocks <= (1 << 24);
}

}  // namespace

// proj (B*T, ld): [q: H x dim | k: G x dim | v: G x vdim | ...]; q (B, G, T, H/G, dim) fp32; raw_k, raw_v (B, G, T + 64, dim | vdim);
// codes, scales and tails as in attention_q8.cuh. dim, vdim <= 512. Sequences that would not fit, and rows past count[b], are left out.
XL_API int xl_q8_append(const void* proj, long long ld, const float* wq, const float* wk, void* q, void* raw_k, void* raw_v, void* kc,
                        void* vc, float* ks, float* vs, void* kt, void* vt, const int* pos, const int* count, int B, int T, int H, int G,
                        int dim, int vdim, int blocks, double eps, int dtype, cudaStream_t s) {
  if (!q8_sizes_ok(B, T, H, G, dim, vdim, blocks) || ld < (long long)(H + G) * dim + (long long)G * vdim || !wq || !wk) return -1;
  const Q8AppendParams p{proj, ld, wq, wk, q, raw_k, raw_v, (int8_t*)kc, (int8_t*)vc, ks, vs, kt, vt, pos, count, T, H, G, dim, vdim,
                         blocks, eps};
  const dim3 grid(q8_touched(T), G, B);
  XL_DISPATCH_DTYPE(dtype, D, {
    const uintptr_t at = (uintptr_t)proj | (uintptr_t)raw_k | (uintptr_t)raw_v | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)kt | (uintptr_t)vt;
    const bool four = dim % 4 == 0 && vdim % 4 == 0 && ld % 4 == 0 && (at & 15) == 0;
    XL_TRY(xl_launch_overlapped(four ? q8_append_kernel<D, 4> : q8_append_kernel<D, 1>, grid, dim3(256), (size_t)0, s, p));
  });
  return (int)cudaGetLastError();
}

// After xl_q8_append. gate: first gate column of the projections (row stride ldg), or null; out (B*T, ldo). sink -inf: none.
XL_API int xl_q8_attn_general(const float* q, const void* raw_k, const void* raw_v, const void* kc, const void* vc, const float* ks,
                              const float* vs, const void* gate, long long ldg, void* out, long long ldo, const int* pos,
                              const int* count, int B, int T, int H, int G, int dim, int vdim, int blocks, int window, int keep_first,
                              float scale, float sink, int dtype, cudaStream_t s) {
  if (!q8_sizes_ok(B, T, H, G, dim, vdim, blocks) || window < 0 || keep_first < 0 || !(scale > 0.f) || ldo < (long long)H * vdim) return -1;
  const Q8AttnParams p{q, raw_k, raw_v, (const int8_t*)kc, (const int8_t*)vc, ks, vs, gate, ldg, out, ldo, pos, count, T, H, G, dim, vdim,
                       blocks, window, keep_first, scale, sink};
  // a CTA per row while that is no more than about two CTAs of eight warps per SM; longer portions fill the SMs with a warp per row
  const bool split = (long long)T * H * B <= 2 * 148;
  const dim3 grid(split ? T : (T + 3) / 4, H, B), block(split ? 256 : 128);
  XL_DISPATCH_DTYPE(dtype, D, {
    const bool wide = vdim % 4 == 0 && (((uintptr_t)raw_v | (uintptr_t)vc) & 15) == 0;
    void (*kernel)(const Q8AttnParams);
    if (wide)
      kernel = vdim <= 128 ? (split ? q8_attn_general_kernel<D, 4, 8, true> : q8_attn_general_kernel<D, 4, 1, true>)
                           : (split ? q8_attn_general_kernel<D, 16, 8, true> : q8_attn_general_kernel<D, 16, 1, true>);
    else
      kernel = vdim <= 128 ? (split ? q8_attn_general_kernel<D, 4, 8, false> : q8_attn_general_kernel<D, 4, 1, false>)
                           : (split ? q8_attn_general_kernel<D, 16, 8, false> : q8_attn_general_kernel<D, 16, 1, false>);
    XL_TRY(xl_launch_overlapped(kernel, grid, block, (size_t)0, s, p));
  });
  return (int)cudaGetLastError();
}

// Few rows per sequence, bf16: dim, vdim multiples of 16 up to 128, ld, ldo and all pointers as the 16-byte accesses need them.
// T = 1: the kernel normalises, appends and completes blocks itself (q and raw rows are null). T > 1: after xl_q8_append, on its q and
// raw rows, with read_ahead 0. part: B * G * ceil(T H/G / 8 RT) * splits * 8 RT * (vdim + 2) floats with RT = 1 where T H/G <= 8, else
// 2; counters: B * G * ceil(...) zero-initialised words (left zeroed). read_ahead: positions, counts, the cache and the factors of both norms
// were complete before the previous launch. err: device int for the code of a wait that gave up.
XL_API int xl_q8_attn_few(const void* proj, long long ld, const float* wq, const float* wk, const float* q, const void* raw_k,
                          const void* raw_v, void* kc, void* vc, float* ks, float* vs, void* kt, void* vt, void* out, long long ldo,
                          const int* pos, const int* count, int B, int T, int H, int G, int dim, int vdim, int blocks, int window,
                          int keep_first, int gated, float scale, float sink, double eps, int splits, float* part, unsigned int* counters,
                          int read_ahead, int* err, cudaStream_t s) {
  if (!q8_sizes_ok(B, T, H, G, dim, vdim, blocks) || window < 0 || keep_first < 0 || !(scale > 0.f) || !wq || !wk) return -1;
  if (dim % 16 || vdim % 16 || dim > 128 || vdim > 128 || ld % 8 || ldo < (long long)H * vdim || splits < 1 || splits > QD_MAX_SPLITS ||
      ld < (long long)(H + G) * dim + (long long)G * vdim + (gated ? (long long)H * vdim : 0) || (T > 1 && (read_ahead || !q || !raw_k || !raw_v)))
    return -1;
  const uintptr_t at = (uintptr_t)proj | (uintptr_t)raw_k | (uintptr_t)raw_v | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)kt | (uintptr_t)vt;
  if ((at & 15) || (splits > 1 && (!part || ((uintptr_t)part & 15) || !counters)) || !err) return -1;
  const long long chunks = ((long long)T * (H / G) + 7) / 8;
  if ((long long)B * G * blocks * Q8_BLOCK > 0x7fffff00LL || G * chunks > 65535) return -1;
  Q8FewParams p = {};
  p.proj = (const __nv_bfloat16*)proj; p.ld = ld; p.wq = wq; p.wk = wk; p.q = q; p.raw_k = (const __nv_bfloat16*)raw_k;
  p.raw_v = (const __nv_bfloat16*)raw_v; p.kc = (int8_t*)kc; p.vc = (int8_t*)vc; p.ks = ks; p.vs = vs; p.kt = (__nv_bfloat16*)kt;
  p.vt = (__nv_bfloat16*)vt; p.out = (__nv_bfloat16*)out; p.ldo = ldo; p.pos = pos; p.count = count; p.T = T; p.H = H; p.G = G;
  p.dim = dim; p.vdim = vdim; p.blocks = blocks; p.window = window; p.keep_first = keep_first; p.gated = gated; p.scale = scale;
  p.sink = sink; p.eps = eps; p.inv_dim = 1.0 / dim; p.part = part; p.counters = counters; p.read_ahead = read_ahead; p.err = err;
  if (dim <= 64) return vdim <= 64 ? q8_few_sizes<64, 64>(p, B, splits, s) : q8_few_sizes<64, 128>(p, B, splits, s);
  return vdim <= 64 ? q8_few_sizes<128, 64>(p, B, splits, s) : q8_few_sizes<128, 128>(p, B, splits, s);
}

// The same as xl_q8_append for xl_q8_attn_tcgen05 (see there): q (B, G, T, H/G, dim) and raw_k (B, G, raw_rows, dim) fp16, raw_v (B, G,
// raw_rows, vdim) bf16 with raw_rows >= T + 128, raw_unit (B, G, (T + 126) / 64) fp32, kx (B, G, held * 64, dim)
// fp16, vx (.., vdim) bf16: complete blocks that the portion can see, in `held` places (q8_held, or more). bf16; dim, vdim multiples of 8 up to 128, ld a multiple of 8, all pointers 16-byte aligned.
XL_API int xl_q8_append_expand(const void* proj, long long ld, const float* wq, const float* wk, void* q, void* raw_k, void* raw_v,
                               int raw_rows, float* raw_unit, void* kx, void* vx, int held, void* kc, void* vc, float* ks, float* vs,
                               void* kt, void* vt, const int* pos, const int* count, int B, int T, int H, int G, int dim, int vdim,
                               int blocks, int window, int keep_first, double eps, cudaStream_t s) {
  if (!q8_sizes_ok(B, T, H, G, dim, vdim, blocks) || dim % 8 || vdim % 8 || dim > 128 || vdim > 128 || ld % 8 || !wq || !wk || !raw_unit ||
      ld < (long long)(H + G) * dim + (long long)G * vdim || raw_rows < T + 2 * Q8_BLOCK || window < 0 || keep_first < 0 ||
      held < q8_held(T, blocks, window, keep_first))
    return -1;
  const uintptr_t at = (uintptr_t)proj | (uintptr_t)q | (uintptr_t)raw_k | (uintptr_t)raw_v | (uintptr_t)kx | (uintptr_t)vx | (uintptr_t)kc |
                       (uintptr_t)vc | (uintptr_t)kt | (uintptr_t)vt;
  if (at & 15) return -1;
  const Q8ExpandParams p{(const __nv_bfloat16*)proj, ld, wq, wk, (__half*)q, (__half*)raw_k, (__nv_bfloat16*)raw_v, raw_unit, (__half*)kx,
                         (__nv_bfloat16*)vx, (int8_t*)kc, (int8_t*)vc, ks, vs, (__nv_bfloat16*)kt, (__nv_bfloat16*)vt, pos, count, T, H, G, dim,
                         vdim, blocks, held, raw_rows, window, keep_first, eps, 1.0 / dim};
  XL_TRY(xl_launch_overlapped(q8_append_expand_kernel, dim3(q8_touched(T), G, B), dim3(256), (size_t)0, s, p));
  XL_TRY(xl_launch_overlapped(q8_expand_kernel, dim3((blocks + Q8_EXPAND_GROUP - 1) / Q8_EXPAND_GROUP, G, B), dim3(256), (size_t)0, s, p));
  return (int)cudaGetLastError();
}
