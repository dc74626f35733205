// Sliding-window attention against a key / value cache of 8 bits: normalised queries and keys, kept first tokens, a sink, a gate
// (the mathematics of attention_window.cu; layouts in attention_q8.cuh). Keys are normalised in 64 bits and rounded once to the
// model's type, so that every kernel and every division into portions comes to the same codes. Queries are not rounded to it.
//
//   xl_q8_append          queries to their buffer, keys and values to `raw`; complete blocks to codes, the rest to the tails
//   xl_q8_attn_general    any sizes and types, scores and weights in fp32 on the CUDA cores: one warp per row and head
#include "attention_q8.cuh"

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
  for (int i = warp; i < (r1 - first) * items + 2 * (first - r0); i += WARPS) {
    float x[NP][V];
    const int k = i - (r1 - first) * items;
    if (k >= 0) {  // a token that was there before
      const int r = r0 + (k >> 1), kind = k & 1;
      load(tail[kind] + (long long)r * width[kind], width[kind], x);
      store(raw[kind] + (long long)r * width[kind], width[kind], x);
#pragma unroll
      for (int u = 0; u < NP; ++u)
#pragma unroll
        for (int e = 0; e < V; ++e) top[kind] = fmaxf(top[kind], fabsf(x[u][e]));
      continue;
    }
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
      for (int e = 0; e < V; ++e) top[kind] = fmaxf(top[kind], fabsf(x[u][e]));
  }
  if (complete) {
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const float m = xl_warp_max(top[kind]);
      if (lane == 0) tops[kind][warp] = m;
    }
    __syncthreads();  // the raw rows of this block are written
    const long long at = head * p.blocks + pos / Q8_BLOCK + blk;
    if (threadIdx.x < 2) {
      const int kind = threadIdx.x;
      float m = 0.f;
      for (int w = 0; w < WARPS; ++w) m = fmaxf(m, tops[kind][w]);
      scales[kind] = __fdiv_rn(m, 127.f);
      (kind ? p.vs : p.ks)[at] = scales[kind];
    }
    __syncthreads();
#pragma unroll
    for (int kind = 0; kind < 2; ++kind) {
      const T* src = raw[kind] + (long long)r0 * width[kind];
      int8_t* dst = (kind ? p.vc : p.kc) + at * Q8_BLOCK * width[kind];
      const float scale = scales[kind];
      for (int i = threadIdx.x * V; i < Q8_BLOCK * width[kind]; i += 256 * V) {
        const Q8Piece<T, V> piece = *reinterpret_cast<const Q8Piece<T, V>*>(src + i);
        Q8Piece<int8_t, V> code;
#pragma unroll
        for (int e = 0; e < V; ++e) code.v[e] = (int8_t)q8_code(xl_to_float(piece.v[e]), scale);
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

// Keys of one query position: earlier blocks from the codes, its own block from `raw`; in both a kept range and a window.
struct Q8Ranges { int kept, first, own; };  // [0, kept) and [first, p]; positions from `own` on are raw
__device__ __forceinline__ Q8Ranges q8_ranges(int p, int window, int keep_first) {
  const WindowRange seen = window_range(p, window, keep_first);
  return {seen.kept, seen.first, p / Q8_BLOCK * Q8_BLOCK};
}

// dot product of n values in shared memory with a row of codes
__device__ __forceinline__ float q8_row_dot(const float* a, const int8_t* row, int n) {
  float s = 0.f;
  if ((n & 3) == 0 && (((uintptr_t)row) & 3) == 0) {
#pragma unroll 8
    for (int d = 0; d < n; d += 4) {
      const char4 c = *reinterpret_cast<const char4*>(row + d);
      s = fmaf(a[d], (float)c.x, s);
      s = fmaf(a[d + 1], (float)c.y, s);
      s = fmaf(a[d + 2], (float)c.z, s);
      s = fmaf(a[d + 3], (float)c.w, s);
    }
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
// and merge their parts of the softmax in shared memory, for the few rows of a decoding step.
template <typename T, int VPL, int SPLIT>  // VPL: value features per lane
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
  float o[VPL], mx = part ? -INFINITY : p.sink, l = part || p.sink == -INFINITY ? 0.f : 1.f;  // the sink is the first part's
#pragma unroll
  for (int e = 0; e < VPL; ++e) o[e] = 0.f;
  auto walk = [&](int begin, int end, auto is_raw) {
    constexpr bool RAW = decltype(is_raw)::value;
    for (int j0 = begin + part * 32; j0 < end; j0 += 32 * SPLIT) {
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
#pragma unroll 4
      for (int k = 0; k < m; ++k) {
        const float wk = __shfl_sync(0xffffffffu, wv, k);
#pragma unroll
        for (int e = 0; e < VPL; ++e) {
          const int c = lane + 32 * e;
          if (c < p.vdim)
            o[e] = fmaf(wk, RAW ? xl_to_float(vr[(long long)(j0 + k - base) * p.vdim + c]) : (float)vc[(long long)(j0 + k) * p.vdim + c],
                        o[e]);
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
    const int c = lane + 32 * e;
    if (c < p.vdim) {
      float v = o[e] / l;
      if (gr) v *= 1.f / (1.f + expf(-xl_to_float(gr[c])));
      ((T*)p.out)[row * p.ldo + (long long)h * p.vdim + c] = xl_from_float<T>(v);
    }
  }
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
  const dim3 grid((T + 2 * Q8_BLOCK - 2) / Q8_BLOCK, G, B);
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
    void (*kernel)(const Q8AttnParams) = vdim <= 128 ? (split ? q8_attn_general_kernel<D, 4, 8> : q8_attn_general_kernel<D, 4, 1>)
                                                     : (split ? q8_attn_general_kernel<D, 16, 8> : q8_attn_general_kernel<D, 16, 1>);
    XL_TRY(xl_launch_overlapped(kernel, grid, block, (size_t)0, s, p));
  });
  return (int)cudaGetLastError();
}
