// Logits shaped by the rules of a slot, and the choice of a token from them.
//
//   x = l                                            seen:  the token occurs among the slot's first `length` tokens
//   x = x > 0 ? x / repetition : x * repetition      where seen
//   x = x - frequency * times - presence             where times > 0: occurrences since the prompt
//   x = x + sum of the slot's biases of the token
//   x = -inf                                         where the slot's mask has no bit for the token
//
// A pass reads the logits once and writes the shaped row, or only the token chosen. What a slot remembers is its tokens, not a
// count for every entry of the vocabulary: a CTA counts the tokens of its slice of the vocabulary in shared memory, one word per
// entry, and an entry whose word is zero needs its mask bit and nothing else. Sums and quotients are rounded one by one (no
// contraction), so the results are those of the formula in 32 bits, bit for bit, and ties stay ties.
#include "common.cuh"

#include <cooperative_groups.h>
#include <math.h>

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 8192;        // entries of the vocabulary counted at a time: 32 KB of words
constexpr int LG_MAX_BIASES = 1024;
// word of an entry: bit 31 seen, bits 20 .. 30 one more than the place of its bias in the list, bits 0 .. 19 times
constexpr uint32_t LG_SEEN = 1u << 31, LG_TIMES = (1u << 20) - 1;
constexpr int LG_BIAS_SHIFT = 20;

struct LogitRulesArgs {
  int* history;
  const int* start;
  const float* penalties;
  const int* bias_tokens;
  const float* bias_values;
  const uint32_t* allowed;
  int slots, length, biases, words;  // rows of the rules; columns of history, bias lists, masks
};

struct Best { float v; int i; };
__device__ __forceinline__ void best_of(Best& b, float v, int i) {
  if (v > b.v || (v == b.v && i < b.i)) { b.v = v; b.i = i; }
}

__device__ __forceinline__ float shaped(float x, uint32_t word, bool ok, float repetition, float frequency, float presence,
                                        const float* bias_sum) {
  if (word) {
    if (word & LG_SEEN) x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
    const uint32_t times = word & LG_TIMES;
    if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)times)), presence);
    const uint32_t k = (word & ~LG_SEEN) >> LG_BIAS_SHIFT;
    if (k) x = __fadd_rn(x, bias_sum[k - 1]);
  }
  return ok ? x : -INFINITY;
}

// What the choice does with its token (see xl_take_shaped).
struct ShapedTake {
  int *current, *buf, *pos;
  const int* count;
  int buf_rows, base, ahead, advance, rows;
  unsigned int* counter;
};

// Grid (parts, rows). Entries are numbered from the 16-byte boundary at or before the row's first logit (`phase` entries earlier),
// so that groups of N entries are whole 16-byte pieces of the logits; a part is a whole number of groups.
// CHOOSE: the parts of a row are a cluster, whose winners meet in the first CTA.
template <typename T, bool CHOOSE>
__global__ void __launch_bounds__(LG_THREADS)
    logits_kernel(const T* logits, float* out, const int* slot_of, const int* length_of, const LogitRulesArgs r, int V, int valid,
                  int per_part, const ShapedTake take) {
  constexpr int N = XlVec<T>::N;
  __shared__ __align__(16) uint32_t words[LG_CHUNK];
  __shared__ __align__(16) int tokens[LG_MAX_BIASES];
  __shared__ float sums[LG_MAX_BIASES];
  const int part = blockIdx.x, tid = threadIdx.x;
  const long long row = blockIdx.y;
  const int phase = (int)((row * V) % N);
  const int u_end = phase + valid, u0 = part * per_part, u1 = min(u0 + per_part, u_end);
  auto clear = [&](int n) {
    for (int i = tid * 4; i < n; i += LG_THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0u, 0u, 0u, 0u);
  };
  clear(min(per_part, LG_CHUNK));
  xl_grid_dependency_wait();
  if (!CHOOSE) xl_grid_launch_dependents();
  const int slot = CHOOSE ? (int)row : slot_of[row];
  const bool ruled = slot >= 0 && slot < r.slots, live = !CHOOSE || take.count[row] > 0;
  const T* p = logits + row * V - phase;
  float* o = CHOOSE ? nullptr : out + row * V - phase;
  Best best{-INFINITY, 0};
  if (live) {
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    int held = 0, start = 0, biases = 0;
    const int* past = r.history;
    const uint32_t* mask = r.allowed;
    if (ruled) {
      repetition = r.penalties[slot * 3];
      frequency = r.penalties[slot * 3 + 1];
      presence = r.penalties[slot * 3 + 2];
      past += (long long)slot * r.length;
      mask += (long long)slot * r.words;
      held = max(0, min(length_of[row], r.length));
      start = r.start[slot];
      biases = r.biases;
      if (repetition == 1.f && frequency == 0.f && presence == 0.f) held = 0;  // nothing that the tokens would change
      for (int k = tid; k < biases; k += LG_THREADS) tokens[k] = r.bias_tokens[(long long)slot * biases + k];
      for (int k = biases + tid; k < (biases + 3) / 4 * 4; k += LG_THREADS) tokens[k] = -1;
    }
    __syncthreads();
    for (int c0 = u0; c0 < u1; c0 += LG_CHUNK) {
      const int c1 = min(c0 + LG_CHUNK, u1);
      if (c0 > u0) {
        __syncthreads();
        clear(c1 - c0);
        __syncthreads();
      }
      const int lo = c0 - phase, n = c1 - c0;  // token of the first word (negative before the row), words
#pragma unroll 8
      for (int i = tid; i < held; i += LG_THREADS) {
        const int t = past[i];
        const unsigned w = (unsigned)(t - lo);
        if (t >= 0 && w < (unsigned)n) {
          if (i >= start) atomicAdd(words + w, 1u);
          atomicOr(words + w, LG_SEEN);
        }
      }
      // a token's first entry in the list takes the sum of all of them, in the order of the list
      for (int k = tid; k < biases; k += LG_THREADS) {
        const int t = tokens[k];
        const unsigned w = (unsigned)(t - lo);
        if (t >= 0 && w < (unsigned)n) {
          bool first = true;
          float sum = 0.f;
          for (int q = 0; q < biases; q += 4) {
            const int4 other = *reinterpret_cast<const int4*>(tokens + q);
            const int at[4] = {other.x, other.y, other.z, other.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (at[e] == t) {
                first &= q + e >= k;
                sum = __fadd_rn(sum, r.bias_values[(long long)slot * biases + q + e]);
              }
          }
          if (first) {
            sums[k] = sum;
            atomicOr(words + w, (uint32_t)(k + 1) << LG_BIAS_SHIFT);
          }
        }
      }
      __syncthreads();
      for (int u = c0 + tid * N; u < c1; u += LG_THREADS * N) {
        const int e0 = u - phase;  // token of the group's first entry
        float x[N];
        uint32_t bits = 0xffffffffu;
        if (e0 >= 0 && u + N <= u_end) {
          xl_load16(p + u, x);
          if (ruled) {
            const int w = e0 >> 5, s = e0 & 31;
            const uint32_t w0 = mask[w], w1 = s + N > 32 ? mask[w + 1] : 0u;  // the group's last token is below `valid`
            bits = __funnelshift_r(w0, w1, s);
          }
          uint32_t word[N];
#pragma unroll
          for (int i = 0; i < N; i += 4) {
            const uint4 q = *reinterpret_cast<const uint4*>(words + (u - c0) + i);
            word[i] = q.x; word[i + 1] = q.y; word[i + 2] = q.z; word[i + 3] = q.w;
          }
#pragma unroll
          for (int i = 0; i < N; ++i) {
            x[i] = shaped(x[i], word[i], (bits >> i) & 1u, repetition, frequency, presence, sums);
            if (CHOOSE) best_of(best, x[i], e0 + i);
          }
          if (!CHOOSE) {
#pragma unroll
            for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(o + u + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
          }
        } else {  // the row's first and last group
          for (int i = 0; i < N; ++i) {
            const int t = e0 + i;
            if (t < 0 || t >= valid) continue;
            const bool ok = !ruled || ((mask[t >> 5] >> (t & 31)) & 1u);
            const float y = shaped(xl_to_float(p[u + i]), words[u - c0 + i], ok, repetition, frequency, presence, sums);
            if (CHOOSE) best_of(best, y, t);
            else o[u + i] = y;
          }
        }
      }
    }
  }
  if (CHOOSE) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    const int parts = (int)cluster.num_blocks();
    __shared__ Best warps[LG_THREADS / 32], ctas[8];
    const int warp = tid >> 5, lane = tid & 31;
    auto warp_best = [&]() {
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best.v, d);
        const int i = __shfl_xor_sync(0xffffffffu, best.i, d);
        best_of(best, v, i);
      }
    };
    warp_best();
    if (lane == 0) warps[warp] = best;
    __syncthreads();
    if (parts > 1) cluster.sync();  // every CTA of the cluster runs before its shared memory is written from outside
    if (warp == 0) {
      best = lane < LG_THREADS / 32 ? warps[lane] : Best{-INFINITY, 0};
      warp_best();
      if (lane == 0) *(parts > 1 ? cluster.map_shared_rank(&ctas[part], 0) : &ctas[0]) = best;
    }
    if (parts > 1) cluster.sync();
    if (part == 0 && tid == 0) {
      best = ctas[0];
      for (int k = 1; k < parts; ++k) best_of(best, ctas[k].v, ctas[k].i);
      const int at = *take.pos, to = at + take.ahead - take.base;
      if (live) {
        take.current[row] = best.i;
        if (to >= 0 && to < take.buf_rows) take.buf[(long long)to * take.rows + row] = best.i;
        const int len = length_of[row];
        if (len >= 0 && len < r.length) r.history[row * r.length + len] = best.i;
      }
      if (take.advance) {
        __threadfence();  // every row has read the position before the last one moves it
        if (atomicAdd(take.counter, 1u) == (unsigned int)take.rows - 1) {
          *take.counter = 0;
          *take.pos = at + 1;
        }
      }
    }
  }
}

__global__ void append_tokens_kernel(int* history, const int* tokens, const int* pos, const int* count, int T, int length) {
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int b = blockIdx.y, p = pos[b], n = min(count[b], T);
  for (int t = blockIdx.x * blockDim.x + threadIdx.x; t < n; t += gridDim.x * blockDim.x)
    if (p + t >= 0 && p + t < length) history[(long long)b * length + p + t] = tokens[(long long)b * T + t];
}

bool rules_ok(const LogitRulesArgs& r, int valid) {
  return r.slots >= 1 && r.length >= 1 && r.length <= (int)LG_TIMES && r.biases >= 0 && r.biases <= LG_MAX_BIASES &&
         (long long)r.words * 32 >= valid && r.history && r.start && r.penalties && r.allowed &&
         (r.biases == 0 || (r.bias_tokens && r.bias_values));
}

// entries of one part: whole groups of 16 bytes of logits, whatever their type
int part_size(int valid, int parts) { return ((valid + 8 + parts - 1) / parts + 31) / 32 * 32; }

template <typename T, bool CHOOSE>
int launch(const void* logits, float* out, const int* slot, const int* length, const LogitRulesArgs& r, int rows, int V, int valid,
           int parts, const ShapedTake& take, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)parts, (unsigned)rows, 1);
  cfg.blockDim = dim3(LG_THREADS, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CHOOSE ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logits_kernel<T, CHOOSE>, (const T*)logits, out, slot, length, r, V, valid,
                                           part_size(valid, parts), take);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

// logits (rows, V), 16-byte aligned -> out (rows, V) fp32, 16-byte aligned. slot, length (rows). Rules by slot: history (slots, L)
// with L < 2^20, start (slots), penalties (slots, 3), bias lists (slots, biases <= 1024), allowed (slots, words) with words * 32 >= V.
// At most 65535 rows.
XL_API int xl_shape_logits(const void* logits, float* out, const int* slot, const int* length, const int* history, const int* start,
                           const float* penalties, const int* bias_tokens, const float* bias_values, const void* allowed, int rows,
                           int V, int slots, int L, int biases, int words, int dtype, cudaStream_t s) {
  const LogitRulesArgs r{const_cast<int*>(history), start, penalties, bias_tokens, bias_values, (const uint32_t*)allowed,
                         slots, L, biases, words};
  if (rows < 1 || rows > 65535 || V < 1 || V > 0x7fff0000 || !slot || !length || !rules_ok(r, V)) return -1;
  if (((uintptr_t)logits | (uintptr_t)out) & 15) return -1;
  // one group of entries per thread is enough work; no more CTAs than four per SM together
  int parts = 1;
  while (parts < 32 && V > LG_THREADS * 4 * parts && (long long)rows * parts * 2 <= 4 * 148) parts *= 2;
  XL_DISPATCH_DTYPE(dtype, T, { return launch<T, false>(logits, out, slot, length, r, rows, V, V, parts, ShapedTake{}, s); });
  return -1;
}

// The choice of every row b of logits (rows, V) among its first `valid` entries under the rules of slot b, after length[b] tokens:
// it becomes current[b], buf[*pos + ahead - base][b] (buf: (buf_rows, rows)) and history[b][length[b]] where there is such a place.
// Rows with count[b] <= 0 are left out. With `advance` *pos moves on by one. counter: a zero-initialised word (left zeroed).
XL_API int xl_take_shaped(const void* logits, int* current, int* buf, int* pos, const int* length, const int* count, int* history,
                          const int* start, const float* penalties, const int* bias_tokens, const float* bias_values,
                          const void* allowed, unsigned int* counter, int rows, int V, int valid, int buf_rows, int base, int ahead,
                          int advance, int L, int biases, int words, int dtype, cudaStream_t s) {
  const LogitRulesArgs r{history, start, penalties, bias_tokens, bias_values, (const uint32_t*)allowed, rows, L, biases, words};
  if (rows < 1 || rows > 65535 || valid < 1 || valid > V || V > 0x7fff0000 || !current || !buf || !pos || !length || !count ||
      !counter || !rules_ok(r, valid) || ((uintptr_t)logits & 15))
    return -1;
  int parts = 1;
  while (parts < 8 && valid > LG_THREADS * 4 * parts && (long long)rows * parts * 2 <= 4 * 148) parts *= 2;
  const ShapedTake take{current, buf, pos, count, buf_rows, base, ahead, advance, rows, counter};
  XL_DISPATCH_DTYPE(dtype, T, { return launch<T, true>(logits, nullptr, nullptr, length, r, rows, V, valid, parts, take, s); });
  return -1;
}

// tokens (B * T): the first count[b] of each sequence go to history[b][pos[b] ...] where there is such a place.
XL_API int xl_append_tokens(int* history, const int* tokens, const int* pos, const int* count, int B, int T, int length, cudaStream_t s) {
  if (B < 1 || B > 65535 || T < 1 || length < 1) return -1;
  const cudaError_t e = xl_launch_overlapped(append_tokens_kernel, dim3((T + 255) / 256 < 32 ? (T + 255) / 256 : 32, B), dim3(256), (size_t)0,
                                             s, history, tokens, pos, count, T, length);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
