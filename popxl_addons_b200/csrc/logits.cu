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
// entry. The words that are not zero go through the formula by themselves, from a list (a quotient takes some sixty instructions, and with
// one entry in seventy on the list a third of all warps would take them for every entry); the pass over the row then takes the word or
// the logit, and its mask bit. Sums and quotients are rounded one by one (no contraction), so the results are those of the formula in 32
// bits, and ties stay ties.
#include "common.cuh"

#include <cooperative_groups.h>
#include <math.h>

namespace {

constexpr int LG_THREADS = 256;
constexpr int LG_CHUNK = 8192;        // entries of the vocabulary that a CTA holds at a time, at most
constexpr int LG_MAX_BIASES = 1024;
// word of an entry: bit 31 seen in the prompt, bits 20 .. 30 one more than the place of its bias in the list, bits 0 .. 19 times since
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

__device__ __forceinline__ float shaped(float x, uint32_t word, float repetition, float frequency, float presence, const float* bias_sum) {
  const uint32_t times = word & LG_TIMES, k = (word & ~LG_SEEN) >> LG_BIAS_SHIFT;
  if ((word & LG_SEEN) || times) x = x > 0.f ? __fdiv_rn(x, repetition) : __fmul_rn(x, repetition);
  if (times) x = __fsub_rn(__fsub_rn(x, __fmul_rn(frequency, (float)times)), presence);
  return k ? __fadd_rn(x, bias_sum[k - 1]) : x;
}

// mask words of `chunk` entries from anywhere in a word, and one behind them; whole pieces of 16 bytes
__host__ __device__ __forceinline__ int mask_room(int chunk) { return (chunk / 32 + 7) / 4 * 4; }

// What the choice does with its token (see xl_take_shaped).
struct ShapedTake {
  int *current, *buf, *pos;
  const int* count;
  int buf_rows, base, ahead, advance, rows;
  unsigned int* counter;
};

// Grid (parts, rows). Entries are numbered from the 16-byte boundary at or before the row's first logit (`phase` entries earlier),
// so that groups of N entries are whole 16-byte pieces of the logits; a part is a whole number of groups, taken `chunk` entries at a time.
// CHOOSE: the parts of a row are a cluster, whose winners meet in the first CTA.
// What bounds it is latency: a row's scalars, its tokens, the count, the logits. The logits go to shared memory by asynchronous copies
// that are asked for first, and the first eight tokens of every thread at once with the scalars that say how many there are. With
// the logits in registers four CTAs fitted an SM and 96 rows of 50400 took two waves. 96 rows of 50400 fp32 logits, 2048 tokens, 64 biases:
// 16.5 us (the bytes alone: 6); the choice from 48 rows in bf16: 12.4; one row of 32000: 4.1.
template <typename T, bool CHOOSE>
__global__ void __launch_bounds__(LG_THREADS)
    logits_kernel(const T* logits, float* out, const int* slot_of, const int* length_of, const LogitRulesArgs r, int V, int valid,
                  int per_part, int chunk, const ShapedTake take) {
  constexpr int N = XlVec<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  uint32_t* words = reinterpret_cast<uint32_t*>(smem);                      // [chunk]
  T* held_logits = reinterpret_cast<T*>(words + chunk);                     // [chunk]
  uint32_t* masks = reinterpret_cast<uint32_t*>(held_logits + chunk);       // [mask_room] from the word of the first entry on
  int* tokens = reinterpret_cast<int*>(masks + mask_room(chunk));           // [biases rounded up to 4], read four at a time
  float* values = reinterpret_cast<float*>(tokens + (r.biases + 3) / 4 * 4);  // [biases]
  float* sums = values + r.biases;                                            // [biases]
  uint16_t* changed = reinterpret_cast<uint16_t*>(sums + r.biases);           // [changes_room] entries whose word is not zero
  __shared__ int changes;
  const int part = blockIdx.x, tid = threadIdx.x;
  const long long row = blockIdx.y;
  const int phase = (int)((row * V) % N);
  const int u_end = phase + valid, u0 = part * per_part, u1 = min(u0 + per_part, u_end);
  auto clear = [&](int n) {
    for (int i = tid * 4; i < n; i += LG_THREADS * 4) *reinterpret_cast<uint4*>(words + i) = make_uint4(0u, 0u, 0u, 0u);
  };
  clear(chunk);
  if (tid == 0) changes = 0;
  xl_grid_dependency_wait();
  if (!CHOOSE) xl_grid_launch_dependents();
  const T* p = logits + row * V - phase;
  float* o = CHOOSE ? nullptr : out + row * V - phase;
  auto whole = [&](int u) { return u >= phase && u + N <= u_end; };  // groups inside the row
  auto fetch = [&](int c0, int c1) {
    for (int u = c0 + tid * N; u < c1; u += LG_THREADS * N) {
      if (whole(u)) xl_cp_async16(held_logits + (u - c0), p + u, true);
      else  // the row's first and last group
        for (int i = u; i < min(u + N, c1); ++i)
          if (i >= phase) held_logits[i - c0] = p[i];
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const bool live = !CHOOSE || take.count[row] > 0;
  if (u0 < u1) fetch(u0, min(u0 + chunk, u1));
  const int slot = CHOOSE ? (int)row : slot_of[row];
  const bool ruled = slot >= 0 && slot < r.slots;
  Best best{-INFINITY, 0};
  if (live) {
    constexpr int EARLY = 8;
    float repetition = 1.f, frequency = 0.f, presence = 0.f;
    int held = 0, start = 0, biases = 0, early[EARLY];
    const int* past = r.history + (long long)(ruled ? slot : 0) * r.length;
    const uint32_t* mask = r.allowed + (long long)(ruled ? slot : 0) * r.words;
    auto fetch_masks = [&](int c0, int c1) {
      const int first = max(c0 - phase, 0) >> 5, last = (c1 - 1 - phase) >> 5;
      for (int i = tid; i <= last - first; i += LG_THREADS) masks[i] = mask[first + i];
      if (tid == 0) masks[last - first + 1] = 0u;  // read by a group that ends with the row, for nothing
    };
    if (ruled) {
      if (u0 < u1) fetch_masks(u0, min(u0 + chunk, u1));
#pragma unroll
      for (int q = 0; q < EARLY; ++q) early[q] = tid + q * LG_THREADS < r.length ? past[tid + q * LG_THREADS] : -1;
      repetition = r.penalties[slot * 3];
      frequency = r.penalties[slot * 3 + 1];
      presence = r.penalties[slot * 3 + 2];
      held = max(0, min(length_of[row], r.length));
      start = r.start[slot];
      biases = r.biases;
      for (int k = tid; k < biases; k += LG_THREADS) {
        tokens[k] = r.bias_tokens[(long long)slot * biases + k];
        values[k] = r.bias_values[(long long)slot * biases + k];
      }
      for (int k = biases + tid; k < (biases + 3) / 4 * 4; k += LG_THREADS) tokens[k] = -1;
      if (repetition == 1.f && frequency == 0.f && presence == 0.f) held = 0;  // nothing that the tokens would change
    }
    __syncthreads();
    for (int c0 = u0; c0 < u1; c0 += chunk) {
      const int c1 = min(c0 + chunk, u1);
      if (c0 > u0) {
        __syncthreads();
        fetch(c0, c1);
        if (ruled) fetch_masks(c0, c1);
        clear(c1 - c0);
        if (tid == 0) changes = 0;
        __syncthreads();
      }
      const int lo = c0 - phase, n = c1 - c0;  // token of the first word (negative before the row), words
      auto count = [&](int i, int t) {  // whoever finds a word at zero puts it on the list
        const unsigned w = (unsigned)(t - lo);
        if (t >= 0 && w < (unsigned)n) {
          const uint32_t old = i >= start ? atomicAdd(words + w, 1u) : atomicOr(words + w, LG_SEEN);
          if (old == 0) changed[atomicAdd(&changes, 1)] = (uint16_t)w;
        }
      };
      if (held > 0) {
#pragma unroll
        for (int q = 0; q < EARLY; ++q)
          if (tid + q * LG_THREADS < held) count(tid + q * LG_THREADS, early[q]);
#pragma unroll 8
        for (int i = tid + EARLY * LG_THREADS; i < held; i += LG_THREADS) count(i, past[i]);
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
                sum = __fadd_rn(sum, values[q + e]);
              }
          }
          if (first) {
            sums[k] = sum;
            if (atomicOr(words + w, (uint32_t)(k + 1) << LG_BIAS_SHIFT) == 0) changed[atomicAdd(&changes, 1)] = (uint16_t)w;
          }
        }
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncthreads();
      // the words that are not zero become the shaped logits, inverted: then no number is zero (all ones is one of the NaN)
      for (int i = tid; i < changes; i += LG_THREADS) {
        const int w = changed[i];
        const uint32_t y = __float_as_uint(shaped(xl_to_float(held_logits[w]), words[w], repetition, frequency, presence, sums));
        words[w] = y != 0xffffffffu ? ~y : 0x80000000u;
      }
      __syncthreads();
#pragma unroll 2
      for (int u = c0 + tid * N; u < c1; u += LG_THREADS * N) {
        const int e0 = u - phase;  // token of the group's first entry
        const bool all = whole(u);
        uint32_t bits = 0xffffffffu;
        if (ruled) {
          const int e1 = max(e0, 0), w = (e1 >> 5) - (max(lo, 0) >> 5);
          bits = __funnelshift_r(masks[w], masks[w + 1], e1 & 31) << (e1 - e0);
        }
        float x[N];
        xl_load16(held_logits + (u - c0), x);
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const uint4 w = *reinterpret_cast<const uint4*>(words + (u - c0) + i);
          const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            x[i + k] = word[k] ? __uint_as_float(~word[k]) : x[i + k];
            x[i + k] = (bits >> (i + k)) & 1u ? x[i + k] : -INFINITY;
          }
        }
        if (CHOOSE) {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (all || (e0 + i >= 0 && e0 + i < valid)) best_of(best, x[i], e0 + i);
        } else if (all) {
#pragma unroll
          for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(o + u + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i)
            if (e0 + i >= 0 && e0 + i < valid) o[u + i] = x[i];
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
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
  const int per_part = part_size(valid, parts), chunk = per_part < LG_CHUNK ? per_part : LG_CHUNK;
  const int room = r.length + r.biases < chunk ? r.length + r.biases : chunk;  // entries that tokens and biases can name
  const int bytes = chunk * (4 + (int)sizeof(T)) + mask_room(chunk) * 4 + (r.biases + 3) / 4 * 4 * 12 + (room + 7) / 8 * 16;
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(logits_kernel<T, CHOOSE>, bytes, smem));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)parts, (unsigned)rows, 1);
  cfg.blockDim = dim3(LG_THREADS, 1, 1);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)parts;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CHOOSE ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, logits_kernel<T, CHOOSE>, (const T*)logits, out, slot, length, r, V, valid, per_part,
                                           chunk, take);
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
  // about 4096 entries of a row for a CTA, or fewer (one group of entries per thread is enough work) while that is no more than four CTAs
  // per SM
  const int chunk = 4096;
  int parts = 1;
  while (parts < 32 && V > LG_THREADS * 4 * parts && (long long)rows * parts * 2 <= 4 * 148) parts *= 2;
  if (parts < (V + chunk - 1) / chunk) parts = min((V + chunk - 1) / chunk, 1024);
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
