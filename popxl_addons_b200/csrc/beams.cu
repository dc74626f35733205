// Beam search: the best continuations of a group of beams, and the states that follow them.
//
//   c(k, v) = score_k + x_kv - M_k - log sum_v exp(x_kv - M_k)     beam k of a group goes on with token v; M_k: the largest of its row
//   c(k, end) = score_k                                            the only continuation of a beam that has ended
//   the K largest c / tokens^penalty of the K V ones of a group; of equal ones the lowest k, then the lowest v
//
// Nothing but reading the logits once bounds this, so a row is cut into parts until there are some CTAs for every SM, and a part leaves
// its maximum, its sum and its K largest entries. No part needs more than that: its (K + 1)st entry has K better ones. The CTA of a group that
// arrives last merges. Which entries a part keeps: of its first 4096 entries every thread has 16, and the K-th largest of the threads' maxima
// is a bound that K entries reach; the few entries that reach it go to a list, those of later chunks if they pass it, and the list is
// ranked at the end. A list that grows long (sorted or equal logits) is cut to its K best between two chunks.
//
// 48 x 8 beams of 50400 entries: 42.5 us (77 MB, 1.8 TB/s), 16 x 16 of 32000 in bf16: 31 us (each 768 CTAs, of which 740 run at a time); one prompt's 4 beams of 32000: 15 us, dependent loads and
// barriers.
//
// Continuations are compared in 64 bits. Within a row that takes no more than the logits; between rows it takes the logarithms of sums over 50000
// entries each. Those are first formed from exponentials in 32 bits, 16 of them added in 32 bits and the rest in 64 (off by 2e-6 at most,
// 5e-8 as a rule). Where the choice hangs on less than that, the last CTA forms the sums of the rows concerned again with exponentials in 64
// bits, in an order that does not depend on where a row lies, and merges once more: equal rows are equal.
// That is rare, and takes 35 us for a row of 50400 entries.
#include "common.cuh"

#include <math.h>

namespace {

constexpr int BM_THREADS = 256;
constexpr int BM_EACH = 16;                       // entries of a thread in a chunk
constexpr int BM_CHUNK = BM_THREADS * BM_EACH;
constexpr int BM_MAX_BEAMS = 32;
constexpr double BM_MAX_PENALTY = 32.0;           // any number of tokens to this power is finite
constexpr int BM_MAX_PARTS = 16;                  // each part costs the merge its loads
constexpr int BM_KEEP = 512;                      // a longer list is cut to its best between two chunks
constexpr int BM_MERGED = 2048;                   // entries that the parts of a group leave, at most
constexpr int BM_GROUP = 4;                       // threads whose largest entry counts as one for the bound

template <typename V> __device__ __forceinline__ bool better(V a, int i, V b, int j) { return a > b || (a == b && i < j); }

// The `most` best of n entries in shared memory, in order, to best_v / best_i (elsewhere in shared memory). Returns how many there are.
// All threads call it, the entries are in place for all of them before, and the results are after.
template <typename V> __device__ int best_of_list(const V* v, const int* id, int n, int most, V* best_v, int* best_i) {
  const int tid = threadIdx.x;
  if (n <= 2 * BM_THREADS) {
    for (int e = tid; e < n; e += BM_THREADS) {
      const V mine = v[e];
      const int at = id[e];
      int rank = 0;
#pragma unroll 2
      for (int o = 0; o < n; ++o) rank += better(v[o], id[o], mine, at) ? 1 : 0;
      if (rank < most) {
        best_v[rank] = mine;
        best_i[rank] = at;
      }
    }
    __syncthreads();
    return min(n, most);
  }
  __shared__ V top_v[BM_THREADS / 32];
  __shared__ int top_i[BM_THREADS / 32];
  V last = (V)INFINITY;
  int last_i = -1;
  for (int r = 0; r < most; ++r) {  // the best entry behind the last one
    V bv = (V)-INFINITY;
    int bi = 0x7fffffff;
    for (int e = tid; e < n; e += BM_THREADS)
      if (better(last, last_i, v[e], id[e]) && better(v[e], id[e], bv, bi)) { bv = v[e]; bi = id[e]; }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const V ov = __shfl_xor_sync(0xffffffffu, bv, d);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, d);
      if (better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
    }
    if ((tid & 31) == 0) { top_v[tid >> 5] = bv; top_i[tid >> 5] = bi; }
    __syncthreads();
    last = top_v[0];
    last_i = top_i[0];
    for (int w = 1; w < BM_THREADS / 32; ++w)
      if (better(top_v[w], top_i[w], last, last_i)) { last = top_v[w]; last_i = top_i[w]; }
    if (tid == 0) { best_v[r] = last; best_i[r] = last_i; }
    __syncthreads();
  }
  return most;
}

// A bound that at least `most` (up to 64) of the threads' values reach (-inf where fewer than that are finite): the `most`-th largest of the maxima of
// BM_GROUP threads each. (Of all threads: 1.1 us of every CTA instead of 0.2, for a list that is hardly shorter.)
template <typename V> __device__ V bound_of(V mine, int most, V* room, V* result) {
  constexpr int GROUPS = BM_THREADS / BM_GROUP;
  const int tid = threadIdx.x;
#pragma unroll
  for (int d = 1; d < BM_GROUP; d <<= 1) {
    const V other = __shfl_xor_sync(0xffffffffu, mine, d);
    mine = other > mine ? other : mine;
  }
  if (tid % BM_GROUP == 0) room[tid / BM_GROUP] = mine;
  __syncthreads();
  if (tid < GROUPS) {
    const V own = room[tid];
    int rank = 0;
#pragma unroll 4
    for (int o = 0; o < GROUPS; ++o) rank += better(room[o], o, own, tid) ? 1 : 0;
    if (rank == most - 1) *result = own;
  }
  __syncthreads();
  return *result;
}

// the next lower number (of what is finite)
__device__ __forceinline__ float below(float x) {
  const int i = __float_as_int(x);
  return !isfinite(x) ? x : x > 0.f ? __int_as_float(i - 1) : x < 0.f ? __int_as_float(i + 1) : __int_as_float((int)0x80000001u);
}
// e^d for d <= 0 (or d = -inf): the rounding of d * log2(e) is made good, the rest is the special-function unit's (2^-22 relative)
__device__ __forceinline__ float exp_below(float d) {
  constexpr float HI = 1.44269502f, LO = 1.92596299e-8f;  // of log2(e)
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(fmaf(d, HI, d * LO)));
  return y;
}

struct BeamArgs {
  const float* scores;
  const int *ended, *length;
  const int* rule_end;          // what `end` and `penalty` are, if the device holds them, else null
  const double* rule_penalty;
  float* to_scores;
  int *to_ended, *to_length;
  int *current, *parent, *buf, *parents, *step;
  float4* stats;  // [rows][parts]: maximum, sum, entries kept
  float* part_v;  // [rows][parts][beams]
  int* part_i;
  unsigned int* counters;  // [groups + 1], zero between launches
  int rows, V, valid, beams, parts, per_part, end, buf_rows, base, ahead, advance;
  double penalty;
  double slack;  // how far the logarithm of a row's sum may be off, see xl_take_beams
};

// the token that ends a beam, or a negative number
__device__ __forceinline__ int end_of(const BeamArgs& a) {
  int end = a.end;
  if (a.rule_end) end = *a.rule_end;
  return end < a.valid ? end : -1;
}

// A sum of exponentials relative to `m` as one relative to `now`, the larger one: rare, and out of the way of the loop's registers.
__device__ __noinline__ double rescaled(double sum, float m, float now) { return m > -INFINITY ? sum * exp((double)m - (double)now) : 0.0; }

// The sum over a row of e^(x - top), in 64 bits and in an order that only depends on the number of entries, for all threads.
template <typename T> __device__ __noinline__ double exact_sum(const T* row, int valid, double top, double* room) {
  constexpr int AHEAD = 8;
  double sum = 0.0;
#pragma unroll 1
  for (long long v = threadIdx.x; v < valid; v += AHEAD * BM_THREADS) {
    float x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) x[i] = v + i * BM_THREADS < valid ? fmaxf(xl_to_float(row[v + i * BM_THREADS]), -INFINITY) : -INFINITY;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) sum += exp((double)x[i] - top);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = sum;
  __syncthreads();
  sum = 0.0;
  for (int w = 0; w < BM_THREADS / 32; ++w) sum += room[w];
  return sum;
}

template <typename T> __global__ void __launch_bounds__(BM_THREADS, 5) take_beams_kernel(const T* logits, const BeamArgs a) {
  constexpr int N = XlVec<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float best_v[BM_MAX_BEAMS];
  __shared__ int best_i[BM_MAX_BEAMS], listed;
  __shared__ float tau_s, warp_m[BM_THREADS / 32];
  __shared__ double warp_s[BM_THREADS / 32];
  __shared__ unsigned int is_last;
  float* list_v = reinterpret_cast<float*>(smem);         // [BM_CHUNK + BM_KEEP]
  int* list_i = reinterpret_cast<int*>(list_v + BM_CHUNK + BM_KEEP);
  const int tid = threadIdx.x, part = blockIdx.x, row = blockIdx.y, K = a.beams, group = row / K;
  if (tid == 0) listed = 0;
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const bool live = isfinite(a.scores[row]) && !(end_of(a) >= 0 && a.ended[row] != 0);
  __syncthreads();
  if (live) {
    const T* p = logits + (long long)row * a.V;
    const int phase = (int)(((uintptr_t)p & 15) / sizeof(T));  // places are counted from the 16-byte boundary before the row
    const int u0 = max(part * a.per_part, phase), u1 = min((part + 1) * a.per_part, a.valid + phase);
    p -= phase;
    float m = -INFINITY, tau = -INFINITY;  // m: of the warp; tau: entries above it go to the list
    double sum = 0.0;
    constexpr int LOADS = BM_EACH / N;
    uint4 raw[LOADS];
    auto fetch = [&](int c0) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int u = c0 + (i * BM_THREADS + tid) * N;
        if (u >= u0 && u + N <= u1) raw[i] = __ldcs(reinterpret_cast<const uint4*>(p + u));
      }
    };
    bool first = true;
    const int begin = part * a.per_part;
    if (begin < u1) fetch(begin);
#pragma unroll 1
    for (int c0 = begin; c0 < u1; c0 += BM_CHUNK) {
      float x[BM_EACH];
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        const int u = c0 + (i * BM_THREADS + tid) * N;
        const T* e = reinterpret_cast<const T*>(&raw[i]);
        const bool whole = u >= u0 && u + N <= u1;  // else the first or the last group of the part, or none of it
#pragma unroll
        for (int k = 0; k < N; ++k) {
          x[i * N + k] = -INFINITY;
          if (whole) x[i * N + k] = fmaxf(xl_to_float(e[k]), -INFINITY);  // NaN: minus infinity
        }
        if (!whole && u + N > u0 && u < u1)
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (u + k >= u0 && u + k < u1) x[i * N + k] = fmaxf(xl_to_float(p[u + k]), -INFINITY);
      }
      if (c0 + BM_CHUNK < u1) fetch(c0 + BM_CHUNK);  // under way while these are looked at
      float top = x[0];
#pragma unroll
      for (int i = 1; i < BM_EACH; ++i) top = fmaxf(top, x[i]);
      const float now = fmaxf(m, xl_warp_max(top));
      if (now > m) {
        sum = rescaled(sum, m, now);
        m = now;
      }
      if (m > -INFINITY) {
        float e[BM_EACH];
#pragma unroll
        for (int i = 0; i < BM_EACH; ++i) e[i] = exp_below(x[i] - m);
#pragma unroll
        for (int w = BM_EACH / 2; w; w >>= 1)
#pragma unroll
          for (int i = 0; i < w; ++i) e[i] += e[i + w];
        sum += (double)e[0];
      }
      // of the first chunk entries that reach the bound, of later ones those that pass it: equal ones have K before them
      float bound = tau;
      if (first) {
        tau = bound_of(top, K, list_v, &tau_s);  // (the list is empty)
        bound = below(tau);
      }
      first = false;
      int places = 0;
      if (top > bound) {
        unsigned int hits = 0;
#pragma unroll
        for (int i = 0; i < BM_EACH; ++i) hits |= x[i] > bound ? 1u << i : 0u;
        places = atomicAdd(&listed, __popc(hits));
        int at = places;
#pragma unroll
        for (int i = 0; i < BM_EACH; ++i)
          if (hits >> i & 1) {
            list_v[at] = x[i];
            list_i[at++] = c0 + (i / N * BM_THREADS + tid) * N + i % N - phase;
          }
        places = at;
      }
      if (__syncthreads_or(places > BM_KEEP) && c0 + BM_CHUNK < u1) {  // (the same for all threads, and nobody adds before all are here)
        const int kept = best_of_list(list_v, list_i, listed, K, best_v, best_i);
        if (tid < kept) {
          list_v[tid] = best_v[tid];
          list_i[tid] = best_i[tid];
        }
        tau = best_v[K - 1];
        if (tid == 0) listed = K;
        __syncthreads();
      }
    }
    // ---- the part's maximum and sum, and its best entries -----------------------------------------------------------------------
    const int kept = best_of_list(list_v, list_i, listed, K, best_v, best_i);
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if ((tid & 31) == 0) {
      warp_m[tid >> 5] = m;
      warp_s[tid >> 5] = sum;
    }
    __syncthreads();
    const long long at = (long long)row * a.parts + part;
    if (tid < kept) {
      __stcg(a.part_v + at * K + tid, best_v[tid]);
      __stcg(a.part_i + at * K + tid, best_i[tid]);
    }
    if (tid < 32) {
      constexpr int WARPS = BM_THREADS / 32;
      const float pm = xl_warp_max(tid < WARPS ? warp_m[tid] : -INFINITY);
      sum = tid < WARPS && warp_m[tid] > -INFINITY ? warp_s[tid] * exp((double)warp_m[tid] - (double)pm) : 0.0;
#pragma unroll
      for (int d = WARPS / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      const float up = (float)sum;  // and what it leaves
      if (tid == 0) __stcg(a.stats + at, make_float4(pm, up, (float)(sum - (double)up), __int_as_float(kept)));
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) is_last = atomicAdd(a.counters + group, 1u) == (unsigned int)(K * a.parts) - 1;
  __syncthreads();
  if (!is_last) return;
  __threadfence();

  // ---- the group's last CTA: continuations of all its beams ---------------------------------------------------------------------------
  __shared__ double top[BM_MAX_BEAMS], log_sum[BM_MAX_BEAMS], divisor[BM_MAX_BEAMS], score[BM_MAX_BEAMS], chosen_rank[BM_MAX_BEAMS], tau_d;
  __shared__ double slack[BM_MAX_BEAMS];
  __shared__ unsigned int doubt;  // rows whose sums have to be better than they are
  __shared__ int chosen[BM_MAX_BEAMS], state[BM_MAX_BEAMS], after[BM_MAX_BEAMS], slot_of[BM_MAX_BEAMS], row_of[BM_MAX_BEAMS];  // state 0: no beam, 1: live, 2: ended, 3: no beam, but marked as ended
  const int row0 = group * K;
  double* room = reinterpret_cast<double*>(smem);  // [BM_THREADS] for the bound
  const int end = end_of(a);
  double penalty = a.penalty;
  if (a.rule_penalty) penalty = *a.rule_penalty;
  if (!(fabs(penalty) <= BM_MAX_PENALTY)) penalty = 0.0;
  if (tid < K) {
    const float f = a.scores[row0 + tid];
    const bool ended = end >= 0 && a.ended[row0 + tid] != 0;
    state[tid] = !isfinite(f) ? (ended ? 3 : 0) : ended ? 2 : 1;
    score[tid] = (double)f;
    after[tid] = a.length[row0 + tid] + (ended ? 0 : 1);
    divisor[tid] = penalty == 0.0 ? 1.0 : pow((double)max(after[tid], 1), penalty);
    slack[tid] = state[tid] == 1 ? a.slack / divisor[tid] : 0.0;  // (the only continuation of an ended beam has the sum that the beam has)
  }
  if (tid == 0) doubt = 0;
  __syncthreads();
  {  // maxima and sums of all rows side by side
    const int lanes = K <= 8 ? 32 : K <= 16 ? 16 : 8, k = tid / lanes, lane = tid & (lanes - 1);
    const bool on = k < K && state[min(k, K - 1)] == 1;
    const float4* st = a.stats + (long long)(row0 + k) * a.parts;
    float m = -INFINITY;
    for (int q = lane; on && q < a.parts; q += lanes) m = fmaxf(m, __ldcg(&st[q]).x);
    for (int d = lanes / 2; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    double sum = 0.0;
#pragma unroll 1
    for (int q = lane; on && q < a.parts; q += lanes) {
      const float4 x = __ldcg(&st[q]);
      if (x.x > -INFINITY) sum += ((double)x.y + (double)x.z) * (x.x == m ? 1.0 : exp((double)x.x - (double)m));
    }
    for (int d = lanes / 2; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (on && lane == 0) {
      top[k] = (double)m;
      log_sum[k] = log(sum);
    }
  }
  __syncthreads();
  // the sum that beam k has with an entry x; where its row has no finite largest entry: not a number, or minus infinity
  auto with = [&](int k, float x) { return score[k] + (((double)x - top[k]) - log_sum[k]); };
  // 2^n lanes for the entries of one row and part, several of these for a warp at a time
  const int parts_all = a.parts * K;
  double* all_r = room + BM_THREADS;  // [BM_MERGED] ranks, then [BM_MERGED] entries
  int* all_i = reinterpret_cast<int*>(all_r + BM_MERGED);
  __shared__ int at_list;
  double widest = 0.0;
  for (int k = 0; k < K; ++k) widest = fmax(widest, slack[k]);
  int found;
#pragma unroll 1
  for (bool again = false;; again = true) {
    double most = -INFINITY;
    {
      int lanes = 1;
      while (lanes < K) lanes *= 2;
      const int at = tid & (lanes - 1), stride = BM_THREADS / lanes;
      int from = tid / lanes, k = from / a.parts, q = from - k * a.parts;
#pragma unroll 2
      for (; from < parts_all; from += stride) {
        if (at < K) {
          double r = -INFINITY;
          int flat = 0;
          if (state[k] == 1) {
            const long long place = (long long)(row0 + k) * a.parts + q;
            const float kept = __ldcg(&a.stats[place].w), x = __ldcg(a.part_v + place * K + at);
            const int v = __ldcg(a.part_i + place * K + at);
            if (at < __float_as_int(kept)) {
              r = with(k, x);
              if (penalty != 0.0) r /= divisor[k];
              flat = k * a.valid + v;
            }
          } else if (state[k] == 2 && q == 0 && at == 0) {
            r = score[k] / divisor[k];
            flat = k * a.valid + end;
          }
          if (!isfinite(r)) r = -INFINITY;
          all_r[from * K + at] = r;
          all_i[from * K + at] = flat;
          most = r > most ? r : most;
        }
        for (q += stride; q >= a.parts; q -= a.parts) ++k;
      }
    }
    const double tau = bound_of(most, K, room, &tau_d);
    // The list takes the place of the ranks that have been looked at: no more entries are before an entry than in front of it.
    if (tid == 0) at_list = 0;
    __syncthreads();
#pragma unroll 1
    for (int e0 = 0; e0 < parts_all * K; e0 += BM_THREADS) {
      const int e = e0 + tid;
      const double r = e < parts_all * K ? all_r[e] : -INFINITY;
      const int flat = e < parts_all * K ? all_i[e] : 0;
      __syncthreads();
      if (r >= tau - 2.0 * widest && r > -INFINITY) {
        const int at = atomicAdd(&at_list, 1);
        all_r[at] = r;
        all_i[at] = flat;
      }
      __syncthreads();
    }
    found = best_of_list(all_r, all_i, at_list, K, chosen_rank, chosen);
    if (again) break;
    // Continuations of different rows, one of them chosen, that are closer than the logarithms of their sums are known. (Two that are neither chosen
    // nor as close as that to one that is need no order.)
    if (tid < found) row_of[tid] = chosen[tid] / a.valid;
    __syncthreads();
#pragma unroll 1
    for (int e = tid; e < at_list; e += BM_THREADS) {
      const int k = all_i[e] / a.valid;
      const double r = all_r[e];
      unsigned int rows = 0;
      for (int j = 0; j < found; ++j) {
        const int o = row_of[j];
        if (o != k && fabs(r - chosen_rank[j]) <= slack[k] + slack[o]) rows |= 1u << k | 1u << o;
      }
      if (rows) atomicOr(&doubt, rows);
    }
    __syncthreads();
    bool better_sums = false;
    for (unsigned int rows = doubt; rows; rows &= rows - 1) {
      const int k = __ffs(rows) - 1;
      if (state[k] != 1) continue;
      const double sum = exact_sum(logits + (long long)(row0 + k) * a.V, a.valid, top[k], chosen_rank);
      if (tid == 0) log_sum[k] = log(sum);
      better_sums = true;
    }
    if (!better_sums) break;
    __syncthreads();
  }
  bool any = false;
  for (int k = 0; k < K; ++k) any |= state[k] == 1 || state[k] == 2;
  if (any) {
    if (found < K) {
      if (tid == 0)
        for (int n = found, i = 0; n < K; ++i) {  // too few: those at minus infinity follow, the lowest first
          bool in = false;
          for (int j = 0; j < found; ++j) in |= chosen[j] == i;
          if (!in) chosen[n++] = i;
        }
      __syncthreads();
    }
    if (tid < 32) {  // slots by rank: the beam's own for its best continuation, the spare ones in order for others
      const unsigned int all = K == 32 ? ~0u : (1u << K) - 1, mine = 1u << tid;
      const int k = tid < K ? chosen[tid] / a.valid : -1;
      const unsigned int same = __match_any_sync(0xffffffffu, k);
      const unsigned int spare = ~__reduce_or_sync(0xffffffffu, k >= 0 ? 1u << k : 0u) & all;
      const bool again = k >= 0 && (same & (mine - 1));
      const unsigned int others = __ballot_sync(0xffffffffu, again);
      if (k >= 0) slot_of[tid] = again ? (int)__fns(spare, 0, __popc(others & (mine - 1)) + 1) : k;
    }
    __syncthreads();
    if (tid < K) {
      const int k = chosen[tid] / a.valid, token = chosen[tid] - k * a.valid, to = row0 + slot_of[tid];
      double c = -INFINITY;
      if (tid < found) c = state[k] == 2 ? score[k] : with(k, xl_to_float(logits[(long long)(row0 + k) * a.V + token]));
      a.to_scores[to] = (float)c;
      a.to_ended[to] = state[k] >= 2 || token == end;
      a.to_length[to] = after[k];
      a.current[to] = token;
      a.parent[to] = row0 + k;
      const int at = *a.step + a.ahead - a.base;
      if (at >= 0 && at < a.buf_rows) {
        a.buf[(long long)at * a.rows + to] = token;
        a.parents[(long long)at * a.rows + to] = row0 + k;
      }
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    a.counters[group] = 0;
    if (a.advance && atomicAdd(a.counters + a.rows / K, 1u) == (unsigned int)(a.rows / K) - 1) {  // every group has read the step
      a.counters[a.rows / K] = 0;
      *a.step += 1;
    }
  }
}

template <typename T> int launch_take(const void* logits, const BeamArgs& a, cudaStream_t s) {
  const int bytes = (BM_CHUNK + BM_KEEP) * 8;
  static_assert(BM_THREADS * 8 + BM_MERGED * 12 <= (BM_CHUNK + BM_KEEP) * 8, "the merge has room in the list");
  const cudaError_t e = xl_launch_overlapped(take_beams_kernel<T>, dim3(a.parts, a.rows), dim3(BM_THREADS), (size_t)bytes, s, (const T*)logits, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Into how many parts a row is cut: about six CTAs for every SM, of which five run at a time (384 rows of 50400 entries: 1 part 50 us, 2 parts 43).
int parts_of(int rows, int beams, int valid) {
  int parts = 6 * 148 / rows < 1 ? 1 : 6 * 148 / rows;
  if (parts > (valid + 2047) / 2048) parts = (valid + 2047) / 2048;
  if (parts > BM_MERGED / (beams * beams)) parts = BM_MERGED / (beams * beams);
  return parts < BM_MAX_PARTS ? parts : BM_MAX_PARTS;
}

// ---- reordering of states ---------------------------------------------------------------------------------------------------
// A CTA takes a span of one state, group and outer index. A thread takes the same 16 bytes of all rows of the group that move: it
// has them all before it writes the first, so that rows may be read and written in any pattern, without a copy elsewhere. Bytes bound it: each
// distinct source once, each moved row once. 32 x 8 beams, 8 layers of 8 heads of 128, up to 230 positions: 944 MB in 156 to 172 us (5.5 to 6.1 TB/s).
constexpr int RO_MAX_STATES = 64;
constexpr int RO_THREADS = 256;

struct ReorderState {
  uint8_t* base;
  long long row_bytes, outer_bytes;  // from one row to the next, from one outer index to the next
  int outer, entries, unit, per;     // outer indexes, entries along the positions, bytes of one, positions of one (0: no positions)
  int piece;                         // bytes that a thread moves at a time: what alignment allows
};
struct ReorderArgs {
  ReorderState state[RO_MAX_STATES];
  int first[RO_MAX_STATES + 1];  // CTAs of the states before, along x
  const int *parent, *begin, *end;
  int states, rows, beams;
};

template <typename P, int K>
__device__ __forceinline__ void move_pieces(uint8_t* base, long long row_bytes, const int* dst, const int* src, const long long* lo, const long long* hi,
                                            int moved, long long from, long long to) {
  for (long long at = from + (long long)threadIdx.x * sizeof(P); at < to; at += (long long)RO_THREADS * sizeof(P)) {
    P v[K];
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < moved && at >= lo[i] && at < hi[i]) v[i] = *reinterpret_cast<const P*>(base + src[i] * row_bytes + at);
#pragma unroll
    for (int i = 0; i < K; ++i)
      if (i < moved && at >= lo[i] && at < hi[i]) *reinterpret_cast<P*>(base + dst[i] * row_bytes + at) = v[i];
  }
}

template <int K> __global__ void __launch_bounds__(RO_THREADS) reorder_kernel(const __grid_constant__ ReorderArgs a) {
  __shared__ int dst[BM_MAX_BEAMS], src[BM_MAX_BEAMS], moved;
  __shared__ long long lo[BM_MAX_BEAMS], hi[BM_MAX_BEAMS];  // bytes of the moved rows that move
  int t = 0;
  while (t + 1 < a.states && (int)blockIdx.x >= a.first[t + 1]) ++t;
  const ReorderState& st = a.state[t];
  const int item = blockIdx.x - a.first[t], group = item / st.outer, outer = item - group * st.outer;
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  if (threadIdx.x < 32) {
    const int k = threadIdx.x, row = group * a.beams + k;
    int from = row;
    long long l = 0, h = 0;
    if (k < a.beams) {
      from = a.parent[row];
      if (from < group * a.beams || from >= (group + 1) * a.beams) from = row;
      h = st.entries;
      if (st.per) {
        const int b = max(a.begin[row], 0), e = max(a.end[row], 0);
        l = b / st.per;
        h = b < e ? min((long long)st.entries, ((long long)e + st.per - 1) / st.per) : 0;
      }
    }
    const unsigned int moves = __ballot_sync(0xffffffffu, from != row && l < h);
    const int at = __popc(moves & ((1u << k) - 1));
    if (moves >> k & 1) {
      dst[at] = row;
      src[at] = from;
      lo[at] = l * st.unit;
      hi[at] = h * st.unit;
    }
    if (k == 0) moved = __popc(moves);
  }
  __syncthreads();
  const int n = moved;
  if (n == 0) return;
  long long from = lo[0], to = hi[0];
  for (int i = 1; i < n; ++i) {
    from = min(from, lo[i]);
    to = max(to, hi[i]);
  }
  // the span of this CTA among those of the same item, in whole pieces
  const long long pieces = (to - from) / st.piece, p0 = pieces * blockIdx.y / gridDim.y, p1 = pieces * (blockIdx.y + 1) / gridDim.y;
  to = from + p1 * st.piece;
  from += p0 * st.piece;
  uint8_t* base = st.base + outer * st.outer_bytes;
  switch (st.piece) {
    case 16: move_pieces<uint4, K>(base, st.row_bytes, dst, src, lo, hi, n, from, to); break;
    case 8: move_pieces<uint2, K>(base, st.row_bytes, dst, src, lo, hi, n, from, to); break;
    case 4: move_pieces<uint32_t, K>(base, st.row_bytes, dst, src, lo, hi, n, from, to); break;
    case 2: move_pieces<uint16_t, K>(base, st.row_bytes, dst, src, lo, hi, n, from, to); break;
    default: move_pieces<uint8_t, K>(base, st.row_bytes, dst, src, lo, hi, n, from, to);
  }
}

template <int K> int launch_reorder(const ReorderArgs& a, int slices, cudaStream_t s) {
  const cudaError_t e = xl_launch_overlapped(reorder_kernel<K>, dim3(a.first[a.states], slices), dim3(RO_THREADS), (size_t)0, s, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

}  // namespace

XL_API int xl_take_beams_parts(int rows, int beams, int valid) {
  return rows < 1 || beams < 1 || beams > BM_MAX_BEAMS || valid < 1 ? 0 : parts_of(rows, beams, valid);
}

// logits (rows, V), of which the first `valid` entries count; rows are groups of `beams`. scores, ended, length (rows) -> to_* (rows, may be the same).
// The choices become current, parent (rows) and row *step + ahead - base of buf, parents (buf_rows, rows); with `advance` *step moves on. end < 0: no beam
// ends. scratch: rows * parts * (16 + 8 beams) bytes, 16-byte aligned, with parts = xl_take_beams_parts; counters: rows / beams + 1 zero-initialised
// words (left zeroed). rule_end, rule_penalty: both null, or one number each that is read instead of `end` and `penalty`.
XL_API int xl_take_beams(const void* logits, const float* scores, const int* ended, const int* length, float* to_scores, int* to_ended,
                         int* to_length, int* current, int* parent, int* buf, int* parents, int* step, void* scratch, unsigned int* counters,
                         const int* rule_end, const double* rule_penalty, int rows, int V, int valid, int beams, int end, double penalty, int buf_rows, int base, int ahead, int advance, int dtype,
                         cudaStream_t s) {
  if (rows < 1 || rows > 65535 || beams < 1 || beams > BM_MAX_BEAMS || rows % beams || valid < 1 || valid > V || V > 0x7fff0000 ||
      (long long)valid * beams > 0x7fffffffLL || end >= valid || !scores || !ended || !length || !to_scores || !to_ended || !to_length ||
      !current || !parent || !buf || !parents || !step || !scratch || !rule_end != !rule_penalty || ((uintptr_t)rule_penalty & 7) || ((uintptr_t)scratch & 15) || !counters)
    return -1;
  BeamArgs a = {};
  a.scores = scores; a.ended = ended; a.length = length; a.to_scores = to_scores; a.to_ended = to_ended; a.to_length = to_length;
  a.current = current; a.parent = parent; a.buf = buf; a.parents = parents; a.step = step; a.counters = counters;
  a.rule_end = rule_end; a.rule_penalty = rule_penalty;
  a.rows = rows; a.V = V; a.valid = valid; a.beams = beams; a.end = end; a.buf_rows = buf_rows; a.base = base; a.ahead = ahead;
  a.advance = advance; a.penalty = penalty;
  // What a sum's logarithm may be off, relative errors of the sum: a difference x - m and its product with log2(e) are rounded to 2^-24 of themselves,
  // together 2^-23 |x - m| of the exponential, on average over the sum at most 2^-23 log(entries); the exponential itself 2^-22, four sums in 32 bits 2^-22.
  a.slack = ldexp(4.0 + log((double)valid), -23);
  a.parts = parts_of(rows, beams, valid);
  a.per_part = ((valid + 8 + a.parts - 1) / a.parts + 31) / 32 * 32;  // whole 16 bytes of any type, with room for a row that starts off a boundary
  a.stats = (float4*)scratch;
  a.part_v = (float*)(a.stats + (long long)rows * a.parts);
  a.part_i = (int*)(a.part_v + (long long)rows * a.parts * beams);
  XL_DISPATCH_DTYPE(dtype, T, {
    if ((uintptr_t)logits % sizeof(T)) return -1;
    return launch_take<T>(logits, a, s);
  });
  return -1;
}

// states: n descriptions of 7 numbers each: address, bytes from row to row, outer indexes, bytes from one to the next, entries along the
// positions, bytes of an entry, positions of an entry (0: the state has none). parent, begin, end (rows). n <= 64.
XL_API int xl_reorder(const long long* states, int n, const int* parent, const int* begin, const int* end, int rows, int beams, cudaStream_t s) {
  if (n < 1 || n > RO_MAX_STATES || rows < 1 || beams < 1 || beams > BM_MAX_BEAMS || rows % beams || !parent || !begin || !end) return -1;
  ReorderArgs a = {};
  a.parent = parent; a.begin = begin; a.end = end; a.states = n; a.rows = rows; a.beams = beams;
  long long items = 0, most = 0;
  for (int i = 0; i < n; ++i) {
    const long long* d = states + 7 * i;
    if (!d[0] || d[1] < 1 || d[2] < 1 || d[4] < 1 || d[4] > 0x7fffffffLL || d[5] < 1 || d[5] > 0x7fffffffLL || d[6] < 0 || d[6] > 0x7fffffffLL) return -1;
    ReorderState& st = a.state[i];
    st.base = (uint8_t*)d[0];
    st.row_bytes = d[1]; st.outer_bytes = d[3];
    st.outer = (int)d[2]; st.entries = (int)d[4]; st.unit = (int)d[5]; st.per = (int)d[6];
    const unsigned long long all = (unsigned long long)d[0] | d[1] | d[3] | d[5];
    st.piece = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : all % 2 == 0 ? 2 : 1;
    a.first[i] = (int)items;
    items += d[2] * (rows / beams);
    if (d[2] > 0x7fffffffLL || items > 0x7fffffffLL) return -1;
    if (d[4] * d[5] > most) most = d[4] * d[5];
  }
  a.first[n] = (int)items;
  // spans of 16 KB or more of the longest state, while there are no more than about eight CTAs per SM
  int slices = 1;
  while (slices < 64 && items * slices * 2 <= 8 * 148 && most / (2 * slices) >= 16384) slices *= 2;
  if (beams <= 4) return launch_reorder<4>(a, slices, s);
  if (beams <= 8) return launch_reorder<8>(a, slices, s);
  if (beams <= 16) return launch_reorder<16>(a, slices, s);
  return launch_reorder<32>(a, slices, s);
}
