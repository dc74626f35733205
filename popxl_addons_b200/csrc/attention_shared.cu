// Sliding-window attention where the first positions of a sequence lie in the cache of another slot (attention_window.cuh): beams of one
// prompt, requests behind one system prompt. Same mathematics and layouts as attention_window.cu.
//
//   xl_shared_append           new keys (norms in 64 bits, rounded to 32 and then to the type) and values into the caches; for the general kernel queries in fp32
//   xl_shared_attn_groups      few rows per sequence, bf16: the keys that a group of sequences shares, once for the group, on the tensor cores
//                              (tcgen05), and behind it the sum of its parts
//   xl_shared_attn_portion     portions of many rows per sequence on the tensor cores, bf16
//   xl_shared_attn_general     any sizes and types (attention_window.cu)
//
// Queries enter the products as two bf16 numbers, value and rounding error, as the weights do: a rounded query would move every score by
// 2^-9 of itself, more than all other roundings together.
#include "attention_decode.cuh"
#include "attention_window.cuh"
#include "tcgen05.cuh"

#include <math.h>

namespace {

using namespace xl_tc;

constexpr int SA_MAX_DIM = 512;

// Waits as in tcgen05.cuh, in loops that are not unrolled: code that is run for the first time comes from L2, 128 bytes at a time, and these kernels
// are short.
__device__ __forceinline__ bool bar_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
#pragma unroll 1
  for (uint32_t i = 0; i < MBAR_SPIN_LIMIT; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 1023u) == 1023u && *abort_flag) return false;
  }
  *abort_flag = 1;
  if (err) atomicCAS(err, 0, code);
  return false;
}
__device__ __forceinline__ bool bar_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err, int code) {
#pragma unroll 1
  for (uint32_t i = 0; i < MBAR_SPIN_LIMIT; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 1023u) == 1023u && __any_sync(0xffffffffu, *abort_flag)) return false;
  }
  *abort_flag = 1;
  if (err) atomicCAS(err, 0, code);
  return false;
}

// ---- new keys and values ------------------------------------------------------------------------------------------------------
// One CTA per row, a warp per head. What it reads and the kernels behind it write was complete or is no longer read when it lets them start: they
// may do all but look at the new keys and values at once. Latency bounds it, so a head's key, weights and value are all under way before position and
// count are looked at, V features at a time (4 where sizes and addresses allow, else 1). 4 us for 128 rows of 8 heads, 20 us for 4000 rows (33 MB;
// 33 us with one feature at a time and values before keys).
template <typename T, int V>
struct alignas(sizeof(T) * V) Features {
  T v[V];
};

template <typename T, int V>
__global__ void __launch_bounds__(256)
    shared_append_kernel(const T* proj, long long ld, const float* wq, const float* wk, float* qn, T* kc, T* vc, const int* pos, const int* count,
                         int T_len, int H, int G, int dim, int vdim, int Smax, float eps) {
  using Raw = Features<T, V>;
  using Real = Features<float, V>;
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int b = blockIdx.y, t = blockIdx.x, at = pos[b], n = count[b];
  const T* row = proj + ((long long)b * T_len + t) * ld;
  const int R = H / G, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int NP = SA_MAX_DIM / (32 * V);
  for (int h = qn ? warp : H + warp; h < H + G; h += blockDim.x >> 5) {
    const T* head = row + (long long)h * dim;
    const T* value = row + (long long)(H + G) * dim + (long long)(h - H) * vdim;
    const float* weight = h < H ? wq : wk;
    Raw x[NP], val[NP];
    Real w[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (lane + 32 * i) * V;
      if (c < dim) x[i] = *(const Raw*)(head + c), w[i] = *(const Real*)(weight + c);
      if (h >= H && c < vdim) val[i] = *(const Raw*)(value + c);
    }
    if (t >= n || !window_fits(at, n, T_len, Smax)) return;
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if ((lane + 32 * i) * V < dim)
#pragma unroll
        for (int e = 0; e < V; ++e) sq += (double)xl_to_float(x[i].v[e]) * (double)xl_to_float(x[i].v[e]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const double f = 1.0 / sqrt(sq / dim + (double)eps);
    const long long entry = h < H ? (((long long)b * G + h / R) * T_len + t) * R + h % R : ((long long)b * G + (h - H)) * Smax + at + t;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (lane + 32 * i) * V;
      Real y;
      Raw r;
      if (c < dim) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          y.v[e] = (float)((double)xl_to_float(x[i].v[e]) * f * (double)w[i].v[e]);
          r.v[e] = xl_from_float<T>(y.v[e]);
        }
        if (h < H) *(Real*)(qn + entry * dim + c) = y;
        else *(Raw*)(kc + entry * dim + c) = r;
      }
      if (h >= H && c < vdim) *(Raw*)(vc + entry * vdim + c) = val[i];
    }
  }
}

// ---- portions on the tensor cores -----------------------------------------------------------------------------------------------
// The R query heads that read one key / value head are consecutive rows (token-major). A CTA owns 256 of these rows as two tiles of 128
// and walks the keys visible to any of them in blocks of 128: those of the lead, then its own ones. Key and value tiles serve both row
// tiles, which take turns on the tensor cores while the other one's softmax runs:
//   warp 0       TMA: key and value tiles in turn through one ring
//   warp 1       MMA: S_m = Q_m K^T into TMEM (both halves of the queries), then O_m += P_m V
//   warps 4..7   tile 0, warps 8..11 tile 1: norms of the queries, from the projections straight to shared memory; then the softmax, one thread
//                per row, running maximum and sum in fp32, lazy rescaling of O_m in TMEM (warps 2, 3: none)
// P replaces S in TMEM as two bf16 numbers per weight. Keys beyond a range, and those that no row of the tiles sees, are masked in the scores, and their
// values are zeroed in shared memory: they belong to others, and a weight of zero times anything that is not finite would reach the sum.
//
// TMEM columns: [0, 128) S_0 / P_0, [128, 256) S_1 / P_1, [256, 256 + VD) O_0, [256 + VD, 256 + 2 VD) O_1. One CTA per SM. Every wait is
// bounded (see tcgen05.cuh).
//
// The chain of a tile bounds this: scores, softmax, product. 16 x 250 tokens behind 4000, 32 heads on 8 of 128: 562 us by itself, 569 with the append (448 TFLOP/s
// of 255 GFLOP; the two numbers of queries and weights make it twice that in the tensor cores). 7700 clocks for a block of both tiles, 4096 of them products.
// Two tiles, since a tile's softmax then has the other's products to run under, and keys are read half as often.
constexpr int TILE_M = 128;
constexpr int BKV = 128;
constexpr int UMMA_K = 16;
constexpr int SA_THREADS = 128 + 2 * 128;
constexpr uint32_t TMEM_COLS = 512;
// Registers of a thread of a kernel that holds rows of scores: of the first warpgroup, which only issues, and of the two others (together what the
// launch gives, 384 x 168: with 168 each the rows spilled). The settings stand at the head of branches that only join again at the end: behind a join the
// smaller one would hold.
constexpr int REGS_CONTROL = 72, REGS_SOFTMAX = 216;
static_assert(REGS_CONTROL + 2 * REGS_SOFTMAX <= 3 * 168, "more than the launch gives would never be granted");
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

enum { ERR_Q = 111, ERR_KV_FULL = 112, ERR_KV_EMPTY = 113, ERR_S = 114, ERR_P = 115, ERR_PV = 116, ERR_MEET = 117, ERR_TABLE = 118, ERR_ROOM = 119 };

struct SharedParams {
  const __nv_bfloat16* proj;
  long long ld;
  const float* wq;
  const int *pos, *count;
  SharedPrefix prefix;
  __nv_bfloat16* out;
  long long ldo;
  int B, T, H, G, dim, vdim, Smax, window, keep_first, gated;
  float scale, sink, eps;
  int* err;
};

// DK, VD: 64 or 128, features of queries and values rounded up. Features past the real sizes are zero in the query tiles (and what TMA fills in
// for those of keys and values), so they add nothing.
template <int DK, int VD> struct SharedTiles {
  static constexpr int Q_HALF = TILE_M * DK * 2;                     // DK/64 blocks of (128 rows x 128 B)
  static constexpr int Q_BYTES = 2 * Q_HALF;                         // values, then rounding errors
  static constexpr int K_BYTES = BKV * DK * 2;
  static constexpr int V_BYTES = BKV * VD * 2;                       // 2 blocks of VD/64 boxes of (64 rows x 128 B)
  static constexpr int SLOT = K_BYTES > V_BYTES ? K_BYTES : V_BYTES;
};

// Rows of a tile by `warps` warps, of which this is number `i`, as two K-major operands of 128-byte swizzle: copied as they are to where their rounded
// values will be, all of them under way together, and then normalised. Loops are not unrolled: code that runs once is fetched from L2 as slowly as the
// rows are. `row(r)`: where the projections have the head of row r of the tile (rows of an even number of passes), or null.
template <int DK, typename F>
__device__ __forceinline__ void load_queries(uint8_t* tile, int i, int warps, int end, const F& row, const float* wq, int dim, float eps) {
  constexpr int LANES = DK / 8, ROWS = 32 / LANES;  // lanes of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % LANES;
  const bool on = chunk * 8 < dim;
  auto place = [&](int r) { return tile + (chunk >> 3) * (TILE_M * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4); };
#pragma unroll 1
  for (int r0 = i * ROWS; r0 < end; r0 += warps * ROWS) {
    const int r = r0 + lane / LANES;
    const __nv_bfloat16* src = on ? row(r) : nullptr;
    dd_cp16_zfill(place(r), src ? src + chunk * 8 : (const __nv_bfloat16*)wq, src != nullptr);
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  const float per = 1.f / dim;
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = on ? wq[chunk * 8 + e] : 0.f;
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();
#pragma unroll 1
  for (int r0 = i * ROWS; r0 < end; r0 += warps * ROWS) {
    uint8_t* dst = place(r0 + lane / LANES);
    float x[8], lo[8], sq = 0.f;
    xl_load16<__nv_bfloat16>(reinterpret_cast<const __nv_bfloat16*>(dst), x);
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += x[e] * x[e];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float f = rsqrtf(fmaf(sq, per, eps));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f * w[e];
    const uint4 hi = pack8_16bit(x, false);
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[2 * e] = x[2 * e] - dd_lo(h[e]);
      lo[2 * e + 1] = x[2 * e + 1] - dd_hi(h[e]);
    }
    *reinterpret_cast<uint4*>(dst) = hi;
    *reinterpret_cast<uint4*>(dst + TILE_M * DK * 2) = pack8_16bit(lo, false);
  }
}

// Descriptors of a product's steps differ by whole 16 bytes of address, which stay inside the address field. The first one is hidden from the
// compiler, which would keep those of all steps in registers across the loop over blocks.
__device__ __forceinline__ uint64_t first_desc(uint32_t addr, uint32_t lbo_bytes) {
  uint64_t d = make_smem_desc(addr, lbo_bytes);
  asm volatile("" : "+l"(d));
  return d;
}

// steps of 16 keys that a block of `keys` has
__device__ __forceinline__ int key_steps(int keys) { return (min(keys, BKV) + UMMA_K - 1) / UMMA_K; }

// S_m = Q K^T, both halves of the queries, for `steps` times 16 keys
template <int DK> __device__ __forceinline__ void issue_score_product(uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr, int steps) {
  // bf16 operands, fp32 accumulator, both K-major, N = 16 steps
  const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(2 * steps) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
  const uint64_t dq = first_desc(q_addr, 16), dk = first_desc(k_addr, 16);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int kb = 0; kb < DK / 64; ++kb)
#pragma unroll
      for (int k = 0; k < 64 / UMMA_K; ++k)
        tcgen05_mma_f16(tmem_s, dq + ((half * (TILE_M * DK * 2) + kb * (TILE_M * 128) + k * (UMMA_K * 2)) >> 4),
                        dk + ((kb * (BKV * 128) + k * (UMMA_K * 2)) >> 4), idesc, (half | kb | k) ? 1u : 0u);
}

// O_m (+)= P V, both halves of the weights, over `steps` times 16 keys
template <int VD> __device__ __forceinline__ void issue_value_product(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr, bool add, int steps) {
  // A (P) from TMEM, B (V) MN-major (bit 16), N = VD
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(VD >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
  const uint64_t dv = first_desc(v_addr, 8192);
#pragma unroll
  for (int k = 0; k < BKV / UMMA_K; ++k) {
    if (k == steps) break;
#pragma unroll
    for (int half = 0; half < 2; ++half)
      tcgen05_mma_f16_ts(tmem_o, tmem_p + (k >> 1) * 32 + half * 16 + (k & 1) * (UMMA_K / 2),
                         dv + (((k >> 2) * (VD / 64) * 8192 + (k & 3) * (UMMA_K * 128)) >> 4), idesc, (add || half || k) ? 1u : 0u);
  }
}

// the lowest n bits (n may be anything)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }
// Keys 32 w .. 32 w + 31 of a block that begins at key0 which a row sees: below `end`, and from `lo` on or below `keep`.
__device__ __forceinline__ uint32_t visible_bits(int key0, int w, int end, int lo, int keep) {
  const int k = key0 + 32 * w;
  return low_bits(end - k) & (~low_bits(lo - k) | low_bits(keep - k));
}

// Which keys of a block a row sees; `unknown`: keys whose scores are not numbers, by 32 of them, or null.
struct RowMask {
  bool cut;  // some row of the warp does not see them all: the same for all lanes, which vote where it holds
  int key0, end, lo, keep;
  const uint32_t* unknown;
};

// 32 scores of a row, masked
__device__ __forceinline__ void masked_scores(uint32_t taddr, const RowMask& mask, int w, float (&s)[32]) {
  uint32_t raw[32];
  tmem_ld_32x32b_x32(taddr + w * 32, raw);
  tmem_ld_wait();
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(raw[i]);
  if (mask.cut) {
    const uint32_t visible = visible_bits(mask.key0, w, mask.end, mask.lo, mask.keep);
    if (mask.unknown) {
      const uint32_t unknown = mask.unknown[w];
#pragma unroll
      for (int i = 0; i < 32; ++i) s[i] = unknown >> i & 1 ? NAN : s[i];
    }
    if (!__all_sync(0xffffffffu, visible == 0xffffffffu)) {
#pragma unroll
      for (int i = 0; i < 32; ++i) s[i] = visible >> i & 1 ? s[i] : -INFINITY;
    }
  }
}

// One block's scores (in units of 1 / scale) of a row become weights in their place, 32 at a time: 16 columns of pairs of bf16 numbers, and 16 of their
// rounding errors. mx, l: running maximum and sum; c = scale * log2(e). Returns the factor of what O holds: the maximum moves only when an exponent
// would exceed 2^8, as a rule with the first scores of a row, and then what is stored of the block follows. A short loop: a row of 128 scores in
// registers took 1500 instructions, whose first run cost 6000 cycles.
__device__ __forceinline__ float weigh(uint32_t tmem_s, const RowMask& mask, int steps, float& mx, float& l, float c) {
  float alpha = 1.f, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int w = 0; w < (steps + 1) / 2; ++w) {  // (scores behind the steps are those of another block: masked)
    float s[32];
    masked_scores(tmem_s, mask, w, s);
    float top[4] = {s[0], s[1], s[2], s[3]};  // chains of their own
#pragma unroll
    for (int i = 4; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
    const float m_new = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
    const bool move = m_new > -INFINITY && (mx == -INFINITY || (m_new - mx) * c > 8.f);
    if (__any_sync(0xffffffffu, move)) {
      const float f = move && mx != -INFINITY ? fast_exp2((mx - m_new) * c) : 1.f;
      if (move) mx = m_new;
      alpha *= f;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] *= f;
      if (w && __any_sync(0xffffffffu, f != 1.f)) {
        tmem_st_wait();
#pragma unroll 1
        for (int v = 0; v < w; ++v) {
          uint32_t pairs[32];
          tmem_ld_32x32b_x32(tmem_s + v * 32, pairs);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float x = (dd_lo(pairs[i]) + dd_lo(pairs[16 + i])) * f, y = (dd_hi(pairs[i]) + dd_hi(pairs[16 + i])) * f;
            pairs[i] = dd_pack(x, y);
            pairs[16 + i] = dd_pack(x - dd_lo(pairs[i]), y - dd_hi(pairs[i]));
          }
          tmem_st_32x32b_x32(tmem_s + v * 32, pairs);
        }
      }
    }
    const float mc = mx == -INFINITY ? 0.f : mx * c;  // a row without a visible key yet keeps weight 0
    uint32_t pairs[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      s[i] = fast_exp2(fmaf(s[i], c, -mc));
      sum[i & 3] += s[i];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      pairs[i] = dd_pack(s[2 * i], s[2 * i + 1]);
      pairs[16 + i] = dd_pack(s[2 * i] - dd_lo(pairs[i]), s[2 * i + 1] - dd_hi(pairs[i]));
    }
    tmem_st_32x32b_x32(tmem_s + w * 32, pairs);
  }
  l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
  return alpha;
}

// The same with the whole row in registers: more code, and less time for each block where there are many (16 x 250 tokens behind 4000: 630 -> 583 us).
// The maximum from before the block serves for all of the row.
__device__ __forceinline__ float weigh_row(uint32_t tmem_s, const RowMask& mask, float& mx, float& l, float c) {
  float s[BKV];
#pragma unroll
  for (int w = 0; w < BKV / 32; ++w) {
    float part[32];
    masked_scores(tmem_s, mask, w, part);
#pragma unroll
    for (int i = 0; i < 32; ++i) s[w * 32 + i] = part[i];
  }
  float top[4] = {s[0], s[1], s[2], s[3]}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 4; i < BKV; ++i) top[i & 3] = fmaxf(top[i & 3], s[i]);
  const float m_blk = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
  const bool move = m_blk > -INFINITY && (mx == -INFINITY || (m_blk - mx) * c > 8.f);
  const float alpha = move && mx != -INFINITY ? fast_exp2((mx - m_blk) * c) : 1.f;
  if (move) mx = m_blk;
  const float mc = mx == -INFINITY ? 0.f : mx * c;
#pragma unroll
  for (int w = 0; w < BKV / 32; ++w) {
    uint32_t pairs[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      float& x = s[w * 32 + i];
      x = fast_exp2(fmaf(x, c, -mc));
      sum[i & 3] += x;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float x = s[w * 32 + 2 * i], y = s[w * 32 + 2 * i + 1];
      pairs[i] = dd_pack(x, y);
      pairs[16 + i] = dd_pack(x - dd_lo(pairs[i]), y - dd_hi(pairs[i]));
    }
    tmem_st_32x32b_x32(tmem_s + w * 32, pairs);
  }
  l = l * alpha + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
  return alpha;
}

template <int VD> __device__ __forceinline__ void rescale_output(uint32_t tmem_o, float alpha) {
#pragma unroll 1
  for (int ch = 0; ch < VD / 32; ++ch) {
    uint32_t raw[32];
    tmem_ld_32x32b_x32(tmem_o + ch * 32, raw);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) raw[i] = __float_as_uint(__uint_as_float(raw[i]) * alpha);
    tmem_st_32x32b_x32(tmem_o + ch * 32, raw);
  }
}

// piece i (of eight) of the 64-feature block jn of value row r in shared memory; neighbouring rows' pieces of one number lie in different banks
template <int VD> __device__ __forceinline__ uint4* value_piece(uint8_t* tile, int r, int jn, int i) {
  return reinterpret_cast<uint4*>(tile + ((r >> 6) * (VD / 64) + jn) * 8192 + (r & 63) * 128) + ((i + r) & 7);
}
template <int VD> __device__ __forceinline__ void clear_value_row(uint8_t* tile, int r) {
#pragma unroll 1
  for (int jn = 0; jn < VD / 64; ++jn)
#pragma unroll 4
    for (int i = 0; i < 8; ++i) *value_piece<VD>(tile, r, jn, i) = make_uint4(0u, 0u, 0u, 0u);
}
// The rows of a block of `keys` keys that the product's last step reads behind them, by the 128 threads of a warpgroup.
template <int VD> __device__ __forceinline__ void clear_step_rest(uint8_t* tile, int keys, int thread) {
  const int rows = key_steps(keys) * UMMA_K - keys;
#pragma unroll 1
  for (int i = thread; i < rows * (VD / 8); i += 128) {
    const int r = keys + i / (VD / 8), piece = i % (VD / 8);
    *value_piece<VD>(tile, r, piece >> 3, piece & 7) = make_uint4(0u, 0u, 0u, 0u);
  }
}
template <int VD> __device__ __forceinline__ bool finite_value_row(uint8_t* tile, int r) {
  bool finite = true;
#pragma unroll 1
  for (int jn = 0; jn < VD / 64; ++jn)
#pragma unroll 4
    for (int i = 0; i < 8; ++i) {
      const uint4 v = *value_piece<VD>(tile, r, jn, i);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) finite &= (w[e] & 0x7f80u) != 0x7f80u && (w[e] & 0x7f800000u) != 0x7f800000u;
    }
  return finite;
}

struct KeyRange {
  int slot, begin, end;
};
// The keys that rows at positions p_first .. p_last of sequence b see, as up to four ranges of the lead's and its own cache, in blocks of BKV.
struct KeyRanges {  // in shared memory
  KeyRange r[4];
  int until[4];  // blocks of the ranges up to and with this one
  int kept, first;  // the keys from `kept` to `first` are seen by no row, though blocks may have them
};
__device__ __forceinline__ int key_blocks(int begin, int end) { return begin < end ? (end - begin + BKV - 1) / BKV : 0; }
__device__ __forceinline__ void set_ranges(KeyRanges& k, int b, int lead, int edge, int p_first, int p_last, int window, int keep_first) {
  WindowRange seen = window_range(p_first, window, keep_first);
  const int all = key_blocks(0, edge) + key_blocks(edge, p_last + 1);
  const int visible = key_blocks(0, min(seen.kept, edge)) + key_blocks(seen.first, edge) + key_blocks(edge, seen.kept) +
                      key_blocks(max(seen.first, edge), p_last + 1);
  k.kept = seen.kept;
  k.first = seen.first;
  if (visible >= all) seen = {0, 0};  // leaving keys out saves no block
  k.r[0] = {lead, 0, min(seen.kept, edge)};
  k.r[1] = {lead, seen.first, edge};
  k.r[2] = {b, edge, seen.kept};
  k.r[3] = {b, max(seen.first, edge), p_last + 1};
  int n = 0;
  for (int i = 0; i < 4; ++i) k.until[i] = n += key_blocks(k.r[i].begin, k.r[i].end);
}
// whether a block of keys from `begin` on has some that no row sees
__device__ __forceinline__ bool has_unseen(int begin, int end, int kept, int first) { return begin < first && end > kept; }
// slot, first key, and end of the range, of block j
__device__ __forceinline__ KeyRange key_block(const KeyRanges& k, int j) {
  int i = 0;
  while (i < 3 && j >= k.until[i]) ++i;
  const KeyRange x = k.r[i];
  return {x.slot, x.begin + (j - (i ? k.until[i - 1] : 0)) * BKV, x.end};
}

template <int DK, int VD> struct PortionSmem : SharedTiles<DK, VD> {
  using L = SharedTiles<DK, VD>;
  static constexpr int SLOTS = L::SLOT > 16384 ? 3 : 6;
  static constexpr int TILE_BYTES = 2 * L::Q_BYTES + SLOTS * L::SLOT;
  static constexpr int NEEDED = TILE_BYTES + 1024 /*alignment*/ + 256 /*barriers*/;
  // more than half of an SM's shared memory: two CTAs, each holding all of TMEM, never meet on an SM
  static constexpr int TOTAL = NEEDED > 120 * 1024 ? NEEDED : 120 * 1024;
};

template <int DK, int VD>
__global__ void __launch_bounds__(SA_THREADS, 1)
    shared_attn_portion_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedParams p) {
  using L = PortionSmem<DK, VD>;
  static_assert(L::TOTAL <= 227 * 1024, "shared memory");
  constexpr int SLOTS = L::SLOTS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* ring = smem + 2 * L::Q_BYTES;
  uint64_t* bars = (uint64_t*)(smem + L::TILE_BYTES);
  uint64_t* q_full = bars;         // [2] per tile
  uint64_t* s_full = bars + 2;     // [2]
  uint64_t* p_full = bars + 4;     // [2]
  uint64_t* pv_done = bars + 6;    // [2]
  uint64_t* full = bars + 8;       // [SLOTS]
  uint64_t* empty = bars + 8 + SLOTS;
  uint32_t* tmem_base_slot = (uint32_t*)(bars + 8 + 2 * SLOTS);
  volatile int* abort_flag = (volatile int*)(tmem_base_slot + 1);
  KeyRanges& keys = *(KeyRanges*)(tmem_base_slot + 2);
  static_assert((8 + 2 * SLOTS) * 8 + 8 + sizeof(KeyRanges) <= 256, "room behind the tiles");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x, b = blockIdx.z, R = p.H / p.G;
  const int cnt = min(p.count[b], p.T), pos = p.pos[b];
  const long long rows = (long long)cnt * R;                                  // real rows of this sequence and key / value head
  const long long f0 = (long long)(gridDim.y - 1 - blockIdx.y) * 2 * TILE_M;  // the blocks with the most keys first
  if (f0 >= rows || !window_fits(pos, cnt, p.T, p.Smax)) {
    xl_grid_dependency_wait();
    return;
  }
  const int tiles = f0 + TILE_M < rows ? 2 : 1;
  const int p_first = pos + (int)(f0 / R), p_last = pos + (int)((min(rows, f0 + 2 * TILE_M) - 1) / R);
  int lead;
  const int edge = shared_edge(p.prefix, p.pos, b, pos, p.B, lead);
  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 4);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
    }
    for (int s = 0; s < 2 * SLOTS; ++s) mbar_init(&full[s], 1);
    set_ranges(keys, b, lead, edge, p_first, p_last, p.window, p.keep_first);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    tmem_alloc(tmem_base_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;
  const int n_kv = keys.until[3];

  if (warp < 4) {
    fewer_registers<REGS_CONTROL>();
    if (warp == 0 && lane == 0) {
      xl_grid_dependency_wait();    // the new keys and values; nothing else here depends on the kernel that appends them
      xl_grid_launch_dependents();  // TMEM is held: a successor that allocates some on this SM cannot come first
      bool ok = true;
      int issued = 0;
      for (int n = 0; n < 2 * n_kv && ok; ++n) {  // key tile of block 0, value tile of block 0, key tile of block 1, ...
        const int st = n % SLOTS;
        const KeyRange x = key_block(keys, n >> 1);
        const int row = (x.slot * p.G + g) * p.Smax + x.begin;
        if (n >= SLOTS) ok = bar_wait(&empty[st], (uint32_t)(n / SLOTS - 1) & 1u, abort_flag, p.err, ERR_KV_EMPTY);
        if (!ok) break;
        uint8_t* dst = ring + st * L::SLOT;
        if (n & 1) {
          mbar_expect_tx(&full[st], L::V_BYTES);
#pragma unroll
          for (int kk = 0; kk < BKV / 64; ++kk)
#pragma unroll
            for (int jn = 0; jn < VD / 64; ++jn)
              tma_load_2d(dst + (kk * (VD / 64) + jn) * 8192, &map_v, &full[st], jn * 64, row + kk * 64);
        } else {
          mbar_expect_tx(&full[st], L::K_BYTES);
#pragma unroll
          for (int kb = 0; kb < DK / 64; ++kb) tma_load_2d(dst + kb * (BKV * 128), &map_k, &full[st], kb * 64, row);
        }
        issued = n + 1;
      }
      if (!ok || *abort_flag) {
        // loads in flight target this CTA's shared memory: give them a bounded time to land before the CTA ends
        for (int n = max(0, issued - SLOTS); n < issued; ++n)
#pragma unroll 1
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u); ++i) {}
      }
    } else if (warp == 1 && elect_one()) {
      auto wait_full = [&](int n) { return bar_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL); };
      auto issue_scores = [&](int j, int m) -> bool {
        if (j == 0 && !bar_wait(&q_full[m], 0, abort_flag, p.err, ERR_Q)) return false;
        if (!wait_full(2 * j)) return false;
        // the buffer still holds P of the previous block until its product has been taken
        if (j > 0 && !bar_wait(&pv_done[m], (uint32_t)(j - 1) & 1u, abort_flag, p.err, ERR_PV)) return false;
        tcgen05_fence_after();
        const int st = 2 * j % SLOTS;
        const KeyRange x = key_block(keys, j);
        issue_score_product<DK>(tmem_base + m * BKV, smem_u32(sQ + m * L::Q_BYTES), smem_u32(ring + st * L::SLOT), key_steps(x.end - x.begin));
        if (m == tiles - 1) tcgen05_commit(&empty[st]);
        tcgen05_commit(&s_full[m]);
        return true;
      };
      bool ok = true;
      for (int m = 0; m < tiles && ok; ++m) ok = issue_scores(0, m);
      for (int j = 0; j < n_kv && ok; ++j) {
        const int st = (2 * j + 1) % SLOTS;
        const KeyRange x = key_block(keys, j);
        const int steps = key_steps(x.end - x.begin);
        ok = wait_full(2 * j + 1);
        for (int m = 0; m < tiles && ok; ++m) {
          ok = bar_wait(&p_full[m], (uint32_t)j & 1u, abort_flag, p.err, ERR_P);
          if (!ok) break;
          tcgen05_fence_after();
          issue_value_product<VD>(tmem_base + 2 * BKV + m * VD, tmem_base + m * BKV, smem_u32(ring + st * L::SLOT), j > 0, steps);
          if (m == tiles - 1) tcgen05_commit(&empty[st]);
          tcgen05_commit(&pv_done[m]);
          if (j + 1 < n_kv) ok = issue_scores(j + 1, m);
        }
      }
    }
  } else {
    more_registers<REGS_SOFTMAX>();
    if ((warp < 8 ? 0 : 1) < tiles) {
    const int m = warp < 8 ? 0 : 1;           // row tile of this warpgroup
    const int qtr = warp & 3;                 // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;            // row inside the tile
    const long long f = f0 + m * TILE_M + r;  // (token, head of the group)
    const int t = (int)(f / R), hh = (int)(f - (long long)t * R);
    load_queries<DK>(sQ + m * L::Q_BYTES, qtr, 4, TILE_M, [&](int row) -> const __nv_bfloat16* {
      const long long at = f0 + m * TILE_M + row;
      if (at >= rows) return nullptr;
      const int tt = (int)(at / R);
      return p.proj + ((long long)b * p.T + tt) * p.ld + (long long)(g * R + (int)(at - (long long)tt * R)) * p.dim;
    }, p.wq, p.dim, p.eps);
    fence_proxy_async_smem();
    __syncwarp();
    if (lane == 0) mbar_arrive(&q_full[m]);
    const int qpos = pos + t;
    const int lo = window_range(qpos, p.window, 0).first;
    const uint32_t lane_base = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_s = tmem_base + lane_base + m * BKV;
    const uint32_t tmem_o = tmem_base + lane_base + 2 * BKV + m * VD;
    const float c = p.scale * 1.4426950408889634f;
    float mx = p.sink / p.scale, l = mx == -INFINITY ? 0.f : 1.f;  // (in units of the scores a sink far below them all is none)
    bool ok = true;
    for (int j = 0; j < n_kv && ok; ++j) {
      const KeyRange x = key_block(keys, j);
      const int col0 = x.begin, hi = min(qpos, x.end - 1);
      const bool unseen = has_unseen(col0, min(col0 + BKV, x.end), keys.kept, keys.first);
      if (m == 0 && (col0 + BKV > x.end || unseen)) {  // the values beyond the range, and those that no row sees
        const int n = 2 * j + 1;
        ok = bar_wait_warp(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL);
        if (!ok) break;
        uint8_t* tile = ring + n % SLOTS * L::SLOT;
        if (col0 + BKV > x.end) clear_step_rest<VD>(tile, x.end - col0, r);
        if (unseen && col0 + r >= keys.kept && col0 + r < keys.first) clear_value_row<VD>(tile, r);
        fence_proxy_async_smem();
      }
      ok = bar_wait_warp(&s_full[m], (uint32_t)j & 1u, abort_flag, p.err, ERR_S);
      if (!ok) break;
      tcgen05_fence_after();
      const bool cut = __any_sync(0xffffffffu, col0 + BKV - 1 > hi || (col0 < lo && col0 + BKV > p.keep_first));  // for all lanes alike
      const RowMask mask{cut, col0, hi + 1, lo, p.keep_first, nullptr};
      const float alpha = weigh_row(tmem_s, mask, mx, l, c);
      // the scores of block j are only computed after P V of block j - 1: O is at rest here
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) rescale_output<VD>(tmem_o, alpha);
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[m]);
    }
    // ---- output: divided by the sum, gated -------------------------------------------------------------------------------
    ok = ok && bar_wait_warp(&pv_done[m], (uint32_t)(n_kv - 1) & 1u, abort_flag, p.err, ERR_PV);
    if (ok) {
      tcgen05_fence_after();
      const float inv = 1.f / l;
      const long long at = (long long)b * p.T + t, col = (long long)(g * R + hh) * p.vdim;
      const __nv_bfloat16* grow = p.gated ? p.proj + at * p.ld + (long long)(p.H + p.G) * p.dim + (long long)p.G * p.vdim + col : nullptr;
      __nv_bfloat16* orow = p.out + at * p.ldo + col;
#pragma unroll 1
      for (int ch = 0; ch < VD / 32; ++ch) {
        uint32_t raw[32];
        tmem_ld_32x32b_x32(tmem_o + ch * 32, raw);
        tmem_ld_wait();
        if (f < rows) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c0 = ch * 32 + q * 8;
            if (c0 < p.vdim) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(raw[q * 8 + e]) * inv;
              if (grow) {
                float gt[8];
                xl_load16<__nv_bfloat16>(grow + c0, gt);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= __fdividef(1.f, 1.f + __expf(-gt[e]));
              }
              *(uint4*)(orow + c0) = pack8_16bit(v, false);
            }
          }
        }
      }
    }
  }
  }
  // ---- teardown: every role arrives here, also after an abort --------------------------------------------------------
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

template <int DK, int VD> int launch_portion(const void* kc, const void* vc, const SharedParams& p, cudaStream_t s) {
  using L = PortionSmem<DK, VD>;
  CUtensorMap mk, mv;
  int r = make_map_bf16(&mk, kc, (long long)p.B * p.G * p.Smax, p.dim, p.dim, BKV);
  if (r) return r;
  r = make_map_bf16(&mv, vc, (long long)p.B * p.G * p.Smax, p.vdim, p.vdim, 64);
  if (r) return r;
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(shared_attn_portion_kernel<DK, VD>, L::TOTAL, smem));
  const long long rows = (long long)p.T * (p.H / p.G);
  const dim3 grid(p.G, (unsigned)((rows + 2 * TILE_M - 1) / (2 * TILE_M)), p.B);
  const cudaError_t e = xl_launch_overlapped(shared_attn_portion_kernel<DK, VD>, grid, dim3(SA_THREADS), (size_t)L::TOTAL, s, mk, mv, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// ---- few rows per sequence: shared keys once for all that share them -------------------------------------------------------------------
// The rows (tokens and query heads) of all sequences of a group, those with the same lead, that read one key / value head make tiles of 128, so a
// group's shared keys and values are read once per tile and not once per sequence. A sequence's own keys, with the new ones, are tiles of its own
// rows: reading bounds them, and the tensor cores work on empty rows for nothing else. All tiles' blocks of 128 keys, by group and by sequence, are one
// long list of which every CTA (one per SM) takes an equal run; a tile whose blocks belong to several CTAs leaves as many parts of its sums, and so does
// each of the two warpgroups, which take a CTA's blocks in turn: one block's softmax runs under the other's products. The kernel behind this one
// (shared_attn_sum_kernel) adds the parts.
//   warp 0       TMA: key and value tiles in turn through one ring
//   warp 1       MMA: S_m = Q K^T, O_m += P_m V
//   warp 2       queries of the next tile, if they are few, normalised, from the projections to shared memory;  warp 3  the list of this CTA's tiles
//   warps 4..7, 8..11   queries of large tiles; softmax of every second block (warps without rows only keep step)
//
// 16 x 8 beams behind 2000, up to 130 own positions, 32 heads on 8 of 128: 73 us by itself, 79 with the append and the sum (176 MB, 2.2 TB/s); 64 requests
// behind 8000, up to 700 own: 80 and 86 us (183 MB). About 9 us pass before a CTA's first product; then about 2900 clocks per block, and what it takes to
// change from tile to tile.
// Equal runs and not a CTA per tile and slice: groups and own parts are of unlike lengths, and one wave has to end together.
//
// Every CTA makes the list by itself, from positions and leads in shared memory: counts, key ranges and offsets by slot, ranks of the members by
// votes. CTA 0 leaves a copy for the kernel behind.
//
// Keys that only some rows of a tile see are masked, and values that none sees zeroed; a value that is not finite in a block that some row does not see whole is taken out, and
// the scores of its key become NaN for the rows that see it: a weight of zero times anything would reach the others.
constexpr int PF_MAX_BATCH = 448;
constexpr int PF_SLOTS_LARGE = 4, PF_SLOTS_SMALL = 8;
constexpr int PF_HALF = 32;  // rows of a tile whose queries one warp makes ready ahead; those of larger tiles are made by the softmax warps

struct GroupPlan {  // where a sequence's parts are
  int first, blocks, tiles, row;        // first block of the group, blocks of a tile, tiles of a head, the sequence's first row in the group
  int packed, total, ctas, own_blocks;  // rows of the groups before, blocks in all, CTAs that share them, blocks of a tile of its own keys
  int own_first, unused[3];             // first block of those
};

struct GroupParams {
  SharedParams p;
  float *main_o, *extra_o;    // parts that begin with a tile's first block: [groups, own][2][G][B T R][vdim]; others, by CTA: [ctas][2][TILE_M][vdim]
  float2 *main_s, *extra_s;   // their maxima (powers of two) and sums
  GroupPlan* plan;            // [B]
};

struct GroupLists {  // by slot or by sequence
  int *pos, *tokens, *edge, *hi, *lo, *least, *latest, *members, *run, *own_n, *own_key, *begin;  // begin: of groups, then of sequences
  short *lead, *offset, *rank, *order;
  __host__ __device__ static int padded(int B) { return (B + 7) / 8 * 8; }
  __host__ __device__ static int bytes(int B) { return padded(B) * (13 * 4 + 4 * 2); }
  __device__ __forceinline__ GroupLists(void* at, int B) {
    const int n = padded(B);
    pos = (int*)at; tokens = pos + n; edge = tokens + n; hi = edge + n; lo = hi + n; least = lo + n; latest = least + n; members = latest + n; run = members + n;
    own_n = run + n; own_key = own_n + n; begin = own_key + n;
    lead = (short*)(begin + 2 * n); offset = lead + n; rank = offset + n; order = rank + n;
  }
};

// A tile's keys: kept ones [low, kept), then [first, end).
struct TileKeys {
  int low, kept, first, end, kept_blocks, total;
  // of a group: somebody sees each key from `lo` to `hi`, and kept ones below
  __device__ __forceinline__ TileKeys(int lo, int hi, int keep_first) : low(0), kept(min(keep_first, lo)), first(lo), end(hi) {
    kept_blocks = key_blocks(0, kept);
    total = kept_blocks + key_blocks(first, hi);
    if (total >= key_blocks(0, hi)) {  // leaving keys out saves no block
      kept = first = kept_blocks = 0;
      total = key_blocks(0, hi);
    }
  }
  // of a sequence: its own from `edge` on, window from `lo`
  __device__ __forceinline__ TileKeys(int edge, int lo, int hi, int keep_first) : low(edge), kept(min(keep_first, lo)), first(lo), end(hi) {
    kept_blocks = key_blocks(edge, kept);
    total = kept_blocks + key_blocks(first, hi);
    if (total >= key_blocks(edge, hi)) {
      first = edge;
      kept_blocks = 0;
      total = key_blocks(edge, hi);
    }
  }
  __device__ __forceinline__ int key(int j) const { return j < kept_blocks ? low + j * BKV : first + (j - kept_blocks) * BKV; }
  __device__ __forceinline__ int until(int j) const { return j < kept_blocks ? kept : end; }
};

// a / n for numbers whose quotient is below 2^20: the software division is a hundred instructions
__device__ __forceinline__ int small_quotient(int a, int n) {
  int q = (int)__fdividef((float)a, (float)n);
  const int r = a - q * n;
  q += r >= n ? 1 : 0;
  return q - (r < 0 ? 1 : 0);
}

struct alignas(16) GroupSegment {  // blocks [block, block + count) of one tile
  int own, slot, g, tile, block, count, rows;
  int least, latest;  // every row of the tile sees the keys below `least` and from `latest` on
  int first;          // own keys below this one that are not kept are seen by no row, though blocks may have them
  TileKeys keys;
  __device__ __forceinline__ GroupSegment() : keys(0, 0, 0) {}
};
constexpr int PF_SEGMENTS = 64;  // places of the table of a CTA's segments, used in turn

template <int DK, int VD> struct GroupSmem : SharedTiles<DK, VD> {
  using L = SharedTiles<DK, VD>;
  static constexpr int SLOTS = L::SLOT > 16384 ? PF_SLOTS_LARGE : PF_SLOTS_SMALL;
  static constexpr int TILE_BYTES = L::Q_BYTES + SLOTS * L::SLOT;
  static int total(int B) {
    const int needed = TILE_BYTES + 1024 /*alignment*/ + 640 /*barriers*/ + PF_SEGMENTS * (int)sizeof(GroupSegment) + GroupLists::bytes(B);
    // more than half of an SM's shared memory: two CTAs, each holding all of TMEM, never meet on an SM
    return needed > 120 * 1024 ? needed : 120 * 1024;
  }
};

// A barrier of warps whose wait is bounded: every warp arrives and waits for its phase.
__device__ __forceinline__ bool warps_meet(uint64_t* bar, uint32_t& phase, volatile int* abort_flag, int* err) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  const bool ok = bar_wait_warp(bar, phase & 1u, abort_flag, err, ERR_MEET);
  ++phase;
  return ok;
}

// Where a tile's queries are: small tiles take the first rows of the room and the next ones in turn, so that one can be made ready while the other is in
// use; a large tile takes all of it, under number 0, and so does a CTA's first one. Everybody counts alike.
struct QueryRoom {
  int next = 0, used0 = 0, used1 = 0;           // how often each place was taken
  int ahead0 = 0, ahead1 = 0, at_once = 0;      // and was filled ahead, or the room at once
  bool large = false;                           // of the tile that took it last
  __device__ __forceinline__ int take(int rows, bool first) {
    large = first || rows > PF_HALF;
    const int h = large ? 0 : next;
    next = large ? (rows > PF_HALF ? 0 : 1) : next ^ 1;
    return h;
  }
  __device__ __forceinline__ void count(int h) {
    h ? ++used1 : ++used0;
    if (large) ++at_once;
    else h ? ++ahead1 : ++ahead0;
  }
};

template <int DK, int VD>
__global__ void __launch_bounds__(SA_THREADS, 1)
    shared_attn_groups_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const GroupParams a) {
  using L = GroupSmem<DK, VD>;
  constexpr int SLOTS = L::SLOTS;
  const SharedParams& p = a.p;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* ring = smem + L::Q_BYTES;
  uint64_t* bars = (uint64_t*)(smem + L::TILE_BYTES);
  uint64_t* q_full = bars;       // [2] by half
  uint64_t* q_empty = bars + 2;  // [2]
  uint64_t* s_full = bars + 4;   // [2] per warpgroup
  uint64_t* p_full = bars + 6;   // [2]
  uint64_t* pv_done = bars + 8;  // [2]
  uint64_t* wg_meet = bars + 10;  // [2]
  uint64_t* q_large = bars + 12;  // queries of large tiles
  uint64_t* q_free = bars + 13;   // no product needs the queries' room any more, for the next large tile
  uint64_t* full = bars + 14;     // [SLOTS]
  uint64_t* empty = bars + 14 + SLOTS;
  uint32_t* tmem_base_slot = (uint32_t*)(bars + 14 + 2 * SLOTS);
  volatile int* abort_flag = (volatile int*)(tmem_base_slot + 1);
  uint32_t* unknown = tmem_base_slot + 2;  // [2][4] keys whose values are not finite
  int* total_blocks = (int*)(unknown + 8);
  int* chunk_rows = total_blocks + 1;  // [32]
  int* chunk_blocks = chunk_rows + 32;
  volatile int* ready = (volatile int*)(chunk_blocks + 32);  // segments that were in the table so far
  volatile int* begun = ready + 1;                           // the segment that the MMA warp has come to
  static_assert((14 + 2 * SLOTS) * 8 + 8 + (9 + 66) * 4 <= 640, "room behind the tiles");
  static_assert(2 * PF_MAX_BATCH <= 32 * 32, "sums of 32 by one warp");
  GroupSegment* table = (GroupSegment*)(smem + L::TILE_BYTES + 640);
  const GroupLists list(table + PF_SEGMENTS, p.B);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, R = p.H / p.G, M = p.T * R;  // M: rows of a sequence
  // The kernel before this one appends keys and values, and all that came before that one has ended: only blocks with new keys wait for it.
  // ---- the list of blocks ------------------------------------------------------------------------------------------------------
#pragma unroll 1
  for (int b = tid; b < p.B; b += SA_THREADS) {
    list.members[b] = list.run[b] = list.hi[b] = list.latest[b] = 0;
    list.lo[b] = list.least[b] = 0x7fffffff;
  }
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
      mbar_init(&wg_meet[s], 4);
    }
    mbar_init(q_large, 8);
    mbar_init(q_free, 1);
    for (int s = 0; s < 2 * SLOTS; ++s) mbar_init(&full[s], 1);
    *ready = *begun = 0;
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
#pragma unroll 1
  for (int b = tid; b < p.B; b += SA_THREADS) {
    const int pos = p.pos[b], count = p.count[b], of = p.prefix.lead[b], shared = p.prefix.shared[b];  // asked for together
    const bool there = of >= 0 && of < p.B;
    const int held = p.pos[there ? of : b], tokens = min(count, p.T);
    int e = 0, first = 0, last = 0, n = 0;  // first, last: where the windows of the first and the last row begin
    bool sees = false;
    if (tokens > 0 && window_fits(pos, tokens, p.T, p.Smax)) {
      e = there ? max(0, min(min(shared, pos), held)) : 0;  // as shared_edge
      first = window_range(pos, p.window, 0).first;
      last = window_range(pos + tokens - 1, p.window, 0).first;
      sees = e > 0 && (first < e || p.keep_first > 0);
      n = TileKeys(e, max(first, e), pos + tokens, p.keep_first).total;
    }
    list.pos[b] = pos;
    list.tokens[b] = tokens;
    list.edge[b] = e;
    list.lead[b] = (short)(sees ? of : -1);
    list.own_key[b] = max(first, e);
    list.own_n[b] = n;
    if (sees) {
      atomicAdd(list.members + of, 1);
      atomicMax(list.hi + of, e);
      atomicMin(list.lo + of, min(first, e));
      atomicMin(list.least + of, e);
      atomicMax(list.latest + of, last);
    }
  }
  __syncthreads();
  // offsets by slot, then by sequence: sums of 32 by the warps, then of those
  const int n_list = GroupLists::padded(p.B), own_tiles = (M + TILE_M - 1) / TILE_M, chunks = (2 * n_list + 31) / 32;
  if (warp == 1) {  // ranks of the members
#pragma unroll 1
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane, s = b < p.B ? list.lead[b] : -1;
      const unsigned int same = __match_any_sync(0xffffffffu, s);
      const int before = __popc(same & ((1u << lane) - 1)), old = s >= 0 ? list.run[s] : 0;
      __syncwarp();
      if (s >= 0 && before == 0) list.run[s] = old + __popc(same);
      __syncwarp();
      if (b < p.B) list.rank[b] = (short)(old + before);
    }
  } else {
#pragma unroll 1
    for (int k = warp ? warp - 1 : 0; k < chunks; k += SA_THREADS / 32 - 1) {
      const int i = k * 32 + lane, s = i < n_list ? i : i - n_list;
      int n = 0, work = 0;
      if (i < n_list && s < p.B) {
        n = list.members[s];
        if (n) work = (n * M + TILE_M - 1) / TILE_M * p.G * TileKeys(list.lo[s], list.hi[s], p.keep_first).total;
      } else if (i >= n_list && s < p.B) {
        work = list.own_n[s] * own_tiles * p.G;
      }
      int up_n = n, up_w = work;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, up_n, d), y = __shfl_up_sync(0xffffffffu, up_w, d);
        if (lane >= d) { up_n += x; up_w += y; }
      }
      if (i < n_list) list.offset[i] = (short)(up_n - n);
      if (i < 2 * n_list) list.begin[i] = up_w - work;
      if (lane == 31) {
        chunk_rows[k] = up_n;
        chunk_blocks[k] = up_w;
      }
    }
  }
  __syncthreads();
  if (warp == 0) {
    int n = lane < chunks ? chunk_rows[lane] : 0, w = lane < chunks ? chunk_blocks[lane] : 0;
    const int n0 = n, w0 = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, n, d), y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) { n += x; w += y; }
    }
    if (lane < chunks) {
      chunk_rows[lane] = n - n0;
      chunk_blocks[lane] = w - w0;
    }
    if (lane == 31) *total_blocks = w;
  }
  __syncthreads();
#pragma unroll 1
  for (int i = tid; i < 2 * n_list; i += SA_THREADS) {
    if (i < n_list) list.offset[i] += (short)chunk_rows[i >> 5];
    list.begin[i] += chunk_blocks[i >> 5];
  }
  __syncthreads();
  const int total = *total_blocks, ctas = min((int)gridDim.x, total);
#pragma unroll 1
  for (int b = tid; b < p.B; b += SA_THREADS) {
    const int s = list.lead[b];
    if (s >= 0) list.order[list.offset[s] + list.rank[b]] = (short)b;
    if (blockIdx.x == 0) {
      GroupPlan x = {};
      x.total = total;
      x.ctas = ctas;
      x.own_blocks = list.own_n[b];
      x.own_first = list.begin[n_list + b];
      if (s >= 0) {
        x.first = list.begin[s];
        x.blocks = TileKeys(list.lo[s], list.hi[s], p.keep_first).total;
        x.tiles = (list.members[s] * M + TILE_M - 1) / TILE_M;
        x.row = list.rank[b] * M;
        x.packed = list.offset[s] * M;
      }
      a.plan[b] = x;
    }
  }
  if ((int)blockIdx.x >= ctas) {
    xl_grid_dependency_wait();
    return;
  }
  const XlRanges ranges{total / ctas, total % ctas};
  const int x0 = ranges.begin(blockIdx.x), x1 = ranges.begin(blockIdx.x + 1);
  // segment number n of this CTA, when it is in the table; null: the wait for it gave up
  auto segment = [&](int n) -> const GroupSegment* {
#pragma unroll 1
    for (uint32_t i = 0; *ready <= n; ++i) {
      if (i == MBAR_SPIN_LIMIT || *abort_flag) {
        *abort_flag = 1;
        atomicCAS(p.err, 0, (int)ERR_TABLE);
        return nullptr;
      }
      if (i > 64) __nanosleep(200);  // (a wait that gives up does so behind the barriers' waits, which have the reason)
    }
    __threadfence_block();
    return table + n % PF_SEGMENTS;
  };

  // a tile's queries by `count` warps, of which this is number i
  auto fill_queries = [&](const GroupSegment& g, int half, int i, int count) {
    const short* members = list.order + (g.own ? 0 : list.offset[g.slot]);
    load_queries<DK>(sQ + half * PF_HALF * 128, i, count, g.rows, [&](int row) -> const __nv_bfloat16* {
      if (row >= g.rows) return nullptr;
      const int at = g.tile * TILE_M + row, k = g.own ? 0 : small_quotient(at, M), b = g.own ? g.slot : members[k], t = p.T > 1 ? small_quotient(at - k * M, R) : 0;
      return p.proj + ((long long)b * p.T + t) * p.ld + (long long)(g.g * R + at - k * M - t * R) * p.dim;
    }, p.wq, p.dim, p.eps);
  };

  if (warp == 1) {
    tmem_alloc(tmem_base_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;

  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int issued = 0;
#pragma unroll 1
      for (int x = x0, sn = 0; x < x1 && ok; ++sn) {
        const GroupSegment* sg = segment(sn);
        if (!sg) break;
        const TileKeys keys = sg->keys;
        const int row0 = (sg->slot * p.G + sg->g) * p.Smax, j0 = sg->block, j1 = j0 + sg->count;
        if (sg->own) xl_grid_dependency_wait();
#pragma unroll 1
        for (int j = j0; j < j1 && ok; ++j, ++x) {
          const int row = row0 + keys.key(j);
          const int halves = keys.until(j) - keys.key(j) > BKV / 2 ? 2 : 1;  // of which somebody sees a key
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            const int n = 2 * (x - x0) + kv, st = n % SLOTS;
            if (n >= SLOTS) ok = bar_wait(&empty[st], (uint32_t)(n / SLOTS - 1) & 1u, abort_flag, p.err, ERR_KV_EMPTY);
            if (!ok) break;
            uint8_t* dst = ring + st * L::SLOT;
            if (kv) {
              mbar_expect_tx(&full[st], L::V_BYTES / 2 * halves);
#pragma unroll 1
              for (int kk = 0; kk < halves; ++kk)
#pragma unroll
                for (int jn = 0; jn < VD / 64; ++jn)
                  tma_load_2d(dst + (kk * (VD / 64) + jn) * 8192, &map_v, &full[st], jn * 64, row + kk * 64);
            } else {
              mbar_expect_tx(&full[st], L::K_BYTES / 2 * halves);
#pragma unroll 1
              for (int kk = 0; kk < halves; ++kk)
#pragma unroll
                for (int kb = 0; kb < DK / 64; ++kb) tma_load_2d(dst + kb * (BKV * 128) + kk * 8192, &map_k, &full[st], kb * 64, row + kk * 64);
            }
            issued = n + 1;
          }
        }
      }
      if (!ok || *abort_flag) {
        // loads in flight target this CTA's shared memory: give them a bounded time to land before the CTA ends
#pragma unroll 1
        for (int n = max(0, issued - SLOTS); n < issued; ++n)
#pragma unroll 1
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u); ++i) {}
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      xl_grid_dependency_wait();    // the successor reads what came before this kernel
      xl_grid_launch_dependents();  // TMEM is held: a successor that allocates some on this SM cannot come first
      auto wait_full = [&](int n) { return bar_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL); };
      // block `it` of this CTA: warpgroup it & 1, its block it >> 1
      auto issue_scores = [&](int it, int half, int steps) -> bool {
        const int m = it & 1, st = 2 * it % SLOTS;
        if (!wait_full(2 * it)) return false;
        // the buffer still holds P of the warpgroup's previous block until its product has been taken
        if (it >= 2 && !bar_wait(&pv_done[m], (uint32_t)((it >> 1) - 1) & 1u, abort_flag, p.err, ERR_PV)) return false;
        tcgen05_fence_after();
        issue_score_product<DK>(tmem_base + m * BKV, smem_u32(sQ) + half * PF_HALF * 128, smem_u32(ring + st * L::SLOT), steps);
        tcgen05_commit(&empty[st]);
        tcgen05_commit(&s_full[m]);
        return true;
      };
      auto issue_values = [&](int it, bool add, int steps) -> bool {
        const int m = it & 1, st = (2 * it + 1) % SLOTS;
        if (!wait_full(2 * it + 1)) return false;
        if (!bar_wait(&p_full[m], (uint32_t)(it >> 1) & 1u, abort_flag, p.err, ERR_P)) return false;
        tcgen05_fence_after();
        issue_value_product<VD>(tmem_base + 2 * BKV + m * VD, tmem_base + m * BKV, smem_u32(ring + st * L::SLOT), add, steps);
        tcgen05_commit(&empty[st]);
        tcgen05_commit(&pv_done[m]);
        return true;
      };
      QueryRoom room;
      bool ok = true, add = false, pending = false;  // pending: block it - 1 has no product with the values yet
      int it = 0, steps = 0;
#pragma unroll 1
      for (int x = x0, sn = 0; x < x1 && ok; ++sn) {
        const GroupSegment* sg = segment(sn);
        if (!sg) break;
        const int half = room.take(sg->rows, sn == 0), count = sg->count, block = sg->block;
        const TileKeys keys = sg->keys;
        *begun = sn;
        if (room.large && pending) {  // the warps that make these queries ready end their last tile first
          ok = bar_wait(&s_full[(it - 1) & 1], (uint32_t)((it - 1) >> 1) & 1u, abort_flag, p.err, ERR_S);  // and with it all products before
          if (!ok) break;
          mbar_arrive(q_free);
          ok = issue_values(it - 1, add, steps);
          pending = false;
          if (!ok) break;
        }
        ok = room.large ? bar_wait(q_large, (uint32_t)room.at_once & 1u, abort_flag, p.err, ERR_Q)
                        : bar_wait(&q_full[half], (uint32_t)(half ? room.ahead1 : room.ahead0) & 1u, abort_flag, p.err, ERR_Q);
#pragma unroll 1
        for (int j = 0; j < count && ok; ++j, ++it) {
          const int now = key_steps(keys.until(block + j) - keys.key(block + j));
          ok = issue_scores(it, half, now);
          if (ok && j + 1 == count) tcgen05_commit(&q_empty[half]);
          if (ok && pending) ok = issue_values(it - 1, add, steps);
          pending = true;
          add = j >= 2;  // of this block: the warpgroup has had one of this segment
          steps = now;
        }
        room.count(half);
        x += count;
      }
      if (ok && pending) issue_values(it - 1, add, steps);
    }
  } else if (warp == 2) {  // queries of small tiles
    QueryRoom room;
    bool ok = true;
#pragma unroll 1
    for (int x = x0, sn = 0; x < x1; ++sn) {
      const GroupSegment* sg = segment(sn);
      if (!sg) break;
      const int half = room.take(sg->rows, sn == 0);
      // The products that used the place before. (Place 1 comes behind a small tile in place 0, whose wait was for a large one's products.) Every use is
      // waited for, in order, those of large tiles too: a barrier only tells apart the phase that runs and the one before.
      const int used = half ? room.used1 : room.used0;
      if (used) ok = bar_wait_warp(&q_empty[half], (uint32_t)(used - 1) & 1u, abort_flag, p.err, ERR_Q);
      if (!ok) break;
      if (!room.large) {
        fill_queries(*sg, half, 0, 1);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[half]);
      }
      room.count(half);
      x += sg->count;
    }
  } else if (warp == 3) {  // the table of this CTA's segments
    if (lane == 0) {
      int i = 0;  // the last group or sequence whose blocks begin at x0 or before
#pragma unroll 1
      for (int step = 512; step; step >>= 1)
        if (i + step < 2 * n_list && list.begin[i + step] <= x0) i += step;
#pragma unroll 1
      for (int x = x0, sn = 0; x < x1; ++i) {
        const bool own = i >= n_list;
        const int slot = own ? i - n_list : i;
        const int end = i + 1 < 2 * n_list ? list.begin[i + 1] : total;  // of its blocks
        if (end <= x) continue;
        GroupSegment g;
        g.own = own;
        g.slot = slot;
        g.keys = own ? TileKeys(list.edge[slot], list.own_key[slot], list.pos[slot] + list.tokens[slot], p.keep_first)
                     : TileKeys(list.lo[slot], list.hi[slot], p.keep_first);
        g.least = own ? list.pos[slot] + 1 : list.least[slot];
        g.latest = own ? window_range(list.pos[slot] + list.tokens[slot] - 1, p.window, 0).first : list.latest[slot];
        g.first = own ? list.own_key[slot] : 0;
        const int n = g.keys.total, rows = own ? M : list.members[slot] * M, tiles = (rows + TILE_M - 1) / TILE_M;
        int unit = small_quotient(x - list.begin[i], n);  // tiles by head
        g.g = small_quotient(unit, tiles);
        g.tile = unit - g.g * tiles;
        g.block = x - list.begin[i] - unit * n;
#pragma unroll 1
        for (; x < min(end, x1); ++sn) {
          // the other warps are a few blocks apart from each other: half a table is more than that
#pragma unroll 1
          for (uint32_t k = 0; sn - *begun >= PF_SEGMENTS / 2 && k < MBAR_SPIN_LIMIT && !*abort_flag; ++k) __nanosleep(200);
          if (sn - *begun >= PF_SEGMENTS / 2) {
            *abort_flag = 1;
            atomicCAS(p.err, 0, (int)ERR_ROOM);
            x = x1;
            break;
          }
          g.count = min(n - g.block, x1 - x);
          g.rows = min(TILE_M, rows - g.tile * TILE_M);
          table[sn % PF_SEGMENTS] = g;
          __threadfence_block();
          *ready = sn + 1;
          x += g.count;
          g.block = 0;
          if (++g.tile == tiles) {
            g.tile = 0;
            ++g.g;
          }
        }
      }
    }
  } else {
    const int m = warp < 8 ? 0 : 1;  // warpgroup
    const int qtr = warp & 3;        // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;   // row inside the tile
    const uint32_t lane_base = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_s = tmem_base + lane_base + m * BKV;
    const uint32_t tmem_o = tmem_base + lane_base + 2 * BKV + m * VD;
    const float c = p.scale * 1.4426950408889634f;
    bool ok = true;
    uint32_t met = 0;
    QueryRoom room;
#pragma unroll 1
    for (int x = x0, sn = 0; x < x1 && ok; ++sn) {
      const GroupSegment* at_table = segment(sn);
      if (!at_table) break;
      const GroupSegment sg = *at_table;
      const TileKeys& keys = sg.keys;
      const int half = room.take(sg.rows, sn == 0);
      if (room.large) {
        // The MMA warp says when the room is free, once for every large tile. (The products' own barriers cannot: who skips the uses of small tiles may
        // come here two uses ahead of one, and a barrier only tells apart the phase that runs and the one before.)
        if (sn) ok = bar_wait_warp(q_free, (uint32_t)(room.at_once - 1) & 1u, abort_flag, p.err, ERR_Q);
        if (!ok) break;
        fill_queries(sg, 0, warp - 4, 8);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_large);
      }
      room.count(half);
      // row r: its sequence and position; the keys that it sees end at `edge` and begin with its window at `lo`
      const int at_row = sg.tile * TILE_M + r, member = sg.own ? 0 : small_quotient(at_row, M);
      bool row_on = r < sg.rows;
      const bool warp_on = qtr * 32 < sg.rows;
      int edge = 0x7fffffff, lo = 0;
      const int b = sg.own ? sg.slot : list.order[list.offset[sg.slot] + (row_on ? member : 0)], t = p.T > 1 ? small_quotient(at_row - member * M, R) : 0;
      const int pos = list.pos[b], tokens = list.tokens[b];
      row_on = row_on && t < tokens;
      if (row_on) {
        edge = sg.own ? pos + t + 1 : list.edge[b];
        lo = window_range(pos + t, p.window, 0).first;
      }
      float mx = -INFINITY, l = 0.f;
      int mine = 0, last = 0;
#pragma unroll 1
      for (int j = sg.block; j < sg.block + sg.count && ok; ++j, ++x) {
        const int it = x - x0;
        if ((it & 1) != m) continue;
        ok = bar_wait_warp(&s_full[m], (uint32_t)(it >> 1) & 1u, abort_flag, p.err, ERR_S);
        if (!ok) break;
        tcgen05_fence_after();
        const int key0 = keys.key(j), end = keys.until(j);
        // not every row sees every key; and, of a group, not all rows see the same ones
        const bool cut = key0 + BKV > end || key0 + BKV > sg.least || (key0 < sg.latest && key0 + BKV > p.keep_first);
        const bool uneven = cut && !sg.own && (min(key0 + BKV, end) > sg.least || (key0 < sg.latest && key0 + BKV > p.keep_first));
        const bool unseen = has_unseen(key0, min(key0 + BKV, end), p.keep_first, sg.first);
        if (uneven || unseen || (end - key0 < BKV && (end - key0) % UMMA_K)) {
          const int n = 2 * it + 1;
          ok = bar_wait_warp(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL);
          if (!ok) break;
          uint8_t* tile = ring + n % SLOTS * L::SLOT;
          if (end - key0 < BKV) clear_step_rest<VD>(tile, end - key0, r);
          const bool finite = !uneven || key0 + r >= end || finite_value_row<VD>(tile, r);  // thread r looks at the value of key r
          if (!finite || (unseen && key0 + r >= p.keep_first && key0 + r < sg.first)) clear_value_row<VD>(tile, r);
          fence_proxy_async_smem();
          if (uneven) {
            const unsigned int bits = __ballot_sync(0xffffffffu, !finite);
            if (lane == 0) unknown[m * 4 + qtr] = bits;
            ok = warps_meet(&wg_meet[m], met, abort_flag, p.err);
            if (!ok) break;
          }
        }
        if (warp_on) {
          const RowMask mask{cut, key0, min(end, edge), lo, p.keep_first, uneven ? unknown + m * 4 : nullptr};
          const float alpha = weigh(tmem_s, mask, key_steps(end - key0), mx, l, c);
          // the scores of a block are only computed after P V of the warpgroup's block before: O is at rest here
          if (mine && __any_sync(0xffffffffu, alpha != 1.f)) rescale_output<VD>(tmem_o, alpha);
          tmem_st_wait();
        }
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[m]);
        ++mine;
        last = it >> 1;
      }
      // ---- this part's sums ------------------------------------------------------------------------------------------------
      if (!ok || !warp_on) continue;
      const bool main = sg.block == 0;
      const long long at = main ? (((long long)sg.own * 2 + m) * p.G + sg.g) * p.B * M +
                                      (sg.own ? sg.slot : list.offset[sg.slot]) * (long long)M + at_row
                                : ((long long)blockIdx.x * 2 + m) * TILE_M + r;
      if (row_on) (main ? a.main_s : a.extra_s)[at] = make_float2(mx * c, l);
      if (mine) {
        ok = bar_wait_warp(&pv_done[m], (uint32_t)last & 1u, abort_flag, p.err, ERR_PV);
        if (!ok) break;
        tcgen05_fence_after();
        float* o = (main ? a.main_o : a.extra_o) + at * p.vdim;
#pragma unroll 1
        for (int ch = 0; ch < VD / 32; ++ch) {
          uint32_t raw[32];
          tmem_ld_32x32b_x32(tmem_o + ch * 32, raw);
          tmem_ld_wait();
          if (row_on)
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (ch * 32 + q * 4 < p.vdim)
                *reinterpret_cast<uint4*>(o + ch * 32 + q * 4) = make_uint4(raw[q * 4], raw[q * 4 + 1], raw[q * 4 + 2], raw[q * 4 + 3]);
        }
        tcgen05_fence_before();
      }
    }
  }

  // ---- teardown: every role arrives here, also after an abort --------------------------------------------------------
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcgen05_fence_after();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---- the sum of all parts -----------------------------------------------------------------------------------------------------------
// A warp per row and head, four features per lane. Reading bounds it: 2 + 2 parts of a row, and two more for every further CTA that had blocks of its
// tiles. 9 us for 64 rows of 32 heads with about 20 parts (12.6 with one part after the other).
__global__ void __launch_bounds__(128) shared_attn_sum_kernel(const GroupParams a) {
  const SharedParams& p = a.p;
  const int R = p.H / p.G, M = p.T * R, lane = threadIdx.x & 31;
  const int row = blockIdx.x * 4 + (threadIdx.x >> 5), h = blockIdx.y;  // (sequence, token)
  const int b = row / p.T, t = row - b * p.T, g = h / R;
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  if (b >= p.B) return;
  const int4* at = reinterpret_cast<const int4*>(a.plan + b);
  const int4 pa = __ldcg(at), pb = __ldcg(at + 1), pc = __ldcg(at + 2);
  const int pos = p.pos[b], n = min(p.count[b], p.T);
  const int c = lane * 4;
  uint2 gate = make_uint2(0u, 0u);
  if (p.gated && c < p.vdim)
    gate = *reinterpret_cast<const uint2*>(p.proj + (long long)row * p.ld + (long long)(p.H + p.G) * p.dim + (long long)p.G * p.vdim +
                                           (long long)h * p.vdim + c);
  if (t >= n || !window_fits(pos, n, p.T, p.Smax)) return;
  const int per = pb.y / pb.z;  // (there are blocks: the row's own key is among them)
  const XlRanges ranges{per, pb.y - per * pb.z};
  auto owner = [&](int x) {  // ranges.owner(x)
    const int head = ranges.rem * (per + 1);
    return x < head ? small_quotient(x, per + 1) : ranges.rem + small_quotient(x - head, per);
  };
  float sink = p.sink * 1.4426950408889634f;
  if (sink > 3.4e38f) sink = 3.4e38f;  // (infinite in these units, it would leave no number in the difference below)
  // two sources: the tile of the group and the tile of the sequence; of each one CTA's part for each warpgroup from its first block on, then those of
  // the CTAs that follow
  const int own = t * R + h - g * R;  // row in the sequence's tiles
  const int idx[2] = {pa.w + own, own}, blocks[2] = {pa.y, pb.w};
  int c0[2] = {0, 0}, parts[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (blocks[k]) {
      const int tiles = k ? (M + TILE_M - 1) / TILE_M : pa.z, x = (k ? pc.x : pa.x) + (g * tiles + idx[k] / TILE_M) * blocks[k];
      c0[k] = owner(x);
      parts[k] = 2 * (owner(x + blocks[k] - 1) - c0[k] + 1);
    }
  const int all = parts[0] + parts[1];
  auto place = [&](int k, bool& main) -> long long {
    const int src = k < parts[0] ? 0 : 1, q = src ? k - parts[0] : k, m = q & 1, i = q >> 1;
    main = i == 0;
    return main ? ((long long)(src * 2 + m) * p.G + g) * p.B * M + (src ? (long long)b * M + idx[1] : (long long)pb.x + idx[0])
                : ((long long)((src ? c0[1] : c0[0]) + i) * 2 + m) * TILE_M + (src ? idx[1] : idx[0]) % TILE_M;
  };
  auto stat = [&](int k) {
    bool main;
    const long long e = place(k, main);
    return __ldcg((main ? a.main_s : a.extra_s) + e);
  };
  float2 mine = lane < all ? stat(lane) : make_float2(-INFINITY, 0.f);  // of the first 32 parts
  float m = fmaxf(sink, mine.x);
#pragma unroll 1
  for (int k = lane + 32; k < all; k += 32) m = fmaxf(m, stat(k).x);
  m = xl_warp_max(m);
  float total = sink == -INFINITY ? 0.f : exp2f(sink - m);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
  for (int k0 = 0; k0 < all; k0 += 32) {
    if (k0) mine = k0 + lane < all ? stat(k0 + lane) : make_float2(-INFINITY, 0.f);
    const float f = mine.x == -INFINITY ? 0.f : exp2f(mine.x - m);
    total += xl_warp_sum(f * mine.y);  // (a sum that is not a number stays none)
    const unsigned int holds = __ballot_sync(0xffffffffu, mine.x > -INFINITY);  // parts that had a score (others were not written, or l is no number)
    const int now = min(32, all - k0);
#pragma unroll 1
    for (int k = 0; k < now; k += 4) {  // four parts under way together, those that hold nothing among them
      float fk[4];
      float4 x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int q = min(k + u, now - 1);
        const float fq = __shfl_sync(0xffffffffu, f, q);
        fk[u] = k + u < now ? fq : 0.f;
        bool main;
        const long long e = place(k0 + q, main);
        if (c < p.vdim) x[u] = __ldcg(reinterpret_cast<const float4*>((main ? a.main_o : a.extra_o) + e * p.vdim + c));
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (k + u < now && holds >> (k + u) & 1)  // (with a factor of zero too: what is not finite stays so)
          acc = make_float4(acc.x + x[u].x * fk[u], acc.y + x[u].y * fk[u], acc.z + x[u].z * fk[u], acc.w + x[u].w * fk[u]);
    }
  }
  if (c >= p.vdim) return;
  float v[4] = {acc.x / total, acc.y / total, acc.z / total, acc.w / total};
  if (p.gated) {
    v[0] *= 1.f / (1.f + expf(-dd_lo(gate.x)));
    v[1] *= 1.f / (1.f + expf(-dd_hi(gate.x)));
    v[2] *= 1.f / (1.f + expf(-dd_lo(gate.y)));
    v[3] *= 1.f / (1.f + expf(-dd_hi(gate.y)));
  }
  *reinterpret_cast<uint2*>(p.out + (long long)row * p.ldo + (long long)h * p.vdim + c) = make_uint2(dd_pack(v[0], v[1]), dd_pack(v[2], v[3]));
}

template <int DK, int VD> int launch_groups(const GroupParams& a, const void* kc, const void* vc, int ctas, cudaStream_t s) {
  using L = GroupSmem<DK, VD>;
  const SharedParams& p = a.p;
  CUtensorMap mk, mv;
  int r = make_map_bf16(&mk, kc, (long long)p.B * p.G * p.Smax, p.dim, p.dim, BKV / 2);
  if (r) return r;
  r = make_map_bf16(&mv, vc, (long long)p.B * p.G * p.Smax, p.vdim, p.vdim, 64);
  if (r) return r;
  const int bytes = L::total(p.B);
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(shared_attn_groups_kernel<DK, VD>, bytes, smem));
  XL_TRY(xl_launch_overlapped(shared_attn_groups_kernel<DK, VD>, dim3(ctas), dim3(SA_THREADS), (size_t)bytes, s, mk, mv, a));
  const cudaError_t e = xl_launch_overlapped(shared_attn_sum_kernel, dim3((p.B * p.T + 3) / 4, p.H), dim3(128), (size_t)0, s, a);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

SharedParams shared_params(const void* proj, long long ld, const float* wq, void* out, long long ldo, const int* pos, const int* count, const int* lead,
                           const int* shared, int B, int T, int H, int G, int dim, int vdim, int Smax, int window, int keep_first, int gated,
                           float scale, float sink, float eps, int* err) {
  SharedParams p = {};
  p.proj = (const __nv_bfloat16*)proj; p.ld = ld; p.wq = wq; p.pos = pos; p.count = count; p.prefix = {lead, shared};
  p.out = (__nv_bfloat16*)out; p.ldo = ldo; p.B = B; p.T = T; p.H = H; p.G = G; p.dim = dim; p.vdim = vdim; p.Smax = Smax;
  p.window = window; p.keep_first = keep_first; p.gated = gated; p.scale = scale; p.sink = sink; p.eps = eps; p.err = err;
  return p;
}

// whether the tensor-core kernels take such operands
bool tensor_sizes(const void* proj, long long ld, const void* kc, const void* vc, const void* out, long long ldo, int B, int T, int H, int G, int dim,
                  int vdim, int Smax, int gated) {
  if (dim < 8 || dim > 128 || dim % 8 || vdim < 8 || vdim > 128 || vdim % 8 || ld % 8 || ldo % 8 || ldo < (long long)H * vdim ||
      ld < (long long)(H + G) * dim + (long long)G * vdim + (gated ? (long long)H * vdim : 0))
    return false;
  if ((((uintptr_t)proj) | ((uintptr_t)kc) | ((uintptr_t)vc) | ((uintptr_t)out)) & 15) return false;
  return (long long)B * G * Smax <= 0x7fffffffLL - 2 * BKV && (long long)B * T * H <= 0x7fffffffLL - 4 * TILE_M &&
         ((long long)T * (H / G) + 2 * TILE_M - 1) / (2 * TILE_M) <= 65535;
}

}  // namespace

// proj: (B*T, ld) as in attention_window.cu; wq, wk (dim) fp32. New keys and values go to the caches, of sequences whose rows all fit; with qn (B, G,
// T, H/G, dim) the queries go there. dim, vdim <= 512.
XL_API int xl_shared_append(const void* proj, long long ld, const float* wq, const float* wk, float* qn, void* kc, void* vc, const int* pos,
                            const int* count, int B, int T, int H, int G, int dim, int vdim, int Smax, float eps, int dtype, cudaStream_t s) {
  if (B < 1 || B > 65535 || T < 1 || G < 1 || H < 1 || H % G || dim < 1 || dim > SA_MAX_DIM || vdim < 1 || vdim > SA_MAX_DIM || Smax < 1 ||
      ld < (long long)(H + G) * dim + (long long)G * vdim || !wq || !wk)
    return -1;
  const int warps = min(8, qn ? H + G : G);
  XL_DISPATCH_DTYPE(dtype, X, {
    const auto all = (uintptr_t)proj | (uintptr_t)kc | (uintptr_t)vc;
    const auto real = (uintptr_t)wq | (uintptr_t)wk | (uintptr_t)qn;
    const bool wide = dim % 4 == 0 && vdim % 4 == 0 && ld % 4 == 0 && all % (4 * sizeof(X)) == 0 && real % 16 == 0;
    const auto kernel = wide ? shared_append_kernel<X, 4> : shared_append_kernel<X, 1>;
    XL_TRY(xl_launch_overlapped(kernel, dim3(T, B), dim3(32 * warps), (size_t)0, s, (const X*)proj, ld, wq, wk, qn, (X*)kc, (X*)vc, pos, count, T, H, G, dim,
                                vdim, Smax, eps));
  });
  return (int)cudaGetLastError();
}

// Attention of a portion whose keys and values are in the caches (launched behind xl_shared_append), bf16. dim, vdim multiples of 8 and at most
// 128; ld, ldo multiples of 8; proj, caches and out 16-byte aligned. Rows past count[b], and sequences that do not fit, are not written. err: device int
// for the code of a wait that gave up. Returns 0, a CUDA error code, or a negative value for arguments this kernel does not take.
XL_API int xl_shared_attn_portion(const void* proj, long long ld, const float* wq, const void* kc, const void* vc, void* out, long long ldo,
                                  const int* pos, const int* count, const int* lead, const int* shared, int B, int T, int H, int G, int dim,
                                  int vdim, int Smax, int window, int keep_first, int gated, float scale, float sink, float eps, int* err,
                                  cudaStream_t s) {
  if (B < 1 || B > 65535 || T < 1 || G < 1 || H < 1 || H % G || Smax < 1 || window < 0 || keep_first < 0 || !(scale > 0.f) || !lead || !shared || !wq)
    return -1;
  if (!tensor_sizes(proj, ld, kc, vc, out, ldo, B, T, H, G, dim, vdim, Smax, gated)) return -1;
  const SharedParams p =
      shared_params(proj, ld, wq, out, ldo, pos, count, lead, shared, B, T, H, G, dim, vdim, Smax, window, keep_first, gated, scale, sink, eps, err);
  if (dim <= 64) return vdim <= 64 ? launch_portion<64, 64>(kc, vc, p, s) : launch_portion<64, 128>(kc, vc, p, s);
  return vdim <= 64 ? launch_portion<128, 64>(kc, vc, p, s) : launch_portion<128, 128>(kc, vc, p, s);
}

// floats of scratch memory for xl_shared_attn_groups with `ctas` CTAs
XL_API long long xl_shared_attn_groups_scratch(int B, int T, int H, int vdim, int ctas) {
  return B * 12LL + (4LL * B * T * H + ctas * 2LL * TILE_M) * (vdim + 2);
}

// The same for few rows per sequence, whose shared keys are read once for all that share them: two launches behind xl_shared_append, which has to be the
// launch before. At most 448 sequences. ctas: SMs of the device. scratch: xl_shared_attn_groups_scratch floats, 16-byte aligned.
XL_API int xl_shared_attn_groups(const void* proj, long long ld, const float* wq, const void* kc, const void* vc, void* out, long long ldo,
                                 const int* pos, const int* count, const int* lead, const int* shared, int B, int T, int H, int G, int dim,
                                 int vdim, int Smax, int window, int keep_first, int gated, float scale, float sink, float eps, int ctas,
                                 float* scratch, int* err, cudaStream_t s) {
  if (B < 1 || B > PF_MAX_BATCH || T < 1 || G < 1 || H < 1 || H % G || H > 65535 || Smax < 1 || window < 0 || keep_first < 0 || !(scale > 0.f) || !lead ||
      !shared || !wq || ctas < 1 || ctas > 4096 || !scratch || ((uintptr_t)scratch & 15))
    return -1;
  if (!tensor_sizes(proj, ld, kc, vc, out, ldo, B, T, H, G, dim, vdim, Smax, gated)) return -1;
  GroupParams a = {};
  a.p = shared_params(proj, ld, wq, out, ldo, pos, count, lead, shared, B, T, H, G, dim, vdim, Smax, window, keep_first, gated, scale, sink, eps, err);
  static_assert(sizeof(GroupPlan) == 48, "12 floats of scratch memory per sequence");
  a.plan = (GroupPlan*)scratch;
  a.main_o = scratch + 12LL * B;
  a.extra_o = a.main_o + 4LL * B * T * H * vdim;
  a.main_s = (float2*)(a.extra_o + 2LL * ctas * TILE_M * vdim);
  a.extra_s = a.main_s + 4LL * B * T * H;
  if (dim <= 64) return vdim <= 64 ? launch_groups<64, 64>(a, kc, vc, ctas, s) : launch_groups<64, 128>(a, kc, vc, ctas, s);
  return vdim <= 64 ? launch_groups<128, 64>(a, kc, vc, ctas, s) : launch_groups<128, 128>(a, kc, vc, ctas, s);
}
