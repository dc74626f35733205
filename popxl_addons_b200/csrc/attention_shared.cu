// Sliding-window attention where the first positions of a sequence lie in the cache of another slot (attention_window.cuh): beams of one
// prompt, requests behind one system prompt. Same mathematics and layouts as attention_window.cu.
//
//   xl_shared_append           new keys (norms in 64 bits, rounded once) and values into the caches; for the general kernel queries in fp32
//   xl_shared_attn_portion     portions of tokens on the tensor cores (tcgen05), bf16
//   xl_shared_attn_general     any sizes and types (attention_window.cu)
//
// Queries enter the products as two bf16 numbers, value and rounding error, as the weights do: a rounded query would move every score by
// 2^-9 of itself, more than all other roundings together.
#include "attention_window.cuh"
#include "tcgen05.cuh"

#include <math.h>

namespace {

using namespace xl_tc;

constexpr int SA_MAX_DIM = 512;

// ---- new keys and values ------------------------------------------------------------------------------------------------------
// One CTA per row, a warp per head.
template <typename T>
__global__ void __launch_bounds__(256)
    shared_append_kernel(const T* proj, long long ld, const float* wq, const float* wk, float* qn, T* kc, T* vc, const int* pos, const int* count,
                         int T_len, int H, int G, int dim, int vdim, int Smax, float eps) {
  xl_grid_launch_dependents();
  const int b = blockIdx.y, t = blockIdx.x, p = pos[b] + t;
  if (t >= count[b] || !window_fits(pos[b], count[b], T_len, Smax)) return;
  const T* row = proj + ((long long)b * T_len + t) * ld;
  const int R = H / G, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int NP = SA_MAX_DIM / 32;
  for (int h = qn ? warp : H + warp; h < H + G; h += 8) {
    float x[NP];
    double sq = 0.0;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = lane + 32 * i;
      x[i] = c < dim ? xl_to_float(row[(long long)h * dim + c]) : 0.f;
      if (c < dim) sq += (double)x[i] * (double)x[i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const double f = 1.0 / sqrt(sq / dim + (double)eps);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = lane + 32 * i;
      if (c >= dim) break;
      const float y = (float)((double)x[i] * f * (double)(h < H ? wq : wk)[c]);
      if (h < H) qn[((((long long)b * G + h / R) * T_len + t) * R + h % R) * dim + c] = y;
      else kc[(((long long)b * G + (h - H)) * Smax + p) * dim + c] = xl_from_float<T>(y);
    }
  }
  const T* src = row + (long long)(H + G) * dim;
  for (int i = threadIdx.x; i < G * vdim; i += blockDim.x) {
    const int g = i / vdim, c = i - g * vdim;
    vc[(((long long)b * G + g) * Smax + p) * vdim + c] = src[i];
  }
}

// ---- portions on the tensor cores -----------------------------------------------------------------------------------------------
// The R query heads that read one key / value head are consecutive rows (token-major). A CTA owns 256 of these rows as two tiles of 128
// and walks the keys visible to any of them in blocks of 128: those of the lead, then its own ones. Key and value tiles serve both row
// tiles, which take turns on the tensor cores while the other one's softmax runs:
//   warp 0       TMA: key and value tiles in turn through one ring
//   warp 1       MMA: S_m = Q_m K^T into TMEM (both halves of the queries), then O_m += P_m V
//   warps 2..5   tile 0, warps 6..9 tile 1: norms of the queries, from the projections straight to shared memory; then the softmax, one thread
//                per row, running maximum and sum in fp32, lazy rescaling of O_m in TMEM
// P replaces S in TMEM as two bf16 numbers per weight. Keys beyond a range are masked in the scores, and their values are zeroed in shared
// memory: what lies there belongs to others, and a weight of zero times anything that is not finite would reach the sum.
//
// TMEM columns: [0, 128) S_0 / P_0, [128, 256) S_1 / P_1, [256, 256 + VD) O_0, [256 + VD, 256 + 2 VD) O_1. One CTA per SM. Every wait is
// bounded (see tcgen05.cuh).
constexpr int TILE_M = 128;
constexpr int BKV = 128;
constexpr int UMMA_K = 16;
constexpr int SA_THREADS = 64 + 2 * 128;
constexpr uint32_t TMEM_COLS = 512;

enum { ERR_Q = 101, ERR_KV_FULL = 102, ERR_KV_EMPTY = 103, ERR_S = 104, ERR_P = 105, ERR_PV = 106 };

struct SharedParams {
  const __nv_bfloat16* proj;
  long long ld;
  const float *wq, *wk;
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

// Rows of a tile, normalised, to shared memory as two K-major operands of 128-byte swizzle: the 32 rows of one warp. `row(r)`: where the
// projections have the head of row r of the tile, or null.
template <int DK, typename F>
__device__ __forceinline__ void load_queries(uint8_t* tile, int first_row, const F& row, const float* wq, int dim, float eps) {
  constexpr int LANES = DK / 8, ROWS = 32 / LANES;  // lanes of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % LANES;
  const bool on = chunk * 8 < dim;
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = on ? wq[chunk * 8 + e] : 0.f;
#pragma unroll 4
  for (int i = 0; i < 32; i += ROWS) {
    const int r = first_row + i + lane / LANES;
    const __nv_bfloat16* src = row(r);
    float x[8], sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.f;
    if (src && on) xl_load16<__nv_bfloat16>(src + chunk * 8, x);
#pragma unroll
    for (int e = 0; e < 8; ++e) sq += x[e] * x[e];
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, o);
    const float f = 1.f / sqrtf(sq / dim + eps);
    float lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= f * w[e];
    const uint4 hi = pack8_16bit(x, false);
    const uint32_t h[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo[2 * e] = x[2 * e] - __uint_as_float(h[e] << 16);
      lo[2 * e + 1] = x[2 * e + 1] - __uint_as_float(h[e] & 0xffff0000u);
    }
    uint8_t* dst = tile + (chunk >> 3) * (TILE_M * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4);
    *reinterpret_cast<uint4*>(dst) = hi;
    *reinterpret_cast<uint4*>(dst + TILE_M * DK * 2) = pack8_16bit(lo, false);
  }
}

// S_m = Q K^T, both halves of the queries
template <int DK> __device__ __forceinline__ void issue_score_product(uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr) {
  // bf16 operands, fp32 accumulator, both K-major, N = BKV
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BKV >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int kb = 0; kb < DK / 64; ++kb)
#pragma unroll
      for (int k = 0; k < 64 / UMMA_K; ++k)
        tcgen05_mma_f16(tmem_s, make_smem_desc(q_addr + half * (TILE_M * DK * 2) + kb * (TILE_M * 128) + k * (UMMA_K * 2), 16),
                        make_smem_desc(k_addr + kb * (BKV * 128) + k * (UMMA_K * 2), 16), idesc, (half | kb | k) ? 1u : 0u);
}

// O_m (+)= P V, both halves of the weights
template <int VD> __device__ __forceinline__ void issue_value_product(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr, bool add) {
  // A (P) from TMEM, B (V) MN-major (bit 16), N = VD
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(VD >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int k = 0; k < BKV / UMMA_K; ++k)
      tcgen05_mma_f16_ts(tmem_o, tmem_p + half * (BKV / 2) + k * (UMMA_K / 2),
                         make_smem_desc(v_addr + (k >> 2) * (VD / 64) * 8192 + (k & 3) * (UMMA_K * 128), 8192), idesc,
                         (add || half || k) ? 1u : 0u);
}

__device__ __forceinline__ void load_scores(uint32_t tmem_s, float (&s)[BKV]) {
#pragma unroll
  for (int ch = 0; ch < BKV / 32; ++ch) {
    uint32_t raw[32];
    tmem_ld_32x32b_x32(tmem_s + ch * 32, raw);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; ++i) s[ch * 32 + i] = __uint_as_float(raw[i]);
  }
}

// Scores of one block (in units of 1 / scale, -inf where masked) become weights; mx, l: running maximum and sum; c = scale * log2(e). Returns the
// factor of what O holds. The maximum moves only when an exponent would exceed 2^8.
__device__ __forceinline__ float weigh(float (&s)[BKV], float& mx, float& l, float c) {
  float m_blk = -INFINITY;
#pragma unroll
  for (int i = 0; i < BKV; ++i) m_blk = fmaxf(m_blk, s[i]);
  const bool move = m_blk > -INFINITY && (mx == -INFINITY || (m_blk - mx) * c > 8.f);
  const float m_new = move ? m_blk : mx;
  const float m_use = m_new == -INFINITY ? 0.f : m_new;  // a row without a visible key yet keeps weight 0
  const float alpha = (move && mx != -INFINITY) ? fast_exp2((mx - m_use) * c) : 1.f;
  const float mc = m_use * c;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < BKV; ++i) {
    s[i] = fast_exp2(fmaf(s[i], c, -mc));
    sum += s[i];
  }
  l = l * alpha + sum;
  mx = m_new;
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

// the features of value row r of a tile in shared memory
template <int VD> __device__ __forceinline__ uint4* value_row(uint8_t* tile, int r, int jn) {
  return reinterpret_cast<uint4*>(tile + ((r >> 6) * (VD / 64) + jn) * 8192 + (r & 63) * 128);
}

struct KeyRange {
  int slot, begin, end;
};
// The keys that rows at positions p_first .. p_last of sequence b see, as up to four ranges of the lead's and its own cache, in blocks of BKV.
struct KeyRanges {  // in shared memory
  KeyRange r[4];
  int until[4];  // blocks of the ranges up to and with this one
};
__device__ __forceinline__ int key_blocks(int begin, int end) { return begin < end ? (end - begin + BKV - 1) / BKV : 0; }
__device__ __forceinline__ void set_ranges(KeyRanges& k, int b, int lead, int edge, int p_first, int p_last, int window, int keep_first) {
  WindowRange seen = window_range(p_first, window, keep_first);
  const int all = key_blocks(0, edge) + key_blocks(edge, p_last + 1);
  const int visible = key_blocks(0, min(seen.kept, edge)) + key_blocks(seen.first, edge) + key_blocks(edge, seen.kept) +
                      key_blocks(max(seen.first, edge), p_last + 1);
  if (visible >= all) seen = {0, 0};  // leaving keys out saves no block
  k.r[0] = {lead, 0, min(seen.kept, edge)};
  k.r[1] = {lead, seen.first, edge};
  k.r[2] = {b, edge, seen.kept};
  k.r[3] = {b, max(seen.first, edge), p_last + 1};
  int n = 0;
  for (int i = 0; i < 4; ++i) k.until[i] = n += key_blocks(k.r[i].begin, k.r[i].end);
}
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

  if (warp == 0) {
    if (lane == 0) {
      xl_grid_dependency_wait();    // the new keys and values; nothing else here depends on the kernel that appends them
      xl_grid_launch_dependents();  // TMEM is held: a successor that allocates some on this SM cannot come first
      bool ok = true;
      int issued = 0;
      for (int n = 0; n < 2 * n_kv && ok; ++n) {  // key tile of block 0, value tile of block 0, key tile of block 1, ...
        const int st = n % SLOTS;
        const KeyRange x = key_block(keys, n >> 1);
        const int row = (x.slot * p.G + g) * p.Smax + x.begin;
        if (n >= SLOTS) ok = mbar_wait(&empty[st], (uint32_t)(n / SLOTS - 1) & 1u, abort_flag, p.err, ERR_KV_EMPTY);
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
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u); ++i) {}
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      auto wait_full = [&](int n) { return mbar_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL); };
      auto issue_scores = [&](int j, int m) -> bool {
        if (j == 0 && !mbar_wait(&q_full[m], 0, abort_flag, p.err, ERR_Q)) return false;
        if (!wait_full(2 * j)) return false;
        // the buffer still holds P of the previous block until its product has been taken
        if (j > 0 && !mbar_wait(&pv_done[m], (uint32_t)(j - 1) & 1u, abort_flag, p.err, ERR_PV)) return false;
        tcgen05_fence_after();
        const int st = 2 * j % SLOTS;
        issue_score_product<DK>(tmem_base + m * BKV, smem_u32(sQ + m * L::Q_BYTES), smem_u32(ring + st * L::SLOT));
        if (m == tiles - 1) tcgen05_commit(&empty[st]);
        tcgen05_commit(&s_full[m]);
        return true;
      };
      bool ok = true;
      for (int m = 0; m < tiles && ok; ++m) ok = issue_scores(0, m);
      for (int j = 0; j < n_kv && ok; ++j) {
        const int st = (2 * j + 1) % SLOTS;
        ok = wait_full(2 * j + 1);
        for (int m = 0; m < tiles && ok; ++m) {
          ok = mbar_wait(&p_full[m], (uint32_t)j & 1u, abort_flag, p.err, ERR_P);
          if (!ok) break;
          tcgen05_fence_after();
          issue_value_product<VD>(tmem_base + 2 * BKV + m * VD, tmem_base + m * BKV, smem_u32(ring + st * L::SLOT), j > 0);
          if (m == tiles - 1) tcgen05_commit(&empty[st]);
          tcgen05_commit(&pv_done[m]);
          if (j + 1 < n_kv) ok = issue_scores(j + 1, m);
        }
      }
    }
  } else if ((warp < 6 ? 0 : 1) < tiles) {
    const int m = warp < 6 ? 0 : 1;           // row tile of this warpgroup
    const int qtr = warp & 3;                 // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;            // row inside the tile
    const long long f = f0 + m * TILE_M + r;  // (token, head of the group)
    const int t = (int)(f / R), hh = (int)(f - (long long)t * R);
    load_queries<DK>(sQ + m * L::Q_BYTES, qtr * 32, [&](int row) -> const __nv_bfloat16* {
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
    float mx = p.sink / p.scale, l = p.sink == -INFINITY ? 0.f : 1.f;
    bool ok = true;
    for (int j = 0; j < n_kv && ok; ++j) {
      const KeyRange x = key_block(keys, j);
      const int col0 = x.begin, hi = min(qpos, x.end - 1);
      if (m == 0 && col0 + BKV > x.end) {  // the values beyond the range
        const int n = 2 * j + 1;
        ok = mbar_wait_warp(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL);
        if (!ok) break;
        if (col0 + r >= x.end)
#pragma unroll
          for (int jn = 0; jn < VD / 64; ++jn)
#pragma unroll
            for (int i = 0; i < 8; ++i) value_row<VD>(ring + n % SLOTS * L::SLOT, r, jn)[i] = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
      }
      ok = mbar_wait_warp(&s_full[m], (uint32_t)j & 1u, abort_flag, p.err, ERR_S);
      if (!ok) break;
      tcgen05_fence_after();
      float s[BKV];
      load_scores(tmem_s, s);
      if (col0 + BKV - 1 > hi || (col0 < lo && col0 + BKV > p.keep_first)) {
#pragma unroll
        for (int i = 0; i < BKV; ++i)
          if (col0 + i > hi || (col0 + i < lo && col0 + i >= p.keep_first)) s[i] = -INFINITY;
      }
      const float alpha = weigh(s, mx, l, c);
      // the scores of block j are only computed after P V of block j - 1: O is at rest here
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) rescale_output<VD>(tmem_o, alpha);
      store_split_weights<BKV>(tmem_s, s);
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[m]);
    }
    // ---- output: divided by the sum, gated -------------------------------------------------------------------------------
    ok = ok && mbar_wait_warp(&pv_done[m], (uint32_t)(n_kv - 1) & 1u, abort_flag, p.err, ERR_PV);
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
// T, H/G, dim) the queries go there. dim <= 512.
XL_API int xl_shared_append(const void* proj, long long ld, const float* wq, const float* wk, float* qn, void* kc, void* vc, const int* pos,
                            const int* count, int B, int T, int H, int G, int dim, int vdim, int Smax, float eps, int dtype, cudaStream_t s) {
  if (B < 1 || B > 65535 || T < 1 || G < 1 || H < 1 || H % G || dim < 1 || dim > SA_MAX_DIM || vdim < 1 || Smax < 1 ||
      ld < (long long)(H + G) * dim + (long long)G * vdim || !wq || !wk)
    return -1;
  XL_DISPATCH_DTYPE(dtype, X, {
    shared_append_kernel<X><<<dim3(T, B), 256, 0, s>>>((const X*)proj, ld, wq, wk, qn, (X*)kc, (X*)vc, pos, count, T, H, G, dim, vdim, Smax, eps);
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
  SharedParams p = {};
  p.proj = (const __nv_bfloat16*)proj; p.ld = ld; p.wq = wq; p.pos = pos; p.count = count; p.prefix = {lead, shared};
  p.out = (__nv_bfloat16*)out; p.ldo = ldo; p.B = B; p.T = T; p.H = H; p.G = G; p.dim = dim; p.vdim = vdim; p.Smax = Smax;
  p.window = window; p.keep_first = keep_first; p.gated = gated; p.scale = scale; p.sink = sink; p.eps = eps; p.err = err;
  if (dim <= 64) return vdim <= 64 ? launch_portion<64, 64>(kc, vc, p, s) : launch_portion<64, 128>(kc, vc, p, s);
  return vdim <= 64 ? launch_portion<128, 64>(kc, vc, p, s) : launch_portion<128, 128>(kc, vc, p, s);
}
