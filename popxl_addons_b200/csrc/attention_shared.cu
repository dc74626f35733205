// Sliding-window attention where the first positions of a sequence lie in the cache of another slot (attention_window.cuh): beams of one
// prompt, requests behind one system prompt. Same mathematics and layouts as attention_window.cu.
//
//   xl_shared_append           new keys (norms in 64 bits, rounded once) and values into the caches; for the general kernel queries in fp32
//   xl_shared_attn_portion     portions of tokens on the tensor cores (tcgen05), bf16
//   xl_shared_attn_decode      one token per sequence, bf16: the keys that a group of sequences shares, once for the group (tcgen05), and each
//                              sequence's own keys (mma.sync)
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
//   warps 4..7   tile 0, warps 8..11 tile 1: norms of the queries, from the projections straight to shared memory; then the softmax, one thread
//                per row, running maximum and sum in fp32, lazy rescaling of O_m in TMEM (warps 2, 3: none)
// P replaces S in TMEM as two bf16 numbers per weight. Keys beyond a range are masked in the scores, and their values are zeroed in shared
// memory: what lies there belongs to others, and a weight of zero times anything that is not finite would reach the sum.
//
// TMEM columns: [0, 128) S_0 / P_0, [128, 256) S_1 / P_1, [256, 256 + VD) O_0, [256 + VD, 256 + 2 VD) O_1. One CTA per SM. Every wait is
// bounded (see tcgen05.cuh).
constexpr int TILE_M = 128;
constexpr int BKV = 128;
constexpr int UMMA_K = 16;
constexpr int SA_THREADS = 128 + 2 * 128;
// registers of a thread: of the first warpgroup, which only issues, and of the two that hold a row of scores each (together what the
// launch gives, 384 x 168: with 168 each the softmax spilled, and a block took twice as long)
constexpr int REGS_CONTROL = 72, REGS_SOFTMAX = 216;
static_assert(REGS_CONTROL + 2 * REGS_SOFTMAX <= 3 * 168, "more than the launch gives would never be granted");
template <int N> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
constexpr uint32_t TMEM_COLS = 512;

enum { ERR_Q = 101, ERR_KV_FULL = 102, ERR_KV_EMPTY = 103, ERR_S = 104, ERR_P = 105, ERR_PV = 106, ERR_MEET = 107 };

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

// Rows first, first + step, ... below `end` (LANES lanes each, as many at a time as a warp has lanes for) of a tile, normalised, to shared memory as
// two K-major operands of 128-byte swizzle. `row(r)`: where the projections have the head of row r of the tile, or null.
template <int DK, int UNROLL, typename F>
__device__ __forceinline__ void load_queries(uint8_t* tile, int first, int step, int end, const F& row, const float* wq, int dim, float eps) {
  constexpr int LANES = DK / 8, ROWS = 32 / LANES;  // lanes of a row, rows at a time
  const int lane = threadIdx.x & 31, chunk = lane % LANES;
  const bool on = chunk * 8 < dim;
  float w[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) w[e] = on ? wq[chunk * 8 + e] : 0.f;
#pragma unroll UNROLL
  for (int i = first * ROWS; i < end; i += step * ROWS) {
    const int r = i + lane / LANES;
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

// Descriptors of a product's steps differ by whole 16 bytes of address, which stay inside the address field. The first one is hidden from the
// compiler, which would keep those of all steps in registers across the loop over blocks.
__device__ __forceinline__ uint64_t first_desc(uint32_t addr, uint32_t lbo_bytes) {
  uint64_t d = make_smem_desc(addr, lbo_bytes);
  asm volatile("" : "+l"(d));
  return d;
}

// S_m = Q K^T, both halves of the queries
template <int DK> __device__ __forceinline__ void issue_score_product(uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr) {
  // bf16 operands, fp32 accumulator, both K-major, N = BKV
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BKV >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
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

// O_m (+)= P V, both halves of the weights
template <int VD> __device__ __forceinline__ void issue_value_product(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr, bool add) {
  // A (P) from TMEM, B (V) MN-major (bit 16), N = VD
  constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(VD >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
  const uint64_t dv = first_desc(v_addr, 8192);
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int k = 0; k < BKV / UMMA_K; ++k)
      tcgen05_mma_f16_ts(tmem_o, tmem_p + half * (BKV / 2) + k * (UMMA_K / 2),
                         dv + (((k >> 2) * (VD / 64) * 8192 + (k & 3) * (UMMA_K * 128)) >> 4), idesc, (add || half || k) ? 1u : 0u);
}

// 64 columns, and the wait for them: nothing may touch the registers in between
__device__ __forceinline__ void load_scores_64(uint32_t taddr, float* s) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(s[0]), "=f"(s[1]), "=f"(s[2]), "=f"(s[3]), "=f"(s[4]), "=f"(s[5]), "=f"(s[6]), "=f"(s[7]),
        "=f"(s[8]), "=f"(s[9]), "=f"(s[10]), "=f"(s[11]), "=f"(s[12]), "=f"(s[13]), "=f"(s[14]), "=f"(s[15]),
        "=f"(s[16]), "=f"(s[17]), "=f"(s[18]), "=f"(s[19]), "=f"(s[20]), "=f"(s[21]), "=f"(s[22]), "=f"(s[23]),
        "=f"(s[24]), "=f"(s[25]), "=f"(s[26]), "=f"(s[27]), "=f"(s[28]), "=f"(s[29]), "=f"(s[30]), "=f"(s[31]),
        "=f"(s[32]), "=f"(s[33]), "=f"(s[34]), "=f"(s[35]), "=f"(s[36]), "=f"(s[37]), "=f"(s[38]), "=f"(s[39]),
        "=f"(s[40]), "=f"(s[41]), "=f"(s[42]), "=f"(s[43]), "=f"(s[44]), "=f"(s[45]), "=f"(s[46]), "=f"(s[47]),
        "=f"(s[48]), "=f"(s[49]), "=f"(s[50]), "=f"(s[51]), "=f"(s[52]), "=f"(s[53]), "=f"(s[54]), "=f"(s[55]),
        "=f"(s[56]), "=f"(s[57]), "=f"(s[58]), "=f"(s[59]), "=f"(s[60]), "=f"(s[61]), "=f"(s[62]), "=f"(s[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void load_scores(uint32_t tmem_s, float (&s)[BKV]) {
  load_scores_64(tmem_s, s);
  load_scores_64(tmem_s + 64, s + 64);
}

// the lowest n bits (n may be anything)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1; }
// Keys 32 w .. 32 w + 31 of a block that begins at key0 which a row sees: below `end`, and from `lo` on or below `keep`.
__device__ __forceinline__ uint32_t visible_bits(int key0, int w, int end, int lo, int keep) {
  const int k = key0 + 32 * w;
  return low_bits(end - k) & (~low_bits(lo - k) | low_bits(keep - k));
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

  // (the two settings stand at the head of branches that only join again at the end: behind a join the smaller one would hold)
  if (warp < 4) {
  fewer_registers<REGS_CONTROL>();
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
  }
  } else {
  more_registers<REGS_SOFTMAX>();
  if ((warp < 8 ? 0 : 1) < tiles) {
    const int m = warp < 8 ? 0 : 1;           // row tile of this warpgroup
    const int qtr = warp & 3;                 // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;            // row inside the tile
    const long long f = f0 + m * TILE_M + r;  // (token, head of the group)
    const int t = (int)(f / R), hh = (int)(f - (long long)t * R);
    load_queries<DK, 4>(sQ + m * L::Q_BYTES, qtr, 4, TILE_M, [&](int row) -> const __nv_bfloat16* {
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
        for (int w = 0; w < BKV / 32; ++w) {
          const uint32_t visible = visible_bits(col0, w, hi + 1, lo, p.keep_first);
#pragma unroll
          for (int i = 0; i < 32; ++i) s[w * 32 + i] = visible >> i & 1 ? s[w * 32 + i] : -INFINITY;
        }
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

// ---- single tokens: long runs of keys, the shared ones once for all that share them ----------------------------------------------------
// The query heads of all sequences of a group (those with the same lead) that read one key / value head are the rows of tiles of 128, so a
// group's shared keys and values are read once per tile and not once per sequence. Of a sequence's own keys whole blocks of 128 are tiles of
// R rows, if there are two at least: reading bounds them, and the tensor cores work on empty rows for nothing else. All tiles' blocks, by group and
// by sequence, are one long list of which every CTA (one per SM) takes an equal run; a tile whose blocks belong to several CTAs leaves as many parts
// of its sums, and so does each of the two warpgroups, which take a CTA's blocks in turn: one block's softmax runs under the other's products.
// The kernel behind this one (shared_attn_decode_kernel) adds the parts to what is left of the sequences' own keys.
//   warp 0       TMA: key and value tiles in turn through one ring
//   warp 1       MMA: S_m = Q K^T, O_m += P_m V
//   warps 2, 3   queries of the next tile, normalised, from the projections to shared memory; tiles of up to 64 rows take halves of the room in turn
//   warps 4..7, 8..11   softmax of every second block; warps without rows only keep step
//
// Every CTA makes the list by itself, from positions and leads in shared memory: counts, key ranges and offsets by slot, ranks of the members by
// votes. CTA 0 leaves a copy for the kernel behind.
//
// Keys that only some rows of a tile see are masked; a value that is not finite in a block that some row does not see whole is taken out, and
// the scores of its key become NaN for the rows that see it: a weight of zero times anything would reach the others.
constexpr int PF_MAX_BATCH = 512;
constexpr int PF_SLOTS_LARGE = 4, PF_SLOTS_SMALL = 8;
constexpr int PF_HALF = TILE_M / 2;

// A sequence's own visible keys before its new one, from `first` on: whole blocks for the prefix kernel (0 or at least two).
__device__ __forceinline__ int own_blocks(int first, int pos) { return pos - first >= 2 * BKV ? (pos - first) / BKV : 0; }

struct PrefixPlan {  // where a sequence's parts are
  int first, blocks, tiles, row;  // first block of the group, blocks of a tile, tiles of a head, the sequence's first row in the group
  int packed, total, ctas, own_blocks;  // rows of the groups before, blocks in all, CTAs that share them, blocks of a tile of its own keys
  int own_first, unused[3];       // first block of those
};

struct PrefixParams {
  SharedParams p;
  float *main_o, *extra_o;    // parts that begin with a tile's first block: [groups, own][2][G][B R][vdim]; others, by CTA: [ctas][2][TILE_M][vdim]
  float2 *main_s, *extra_s;   // their maxima (powers of two) and sums
  PrefixPlan* plan;           // [B]
  int read_ahead;             // positions, counts, leads and the caches were complete before the previous launch
};

struct PrefixLists {  // by slot or by sequence
  int *edge, *hi, *lo, *least, *latest, *members, *run, *own_n, *own_key, *begin;  // begin: of groups, then of sequences
  short *lead, *offset, *rank, *order;
  __host__ __device__ static int padded(int B) { return (B + 7) / 8 * 8; }
  __host__ __device__ static int bytes(int B) { return padded(B) * (11 * 4 + 4 * 2); }
  __device__ __forceinline__ PrefixLists(void* at, int B) {
    const int n = padded(B);
    edge = (int*)at; hi = edge + n; lo = hi + n; least = lo + n; latest = least + n; members = latest + n; run = members + n;
    own_n = run + n; own_key = own_n + n; begin = own_key + n;
    lead = (short*)(begin + 2 * n); offset = lead + n; rank = offset + n; order = rank + n;
  }
};

// the blocks of a group's shared keys: those of the kept tokens, then those from `first` on
struct PrefixBlocks {
  int kept, first, end, kept_blocks, total;
  __device__ __forceinline__ PrefixBlocks(int lo, int hi, int keep_first) {
    kept = min(keep_first, lo);
    first = lo;
    end = hi;
    kept_blocks = key_blocks(0, kept);
    total = kept_blocks + key_blocks(first, hi);
    if (total >= key_blocks(0, hi)) {  // leaving keys out saves no block
      kept = first = kept_blocks = 0;
      total = key_blocks(0, hi);
    }
  }
  __device__ __forceinline__ int key(int j) const { return j < kept_blocks ? j * BKV : first + (j - kept_blocks) * BKV; }
  __device__ __forceinline__ int until(int j) const { return j < kept_blocks ? kept : end; }
};

struct PrefixSegment {  // blocks [block, block + count) of one tile
  bool own;
  int slot, g, tile, block, count, rows;
};

template <int DK, int VD> struct PrefixSmem : SharedTiles<DK, VD> {
  using L = SharedTiles<DK, VD>;
  static constexpr int SLOTS = L::SLOT > 16384 ? PF_SLOTS_LARGE : PF_SLOTS_SMALL;
  static constexpr int TILE_BYTES = L::Q_BYTES + SLOTS * L::SLOT;
  static int total(int B) {
    const int needed = TILE_BYTES + 1024 /*alignment*/ + 512 /*barriers*/ + PrefixLists::bytes(B);
    // more than half of an SM's shared memory: two CTAs, each holding all of TMEM, never meet on an SM
    return needed > 120 * 1024 ? needed : 120 * 1024;
  }
};

// A barrier of warps whose wait is bounded: every warp arrives and waits for its phase.
__device__ __forceinline__ bool warps_meet(uint64_t* bar, uint32_t& phase, volatile int* abort_flag, int* err) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  const bool ok = mbar_wait_warp(bar, phase & 1u, abort_flag, err, ERR_MEET);
  ++phase;
  return ok;
}

// Which half of the queries' room a tile takes, and how often it was taken before: the warps that fill it and the one that uses it count alike.
struct QueryRoom {
  int next = 0, used[2] = {0, 0};
  __device__ __forceinline__ int take(int rows) {  // 0 or 1; a tile of more than half takes both, under number 0
    if (rows > PF_HALF) {
      next = 0;
      return 0;
    }
    const int h = next;
    next ^= 1;
    return h;
  }
};

template <int DK, int VD>
__global__ void __launch_bounds__(SA_THREADS, 1)
    shared_attn_prefix_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const PrefixParams a) {
  using L = PrefixSmem<DK, VD>;
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
  uint64_t* full = bars + 12;     // [SLOTS]
  uint64_t* empty = bars + 12 + SLOTS;
  uint32_t* tmem_base_slot = (uint32_t*)(bars + 12 + 2 * SLOTS);
  volatile int* abort_flag = (volatile int*)(tmem_base_slot + 1);
  uint32_t* unknown = tmem_base_slot + 2;  // [2][4] keys whose values are not finite
  int* total_blocks = (int*)(unknown + 8);
  static_assert((12 + 2 * SLOTS) * 8 + 8 + 9 * 4 <= 512, "room behind the tiles");
  const PrefixLists list(smem + L::TILE_BYTES + 512, p.B);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, R = p.H / p.G;
  if (!a.read_ahead) xl_grid_dependency_wait();
  // ---- the list of blocks ------------------------------------------------------------------------------------------------------
  for (int b = tid; b < p.B; b += SA_THREADS) {
    list.members[b] = list.run[b] = list.hi[b] = list.latest[b] = 0;
    list.lo[b] = list.least[b] = 0x7fffffff;
  }
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 2);
      mbar_init(&q_empty[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
      mbar_init(&wg_meet[s], 4);
    }
    for (int s = 0; s < 2 * SLOTS; ++s) mbar_init(&full[s], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  for (int b = tid; b < p.B; b += SA_THREADS) {
    int lead = b, e = 0, first = 0, n = 0;
    const int pos = p.pos[b];
    bool sees = false;
    if (p.count[b] > 0 && window_fits(pos, p.count[b], 1, p.Smax)) {
      e = shared_edge(p.prefix, p.pos, b, pos, p.B, lead);
      first = window_range(pos, p.window, 0).first;
      sees = e > 0 && (first < e || p.keep_first > 0);
      n = own_blocks(max(first, e), pos);
    }
    list.edge[b] = e;
    list.lead[b] = (short)(sees ? lead : -1);
    list.own_key[b] = max(first, e);
    list.own_n[b] = n;
    if (sees) {
      atomicAdd(list.members + lead, 1);
      atomicMax(list.hi + lead, e);
      atomicMin(list.lo + lead, min(first, e));
      atomicMin(list.least + lead, e);
      atomicMax(list.latest + lead, first);
    }
  }
  __syncthreads();
  const int n_list = PrefixLists::padded(p.B), own_tiles = (R + TILE_M - 1) / TILE_M;
  if (warp == 0) {  // offsets by slot, then by sequence
    int rows = 0, blocks = 0;
    for (int s0 = 0; s0 < 2 * n_list; s0 += 32) {
      const int i = s0 + lane, s = i < n_list ? i : i - n_list;
      int n = 0, work = 0;
      if (i < n_list && s < p.B) {
        n = list.members[s];
        if (n) work = (n * R + TILE_M - 1) / TILE_M * p.G * PrefixBlocks(list.lo[s], list.hi[s], p.keep_first).total;
      } else if (i >= n_list && i < 2 * n_list && s < p.B) {
        work = list.own_n[s] * own_tiles * p.G;
      }
      int up_n = n, up_w = work;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, up_n, d), y = __shfl_up_sync(0xffffffffu, up_w, d);
        if (lane >= d) { up_n += x; up_w += y; }
      }
      if (i < n_list) list.offset[i] = (short)(rows + up_n - n);
      if (i < 2 * n_list) list.begin[i] = blocks + up_w - work;
      rows += __shfl_sync(0xffffffffu, up_n, 31);
      blocks += __shfl_sync(0xffffffffu, up_w, 31);
    }
    if (lane == 0) *total_blocks = blocks;
  } else if (warp == 1) {  // ranks of the members
    for (int b0 = 0; b0 < p.B; b0 += 32) {
      const int b = b0 + lane, s = b < p.B ? list.lead[b] : -1;
      const unsigned int same = __match_any_sync(0xffffffffu, s);
      const int before = __popc(same & ((1u << lane) - 1)), old = s >= 0 ? list.run[s] : 0;
      __syncwarp();
      if (s >= 0 && before == 0) list.run[s] = old + __popc(same);
      __syncwarp();
      if (b < p.B) list.rank[b] = (short)(old + before);
    }
  }
  __syncthreads();
  const int total = *total_blocks, ctas = min((int)gridDim.x, total);
  if (blockIdx.x == 0) xl_grid_dependency_wait();  // an earlier attention may still read its plan
  for (int b = tid; b < p.B; b += SA_THREADS) {
    const int s = list.lead[b];
    if (s >= 0) list.order[list.offset[s] + list.rank[b]] = (short)b;
    if (blockIdx.x == 0) {
      PrefixPlan x = {};
      x.total = total;
      x.ctas = ctas;
      x.own_blocks = list.own_n[b];
      x.own_first = list.begin[n_list + b];
      if (s >= 0) {
        x.first = list.begin[s];
        x.blocks = PrefixBlocks(list.lo[s], list.hi[s], p.keep_first).total;
        x.tiles = (list.members[s] * R + TILE_M - 1) / TILE_M;
        x.row = list.rank[b] * R;
        x.packed = list.offset[s] * R;
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
  // the run of blocks from x on that belong to one tile
  auto segment = [&](int x) {
    int i = 0;  // the last group or sequence whose blocks begin at x or before
    for (int step = 2 * PF_MAX_BATCH / 2; step; step >>= 1)
      if (i + step < 2 * n_list && list.begin[i + step] <= x) i += step;
    PrefixSegment g;
    g.own = i >= n_list;
    g.slot = g.own ? i - n_list : i;
    const int n = g.own ? list.own_n[g.slot] : PrefixBlocks(list.lo[g.slot], list.hi[g.slot], p.keep_first).total;
    const int rows = g.own ? R : list.members[g.slot] * R, tiles = (rows + TILE_M - 1) / TILE_M, unit = (x - list.begin[i]) / n;
    g.g = unit / tiles;
    g.tile = unit % tiles;
    g.block = x - list.begin[i] - unit * n;
    g.count = min(n - g.block, x1 - x);
    g.rows = min(TILE_M, rows - g.tile * TILE_M);
    return g;
  };

  if (warp == 1) {
    tmem_alloc(tmem_base_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  const uint32_t tmem_base = *tmem_base_slot;

  // (the two settings stand at the head of branches that only join again at the end: behind a join the smaller one would hold)
  if (warp < 4) {
  fewer_registers<REGS_CONTROL>();
  if (warp == 0) {
    if (lane == 0) {
      bool ok = true;
      int issued = 0;
      for (int x = x0; x < x1 && ok;) {
        const PrefixSegment sg = segment(x);
        const PrefixBlocks keys(list.lo[sg.slot], list.hi[sg.slot], p.keep_first);
        for (int j = sg.block; j < sg.block + sg.count && ok; ++j, ++x) {
          const int row = (sg.slot * p.G + sg.g) * p.Smax + (sg.own ? list.own_key[sg.slot] + j * BKV : keys.key(j));
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            const int n = 2 * (x - x0) + kv, st = n % SLOTS;
            if (n >= SLOTS) ok = mbar_wait(&empty[st], (uint32_t)(n / SLOTS - 1) & 1u, abort_flag, p.err, ERR_KV_EMPTY);
            if (!ok) break;
            uint8_t* dst = ring + st * L::SLOT;
            if (kv) {
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
        }
      }
      if (!ok || *abort_flag) {
        // loads in flight target this CTA's shared memory: give them a bounded time to land before the CTA ends
        for (int n = max(0, issued - SLOTS); n < issued; ++n)
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u); ++i) {}
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      xl_grid_dependency_wait();    // the successor takes whatever came before this kernel as complete
      xl_grid_launch_dependents();  // TMEM is held: a successor that allocates some on this SM cannot come first
      auto wait_full = [&](int n) { return mbar_wait(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL); };
      // block `it` of this CTA: warpgroup it & 1, its block it >> 1
      auto issue_scores = [&](int it, int half) -> bool {
        const int m = it & 1, st = 2 * it % SLOTS;
        if (!wait_full(2 * it)) return false;
        // the buffer still holds P of the warpgroup's previous block until its product has been taken
        if (it >= 2 && !mbar_wait(&pv_done[m], (uint32_t)((it >> 1) - 1) & 1u, abort_flag, p.err, ERR_PV)) return false;
        tcgen05_fence_after();
        issue_score_product<DK>(tmem_base + m * BKV, smem_u32(sQ) + half * PF_HALF * 128, smem_u32(ring + st * L::SLOT));
        tcgen05_commit(&empty[st]);
        tcgen05_commit(&s_full[m]);
        return true;
      };
      auto issue_values = [&](int it, bool add) -> bool {
        const int m = it & 1, st = (2 * it + 1) % SLOTS;
        if (!wait_full(2 * it + 1)) return false;
        if (!mbar_wait(&p_full[m], (uint32_t)(it >> 1) & 1u, abort_flag, p.err, ERR_P)) return false;
        tcgen05_fence_after();
        issue_value_product<VD>(tmem_base + 2 * BKV + m * VD, tmem_base + m * BKV, smem_u32(ring + st * L::SLOT), add);
        tcgen05_commit(&empty[st]);
        tcgen05_commit(&pv_done[m]);
        return true;
      };
      QueryRoom room;
      bool ok = true, add = false;
      int it = 0;
      for (int x = x0; x < x1 && ok;) {
        const PrefixSegment sg = segment(x);
        const int half = room.take(sg.rows);
        ok = mbar_wait(&q_full[half], (uint32_t)room.used[half] & 1u, abort_flag, p.err, ERR_Q);
        for (int j = 0; j < sg.count && ok; ++j, ++it) {
          ok = issue_scores(it, half);
          if (ok && j + 1 == sg.count) tcgen05_commit(&q_empty[half]);
          if (ok && it) ok = issue_values(it - 1, add);
          add = j >= 2;  // of this block: the warpgroup has had one of this segment
        }
        ++room.used[half];
        x += sg.count;
      }
      if (ok && it) issue_values(it - 1, add);
    }
  } else {
    xl_grid_dependency_wait();  // the projections
    QueryRoom room;
    bool ok = true;
    for (int x = x0; x < x1 && ok;) {
      const PrefixSegment sg = segment(x);
      const int half = room.take(sg.rows);
      // the products that used the room before: of this half, or of both
      if (room.used[half]) ok = mbar_wait_warp(&q_empty[half], (uint32_t)(room.used[half] - 1) & 1u, abort_flag, p.err, ERR_Q);
      if (ok && sg.rows > PF_HALF && room.used[1]) ok = mbar_wait_warp(&q_empty[1], (uint32_t)(room.used[1] - 1) & 1u, abort_flag, p.err, ERR_Q);
      if (!ok) break;
      const short* members = list.order + (sg.own ? 0 : list.offset[sg.slot]);
      load_queries<DK, 2>(sQ + half * PF_HALF * 128, warp - 2, 2, sg.rows, [&](int row) -> const __nv_bfloat16* {
        if (row >= sg.rows) return nullptr;
        const int at = sg.tile * TILE_M + row, i = sg.own ? 0 : at / R, b = sg.own ? sg.slot : members[i];
        return p.proj + (long long)b * p.ld + (long long)(sg.g * R + at - i * R) * p.dim;
      }, p.wq, p.dim, p.eps);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[half]);
      ++room.used[half];
      x += sg.count;
    }
  }
  } else {
    more_registers<REGS_SOFTMAX>();
    const int m = warp < 8 ? 0 : 1;  // warpgroup
    const int qtr = warp & 3;        // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;   // row inside the tile
    const uint32_t lane_base = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_s = tmem_base + lane_base + m * BKV;
    const uint32_t tmem_o = tmem_base + lane_base + 2 * BKV + m * VD;
    const float c = p.scale * 1.4426950408889634f;
    xl_grid_dependency_wait();  // what is written here an earlier attention may still read
    bool ok = true;
    uint32_t met = 0;
    for (int x = x0; x < x1 && ok;) {
      const PrefixSegment sg = segment(x);
      const PrefixBlocks keys(list.lo[sg.slot], list.hi[sg.slot], p.keep_first);
      const bool row_on = r < sg.rows, warp_on = qtr * 32 < sg.rows;
      int edge = 0x7fffffff, lo = 0, least = 0x7fffffff, latest = 0;
      if (!sg.own) {
        least = list.least[sg.slot];
        latest = list.latest[sg.slot];
        if (row_on) {
          const int b = list.order[list.offset[sg.slot] + (sg.tile * TILE_M + r) / R];
          edge = list.edge[b];
          lo = window_range(p.pos[b], p.window, 0).first;
        }
      }
      float mx = -INFINITY, l = 0.f;
      int mine = 0, last = 0;
      for (int j = sg.block; j < sg.block + sg.count && ok; ++j, ++x) {
        const int it = x - x0;
        if ((it & 1) != m) continue;
        ok = mbar_wait_warp(&s_full[m], (uint32_t)(it >> 1) & 1u, abort_flag, p.err, ERR_S);
        if (!ok) break;
        tcgen05_fence_after();
        const int key0 = keys.key(j), end = keys.until(j);
        const bool cut = !sg.own && (key0 + BKV > end || key0 + BKV > least || (key0 < latest && key0 + BKV > p.keep_first));
        if (cut) {  // not every row sees every key: thread r looks at the value of key r
          const int n = 2 * it + 1;
          ok = mbar_wait_warp(&full[n % SLOTS], (uint32_t)(n / SLOTS) & 1u, abort_flag, p.err, ERR_KV_FULL);
          if (!ok) break;
          uint8_t* tile = ring + n % SLOTS * L::SLOT;
          bool finite = true;
#pragma unroll
          for (int jn = 0; jn < VD / 64; ++jn)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = value_row<VD>(tile, r, jn)[i];
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
              for (int e = 0; e < 4; ++e) finite &= (w[e] & 0x7f80u) != 0x7f80u && (w[e] & 0x7f800000u) != 0x7f800000u;
            }
          const bool beyond = key0 + r >= end;  // nobody sees it
          const unsigned int bits = __ballot_sync(0xffffffffu, !finite && !beyond);
          if (lane == 0) unknown[m * 4 + qtr] = bits;
          if (!finite || beyond)
#pragma unroll
            for (int jn = 0; jn < VD / 64; ++jn)
#pragma unroll
              for (int i = 0; i < 8; ++i) value_row<VD>(tile, r, jn)[i] = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_smem();
          ok = warps_meet(&wg_meet[m], met, abort_flag, p.err);
          if (!ok) break;
        }
        if (warp_on) {
          float s[BKV];
          load_scores(tmem_s, s);
          if (cut) {
#pragma unroll
            for (int w = 0; w < BKV / 32; ++w) {
              const uint32_t not_known = unknown[m * 4 + w];
              const uint32_t visible = visible_bits(key0, w, min(end, edge), lo, p.keep_first);
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                s[w * 32 + i] = not_known >> i & 1 ? NAN : s[w * 32 + i];
                s[w * 32 + i] = visible >> i & 1 ? s[w * 32 + i] : -INFINITY;
              }
            }
          }
          const float alpha = weigh(s, mx, l, c);
          // the scores of a block are only computed after P V of the warpgroup's block before: O is at rest here
          if (mine && __any_sync(0xffffffffu, alpha != 1.f)) rescale_output<VD>(tmem_o, alpha);
          store_split_weights<BKV>(tmem_s, s);
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
      const long long at = main ? (((long long)sg.own * 2 + m) * p.G + sg.g) * p.B * R +
                                      (sg.own ? sg.slot : list.offset[sg.slot]) * (long long)R + sg.tile * TILE_M + r
                                : ((long long)blockIdx.x * 2 + m) * TILE_M + r;
      if (row_on) (main ? a.main_s : a.extra_s)[at] = make_float2(mx * c, l);
      if (mine) {
        ok = mbar_wait_warp(&pv_done[m], (uint32_t)last & 1u, abort_flag, p.err, ERR_PV);
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

// ---- single tokens: the rest of each sequence's own keys, and the sum of all parts -------------------------------------------------------
// As window_attn_decode_kernel (attention_window.cu): a CTA takes up to 8 RT query heads of one key / value head, each of its 4 warps every fourth
// block of keys through a cp.async ring of its own, products on mma.sync. There are fewer than 256 keys besides kept ones: the prefix kernel has the
// others. It starts under that kernel's tail: everything but its parts was complete when it let this one start.
constexpr int SD_WARPS = 4;

struct SharedDecodeParams {
  SharedParams p;
  __nv_bfloat16 *kc, *vc;
  const float *wk;
  const float *main_o, *extra_o;
  const float2 *main_s, *extra_s;
  const PrefixPlan* plan;
  int stages;
};

__host__ __device__ constexpr int sd_keys(int kd, int vt) { return 4 * kd + vt <= 16 ? 32 : 16; }
// bytes of one ring stage of one warp: the keys as KD pieces of 64 B, then the value rows of vdim + 8 elements
__host__ __device__ constexpr int sd_stage_bytes(int keys, int kd, int vdim) { return keys * kd * 64 + keys * (vdim + 8) * 2; }

// KD: 32-feature steps of a query / key row (dim <= 32 KD); VT: 8-feature tiles of a value row (vdim <= 8 VT)
template <int KD, int VT, int RT>
__global__ void __launch_bounds__(SD_WARPS * 32, RT == 1 ? 3 : 2) shared_attn_decode_kernel(const SharedDecodeParams d) {
  constexpr int KEYS = sd_keys(KD, VT), KT = KEYS / 8;  // keys per block, tiles of eight keys
  constexpr int HEADS = 8 * RT;
  const SharedParams& p = d.p;
  extern __shared__ __align__(16) uint8_t smem[];
  // normalised queries and their rounding errors; the last row is the new key
  __shared__ __align__(16) __nv_bfloat16 sq[2][HEADS + 1][KD * 32];
  __shared__ float sm[SD_WARPS][HEADS], sl[SD_WARPS][HEADS], fw[SD_WARPS][HEADS];
  __shared__ float2 own[HEADS];  // this CTA's maxima and sums
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, j = lane & 3;
  const int R = p.H / p.G, hchunks = (R + HEADS - 1) / HEADS;
  const int g = blockIdx.x / hchunks, b = blockIdx.y;
  const int h0 = g * R + (blockIdx.x % hchunks) * HEADS;  // first query head of this CTA
  const int nh = min(HEADS, (g + 1) * R - h0);
  const int pos = p.pos[b];
  if (p.count[b] <= 0 || !window_fits(pos, p.count[b], 1, p.Smax)) {
    xl_grid_dependency_wait();  // no kernel of a chain ends before its predecessor
    return;
  }
  int lead;
  const int edge = shared_edge(p.prefix, p.pos, b, pos, p.B, lead);
  WindowRange seen = window_range(pos, p.window, p.keep_first);
  seen.first = max(seen.first, edge);
  seen.kept = max(seen.kept, edge);  // kept tokens of its own: [edge, kept)
  seen.first += own_blocks(seen.first, pos) * BKV;
  const int kept_blocks = (seen.kept - edge + KEYS - 1) / KEYS;
  const int blocks = kept_blocks + (pos - seen.first) / KEYS + 1;
  const __nv_bfloat16* row = p.proj + (long long)b * p.ld;
  const __nv_bfloat16* kb = d.kc + ((long long)b * p.G + g) * p.Smax * p.dim;
  const __nv_bfloat16* vb = d.vc + ((long long)b * p.G + g) * p.Smax * p.vdim;
  auto first_key = [&](int blk) { return blk < kept_blocks ? edge + blk * KEYS : seen.first + (blk - kept_blocks) * KEYS; };
  // visible keys of a block lie below this; so do those that are in the cache already, except the new one
  auto end_key = [&](int blk) { return blk < kept_blocks ? seen.kept : pos + 1; };

  // ---- the ring of key / value blocks -------------------------------------------------------------------------------------
  const int stage_bytes = sd_stage_bytes(KEYS, KD, p.vdim), vld = p.vdim + 8;
  uint8_t* ring = smem + (long long)warp * d.stages * stage_bytes;
  const int mine = (blocks - warp + SD_WARPS - 1) / SD_WARPS;  // this warp's blocks: warp, warp + SD_WARPS, ...
  constexpr int V_ROWS = 32 / VT, V_PASSES = KEYS / V_ROWS;  // value rows that a warp copies at a time, one piece per lane
  const int v_row = lane / VT, v_col = (lane % VT) * 8;
  const bool v_on = v_col < p.vdim;
  auto prefetch = [&](int n) {
    if (n < mine) {
      uint8_t* st = ring + (n % d.stages) * stage_bytes;
      const int blk = warp + n * SD_WARPS, key0 = first_key(blk), end = min(end_key(blk), pos);
      const bool full = key0 + KEYS <= end;  // else rows from `end` on are zero-filled
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const bool row_on = full || key0 + t * 8 + quad < end;
        const __nv_bfloat16* src = kb + (row_on ? (long long)(key0 + t * 8 + quad) * p.dim + j * 8 : 0);
#pragma unroll
        for (int i = 0; i < KD; ++i) {
          const bool on = row_on && i * 32 + j * 8 < p.dim;
          dd_cp16_zfill(st + ((t * KD + i) * 32 + lane) * 16, on ? src + i * 32 : kb, on);
        }
      }
      if (v_on) {
        uint8_t* dst = st + KEYS * KD * 64 + (v_row * vld + v_col) * 2;
        const __nv_bfloat16* src = vb + (long long)(key0 + v_row) * p.vdim + v_col;
#pragma unroll
        for (int i = 0; i < V_PASSES; ++i) {
          const bool on = full || key0 + v_row + i * V_ROWS < end;
          dd_cp16_zfill(dst + i * V_ROWS * vld * 2, on ? src + (long long)i * V_ROWS * p.vdim : vb, on);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");  // possibly empty: keeps the group count per block fixed
  };
  for (int n = 0; n < d.stages - 1; ++n) prefetch(n);
  // ---- normalised queries and new key to shared memory, new key and value to the caches (the same data from each chunk of heads) -----
  const __nv_bfloat16* v_src = row + (long long)(p.H + p.G) * p.dim + (long long)g * p.vdim;
  uint4 v_new = make_uint4(0, 0, 0, 0);  // lane's piece of the new value, in every warp
  {
    constexpr int QUERIES = HEADS / SD_WARPS;  // of a warp
    uint32_t raw[QUERIES + 1][2];              // dim <= 128; the last one is the new key
#pragma unroll
    for (int i = 0; i <= QUERIES; ++i) {
      const int r = warp + i * SD_WARPS;
      const __nv_bfloat16* src = row + (long long)(i < QUERIES ? h0 + r : p.H + g) * p.dim;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * lane + 64 * u;
        raw[i][u] = (r < nh || i == QUERIES) && e < p.dim ? *reinterpret_cast<const uint32_t*>(src + e) : 0u;
      }
    }
    float w[2][4];  // query and key factors
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int e = 2 * lane + 64 * u;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        w[0][2 * u + c] = e < p.dim ? p.wq[e + c] : 0.f;
        w[1][2 * u + c] = e < p.dim ? d.wk[e + c] : 0.f;
      }
    }
    if (lane < p.vdim / 8) v_new = *reinterpret_cast<const uint4*>(v_src + lane * 8);
    float sum[QUERIES];
    double key_sum = 0.0;  // the key's norm is taken in 64 bits, as in every kernel, so that all come to the same number
#pragma unroll
    for (int i = 0; i < QUERIES; ++i) {
      sum[i] = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const float y0 = dd_lo(raw[i][u]), y1 = dd_hi(raw[i][u]);
        sum[i] += y0 * y0 + y1 * y1;
      }
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const double y0 = dd_lo(raw[QUERIES][u]), y1 = dd_hi(raw[QUERIES][u]);
      key_sum += y0 * y0 + y1 * y1;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {  // the rows' sums side by side
#pragma unroll
      for (int i = 0; i < QUERIES; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      key_sum += __shfl_xor_sync(0xffffffffu, key_sum, o);
    }
#pragma unroll
    for (int i = 0; i < QUERIES; ++i) {
      const int r = warp + i * SD_WARPS;
      const float f = 1.f / sqrtf(sum[i] / p.dim + p.eps);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * lane + 64 * u;
        if (e < KD * 32) {  // rows and features that are not in use: zero
          const float y0 = dd_lo(raw[i][u]) * f * w[0][2 * u], y1 = dd_hi(raw[i][u]) * f * w[0][2 * u + 1];
          const uint32_t hi = dd_pack(y0, y1);
          *reinterpret_cast<uint32_t*>(&sq[0][r][e]) = hi;
          *reinterpret_cast<uint32_t*>(&sq[1][r][e]) = dd_pack(y0 - dd_lo(hi), y1 - dd_hi(hi));
        }
      }
    }
    if (warp == 0) {
      const double f = 1.0 / sqrt(key_sum / p.dim + (double)p.eps);
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int e = 2 * lane + 64 * u;
        if (e < KD * 32) {
          const uint32_t y = dd_pack((float)((double)dd_lo(raw[QUERIES][u]) * f * (double)w[1][2 * u]),
                                     (float)((double)dd_hi(raw[QUERIES][u]) * f * (double)w[1][2 * u + 1]));
          *reinterpret_cast<uint32_t*>(&sq[0][HEADS][e]) = y;
          if (e < p.dim) *reinterpret_cast<uint32_t*>(d.kc + (((long long)b * p.G + g) * p.Smax + pos) * p.dim + e) = y;
        }
      }
    }
    if (threadIdx.x < p.vdim / 8)
      *reinterpret_cast<uint4*>(d.vc + (((long long)b * p.G + g) * p.Smax + pos) * p.vdim + threadIdx.x * 8) = v_new;
  }
  __syncthreads();
  uint4 q[2][RT][KD];  // rows quad (and quad + 8)
#pragma unroll
  for (int half = 0; half < 2; ++half)
#pragma unroll
    for (int m = 0; m < RT; ++m)
#pragma unroll
      for (int i = 0; i < KD; ++i) q[half][m][i] = *reinterpret_cast<const uint4*>(&sq[half][quad + 8 * m][i * 32 + j * 8]);
  float o[VT][2 * RT];
#pragma unroll
  for (int t = 0; t < VT; ++t)
#pragma unroll
    for (int e = 0; e < 2 * RT; ++e) o[t][e] = 0.f;
  float mx[RT], l[RT];
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    mx[m] = -INFINITY;
    l[m] = 0.f;
  }
  const float sc = p.scale * 1.4426950408889634f;
  for (int n = 0; n < mine; ++n) {
    prefetch(n + d.stages - 1);
    if (d.stages == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (d.stages == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
    __syncwarp();
    uint8_t* st = ring + (n % d.stages) * stage_bytes;
    const int blk = warp + n * SD_WARPS, key0 = first_key(blk), end = end_key(blk);
    if (blk == blocks - 1) {  // the new key and value take their place
      const int k = pos - key0;
      for (int i = lane; i < KD * 4; i += 32)
        *reinterpret_cast<uint4*>(st + (((k >> 3) * KD + (i >> 2)) * 32 + (k & 7) * 4 + (i & 3)) * 16) =
            *reinterpret_cast<const uint4*>(&sq[0][HEADS][i * 8]);
      if (lane < p.vdim / 8) *reinterpret_cast<uint4*>(st + KEYS * KD * 64 + (k * vld + lane * 8) * 2) = v_new;
      __syncwarp();
    }
    float s[KT][2 * RT];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int e = 0; e < 2 * RT; ++e) s[t][e] = 0.f;
#pragma unroll
      for (int i = 0; i < KD; ++i) {
        const uint4 k = *reinterpret_cast<const uint4*>(st + ((t * KD + i) * 32 + lane) * 16);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint4 &lo = q[half][0][i], &hi = q[half][RT - 1][i];
          wd_mma(s[t], make_uint2(lo.x, lo.y), make_uint2(hi.x, hi.y), k.x, k.y);
          wd_mma(s[t], make_uint2(lo.z, lo.w), make_uint2(hi.z, hi.w), k.z, k.w);
        }
      }
#pragma unroll
      for (int e = 0; e < 2 * RT; ++e)
        s[t][e] = key0 + t * 8 + 2 * j + (e & 1) < end ? s[t][e] * sc : -INFINITY;
    }
    float alpha[RT];
    uint2 ph[KT / 2][RT], pl[KT / 2][RT];  // weights as operands of the second product, and their rounding errors
#pragma unroll
    for (int m = 0; m < RT; ++m) {
      float v = -INFINITY;
#pragma unroll
      for (int t = 0; t < KT; ++t) v = fmaxf(v, fmaxf(s[t][2 * m], s[t][2 * m + 1]));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
      const float m_new = fmaxf(mx[m], v), use = m_new == -INFINITY ? 0.f : m_new;  // (no score is a number: the sum is none either)
      alpha[m] = exp2f(mx[m] - use);
      mx[m] = m_new;
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < KT; ++t) {
        const float x = exp2f(s[t][2 * m] - use), y = exp2f(s[t][2 * m + 1] - use);
        sum += x + y;
        const uint32_t hi = dd_pack(x, y), lo = dd_pack(x - dd_lo(hi), y - dd_hi(hi));
        uint2 &h = ph[t / 2][m], &r = pl[t / 2][m];
        (t % 2 ? h.y : h.x) = hi;
        (t % 2 ? r.y : r.x) = lo;
      }
      l[m] = l[m] * alpha[m] + sum;  // this lane's share of the row sum
    }
    bool moved = false;
#pragma unroll
    for (int m = 0; m < RT; ++m) moved |= alpha[m] != 1.f;
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int t = 0; t < VT; ++t)
#pragma unroll
        for (int e = 0; e < 2 * RT; ++e) o[t][e] *= alpha[e >> 1];
    }
    const uint32_t sv = (uint32_t)__cvta_generic_to_shared(st + KEYS * KD * 64);
    const uint32_t vaddr = sv + (((lane & 7) + ((lane >> 3) & 1) * 8) * vld + (lane >> 4) * 8) * 2;
#pragma unroll
    for (int t = 0; t < VT; t += 2) {
      if (t * 8 < p.vdim) {
#pragma unroll
        for (int k = 0; k < KT / 2; ++k) {
          uint32_t v0, v1, v2, v3;  // 16 keys of value tiles t (v0, v1) and t + 1 (v2, v3)
          asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                       : "=r"(v0), "=r"(v1), "=r"(v2), "=r"(v3)
                       : "r"(vaddr + k * 32 * vld + t * 16));
          wd_mma(o[t], ph[k][0], ph[k][RT - 1], v0, v1);
          wd_mma(o[t + 1], ph[k][0], ph[k][RT - 1], v2, v3);
          wd_mma(o[t], pl[k][0], pl[k][RT - 1], v0, v1);
          wd_mma(o[t + 1], pl[k][0], pl[k][RT - 1], v2, v3);
        }
      }
    }
    __syncwarp();  // every lane has read the stage before it is refilled
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  // From here on one warp per head; features c of a lane: (lane + 32 u) * 4 .. The gates are asked for before they are needed.
  constexpr int CH = (VT * 8 + 127) / 128, MINE = HEADS / SD_WARPS;
  uint2 gates[MINE][CH];
  {
    const __nv_bfloat16* gate = row + (long long)(p.H + p.G) * p.dim + (long long)p.G * p.vdim + (long long)h0 * p.vdim;
#pragma unroll
    for (int i = 0; i < MINE; ++i)
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const int r = warp + i * SD_WARPS, c = (lane + 32 * u) * 4;
        gates[i][u] = p.gated && r < nh && c < p.vdim ? *reinterpret_cast<const uint2*>(gate + (long long)r * p.vdim + c)
                                                      : make_uint2(0u, 0u);
      }
  }
#pragma unroll
  for (int m = 0; m < RT; ++m) {
    l[m] += __shfl_xor_sync(0xffffffffu, l[m], 1);
    l[m] += __shfl_xor_sync(0xffffffffu, l[m], 2);
    if (j == 0) {
      sm[warp][quad + 8 * m] = mx[m];
      sl[warp][quad + 8 * m] = l[m];
    }
  }
  __syncthreads();  // all rings are idle: their memory holds the warps' outputs from here on
  float* so = reinterpret_cast<float*>(smem);  // [SD_WARPS][HEADS][vdim + 8]
  const int old = p.vdim + 8;                  // the padding keeps the quads' stores in different banks
#pragma unroll
  for (int t = 0; t < VT; ++t) {
    if (t * 8 < p.vdim) {
#pragma unroll
      for (int m = 0; m < RT; ++m)
        *reinterpret_cast<float2*>(so + (warp * HEADS + quad + 8 * m) * old + t * 8 + 2 * j) =
            make_float2(o[t][2 * m], o[t][2 * m + 1]);
    }
  }
  // ---- merge of the warps: their weights, and the sums of the weights --------------------------------------------------------
  if (threadIdx.x < HEADS) {
    const int r = threadIdx.x;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < SD_WARPS; ++w) m = fmaxf(m, sm[w][r]);
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < SD_WARPS; ++w) {
      const float f = sm[w][r] == -INFINITY ? 0.f : exp2f(sm[w][r] - m);
      fw[w][r] = f;
      ll += sl[w][r] * f;  // (a sum that is not a number stays none)
    }
    own[r] = make_float2(m, ll);
  }
  __syncthreads();
  auto merged = [&](int r, int c) {  // head r, features c .. c + 3, over this CTA's warps
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < SD_WARPS; ++w) {
      const float f = fw[w][r];
      const float4 x = *reinterpret_cast<const float4*>(so + (w * HEADS + r) * old + c);
      if (f != 0.f) a = make_float4(a.x + x.x * f, a.y + x.y * f, a.z + x.z * f, a.w + x.w * f);
    }
    return a;
  };
  // ---- all parts: these keys, then what the prefix kernel has of the shared and of the sequence's own ones ----------------------------------
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int4* at = reinterpret_cast<const int4*>(d.plan + b);
  const int4 pa = __ldcg(at), pb = __ldcg(at + 1), pc = __ldcg(at + 2);
  const XlRanges ranges{pb.z ? pb.y / pb.z : 1, pb.z ? pb.y % pb.z : 0};
  const float sink = p.sink * 1.4426950408889634f;
#pragma unroll
  for (int i = 0; i < MINE; ++i) {
    const int r = warp + i * SD_WARPS;
    if (r >= nh) break;
    const int hh = h0 - g * R + r;
    // two sources: the tile of the group and the tile of the sequence; of each one CTA's part for each warpgroup from its first block on, then those of
    // the CTAs that follow
    int idx[2] = {pa.w + hh, hh}, c0[2] = {0, 0}, parts[2] = {0, 0};
    const int n_of[2] = {pa.y, pb.w};
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (n_of[k]) {
        const int x = k ? pc.x + (g * ((R + TILE_M - 1) / TILE_M) + idx[k] / TILE_M) * n_of[k] : pa.x + (g * pa.z + idx[k] / TILE_M) * n_of[k];
        c0[k] = ranges.owner(x);
        parts[k] = 2 * (ranges.owner(x + n_of[k] - 1) - c0[k] + 1);
      }
    const long long row0[2] = {pb.x + idx[0], (long long)b * R + idx[1]};
    const int all = parts[0] + parts[1];
    auto place = [&](int k, bool& main) -> long long {
      const int q = k < parts[0] ? k : k - parts[0], src = k < parts[0] ? 0 : 1, m = q & 1, c = q >> 1;
      main = c == 0;
      return main ? ((long long)(src * 2 + m) * p.G + g) * p.B * R + (src ? row0[1] : row0[0])
                  : ((long long)((src ? c0[1] : c0[0]) + c) * 2 + m) * TILE_M + (src ? idx[1] : idx[0]) % TILE_M;
    };
    auto stat = [&](int k) {
      bool main;
      const long long e = place(k, main);
      return __ldcg((main ? d.main_s : d.extra_s) + e);
    };
    float2 mine_s = lane < all ? stat(lane) : make_float2(-INFINITY, 0.f);  // of the first 32 parts
    float m = fmaxf(fmaxf(sink, own[r].x), mine_s.x);
    for (int k = lane + 32; k < all; k += 32) m = fmaxf(m, stat(k).x);
    m = xl_warp_max(m);
    float4 acc[CH];
    float total = sink == -INFINITY ? 0.f : exp2f(sink - m);
    {
      const float f = own[r].x == -INFINITY ? 0.f : exp2f(own[r].x - m);
      total += f * own[r].y;  // (a sum that is not a number stays none)
#pragma unroll
      for (int u = 0; u < CH; ++u) {
        const int c = (lane + 32 * u) * 4;
        acc[u] = c < p.vdim ? merged(r, c) : make_float4(0.f, 0.f, 0.f, 0.f);
        acc[u] = make_float4(acc[u].x * f, acc[u].y * f, acc[u].z * f, acc[u].w * f);
      }
    }
    for (int k0 = 0; k0 < all; k0 += 32) {
      if (k0) mine_s = k0 + lane < all ? stat(k0 + lane) : make_float2(-INFINITY, 0.f);
      const float f = mine_s.x == -INFINITY ? 0.f : exp2f(mine_s.x - m);
      total += xl_warp_sum(f * mine_s.y);
      const int n = min(32, all - k0);
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        if (fk == 0.f) continue;
        bool main;
        const long long e = place(k0 + k, main);
        const float* src = (main ? d.main_o : d.extra_o) + e * p.vdim;
#pragma unroll
        for (int u = 0; u < CH; ++u) {
          const int c = (lane + 32 * u) * 4;
          if (c < p.vdim) {
            const float4 x = __ldcg(reinterpret_cast<const float4*>(src + c));
            acc[u] = make_float4(acc[u].x + x.x * fk, acc[u].y + x.y * fk, acc[u].z + x.z * fk, acc[u].w + x.w * fk);
          }
        }
      }
    }
    __nv_bfloat16* out = p.out + (long long)b * p.ldo + (long long)(h0 + r) * p.vdim;
#pragma unroll
    for (int u = 0; u < CH; ++u) {
      const int c = (lane + 32 * u) * 4;
      if (c >= p.vdim) continue;
      float v[4] = {acc[u].x / total, acc[u].y / total, acc[u].z / total, acc[u].w / total};
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

constexpr int SD_RING_LIMIT = 68 * 1024;  // three CTAs per SM

template <int KD, int VT, int RT> int launch_decode_rows(SharedDecodeParams d, cudaStream_t s) {
  const SharedParams& p = d.p;
  const int stage = sd_stage_bytes(sd_keys(KD, VT), KD, p.vdim) * SD_WARPS;
  d.stages = 4 * stage <= SD_RING_LIMIT ? 4 : (3 * stage <= SD_RING_LIMIT ? 3 : 2);
  int bytes = d.stages * stage;
  const int merge = SD_WARPS * 8 * RT * (p.vdim + 8) * 4;
  if (bytes < merge) bytes = merge;
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(shared_attn_decode_kernel<KD, VT, RT>, bytes, smem));
  const int hchunks = (p.H / p.G + 8 * RT - 1) / (8 * RT);
  const cudaError_t e = xl_launch_overlapped(shared_attn_decode_kernel<KD, VT, RT>, dim3(p.G * hchunks, p.B), dim3(SD_WARPS * 32),
                                             (size_t)bytes, s, d);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

template <int KD, int VT> int launch_decode(const SharedDecodeParams& d, cudaStream_t s) {
  return d.p.H / d.p.G <= 8 ? launch_decode_rows<KD, VT, 1>(d, s) : launch_decode_rows<KD, VT, 2>(d, s);
}

template <int DK, int VD> int launch_prefix(const PrefixParams& a, const void* kc, const void* vc, int ctas, cudaStream_t s) {
  using L = PrefixSmem<DK, VD>;
  const SharedParams& p = a.p;
  CUtensorMap mk, mv;
  int r = make_map_bf16(&mk, kc, (long long)p.B * p.G * p.Smax, p.dim, p.dim, BKV);
  if (r) return r;
  r = make_map_bf16(&mv, vc, (long long)p.B * p.G * p.Smax, p.vdim, p.vdim, 64);
  if (r) return r;
  const int bytes = L::total(p.B);
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(shared_attn_prefix_kernel<DK, VD>, bytes, smem));
  const cudaError_t e = xl_launch_overlapped(shared_attn_prefix_kernel<DK, VD>, dim3(ctas), dim3(SA_THREADS), (size_t)bytes, s, mk, mv, a);
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

// floats of scratch memory for xl_shared_attn_decode with `ctas` CTAs for long runs of keys
XL_API long long xl_shared_attn_decode_scratch(int B, int H, int vdim, int ctas) { return B * 12LL + (4LL * B * H + ctas * 2LL * TILE_M) * (vdim + 2); }

// One token per sequence (rows of proj = sequences), bf16, in two launches. Sizes and alignment as for portions, at most 512 sequences. Queries and
// keys are normalised and keys and values appended here. ctas: SMs of the device. scratch: xl_shared_attn_decode_scratch floats, 16-byte aligned.
// read_ahead: positions, counts, leads and caches were complete before the previous launch of the stream.
XL_API int xl_shared_attn_decode(const void* proj, long long ld, const float* wq, const float* wk, void* kc, void* vc, void* out, long long ldo,
                                 const int* pos, const int* count, const int* lead, const int* shared, int B, int H, int G, int dim, int vdim,
                                 int Smax, int window, int keep_first, int gated, float scale, float sink, float eps, int ctas,
                                 float* scratch, int read_ahead, int* err, cudaStream_t s) {
  if (B < 1 || B > PF_MAX_BATCH || G < 1 || H < 1 || H % G || H > 4096 || Smax < 1 || window < 0 || keep_first < 0 || !(scale > 0.f) || !lead || !shared ||
      !wq || !wk || ctas < 1 || ctas > 4096 || !scratch || ((uintptr_t)scratch & 15))
    return -1;
  if (!tensor_sizes(proj, ld, kc, vc, out, ldo, B, 1, H, G, dim, vdim, Smax, gated)) return -1;
  SharedParams p = {};
  p.proj = (const __nv_bfloat16*)proj; p.ld = ld; p.wq = wq; p.pos = pos; p.count = count; p.prefix = {lead, shared};
  p.out = (__nv_bfloat16*)out; p.ldo = ldo; p.B = B; p.T = 1; p.H = H; p.G = G; p.dim = dim; p.vdim = vdim; p.Smax = Smax;
  p.window = window; p.keep_first = keep_first; p.gated = gated; p.scale = scale; p.sink = sink; p.eps = eps; p.err = err;
  PrefixParams a = {};
  a.p = p;
  a.plan = (PrefixPlan*)scratch;
  static_assert(sizeof(PrefixPlan) == 48, "12 floats of scratch memory per sequence");
  a.main_o = scratch + 12LL * B;
  a.extra_o = a.main_o + 4LL * B * H * vdim;
  a.main_s = (float2*)(a.extra_o + 2LL * ctas * TILE_M * vdim);
  a.extra_s = a.main_s + 4LL * B * H;
  a.read_ahead = read_ahead;
  SharedDecodeParams d = {};
  d.p = p; d.kc = (__nv_bfloat16*)kc; d.vc = (__nv_bfloat16*)vc; d.wk = wk;
  d.main_o = a.main_o; d.extra_o = a.extra_o; d.main_s = a.main_s; d.extra_s = a.extra_s; d.plan = a.plan;
  int r;
  if (dim <= 64) r = vdim <= 64 ? launch_prefix<64, 64>(a, kc, vc, ctas, s) : launch_prefix<64, 128>(a, kc, vc, ctas, s);
  else r = vdim <= 64 ? launch_prefix<128, 64>(a, kc, vc, ctas, s) : launch_prefix<128, 128>(a, kc, vc, ctas, s);
  if (r) return r;
#define XL_SD(KD) return vdim <= 64 ? launch_decode<KD, 8>(d, s) : launch_decode<KD, 16>(d, s);
  if (dim <= 32) { XL_SD(1) }
  if (dim <= 64) { XL_SD(2) }
  XL_SD(4)
#undef XL_SD
}
