// Sliding-window attention of a portion of tokens against a key / value cache of 8 bits on the 5th-generation tensor cores (tcgen05).
// Mathematics of attention_window.cu, layouts of attention_q8.cuh; xl_q8_append_expand (attention_q8.cu) lays out what is read here.
//
// The R query heads that read one key / value head are consecutive rows (token-major) of the normalised queries. One CTA owns
// 256 of these rows as two tiles of 128 and walks the blocks of 64 keys that any of them sees: the codes of the kept first tokens, those
// of the windows, then the raw rows of the portion from the start of the block in progress. A query sees raw rows of its own block and
// codes of earlier blocks; which is which is a mask like any other.
//   warp 0       TMA producer : both query tiles once, key blocks (lane 0) and value blocks (lane 1) through rings
//   warps 1, 10  MMA issuers  : of a tile each, S_m = Q_m K^T into TMEM, O_m += P_m V
//   warps 2..5   softmax of tile 0, warps 6..9 of tile 1: one thread per row; running maximum and sum in fp32 start with the
//                               sink, lazy rescaling of O_m in TMEM
// Codes are fp16 keys and bf16 values, both exact: the scale of a block multiplies the scores, that of its values the weights, which
// replace S in TMEM as two bf16 numbers each (value and rounding error): rounded once to bf16 they would add as much error as the
// rounding of the result does, and save 7 % of the time. Queries and raw keys are fp16 in units of a power of two above their norm's
// factors.
//
// 32 heads on 8 of 128 features: 2 x 4096 tokens, window 1024, 266 us; 2 x 515 tokens after 6000, 170 us (600 TFLOP/s of visible keys,
// the tensor pipe 46 % busy). What bounds it is the chain of a tile: scores, softmax, weights, product. A tile has two buffers of scores
// of 64 keys each, so that the next scores are there when a softmax ends, and an issuer of its own, so that no tile's products wait
// behind what holds up the other's: with one buffer of 128 keys a tile's warps waited 1700 of 4500 cycles per 128 keys for the tensor
// core's answer, with one issuer for both tiles, in a fixed order or going by what is ready, 1500 of 3000 cycles per 64 keys (clock stamps
// of the second call). The softmax takes a block's scores into registers at once and works on pairs of fp32 numbers (fma.rn.f32x2); its
// exponentials alone occupy the special-function unit half of the time.
// Expanding codes outside this kernel moves five bytes per code once per portion, where every CTA would convert every block again next to a
// softmax that fills the issue slots.
//
// TMEM columns: [m * 128 + 64 * buffer, + 64) S_m / P_m, [256, 256 + VD) O_0, [256 + VD, 256 + 2 VD) O_1. One CTA per SM. Every wait
// is bounded (see tcgen05.cuh).
#include "attention_q8.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int TILE_M = 128;
constexpr int BKV = Q8_BLOCK;
constexpr int UMMA_K = 16;
constexpr int NUM_THREADS = 96 + 2 * 128;
constexpr uint32_t TMEM_COLS = 512;

enum { ERR_Q = 92, ERR_KV_FULL = 93, ERR_KV_EMPTY = 94, ERR_S = 95, ERR_P = 96, ERR_PV = 97 };

struct Q8PortionParams {
  const int *pos, *count;
  const __nv_bfloat16* gate;  // first gate column of the projections, or null
  long long ldg;
  __nv_bfloat16* out;
  long long ldo;
  int T, H, G, dim, vdim, blocks, held, raw_rows, window, keep_first;
  float scale, sink;
  const float *ks, *vs, *wq, *wk;  // scales of the blocks (B, G, blocks), factors of the norms
  const float* raw_unit;           // (B, G, q8_touched(T)): 1, or NaN for a raw block with a value that is not finite
  int* err;
};

using namespace xl_tc;

// two fp32 numbers in a register pair
__device__ __forceinline__ uint64_t pair_of(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void halves_of(uint64_t p, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p)); }
__device__ __forceinline__ uint64_t pair_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t pair_mul(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t pair_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// Descriptors of 128-byte-swizzled tiles (see make_smem_desc) in two words: the upper one is the same for all of them, in the lower one
// an offset inside a tile is an addition. Building each of a block's 24 descriptors from its address kept the one issuing thread busy
// for longer than the softmax takes.
constexpr uint32_t DESC_HI = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t lbo_bytes) { return ((addr & 0x3FFFFu) >> 4) | ((lbo_bytes >> 4) << 16); }
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
      ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(DESC_HI), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
      ::"r"(d), "r"(a), "r"(b_lo), "r"(DESC_HI), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
// bits a .. b - 1 of a word, whatever lies outside it
__device__ __forceinline__ uint32_t bits_of(int a, int b) {
  a = max(a, 0);
  b = min(b, 32);
  return b > a ? (0xffffffffu >> (32 - (b - a))) << a : 0u;
}

// DK: 64 or 128, query / key features rounded up; VD: 64 or 128, value features rounded up. Features past the real sizes are zero
// in the key and value blocks (TMA fills what lies outside the rows), so they add nothing.
template <int DK, int VD> struct Q8Smem {
  static constexpr int K_STAGES = DK == 64 ? 6 : 4;
  static constexpr int V_STAGES = VD == 64 ? 6 : 4;
  static constexpr int Q_BYTES = TILE_M * DK * 2;  // per tile: DK/64 boxes of (128 rows x 128 B)
  static constexpr int K_BYTES = BKV * DK * 2;     // DK/64 boxes of (64 rows x 128 B)
  static constexpr int V_BYTES = BKV * VD * 2;     // VD/64 boxes of (64 rows x 128 B)
  static constexpr int TILE_BYTES = 2 * Q_BYTES + K_STAGES * K_BYTES + V_STAGES * V_BYTES;
  static constexpr int NEEDED = TILE_BYTES + 1024 /*alignment*/ + 512 /*barriers*/;
  // more than half of an SM's shared memory: two CTAs, each holding all of TMEM, never meet on an SM
  static constexpr int TOTAL = NEEDED > 120 * 1024 ? NEEDED : 120 * 1024;
};

template <int DK, int VD>
__global__ void __launch_bounds__(NUM_THREADS, 1)
    q8_attn_tcgen05_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                           const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_raw_k,
                           const __grid_constant__ CUtensorMap map_raw_v, const Q8PortionParams p) {
  using L = Q8Smem<DK, VD>;
  static_assert(L::TOTAL <= 227 * 1024, "shared memory");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* sK = smem + 2 * L::Q_BYTES;
  uint8_t* sV = sK + L::K_STAGES * L::K_BYTES;
  uint64_t* bars = (uint64_t*)(smem + L::TILE_BYTES);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;    // [6]
  uint64_t* k_empty = bars + 7;   // [6]
  uint64_t* v_full = bars + 13;   // [6]
  uint64_t* v_empty = bars + 19;  // [6]
  uint64_t* s_full = bars + 25;   // [2 m + buffer]
  uint64_t* p_full = bars + 29;
  uint64_t* pv_done = bars + 33;
  uint32_t* tmem_base_slot = (uint32_t*)(bars + 37);
  volatile int* abort_flag = (volatile int*)(tmem_base_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x, b = blockIdx.z, R = p.H / p.G;
  const int cnt = min(p.count[b], p.T), pos = p.pos[b];
  const long long rows = (long long)cnt * R;                                  // real rows of this sequence and key / value head
  const long long f0 = (long long)(gridDim.y - 1 - blockIdx.y) * 2 * TILE_M;  // the tiles with the most keys first
  if (f0 >= rows || pos < 0 || (long long)pos + cnt > (long long)p.blocks * BKV) return;
  const int tiles = f0 + TILE_M < rows ? 2 : 1;
  const int p_first = pos + (int)(f0 / R), p_last = pos + (int)((min(rows, f0 + 2 * TILE_M) - 1) / R);
  // blocks: codes of kept tokens before every window of this CTA, codes from there to the last block in progress, raw ones
  const int base = pos / BKV, own_first = p_first / BKV, own_last = p_last / BKV;  // base: block of the first raw row
  const int w0 = window_range(p_first, p.window, 0).first / BKV;
  const int kept = min(min((int)(((long long)p.keep_first + BKV - 1) / BKV), w0), own_last);
  const int n_code = kept + max(0, own_last - w0), n_kv = n_code + own_last - own_first + 1;
  auto block_of = [&](int j) { return j < kept ? j : (j < n_code ? w0 + j - kept : own_first + j - n_code); };

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < 6; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], tiles);
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], tiles);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&s_full[s], 1);
      mbar_init(&p_full[s], 4);
      mbar_init(&pv_done[s], 1);
    }
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
  xl_grid_launch_dependents();  // TMEM is held: a successor that allocates some on this SM cannot come first

  if (warp == 0) {
    // lane 0: queries and key blocks, lane 1: value blocks; each waits only on its own ring
    if (lane < 2) {
      const bool for_k = lane == 0;
      if (for_k) {
        mbar_expect_tx(q_full, tiles * L::Q_BYTES);
        for (int m = 0; m < tiles; ++m)
#pragma unroll
          for (int kb = 0; kb < DK / 64; ++kb)
            tma_load_2d(sQ + m * L::Q_BYTES + kb * (TILE_M * 128), &map_q, q_full, kb * 64,
                        (int)((long long)(b * p.G + g) * p.T * R + f0) + m * TILE_M);
      }
      const int stages = for_k ? L::K_STAGES : L::V_STAGES;
      uint64_t* full = for_k ? k_full : v_full;
      uint64_t* empty = for_k ? k_empty : v_empty;
      const Q8Slots slots = q8_slots(pos, p.window, p.keep_first);
      bool ok = true;
      int issued = 0;
      for (int j = 0; j < n_kv && ok; ++j) {
        const bool raw = j >= n_code;
        const int st = j % stages, blk = block_of(j);
        const int row = raw ? (b * p.G + g) * p.raw_rows + (blk - base) * BKV : ((b * p.G + g) * p.held + slots.of(blk)) * BKV;
        if (j >= stages) {
          ok = mbar_wait(&empty[st], (uint32_t)(j / stages - 1) & 1u, abort_flag, p.err, ERR_KV_EMPTY);
          if (!ok) break;
        }
        if (for_k) {
          mbar_expect_tx(&full[st], L::K_BYTES);
#pragma unroll
          for (int kb = 0; kb < DK / 64; ++kb)
            tma_load_2d(sK + st * L::K_BYTES + kb * (BKV * 128), raw ? &map_raw_k : &map_k, &full[st], kb * 64, row);
        } else {
          mbar_expect_tx(&full[st], L::V_BYTES);
#pragma unroll
          for (int jn = 0; jn < VD / 64; ++jn)
            tma_load_2d(sV + st * L::V_BYTES + jn * (BKV * 128), raw ? &map_raw_v : &map_v, &full[st], jn * 64, row);
        }
        issued = j + 1;
      }
      if (!ok || *abort_flag) {
        // loads in flight target this CTA's shared memory: give them a bounded time to land before the CTA ends
        if (for_k)
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(q_full, 0); ++i) {}
        for (int j = max(0, issued - stages); j < issued; ++j)
          for (uint32_t i = 0; i < MBAR_SPIN_LIMIT && !mbar_try_wait(&full[j % stages], (uint32_t)(j / stages) & 1u); ++i) {}
      }
    }
  } else if (warp == 1 || warp == 10) {
    const int m = warp == 1 ? 0 : 1;  // row tile whose products this warp issues
    if (m < tiles && elect_one()) {
      // fp32 accumulators. S: fp16, both K-major, N = BKV. O: bf16, A (P) from TMEM, B (V) MN-major (bit 16), N = VD.
      const uint32_t idesc_s = (1u << 4) | ((uint32_t)(BKV >> 3) << 17) | ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t idesc_o = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(VD >> 3) << 17) |
                               ((uint32_t)(TILE_M >> 4) << 24);
      const uint32_t q_lo = desc_lo(smem_u32(sQ + m * L::Q_BYTES), 16), k_desc = desc_lo(smem_u32(sK), 16),
                     v_desc = desc_lo(smem_u32(sV), BKV * 128);
      bool ok = mbar_wait(q_full, 0, abort_flag, p.err, ERR_Q);
      auto issue_scores = [&](int j) -> bool {
        const int st = j % L::K_STAGES, buf = 2 * m + (j & 1);
        if (!mbar_wait(&k_full[st], (uint32_t)(j / L::K_STAGES) & 1u, abort_flag, p.err, ERR_KV_FULL)) return false;
        // the buffer still holds P of the block before the last one until its product has been taken
        if (j > 1 && !mbar_wait(&pv_done[buf], (uint32_t)((j - 2) >> 1) & 1u, abort_flag, p.err, ERR_PV)) return false;
        tcgen05_fence_after();
        const uint32_t k_lo = k_desc + st * (L::K_BYTES >> 4);
#pragma unroll
        for (int kb = 0; kb < DK / 64; ++kb)
#pragma unroll
          for (int k = 0; k < 64 / UMMA_K; ++k)
            mma_ss(tmem_base + buf * BKV, q_lo + ((kb * (TILE_M * 128) + k * (UMMA_K * 2)) >> 4),
                   k_lo + ((kb * (BKV * 128) + k * (UMMA_K * 2)) >> 4), idesc_s, (kb | k) != 0);
        tcgen05_commit(&k_empty[st]);
        tcgen05_commit(&s_full[buf]);
        return true;
      };
      for (int j = 0; j < min(2, n_kv) && ok; ++j) ok = issue_scores(j);
      for (int j = 0; j < n_kv && ok; ++j) {
        const int st = j % L::V_STAGES, buf = 2 * m + (j & 1);
        ok = mbar_wait(&v_full[st], (uint32_t)(j / L::V_STAGES) & 1u, abort_flag, p.err, ERR_KV_FULL) &&
             mbar_wait(&p_full[buf], (uint32_t)(j >> 1) & 1u, abort_flag, p.err, ERR_P);
        if (!ok) break;
        tcgen05_fence_after();
        const uint32_t v_lo = v_desc + st * (L::V_BYTES >> 4);
#pragma unroll
        for (int part = 0; part < 2; ++part)  // rounded weights, then their rounding errors
#pragma unroll
          for (int k = 0; k < BKV / UMMA_K; ++k)
            mma_ts(tmem_base + 4 * BKV + m * VD, tmem_base + buf * BKV + part * (BKV / 2) + k * (UMMA_K / 2),
                   v_lo + ((k * (UMMA_K * 128)) >> 4), idesc_o, (j | part | k) != 0);
        tcgen05_commit(&v_empty[st]);
        tcgen05_commit(&pv_done[buf]);
        if (j + 2 < n_kv) ok = issue_scores(j + 2);
      }
    }
  } else if ((warp < 6 ? 0 : 1) < tiles) {
    const int m = warp < 6 ? 0 : 1;           // row tile of this warpgroup
    const int qtr = warp & 3;                 // TMEM lane quarter this warp may access
    const int r = qtr * 32 + lane;            // row inside the tile
    const long long f = f0 + m * TILE_M + r;  // (token, head of the group)
    const int t = (int)(f / R), hh = (int)(f - (long long)t * R);
    const int qpos = pos + t, own = qpos / BKV * BKV;
    const int lo = window_range(qpos, p.window, 0).first, lo_last = window_range(p_last, p.window, 0).first;
    const uint32_t lane_base = (uint32_t)(qtr * 32) << 16;
    const uint32_t tmem_o = tmem_base + lane_base + 4 * BKV + m * VD;
    const float unit_q = q8_norm_unit(p.wq, p.dim, lane), unit_k = q8_norm_unit(p.wk, p.dim, lane);
    const float c = p.scale * 1.4426950408889634f * unit_q;
    const float *ks = p.ks + (long long)(b * p.G + g) * p.blocks, *vs = p.vs + (long long)(b * p.G + g) * p.blocks;
    const float* raw_unit = p.raw_unit + (long long)(b * p.G + g) * q8_touched(p.T);
    // Scores differ in their factors: the maximum is held in units of the exponent. A factor is never zero (the scale of a block of zeros):
    // minus infinity, a masked score, has to stay what it is; the values' factor is finite: a weight of zero has to stay zero. Where the
    // scale is NaN (a block that held a number that is not finite; its codes are zero) the sum of every row that reads the block becomes NaN,
    // and no other.
    float mx = p.sink * 1.4426950408889634f, l = p.sink == -INFINITY ? 0.f : 1.f;
    float ch = 0.f, vh = 0.f;  // factors of the next block
    auto ask = [&](int j) {
      if (j < n_code) {
        const int blk = block_of(j);
        ch = ks[blk];
        vh = vs[blk];
      } else {
        ch = unit_k;
        vh = raw_unit[block_of(j) - base];
      }
    };
    ask(0);
    bool ok = true;
    for (int j = 0; j < n_kv && ok; ++j) {
      const int buf = 2 * m + (j & 1);
      const bool raw = j >= n_code;
      const float fs = fmaxf(c * ch, 1e-37f), fv = fminf(vh, 1e37f);
      const bool spoiled = q8_spoiled(ch, vh);
      if (j + 1 < n_kv) ask(j + 1);
      // keys that the row sees: of a raw block its own, of codes the earlier ones; its window, and the kept first tokens
      const int blk = block_of(j), col0 = blk * BKV;
      uint32_t vis[2] = {0xffffffffu, 0xffffffffu};
      if (raw || blk >= own_first || (col0 < lo_last && col0 + BKV > p.keep_first)) {  // else every row of this CTA sees all of it
        const int first = raw ? own : 0, end = raw ? qpos + 1 : own, from = max(lo, first);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = col0 + k * 32;
          vis[k] = bits_of(from - at, end - at) | bits_of(first - at, min(p.keep_first, end) - at);
        }
      }
      if (spoiled && (vis[0] | vis[1])) l = __uint_as_float(0x7fc00000u);
      const uint32_t tmem_s = tmem_base + lane_base + buf * BKV;
      ok = mbar_wait_warp(&s_full[buf], (uint32_t)(j >> 1) & 1u, abort_flag, p.err, ERR_S);
      if (!ok) break;
      tcgen05_fence_after();
      uint32_t s[2][32];
      tmem_ld_32x32b_x32(tmem_s, s[0]);
      tmem_ld_32x32b_x32(tmem_s + 32, s[1]);
      tmem_ld_wait();
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        if (vis[k] != 0xffffffffu) {
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(vis[k] >> i & 1u)) s[k][i] = 0xff800000u;
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) top[i & 3] = fmaxf(top[i & 3], __uint_as_float(s[k][i]));
      }
      const float m_blk = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * fs;
      // the reference maximum moves (and O, l are rescaled) only when the exponent would exceed 2^8
      const bool move = m_blk > -INFINITY && (mx == -INFINITY || m_blk - mx > 8.f);
      const float m_new = move ? m_blk : mx;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;  // a row without a visible key yet keeps weight 0
      const float alpha = (move && mx != -INFINITY) ? fast_exp2(mx - m_use) : 1.f;
      uint64_t sums[2] = {0, 0};
      const uint64_t f2 = pair_of(fs, fs), v2 = pair_of(fv, fv), m2 = pair_of(-m_use, -m_use), minus_one = pair_of(-1.f, -1.f);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t w[16], err[16];  // rounded weights, their rounding errors
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x, y;
          halves_of(pair_fma(pair_of(__uint_as_float(s[k][2 * i]), __uint_as_float(s[k][2 * i + 1])), f2, m2), x, y);
          const uint64_t e2 = pair_of(fast_exp2(x), fast_exp2(y));
          sums[i & 1] = pair_add(sums[i & 1], e2);
          const uint64_t x2 = pair_mul(e2, v2);
          halves_of(x2, x, y);
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[i]) : "f"(y), "f"(x));
          halves_of(pair_fma(pair_of(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), minus_one, x2), x, y);
          asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(err[i]) : "f"(y), "f"(x));
        }
        tmem_st_32x32b_x16(tmem_s + k * 16, w);
        tmem_st_32x32b_x16(tmem_s + BKV / 2 + k * 16, err);
      }
      float x, y;
      halves_of(pair_add(sums[0], sums[1]), x, y);
      l = l * alpha + (x + y);
      mx = m_new;
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
        // O is at rest once the product of the block before this one has been taken: the next one waits for these weights
        ok = mbar_wait_warp(&pv_done[2 * m + ((j - 1) & 1)], (uint32_t)((j - 1) >> 1) & 1u, abort_flag, p.err, ERR_PV);
        if (!ok) break;
        tcgen05_fence_after();
#pragma unroll 1
        for (int k = 0; k < VD / 32; ++k) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tmem_o + k * 32, o);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
          tmem_st_32x32b_x32(tmem_o + k * 32, o);
        }
      }
      tmem_st_wait();
      tcgen05_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf]);
    }
    // ---- output: divided by the sum, gated -------------------------------------------------------------------------------
    ok = ok && mbar_wait_warp(&pv_done[2 * m + ((n_kv - 1) & 1)], (uint32_t)((n_kv - 1) >> 1) & 1u, abort_flag, p.err, ERR_PV);
    if (ok) {
      tcgen05_fence_after();
      const float inv = 1.f / l;
      const long long at = (long long)b * p.T + t, col = (long long)(g * R + hh) * p.vdim;
      const __nv_bfloat16* grow = p.gate ? p.gate + at * p.ldg + col : nullptr;
      __nv_bfloat16* orow = p.out + at * p.ldo + col;
#pragma unroll 1
      for (int k = 0; k < VD / 32; ++k) {
        uint4 gates[4];
        if (grow && f < rows) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (k * 32 + q * 8 < p.vdim) gates[q] = *reinterpret_cast<const uint4*>(grow + k * 32 + q * 8);
        }
        uint32_t o[32];
        tmem_ld_32x32b_x32(tmem_o + k * 32, o);
        tmem_ld_wait();
        if (f < rows) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int c0 = k * 32 + q * 8;
            if (c0 < p.vdim) {
              float v[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(o[q * 8 + e]) * inv;
              if (grow) {
                const uint32_t gw[4] = {gates[q].x, gates[q].y, gates[q].z, gates[q].w};
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  v[e] *= __fdividef(1.f, 1.f + __expf(-(e & 1 ? __uint_as_float(gw[e >> 1] & 0xffff0000u) : __uint_as_float(gw[e >> 1] << 16))));
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

template <int DK, int VD>
int launch(const void* q, const void* kx, const void* vx, const void* raw_k, const void* raw_v, const Q8PortionParams& p, int B, cudaStream_t s) {
  using L = Q8Smem<DK, VD>;
  CUtensorMap mq, mk, mv, mrk, mrv;  // fp16 rows travel like bf16 ones
  const long long heads = (long long)B * p.G;
  int r = make_map_bf16(&mq, q, (long long)B * p.T * p.H, p.dim, p.dim, TILE_M);
  if (!r) r = make_map_bf16(&mk, kx, heads * p.held * BKV, p.dim, p.dim, BKV);
  if (!r) r = make_map_bf16(&mv, vx, heads * p.held * BKV, p.vdim, p.vdim, BKV);
  if (!r) r = make_map_bf16(&mrk, raw_k, heads * p.raw_rows, p.dim, p.dim, BKV);
  if (!r) r = make_map_bf16(&mrv, raw_v, heads * p.raw_rows, p.vdim, p.vdim, BKV);
  if (r) return r;
  static XlPerDevice smem;
  XL_TRY(xl_allow_smem(q8_attn_tcgen05_kernel<DK, VD>, L::TOTAL, smem));
  const long long rows = (long long)p.T * (p.H / p.G);
  const dim3 grid(p.G, (unsigned)((rows + 2 * TILE_M - 1) / (2 * TILE_M)), B);
  q8_attn_tcgen05_kernel<DK, VD><<<grid, NUM_THREADS, L::TOTAL, s>>>(mq, mk, mv, mrk, mrv, p);
  return (int)cudaGetLastError();
}

}  // namespace

// After xl_q8_append_expand: q16 (B, G, T, H/G, dim) fp16, codes as fp16 kx (B, G, held * 64, dim) and bf16 vx (.., vdim), raw rows as
// fp16 raw_k and bf16 raw_v (B, G, raw_rows, dim | vdim), raw_unit (B, G, (T + 126) / 64); ks, vs (B, G, blocks) the scales, wq and wk
// the factors of the norms; gate: first gate column of the projections (row stride ldg), or null; out (B*T, ldo). dim, vdim multiples of
// 8 and at most 128; ldg, ldo multiples of 8; all pointers but those of fp32 numbers 16-byte aligned. Rows past count[b] are not written. err: device int for the code of a wait that gave up.
// Returns 0, a CUDA error code, or a negative value for arguments this kernel does not take.
XL_API int xl_q8_attn_tcgen05(const void* q16, const void* kx, const void* vx, int held, const void* raw_k, const void* raw_v,
                              int raw_rows, const float* raw_unit, const float* ks, const float* vs, const float* wq, const float* wk, const void* gate,
                              long long ldg, void* out, long long ldo, const int* pos, const int* count, int B, int T, int H, int G, int dim, int vdim,
                              int blocks, int window, int keep_first, float scale, float sink, int* err, cudaStream_t s) {
  if (B < 1 || B > 65535 || T < 1 || G < 1 || H < 1 || H % G || blocks < 1 || blocks > (1 << 24) || window < 0 || keep_first < 0 || !(scale > 0.f))
    return -1;
  if (dim < 8 || dim > 128 || dim % 8 || vdim < 8 || vdim > 128 || vdim % 8 || ldo % 8 || ldo < (long long)H * vdim ||
      (gate && (ldg % 8 || ldg < (long long)H * vdim)) || raw_rows < T + 2 * Q8_BLOCK || !raw_unit ||
      held < q8_held(T, blocks, window, keep_first))
    return -1;
  if (((uintptr_t)q16 | (uintptr_t)kx | (uintptr_t)vx | (uintptr_t)raw_k | (uintptr_t)raw_v | (uintptr_t)gate | (uintptr_t)out) & 15) return -1;
  const long long limit = 0x7fffffffLL - 4 * TILE_M;
  if ((long long)B * G * held * BKV > limit || (long long)B * G * raw_rows > limit || (long long)B * T * H > limit ||
      ((long long)T * (H / G) + 2 * TILE_M - 1) / (2 * TILE_M) > 65535)
    return -1;
  Q8PortionParams p = {};
  p.pos = pos; p.count = count; p.gate = (const __nv_bfloat16*)gate; p.ldg = ldg; p.out = (__nv_bfloat16*)out; p.ldo = ldo;
  p.T = T; p.H = H; p.G = G; p.dim = dim; p.vdim = vdim; p.blocks = blocks; p.held = held; p.raw_rows = raw_rows; p.window = window;
  p.keep_first = keep_first; p.scale = scale; p.sink = sink; p.ks = ks; p.vs = vs; p.wq = wq; p.wk = wk; p.raw_unit = raw_unit; p.err = err;
  if (dim <= 64) return vdim <= 64 ? launch<64, 64>(q16, kx, vx, raw_k, raw_v, p, B, s) : launch<64, 128>(q16, kx, vx, raw_k, raw_v, p, B, s);
  return vdim <= 64 ? launch<128, 64>(q16, kx, vx, raw_k, raw_v, p, B, s) : launch<128, 128>(q16, kx, vx, raw_k, raw_v, p, B, s);
}
