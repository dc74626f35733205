// Low-rank adapters of many requests beside a shared projection.
//
//   y[i] = x[i] W^T + scale[s] (x[i] A[s]^T) B[s]^T,   s = slot[i / T]: the adapter of row i's sequence (none: the second term is zero)
//
// The shared product is a kernel of its own (few rows: bound by reading W; many: by the tensor cores). Here are the two narrow ones,
// with the r numbers between them in fp32, `low` (rows, rp), rp = r rounded up to 16, filled with zeros, scale included:
//   xl_adapter_down        any type: one warp per number, which reads one row of A (40 rows x 4096, rank 16: 8 us)
//   xl_adapter_up          any type: adds the second term to the shared product in fp32 and rounds once (40 rows x 32256: 11 us)
//   xl_adapter_down_mma, xl_adapter_up_mma   the same for 16-bit types and many rows of a sequence, on mma.sync
// Either second half takes the shared product in 32 bits and rounds the sum once. An adapters' term in 16 bits, for the shared product to
// accumulate on, would move 4 bytes less per value (4096 x 32256: 82 us of 845), but its rounding is half a step of the term, which
// nothing keeps below the sum: where the two cancel it would be all there is, and in fp16 the term may be past 65504 where the sum is not.
#include "common.cuh"

#include <type_traits>

namespace {

constexpr int AD_MAX_RANK = 128;

struct AdapterParams {
  const void *x, *a, *b;
  const float* scale;
  const int* slot;
  float* low;
  const float* y;  // shared product (rows, N), fp32
  void* out;       // (rows, N)
  long long rows;
  int T, K, N, n, r, rp;
  int tile;        // xl_adapter_up_mma: rows of a CTA
};

__device__ __forceinline__ int adapter_of(const AdapterParams& p, long long seq) {
  const int s = p.slot[seq];
  return s >= 0 && s < p.n ? s : -1;
}

// ---- one warp per number ----------------------------------------------------------------------------------------------------
template <typename T, bool VEC> __global__ void __launch_bounds__(256) adapter_down_kernel(const AdapterParams p) {
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (i >= p.rows * p.rp) return;
  const long long row = i / p.rp;
  const int j = (int)(i - row * p.rp), s = adapter_of(p, row / p.T);
  float sum = 0.f;
  if (j < p.r && s >= 0) {
    const T* x = (const T*)p.x + row * p.K;
    const T* a = (const T*)p.a + ((long long)s * p.r + j) * p.K;
    if (VEC) {
      constexpr int V = XlVec<T>::N;
#pragma unroll 8
      for (int k = lane * V; k < p.K; k += 32 * V) {
        float u[V], v[V];
        xl_load16(x + k, u);
        xl_load16(a + k, v);
#pragma unroll
        for (int e = 0; e < V; ++e) sum = fmaf(u[e], v[e], sum);
      }
    } else {
      for (int k = lane; k < p.K; k += 32) sum = fmaf(xl_to_float(x[k]), xl_to_float(a[k]), sum);
    }
    sum = xl_warp_sum(sum) * p.scale[s];
  }
  if (lane == 0) p.low[i] = sum;
}

// ---- shared product + second term, rounded once -------------------------------------------------------------------------------
// Grid (columns / 256, groups of eight rows): a thread has one column of every row of the group, and with it one row of each row's B[s],
// r numbers side by side. The group's slots and numbers are fetched once, side by side: a CTA per row and 256 columns spent its time on
// that chain of loads (40 rows x 32256: 17 us). W: bytes that a load of B takes, 0: single elements.
constexpr int AD_ROWS = 8;
template <typename T, typename O, int W> __global__ void __launch_bounds__(256) adapter_up_kernel(const AdapterParams p) {
  __shared__ __align__(16) float low[AD_ROWS][AD_MAX_RANK];
  __shared__ int slots[AD_ROWS];
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int c = blockIdx.x * 256 + threadIdx.x;
  const long long row0 = (long long)blockIdx.y * AD_ROWS;
  const int rows = (int)(p.rows - row0 < AD_ROWS ? p.rows - row0 : AD_ROWS);
  float v[AD_ROWS];
#pragma unroll
  for (int i = 0; i < AD_ROWS; ++i) v[i] = i < rows && c < p.N ? p.y[(row0 + i) * p.N + c] : 0.f;
  for (int i = threadIdx.x; i < rows * p.rp; i += 256) low[i / p.rp][i % p.rp] = p.low[row0 * p.rp + i];
  if ((int)threadIdx.x < rows) slots[threadIdx.x] = adapter_of(p, (row0 + threadIdx.x) / p.T);
  __syncthreads();
  if (c >= p.N) return;
#pragma unroll
  for (int i = 0; i < AD_ROWS; ++i) {
    if (i < rows && slots[i] >= 0) {
      const T* b = (const T*)p.b + ((long long)slots[i] * p.N + c) * p.r;
      float sum = 0.f;
      if (W > 0) {
        constexpr int E = W > 0 ? W / (int)sizeof(T) : 1;
#pragma unroll 2
        for (int j = 0; j < p.r; j += E) {
          uint32_t w[W > 0 ? W / 4 : 1];
          if (W == 16) *reinterpret_cast<uint4*>(w) = *reinterpret_cast<const uint4*>(b + j);
          else if (W == 8) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(b + j);
          else w[0] = *reinterpret_cast<const uint32_t*>(b + j);
          const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
          for (int q = 0; q < E; ++q) sum = fmaf(low[i][j + q], xl_to_float(e[q]), sum);
        }
      } else {
        for (int j = 0; j < p.r; ++j) sum = fmaf(low[i][j], xl_to_float(b[j]), sum);
      }
      v[i] += sum;
    }
  }
#pragma unroll
  for (int i = 0; i < AD_ROWS; ++i)
    if (i < rows) ((O*)p.out)[(row0 + i) * p.N + c] = xl_from_float<O>(v[i]);
}

// ---- many rows of a sequence: mma.sync ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ void ad_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void ad_mma<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void ad_mma<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t ad_pack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t ad_pack<__nv_bfloat16>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
template <> __device__ __forceinline__ uint32_t ad_pack<__half>(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Grid (row tiles of 16, sequences). Sixteen warps (eight where their sums would not fit) share a tile and take parts of K, 32 features at a
// time: a lane reads 16 bytes of its two rows of x and of each of its rows of A, which are the operands of two products (the order of
// features is free as long as both sides agree). Their sums meet in shared memory. 4 x 1024 rows x 4096, rank 16: 13 us, of which reading x
// is 5. NT: tiles of eight numbers.
template <typename T, int NT> __global__ void __launch_bounds__(NT <= 2 ? 512 : 256, 2) adapter_down_mma_kernel(const AdapterParams p) {
  constexpr int WARPS = NT <= 2 ? 16 : 8, THREADS = WARPS * 32;
  __shared__ float part[WARPS][16][NT * 8 + 1];
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, j = lane & 3;
  const long long seq = blockIdx.y;
  const int t0 = blockIdx.x * 16, s = adapter_of(p, seq);
  float* low = p.low + (seq * p.T + t0) * p.rp;
  const int rows = min(16, p.T - t0);
  if (s < 0) {
    for (int i = threadIdx.x; i < rows * p.rp; i += THREADS) low[i] = 0.f;
    return;
  }
  const T* x = (const T*)p.x + (seq * p.T + t0) * p.K;
  const T* a = (const T*)p.a + (long long)s * p.r * p.K;
  float c[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) c[n][e] = 0.f;
  const int steps = (p.K + 31) / 32;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 2
  for (int i = warp; i < steps; i += WARPS) {
    const int k = i * 32 + j * 8;
    const bool on = k < p.K;
    const uint4 lo = on && quad < rows ? *reinterpret_cast<const uint4*>(x + (long long)quad * p.K + k) : zero;
    const uint4 hi = on && quad + 8 < rows ? *reinterpret_cast<const uint4*>(x + (long long)(quad + 8) * p.K + k) : zero;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4 w = on && n * 8 + quad < p.r ? *reinterpret_cast<const uint4*>(a + (long long)(n * 8 + quad) * p.K + k) : zero;
      ad_mma<T>(c[n], lo.x, hi.x, lo.y, hi.y, w.x, w.y);
      ad_mma<T>(c[n], lo.z, hi.z, lo.w, hi.w, w.z, w.w);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][quad + 8 * (e >> 1)][n * 8 + 2 * j + (e & 1)] = c[n][e];
  __syncthreads();
  const float scale = p.scale[s];
  for (int i = threadIdx.x; i < rows * p.rp; i += THREADS) {
    const int r = i / p.rp, q = i - r * p.rp;
    float sum = 0.f;
    if (q < NT * 8) {
#pragma unroll
      for (int w = 0; w < WARPS; ++w) sum += part[w][r][q];
    }
    low[i] = sum * scale;
  }
}

// Grid (columns / 128, row tiles, sequences): the shared product + the adapters' term, rounded to T. A warp has 32 columns for all rows of
// the tile, whose row of B[s] it holds; its lanes' columns are chosen so that each ends up with eight neighbours, which arrive in two loads
// and leave in one store. `low` enters as sums of two T (value and rounding error). Moving the results bounds it: 4 x 1024 rows x 32256 take
// 132 us (793 MB, 6.0 TB/s). KS: steps of 16 numbers.
constexpr int AD_TILE = 256;  // rows of a CTA, at most
template <typename T, int KS> __global__ void __launch_bounds__(128) adapter_up_mma_kernel(const AdapterParams p) {
  xl_grid_dependency_wait();
  xl_grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, quad = lane >> 2, j = lane & 3;
  const long long seq = blockIdx.z;
  const int t0 = blockIdx.y * p.tile, s = adapter_of(p, seq), rows = min(p.tile, p.T - t0), c0 = blockIdx.x * 128 + warp * 32;
  if (c0 >= p.N) return;
  T* out = (T*)p.out + (seq * p.T + t0) * p.N;
  const float* y = p.y + (seq * p.T + t0) * p.N;
  const float* low = p.low + (seq * p.T + t0) * p.rp;
  const bool wide = p.N % 8 == 0;
  uint32_t b[4][KS][2];
  if (s >= 0) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 8 * (quad >> 1) + 2 * u + (quad & 1);
      const T* row = (const T*)p.b + ((long long)s * p.N + c) * p.r;
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int q = k * 16 + h * 8 + 2 * j;
          uint32_t w = 0u;
          if (c < p.N) {
            if (p.r % 2 == 0) {
              if (q < p.r) w = *reinterpret_cast<const uint32_t*>(row + q);
            } else {
              const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
              w = (q < p.r ? e[q] : 0u) | (q + 1 < p.r ? (uint32_t)e[q + 1] << 16 : 0u);
            }
          }
          b[u][k][h] = w;
        }
    }
  }
#pragma unroll 2
  for (int m = 0; m * 16 < rows; ++m) {
    float sum[2][8];  // rows quad, quad + 8: the shared product, asked for ahead of what is added to it
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = m * 16 + quad + 8 * h, c1 = c0 + 8 * j;
      const float* src = y + (long long)r * p.N + c1;
      if (wide && r < rows && c1 < p.N) {
        *reinterpret_cast<float4*>(&sum[h][0]) = __ldcs(reinterpret_cast<const float4*>(src));
        *reinterpret_cast<float4*>(&sum[h][4]) = __ldcs(reinterpret_cast<const float4*>(src + 4));
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) sum[h][q] = r < rows && c1 + q < p.N ? src[q] : 0.f;
      }
    }
    float c[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[u][e] = 0.f;
    float up[2] = {1.f, 1.f};  // rows quad, quad + 8
    if (s >= 0) {
      float down[2] = {1.f, 1.f};
      if constexpr (std::is_same<T, __half>::value) {  // fp16 ends at 65504, and keeps ever fewer bits below 2^-14: every row is brought
                                                       // to numbers of up to 2^15 by a power of two on the way
        float top[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < KS * 4; ++i) {
          const int r = m * 16 + quad + 8 * (i & 1);
          if (r < rows) {
            const float2 v = *reinterpret_cast<const float2*>(low + r * p.rp + 8 * (i >> 1) + 2 * j);
            top[i & 1] = fmaxf(top[i & 1], fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
          top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
          if (top[i] > 0.f && top[i] < INFINITY) {
            const int by = max(ilogbf(top[i]) - 14, -126);  // both powers are normal numbers
            down[i] = ldexpf(1.f, -by);
            up[i] = ldexpf(1.f, by);
          }
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t h[4], e[4];  // rows quad, quad + 8; numbers 2 j, 2 j + 1, then 2 j + 8, 2 j + 9
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = m * 16 + quad + 8 * (i & 1);
          float2 v = r < rows ? *reinterpret_cast<const float2*>(low + r * p.rp + k * 16 + 8 * (i >> 1) + 2 * j) : make_float2(0.f, 0.f);
          if constexpr (std::is_same<T, __half>::value) v = make_float2(v.x * down[i & 1], v.y * down[i & 1]);
          h[i] = ad_pack<T>(v.x, v.y);
          const float2 back = xl_pair_to_float2<T>(h[i]);  // infinite: there is no rest
          e[i] = ad_pack<T>(fabsf(back.x) < INFINITY ? v.x - back.x : 0.f, fabsf(back.y) < INFINITY ? v.y - back.y : 0.f);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          ad_mma<T>(c[u], h[0], h[1], h[2], h[3], b[u][k][0], b[u][k][1]);
          ad_mma<T>(c[u], e[0], e[1], e[2], e[3], b[u][k][0], b[u][k][1]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = m * 16 + quad + 8 * h, c1 = c0 + 8 * j;
      if (r >= rows) continue;
      T* dst = out + (long long)r * p.N + c1;
      uint32_t w[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if constexpr (std::is_same<T, __half>::value)
          w[u] = ad_pack<T>(fmaf(c[u][2 * h], up[h], sum[h][2 * u]), fmaf(c[u][2 * h + 1], up[h], sum[h][2 * u + 1]));
        else w[u] = ad_pack<T>(sum[h][2 * u] + c[u][2 * h], sum[h][2 * u + 1] + c[u][2 * h + 1]);
      }
      if (wide) {
        if (c1 < p.N) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          if (c1 + q < p.N) dst[q] = e[q];
      }
    }
  }
}

bool adapter_sizes_ok(long long rows, int T, int K, int N, int n, int r) {
  return rows >= 1 && T >= 1 && rows % T == 0 && K >= 1 && N >= 1 && n >= 1 && r >= 1 && r <= AD_MAX_RANK && rows <= 0x7fffffffLL;
}

}  // namespace

// x (rows, K), a (n, r, K), scale (n), slot (rows / T) -> low (rows, rp) fp32, rp = r rounded up to 16. r <= 128.
XL_API int xl_adapter_down(const void* x, const void* a, const float* scale, const int* slot, float* low, long long rows, int T, int K,
                           int n, int r, int dtype, cudaStream_t s) {
  if (!adapter_sizes_ok(rows, T, K, 1, n, r)) return -1;
  AdapterParams p = {};
  p.x = x; p.a = a; p.scale = scale; p.slot = slot; p.low = low; p.rows = rows; p.T = T; p.K = K; p.n = n; p.r = r; p.rp = (r + 15) / 16 * 16;
  const long long ctas = (rows * p.rp + 7) / 8;
  if (ctas > 0x7fffffffLL) return -1;
  XL_DISPATCH_DTYPE(dtype, D, {
    const bool vec = K % XlVec<D>::N == 0 && (((uintptr_t)x | (uintptr_t)a) & 15) == 0;
    XL_TRY(xl_launch_overlapped(vec ? adapter_down_kernel<D, true> : adapter_down_kernel<D, false>, dim3((unsigned)ctas), dim3(256), (size_t)0, s, p));
  });
  return (int)cudaGetLastError();
}

// out (rows, N) of type `out_dtype` (that of b, or fp32) = y (rows, N) fp32 + low b[slot]^T. out may be y.
XL_API int xl_adapter_up(const float* low, const void* b, const int* slot, const float* y, void* out, long long rows, int T, int N, int n,
                         int r, int dtype, int out_dtype, cudaStream_t s) {
  if (!adapter_sizes_ok(rows, T, 1, N, n, r) || (out_dtype != dtype && out_dtype != XL_F32)) return -1;
  AdapterParams p = {};
  p.b = b; p.slot = slot; p.low = const_cast<float*>(low); p.y = y; p.out = out; p.rows = rows; p.T = T; p.N = N; p.n = n; p.r = r;
  p.rp = (r + 15) / 16 * 16;
  if ((rows + AD_ROWS - 1) / AD_ROWS > 65535) return -1;
  const dim3 grid((N + 255) / 256, (unsigned)((rows + AD_ROWS - 1) / AD_ROWS));
  XL_DISPATCH_DTYPE(dtype, D, {
    const int bytes = r * (int)sizeof(D);
    const uintptr_t at = (uintptr_t)b;
    const int w = bytes % 16 == 0 && at % 16 == 0 ? 16 : (bytes % 8 == 0 && at % 8 == 0 ? 8 : (bytes % 4 == 0 && at % 4 == 0 ? 4 : 0));
    void (*kernel)(const AdapterParams);
    if (out_dtype == XL_F32)
      kernel = w == 16 ? adapter_up_kernel<D, float, 16> : (w == 8 ? adapter_up_kernel<D, float, 8> : (w == 4 ? adapter_up_kernel<D, float, 4> : adapter_up_kernel<D, float, 0>));
    else
      kernel = w == 16 ? adapter_up_kernel<D, D, 16> : (w == 8 ? adapter_up_kernel<D, D, 8> : (w == 4 ? adapter_up_kernel<D, D, 4> : adapter_up_kernel<D, D, 0>));
    XL_TRY(xl_launch_overlapped(kernel, grid, dim3(256), (size_t)0, s, p));
  });
  return (int)cudaGetLastError();
}

// The first half for 16-bit types; K a multiple of 8, x and a 16-byte aligned.
XL_API int xl_adapter_down_mma(const void* x, const void* a, const float* scale, const int* slot, float* low, long long rows, int T, int K,
                               int n, int r, int dtype, cudaStream_t s) {
  if (!adapter_sizes_ok(rows, T, K, 1, n, r) || dtype == XL_F32 || K % 8 || (((uintptr_t)x | (uintptr_t)a) & 15) || rows / T > 65535) return -1;
  AdapterParams p = {};
  p.x = x; p.a = a; p.scale = scale; p.slot = slot; p.low = low; p.rows = rows; p.T = T; p.K = K; p.n = n; p.r = r; p.rp = (r + 15) / 16 * 16;
  const dim3 grid((T + 15) / 16, (unsigned)(rows / T));
  void (*kernel)(const AdapterParams);
#define XL_AD(D) \
  kernel = r <= 8 ? adapter_down_mma_kernel<D, 1> : (r <= 16 ? adapter_down_mma_kernel<D, 2> : (r <= 32 ? adapter_down_mma_kernel<D, 4> : (r <= 64 ? adapter_down_mma_kernel<D, 8> : nullptr)))
  if (dtype == XL_BF16) XL_AD(__nv_bfloat16);
  else XL_AD(__half);
#undef XL_AD
  if (!kernel) return -1;
  XL_TRY(xl_launch_overlapped(kernel, grid, dim3(r <= 16 ? 512 : 256), (size_t)0, s, p));
  return (int)cudaGetLastError();
}

// out (rows, N) of b's type = y (rows, N) fp32 + low b[slot]^T. 16-bit types, r <= 64; y and out 16-byte aligned, b to 4 bytes.
XL_API int xl_adapter_up_mma(const float* low, const void* b, const int* slot, const float* y, void* out, long long rows, int T, int N, int n, int r,
                             int dtype, cudaStream_t s) {
  if (!adapter_sizes_ok(rows, T, 1, N, n, r) || dtype == XL_F32 || (((uintptr_t)y | (uintptr_t)out) & 15) || (((uintptr_t)b) & 3) || rows / T > 65535 ||
      (T + 31) / 32 > 65535)
    return -1;
  AdapterParams p = {};
  p.b = b; p.slot = slot; p.low = const_cast<float*>(low); p.y = y; p.out = out; p.rows = rows; p.T = T; p.N = N; p.n = n; p.r = r;
  p.rp = (r + 15) / 16 * 16;
  // Fewer rows per CTA while there are fewer than four CTAs per SM, which then wait for their loads one after another (the whole op, in tiles of
  // 256 and by this rule: 1000 rows, 4096 x 4096, rank 64 100 and 78 us, 2048 x 2048, rank 8 33 and 23). More rows otherwise: B[s] is
  // read once per tile.
  p.tile = AD_TILE;
  while (p.tile > 32 && (long long)((N + 127) / 128) * ((T + p.tile - 1) / p.tile) * (rows / T) < 4 * 148) p.tile /= 2;
  const dim3 grid((N + 127) / 128, (T + p.tile - 1) / p.tile, (unsigned)(rows / T));
  void (*kernel)(const AdapterParams);
#define XL_AD(D) \
  kernel = p.rp == 16 ? adapter_up_mma_kernel<D, 1> : (p.rp == 32 ? adapter_up_mma_kernel<D, 2> : (p.rp == 48 ? adapter_up_mma_kernel<D, 3> : (p.rp == 64 ? adapter_up_mma_kernel<D, 4> : nullptr)))
  if (dtype == XL_BF16) XL_AD(__nv_bfloat16);
  else XL_AD(__half);
#undef XL_AD
  if (!kernel) return -1;
  XL_TRY(xl_launch_overlapped(kernel, grid, dim3(128), (size_t)0, s, p));
  return (int)cudaGetLastError();
}
