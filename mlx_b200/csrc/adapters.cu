// Low-rank adapters beside a shared projection: out[t] = y[t] + c_l B_l (A_l x[t]) with l the adapter of row t, and the gradients.
//
//   forward   h = A x           down (weights [r, K])              out = y + c B h    up (weights [N, r])
//   backward  g = c B^T dy      down (weights [N, r], "tall")      dx = A^T g         up (weights [r, K], "wide")
//             dA = sum g x^T    outer                              dB = c sum dy h^T  outer, transposed
//
// Rows come sorted by adapter (b200q_group_rows), in tiles of up to 64 rows of one adapter.  A rank of 8 to 64 makes r operations per
// byte of activations, far below what the tensor cores do per byte of HBM, so the kernels are built for the memory: activations are read
// once, straight from HBM into the fragments of mma.sync (no shared memory, no transposed copies), 16 bytes per lane.  That works because
// the k index of a product may be permuted as long as both operands agree, and the columns of its result as long as the stores do:
// a lane's 8 consecutive values are its fragments of four (or two) steps.  Operands that lie the other way round are transposed 8 x 8 in
// registers (movmatrix).
//
// h and g are kept in fp32.  As operands of the second product they are split into two bf16 numbers, high and low part (2^-17 of the
// value is lost), and multiplied as such; 16-bit floats of type f16 are split too, exactly, so that no value leaves a type's range.
#include <cooperative_groups.h>

#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace b200q {
namespace {
namespace cg = cooperative_groups;

constexpr int kRows = kAdapterRows, kWarps = 8, kThreads = 32 * kWarps;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (sizeof(T) == 2 && std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// An 8 x 8 matrix of 16-bit values, lane (i, q) having (i, 2q) and (i, 2q + 1): afterwards (2q, i) and (2q + 1, i).
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {   // two bf16, the first in the lower half
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The high part's rounding is away from infinity where the nearest bf16 would be one; what is not finite has no low part.
__device__ __forceinline__ void split(float a, float b, uint32_t* hi, uint32_t* lo) {
  __nv_bfloat16 ha = __float2bfloat16_rn(a), hb = __float2bfloat16_rn(b);
  if (isinf(__bfloat162float(ha))) ha = __float2bfloat16_rz(a);
  if (isinf(__bfloat162float(hb))) hb = __float2bfloat16_rz(b);
  const float fa = __bfloat162float(ha), fb = __bfloat162float(hb);
  *hi = pack(fa, fb);
  *lo = pack(isinf(fa) ? 0.0f : a - fa, isinf(fb) ? 0.0f : b - fb);
}
// A pair of T as bf16 numbers: itself, or (f16) high and low part.
template <typename T>
__device__ __forceinline__ void as_bf16(uint32_t v, uint32_t* hi, uint32_t* lo) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
    split(f.x, f.y, hi, lo);
  } else {
    *hi = v;
    *lo = 0;
  }
}

// 8 consecutive values from p on, of which `have` are there (others: 0); whole: 16 bytes aligned, all or none there.
// (fixed: no kernel running now writes them)
template <bool WHOLE, bool FIXED = true, typename T>
__device__ __forceinline__ uint4 load8(const T* p, int64_t have) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if constexpr (WHOLE) {
    if (have > 0) v = FIXED ? __ldg(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
    uint32_t* w = &v.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < have) w[i / 2] |= (uint32_t)(FIXED ? __ldg(q + i) : q[i]) << (16 * (i & 1));
  }
  return v;
}
// N consecutive values (4 or 8) in the widest pieces that the rows' alignment allows (`width` bytes).
template <int N, typename T>
__device__ __forceinline__ void load_few(const T* p, int64_t have, int width, uint32_t (&w)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) w[i] = 0;
  if (N == 8 && width == 16) {
    if (have > 0) {
      const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
      w[0] = v.x; w[1] = v.y; w[N / 2 - 2] = v.z; w[N / 2 - 1] = v.w;
    }
  } else if (width >= 8) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i)
      if (4 * i < have) {
        const uint2 v = __ldg(reinterpret_cast<const uint2*>(p) + i);
        w[2 * i] = v.x; w[2 * i + 1] = v.y;
      }
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      if (2 * i < have) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < have) w[i / 2] |= (uint32_t)__ldg(q + i) << (16 * (i & 1));
  }
}

struct Params {
  const void *x, *w;       // activations; weights of all adapters
  const float* h;          // up, outer: [T, r]
  const void* y;           // up: what is added to (null: zeros)
  void* out;               // down: float [T, r]
  const float* scales;     // null: 1
  const int *order, *sizes, *starts;
  const int4* tiles;
  int64_t T, C;            // rows; the long dimension (K or N)
  int64_t tiles_n;
  int L, r, width;         // width: bytes that a row of weights' pieces are aligned to
  int split;               // blocks per cluster
};

// A tile, or none (rows == 0) where the table does not fit the operands.
__device__ __forceinline__ int4 tile_of(const Params& p, int64_t k) {
  int4 t = p.tiles[k];
  if (t.z <= 0 || t.z > kRows || t.y < 0 || (int64_t)t.y + t.z > p.T || t.x >= p.L) t.z = 0;
  return t;
}
// The row at a place of the order; -1 where there is none.
__device__ __forceinline__ int64_t row_at(const Params& p, int64_t place) {
  int64_t row = p.order[place];
  if (row < 0) row = -1 - row;
  return row < p.T ? row : -1;
}

// ---- h[place] = (c) sum over the long dimension of x[row] w.  Blocks by (tile, part of the long dimension, 8 NT ranks); the parts are a cluster.
// TALL: weights [C, r], else [r, C].
template <typename T, bool TALL, bool WHOLE, int NT>
__global__ void __launch_bounds__(kThreads) down_kernel(const Params p) {
  constexpr int kRanks = 8 * NT;
  extern __shared__ __align__(16) float red[];   // [kWarps][kRows][kRanks]
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int part = (int)(blockIdx.x % p.split);
  const int4 tile = tile_of(p, blockIdx.x / p.split);
  if (tile.z == 0 || tile.x < 0) return;   // the whole cluster
  const int subs = (tile.z + 15) / 16, r0 = blockIdx.y * kRanks;
  const int64_t C = p.C;
  const T* x[4][2];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m * 16 + i * 8 + g;
      const int64_t at = row < tile.z ? row_at(p, tile.y + row) : -1;
      x[m][i] = at < 0 ? nullptr : static_cast<const T*>(p.x) + at * C;
    }
  const T* w = static_cast<const T*>(p.w) + (int64_t)tile.x * p.r * C;
  float acc[4][NT][4] = {};
  struct Stage {
    uint4 x[4][2];
    uint32_t w[TALL ? 4 : NT][TALL ? NT : 4];
  };
  auto load = [&](int64_t k0, Stage& s) {
    const int64_t k = k0 + q * 8;
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (m < subs) {
#pragma unroll
        for (int i = 0; i < 2; ++i) s.x[m][i] = x[m][i] ? load8<WHOLE>(x[m][i] + k, C - k) : make_uint4(0, 0, 0, 0);
      }
    if constexpr (TALL) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {   // rows of pair j of every lane's 8
        const int64_t kr = k0 + (g >> 1) * 8 + j * 2 + (g & 1);
        const int rank = r0 + q * 2 * NT;
        load_few<2 * NT>(w + kr * p.r + rank, kr < C ? p.r - rank : 0, p.width, s.w[j]);
      }
    } else {
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int rank = r0 + (g >> 1) * 2 * NT + t * 2 + (g & 1);
        const uint4 v = rank < p.r ? load8<WHOLE>(w + (int64_t)rank * C + k, C - k) : make_uint4(0, 0, 0, 0);
        s.w[t][0] = v.x; s.w[t][1] = v.y; s.w[t][2] = v.z; s.w[t][3] = v.w;
      }
    }
  };
  auto multiply = [&](Stage& s) {
    uint32_t b[NT][4];   // pair j of the lane's 8, of column tile t
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (TALL) b[t][j] = transposed(s.w[j][t]);
        else b[t][j] = s.w[t][j];
      }
#pragma unroll
    for (int m = 0; m < 4; ++m)
      if (m < subs) {
        const uint4 u = s.x[m][0], v = s.x[m][1];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          mma<T>(acc[m][t], u.x, v.x, u.y, v.y, b[t][0], b[t][1]);
          mma<T>(acc[m][t], u.z, v.z, u.w, v.w, b[t][2], b[t][3]);
        }
      }
  };
  const int64_t step = (int64_t)p.split * kWarps * 32;
  int64_t k = ((int64_t)part * kWarps + warp) * 32;
  Stage a, b;
  if (k < C) load(k, a);
  while (k < C) {
    if (k + step < C) load(k + step, b);
    multiply(a);
    k += step;
    if (k >= C) break;
    if (k + step < C) load(k + step, a);
    multiply(b);
    k += step;
  }
#pragma unroll
  for (int m = 0; m < 4; ++m)
    if (m < subs) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(&red[(warp * kRows + m * 16 + i * 8 + g) * kRanks + q * 2 * NT + t * 2]) = make_float2(acc[m][t][2 * i], acc[m][t][2 * i + 1]);
    }
  __syncthreads();
  const int n = tile.z * kRanks;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    float s = red[i];
#pragma unroll
    for (int v = 1; v < kWarps; ++v) s += red[v * kRows * kRanks + i];
    red[i] = s;
  }
  cluster.sync();
  const float c = p.scales ? p.scales[tile.x] : 1.0f;
  float* h = static_cast<float*>(p.out);
  for (int i = threadIdx.x * p.split + part; i < n; i += kThreads * p.split) {
    float s = 0.0f;
    for (int v = 0; v < p.split; ++v) s += cluster.map_shared_rank(red, v)[i];
    const int rank = r0 + i % kRanks;
    if (rank < p.r) h[(int64_t)(tile.y + i / kRanks) * p.r + rank] = c * s;
  }
  cluster.sync();   // no block leaves while others read its sums
}

// ---- out[row] = y[row] + (c) sum over ranks of h[place] w.  Blocks by (tile, 256 columns), warps by 32 columns; ranks in chunks of 64.
// WIDE: weights [r, C], else [C, r].
constexpr int kChunk = 64, kPitch = kChunk + 16;
template <typename T, bool WIDE, bool WHOLE>
__global__ void __launch_bounds__(kThreads) up_kernel(const Params p) {
  constexpr bool kSplitW = std::is_same_v<T, __half>;
  __shared__ __align__(16) uint16_t hi[kRows * kPitch], lo[kRows * kPitch];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int64_t C = p.C, blocks = (C + 255) / 256;
  const int4 tile = tile_of(p, blockIdx.x / blocks);
  if (tile.z == 0) return;
  const int64_t n0 = (blockIdx.x % blocks) * 256 + warp * 32, n = n0 + q * 8;   // the lane's columns are n .. n + 7
  const int64_t have = C - n;
  const int subs = (tile.z + 15) / 16;
  const T* y = static_cast<const T*>(p.y);
  T* out = static_cast<T*>(p.out);
  const bool plain = tile.x < 0;   // rows without an adapter
  if (plain && p.y == p.out) return;
  float acc[4][4][4] = {};
  if (!plain) {
    const T* w = static_cast<const T*>(p.w) + (int64_t)tile.x * p.r * C;
    const float c = p.scales ? p.scales[tile.x] : 1.0f;
    for (int r0 = 0; r0 < p.r; r0 += kChunk) {
      const int ranks = min(kChunk, p.r - r0), steps = (ranks + 15) / 16;
      if (r0) __syncthreads();
      for (int i = threadIdx.x; i < kRows * (kChunk / 2); i += kThreads) {
        const int row = i / (kChunk / 2), k = i % (kChunk / 2) * 2;
        float a = 0.0f, b = 0.0f;
        if (row < tile.z) {
          const float* h = p.h + (int64_t)(tile.y + row) * p.r + r0 + k;
          if (k < ranks) a = c * h[0];
          if (k + 1 < ranks) b = c * h[1];
        }
        split(a, b, reinterpret_cast<uint32_t*>(&hi[row * kPitch + k]), reinterpret_cast<uint32_t*>(&lo[row * kPitch + k]));
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < kChunk / 16; ++s) {
        if (s >= steps) break;
        uint32_t b[4][2];   // column tile, pair of the lane's 4 ranks
        if constexpr (WIDE) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int rank = r0 + s * 16 + (g >> 1) * 4 + j * 2 + (g & 1);
            const uint4 v = rank < p.r ? load8<WHOLE>(w + (int64_t)rank * C + n, have) : make_uint4(0, 0, 0, 0);
            b[0][j] = transposed(v.x); b[1][j] = transposed(v.y); b[2][j] = transposed(v.z); b[3][j] = transposed(v.w);
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int64_t col = n0 + (g >> 1) * 8 + t * 2 + (g & 1);
            const int rank = r0 + s * 16 + q * 4;
            load_few<4>(w + col * p.r + rank, col < C ? p.r - rank : 0, p.width, b[t]);
          }
        }
        uint32_t bh[4][2], bl[4][2];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) as_bf16<T>(b[t][j], &bh[t][j], &bl[t][j]);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (m >= subs) break;
          const int at = (m * 16 + g) * kPitch + s * 16 + q * 4;
          const uint2 h0 = *reinterpret_cast<const uint2*>(&hi[at]), h1 = *reinterpret_cast<const uint2*>(&hi[at + 8 * kPitch]);
          const uint2 l0 = *reinterpret_cast<const uint2*>(&lo[at]), l1 = *reinterpret_cast<const uint2*>(&lo[at + 8 * kPitch]);
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            mma<__nv_bfloat16>(acc[m][t], h0.x, h1.x, h0.y, h1.y, bh[t][0], bh[t][1]);
            mma<__nv_bfloat16>(acc[m][t], l0.x, l1.x, l0.y, l1.y, bh[t][0], bh[t][1]);
            if constexpr (kSplitW) mma<__nv_bfloat16>(acc[m][t], h0.x, h1.x, h0.y, h1.y, bl[t][0], bl[t][1]);
          }
        }
      }
    }
  }
  if (have <= 0) return;
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m * 16 + i * 8 + g;
      const int64_t at = row < tile.z ? row_at(p, tile.y + row) : -1;
      if (at < 0) continue;
      const uint4 v = y ? load8<WHOLE, false>(y + at * C + n, have) : make_uint4(0, 0, 0, 0);
      T o[8];
      *reinterpret_cast<uint4*>(o) = v;
      if (!plain) {
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] = Elem<T>::from_float(Elem<T>::to_float(o[k]) + acc[m][k / 2][2 * i + (k & 1)]);
      }
      if constexpr (WHOLE) {
        *reinterpret_cast<uint4*>(out + at * C + n) = *reinterpret_cast<const uint4*>(o);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < have) out[at * C + n + k] = o[k];
      }
    }
}

// ---- out_l = (c) sum over l's rows of h[place] x[row]^T.  Blocks by (64 columns, part of the rows; adapter; 16 MT ranks), the parts are a
// cluster; warps by (32 columns, quarter of the rows).  TALL: out [C, r], else [r, C].
template <typename T, bool TALL, bool WHOLE, int MT>
__global__ void __launch_bounds__(kThreads) outer_kernel(const Params p) {
  constexpr int kRanks = 16 * MT, kCols = 64, kLine = kCols + 4;
  extern __shared__ __align__(16) float red[];   // [4][kRanks][kLine]
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3, slot = warp >> 1;
  const int part = (int)(blockIdx.x % p.split), l = blockIdx.y, r0 = blockIdx.z * kRanks;
  const int64_t C = p.C, c0 = (int64_t)(blockIdx.x / p.split) * kCols, col = c0 + (warp & 1) * 32 + q * 8;
  const int64_t lo = max(p.starts[l], 0), hi = min((int64_t)p.starts[l + 1], p.T);
  const T* x = static_cast<const T*>(p.x);
  float acc[MT][4][4] = {};
  struct Stage {
    uint4 x[2];
    float h[MT][8];
  };
  auto load = [&](int64_t t0, Stage& s) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t at = t0 + i * 8 + g, row = at < hi ? row_at(p, at) : -1;
      s.x[i] = row >= 0 ? load8<WHOLE>(x + row * C + col, C - col) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int i = 0; i < 8; ++i) {   // places 2q, 2q + 1, the same + 8; ranks g, g + 8
        const int64_t at = t0 + q * 2 + (i & 1) + (i & 2 ? 8 : 0);
        const int rank = r0 + m * 16 + g + (i & 4 ? 8 : 0);
        s.h[m][i] = at < hi && rank < p.r ? p.h[at * p.r + rank] : 0.0f;
      }
  };
  auto multiply = [&](const Stage& s) {
    uint32_t bh[4][2], bl[4][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      as_bf16<T>(transposed(s.x[i].x), &bh[0][i], &bl[0][i]);
      as_bf16<T>(transposed(s.x[i].y), &bh[1][i], &bl[1][i]);
      as_bf16<T>(transposed(s.x[i].z), &bh[2][i], &bl[2][i]);
      as_bf16<T>(transposed(s.x[i].w), &bh[3][i], &bl[3][i]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      uint32_t ah[4], al[4];
      split(s.h[m][0], s.h[m][1], &ah[0], &al[0]);
      split(s.h[m][4], s.h[m][5], &ah[1], &al[1]);
      split(s.h[m][2], s.h[m][3], &ah[2], &al[2]);
      split(s.h[m][6], s.h[m][7], &ah[3], &al[3]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        mma<__nv_bfloat16>(acc[m][t], ah[0], ah[1], ah[2], ah[3], bh[t][0], bh[t][1]);
        mma<__nv_bfloat16>(acc[m][t], al[0], al[1], al[2], al[3], bh[t][0], bh[t][1]);
        if constexpr (std::is_same_v<T, __half>) mma<__nv_bfloat16>(acc[m][t], ah[0], ah[1], ah[2], ah[3], bl[t][0], bl[t][1]);
      }
    }
  };
  const int64_t step = (int64_t)p.split * 64;
  int64_t t = lo + ((int64_t)part * 4 + slot) * 16;
  Stage a, b;
  if (t < hi) load(t, a);
  while (t < hi) {
    if (t + step < hi) load(t + step, b);
    multiply(a);
    t += step;
    if (t >= hi) break;
    if (t + step < hi) load(t + step, a);
    multiply(b);
    t += step;
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(&red[(slot * kRanks + m * 16 + i * 8 + g) * kLine + (warp & 1) * 32 + q * 8 + t * 2]) = make_float2(acc[m][t][2 * i], acc[m][t][2 * i + 1]);
  __syncthreads();
  for (int i = threadIdx.x; i < kRanks * kCols; i += kThreads) {
    const int at = i / kCols * kLine + i % kCols;
    float s = red[at];
#pragma unroll
    for (int v = 1; v < 4; ++v) s += red[v * kRanks * kLine + at];
    red[at] = s;
  }
  cluster.sync();
  const float c = p.scales ? p.scales[l] : 1.0f;
  T* out = static_cast<T*>(p.out) + (int64_t)l * p.r * C;
  const int each = kRanks * kCols / p.split;   // of the tile's elements: this block's
  for (int i = threadIdx.x; i < each; i += kThreads) {
    const int e = part * each + i, rank = TALL ? e % kRanks : e / kCols, cc = TALL ? e / kRanks : e % kCols;
    float s = 0.0f;
    for (int v = 0; v < p.split; ++v) s += cluster.map_shared_rank(red, v)[rank * kLine + cc];
    if (r0 + rank < p.r && c0 + cc < C) out[TALL ? (c0 + cc) * p.r + r0 + rank : (int64_t)(r0 + rank) * C + c0 + cc] = Elem<T>::from_float(c * s);
  }
  cluster.sync();
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Bytes (2 to 16) that rows of `pitch` bytes from p on are aligned to.
int width_of(const void* p, int64_t pitch) {
  int w = 16;
  while (w > 2 && (!aligned(p, w) || pitch % w != 0)) w /= 2;
  return w;
}
// Blocks per cluster: enough for two blocks per SM, a power of two up to 8, with work for everyone.
int split_of(int64_t blocks, int64_t most) {
  int s = 1;
  while (s < 8 && blocks * s < 2 * 148 && 2 * s <= most) s *= 2;
  return s;
}

template <typename K>
int launch(K kern, const Params& p, dim3 grid, size_t smem, bool cluster, cudaStream_t st) {
  if (smem > 48 * 1024) B200Q_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  if (cluster) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
  B200Q_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p));
  B200Q_LAUNCH_OK("adapter kernel");
  return B200Q_OK;
}

template <typename T, bool TALL, bool WHOLE>
int down(Params p, cudaStream_t st) {
  const int nt = p.r <= 16 ? 2 : 4, chunks = (p.r + 8 * nt - 1) / (8 * nt);
  p.split = split_of(p.tiles_n * chunks, p.C / (kWarps * 32));
  const dim3 grid((unsigned)(p.tiles_n * p.split), chunks);
  const size_t smem = (size_t)kWarps * kRows * 8 * nt * 4;
  return nt == 2 ? launch(down_kernel<T, TALL, WHOLE, 2>, p, grid, smem, true, st) : launch(down_kernel<T, TALL, WHOLE, 4>, p, grid, smem, true, st);
}
template <typename T, bool TALL, bool WHOLE>
int outer(Params p, cudaStream_t st) {
  const int mt = p.r <= 16 ? 1 : (p.r <= 32 ? 2 : 4), chunks = (p.r + 16 * mt - 1) / (16 * mt);
  const int64_t cols = (p.C + 63) / 64;
  p.split = split_of(cols * p.L * chunks, p.T / 64);
  const dim3 grid((unsigned)(cols * p.split), p.L, chunks);
  const size_t smem = (size_t)4 * 16 * mt * 68 * 4;
  if (mt == 1) return launch(outer_kernel<T, TALL, WHOLE, 1>, p, grid, smem, true, st);
  if (mt == 2) return launch(outer_kernel<T, TALL, WHOLE, 2>, p, grid, smem, true, st);
  return launch(outer_kernel<T, TALL, WHOLE, 4>, p, grid, smem, true, st);
}

// Of a call: which form of a kernel.
enum class Step { Down, DownTall, Up, UpWide, Outer, OuterTall };
template <typename T, bool WHOLE>
int run(Step step, const Params& p, cudaStream_t st) {
  const dim3 grid((unsigned)(p.tiles_n * ((p.C + 255) / 256)));
  switch (step) {
    case Step::Down: return down<T, false, WHOLE>(p, st);
    case Step::DownTall: return down<T, true, WHOLE>(p, st);
    case Step::Up: return launch(up_kernel<T, false, WHOLE>, p, grid, 0, false, st);
    case Step::UpWide: return launch(up_kernel<T, true, WHOLE>, p, grid, 0, false, st);
    case Step::Outer: return outer<T, false, WHOLE>(p, st);
    default: return outer<T, true, WHOLE>(p, st);
  }
}
int run(Step step, Params p, int dtype, cudaStream_t st) {
  const bool lies = step == Step::Down || step == Step::UpWide;   // weights' rows are along the long dimension
  bool whole = p.C % 8 == 0;
  for (const void* q : {p.x, p.y, lies ? p.w : nullptr, step == Step::Up || step == Step::UpWide ? static_cast<const void*>(p.out) : nullptr}) whole = whole && aligned(q, 16);
  p.width = p.w && !lies ? width_of(p.w, 2 * p.r) : 2;
  if (dtype == B200Q_F16) return whole ? run<__half, true>(step, p, st) : run<__half, false>(step, p, st);
  return whole ? run<__nv_bfloat16, true>(step, p, st) : run<__nv_bfloat16, false>(step, p, st);
}

int check(const char* tag, int dtype, int64_t T, int64_t L, int64_t N, int64_t K, int64_t r) {
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", tag, dtype);
  if (T < 0 || L < 0 || N < 0 || K < 0 || r < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] negative dimension.", tag);
  if (T > INT32_MAX - 64 || L > 4096 || N > (1 << 24) || K > (1 << 24) || r > 4096)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^31 - 65 rows, 4096 adapters, widths of 2^24 or ranks of 4096.", tag);
  const int64_t tiles = b200q_group_rows_tiles(T, L), most = INT32_MAX;
  if (tiles * 8 > most || tiles > most / ((N + 255) / 256 + 1) || tiles > most / ((K + 255) / 256 + 1))
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^31 - 1 blocks.", tag);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_add_adapters(const void* y, const void* x, const void* a, const void* b, int dtype, int64_t T, int64_t L, int64_t N, int64_t K,
                                  int64_t r, const int32_t* order, const int32_t* tiles, const float* scales, float* h, void* out, void* stream) {
  const char* tag = "add_adapters";
  if (int rc = check(tag, dtype, T, L, N, K, r)) return rc;
  if (T == 0 || N == 0) return B200Q_OK;
  if (!y || !out) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (L == 0 || K == 0 || r == 0) {   // nothing to add
    if (out != y) B200Q_CUDA_OK(cudaMemcpyAsync(out, y, (size_t)T * N * 2, cudaMemcpyDeviceToDevice, st));
    return B200Q_OK;
  }
  if (!x || !a || !b || !order || !tiles || !h) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  for (const void* q : {y, x, a, b, static_cast<const void*>(out)})
    if (!aligned(q, 2)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  if (!aligned(tiles, 16)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] tiles must be 16-byte aligned", tag);
  Params p{};
  p.x = x; p.w = a; p.out = h;
  p.order = order; p.tiles = reinterpret_cast<const int4*>(tiles); p.tiles_n = b200q_group_rows_tiles(T, L);
  p.T = T; p.C = K; p.L = (int)L; p.r = (int)r;
  const ScratchLock lock(h);
  if (int rc = run(Step::Down, p, dtype, st)) return rc;
  p.x = nullptr; p.w = b; p.h = h; p.y = y; p.out = out; p.scales = scales; p.C = N;
  return run(Step::Up, p, dtype, st);
}

extern "C" int b200q_add_adapters_grad(const void* dy, const void* x, const void* a, const void* b, int dtype, int64_t T, int64_t L, int64_t N, int64_t K,
                                       int64_t r, const int32_t* order, const int32_t* starts, const int32_t* tiles, const float* scales, const float* h,
                                       float* g, void* dx, void* da, void* db, void* stream) {
  const char* tag = "add_adapters";
  if (int rc = check(tag, dtype, T, L, N, K, r)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0 || L == 0 || N == 0 || K == 0 || r == 0) {
    if (dx && T * K > 0) B200Q_CUDA_OK(cudaMemsetAsync(dx, 0, (size_t)T * K * 2, st));
    if (da && L * r * K > 0) B200Q_CUDA_OK(cudaMemsetAsync(da, 0, (size_t)L * r * K * 2, st));
    if (db && L * N * r > 0) B200Q_CUDA_OK(cudaMemsetAsync(db, 0, (size_t)L * N * r * 2, st));
    return B200Q_OK;
  }
  if (!dy || !order || !starts || !tiles || (dx && !a) || ((dx || da) && (!b || !g)) || (da && !x) || (db && !h))
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  for (const void* q : {dy, x, a, b, static_cast<const void*>(dx), static_cast<const void*>(da), static_cast<const void*>(db)})
    if (!aligned(q, 2)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  if (!aligned(tiles, 16)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] tiles must be 16-byte aligned", tag);
  Params p{};
  p.order = order; p.starts = starts; p.tiles = reinterpret_cast<const int4*>(tiles); p.tiles_n = b200q_group_rows_tiles(T, L);
  p.T = T; p.L = (int)L; p.r = (int)r;
  const ScratchLock lock(g);
  if (dx || da) {
    Params d = p;
    d.x = dy; d.w = b; d.out = g; d.scales = scales; d.C = N;
    if (int rc = run(Step::DownTall, d, dtype, st)) return rc;
  }
  if (dx) {
    Params d = p;
    d.w = a; d.h = g; d.out = dx; d.C = K;
    if (int rc = run(Step::UpWide, d, dtype, st)) return rc;
  }
  if (da) {
    Params d = p;
    d.x = x; d.h = g; d.out = da; d.C = K;
    if (int rc = run(Step::Outer, d, dtype, st)) return rc;
  }
  if (db) {
    Params d = p;
    d.x = dy; d.h = h; d.out = db; d.scales = scales; d.C = N;
    if (int rc = run(Step::OuterTall, d, dtype, st)) return rc;
  }
  return B200Q_OK;
}
