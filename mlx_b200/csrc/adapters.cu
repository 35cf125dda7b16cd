// Low-rank adapters beside a shared projection: out[t] = y[t] + c_l B_l (A_l x[t]) with l the adapter of row t, and the gradients.
//
//   forward   h = A x           down (weights [r, K])              out = y + c B h    up (weights [N, r])
//   backward  g = c B^T dy      down (weights [N, r], "tall")      dx = A^T g         up (weights [r, K], "wide")
//             dA = sum g x^T    outer                              dB = c sum dy h^T  outer, transposed
//
// Rows come sorted by adapter (b200q_group_rows), in tiles of up to 64 rows of one adapter.  A rank of 8 to 64 makes r operations per byte of
// activations, far below what the tensor cores do per byte of HBM, so the kernels are built for the memory: activations are read once per product and
// nothing is written but h and the results.  The products are mma.sync (545 TFLOP/s measured here): tiles of a few rows whose number only the
// device knows, operands that come in pieces from gathered rows and are split into parts on the way; at rank 64 they take somewhat longer than HBM does.
//
// h and g, summed in fp32, are kept as three bf16 numbers each that add up to them exactly, since that is how the second products take them: fp32's 24 bits are 8
// and two times 8 more with signs.  16-bit floats of type f16 are split too, in two, exactly, so that no value leaves a type's range; of those six products
// the smallest, below 2^-24 of the whole, is left out.
#include <cooperative_groups.h>

#include <algorithm>
#include <cmath>
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
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The matrix instructions truncate their sums: long ones are made of short ones, which are added here with the nearest rounding.
__device__ __forceinline__ void add4(float (&d)[4], const float (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) d[i] += s[i];
}
// An 8 x 8 matrix of 16-bit values, lane (i, q) having (i, 2q) and (i, 2q + 1): afterwards (2q, i) and (2q + 1, i).
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {   // two bf16, the first in the lower half
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// The nearest bf16; toward zero where that would be infinite.
__device__ __forceinline__ float near_bf16(float a) {
  const float f = __bfloat162float(__float2bfloat16_rn(a));
  return isinf(f) ? __bfloat162float(__float2bfloat16_rz(a)) : f;
}
// Two numbers as three bf16 each, exactly.  An infinity is the last one's, and the others have its sign: whatever finite numbers these are multiplied with, of two parts
// of which the second may be zero, the sum is the infinity that it has to be.
__device__ __forceinline__ void split(float a, float b, uint32_t (&part)[3]) {
  const bool ia = isinf(a), ib = isinf(b);
  const float ha = near_bf16(a), hb = near_bf16(b), ra = a - ha, rb = b - hb;
  const float ma = ia ? copysignf(1.0f, a) : near_bf16(ra), mb = ib ? copysignf(1.0f, b) : near_bf16(rb);
  part[0] = pack(ia ? ma : ha, ib ? mb : hb);
  part[1] = pack(ma, mb);
  part[2] = pack(ia ? a : ra - ma, ib ? b : rb - mb);
}
// A pair of T as bf16 numbers: itself, or (f16) high and low part: the upper 8 bits of the 11, and the rest, exactly (0 of what is not finite).
template <typename T>
__device__ __forceinline__ void as_bf16(uint32_t v, uint32_t* hi, uint32_t* lo) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = *reinterpret_cast<const __half2*>(&v);
    const float2 f = __half22float2(h);
    const uint32_t a = __float_as_uint(f.x), b = __float_as_uint(f.y);
    *hi = __byte_perm(a, b, 0x7632);
    const float la = f.x - __uint_as_float(a & 0xffff0000u), lb = f.y - __uint_as_float(b & 0xffff0000u);
    *lo = __byte_perm(__float_as_uint(la), __float_as_uint(lb), 0x7632) & __hlt2_mask(__habs2(h), __half2half2(__ushort_as_half(0x7c00)));
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
// 4 consecutive values in the widest pieces that the rows' alignment allows (`width` bytes).
template <typename T>
__device__ __forceinline__ void load4(const T* p, int64_t have, int width, uint32_t (&w)[2]) {
  w[0] = w[1] = 0;
  if (width >= 8) {
    if (have > 0) {
      const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
      w[0] = v.x; w[1] = v.y;
    }
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (2 * i < have) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p) + i);
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < have) w[i / 2] |= (uint32_t)__ldg(q + i) << (16 * (i & 1));
  }
}

__device__ __forceinline__ uint32_t shared(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// BYTES (4, 8, 16) to shared memory, asynchronously; zeros where there is nothing (p is not read then).
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* p, bool there) {
  if constexpr (BYTES == 16)
    asm volatile("{\n.reg .pred none;\nsetp.eq.s32 none, %2, 0;\ncp.async.cg.shared.global [%0], [%1], 16, none;\n}" ::"r"(dst), "l"(p), "r"((int)there) : "memory");
  else
    asm volatile("{\n.reg .pred none;\nsetp.eq.s32 none, %3, 0;\ncp.async.ca.shared.global [%0], [%1], %2, none;\n}" ::"r"(dst), "l"(p), "n"(BYTES), "r"((int)there) : "memory");
}
__device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_all_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// 8 consecutive values in the widest pieces that the rows' alignment allows, to shared memory.
template <typename T>
__device__ __forceinline__ void copy8(uint32_t dst, const T* p, int have, int width) {
  const char* q = reinterpret_cast<const char*>(p);
  if (width == 16) {
    copy_async<16>(dst, q, have > 0);
  } else if (width == 8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) copy_async<8>(dst + 8 * i, q + 8 * i, 4 * i < have);
  } else if (width == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) copy_async<4>(dst + 4 * i, q + 4 * i, 2 * i < have);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint16_t v = i < have ? __ldg(reinterpret_cast<const uint16_t*>(p) + i) : (uint16_t)0;
      asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + 2 * i), "h"(v) : "memory");
    }
  }
}
__device__ __forceinline__ void store16(uint32_t dst, const uint4& v) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
// (volatile: after the wait for the copy)
__device__ __forceinline__ uint4 load16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
// Four 8 x 8 matrices of 16-bit values, lane 8 i + j naming row j of the i-th: lane (g, q) gets (g, 2q) and (g, 2q + 1) of each, TRANS: (2q, g), (2q + 1, g).
template <bool TRANS>
__device__ __forceinline__ uint4 load_matrices(uint32_t row) {
  uint4 v;
  if constexpr (TRANS) asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(row) : "memory");
  else asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(row) : "memory");
  return v;
}
// Eight values of T, of which `have` are there; whole: on 16 bytes.
template <typename T>
__device__ __forceinline__ void store8(T* p, int have, bool whole, const float (&v)[8]) {
  alignas(16) T e[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) e[j] = Elem<T>::from_float(v[j]);
  if (whole && have >= 8) {
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < have) p[j] = e[j];
  }
}
// a + c * b for eight values of T
template <typename T>
__device__ __forceinline__ uint4 add8(const uint4& a, float c, const float (&b)[8]) {
  uint4 o;
  const uint32_t* in = &a.x;
  uint32_t* to = &o.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    if constexpr (std::is_same_v<T, __half>) f = __half22float2(*reinterpret_cast<const __half2*>(&in[i]));
    else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&in[i]));
    f.x = fmaf(c, b[2 * i], f.x);
    f.y = fmaf(c, b[2 * i + 1], f.y);
    if constexpr (std::is_same_v<T, __half>) { const __half2 h = __float22half2_rn(f); to[i] = *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __float22bfloat162_rn(f); to[i] = *reinterpret_cast<const uint32_t*>(&h); }
  }
  return o;
}

struct Params {
  const void *x, *w;       // activations; weights of all adapters
  uint16_t* h;             // inner products, by place: [T][r16 / 16][3 parts][16] bf16; of 16 ranks 0 1 4 5 8 9 12 13 2 3 6 7 10 11 14 15, as the operands want them
  const void* y;           // up: what is added to (null: zeros)
  void* out;
  const float* scales;     // null: 1
  const int *order, *starts;
  const int4* tiles;
  int64_t T, C;            // rows; the long dimension (K or N)
  int64_t tiles_n;
  int L, r, r16, width;    // r16: r in whole 16s; width: bytes that the rows of weights [C, r] (or of their gradient) are aligned to
  int split, each;         // blocks per cluster; tiles per block (0: the block counts them)
};

// A tile, or none (rows == 0) where the table does not fit the operands.
__device__ __forceinline__ int4 tile_of(const Params& p, int64_t k) {
  int4 t = p.tiles[k];
  if (t.z <= 0 || t.z > kRows || t.y < 0 || (int64_t)t.y + t.z > p.T || t.x >= p.L) t.z = 0;
  return t;
}
// The row at a place of the order; -1 where there is none.
__device__ __forceinline__ int row_at(const Params& p, int64_t place) {
  int row = p.order[place];
  row = row < 0 ? ~row : row;
  return row < (int)p.T ? row : -1;
}

// How many tiles have rows (with_adapter: of an adapter); they come first in the table, so that a search by the whole block finds the end: 256 of them are looked
// at at once.
__device__ int64_t tiles_with_rows(const Params& p, bool with_adapter) {
  int64_t lo = 0, n = p.tiles_n;   // all before lo have rows, none from lo + n on
  while (n > 0) {
    const int64_t each = (n + kThreads - 1) / kThreads, at = lo + threadIdx.x * each;   // of every part its first one
    bool has = false;
    if (threadIdx.x * each < n) {
      const int4 t = p.tiles[at];
      has = t.z > 0 && (!with_adapter || t.x >= 0);
    }
    const int parts = __syncthreads_count(has);
    if (parts == 0) break;
    const int64_t end = lo + n;
    lo += (parts - 1) * each + 1;
    n = min(each - 1, end - lo);
  }
  return lo;
}

// ---- h[place] = (c) sum over the long dimension of x[row] w.  Blocks by (tile, part of the long dimension, 16 MT ranks); the parts are a cluster
// whose blocks add up their sums through distributed shared memory.  Warps take every 8th (of their cluster: 8 split-th) 32 columns of x.
// Ranks are the rows of the products and activations their columns: a column's operands are two registers out of one 16-byte load, where a
// row's would have to be brought together from two.
// TALL: weights [C, r], else [r, C].
//
// Every warp has a ring of its own in shared memory, filled some steps ahead, in pieces of 16 bytes whose places are swizzled so that eight rows of
// a matrix are in different banks; no barrier but the warp's.  4096 rows of 16 adapters of rank 64, bf16: 25 us from K = 4096, 46 from K = 14336
// (2.6 TB/s of x); what bounds it there is L2, from which the weights come again for every 64 rows, as many bytes as x has.  Few rows: latencies, 10 us for
// 57 rows of 40 adapters of rank 20 (K 4096, f16).  The additions of every step's sums in fp32 are 2 to 5 us of the 25 and 46.
template <bool TALL, int MT>
struct Down {
  static constexpr int kRanks = 16 * MT, kW = 2 * MT, kPieces = 8 + kW, kStages = MT == 4 ? 3 : 2;
  static constexpr int kLine = kRows + 8;   // floats per rank of the sums: lanes' pairs are in different banks
  static constexpr size_t kRing = (size_t)kWarps * kStages * kPieces * 512, kSums = (size_t)kWarps * kRanks * kLine * 4;
  static constexpr size_t kBytes = kRing > kSums ? kRing : kSums;   // the sums lie where the ring was
};
template <typename T, bool TALL, bool WHOLE, int MT>
__global__ void __launch_bounds__(kThreads, MT == 4 ? 1 : 2) down_kernel(const Params p) {
  using D = Down<TALL, MT>;
  constexpr int kRanks = D::kRanks, kStages = D::kStages, kLine = D::kLine, kStageBytes = D::kPieces * 512;
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  asm volatile("griddepcontrol.launch_dependents;");   // the second product's blocks begin with what does not depend on this one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3;
  const int part = (int)(blockIdx.x % p.split);
  const int4 tile = tile_of(p, blockIdx.x / p.split);
  if (tile.z == 0 || tile.x < 0) return;   // the whole cluster
  const int eights = (tile.z + 7) / 8, r0 = blockIdx.y * kRanks, C = (int)p.C, step = p.split * kWarps * 32;
  int k = (part * kWarps + warp) * 32;     // of the step that is multiplied
  // Rows along the long dimension (x, weights [r, C]) are copied eight at a time, 8 k per lane: lane (g, q) has k 8 q of row g, which goes to
  // piece 4 g + (q ^ g / 2) of the eight rows' 32.
  int kl = k + q * 8;                      // the lane's, of the step that is loaded
  const uint32_t own = (g * 4 + (q ^ (g >> 1))) * 16;
  const T* x[8];
  bool has[8];
#pragma unroll
  for (int n = 0; n < 8; ++n) {
    const int row = n * 8 + g, at = row < tile.z ? row_at(p, tile.y + row) : -1;
    x[n] = static_cast<const T*>(p.x) + (int64_t)max(at, 0) * C + kl;
    has[n] = at >= 0;
  }
  // TALL: 32 rows of 2 MT pieces, one after the other, piece c of row i at c ^ tall(i).
  auto tall = [](int i) { return MT == 4 ? i & 7 : (MT == 2 ? i >> 1 & 3 : i >> 2 & 1); };
  const T* w = static_cast<const T*>(p.w) + (int64_t)tile.x * p.r * C;
  int kw = k;                              // TALL: of the step that is loaded
  if constexpr (!TALL) w += (int64_t)(r0 + g) * C + kl;
  const uint32_t ring = shared(smem) + warp * kStages * kStageBytes;
  auto load = [&](uint32_t to) {   // the next step
    const bool in = kl < C;
#pragma unroll
    for (int n = 0; n < 8; ++n)
      if (n < eights) {
        if constexpr (WHOLE) copy_async<16>(to + n * 512 + own, x[n], in && has[n]);
        else store16(to + n * 512 + own, has[n] ? load8<false>(x[n], C - kl) : make_uint4(0, 0, 0, 0));
        x[n] += step;
      }
    if constexpr (TALL) {
#pragma unroll
      for (int i = 0; i < 2 * MT; ++i) {
        const int row = (i * 32 + lane) / (2 * MT), c = lane % (2 * MT), rank = r0 + c * 8;
        copy8(to + 4096 + (row * 2 * MT + (c ^ tall(row))) * 16, w + (int64_t)(kw + row) * p.r + rank, kw + row < C ? p.r - rank : 0, p.width);
      }
      kw += step;
    } else {
      const T* v = w;
#pragma unroll
      for (int t = 0; t < 2 * MT; ++t) {
        const bool there = in && r0 + t * 8 + g < p.r;
        if constexpr (WHOLE) copy_async<16>(to + 4096 + t * 512 + own, v, there);
        else store16(to + 4096 + t * 512 + own, there ? load8<false>(v, C - kl) : make_uint4(0, 0, 0, 0));
        v += 8 * C;
      }
      w += step;
    }
    kl += step;
  };
  float acc[MT][8][4] = {};
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (k + s * step < C) load(ring + s * kStageBytes);
    commit();
  }
  // Rows that the lane names: of x, 8 k per matrix; of weights [r, C], two times eight ranks by two times 8 k; of TALL ones, 16 k by two times eight ranks.
  const int mr = lane & 7, mi = lane >> 3;
  const uint32_t x_row = (mr * 4 + (mi ^ (mr >> 1))) * 16;
  const uint32_t w_row[2] = {4096u + (mi & 1) * 512 + (mr * 4 + ((mi >> 1) ^ (mr >> 1))) * 16, 4096u + (mi & 1) * 512 + (mr * 4 + ((mi >> 1 | 2) ^ (mr >> 1))) * 16};
  uint32_t from = ring, to = ring + (kStages - 1) * kStageBytes;
  const uint32_t end = ring + kStages * kStageBytes;
  for (; k < C; k += step) {
    __syncwarp();   // everyone has read the stage that is filled now
    if (k + (kStages - 1) * step < C) load(to);
    commit();
    wait_all_but<kStages - 1>();
    __syncwarp();
    uint4 a[MT][2];   // of the first and the second 16 k
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (TALL) {
          const int row = h * 16 + (mi >> 1) * 8 + mr;
          a[m][h] = load_matrices<true>(from + 4096 + (row * 2 * MT + ((2 * m + (mi & 1)) ^ tall(row))) * 16);
        } else {
          a[m][h] = load_matrices<false>(from + m * 1024 + w_row[h]);
        }
      }
#pragma unroll
    for (int n = 0; n < 8; ++n)
      if (n < eights) {
        const uint4 v = load_matrices<false>(from + n * 512 + x_row);
        float sum[MT][4] = {};
#pragma unroll
        for (int m = 0; m < MT; ++m) mma<T>(sum[m], a[m][0].x, a[m][0].y, a[m][0].z, a[m][0].w, v.x, v.y);
#pragma unroll
        for (int m = 0; m < MT; ++m) mma<T>(sum[m], a[m][1].x, a[m][1].y, a[m][1].z, a[m][1].w, v.z, v.w);
#pragma unroll
        for (int m = 0; m < MT; ++m) add4(acc[m][n], sum[m]);
      }
    to = from;
    from = from + kStageBytes == end ? ring : from + kStageBytes;
  }
  wait_all_but<0>();
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);   // [kWarps][kRanks][kLine]
#pragma unroll
  for (int n = 0; n < 8; ++n)
    if (n < eights) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          *reinterpret_cast<float2*>(&red[(warp * kRanks + m * 16 + i * 8 + g) * kLine + n * 8 + q * 2]) = make_float2(acc[m][n][2 * i], acc[m][n][2 * i + 1]);
    }
  __syncthreads();
  // sums over the block's warps, then over the cluster's blocks; two ranks of a row per thread, rows next to each other
  const int n = kRanks / 2 * (eights * 8);
  auto at = [&](int i) { return i / (eights * 8) * 2 * kLine + i % (eights * 8); };
  for (int i = threadIdx.x; i < n; i += kThreads) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = red[at(i) + e * kLine];
#pragma unroll
      for (int v = 1; v < kWarps; ++v) s += red[v * kRanks * kLine + at(i) + e * kLine];
      red[at(i) + e * kLine] = s;
    }
  }
  if (p.split > 1) cluster.sync();
  else __syncthreads();
  const float c = p.scales ? p.scales[tile.x] : 1.0f;
  for (int i = threadIdx.x * p.split + part; i < n; i += kThreads * p.split) {
    float s[2] = {red[at(i)], red[at(i) + kLine]};
    if (p.split > 1) {
      s[0] = s[1] = 0.0f;
      for (int v = 0; v < p.split; ++v) {
        const float* other = cluster.map_shared_rank(red, v);
        s[0] += other[at(i)];
        s[1] += other[at(i) + kLine];
      }
    }
    const int row = i % (eights * 8), rank = r0 + i / (eights * 8) * 2;
    if (rank < p.r16 && row < tile.z) {
      uint32_t parts[3];
      split(rank < p.r ? c * s[0] : 0.0f, rank + 1 < p.r ? c * s[1] : 0.0f, parts);
      uint16_t* h = p.h + (int64_t)(tile.y + row) * 3 * p.r16 + rank / 16 * 48 + rank % 16 / 4 * 2 + (rank & 2) * 4;
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint32_t*>(h + 16 * i) = parts[i];
    }
  }
  if (p.split > 1) cluster.sync();   // no block leaves while others read its sums
}

// ---- out[row] = y[row] + (c) sum over ranks of h[place] w.  Blocks by (tiles, 256 columns), warps by 32 columns; steps of 16 rows and, inside, 16
// ranks.  Up to 64 ranks (KS steps) have their weights in registers, over all rows that an adapter has among the block's tiles.  More (CHUNKED): the
// sums of a tile stay in registers while its ranks come 32 (f16: 16) at a time.  (4096 rows of rank 64, [14336, 4096], both products, us: 115, CHUNKED 150; rank 32: 74 and 104.  4096 rows of rank
// 128, [4096, 4096]: 93.)
// WIDE: weights [r, C], else [C, r].
//
// Bound by the latency of y and by instructions: every lane copies its own pieces of y, three steps of rows ahead, into a ring in shared memory; the steps'
// rows are looked up once per block; h lies in shared memory as one matrix load per part wants it.  4096 rows of rank 64, bf16, cold: 96 us for C = 14336 (2.1
// TB/s of HBM), 34 for C = 4096: tensor cores 43 %, shared memory 38 %, HBM 26 %, 15 warps on an SM for their registers; a warp's issue waits for fixed latencies, shared memory and the
// tensor cores in turn.  The three parts' products alone would take 41 and 12, HBM 36 and 10.  (Two parts of h, which lose 2^-17: 84 and 31.)
constexpr int kUpStages = 4, kUpTiles = 16, kUpSteps = kUpTiles * kRows / 16;
template <int KS, bool CHUNKED>
struct Up {
  static constexpr int kStep = KS * 1536;   // bytes of h per step of 16 rows: [rank step][part][row][two pieces of 16, swapped in every other four rows]
  static constexpr size_t kBytes = (size_t)kWarps * kUpStages * 1024 + 8 * kStep;
};
template <typename T, bool WIDE, bool WHOLE, int KS, bool CHUNKED>
__global__ void __launch_bounds__(kThreads, CHUNKED ? 2 : (KS == 4 ? 2 : 3) - std::is_same_v<T, __half>) up_kernel(const Params p) {
  constexpr bool kSplitW = std::is_same_v<T, __half>;
  constexpr int kStep = Up<KS, CHUNKED>::kStep;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int4 tiles[kUpTiles];
  __shared__ int rows[kUpSteps + kUpStages][16];   // of every step (-1: none); behind the last one some without any
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3, C = (int)p.C;
  const int blocks = (C + 255) / 256, n0 = (int)(blockIdx.x % blocks) * 256 + warp * 32, n = n0 + q * 8;   // the lane's columns are n .. n + 7
  const int have = C - n;
  const bool in = have > 0, add = p.y != nullptr && in;
  const T* y = static_cast<const T*>(p.y) + n;
  T* out = static_cast<T*>(p.out) + n;
  uint32_t bh[KS][4][2], bl[kSplitW ? KS : 1][4][2];   // rank step, column tile, pair of the lane's 4 ranks
  int loaded = -1;                                     // whose weights they are
  const int64_t part = blockIdx.x / blocks, parts = gridDim.x / blocks, n_tiles = p.each ? p.tiles_n : tiles_with_rows(p, p.y == p.out);
  const int64_t end = p.each ? min((part + 1) * p.each, n_tiles) : n_tiles * (part + 1) / parts;
  for (int64_t first = p.each ? part * p.each : n_tiles * part / parts; first < end; first += kUpTiles) {
    const int count = (int)min((int64_t)kUpTiles, end - first);
    __syncthreads();   // everyone is through with the tiles before
    if (threadIdx.x < count) {
      int4 t = tile_of(p, first + threadIdx.x);
      if (t.x < 0 && p.y == p.out) t.z = 0;   // rows without an adapter are there already
      tiles[threadIdx.x] = t;
    }
    for (int i = threadIdx.x; i < (kUpSteps + kUpStages) * 16; i += kThreads) rows[i / 16][i % 16] = -1;
    __syncthreads();
    int steps = 0;
    for (int k = 0; k < count; ++k) {   // (four tiles at once)
      const int4 t = tiles[k];
      const int i = threadIdx.x % kRows;
      if (k % (kThreads / kRows) == threadIdx.x / kRows && i < t.z) rows[steps + i / 16][i % 16] = row_at(p, t.y + i);
      steps += (t.z + 15) / 16;
    }
    const uint32_t ring = shared(smem) + warp * kUpStages * 1024 + lane * 16, hs = shared(smem) + kWarps * kUpStages * 1024;
    const uint32_t h_row = hs + (lane & 15) * 32 + ((lane >> 4 ^ lane >> 2) & 1) * 16;   // that the lane names: of two times eight rows by two times eight ranks
    auto next_tile = [&](int k) {
      while (k < count && tiles[k].z == 0) ++k;
      return k;
    };
    auto copy_h = [&](int k, int r0, int buffer) {
      if (k >= count || tiles[k].x < 0) return;
      constexpr int kPer = 6 * KS;   // pieces of 16 bytes per row
      const int z = tiles[k].z;
      const uint16_t* src = p.h + (int64_t)tiles[k].y * 3 * p.r16 + r0 * 3;
      for (int i = threadIdx.x; i < z * kPer; i += kThreads) {
        const int row = i / kPer, piece = i % kPer;
        if (KS == 1 || r0 + piece / 6 * 16 < p.r16)
          copy_async<16>(hs + buffer * 4 * kStep + row / 16 * kStep + piece / 2 * 512 + row % 16 * 32 + ((piece ^ row >> 2) & 1) * 16, src + row * 3 * p.r16 + piece * 8, true);
      }
    };
    const T* w = nullptr;
    auto weights = [&](int r0) {
      uint32_t b[KS][4][2];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        if constexpr (WIDE) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int rank = r0 + s * 16 + (g >> 1) * 4 + j * 2 + (g & 1);
            const uint4 v = rank < p.r ? load8<WHOLE>(w + (int64_t)rank * C + n, have) : make_uint4(0, 0, 0, 0);
            b[s][0][j] = v.x; b[s][1][j] = v.y; b[s][2][j] = v.z; b[s][3][j] = v.w;
          }
        } else {
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int col = n0 + (g >> 1) * 8 + t * 2 + (g & 1), rank = r0 + s * 16 + q * 4;
            load4(w + (int64_t)col * p.r + rank, col < C ? p.r - rank : 0, p.width, b[s][t]);
          }
        }
      }
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            uint32_t lo;
            as_bf16<T>(WIDE ? transposed(b[s][t][j]) : b[s][t][j], &bh[s][t][j], &lo);
            if constexpr (kSplitW) bl[s][t][j] = lo;
          }
    };
    int k = next_tile(0), buffer = 0, ahead = 0, now = 0;
    auto issue = [&] {   // y of the next step
      const uint32_t to = ring + (ahead % kUpStages) * 1024;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = rows[ahead][i * 8 + g];
        if constexpr (WHOLE) copy_async<16>(to + i * 512, y + (int64_t)row * C, add && row >= 0);
        else store16(to + i * 512, add && row >= 0 ? load8<false, false>(y + (int64_t)row * C, have) : make_uint4(0, 0, 0, 0));
      }
      commit();
      ++ahead;
    };
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kUpStages - 1; ++i) issue();
    if (!CHUNKED && k < count && tiles[k].x >= 0 && loaded != tiles[k].x) {
      loaded = tiles[k].x;
      w = static_cast<const T*>(p.w) + (int64_t)loaded * p.r * C;
      weights(0);
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");   // all of h, of the launch before
    copy_h(k, 0, 0);
    commit();
    for (int last = 4; k < count;) {
      const int4 tile = tiles[k];
      const bool plain = tile.x < 0;   // rows without an adapter
      float c = 0.0f;
      if (!plain) {
        c = p.scales ? p.scales[tile.x] : 1.0f;
        w = static_cast<const T*>(p.w) + (int64_t)tile.x * p.r * C;
        if (!CHUNKED && loaded != tile.x) {
          weights(0);
          loaded = tile.x;
        }
      }
      const int after = next_tile(k + 1), before = last;
      last = (tile.z + 15) / 16;
      auto finish = [&](const float (&acc)[4][4]) {   // the step's sums to its rows
        wait_all_but<kUpStages - 1>();
        const uint32_t from = ring + (now % kUpStages) * 1024;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int row = rows[now][i * 8 + g];
          if (row < 0 || !in) continue;
          const float sum[8] = {acc[0][2 * i], acc[0][2 * i + 1], acc[1][2 * i], acc[1][2 * i + 1], acc[2][2 * i], acc[2][2 * i + 1], acc[3][2 * i], acc[3][2 * i + 1]};
          uint4 v = load16(from + i * 512);
          if (!plain) v = add8<T>(v, c, sum);
          T* o = out + (int64_t)row * C;
          if constexpr (WHOLE) {
            *reinterpret_cast<uint4*>(o) = v;
          } else {
            T e[8];
            *reinterpret_cast<uint4*>(e) = v;
#pragma unroll
            for (int j = 0; j < 8; ++j)
              if (j < have) o[j] = e[j];
          }
        }
        ++now;
      };
      // The ranks r0 .. r0 + 16 KS of 16 rows, whose h lies at src; the smallest parts first, so that few products are truncated at the whole sum's size.
      auto products = [&](float (&acc)[4][4], int r0, uint32_t src) {
#pragma unroll
        for (int i = 2; i >= 0; --i)
#pragma unroll
          for (int s = 0; s < KS; ++s) {
            if (KS > 1 && r0 + s * 16 >= p.r16) break;
            const uint4 a = load_matrices<false>(src + s * 1536 + i * 512);
            if constexpr (kSplitW) {
              if (i < 2) {
#pragma unroll
                for (int t = 0; t < 4; ++t) mma<__nv_bfloat16>(acc[t], a.x, a.y, a.z, a.w, bl[s][t][0], bl[s][t][1]);
              }
            }
#pragma unroll
            for (int t = 0; t < 4; ++t) mma<__nv_bfloat16>(acc[t], a.x, a.y, a.z, a.w, bh[s][t][0], bh[s][t][1]);
          }
      };
      // (rows behind the tile's last one have what was there before; their products are not stored)
      if constexpr (CHUNKED) {
        float acc[kRows / 16][4][4] = {};
        for (int r0 = 0; r0 == 0 || (r0 < p.r16 && !plain); r0 += 16 * KS, buffer ^= 1) {
          // these ranks' h was issued before the last tile's four steps, or last
          if (r0 == 0 && now != 0 && before == 4) wait_all_but<4>();
          else wait_all_but<0>();
          __syncthreads();
          if (r0 + 16 * KS < p.r16 && !plain) copy_h(k, r0 + 16 * KS, buffer ^ 1);
          else copy_h(after, 0, buffer ^ 1);
          commit();
          if (plain) continue;
          weights(r0);
          const uint32_t src = h_row + buffer * 4 * kStep;
#pragma unroll
          for (int m = 0; m < kRows / 16; ++m)
            if (m < last) {
              float sum[4][4] = {};
              products(sum, r0, src + m * kStep);
#pragma unroll
              for (int t = 0; t < 4; ++t) add4(acc[m][t], sum[t]);
            }
        }
#pragma unroll
        for (int m = 0; m < kRows / 16; ++m)
          if (m < last) {
            issue();
            finish(acc[m]);
          }
      } else {
        // the group with this tile's h was issued with the first step of the tile before, four steps ago if that was a whole one
        if (now == 0 || before < 4) wait_all_but<0>();
        __syncthreads();
        copy_h(after, 0, buffer ^ 1);
        uint32_t src = h_row + buffer * 4 * kStep;
        for (int m = 0; m < last; ++m, src += kStep) {
          issue();
          float acc[4][4] = {};
          if (!plain) products(acc, 0, src);
          finish(acc);
        }
        buffer ^= 1;
      }
      k = after;
    }
    wait_all_but<0>();
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");   // (blocks without work: who comes next waits for the first product through this one)
}

// ---- out_l = (c) sum over l's rows of h[place] x[row]^T.  Blocks by (128 columns, part of the rows; adapter; 16 MT ranks), the parts are a
// cluster; warps by (32 columns, half of a step's 32 rows).  TALL: out [C, r], else [r, C].
//
// Rows lie in shared memory as they come, and matrix loads that transpose make both operands of them; h's parts lie apart there.  Which rows come next is
// copied there, too, a ring ahead, so that no step waits for it.  (4096 rows of one adapter of rank 64 and 4096 columns: 27 us, 90 when every 32 columns' h was
// transposed in registers; HBM 5.  2048 rows of 4 adapters of rank 16, [14336, 4096], forward and all gradients: 98 us, 106 with three stages and rows looked up
// one step ahead; 1000 adapters of a row each have no use for it: 229 and 215; all these with two parts of h.  With three, and every step's sums added in fp32, 39 us, and 99.)  Bound by latencies: a block has few steps, and reads where its rows are
// before it reads them; with 64 ranks and 14336 columns (107 us cold) tensor cores are at 38 %, shared memory at 36.  Two blocks on an SM (rank 64, f16: all gradients
// 223 us with one, 158 with two).
template <bool TALL, int MT>
struct Outer {
  static constexpr int kRanks = 16 * MT, kCols = 128, kSteps = 32, kStages = MT == 1 ? 5 : 4;
  static constexpr int kXPitch = kCols * 2 + 16, kHPitch = kRanks * 2 + 16;   // (eight rows of a matrix are in different banks)
  static constexpr int kStage = kSteps * (kXPitch + 3 * kHPitch);
  static constexpr int kLine = kCols + (TALL ? 2 : 8);   // floats per rank of the sums
  static constexpr size_t kRing = (size_t)kStages * kStage, kSums = (size_t)2 * kRanks * kLine * 4, kBytes = kRing > kSums ? kRing : kSums;
};
template <typename T, bool TALL, bool WHOLE, int MT>
__global__ void __launch_bounds__(kThreads, 2) outer_kernel(const Params p) {
  using O = Outer<TALL, MT>;
  constexpr int kRanks = O::kRanks, kCols = O::kCols, kLine = O::kLine, kStages = O::kStages, kXPitch = O::kXPitch, kHPitch = O::kHPitch;
  constexpr bool kSplitX = std::is_same_v<T, __half>;
  extern __shared__ __align__(16) unsigned char smem[];
  cg::cluster_group cluster = cg::this_cluster();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, q = lane & 3, slot = warp >> 2, C = (int)p.C;
  const int part = (int)(blockIdx.x % p.split), l = blockIdx.y, r0 = blockIdx.z * kRanks, c0 = (int)(blockIdx.x / p.split) * kCols;
  const int lo = max(p.starts[l], 0), hi = min(p.starts[l + 1], (int)p.T), step = p.split * O::kSteps, first = lo + part * O::kSteps;
  const int n = first < hi ? (hi - first + step - 1) / step : 0;
  // Copied per step by a thread: 8 columns of two rows of x; of h, pieces of 8 ranks of a part.
  constexpr int kPer = 6 * MT;   // pieces per row
  const int xr = threadIdx.x / 16, xc = threadIdx.x % 16, have = C - c0 - xc * 8;
  const T* x = static_cast<const T*>(p.x) + c0 + xc * 8;
  __shared__ int order[kStages][O::kSteps];   // of the steps that are loaded next: copied a ring ahead of their rows
  int place = first;   // of the step that is loaded
  auto row_of = [&](int at, int row) { return at < hi && row < (int)p.T ? row : -1; };
  auto look_ahead = [&](int slot) {   // a ring less one ahead
    const int at = place + (kStages - 1) * step + threadIdx.x;
    if (threadIdx.x < O::kSteps) copy_async<4>(shared(&order[slot][threadIdx.x]), p.order + at, at < hi);
  };
  const uint32_t ring = shared(smem);
  auto load = [&](int stage, const int (&row)[2]) {   // the next step
    const uint32_t to = ring + stage * O::kStage;
    look_ahead(stage == 0 ? kStages - 1 : stage - 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t d = to + (xr + i * 16) * kXPitch + xc * 16;
      const T* src = x + (int64_t)row[i] * C;
      if constexpr (WHOLE) copy_async<16>(d, src, row[i] >= 0 && have > 0);
      else store16(d, row[i] >= 0 ? load8<false>(src, have) : make_uint4(0, 0, 0, 0));
    }
#pragma unroll
    for (int i = 0; i < (O::kSteps * kPer + kThreads - 1) / kThreads; ++i) {
      const int id = threadIdx.x + i * kThreads, at = id / kPer, piece = id % kPer;
      if (O::kSteps * kPer % kThreads != 0 && at >= O::kSteps) break;
      copy_async<16>(to + O::kSteps * (kXPitch + piece / 2 % 3 * kHPitch) + at * kHPitch + piece / 6 * 32 + piece % 2 * 16,
                     p.h + (int64_t)(place + at) * 3 * p.r16 + r0 * 3 + piece * 8, place + at < hi && r0 + piece / 6 * 16 < p.r16);
    }
    place += step;
  };
  float acc[MT][4][4] = {};
  int begin[kStages - 1][2];
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int at = first + s * step + xr + i * 16;
      begin[s][i] = row_of(at, at < hi ? p.order[at] : -1);
    }
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    if (s < n) load(s, begin[s]);
    commit();
  }
  const int mr = lane & 7, mi = lane >> 3;
  const uint32_t x_at = (slot * 16 + (mi & 1) * 8 + mr) * kXPitch + ((warp & 3) * 4 + (mi >> 1)) * 16;
  const uint32_t h_at = O::kSteps * kXPitch + (slot * 16 + (mi >> 1) * 8 + mr) * kHPitch + (mi & 1) * 16;
  int from = 0, to = kStages - 1;
  for (int k = 0; k < n; ++k) {
    wait_all_but<kStages - 2>();
    __syncthreads();   // the step is there, and everyone has read the stage that is filled now
    if (k + kStages - 1 < n) {
      const int row[2] = {row_of(place + xr, order[to][xr]), row_of(place + xr + 16, order[to][xr + 16])};
      load(to, row);
    }
    commit();
    const uint32_t src = ring + from * O::kStage;
    uint32_t bh[4][2], bl[4][2];
#pragma unroll
    for (int v = 0; v < 4; v += 2) {
      const uint4 b = load_matrices<true>(src + x_at + v * 16);
      as_bf16<T>(b.x, &bh[v][0], &bl[v][0]);
      as_bf16<T>(b.y, &bh[v][1], &bl[v][1]);
      as_bf16<T>(b.z, &bh[v + 1][0], &bl[v + 1][0]);
      as_bf16<T>(b.w, &bh[v + 1][1], &bl[v + 1][1]);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      if (MT > 1 && r0 + m * 16 >= p.r16) break;
      float sum[4][4] = {};
#pragma unroll
      for (int i = 2; i >= 0; --i) {   // (the smallest products first)
        const uint4 a = load_matrices<true>(src + h_at + m * 32 + i * O::kSteps * kHPitch);
        if constexpr (kSplitX) {
          if (i < 2) {
#pragma unroll
            for (int v = 0; v < 4; ++v) mma<__nv_bfloat16>(sum[v], a.x, a.y, a.z, a.w, bl[v][0], bl[v][1]);
          }
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) mma<__nv_bfloat16>(sum[v], a.x, a.y, a.z, a.w, bh[v][0], bh[v][1]);
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) add4(acc[m][v], sum[v]);
    }
    to = from;
    from = from + 1 == kStages ? 0 : from + 1;
  }
  wait_all_but<0>();
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);   // [2][kRanks][kLine]
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(&red[(slot * kRanks + m * 16 + (g >> 1) * 4 + i * 2 + (g & 1)) * kLine + (warp & 3) * 32 + v * 8 + q * 2]) =
            make_float2(acc[m][v][2 * i], acc[m][v][2 * i + 1]);   // (ranks back in their order)
  __syncthreads();
  if (p.split > 1) {
    for (int i = threadIdx.x; i < kRanks * kCols; i += kThreads) {
      const int at = i / kCols * kLine + i % kCols;
      red[at] += red[kRanks * kLine + at];
    }
    cluster.sync();
  }
  const float c = p.scales ? p.scales[l] : 1.0f;
  T* out = static_cast<T*>(p.out) + (int64_t)l * p.r * C;
  float* sums = red + kRanks * kLine;   // with a cluster: what the block stores
  const int wide = kCols / p.split;     // TALL: its columns
  // A thread stores eight values at once: ranks of a column (lanes: 16 columns by twice 8 ranks, so that pairs fill a sector), or columns of a rank.
  if constexpr (TALL) {
    if (p.split > 1) {   // the others' sums along their rows, then the block's own along its columns
      for (int i = threadIdx.x; i < kRanks * wide / 2; i += kThreads) {
        const int at = i / (wide / 2) * kLine + part * wide + i % (wide / 2) * 2;
        float2 s = make_float2(0.0f, 0.0f);
        for (int v = 0; v < p.split; ++v) {
          const float2 o = *reinterpret_cast<const float2*>(cluster.map_shared_rank(red, v) + at);
          s.x += o.x;
          s.y += o.y;
        }
        *reinterpret_cast<float2*>(sums + at) = s;
      }
      __syncthreads();
    }
    for (int i = threadIdx.x; i < 2 * MT * wide; i += kThreads) {
      const int cc = part * wide + i / (32 * MT) * 16 + i % 16, rank = (i / 32 % MT * 2 + i / 16 % 2) * 8;
      float s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = (rank + j) * kLine + cc;
        s[j] = c * (p.split > 1 ? sums[at] : red[at] + sums[at]);
      }
      if (c0 + cc < C) store8(out + (int64_t)(c0 + cc) * p.r + r0 + rank, p.r - r0 - rank, p.width == 16, s);
    }
  } else {
    const int each = kRanks * kCols / 8 / p.split;
    for (int i = threadIdx.x; i < each; i += kThreads) {
      const int rank = (part * each + i) / (kCols / 8), cc = (part * each + i) % (kCols / 8) * 8, at = rank * kLine + cc;
      float s[8] = {};
      auto add = [&](const float* o) {
        const float4 u = *reinterpret_cast<const float4*>(o), w = *reinterpret_cast<const float4*>(o + 4);
        s[0] += u.x; s[1] += u.y; s[2] += u.z; s[3] += u.w;
        s[4] += w.x; s[5] += w.y; s[6] += w.z; s[7] += w.w;
      };
      if (p.split > 1) {
        for (int v = 0; v < p.split; ++v) add(cluster.map_shared_rank(red, v) + at);
      } else {
        add(red + at);
        add(sums + at);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] *= c;
      if (r0 + rank < p.r) store8(out + (int64_t)(r0 + rank) * C + c0 + cc, C - c0 - cc, WHOLE, s);
    }
  }
  if (p.split > 1) cluster.sync();   // no block leaves while others read its sums
}

bool aligned(const void* p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// Bytes (2 to 16) that rows of `pitch` bytes from p on are aligned to.
int width_of(const void* p, int64_t pitch) {
  int w = 16;
  while (w > 2 && (!aligned(p, w) || pitch % w != 0)) w /= 2;
  return w;
}
// Blocks per cluster: a power of two up to 8, as many as fit on the SMs at once, with work for everyone.  (With at most 1, 2, 4, 8, by graph replay, us: one row of
// rank 16, [14336, 4096], forward 8.6 7.2 6.2 5.7, gradient of x 23.9 14.7 10.0 7.7; 57 rows that choose among 40 adapters of rank 20, f16, [11008, 4096], gradient
// of x 40 26 20 19; 4096 rows of rank 64 123 83 83 83.)  Eight only where a sixth of the SMs is left to blocks of the product after it, which begin beside it: both projections of 2048 rows of 4 adapters of rank
// 16 68 us with four, 70 with eight; 1024 rows of rank 64, [4096, 4096], 24 and 34.
int split_of(int64_t blocks, int64_t slots, int64_t most, bool beside) {
  int s = 1;
  while (s < 8 && blocks * 2 * s <= (beside && s == 4 ? slots * 5 / 6 : slots) && 2 * s <= most) s *= 2;
  return s;
}
// Tiles that there will be, about (the table has room for the most that there can be): rows that choose their adapters at random.
int64_t likely_tiles(const Params& p) {
  const double used = p.L * (1.0 - exp(-(double)p.T / p.L)), rows = p.T / used;
  return std::max<int64_t>(1, std::min<int64_t>(p.T, p.T / kRows + (int64_t)(used * (1.0 - 0.5 * std::min(1.0, rows / kRows)))));
}
// Tiles per block of the second product.  A block takes about as long as its tiles and three quarters of one more; blocks run in waves.  (By graph
// replay, both products, us, with 1, 2, 3, 4, 5, 6, 8 tiles: 57 rows that choose among 40 adapters of rank 20, f16, [11008, 4096] 27 23 23 24 21 24 28; 4096 rows of rank 64,
// [14336, 4096] 135 120 116 120 115 123 127; 2048 rows of rank 16 41 39 37 40 37 40 48: the rule takes 5 for all three.)
int tiles_per_block(const Params& p, int64_t cols, int64_t slots) {
  const int64_t tiles = likely_tiles(p);
  double best = 0;
  int each = 1;
  for (int e = 1; e <= 8; ++e) {
    const double time = (double)(((tiles + e - 1) / e * cols + slots - 1) / slots) * (e + 0.75);
    if (e == 1 || time < best) { best = time; each = e; }
  }
  return each;
}

template <typename K>
int launch(K kern, const Params& p, dim3 grid, int threads, size_t smem, cudaStream_t st, bool beside = false) {
  if (int rc = allow_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  cfg.attrs = at;
  if (p.split > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  } else if (beside) {   // may start while the launch before runs, whose results it waits for
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  }
  B200Q_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p));
  B200Q_LAUNCH_OK("adapter kernel");
  return B200Q_OK;
}

template <typename T, bool TALL, bool WHOLE>
int down(Params p, cudaStream_t st) {
  const int mt = p.r <= 16 ? 1 : (p.r <= 32 ? 2 : 4), chunks = (p.r + 16 * mt - 1) / (16 * mt);
  p.split = split_of(likely_tiles(p) * chunks, 148 * (mt == 4 ? 1 : 2), p.C / (kWarps * 32), true);
  const dim3 grid((unsigned)(p.tiles_n * p.split), chunks);
  if (mt == 1) return launch(down_kernel<T, TALL, WHOLE, 1>, p, grid, kThreads, Down<TALL, 1>::kBytes, st);
  if (mt == 2) return launch(down_kernel<T, TALL, WHOLE, 2>, p, grid, kThreads, Down<TALL, 2>::kBytes, st);
  return launch(down_kernel<T, TALL, WHOLE, 4>, p, grid, kThreads, Down<TALL, 4>::kBytes, st);
}
template <typename T, bool WIDE, bool WHOLE>
int up(Params p, cudaStream_t st) {
  p.split = 1;
  const int64_t cols = (p.C + 255) / 256;
  const int64_t slots = 148 * (p.r > 64 ? 2 : (p.r > 32 ? 2 : 3) - std::is_same_v<T, __half>);
  // Where blocks have 8 tiles or more each, those that fit on the SMs at once count the tiles that have rows and share them evenly, if that leaves hardly any SM without a block or if the sum
  // is in place, where tiles of rows without an adapter are no work.  (Counted / not, graph replay, us: 16384 rows of 16 adapters, [4096, 4096], rank 64 160 / 162, 16 83 / 85, 128 342 / 347; 8192 rows of
  // which 9 in 10 have no adapter, [14336, 2048], in place, rank 64 42 / 54, 16 22 / 27; with an eighth of the SMs left out: 8192 rows of rank 32, [14336, 4096], 143 / 130; a quarter: 4096 of rank 64, f16, 202 / 185.  For
  // fewer tiles the count costs more than a last wave: 16 rows of as many adapters 8.8 / 6.9.)
  const int64_t even = std::max<int64_t>(1, slots / cols);
  p.each = likely_tiles(p) * cols >= 8 * slots && (p.y == p.out || even * cols * 25 >= slots * 24) ? 0 : tiles_per_block(p, cols, slots);
  const int64_t parts = p.each ? (p.tiles_n + p.each - 1) / p.each : even;
  const dim3 grid((unsigned)(cols * parts));
  if (p.r <= 16) return launch(up_kernel<T, WIDE, WHOLE, 1, false>, p, grid, kThreads, Up<1, false>::kBytes, st, true);
  if (p.r <= 32) return launch(up_kernel<T, WIDE, WHOLE, 2, false>, p, grid, kThreads, Up<2, false>::kBytes, st, true);
  if (p.r <= 64) return launch(up_kernel<T, WIDE, WHOLE, 4, false>, p, grid, kThreads, Up<4, false>::kBytes, st, true);
  constexpr int kChunk = std::is_same_v<T, __half> ? 1 : 2;   // (f16: weights of 32 ranks in two parts would be spilled; 4096 rows of rank 128, [4096, 4096], 133 us instead of 115)
  return launch(up_kernel<T, WIDE, WHOLE, kChunk, true>, p, grid, kThreads, Up<kChunk, true>::kBytes, st, true);
}
template <typename T, bool TALL, bool WHOLE>
int outer(Params p, cudaStream_t st) {
  const int mt = p.r <= 16 ? 1 : (p.r <= 32 ? 2 : 4), chunks = (p.r + 16 * mt - 1) / (16 * mt);
  const int64_t cols = (p.C + 127) / 128;
  p.split = split_of(cols * p.L * chunks, 148 * 2, p.T / 64, false);
  const dim3 grid((unsigned)(cols * p.split), p.L, chunks);
  if (mt == 1) return launch(outer_kernel<T, TALL, WHOLE, 1>, p, grid, kThreads, Outer<TALL, 1>::kBytes, st);
  if (mt == 2) return launch(outer_kernel<T, TALL, WHOLE, 2>, p, grid, kThreads, Outer<TALL, 2>::kBytes, st);
  return launch(outer_kernel<T, TALL, WHOLE, 4>, p, grid, kThreads, Outer<TALL, 4>::kBytes, st);
}

// Of a call: which form of a kernel.
enum class Step { Down, DownTall, Up, UpWide, Outer, OuterTall };
template <typename T, bool WHOLE>
int run(Step step, const Params& p, cudaStream_t st) {
  switch (step) {
    case Step::Down: return down<T, false, WHOLE>(p, st);
    case Step::DownTall: return down<T, true, WHOLE>(p, st);
    case Step::Up: return up<T, false, WHOLE>(p, st);
    case Step::UpWide: return up<T, true, WHOLE>(p, st);
    case Step::Outer: return outer<T, false, WHOLE>(p, st);
    default: return outer<T, true, WHOLE>(p, st);
  }
}
int run(Step step, Params p, int dtype, cudaStream_t st) {
  const bool lies = step == Step::Down || step == Step::UpWide;   // weights' rows are along the long dimension
  bool whole = p.C % 8 == 0;
  for (const void* q : {p.x, p.y, lies ? p.w : nullptr, step == Step::OuterTall ? nullptr : static_cast<const void*>(p.out)}) whole = whole && aligned(q, 16);
  p.width = step == Step::OuterTall ? width_of(p.out, 2 * p.r) : (p.w && !lies ? width_of(p.w, 2 * p.r) : 2);
  if (dtype == B200Q_F16) return whole ? run<__half, true>(step, p, st) : run<__half, false>(step, p, st);
  return whole ? run<__nv_bfloat16, true>(step, p, st) : run<__nv_bfloat16, false>(step, p, st);
}

int check(const char* tag, int dtype, int64_t T, int64_t L, int64_t N, int64_t K, int64_t r) {
  if (dtype != B200Q_F16 && dtype != B200Q_BF16) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", tag, dtype);
  if (T < 0 || L < 0 || N < 0 || K < 0 || r < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] negative dimension.", tag);
  if (T > (1 << 30) || L > 4096 || N > (1 << 24) || K > (1 << 24) || r > 4096)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^30 rows, 4096 adapters, widths of 2^24 or ranks of 4096.", tag);
  const int64_t tiles = b200q_group_rows_tiles(T, L), most = INT32_MAX;
  if (tiles * 8 > most || tiles > most / ((N + 255) / 256 + 1) || tiles > most / ((K + 255) / 256 + 1))
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^31 - 1 blocks.", tag);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" size_t b200q_add_adapters_inner_bytes(int64_t T, int64_t r) { return T <= 0 || r <= 0 ? 0 : (size_t)T * ((r + 15) / 16 * 16) * 6; }

extern "C" int b200q_add_adapters(const void* y, const void* x, const void* a, const void* b, int dtype, int64_t T, int64_t L, int64_t N, int64_t K,
                                  int64_t r, const int32_t* order, const int32_t* tiles, const float* scales, void* h, void* out, void* stream) {
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
  if (!on_boundaries({y, x, a, b, out}, 2) || !on_boundaries({order, scales}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  if (!aligned(tiles, 16) || !aligned(h, 16)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] tiles and h must be 16-byte aligned", tag);
  Params p{};
  p.split = 1;
  p.x = x; p.w = a; p.h = static_cast<uint16_t*>(h); p.r16 = (int)(r + 15) / 16 * 16;
  p.order = order; p.tiles = reinterpret_cast<const int4*>(tiles); p.tiles_n = b200q_group_rows_tiles(T, L);
  p.T = T; p.C = K; p.L = (int)L; p.r = (int)r;
  const ScratchLock lock(h);
  if (int rc = run(Step::Down, p, dtype, st)) return rc;
  p.x = nullptr; p.w = b; p.y = y; p.out = out; p.scales = scales; p.C = N;
  return run(Step::Up, p, dtype, st);
}

extern "C" int b200q_add_adapters_grad(const void* dy, const void* x, const void* a, const void* b, int dtype, int64_t T, int64_t L, int64_t N, int64_t K,
                                       int64_t r, const int32_t* order, const int32_t* starts, const int32_t* tiles, const float* scales, const void* h,
                                       void* g, void* dx, void* da, void* db, void* stream) {
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
  if (!on_boundaries({dy, x, a, b, dx, da, db}, 2) || !on_boundaries({order, starts, scales}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  if (!aligned(tiles, 16) || !aligned(h, 16) || !aligned(g, 16)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] tiles, h and g must be 16-byte aligned", tag);
  Params p{};
  p.split = 1;
  p.h = static_cast<uint16_t*>(g); p.r16 = (int)(r + 15) / 16 * 16;
  p.order = order; p.starts = starts; p.tiles = reinterpret_cast<const int4*>(tiles); p.tiles_n = b200q_group_rows_tiles(T, L);
  p.T = T; p.L = (int)L; p.r = (int)r;
  const ScratchLock lock(g);
  if (dx || da) {
    Params d = p;
    d.x = dy; d.w = b; d.scales = scales; d.C = N;
    if (int rc = run(Step::DownTall, d, dtype, st)) return rc;
  }
  if (dx) {
    Params d = p;
    d.w = a; d.out = dx; d.C = K;
    if (int rc = run(Step::UpWide, d, dtype, st)) return rc;
  }
  if (da) {
    Params d = p;
    d.x = x; d.out = da; d.C = K;
    if (int rc = run(Step::Outer, d, dtype, st)) return rc;
  }
  if (db) {
    Params d = p;
    d.x = dy; d.h = static_cast<uint16_t*>(const_cast<void*>(h)); d.out = db; d.scales = scales; d.C = N;
    if (int rc = run(Step::OuterTall, d, dtype, st)) return rc;
  }
  return B200Q_OK;
}
