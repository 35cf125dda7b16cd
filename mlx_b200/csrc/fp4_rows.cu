// 4-bit products of up to 8 rows, dense or grouped, in one launch: y[t] = Gx Gw[e] (quantized x[t]) (wq[e], scales[e])^T.
//
// Every block quantizes all of x into shared memory and goes through its share of the weights once, which lie as the caller has them.  A
// warp has 16 rows of weights and every 2^split-th piece of 256 k, fetched by asynchronous copies while the piece before is multiplied.
// Codes become f16 numbers (e2m1 to f16 is one conversion per pair) for mma.sync (m16n8k16), weights as A and x as B, sums in fp32:
//   nvfp4  times their E4M3 scale before, in both operands: at most 2688, a multiple of 2^-10 of six significant bits, so exact
//   mxfp4  codes alone (a power of two of E8M0's range has no f16 number): a group's 32 products are summed from zero, then times
//          both scales in fp32 (one product where fp32 holds it whatever the weights' scale is, else two factors: kXScale)
// Sums of the warps that share rows go through shared memory and are added in order.  Rows beyond the sum of the sizes are zeroed.
//
// Bound: latencies up to some 10 million weights (4096^2, one row: 6.8 us, of which the launch, x, the first weights and the last sums
// are 5), then instructions: 400 per piece and warp, ALU 61 % and issue slots 64 % busy, 3.6 TB/s (28672 x 8192: 36 us).
#include "fp4.cuh"

namespace b200q {
namespace {

using namespace fp4;

constexpr int kWarps = 16, kThreads = 32 * kWarps;
constexpr int kMostRows = 8;       // of x: columns of one product
constexpr int kPieceK = 256;
constexpr int kPad = 20;            // floats from token to token of a partial sum: eight lanes of four tokens on 32 banks
// mxfp4: x's scales are kept times 2^-6.  Times a scale of the weights (2^-127 to 2^127) that is a fp32 number without loss as long as x's
// own lies between 2^-14 and 2^6 (groups whose largest magnitude is 2^-12 to 512), and all products of a group's sum with it are multiples
// of 2^-149.  Where one of x's scales lies outside, both factors are applied one after the other, the smaller one of x's and 1 first, so
// that nothing passes fp32's range but a result that does (one row: [14336, 4096] 16.0 for 14.0 us).
constexpr float kXScale = 0x1p-6f;
constexpr uint32_t kLeastX = 127 - 14, kMostX = 127 + 6;
constexpr int kStages = 2;          // (three: the same; four: 15 % slower where the weights are many)
constexpr int kRowBytes = 144;      // of codes from row to row of a stage: eight rows' words on 32 banks
constexpr int kStageBytes = 16 * kRowBytes + 16 * 16;
constexpr size_t kSmemMax = 227 * 1024 - 1024;

struct RowsParams {
  const void* x;
  const uint8_t* wq;
  const uint8_t* scales;
  const void* sizes;        // null: one group
  void* y;
  const float *gx, *gw;
  uint32_t* status;
  int T, E, N, K, size_bytes, gw_each;
  int tiles;                // of 16 rows of weights, per group
  int pieces;               // of K
  int half;                 // the last piece has 128 k only
  int pitch;                // bytes of a row of x in shared memory
  int x_stride;             // mxfp4: floats from group to group of x's scales there
};

__device__ __forceinline__ uint32_t times(uint32_t v, __half2 m) {
  const __half2 r = __hmul2(reinterpret_cast<const __half2&>(v), m);
  return reinterpret_cast<const uint32_t&>(r);
}
// The eight codes of a word as four pairs of f16 numbers.
__device__ __forceinline__ void spread(uint32_t w, uint32_t (&r)[4]) {
  asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}
// Two E4M3 scales as f16.
__device__ __forceinline__ __half2 nv_factors(uint32_t codes) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)codes));
  return reinterpret_cast<const __half2&>(h);
}
// Byte q of four E8M0 scales: 2^(code - 127), 255 is NaN (infinity times zero).
__device__ __forceinline__ float mx_factor(uint32_t codes, int q) {
  const float f = __uint_as_float(q == 3 ? (codes >> 1) & 0x7F800000u : (codes << (23 - 8 * q)) & 0x7F800000u);
  return fmaf(f, 0.0f, fmaxf(f, 0x1p-127f));
}

__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a0)[4], const uint32_t (&a8)[4], int j, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0[j]), "r"(a8[j]), "r"(a0[j + 1]), "r"(a8[j + 1]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a0)[4], const uint32_t (&a8)[4], int j, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0[j]), "r"(a8[j]), "r"(a0[j + 1]), "r"(a8[j + 1]), "r"(b0), "r"(b1), "f"(0.0f));
}
// N bytes into shared memory.
template <int N>
__device__ __forceinline__ void copy_async(uint32_t to, const uint8_t* from) {
  if constexpr (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(N) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <typename T, bool MX>
__global__ void __launch_bounds__(kThreads, 1) fp4_rows_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int2 first[kMostRows];          // the group that begins with row r: its number and length
  __shared__ int3 list[kMostRows];           // groups with rows: number, first row, length
  __shared__ int totals[kWarps], count;
  float* const sums = reinterpret_cast<float*>(smem + kWarps * kStages * kStageBytes);   // [2][warp][8][kPad]
  constexpr int kSums = kWarps * 8 * kPad;
  uint8_t* const xs = reinterpret_cast<uint8_t*>(sums + 2 * kSums);
  float* const xscales = reinterpret_cast<float*>(xs + (size_t)p.T * p.pitch);   // mxfp4: [group of K][row]
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* const stages = smem + warp * (kStages * kStageBytes);

  // ---- groups ----
  int rows_end = p.T, groups = 1;
  if (p.sizes) {
    bool bad = false;
    auto size_of = [&](int e) -> int {
      const long long n = p.size_bytes == 8 ? __ldg(static_cast<const long long*>(p.sizes) + e) : (long long)__ldg(static_cast<const int*>(p.sizes) + e);
      bad |= n < 0 || n > p.T;
      return n < 0 ? 0 : (n > p.T ? p.T : (int)n);
    };
    auto add = [&](int a, int b) { bad |= a + b > p.T; return min(a + b, p.T); };
    if (tid < kMostRows) first[tid] = make_int2(0, 0);
    const int per = (p.E + kThreads - 1) / kThreads, lo = min(p.E, tid * per), hi = min(p.E, lo + per);
    int at = 0;
    for (int e = lo; e < hi; ++e) at = add(at, size_of(e));
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int v = __shfl_up_sync(0xFFFFFFFFu, at, d);
      if (lane >= d) at = add(at, v);
    }
    if (lane == 31) totals[warp] = at;
    at = __shfl_up_sync(0xFFFFFFFFu, at, 1);
    if (lane == 0) at = 0;
    __syncthreads();
    int before = 0;
    rows_end = 0;
    for (int w = 0; w < kWarps; ++w) {
      if (w == warp) before = rows_end;
      rows_end = add(rows_end, totals[w]);
    }
    at = add(at, before);
    for (int e = lo; e < hi; ++e) {
      const int r0 = at;
      at = add(at, size_of(e));
      if (at > r0) first[r0] = make_int2(e, at - r0);
    }
    if (bad && blockIdx.x == 0) atomicMax(p.status, 9u);
    __syncthreads();
    if (warp == 0) {
      const int2 f = lane < kMostRows ? first[lane] : make_int2(0, 0);
      const uint32_t some = __ballot_sync(0xFFFFFFFFu, f.y > 0);
      if (f.y > 0) list[__popc(some & ((1u << lane) - 1u))] = make_int3(f.x, lane, f.y);
      if (lane == 0) count = __popc(some);
    }
    __syncthreads();
    groups = count;
  }

  // ---- who does what: warps of a tile (a power of two), so that the longest way is shortest; a round's end counts as a piece ----
  const int total = groups * p.tiles;
  int split = 0, rounds = 0, best = INT_MAX;
  for (int s = 0; s <= 4; ++s) {
    const int at_once = (int)gridDim.x << (4 - s), r = (total + at_once - 1) / at_once, c = r * (((p.pieces - 1) >> s) + 2);
    if (c < best) { best = c; split = s; rounds = r; }
  }
  const int part = warp & ((1 << split) - 1), stride = 1 << split;

  // ---- the way through the weights, a piece ahead: a lane copies 16 bytes of rows lane / 8 + {0, 4, 8, 12}, and scales ----
  const int from_row = lane >> 3, from_byte = (lane & 7) * 16;
  constexpr int kScaleCopy = MX ? 4 : 8;      // bytes of 128 k
  int ahead_round = 0, ahead = part, ahead_slot = 0;
  const int64_t four_rows = (int64_t)p.K * 2;
  bool there = false;
  const uint8_t *w0 = nullptr, *s0 = nullptr;
  auto tile_of = [&](int round) { return (round * (int)gridDim.x + (int)blockIdx.x) * (kWarps >> split) + (warp >> split); };
  // first row of a tile: the last one of a group begins earlier where 16 do not divide N (some rows are computed twice, alike)
  auto row_of = [&](int tile_in_group) { return min(tile_in_group * 16, p.N - 16); };
  auto begin_tile = [&]() {
    const int tile = tile_of(ahead_round);
    there = ahead_round < rounds && tile < total;
    if (!there) return;
    const int gi = tile / p.tiles;
    const int64_t row = (int64_t)(p.sizes ? list[gi].x : 0) * p.N + row_of(tile - gi * p.tiles);
    w0 = p.wq + (row + from_row) * (p.K / 2) + from_byte + part * (kPieceK / 2);
    s0 = p.scales + (row + (lane >> 1)) * (p.K / (MX ? 32 : 16)) + (lane & 1) * kScaleCopy + part * (kPieceK / (MX ? 32 : 16));
  };
  auto load = [&]() {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(stages + ahead_slot * kStageBytes) + from_row * kRowBytes + from_byte;
    const uint32_t sto = (uint32_t)__cvta_generic_to_shared(stages + ahead_slot * kStageBytes) + 16 * kRowBytes + lane * kScaleCopy;
    if (there) {
      // the last piece may have one half: the other gets the same codes and scales, which meet zeros of x
      const int half = ahead == p.pieces - 1 ? p.half : 0;
      const uint8_t* at = w0 - ((lane & 4) ? half * 64 : 0);
#pragma unroll
      for (int i = 0; i < 4; ++i, at += four_rows) copy_async<16>(to + 4 * i * kRowBytes, at);
      copy_async<kScaleCopy>(sto, s0 - ((lane & 1) ? half * kScaleCopy : 0));
    }
    copies_done();
    ahead_slot = ahead_slot == kStages - 1 ? 0 : ahead_slot + 1;
    ahead += stride;
    w0 += stride * (kPieceK / 2);
    s0 += stride * (kPieceK / (MX ? 32 : 16));
    if (ahead >= p.pieces) {
      ahead = part;
      ++ahead_round;
      begin_tile();
    }
  };
  begin_tile();
  if (part < p.pieces)
    for (int i = 0; i < kStages - 1; ++i) load();

  // ---- x ----
  int far = 0;   // mxfp4: a group of x that is not zero (or NaN) has a scale outside the range above
  {
    const int units = p.T * (p.pieces * (kPieceK / kUnit));
    const float G = !MX && p.gx ? __ldg(p.gx) : 1.0f;
    for (int u0 = 0; u0 < units; u0 += kThreads) {
      const int u = u0 + tid, row = u / (p.pieces * (kPieceK / kUnit)), k = (u - row * (p.pieces * (kPieceK / kUnit))) * kUnit;
      const bool in = u < units && k < p.K;
      float v[kUnit];
      uint32_t top = 0;
      const T* from = static_cast<const T*>(p.x) + (int64_t)row * p.K + k;
      if (in) top = (reinterpret_cast<uintptr_t>(p.x) & 15) == 0 ? load_unit<T, true>(from, v) : load_unit<T, false>(from, v);
      else
        for (int i = 0; i < kUnit; ++i) v[i] = 0.0f;
      uint32_t codes[2];
      const uint32_t s = quantize_unit<MX>(v, top, G, codes);
      if (u >= units) break;
      uint4* to = reinterpret_cast<uint4*>(xs + (size_t)row * p.pitch + k * 2);
      const __half2 f = nv_factors(s * 0x0101u);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t r[4];
        spread(codes[i], r);
        if (!MX)
#pragma unroll
          for (int j = 0; j < 4; ++j) r[j] = times(r[j], f);
        to[i] = in ? make_uint4(r[0], r[1], r[2], r[3]) : make_uint4(0, 0, 0, 0);
      }
      if (MX && (k & 16) == 0) xscales[(k >> 5) * p.x_stride + row] = in ? e8m0_value(s) * kXScale : 0.0f;
      if (MX) far |= in && (codes[0] | codes[1]) != 0 && (s > kMostX || s < kLeastX);
    }
  }
  // rows of no group
  for (int64_t i = (int64_t)rows_end * p.N + (int64_t)blockIdx.x * kThreads + tid; i < (int64_t)p.T * p.N; i += (int64_t)gridDim.x * kThreads)
    static_cast<T*>(p.y)[i] = Elem<T>::from_float(0.0f);
  const bool wide = __syncthreads_or(far) != 0;

  // ---- products ----
  const float gx = !MX && p.gx ? __ldg(p.gx) : 1.0f;
  int slot = 0;
  for (int round = 0; round < rounds; ++round) {
    const int tile = tile_of(round), gi = tile < total ? tile / p.tiles : 0, row0 = p.sizes ? list[gi].y : 0;
    const int len = tile < total ? (p.sizes ? list[gi].z : p.T) : 0;
    const uint8_t* xrow = xs + (size_t)(row0 + g) * p.pitch + t * 16;
    const float* xscale = xscales + row0 + 2 * t;
    uint4 bs[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};   // columns without a row stay zero
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto pieces = [&](auto form) {
      constexpr bool WIDE = decltype(form)::value;
      for (int piece = part; piece < p.pieces; piece += stride) {
        copies_wait<kStages - 2>();
        __syncwarp();   // everybody's copies are there, and nobody reads the stage before any more
        load();
        const uint8_t* at = stages + slot * kStageBytes;
        slot = slot == kStages - 1 ? 0 : slot + 1;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint8_t* xat = xrow + (piece * 2 + h) * 256;
          uint32_t codes[2];      // mxfp4: four scales per row
          __half2 f[2][4];        // nvfp4: the factor of each word
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const uint8_t* sat = at + 16 * kRowBytes + (g + 8 * r) * (2 * kScaleCopy) + h * kScaleCopy;
            if constexpr (MX) {
              codes[r] = *reinterpret_cast<const uint32_t*>(sat);
            } else {
              const uint2 c = *reinterpret_cast<const uint2*>(sat);
              const __half2 lo = nv_factors(__byte_perm(c.x, 0, t >> 1 ? 0x31 : 0x20)), hi = nv_factors(__byte_perm(c.y, 0, t >> 1 ? 0x31 : 0x20));
              f[r][0] = __low2half2(lo);
              f[r][1] = __high2half2(lo);
              f[r][2] = __low2half2(hi);
              f[r][3] = __high2half2(hi);
            }
          }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t a[2][4];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              spread(*reinterpret_cast<const uint32_t*>(at + (g + 8 * r) * kRowBytes + h * 64 + q * 16 + t * 4), a[r]);
              if constexpr (!MX)
#pragma unroll
                for (int j = 0; j < 4; ++j) a[r][j] = times(a[r][j], f[r][q]);
            }
            uint4& b = bs[q & 1];
            if (g < len) b = *reinterpret_cast<const uint4*>(xat + q * 64);
            if constexpr (MX) {
              float d[4];
              mma_first(d, a[0], a[1], 0, b.x, b.y);
              mma(d, a[0], a[1], 2, b.z, b.w);
              const float* sx = xscale + ((piece * 2 + h) * 4 + q) * p.x_stride;
              const float lo = mx_factor(codes[0], q), hi = mx_factor(codes[1], q), x0 = sx[0], x1 = sx[1];
              if constexpr (WIDE) {
                const float f0 = x0 / kXScale, f1 = x1 / kXScale;
              const float s0 = f0 < 1.0f ? f0 : 1.0f, s1 = f1 < 1.0f ? f1 : 1.0f, b0 = f0 < 1.0f ? 1.0f : f0, b1 = f1 < 1.0f ? 1.0f : f1;
                acc[0] = fmaf(d[0] * s0 * lo, b0, acc[0]);
                acc[1] = fmaf(d[1] * s1 * lo, b1, acc[1]);
                acc[2] = fmaf(d[2] * s0 * hi, b0, acc[2]);
                acc[3] = fmaf(d[3] * s1 * hi, b1, acc[3]);
              } else {
                acc[0] = fmaf(d[0], lo * x0, acc[0]);
                acc[1] = fmaf(d[1], lo * x1, acc[1]);
                acc[2] = fmaf(d[2], hi * x0, acc[2]);
                acc[3] = fmaf(d[3], hi * x1, acc[3]);
              }
            } else {
              mma(acc, a[0], a[1], 0, b.x, b.y);
              mma(acc, a[0], a[1], 2, b.z, b.w);
            }
          }
        }
      }
    };
    if (MX && wide) pieces(std::true_type{});
    else pieces(std::false_type{});
    float* mine = sums + (round & 1) * kSums;
    {
      float* to = mine + (warp * 8 + 2 * t) * kPad + g;
      to[0] = acc[0];
      to[kPad] = acc[1];
      to[8] = acc[2];
      to[kPad + 8] = acc[3];
    }
    __syncthreads();   // (the next round writes the other half of `sums`)
    for (int i = tid; i < (kWarps >> split) * 128; i += kThreads) {
      const int sl = i / 128, token = i / 16 % 8, lane_n = i & 15;
      const int tl = (round * (int)gridDim.x + (int)blockIdx.x) * (kWarps >> split) + sl;
      if (tl >= total) break;
      const int gj = tl / p.tiles, n = row_of(tl - gj * p.tiles) + lane_n;
      const int3 grp = p.sizes ? list[gj] : make_int3(0, 0, p.T);
      if (token >= grp.z) continue;
      float v = 0.0f;
      for (int w = 0; w < stride; ++w) v += mine[(((sl << split) + w) * 8 + token) * kPad + lane_n];
      if constexpr (MX) {
        v *= wide ? 1.0f : 1.0f / kXScale;
      } else {
        v = times_scales(v, gx, p.gw ? __ldg(p.gw + (p.gw_each ? grp.x : 0)) : 1.0f);
      }
      static_cast<T*>(p.y)[(int64_t)(grp.y + token) * p.N + n] = Elem<T>::from_float(v);
    }
  }
  copies_wait<0>();
}

int sm_count() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    cached[dev] = n;
  }
  return cached[dev];
}
int row_pitch(int64_t K) { return (int)((K + kPieceK - 1) / kPieceK * kPieceK * 2 + 64); }   // eight lanes of two rows on 32 banks
// Floats from group to group of x's scales: all rows, and what the lanes of columns without one read.
int scale_stride(int64_t T) { return (int)T + 8; }
size_t smem_bytes(int64_t T, int64_t K, int mode) {
  const size_t xscales = mode == B200Q_MXFP4 ? (size_t)(K + kPieceK - 1) / kPieceK * (kPieceK / 32) * scale_stride(T) * 4 : 0;
  return (size_t)kWarps * kStages * kStageBytes + 2 * (size_t)kWarps * 8 * kPad * 4 + (size_t)T * row_pitch(K) + xscales;
}

}  // namespace

// Where this kernel is the faster one.  In us it takes about 5 + 0.15 per million weights that have rows + 0.1 per thousand values of x
// (which every block quantizes); the tensor-core kernel behind the one that prepares its operands takes 11 at least and rises more
// slowly, by 0.11 per million, but reorders every group's scales first.  nvfp4, here and there:
//   dense, 1 and 8 rows   [4096, 4096] 6.8, 9.2 and 11.8, 12.1; [14336, 4096] 13.7, 16.7 and 15.7, 14.4; [28672, 8192] 36 and 37
//   (mxfp4, 1 and 4 rows  [14336, 4096] 14.2, 14.9 and 14.3, 13.5; [4096, 14336] 13.7, 15.2 and 15.1, 15.4)
//   grouped, 2 and 8 rows of 8 [14336, 4096] 22, 50 and 22.5, 44.5; of 256 [2048, 4096] 7.8, 18 and 24.5, 27
bool fp4_rows_supported(const Fp4Rows& a) {
  const bool mx = a.mode == B200Q_MXFP4;
  if (a.T > kMostRows || a.N < 16 || a.K % 128 != 0 || (reinterpret_cast<uintptr_t>(a.scales) & (mx ? 3 : 7)) != 0 || a.K > 1 << 20) return false;
  const int64_t groups = a.sizes && a.E < a.T ? a.E : (a.sizes ? a.T : 1);
  if (0.15e-6 * (double)groups * (double)a.N * (double)a.K + 0.1e-3 * (double)a.T * (double)a.K > (a.sizes ? 14.0 : 10.3)) return false;
  return smem_bytes(a.T, a.K, a.mode) <= kSmemMax;
}

int fp4_rows(const Fp4Rows& a, cudaStream_t st) {
  RowsParams p{};
  p.x = a.x; p.wq = reinterpret_cast<const uint8_t*>(a.wq); p.scales = a.scales; p.sizes = a.sizes; p.size_bytes = a.size_bytes;
  p.y = a.y; p.gx = a.gx; p.gw = a.gw; p.gw_each = a.gw_each; p.status = a.status;
  p.T = (int)a.T; p.E = (int)a.E; p.N = (int)a.N; p.K = (int)a.K;
  p.tiles = (p.N + 15) / 16;
  p.pieces = (p.K + kPieceK - 1) / kPieceK;
  p.half = p.K % kPieceK != 0;
  p.pitch = row_pitch(a.K);
  p.x_stride = scale_stride(a.T);
  const size_t smem = smem_bytes(a.T, a.K, a.mode);
  const int64_t most = (int64_t)p.tiles * (a.sizes ? (a.E < a.T ? a.E : a.T) : 1);
  const unsigned grid = (unsigned)(most < sm_count() ? most : sm_count());
  auto go = [&](auto kernel) -> int {
    B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
    kernel<<<grid, kThreads, smem, st>>>(p);
    B200Q_LAUNCH_OK("fp4_rows_kernel");
    return B200Q_OK;
  };
  auto typed = [&](auto t) -> int {
    using T = decltype(t);
    return a.mode == B200Q_MXFP4 ? go(fp4_rows_kernel<T, true>) : go(fp4_rows_kernel<T, false>);
  };
  switch (a.dtype) {
    case B200Q_F32: return typed(float{});
    case B200Q_F16: return typed(__half{});
    default: return typed(__nv_bfloat16{});
  }
}

}  // namespace b200q
