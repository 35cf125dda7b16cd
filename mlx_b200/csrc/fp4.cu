// Microscaled 4-bit floating point: quantisation and back.
//
// E2M1, the 4-bit type: sign, two exponent bits, one mantissa bit; magnitudes 0, .5, 1, 1.5, 2, 3, 4, 6.  Eight to a 32-bit
// word, first value in the lowest bits; one 8-bit scale per group:
//   mxfp4, 32 values: 2^e, e = floor(log2(amax)) - 2 (at least -127), stored as e + 127: the largest value comes to lie in
//          [4, 8) and what is beyond 6 becomes 6; scaling is exact
//   nvfp4, 16 values: E4M3 s = amax / (6 G) to the nearest even, at most 448; a value is divided by s G.  G is one fp32
//          number per tensor (or per matrix of a stack): without it, weights of 0.02 would have scales of two or three bits
// Codes are the nearest, ties to the even one.  Every operation is fp32, rounded once, so that any fp32 program that follows
// the formulas gets the same codes.  A group with a NaN or an infinity has the scale's NaN (0xFF, 0x7F) and codes 0.
//
// One pass, a thread per 16 values.  Bound by HBM (mxfp4 6.4 to 6.9 TB/s, back 6.1) but for nvfp4 of 16-bit values, where the
// quotients' five operations make it instructions: 4.4 to 4.7 TB/s (two groups per thread: 3.9).
#include "fp4.cuh"

namespace b200q {
namespace {

using namespace fp4;

constexpr int kQuantThreads = 256;

template <typename T, bool MX, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads)
fp4_quantize_kernel(const T* __restrict__ w, int64_t units, const float* __restrict__ global, int64_t units_per_global,
                    uint2* __restrict__ wq, uint8_t* __restrict__ scales) {
  const int64_t u = (int64_t)blockIdx.x * kQuantThreads + threadIdx.x;
  const bool in = u < units;
  float v[kUnit];
  uint32_t top = 0;
  if (in) top = load_unit<T, ALIGNED>(w + u * kUnit, v);
  else
    for (int i = 0; i < kUnit; ++i) v[i] = 0.0f;
  const float G = !MX && global && in ? __ldg(global + (units_per_global < units ? u / units_per_global : 0)) : 1.0f;
  uint32_t codes[2];
  const uint32_t s = quantize_unit<MX>(v, top, G, codes);
  if (!in) return;
  wq[u] = make_uint2(codes[0], codes[1]);
  if (!MX) scales[u] = (uint8_t)s;
  else if ((u & 1) == 0) scales[u >> 1] = (uint8_t)s;
}

// 4 bytes at any address, of which `left` >= 1 are there (and the rest are zeros): from the one or two words that hold them.
__device__ __forceinline__ uint32_t load4_any(const uint8_t* at, int64_t left) {
  const uint32_t sh = (uint32_t)(reinterpret_cast<uintptr_t>(at) & 3);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(at - sh);
  const uint32_t n = left < 4 ? (uint32_t)left : 4u;
  const uint32_t lo = __ldg(w), hi = sh + n > 4 ? __ldg(w + 1) : 0u;
  const uint32_t v = __funnelshift_r(lo, hi, 8 * sh);
  return n == 4 ? v : v & (0xFFFFFFFFu >> (32 - 8 * n));
}

// Operands of a 4-bit product.  The first blocks bring the weights' scales into the order that tensor memory wants: a block
// has 128 rows and up to 32 words of them.  (Inside the product, warps that read the scales as they lie took 1.3 to 1.6 times as
// long as its MMAs; few rows of many experts would be 5 % faster that way.)  The others quantize x: up to kQuantThreads units
// of one or two rows; four scales become a word.
struct PrepareParams {
  const uint8_t* scales;
  const void* sizes;
  uint32_t* sfw;
  uint8_t* codes;
  uint32_t* sfx;
  const float* global;
  int64_t sf_row, code_pitch, K, T;
  int N, size_bytes, words, word_blocks, row_blocks, blocks_per_row;
  int aligned;               // rows of scales on 16-byte boundaries
  int64_t scale_blocks;
};
constexpr int kPrepareWords = 32;

template <typename T, bool MX, bool ALIGNED, int ROWS>
__global__ void __launch_bounds__(kQuantThreads)
fp4_prepare_kernel(const T* __restrict__ x, const __grid_constant__ PrepareParams p) {
  asm volatile("griddepcontrol.launch_dependents;");   // the product may set itself up; it waits for this grid before it reads
  const int t = threadIdx.x;
  if (blockIdx.x < p.scale_blocks) {
    const int wb = (int)(blockIdx.x % p.word_blocks), rb = (int)(blockIdx.x / p.word_blocks), e = rb / p.row_blocks, n0 = (rb - e * p.row_blocks) * 128;
    if (p.sizes) {
      const long long n = p.size_bytes == 8 ? __ldg(static_cast<const long long*>(p.sizes) + e) : (long long)__ldg(static_cast<const int*>(p.sizes) + e);
      if (n <= 0) return;
    }
    // a thread: rows lane, lane + 32, lane + 64, lane + 96 of four words, which are the four 16-byte pieces that it writes
    const int lane = t & 31, w0 = wb * kPrepareWords + (t >> 5) * 4;
    const int64_t left = p.sf_row - (int64_t)w0 * 4;
    uint4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + 32 * j + lane;
      v[j] = make_uint4(0, 0, 0, 0);
      if (n < p.N && left > 0) {
        const uint8_t* from = p.scales + ((int64_t)e * p.N + n) * p.sf_row + (int64_t)w0 * 4;
        if (p.aligned) {
          v[j] = __ldg(reinterpret_cast<const uint4*>(from));
        } else {
          v[j].x = load4_any(from, left);
          if (left > 4) v[j].y = load4_any(from + 4, left - 4);
          if (left > 8) v[j].z = load4_any(from + 8, left - 8);
          if (left > 12) v[j].w = load4_any(from + 12, left - 12);
        }
      }
    }
    uint4* out = reinterpret_cast<uint4*>(p.sfw) + ((int64_t)rb * p.words + w0) * 32 + lane;
    if (w0 < p.words) {   // (a multiple of 8)
      out[0] = make_uint4(v[0].x, v[1].x, v[2].x, v[3].x);
      out[32] = make_uint4(v[0].y, v[1].y, v[2].y, v[3].y);
      out[64] = make_uint4(v[0].z, v[1].z, v[2].z, v[3].z);
      out[96] = make_uint4(v[0].w, v[1].w, v[2].w, v[3].w);
    }
    return;
  }
  const int64_t b = blockIdx.x - p.scale_blocks, row0 = b / p.blocks_per_row * ROWS;
  const int64_t u = (b % p.blocks_per_row) * kQuantThreads + t, k = u * kUnit;
  const bool in = k < p.K;
  float v[ROWS][kUnit];
  uint32_t top[ROWS];
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    top[j] = 0;
    if (in && row0 + j < p.T) top[j] = load_unit<T, ALIGNED>(x + (row0 + j) * p.K + k, v[j]);
    else
      for (int i = 0; i < kUnit; ++i) v[j][i] = 0.0f;
  }
  const float G = !MX && p.global ? __ldg(p.global) : 1.0f;
#pragma unroll
  for (int j = 0; j < ROWS; ++j) {
    const int64_t row = row0 + j;
    uint32_t codes[2];
    uint32_t s = quantize_unit<MX>(v[j], top[j], G, codes);
    if (row >= p.T) return;   // (of the whole block)
    if (in) *reinterpret_cast<uint2*>(p.codes + row * p.code_pitch + k / 2) = make_uint2(codes[0], codes[1]);
    else s = 0;
    constexpr int kShare = MX ? 8 : 4;   // lanes that share a word
    s |= __shfl_down_sync(0xFFFFFFFFu, s, kShare / 4) << 8;
    s |= __shfl_down_sync(0xFFFFFFFFu, s, kShare / 2) << 16;
    if (t % kShare == 0 && u / kShare < p.words) p.sfx[(u / kShare) * p.T + row] = s;
  }
}

// A thread takes kAhead pieces of 16 bytes of values, kQuantThreads apart, whose codes and scales are all on their way before the
// first is used: whole lines per warp in every access.  (A thread per 16 values: 28672 x 8192 bf16 in 122 us, now 92; fp32 values
// in pairs of stores 32 bytes apart: 4.4 TB/s.)
constexpr int kAhead = 4;
template <typename T, bool MX, bool ALIGNED>
__global__ void __launch_bounds__(kQuantThreads)
fp4_dequantize_kernel(const uint32_t* __restrict__ wq, const uint8_t* __restrict__ scales, int64_t pieces,
                      const float* __restrict__ global, int64_t pieces_per_global, T* __restrict__ out) {
  constexpr int kValues = 16 / sizeof(T), kPerGroup = (MX ? 32 : 16) / kValues;
  using Code = typename std::conditional<kValues == 8, uint32_t, uint16_t>::type;
  const int64_t p0 = (int64_t)blockIdx.x * (kQuantThreads * kAhead) + threadIdx.x;
  uint32_t c[kAhead], code[kAhead];
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t p = p0 + j * kQuantThreads;
    c[j] = p < pieces ? __ldg(reinterpret_cast<const Code*>(wq) + p) : 0u;
    code[j] = p < pieces ? __ldg(scales + p / kPerGroup) : 0u;
  }
#pragma unroll
  for (int j = 0; j < kAhead; ++j) {
    const int64_t p = p0 + j * kQuantThreads;
    if (p >= pieces) return;
    const float s = MX ? e8m0_value(code[j]) : e4m3_value(code[j]);
    const float G = !MX && global ? __ldg(global + (pieces_per_global < pieces ? p / pieces_per_global : 0)) : 1.0f;
    alignas(16) T r[kValues];
#pragma unroll
    for (int i = 0; i < kValues / 2; ++i) {
      const float2 q = e2m1x2_value(c[j] >> (8 * i));
      r[2 * i] = Elem<T>::from_float(q.x * s * G);
      r[2 * i + 1] = Elem<T>::from_float(q.y * s * G);
    }
    T* at = out + p * kValues;
    if constexpr (ALIGNED) {
      *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(r);
    } else {
#pragma unroll
      for (int i = 0; i < kValues; ++i) at[i] = r[i];
    }
  }
}

// A thread makes kPacked times 16 bytes of destination rows, each from the aligned words that hold them.  Index: 32 bits where they
// are enough (with a 64-bit division per 16 bytes the divisions took longer than the copy).
constexpr int kPacked = 4;
template <typename Index>
__global__ void __launch_bounds__(256) repack_rows_kernel(const uint8_t* __restrict__ src, int64_t src_bytes, uint8_t* __restrict__ dst,
                                                          int64_t dst_pitch, Index pieces_per_row, Index pieces) {
  const Index u0 = (Index)blockIdx.x * (256 * kPacked) + threadIdx.x;
  uint32_t v[kPacked][5];
  int sh[kPacked];
  int64_t left[kPacked], to[kPacked];
#pragma unroll
  for (int j = 0; j < kPacked; ++j) {
    const Index u = u0 + j * 256;
    if (u >= pieces) break;
    const Index row = u / pieces_per_row;
    const int64_t at = (int64_t)(u - row * pieces_per_row) * 16;
    const uint8_t* from = src + (int64_t)row * src_bytes + at;
    left[j] = src_bytes - at;   // bytes of the row from here on
    to[j] = (int64_t)row * dst_pitch + at;
    sh[j] = (int)(reinterpret_cast<uintptr_t>(from) & 3);
    const uint32_t* w = reinterpret_cast<const uint32_t*>(from - sh[j]);
#pragma unroll
    for (int i = 0; i < 5; ++i) v[j][i] = 4 * i - sh[j] < left[j] && 4 * i - sh[j] < 16 ? __ldg(w + i) : 0u;   // words that hold a byte of the piece
  }
#pragma unroll
  for (int j = 0; j < kPacked; ++j) {
    if (u0 + j * 256 >= pieces) break;
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = left[j] - 4 * i;
      r[i] = __funnelshift_r(v[j][i], v[j][i + 1], 8 * sh[j]);
      if (n < 4) r[i] = n <= 0 ? 0u : r[i] & (0xFFFFFFFFu >> (32 - 8 * (int)n));
    }
    *reinterpret_cast<uint4*>(dst + to[j]) = make_uint4(r[0], r[1], r[2], r[3]);
  }
}

template <class F>
int with_type(int dtype, F f) {
  switch (dtype) {
    case B200Q_F32: return f(float{});
    case B200Q_F16: return f(__half{});
    default: return f(__nv_bfloat16{});
  }
}
template <class F>
int with_flags(int mode, bool aligned, F f) {
  using Y = std::true_type;
  using N = std::false_type;
  if (mode == B200Q_MXFP4) return aligned ? f(Y{}, Y{}) : f(Y{}, N{});
  return aligned ? f(N{}, Y{}) : f(N{}, N{});
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
constexpr int64_t kMostBlocks = INT32_MAX;

}  // namespace

int fp4_quantize(const void* w, int dtype, int64_t rows, int64_t K, int mode, const float* global, int64_t rows_per_global,
                 uint32_t* wq, uint8_t* scales, cudaStream_t st) {
  const int64_t units = rows * (K / kUnit), blocks = (units + kQuantThreads - 1) / kQuantThreads;
  if (blocks > kMostBlocks) return fail(B200Q_ERR_UNSUPPORTED, "[quantize] No implementation for problem shape: too many values");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_flags(mode, aligned16(w), [&](auto mx, auto al) {
      fp4_quantize_kernel<T, decltype(mx)::value, decltype(al)::value><<<(unsigned)blocks, kQuantThreads, 0, st>>>(
          static_cast<const T*>(w), units, global, rows_per_global * (K / kUnit), reinterpret_cast<uint2*>(wq), scales);
      B200Q_LAUNCH_OK("fp4_quantize_kernel");
      return B200Q_OK;
    });
  });
}

int fp4_dequantize(const uint32_t* wq, const uint8_t* scales, int mode, const float* global, int64_t rows_per_global, int dtype,
                   int64_t rows, int64_t K, void* out, cudaStream_t st) {
  const int values = 16 / (int)dtype_size(dtype);
  const int64_t pieces = rows * (K / values), blocks = (pieces + kQuantThreads * kAhead - 1) / (kQuantThreads * kAhead);
  if (blocks > kMostBlocks) return fail(B200Q_ERR_UNSUPPORTED, "[dequantize] No implementation for problem shape: too many values");
  return with_type(dtype, [&](auto t) {
    using T = decltype(t);
    return with_flags(mode, aligned16(out), [&](auto mx, auto al) {
      fp4_dequantize_kernel<T, decltype(mx)::value, decltype(al)::value><<<(unsigned)blocks, kQuantThreads, 0, st>>>(
          wq, scales, pieces, global, rows_per_global * (K / values), static_cast<T*>(out));
      B200Q_LAUNCH_OK("fp4_dequantize_kernel");
      return B200Q_OK;
    });
  });
}

int fp4_prepare(const Fp4Prepare& a, cudaStream_t st) {
  PrepareParams p{};
  p.scales = a.scales; p.sizes = a.sizes; p.size_bytes = a.size_bytes;
  p.sfw = a.sfw; p.codes = a.codes; p.sfx = a.sfx; p.global = a.global;
  p.sf_row = a.K / fp4_group(a.mode); p.code_pitch = a.code_pitch; p.K = a.K; p.T = a.T;
  p.N = (int)a.N;
  p.words = (int)fp4_words(a.K, a.mode);
  p.word_blocks = (p.words + kPrepareWords - 1) / kPrepareWords;
  p.row_blocks = (p.N + 127) / 128;
  p.scale_blocks = a.E * p.row_blocks * p.word_blocks;
  const int64_t units = (int64_t)p.words * (a.mode == B200Q_MXFP4 ? 8 : 4);
  p.blocks_per_row = (int)((units + kQuantThreads - 1) / kQuantThreads);
  p.aligned = ((reinterpret_cast<uintptr_t>(a.scales) | (uintptr_t)p.sf_row) & 15) == 0;
  const int rows = a.T >= 1024 ? 2 : 1;   // of a block: with two on their way 4096 rows of 4096 take 6.3 us less, few rows end sooner with one
  const int64_t blocks = p.scale_blocks + (a.T + rows - 1) / rows * p.blocks_per_row;
  if (blocks > kMostBlocks) return fail(B200Q_ERR_UNSUPPORTED, "[qqmm] No implementation for problem shape: too many values");
  return with_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    return with_flags(a.mode, aligned16(a.x), [&](auto mx, auto al) {
      if (rows == 2) fp4_prepare_kernel<T, decltype(mx)::value, decltype(al)::value, 2><<<(unsigned)blocks, kQuantThreads, 0, st>>>(static_cast<const T*>(a.x), p);
      else fp4_prepare_kernel<T, decltype(mx)::value, decltype(al)::value, 1><<<(unsigned)blocks, kQuantThreads, 0, st>>>(static_cast<const T*>(a.x), p);
      B200Q_LAUNCH_OK("fp4_prepare_kernel");
      return B200Q_OK;
    });
  });
}

int repack_rows(const void* src, int64_t src_bytes, void* dst, int64_t dst_pitch, int64_t rows, cudaStream_t st) {
  const int64_t per = dst_pitch / 16, pieces = per * rows, blocks = (pieces + 256 * kPacked - 1) / (256 * kPacked);
  if (blocks > kMostBlocks) return fail(B200Q_ERR_UNSUPPORTED, "[grouped product] No implementation for problem shape: too many values");
  const uint8_t* from = static_cast<const uint8_t*>(src);
  uint8_t* to = static_cast<uint8_t*>(dst);
  if (pieces < (int64_t)UINT32_MAX - 256 * kPacked)
    repack_rows_kernel<uint32_t><<<(unsigned)blocks, 256, 0, st>>>(from, src_bytes, to, dst_pitch, (uint32_t)per, (uint32_t)pieces);
  else
    repack_rows_kernel<uint64_t><<<(unsigned)blocks, 256, 0, st>>>(from, src_bytes, to, dst_pitch, (uint64_t)per, (uint64_t)pieces);
  B200Q_LAUNCH_OK("repack_rows_kernel");
  return B200Q_OK;
}

}  // namespace b200q
