// C-ABI entry points of the grouped products and of the microscaled 4-bit modes: argument checks and scratch layout.
#include "common.cuh"
#include "kernels.h"

namespace b200q {
namespace {

constexpr int64_t kMostGroups = 4096;   // the table of groups is in shared memory (16 bytes each)
// Rows of x, and of a matrix in the weights' gradient: the kernel's table holds the number of tiles of 256 of them in 22 bits, and adds two such
// numbers in 31.  Widths: what 256 less one may be added to in 32 bits.
constexpr int64_t kMostRows = (1 << 30) - 256, kMostWidth = INT32_MAX - 255;

size_t up(size_t n) { return (n + 255) / 256 * 256; }
int64_t up16(int64_t n) { return (n + 15) / 16 * 16; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int check_mode(const char* tag, int mode, int64_t K) {
  if (mode != B200Q_MXFP4 && mode != B200Q_NVFP4)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unknown mode %d (0: mxfp4, 1: nvfp4)", tag, mode);
  if (K < 0 || K % fp4_group(mode) != 0)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] K = %lld is not divisible by the group size %d", tag, (long long)K, fp4_group(mode));
  return B200Q_OK;
}
int check_dtype(const char* tag, int dtype, bool f32) {
  if (dtype == B200Q_F16 || dtype == B200Q_BF16 || (f32 && dtype == B200Q_F32)) return B200Q_OK;
  return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", tag, dtype);
}
int check_dims(const char* tag, int64_t T, int64_t E, int64_t N, int64_t K) {
  if (T < 0 || E < 0 || N < 0 || K < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] negative dimension.", tag);
  if (T > kMostRows) return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^30 - 256 rows.", tag);
  if (N > kMostWidth || K > kMostWidth)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: dimension exceeds 2^31 - 256.", tag);
  if (E > kMostGroups)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than %lld groups.", tag, (long long)kMostGroups);
  return B200Q_OK;
}
int check_sizes(const char* tag, const void* sizes, int size_bytes) {
  if (!sizes) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if ((size_bytes != 4 && size_bytes != 8) || reinterpret_cast<uintptr_t>(sizes) % size_bytes != 0)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] sizes are aligned 4- or 8-byte integers", tag);
  return B200Q_OK;
}
// Operands that the copies into shared memory can take, or copies of them in the workspace.
struct Operand {
  const void* at;
  int64_t pitch;
};
size_t packed_bytes(int64_t rows, int64_t row_bytes) { return row_bytes % 16 ? up((size_t)rows * up16(row_bytes)) : 0; }
int pack(const void* src, int64_t rows, int64_t row_bytes, char*& ws, Operand* out, cudaStream_t st) {
  if (row_bytes % 16 == 0) {
    *out = Operand{src, row_bytes};
    return B200Q_OK;
  }
  *out = Operand{ws, up16(row_bytes)};
  char* dst = ws;
  ws += packed_bytes(rows, row_bytes);
  return repack_rows(src, row_bytes, dst, up16(row_bytes), rows, st);
}
int check_ws(const char* tag, const void* ws, size_t have, size_t need) {
  if (!ws || have < need)
    return fail(B200Q_ERR_WORKSPACE, "[%s] workspace of %zu bytes required, %zu given", tag, need, ws ? have : (size_t)0);
  if (!aligned16(ws) || have % 16 != 0)
    return fail(B200Q_ERR_WORKSPACE, "[%s] the workspace and its size must be multiples of 16 bytes", tag);
  return B200Q_OK;
}
uint32_t* status_word(void* ws, size_t bytes) { return reinterpret_cast<uint32_t*>(static_cast<char*>(ws) + bytes - kStatusBytes); }

size_t sfx_bytes(int64_t T, int64_t K, int mode) { return up((size_t)T * fp4_words(K, mode) * 4); }
size_t sfw_bytes(int64_t E, int64_t N, int64_t K, int mode) { return up((size_t)E * ((N + 127) / 128) * fp4_words(K, mode) * 512); }
size_t qqmm_bytes(int64_t T, int64_t E, int64_t N, int64_t K, int mode) {
  return up(grouped_tc_bytes(T, false)) + up((size_t)T * up16(K / 2)) + sfx_bytes(T, K, mode) + sfw_bytes(E, N, K, mode) + packed_bytes(E * N, K / 2) + kStatusBytes;
}
size_t grouped_bytes(int64_t T, int64_t E, int64_t N, int64_t K, bool transpose) {
  return up(grouped_tc_bytes(T, false)) + packed_bytes(T, 2 * K) + (transpose ? packed_bytes(E * N, 2 * K) : packed_bytes(E * K, 2 * N)) + kStatusBytes;
}
size_t dw_bytes(int64_t T, int64_t N, int64_t K) {
  return up(grouped_tc_bytes(T, true)) + packed_bytes(T, 2 * N) + packed_bytes(T, 2 * K) + kStatusBytes;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" int b200q_fp4_quantize(const void* w, int dtype, int64_t rows, int64_t K, int mode, const float* global_scale,
                                  int64_t rows_per_scale, uint32_t* wq, uint8_t* scales, void* stream) {
  if (int rc = check_dtype("quantize", dtype, true)) return rc;
  if (int rc = check_mode("quantize", mode, K)) return rc;
  if (rows < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[quantize] negative dimension.");
  if (global_scale && (mode != B200Q_NVFP4 || rows_per_scale < 1))
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[quantize] a global scale belongs to nvfp4 and to at least one row");
  if (rows == 0 || K == 0) return B200Q_OK;
  if (!w || !wq || !scales) return fail(B200Q_ERR_INVALID_ARGUMENT, "[quantize] null pointer");
  if (reinterpret_cast<uintptr_t>(wq) & 7) return fail(B200Q_ERR_INVALID_ARGUMENT, "[quantize] packed weights must be 8-byte aligned");
  return fp4_quantize(w, dtype, rows, K, mode, global_scale, rows_per_scale, wq, scales, static_cast<cudaStream_t>(stream));
}

extern "C" int b200q_fp4_dequantize(const uint32_t* wq, const uint8_t* scales, int mode, const float* global_scale,
                                    int64_t rows_per_scale, int dtype, int64_t rows, int64_t K, void* out, void* stream) {
  if (int rc = check_dtype("dequantize", dtype, true)) return rc;
  if (int rc = check_mode("dequantize", mode, K)) return rc;
  if (rows < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[dequantize] negative dimension.");
  if (global_scale && (mode != B200Q_NVFP4 || rows_per_scale < 1))
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[dequantize] a global scale belongs to nvfp4 and to at least one row");
  if (rows == 0 || K == 0) return B200Q_OK;
  if (!wq || !scales || !out) return fail(B200Q_ERR_INVALID_ARGUMENT, "[dequantize] null pointer");
  if (reinterpret_cast<uintptr_t>(wq) & 7) return fail(B200Q_ERR_INVALID_ARGUMENT, "[dequantize] packed weights must be 8-byte aligned");
  return fp4_dequantize(wq, scales, mode, global_scale, rows_per_scale, dtype, rows, K, out, static_cast<cudaStream_t>(stream));
}

extern "C" size_t b200q_grouped_qqmm_workspace_bytes(int64_t T, int64_t E, int64_t N, int64_t K, int mode) {
  if (T <= 0 || E <= 0 || N <= 0 || K <= 0 || (mode != B200Q_MXFP4 && mode != B200Q_NVFP4)) return 0;
  return qqmm_bytes(T, E, N, K, mode);
}

extern "C" int b200q_grouped_qqmm(const void* x, const uint32_t* wq, const uint8_t* scales, const void* sizes, int size_bytes,
                                  void* y, int dtype, int64_t T, int64_t E, int64_t N, int64_t K, int mode,
                                  const float* global_scale_x, const float* global_scale_w, int scale_per_group, void* ws,
                                  size_t ws_bytes, void* stream) {
  const char* tag = sizes ? "grouped_qqmm" : "qqmm";
  if (int rc = check_dtype(tag, dtype, true)) return rc;
  if (int rc = check_mode(tag, mode, K)) return rc;
  if (int rc = check_dims(tag, T, E, N, K)) return rc;
  if ((global_scale_x || global_scale_w) && mode != B200Q_NVFP4)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] a global scale belongs to nvfp4", tag);
  if (!sizes && E != 1) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] more than one group needs sizes", tag);
  if (T == 0 || N == 0) return B200Q_OK;
  if (!y) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (E == 0 || K == 0) {
    B200Q_CUDA_OK(cudaMemsetAsync(y, 0, (size_t)T * N * dtype_size(dtype), st));
    return B200Q_OK;
  }
  if (!x || !wq || !scales) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (sizes)
    if (int rc = check_sizes(tag, sizes, size_bytes)) return rc;
  if (!aligned16(wq)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] packed weights must be 16-byte aligned", tag);
  const size_t need = qqmm_bytes(T, E, N, K, mode);
  if (int rc = check_ws(tag, ws, ws_bytes, need)) return rc;
  const Fp4Rows few{x, wq, scales, sizes, size_bytes, y, dtype, mode, T, E, N, K, global_scale_x, global_scale_w, scale_per_group, status_word(ws, ws_bytes)};
  if (fp4_rows_supported(few)) return fp4_rows(few, st);
  const ScratchLock lock(ws);
  char* at = static_cast<char*>(ws) + up(grouped_tc_bytes(T, false));
  uint8_t* codes = reinterpret_cast<uint8_t*>(at);
  at += up((size_t)T * up16(K / 2));
  uint32_t* sfx = reinterpret_cast<uint32_t*>(at);
  at += sfx_bytes(T, K, mode);
  uint32_t* sfw = reinterpret_cast<uint32_t*>(at);
  at += sfw_bytes(E, N, K, mode);
  Operand w;
  if (int rc = pack(wq, E * N, K / 2, at, &w, st)) return rc;
  const Fp4Prepare pr{x, dtype, mode, T, E, N, K, global_scale_x, scales, sizes, size_bytes, codes, up16(K / 2), sfx, sfw};
  if (int rc = fp4_prepare(pr, st)) return rc;
  GroupedTcArgs a{};
  a.form = mode == B200Q_MXFP4 ? GroupedForm::Mx : GroupedForm::Nv;
  a.a = w.at; a.a_pitch = w.pitch;
  a.b = codes; a.b_pitch = up16(K / 2);
  a.sizes = sizes; a.size_bytes = size_bytes;
  a.out = y; a.dtype = dtype;
  a.T = T; a.E = E; a.I = N; a.K = K;
  a.sfa = sfw; a.sfb = sfx; a.sf_words = fp4_words(K, mode);
  a.ga = global_scale_w; a.gb = global_scale_x; a.ga_each = scale_per_group;
  a.ws = ws; a.status = status_word(ws, ws_bytes);
  return grouped_tc(a, st);
}

extern "C" const char* b200q_grouped_qqmm_kernel_name(int64_t T, int64_t E, int64_t N, int64_t K, int mode, int grouped) {
  if (check_mode("qqmm", mode, K) || check_dims("qqmm", T, E, N, K) || (!grouped && E != 1)) return "invalid";
  Fp4Rows few{};
  few.mode = mode;
  few.T = T; few.E = E; few.N = N; few.K = K;
  few.sizes = grouped ? &few : nullptr;   // (whether there are any is all that matters)
  return fp4_rows_supported(few) ? "fp4_rows" : "grouped_tc";
}

extern "C" size_t b200q_grouped_mm_workspace_bytes(int64_t T, int64_t E, int64_t N, int64_t K, int transpose) {
  if (T <= 0 || E <= 0 || N <= 0 || K <= 0) return 0;
  return grouped_bytes(T, E, N, K, transpose != 0);
}

extern "C" int b200q_grouped_mm(const void* x, const void* w, const void* sizes, int size_bytes, void* y, int dtype, int64_t T,
                                int64_t E, int64_t N, int64_t K, int transpose, void* ws, size_t ws_bytes, void* stream) {
  const char* tag = "grouped_mm";
  if (int rc = check_dtype(tag, dtype, false)) return rc;
  if (int rc = check_dims(tag, T, E, N, K)) return rc;
  if (T == 0 || N == 0) return B200Q_OK;
  if (!y) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (E == 0 || K == 0) {
    B200Q_CUDA_OK(cudaMemsetAsync(y, 0, (size_t)T * N * 2, st));
    return B200Q_OK;
  }
  if (!x || !w) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (int rc = check_sizes(tag, sizes, size_bytes)) return rc;
  if (!aligned16(x) || !aligned16(w)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] x and w must be 16-byte aligned", tag);
  const size_t need = grouped_bytes(T, E, N, K, transpose != 0);
  if (int rc = check_ws(tag, ws, ws_bytes, need)) return rc;
  const ScratchLock lock(ws);
  char* at = static_cast<char*>(ws) + up(grouped_tc_bytes(T, false));
  Operand xo, wo;
  if (int rc = pack(x, T, 2 * K, at, &xo, st)) return rc;
  if (int rc = transpose ? pack(w, E * N, 2 * K, at, &wo, st) : pack(w, E * K, 2 * N, at, &wo, st)) return rc;
  GroupedTcArgs a{};
  a.form = transpose ? GroupedForm::KK : GroupedForm::MK;
  a.a = wo.at; a.a_pitch = wo.pitch;
  a.b = xo.at; a.b_pitch = xo.pitch;
  a.sizes = sizes; a.size_bytes = size_bytes;
  a.out = y; a.dtype = dtype;
  a.T = T; a.E = E; a.I = N; a.K = K;
  a.ws = ws; a.status = status_word(ws, ws_bytes);
  return grouped_tc(a, st);
}

extern "C" size_t b200q_grouped_mm_dw_workspace_bytes(int64_t T, int64_t N, int64_t K) {
  if (T <= 0 || N <= 0 || K <= 0) return 0;
  return dw_bytes(T, N, K);
}

extern "C" int b200q_grouped_mm_dw(const void* dy, const void* x, const void* sizes, int size_bytes, void* dw, int dtype, int64_t T,
                                   int64_t E, int64_t N, int64_t K, void* ws, size_t ws_bytes, void* stream) {
  const char* tag = "grouped_mm_dw";
  if (int rc = check_dtype(tag, dtype, false)) return rc;
  if (int rc = check_dims(tag, T, E, N, K)) return rc;
  if (N > kMostRows) return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^30 - 256 rows per matrix.", tag);
  if (E == 0 || N == 0 || K == 0) return B200Q_OK;
  if (!dw) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    B200Q_CUDA_OK(cudaMemsetAsync(dw, 0, (size_t)E * N * K * 2, st));
    return B200Q_OK;
  }
  if (!dy || !x) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (int rc = check_sizes(tag, sizes, size_bytes)) return rc;
  if (!aligned16(dy) || !aligned16(x)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] dy and x must be 16-byte aligned", tag);
  const size_t need = dw_bytes(T, N, K);
  if (int rc = check_ws(tag, ws, ws_bytes, need)) return rc;
  const ScratchLock lock(ws);
  char* at = static_cast<char*>(ws) + up(grouped_tc_bytes(T, true));
  Operand yo, xo;
  if (int rc = pack(dy, T, 2 * N, at, &yo, st)) return rc;
  if (int rc = pack(x, T, 2 * K, at, &xo, st)) return rc;
  GroupedTcArgs a{};
  a.form = GroupedForm::Sum;
  a.a = xo.at; a.a_pitch = xo.pitch;   // [T, K]: k on the accumulator's lanes, contiguous in dw
  a.b = yo.at; a.b_pitch = yo.pitch;
  a.sizes = sizes; a.size_bytes = size_bytes;
  a.out = dw; a.dtype = dtype;
  a.T = T; a.E = E; a.I = K; a.J = N;
  a.ws = ws; a.status = status_word(ws, ws_bytes);
  return grouped_tc(a, st);
}
