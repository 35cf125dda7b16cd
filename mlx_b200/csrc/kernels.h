// Internal interface between the C-ABI dispatch layer (api.cu) and the kernel files.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <mutex>

#include "../../include/b200q.h"

namespace b200q {

// Held while a call launches kernels that pass something on through its workspace.  Stream order keeps one thread's calls apart;
// another thread's launches on the same stream could come between this call's.  (Locks of a small set, by address: 20 ns.)
class ScratchLock {
 public:
  explicit ScratchLock(const void* ws);

 private:
  std::lock_guard<std::mutex> held_;
};

// Output replicated into the buffers of several GPUs (N-sharded linear with the all_gather
// fused into the epilogue): element (m, n) of the local [M, N] result goes to
// y[q][m * ld + col0 + n] for every q < n.  n == 0 means the plain output QmmArgs::y.
constexpr int kMaxPeers = 8;
// Completion signal fused into a kernel whose output goes to peer buffers: when the last thread
// block of the grid has finished (and fenced, at system scope) its peer stores, it adds n to the
// local epoch and 1 to the arrival flag of every rank - what b200q_peer_signal does as a launch of
// its own.  `counter` is a device word of this rank that starts at zero and is left at zero.
struct PeerSignal {
  uint32_t* flags[kMaxPeers];
  uint32_t* epoch;
  uint32_t* counter;
  int n;   // 0: no signal
  // Consumer-side wait: when set, the kernel does not read x or store y before this rank's flag
  // has reached the epoch as the previous kernel of the stream left it, i.e. before every rank
  // has finished the previous exchange step (bounded by wait_limit SM cycles, then status 6).
  const uint32_t* wait_flag;
  long long wait_limit;
  // 1: x is the gathered output of the previous step, so x is not read before the flag either;
  // 0: x comes from elsewhere and only the stores wait (they reuse a buffer the previous step's
  // consumers on other ranks may still be reading).
  int wait_x;
};
struct PeerOut {
  void* y[kMaxPeers];
  int n;
  int64_t ld, col0;
  PeerSignal sig;
};

#ifdef __CUDACC__
// Called by one lane of every warp that is about to touch what the previous exchange step's
// consumers may still be using.  Returns false when the bound ran out (status word set).
__device__ __forceinline__ bool peer_wait_previous(const PeerSignal& ps, uint32_t* status) {
  if (ps.wait_flag == nullptr) return true;
  const uint32_t expected = *reinterpret_cast<const volatile uint32_t*>(ps.epoch);
  const long long t0 = clock64();
  for (;;) {
    uint32_t v;
    asm volatile("ld.acquire.sys.global.u32 %0, [%1];" : "=r"(v) : "l"(ps.wait_flag) : "memory");
    if ((int32_t)(v - expected) >= 0) return true;
    if (clock64() - t0 > ps.wait_limit) {
      if (status) { atomicMax(&status[0], 6u); status[1] = v; }
      return false;
    }
    __nanosleep(100);
  }
}
// Called by ONE thread of every thread block after all peer stores of the block have been issued
// and ordered before this thread (a block- or warp-wide barrier).
__device__ __forceinline__ void peer_signal_tail(const PeerSignal& ps) {
  if (ps.n == 0) return;
  __threadfence_system();
  const unsigned old = atomicAdd(ps.counter, 1u);
  if (old == gridDim.x * gridDim.y * gridDim.z - 1) {
    *ps.counter = 0;
    __threadfence_system();
    *ps.epoch += (uint32_t)ps.n;   // what the local flag must reach before this step's output is complete
    for (int q = 0; q < ps.n; ++q) atomicAdd_system(ps.flags[q], 1u);
  }
}
#endif

struct QmmArgs {
  const void* x;
  const uint32_t* wq;
  const void* scales;
  const void* biases;
  void* y;
  int dtype;
  int64_t batch;  // independent problems (grid z); 1 when W is shared and x is flattened
  int64_t M, N, K;
  int group, bits;
  bool transpose;
  bool w_batched;  // wq/scales/biases hold `batch` matrices
  void* ws;
  size_t ws_bytes;
  PeerOut peers;
};

// Grouped (mixture-of-experts) problem for the tensor-core kernel: activation rows sorted by
// expert; the tile table lives on the device and is produced by the sort kernel of gather.cu.
struct GroupedArgs {
  const void* x_sorted;     // [n_rows, K] bf16, rows in expert order
  const uint32_t* wq;       // [E, N, K*bits/32] packed
  const void* scales;       // [E, N, K/g]
  const void* biases;
  void* y;                  // [n_rows, N]; activation row p is written to row dst_row[p]
  const void* mtiles;       // device: MTile[max_mtiles]
  const int* n_mtiles;      // device scalar
  const int* dst_row;       // device: [n_rows]
  int64_t n_rows, max_mtiles, E, N, K;
  int group, bits, nt;
  uint32_t* status;
  PeerOut peers;            // n > 0: every result row is stored into all of these [n_rows, N] buffers
};

// The row-owning decode kernel over the experts that have rows, for tiles of up to 8 expert-sorted rows (rows_tile: 4 where
// groups of 32 take columns of their own).  With a second matrix the result is silu(x W0^T) * (x W1^T).
int rows_tile(int bits, int group);
// 3, 5 and 6 bits (fields straddle words), and 2 bits in groups of 32 (half a 16-byte unit): that kernel's "runs" form.
constexpr bool runs_form(int bits, int group) { return bits == 3 || bits == 5 || bits == 6 || (bits == 2 && group == 32); }
struct RowsGroup {
  const void* x;            // bf16 rows of K
  const uint32_t* wq[2];    // [E, N, K*bits/32]; the second may be null
  const void* scales[2];
  const void* biases[2];
  void* y;                  // rows of N
  const void* tiles;        // device: (expert, first row, rows, -)[max_tiles]
  const int* n_tiles;       // device scalar
  const int* src_slot;      // device: pair -> the x it multiplies, or null: x is in sorted order
  const int* dst_slot;      // device: pair -> the y it writes, or null: y is in sorted order
  int64_t max_tiles, per_slot, E, N, K;
  int group, bits;
  uint32_t* status;
};
bool qmv_rows_grouped_supported(const RowsGroup& a);
int qmv_rows_grouped(const RowsGroup& a, cudaStream_t st);

// Per-problem operand selection of the gather form: problem i of `batch` multiplies
// x[lhs[i]] with w[rhs[i]].  Indices are range-checked on the device against
// x_batch / n_mats; a bad index zeroes its output and sets status[0].
struct GatherIdx {
  const uint32_t* lhs;
  const uint32_t* rhs;
  uint32_t x_batch, n_mats;
  uint32_t* status;
};

// qmm_generic.cu
int qmm_generic(const QmmArgs& a, cudaStream_t st, const GatherIdx* gi = nullptr);

// qmv_mma.cu : decode path, M <= 16 rows of x against W^T (transpose only, bf16)
bool qmv_mma_supported(const QmmArgs& a);
size_t qmv_mma_workspace_bytes(const QmmArgs& a);
int qmv_mma(const QmmArgs& a, cudaStream_t st);

// qmv_rows.cu : decode path, bf16 and f16, every CTA owns whole weight rows (bulk-copy ring, no scratch)
bool qmv_rows_supported(const QmmArgs& a);
int qmv_rows(const QmmArgs& a, cudaStream_t st);
// Promise that weights are not written by the stream operation preceding a matmul (see qmv_rows.cu).
bool weights_constant();
void set_weights_constant(int on);

// qvm.cu : non-transposed decode (M <= 4, bits 2/4/8): y = x * dequant(W[K, N])
bool qvm_supported(const QmmArgs& a);
size_t qvm_workspace_bytes(const QmmArgs& a);
int qvm(const QmmArgs& a, cudaStream_t st);

// qmm_tcgen05.cu : products with many rows (TMA + tcgen05 + TMEM)
bool qmm_tc_supported(const QmmArgs& a);
size_t qmm_tc_workspace_bytes(const QmmArgs& a);
int qmm_tc(const QmmArgs& a, cudaStream_t st);
int qmm_tc_grouped(const GroupedArgs& a, cudaStream_t st);

// grouped_tc.cu : products over groups of rows with ragged sizes (forms: see there).  Bases and pitches of a and b are
// multiples of 16 bytes; T, I, K >= 1 (Sum: T, I, J >= 1).
enum class GroupedForm { KK, MK, Sum, Mx, Nv };
struct GroupedTcArgs {
  GroupedForm form;
  const void* a;            // [E, I, K], MK: [E, K, I], Sum: [T, I]; rows a_pitch bytes apart
  const void* b;            // [T, K], Sum: [T, J]
  int64_t a_pitch, b_pitch;
  const void* sizes;        // device, [E] of size_bytes each; null: one group of T rows
  int size_bytes;
  void* out;                // [T, I], Sum: [E, J, I]
  int dtype;                // of out (and of 16-bit operands)
  int64_t T, E, I, J, K;    // T, J at most 2^30 - 256; I, K 2^31 - 256
  const uint32_t *sfa, *sfb;        // 4 bits: scales as fp4_prepare leaves them
  int64_t sf_words;                 // of four, per row
  const float *ga, *gb;             // global scales (null: 1); ga_each: one per group
  int ga_each;
  void* ws;                 // grouped_tc_bytes, zeroed once
  uint32_t* status;
};
size_t grouped_tc_bytes(int64_t rows, bool sum);
int grouped_tc(const GroupedTcArgs& a, cudaStream_t st);

// fp4.cu : microscaled 4-bit floating point
constexpr int fp4_group(int mode) { return mode == B200Q_MXFP4 ? 32 : 16; }
int fp4_quantize(const void* w, int dtype, int64_t rows, int64_t K, int mode, const float* global, int64_t rows_per_global,
                 uint32_t* wq, uint8_t* scales, cudaStream_t st);
int fp4_dequantize(const uint32_t* wq, const uint8_t* scales, int mode, const float* global, int64_t rows_per_global, int dtype,
                   int64_t rows, int64_t K, void* out, cudaStream_t st);
// Operands of a 4-bit product in the order that grouped_tc takes, in one launch (the one that its launch has to follow):
//   codes  x quantized, rows code_pitch bytes apart
//   sfx    its scales, words of four consecutive ones, [words][T]
//   sfw    the weights' scales [E * N, K / group] by blocks of 128 rows, [E][blocks][words][32][4]: word (r % 32, r / 32) of a
//          block and word index is row r's.  Groups without rows are left out.
// words: fp4_words(K, mode), zeros after the last.
constexpr int64_t fp4_words(int64_t K, int mode) { return (K / fp4_group(mode) + 31) / 32 * 8; }
struct Fp4Prepare {
  const void* x;
  int dtype, mode;
  int64_t T, E, N, K;
  const float* global;      // x's
  const uint8_t* scales;
  const void* sizes;
  int size_bytes;
  uint8_t* codes;
  int64_t code_pitch;
  uint32_t *sfx, *sfw;
};
int fp4_prepare(const Fp4Prepare& a, cudaStream_t st);
// fp4_rows.cu : 4-bit products of up to 8 rows in one launch; operands as b200q_grouped_qqmm has them
struct Fp4Rows {
  const void* x;
  const uint32_t* wq;
  const uint8_t* scales;
  const void* sizes;        // null: one group
  int size_bytes;
  void* y;
  int dtype, mode;
  int64_t T, E, N, K;
  const float *gx, *gw;
  int gw_each;
  uint32_t* status;
};
bool fp4_rows_supported(const Fp4Rows& a);
int fp4_rows(const Fp4Rows& a, cudaStream_t st);
// Rows per entry of the tile table that b200q_group_rows writes (group or -1, first position, rows, number of rows with a group).
constexpr int kAdapterRows = 64;
// dst rows of dst_pitch bytes (a multiple of 16) from src rows of src_bytes, padded with zeros.
int repack_rows(const void* src, int64_t src_bytes, void* dst, int64_t dst_pitch, int64_t rows, cudaStream_t st);

}  // namespace b200q
