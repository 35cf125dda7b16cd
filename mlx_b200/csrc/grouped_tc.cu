// Products over groups of rows with ragged sizes, on the 5th-generation tensor cores.  Rows of group e are consecutive:
//   KK   out[t, i] = sum_k a[e, i, k] b[t, k]      the weights' reduced dimension is contiguous
//   MK   out[t, i] = sum_k a[e, k, i] b[t, k]      the weights' output dimension is contiguous
//   MM   out[e, j, i] = sum_t a[t, i] b[t, j]      gradient of the weights: the sum goes over the group's rows
//   Mx, Nv  as KK, a and b in microscaled 4-bit floating point (fp4.cu), times the operands' global scales
// One group without sizes is the dense product.
//
// D[i, j] has the output's contiguous dimension on the accumulator's lanes (256 over a pair of thread blocks, cta_group::2)
// and up to 256 rows of the output as columns: a tile costs what its rows cost, in steps of 16, so ragged groups and
// single tokens need no other kernel.  Each block of the pair fetches 128 of the i and half of the j: 64 bytes per clock
// and SM at the tensor cores' full rate, where a block of its own would need 94.
//
//   warps 0, 3  TMA: a's and b's tile of a stage (128 bytes of k per row; MM and MK: 64 k).  A copy costs its thread 100 to 200
//               cycles, so that one warp for both was the bound of MM
//   warp 1      tcgen05.mma (leader block, one thread)
//   warp 2      4 bits: tcgen05.cp of the scales, two or three per 4 scales of 256 rows (leader, one thread: with them in warp
//               1 a stage's instructions took it longer than its MMAs take).  MM: the stage that a group ends in has its
//               foreign rows zeroed in shared memory, in both operands (a foreign infinity times zero would be NaN).  Only
//               those stages go through this warp: with all of them handed on by it a step of the ring took 1600 cycles
//               instead of 700
//   warps 4-11  epilogue: the accumulator is rounded and packed in registers, which frees it for another tile, then goes through
//               stmatrix staging to 16-byte stores.  MM, whose tiles have few stages and are stored as fast as they are
//               multiplied: TMA stores of 32 whole lines
//   warps 12-15 4 bits only: b's scales, from words in global memory into the order that tensor memory wants (a's are in that
//               order already, fp4_prepare_kernel, and come by TMA: warp 3)
//
// The table of groups (first row, first tile, first step) is built in shared memory by every block from `sizes`, which the
// host never reads: no launch in front and no synchronisation.  The roles find their tiles in it through one function (walk_next).
//
// Tiles are dealt to the pairs in whole waves.  What is left over is laid end to end and cut into equal ranges of K where
// that gains more than the partial sums cost; the last pair to arrive adds a tile's parts in order (no atomics on values,
// the same bits every time), and nobody waits for another pair.  (All tiles in equal ranges instead of whole waves: 5 to 40 %
// slower, neighbours no longer share operands in L2.)
//
// What bounds it, measured (bf16 unless said): many rows, power and the tensor cores, 84 to 86 % of whose cycles are busy
// (4096 rows of 8 experts [14336, 4096] 363 us, 1320 TFLOP/s; 8192^3 1476); its gradient of the weights the same with 940 MB written
// (407 us); 4 bits, what is not hidden behind a quarter of the MMA time: of 165,000 cycles that the MMA thread of a pair takes for its 12 tiles of
// 4096 rows through nvfp4 [14336, 4096] (113 us in 124 with fp4_prepare_kernel) it waits 23 % for the epilogue, since tiles of more than
// 128 rows leave tensor memory for one accumulator only (3200 cycles a tile; 60 in bf16, which has two), 26 % for scales in tensor memory
// and 9 % for operands (K = 16384: 8, 38 and 11 %; mxfp4: 25, 23 and 10 %).  L2 gives the bf16 form more (11.3 TB/s against 9.2).  From 19 groups on
// their table leaves four stages instead of five and with them two buffers of scales instead of four: a stage takes 1130 cycles instead of 1020
// (256 rows of each through nvfp4 [6144, 4096]).  Few rows, HBM (8 rows of 5 or 6 experts, 0.95 of its rate) or, below some 20 us, latencies:
// 4000 to 5000 cycles until the first copy is issued, 2500 until it lands, 4000 for a cut tile's end.
//
// Every wait on an mbarrier is bounded: when one runs out, the role raises the block's abort flag and the status word, all roles leave,
// tensor memory is freed and the kernel ends.  What else waits ends by itself: the allocation of tensor memory (for other kernels'
// blocks), the pair's barriers (for its own roles) and the wait for the kernel in front.
#include <cuda.h>

#include <type_traits>

#include "bounded_wait.h"
#include "common.cuh"
#include "fp4.cuh"
#include "kernels.h"
#include "tc_ptx.cuh"

namespace b200q {
namespace {

using namespace tc;

enum class Kind { KK, MK, MM, Mx, Nv };
template <Kind K> constexpr bool kFp4 = K == Kind::Mx || K == Kind::Nv;

constexpr int kLanes = 128;          // i per block
constexpr int kTileI = 2 * kLanes;
constexpr int kMaxNT = 256;
constexpr int kStageA = kLanes * 128;
constexpr int kMaxStages = 12;
constexpr int kSfSlots = 8;          // at most, of chunks of scales: 32 bytes per row each
constexpr int kEpiWarp0 = 4, kEpiWarps = 8;
constexpr int kScaleWarp0 = 12, kScaleWarps = 4;
constexpr int kMaxWarps = kScaleWarp0 + kScaleWarps;
template <Kind K> constexpr int kThreads = 32 * (kFp4<K> ? kMaxWarps : kScaleWarp0);
template <Kind K> constexpr int kStageOut = K == Kind::MM ? 4096 : 2048;   // epilogue staging per warp: 32 rows of 64 bytes; MM: twice
constexpr int kSfColumns = 48;       // tensor memory of a stage's scales: 16 (a) + 32 (b) columns
constexpr int kSfBuffers = 4;        // at most
constexpr size_t kSmemMax = 227 * 1024;

// k per stage, and stages per step: the unit in which K is cut (4 bits: what a chunk of scales covers)
template <Kind K> constexpr int kStageK = kFp4<K> ? 256 : 64;
template <Kind K> constexpr int kSpc = K == Kind::Mx ? 4 : (K == Kind::Nv ? 2 : 1);

struct Maps {
  CUtensorMap a;
  CUtensorMap sfa;    // 4 bits: a's scales, rows of 1024 bytes
  CUtensorMap out;    // MM, rows on 16-byte boundaries: the output, boxes of 64 i x 32 j
  CUtensorMap b[5];   // boxes of 128, 64, 32, 16 and 8 rows (MM: the first only, 64 x 64)
};

struct Params {
  const void* sizes;       // null: one group of T rows
  int size_bytes;          // 4 or 8
  int E, T;
  int I, J, K;             // output width; MM: output rows per group; length of the sum (MM: unused)
  int NT, i_tiles, stages;
  int sf_slots;            // 8 up to 128 rows per tile, else 4 (less where the table of groups needs the room)
  int b_bytes;             // of a stage's b tile
  int blocks;              // MK, MM: a (b) comes in whole blocks of 64 columns, two in one copy (bit 0: a, bit 1: b)
  int sfb_chunk;           // 4 bits: bytes of a chunk of b's scales
  void* out;
  int vec;                 // rows of the output start on 16-byte boundaries
  const uint32_t* sfb;     // b's scales: words of four [.., T]
  int sf_words, i_blocks;  // words of a's (and b's) scales per row, a multiple of 8; blocks of 128 i per group
  const float* ga;         // global scales: one, or (ga_each) one per group
  const float* gb;
  int ga_each;
  float* partial;          // [2 * pairs][block of the pair][NT][128]
  uint32_t* counters;      // [pairs][block of the pair]
  int wait_times;          // how many times kWaitMost a wait for a whole tile may last
  uint32_t* status;
};

struct Piece {
  int e, i0;          // group; first i of the pair
  int row0, rows;     // first output row (MM: row of b's columns) and how many are valid
  int neff;           // the same, rounded up to what the MMA takes
  int t0, len;        // first row of the group and their number
  int ks0, ks1;       // stages
  int parts, part, j0;   // of a cut tile: number of parts, this one's number, first part's pair
};

// Rows of b that are fetched for `half` (a multiple of 8) of them: two boxes at most, since a copy costs its thread more than
// 100 cycles and four of them more than a stage's MMAs.
__host__ __device__ __forceinline__ int box_rows(int half, int* first) {
  int a = 8;
  while (2 * a <= half) a *= 2;
  int b = half > a ? 8 : 0;
  while (b && b < half - a) b *= 2;
  *first = b == a ? 2 * a : a;
  return a + b;
}

// A warp's way through its pair's pieces.
struct __align__(16) Walk {
  Piece c;        // where it is
  int u;          // next whole tile
  int pos, end;   // next step of the pair's range, and its end
  int e;          // group
};

struct __align__(16) Bars {
  uint64_t full[kMaxStages], empty[kMaxStages];
  uint64_t landed[kMaxStages], fixed[kMaxStages];  // MM, a group's last stage: this block's tiles are there; and without foreign rows, in both
  uint64_t sf_full[kSfSlots], sf_empty[kSfSlots];  // chunks of scales in shared memory
  uint64_t sf_ready[kSfBuffers];                   // a stage's scales in tensor memory
  uint64_t acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag, last, seen[2];
  Piece piece[2];                                  // the epilogue's, by turns; what `more` says: whether there is one
  int more[2];
  // schedule
  int full_units, cut_pairs, cut_steps;   // tiles in whole waves; pairs and steps of the rest
  int cut_base;                           // step at which the rest begins
  int rows;                               // rows that belong to a group
  Walk walk[kMaxWarps];
};

// Entry e of the table of groups: first row, first tile and first step of group e; number of tiles of its rows and rows per
// tile (nj << 9 | tr).  The last entry is where everything ends.
using Group = int4;

template <Kind KIND>
__device__ __forceinline__ int group_stages(const Params& p, int len) {
  return KIND == Kind::MM ? max(1, (len + kStageK<KIND> - 1) / kStageK<KIND>) : (p.K + kStageK<KIND> - 1) / kStageK<KIND>;
}
template <Kind KIND>
__device__ __forceinline__ int group_steps(const Params& p, int len) {
  return (group_stages<KIND>(p, len) + kSpc<KIND> - 1) / kSpc<KIND>;
}
// Rows per tile of a group, as even as multiples of 16 allow, and the number of tiles.
template <Kind KIND>
__device__ __forceinline__ int2 tiles_j(const Params& p, int len) {
  if (KIND == Kind::MM) return make_int2(p.NT, (p.J + p.NT - 1) / p.NT);
  if (len <= p.NT) return make_int2((len + 15) & ~15, len > 0);
  const int n = (int)((uint32_t)(len + p.NT - 1) / (uint32_t)p.NT), tr = ((int)((uint32_t)(len + n - 1) / (uint32_t)n) + 15) & ~15;
  return make_int2(tr, (int)((uint32_t)(len + tr - 1) / (uint32_t)tr));
}

// Number of pairs that the n tiles (`rest` steps, `rows` rows each on average) left over from whole waves are cut for; 0: not
// cut.  In cycles: a stage of n busy pairs takes its MMAs, its 16 KB of weights at their share of HBM, or at least 300 (4
// bits, whose scales pass more hands: 450); a cut tile costs its writes (36 a row), the last arriver's reads (20 a row and part)
// and 4000 of fences and latencies.
// The lanes of a warp try lane + 1 parts per tile (most: 8).
template <Kind KIND>
__device__ __forceinline__ int cut_for(int lane, int n, int rest, int rows, int pairs) {
  if ((long long)rest * (pairs + 1) >= INT32_MAX) return 0;
  const float r = (float)max(rows, 16), steps = (float)(rest * kSpc<KIND>);   // stages of all of them
  const int s = lane + 1, busy = min(min(n * s, pairs), rest);
  const float stage = fmaxf(fmaxf(2.0f * r, 700.0f * (float)busy / (float)pairs), kFp4<KIND> ? 450.0f : 300.0f);
  float t = __fdividef(steps, (float)busy) * stage;
  if (s > 1) t += r * (36.0f + 20.0f * (__fdividef((float)busy, (float)n) + (n * s > pairs ? 1.0f : 0.0f))) + 4000.0f;
  if (s > 8 || n * (s - 1) >= pairs) t = 3.0e38f;
  // the least time, with the fewest parts
  uint32_t best = (__float_as_uint(t) & ~31u) | (uint32_t)lane;
#pragma unroll
  for (int d = 16; d; d /= 2) best = min(best, __shfl_xor_sync(0xFFFFFFFFu, best, d));
  const int parts = (int)(best & 31u) + 1;
  return parts == 1 ? 0 : min(min(n * parts, pairs), rest);
}

__device__ __forceinline__ void walk_begin(const Bars& b, Walk& w) {
  const uint32_t pair = blockIdx.x >> 1;
  w.u = (int)pair;
  w.pos = w.end = w.e = 0;
  if ((int)pair < b.cut_pairs) {   // (cut_steps * pairs stays below 2^31)
    w.pos = b.cut_base + (int)((uint32_t)b.cut_steps * pair / (uint32_t)b.cut_pairs);
    w.end = b.cut_base + (int)((uint32_t)b.cut_steps * (pair + 1) / (uint32_t)b.cut_pairs);
  }
}
// One thread: the next piece; false: there is none.  Out of line and through shared memory, so that all roles share its
// instructions and none has a stack: with a copy in each role five of them had to come from memory before the first load
// could start, and what is left of L1 beside the rings keeps no stack.
template <Kind KIND>
__device__ __noinline__ bool walk_next(const Params& p, const Bars& b, const Group* tab, Walk& w) {
  const bool whole = w.u < b.full_units;
  if (!whole && w.pos >= w.end) return false;
  const int at = whole ? w.u : w.pos;
  auto begins = [&](int i) { return whole ? tab[i].y : tab[i].z; };
  int e = w.e;   // the last group that begins at or before `at` is not empty; never one before the last piece's
  if (begins(e + 1) <= at) {
    int hi = p.E;
    while (hi - e > 1) {
      const int mid = (e + hi) >> 1;
      if (begins(mid) <= at) e = mid; else hi = mid;
    }
    w.e = e;
  }
  const Group g = tab[e];
  const int len = tab[e + 1].x - g.x, steps = group_steps<KIND>(p, len), nj = g.w >> 9, tr = g.w & 511;
  uint32_t v;
  int k0 = 0, k1 = steps;
  Piece& c = w.c;
  c.parts = 1;
  if (whole) {
    v = (uint32_t)(at - g.y);
    w.u += gridDim.x >> 1;
  } else {
    const uint32_t off = (uint32_t)(at - g.z);
    v = off / (uint32_t)steps;
    k0 = (int)(off - v * (uint32_t)steps);
    const int first = at - k0;
    k1 = min(steps, w.end - first);
    // the pair whose range holds step s (counted from cut_base) is ((s + 1) cut_pairs - 1) / cut_steps
    const uint32_t s0 = (uint32_t)(first - b.cut_base), s1 = s0 + (uint32_t)steps - 1, n = (uint32_t)b.cut_pairs, all = (uint32_t)b.cut_steps;
    c.j0 = (int)(((s0 + 1) * n - 1) / all);
    c.parts = (int)(((s1 + 1) * n - 1) / all) - c.j0 + 1;
    c.part = (int)(blockIdx.x >> 1) - c.j0;
    w.pos = first + k1;
  }
  const uint32_t it = nj == 1 ? v : v / (uint32_t)nj;
  const int jt = (int)(v - it * (uint32_t)nj);
  c.e = e;
  c.i0 = (int)it * kTileI;
  c.t0 = g.x;
  c.len = len;
  if (KIND == Kind::MM) {
    c.row0 = jt * tr;
    c.rows = min(tr, p.J - c.row0);
    c.neff = (c.rows + 127) & ~127;
  } else {
    c.row0 = g.x + jt * tr;
    c.rows = min(tr, g.x + len - c.row0);
    c.neff = (c.rows + 15) & ~15;
  }
  c.ks0 = k0 * kSpc<KIND>;
  c.ks1 = min(group_stages<KIND>(p, len), k1 * kSpc<KIND>);
  return true;
}

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
// Into this block's shared memory, counted on the pair leader's barrier.
__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(leader_bar)
      : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}
__device__ __forceinline__ void tma_4d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(leader_bar)
      : "memory");
}
// Staged rows to global memory (what lies beyond the tensor is left out).
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];\n\tcp.async.bulk.commit_group;"
               ::"l"(map), "r"(src), "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
// n blocks of 64 columns and 64 rows, from column `col` and row `k` of matrix e: one copy where the map has blocks as a
// dimension of their own (and the box both of them).
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap* map, bool blocks, int n, int col, int k, int e, uint32_t bar, bool own) {
  if (blocks) {
    if (own) tma_4d(dst, map, 0, k, col >> 6, e, bar);
    else tma_4d_pair(dst, map, 0, k, col >> 6, e, bar);
  } else {
    for (int h = 0; h < n; ++h) {
      if (own) tma_3d(dst + h * 8192, map, col + 64 * h, k, e, bar);
      else tma_3d_pair(dst + h * 8192, map, col + 64 * h, k, e, bar);
    }
  }
}
// Bounded waits.  try_wait holds the thread back in hardware: a dozen warps that look again and again take issue slots and
// shared-memory cycles from the tensor core's operands.
constexpr long long kWaitMost = 1ll << 30;   // cycles, about half a second
__device__ __forceinline__ bool wait_local(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitMost) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// For a whole tile, as many times as long as its sum may take.
__device__ __forceinline__ bool wait_tile(uint32_t bar, uint32_t parity, volatile int* abort_flag, int times) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort_flag) return false;
    if ((int)((clock64() - t0) >> 30) >= times) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
// Of the MMA thread, for what the other block's threads have written too.
__device__ __forceinline__ bool try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  if (try_cluster(bar, parity)) return true;
  const long long t0 = clock64();
  while (!try_cluster(bar, parity)) {
    if (*abort_flag) return false;
    if (clock64() - t0 > kWaitMost) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 128-byte-swizzled operand tile.  K-major: rows of 128 bytes of k, 8-row groups 1024 bytes apart.  M-major: rows of 64
// i (or j), one per k, 8-k groups 1024 bytes apart, blocks of 64 i 8192 bytes apart.
__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, bool mn_major) {
  const uint32_t lbo = mn_major ? 8192 : 16;
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// 32 rows of 16 bytes of scales, not swizzled: 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scales_desc(uint32_t addr) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)1 << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}
// The 512 bytes of 128 rows' scales, from each block's shared memory into all four lane quarters of its tensor memory.
__device__ __forceinline__ void tcgen05_cp_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <Kind KIND>
__device__ __forceinline__ void mma_fp4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t acc) {
  if constexpr (KIND == Kind::Nv)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(acc)
        : "memory");
}
// Instruction descriptors, without N (and without the place of the scales in their word).
template <typename T, Kind KIND>
__device__ __forceinline__ uint32_t make_idesc(int n) {
  const uint32_t shape = ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileI >> 4) << 24);
  if constexpr (kFp4<KIND>) return shape | (1u << 7) | (1u << 10) | (KIND == Kind::Mx ? 1u << 23 : 0u);   // E2M1; scales UE8M0 or UE4M3
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return shape | (1u << 4) | (fmt << 7) | (fmt << 10) | (KIND != Kind::KK ? 1u << 15 : 0u) | (KIND == Kind::MM ? 1u << 16 : 0u);
}

__device__ __forceinline__ void lds128(uint32_t at, uint4& v) {
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t at, const uint4& v) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  uint32_t d;
  if constexpr (std::is_same<T, __nv_bfloat16>::value) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
// 32 lanes x 16 columns of the accumulator, as mma fragments.
__device__ __forceinline__ void load_16(uint32_t tmem, uint32_t (&r)[16]) {
  tcgen05_ld_16x16(tmem, r);
  tcgen05_ld_16x16(tmem + (16u << 16), r + 8);
}

// Element (row, i) of the output, of type T.
template <typename T, Kind KIND>
__device__ __forceinline__ T* out_row(const Params& p, const Piece& c, int row) {
  const long long r = (KIND == Kind::MM ? (long long)c.e * p.J : 0) + c.row0 + row;
  return static_cast<T*>(p.out) + r * p.I;
}
// Four consecutive i of one row.
template <typename T>
__device__ __forceinline__ void store4(T* dst, int left, bool vec, float a, float b, float c, float d) {
  if (vec && left >= 4) {
    if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(dst) = make_float4(a, b, c, d);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(a, b), pack2<T>(c, d));
  } else {
    const float v[4] = {a, b, c, d};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) dst[i] = Elem<T>::from_float(v[i]);
  }
}

// nvfp4, global scales whose product is no normal fp32 number (rare, so out of line: a second factor in the kernel
// costs 4 %, the calls 0 to 1.5 %): both
// scales one after the other.  A warp's columns q0 to q1 (of 32) of a tile that is not cut, a lane per i;
template <typename T>
__device__ __noinline__ void store_far(const Params& p, const Piece& c, uint32_t acc, int i, int q0, int q1) {
  const float gx = p.gb ? __ldg(p.gb) : 1.0f, gw = p.ga ? __ldg(p.ga + (p.ga_each ? c.e : 0)) : 1.0f;
  for (int q = q0; q < q1; ++q) {
    uint32_t v[32];
    tcgen05_ld_x32(acc + 32 * q, v);
    tcgen05_wait_ld();
    T* y = static_cast<T*>(p.out) + (long long)(c.row0 + 32 * q) * p.I + i;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (i < p.I && 32 * q + j < c.rows) y[(long long)j * p.I] = Elem<T>::from_float(fp4::times_scales(__uint_as_float(v[j]), gx, gw));
  }
}
// and four i of one row of a cut one.
template <typename T>
__device__ __noinline__ void store4_far(const Params& p, int e, T* dst, int left, float a, float b, float c, float d) {
  const float gx = p.gb ? __ldg(p.gb) : 1.0f, gw = p.ga ? __ldg(p.ga + (p.ga_each ? e : 0)) : 1.0f;
  store4(dst, left, p.vec != 0, fp4::times_scales(a, gx, gw), fp4::times_scales(b, gx, gw), fp4::times_scales(c, gx, gw), fp4::times_scales(d, gx, gw));
}

template <typename T, Kind KIND>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads<KIND>, 1)
grouped_tc_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  constexpr bool kSf = kFp4<KIND>, kSum = KIND == Kind::MM;
  constexpr int kSb = KIND == Kind::Mx ? 8 : 16;   // bytes of scales per row and stage
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t stage_bytes = kStageA + (uint32_t)p.b_bytes;
  unsigned char* ring_sf = smem + (size_t)p.stages * stage_bytes;
  const uint32_t sf_bytes = kSf ? 4096u + (uint32_t)p.sfb_chunk : 0u;
  unsigned char* staging = ring_sf + (kSf ? p.sf_slots : 0) * sf_bytes;
  Bars* bars = reinterpret_cast<Bars*>(staging + (sizeof(T) == 2 ? kEpiWarps * kStageOut<KIND> : 0));
  Group* tab = reinterpret_cast<Group*>(bars + 1);
  volatile int* abort_flag = &bars->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank();

  if (warp == 0) {
    if (lane < p.stages) {
      mbar_init(smem_u32(&bars->full[lane]), 1);
      mbar_init(smem_u32(&bars->empty[lane]), 1);
      if (kSum) { mbar_init(smem_u32(&bars->landed[lane]), 1); mbar_init(smem_u32(&bars->fixed[lane]), 2); }
    }
    if (lane < kSfSlots) { mbar_init(smem_u32(&bars->sf_full[lane]), 3); mbar_init(smem_u32(&bars->sf_empty[lane]), 1); }
    if (lane < kSfBuffers) mbar_init(smem_u32(&bars->sf_ready[lane]), 1);
    if (lane < 2) { mbar_init(smem_u32(&bars->acc_full[lane]), 1); mbar_init(smem_u32(&bars->acc_empty[lane]), 2 * kEpiWarps); }
    if (lane == 0) bars->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncwarp();
  } else if (warp == 1) {
    tcgen05_alloc(smem_u32(&bars->tmem_base), 512);
    tcgen05_relinquish();
  } else if (warp == 3) {
    if (lane == 0) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a) : "memory");
    if (kSf && lane == 1) asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.sfa) : "memory");
    if (lane >= 8 && lane < 13 && (kSum ? lane == 8 : (128 >> (lane - 8)) * 128 <= p.b_bytes))
      asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.b[lane - 8]) : "memory");
  } else if (warp == 2) {
    // The table: a lane takes E / 32 consecutive groups.
    const int per = (p.E + 31) / 32, lo = min(p.E, lane * per), hi = min(p.E, lo + per);
    bool bad = false;
    auto size_of = [&](int e) -> int {
      if (!p.sizes) return p.T;
      const long long n = p.size_bytes == 8 ? __ldg(static_cast<const long long*>(p.sizes) + e) : (long long)__ldg(static_cast<const int*>(p.sizes) + e);
      bad |= n < 0 || n > p.T;
      return n < 0 ? 0 : (n > p.T ? p.T : (int)n);
    };
    auto add = [&](int a, int b) { bad |= a + b > p.T; return min(a + b, p.T); };   // (T is below 2^30)
    int at = 0;
    for (int e = lo; e < hi; ++e) at = add(at, size_of(e));
    int rows_end = at, total, all_steps;   // sums over all groups; a lane keeps those of the lanes before it
    if (p.E > 1) {
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int v = __shfl_up_sync(0xFFFFFFFFu, at, d);
        if (lane >= d) at = add(at, v);
      }
      rows_end = __shfl_sync(0xFFFFFFFFu, at, 31);
      at = __shfl_up_sync(0xFFFFFFFFu, at, 1);
    }
    if (lane == 0) at = 0;
    int units = 0, steps = 0;
    for (int e = lo; e < hi; ++e) {
      const int r0 = at;
      at = add(at, size_of(e));
      const int2 tr = tiles_j<KIND>(p, at - r0);
      tab[e] = make_int4(r0, units, steps, tr.y << 9 | tr.x);
      units += tr.y * p.i_tiles;
      steps += tr.y * p.i_tiles * group_steps<KIND>(p, at - r0);
    }
    total = units;
    all_steps = steps;
    if (p.E > 1) {
      int u0 = units, s0 = steps;
#pragma unroll
      for (int d = 1; d < 32; d *= 2) {
        const int a = __shfl_up_sync(0xFFFFFFFFu, u0, d), b = __shfl_up_sync(0xFFFFFFFFu, s0, d);
        if (lane >= d) { u0 += a; s0 += b; }
      }
      total = __shfl_sync(0xFFFFFFFFu, u0, 31);
      all_steps = __shfl_sync(0xFFFFFFFFu, s0, 31);
      u0 -= units;
      s0 -= steps;
      for (int e = lo; e < hi; ++e) { tab[e].y += u0; tab[e].z += s0; }
    } else {   // one group, in lane 0
      rows_end = __shfl_sync(0xFFFFFFFFu, rows_end, 0);
      total = __shfl_sync(0xFFFFFFFFu, total, 0);
      all_steps = __shfl_sync(0xFFFFFFFFu, all_steps, 0);
    }
    bad = __any_sync(0xFFFFFFFFu, bad);
    if (lane == 0) tab[p.E] = make_int4(rows_end, total, all_steps, 0);
    __syncwarp();
    const int pairs = gridDim.x >> 1, full = (int)((uint32_t)total / (uint32_t)pairs) * pairs;
    int cut_pairs = 0, base = 0, rest = 0;
    if (full < total) {
      int e = 0, h = p.E;   // the group in which the rest begins
      while (h - e > 1) { const int m = (e + h) >> 1; if (tab[m].y <= full) e = m; else h = m; }
      base = tab[e].z + (full - tab[e].y) * group_steps<KIND>(p, tab[e + 1].x - tab[e].x);
      rest = all_steps - base;
      cut_pairs = cut_for<KIND>(lane, total - full, rest, KIND == Kind::MM ? p.NT : (int)__fdividef((float)rows_end * (float)p.i_tiles, (float)total), pairs);
    }
    if (lane == 0) {
      bars->rows = rows_end;
      bars->full_units = cut_pairs ? full : total;
      bars->cut_pairs = cut_pairs;
      bars->cut_steps = rest;
      bars->cut_base = base;
      if (bad && blockIdx.x == 0) atomicMax(p.status, 9u);
    }
  }
  tcgen05_fence_before();
  __syncwarp();
  cluster_sync();   // (every thread of both blocks: the block's own barrier too)
  tcgen05_fence_after();
  const uint32_t tmem = bars->tmem_base;
  const int nacc = 2 * p.NT + (kSf ? 2 * kSfColumns : 0) <= 512 ? 2 : 1;
  const uint32_t tmem_sf = tmem + nacc * p.NT;
  // (fewer than the ring has stages: whoever waits for a stage's MMAs must not miss a turn of its barrier)
  const uint32_t sf_buffers = kSfBuffers * kSfColumns + nacc * p.NT <= 512 && p.stages > kSfBuffers ? kSfBuffers : 2;
  const uint32_t ring = smem_u32(smem);
  Walk& walk = bars->walk[warp];
  if (lane == 0) walk_begin(*bars, walk);
  __syncwarp();
  auto next_of_warp = [&]() -> bool {
    __syncwarp();   // everybody has read the last piece
    bool more = false;
    if (lane == 0) more = walk_next<KIND>(p, *bars, tab, walk);
    __syncwarp();
    return __shfl_sync(0xFFFFFFFFu, more, 0);
  };

  if (warp == 0 || warp == 3) {
    // ------------------------------------------------------------ operands: a warp for each
    if (kSf && warp == 3) asm volatile("griddepcontrol.wait;" ::: "memory");   // 4 bits: the kernel that quantizes b may still be running
    if (elect_one()) {
      const bool of_a = warp == 0;
      const uint32_t full = smem_u32(&bars->full[0]), lfull = leader_addr(full), empty = smem_u32(&bars->empty[0]), landed = smem_u32(&bars->landed[0]);
      uint32_t s = 0, ph = 1, sl = 0, sl_ph = 1;
      bool ok = true;
      while (ok && walk_next<KIND>(p, *bars, tab, walk)) {
        const Piece c = walk.c;
        const int half = c.neff >> 1, i = c.i0 + rank * kLanes, j = c.row0 + rank * half;
        int box0 = 0;
        const int rows = kSum ? half : box_rows(half, &box0);
        const uint32_t bytes = kStageA + (uint32_t)rows * 128u;
        for (int ks = c.ks0; ks < c.ks1; ++ks) {
          if (kSf && !of_a && (ks - c.ks0) % kSpc<KIND> == 0) {   // a's scales of the chunk that begins here
            if (!wait_local(smem_u32(&bars->sf_empty[sl]), sl_ph, abort_flag)) { ok = false; break; }
            if (rank == 0) mbar_expect_tx(smem_u32(&bars->sf_full[sl]), 2 * 4096);
            // (rows of 1024 bytes: two words of 128 rows)
            tma_load_2d_pair(smem_u32(ring_sf) + sl * sf_bytes, &maps.sfa, 0, (c.e * p.i_blocks + c.i0 / kLanes + rank) * (p.sf_words / 2) + ks * kSb / 8,
                             leader_addr(smem_u32(&bars->sf_full[sl])));
            if (++sl == (uint32_t)p.sf_slots) { sl = 0; sl_ph ^= 1; }
          }
          if (!wait_local(empty + s * 8, ph, abort_flag)) { ok = false; break; }
          const uint32_t at = ring + s * stage_bytes + (of_a ? 0 : kStageA);
          // A group's last stage (MM) is counted by this block, for the warp that zeroes foreign rows; any other by the pair's leader.
          const bool ends = kSum && c.len - ks * 64 < 64;
          const uint32_t bar = (ends ? landed : lfull) + s * 8;
          if (of_a) {
            if (ends) mbar_expect_tx(bar, bytes);
            else if (rank == 0) mbar_expect_tx(full + s * 8, 2 * bytes);
          }
          if constexpr (kSum) {
            const CUtensorMap* map = of_a ? &maps.a : &maps.b[0];
            const int col = of_a ? i : j, n = of_a ? 2 : half / 64, t = c.t0 + ks * 64;
            load_columns(at, map, p.blocks & (of_a ? 1 : 2), n, col, t, 0, bar, ends);
          } else if (of_a) {
            if constexpr (KIND == Kind::MK) load_columns(at, &maps.a, p.blocks & 1, 2, i, ks * 64, c.e, bar, false);
            else tma_3d_pair(at, &maps.a, ks * (kSf ? 128 : 64), i, c.e, bar);
          } else {
            const int k = ks * (kSf ? 128 : 64);
            const CUtensorMap* map = &maps.b[4 - (31 - __clz(box0 >> 3))];
            tma_3d_pair(at, map, k, j, 0, bar);
            if (rows > box0) tma_3d_pair(at + box0 * 128, &maps.b[4 - (31 - __clz((rows - box0) >> 3))], k, j + box0, 0, bar);
          }
          if (++s == (uint32_t)p.stages) { s = 0; ph ^= 1; }
        }
      }
      if (!ok) for (int n = 0; n < 100; ++n) __nanosleep(1000);   // copies in flight land before the block ends
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMAs (leader)
    if (rank == 0 && elect_one()) {
      const uint32_t full = smem_u32(&bars->full[0]), empty = smem_u32(&bars->empty[0]);
      const uint32_t sf_ready = smem_u32(&bars->sf_ready[0]);
      const uint32_t fixed = smem_u32(&bars->fixed[0]);
      // A bit per slot: the phase that its barriers `full` and `fixed` are in (MM uses one or the other)
      uint32_t s = 0, full_ph = 0, fixed_ph = 0, n_piece = 0, n_stage = 0;
      bool ok = true;
      while (ok && walk_next<KIND>(p, *bars, tab, walk)) {
        const Piece c = walk.c;
        const uint32_t idesc = make_idesc<T, KIND>(c.neff);
        const uint32_t ab = nacc == 2 ? n_piece & 1 : 0, an = nacc == 2 ? n_piece >> 1 : n_piece;
        const uint32_t acc = tmem + ab * p.NT;
        ++n_piece;
        if (!wait_local(smem_u32(&bars->acc_empty[ab]), (an & 1) ^ 1, abort_flag)) break;
        uint32_t first = 0;
        for (int ks = c.ks0; ks < c.ks1; ++ks) {
          const bool ends = kSum && c.len - ks * 64 < 64;
          if (!wait_cluster((ends ? fixed : full) + s * 8, ((ends ? fixed_ph : full_ph) >> s) & 1, abort_flag)) { ok = false; break; }
          if (ends) fixed_ph ^= 1u << s; else full_ph ^= 1u << s;
          tcgen05_fence_after();
          const uint64_t da = sw128_desc(ring + s * stage_bytes, KIND == Kind::MK || kSum);
          const uint64_t db = sw128_desc(ring + s * stage_bytes + kStageA, kSum);
          if constexpr (kSf) {
            const uint32_t buf = n_stage & (sf_buffers - 1), ta = tmem_sf + buf * kSfColumns, tb = ta + 16;
            if (!wait_local(sf_ready + buf * 8, n_stage / sf_buffers & 1, abort_flag)) { ok = false; break; }
            tcgen05_fence_after();
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const int w = KIND == Kind::Mx ? kk >> 1 : kk, id = KIND == Kind::Mx ? (kk & 1) * 2 : 0;
              mma_fp4<KIND>(acc, da + 2 * kk, db + 2 * kk, idesc | (uint32_t)id << 29 | (uint32_t)id << 4, ta + 4 * w, tb + 8 * w, kk ? 1u : first);
            }
          } else {
            const int a_step = KIND == Kind::KK ? 2 : 128, b_step = kSum ? 128 : 2;
            const int slices = ends ? max(1, (c.len - ks * 64 + 15) >> 4) : 4;   // of 16 k that hold any of the group's rows
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (!kSum || kk < slices) tcgen05_mma_ss(acc, da + a_step * kk, db + b_step * kk, idesc, kk ? 1u : first);
          }
          first = 1;
          ++n_stage;
          tcgen05_commit_pair(empty + s * 8);
          if (++s == (uint32_t)p.stages) s = 0;
        }
        tcgen05_commit_pair(smem_u32(&bars->acc_full[ab]));
      }
    }
  } else if (kSum && warp == 2) {
    // ------------------------------------------------------------ rows of other groups are zeroed
    const uint32_t landed = smem_u32(&bars->landed[0]), lfixed = leader_addr(smem_u32(&bars->fixed[0]));
    uint32_t at = 0, ph = 0;   // stages so far; a bit per slot
    while (next_of_warp()) {
      const Piece c = walk.c;
      at += c.ks1 - c.ks0;
      const int valid = c.len - (c.ks1 - 1) * 64;
      if (valid >= 64) continue;
      const uint32_t s = (at - 1) % (uint32_t)p.stages;
      if (!__all_sync(0xFFFFFFFFu, wait_tile(landed + s * 8, (ph >> s) & 1, abort_flag, p.wait_times))) break;
      ph ^= 1u << s;
      // blocks of 64 columns: two of a, one or two of b; eight lanes for a row of each
      const uint32_t tile = ring + s * stage_bytes + (lane >> 3) * 8192 + (lane & 7) * 16;
      const int from = max(valid, 0), to = max(16, (valid + 15) & ~15);   // the slice of 16 that the group ends in
      if ((lane >> 3) < 2 + (c.neff >> 7))
        for (int r = from; r < to; ++r) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(tile + r * 128), "r"(0u) : "memory");
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(lfixed + s * 8);
    }
  } else if (kSf && warp == 2) {
    // ------------------------------------------------------------ scales, from both blocks' shared memory into their tensor memories
    if (rank == 0 && elect_one()) {
      const uint32_t sf_full = smem_u32(&bars->sf_full[0]), sf_empty = smem_u32(&bars->sf_empty[0]), sf_ready = smem_u32(&bars->sf_ready[0]);
      const uint32_t empty = smem_u32(&bars->empty[0]), at = smem_u32(ring_sf);
      const uint32_t kb = p.sfb_chunk / 8;   // bytes per word of k of b's scales: 512 or 1024
      constexpr int kWords = kSb / 4;
      uint32_t sl = 0, ph = 0, n_stage = 0, done = 0, done_ph = 0;
      bool ok = true;
      while (ok && walk_next<KIND>(p, *bars, tab, walk)) {
        const Piece c = walk.c;
        for (int k0 = c.ks0; ok && k0 < c.ks1; k0 += kSpc<KIND>) {
          if (!wait_cluster(sf_full + sl * 8, ph, abort_flag)) { ok = false; break; }
          tcgen05_fence_after();
          for (int j = 0; j < kSpc<KIND> && k0 + j < c.ks1; ++j, ++n_stage) {
            const uint32_t buf = n_stage & (sf_buffers - 1);
            if (n_stage >= sf_buffers) {   // the stage that used these columns last has been multiplied
              if (!wait_local(empty + done * 8, done_ph, abort_flag)) { ok = false; break; }
              if (++done == (uint32_t)p.stages) { done = 0; done_ph ^= 1; }
              tcgen05_fence_after();
            }
            const uint32_t ta = tmem_sf + buf * kSfColumns, tb = ta + 16;
            const uint32_t sa = at + sl * sf_bytes + j * kWords * 512, sb = at + sl * sf_bytes + 4096 + j * kWords * kb;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              tcgen05_cp_scales(ta + 4 * w, scales_desc(sa + 512 * w));
              tcgen05_cp_scales(tb + 8 * w, scales_desc(sb + kb * w));
              if (c.neff > 128) tcgen05_cp_scales(tb + 8 * w + 4, scales_desc(sb + kb * w + 512));
            }
            tcgen05_commit_pair(sf_ready + buf * 8);
          }
          if (!ok) break;
          tcgen05_commit_pair(sf_empty + sl * 8);
          if (++sl == (uint32_t)p.sf_slots) { sl = 0; ph ^= 1; }
        }
      }
    }
  } else if (kSf && warp >= kScaleWarp0) {
    // ------------------------------------------------------------ b's scales: warps take chunks in turn
    // (no more warps than slots, so that none is ahead of a slot's barrier by more than a turn)
    const uint32_t first = warp - kScaleWarp0, turns = min(kScaleWarps, p.sf_slots), sf_empty = smem_u32(&bars->sf_empty[0]), lsf = leader_addr(smem_u32(&bars->sf_full[0]));
    const int blocks = p.sfb_chunk >> 12;   // of 128 rows: 1 or 2
    uint32_t chunk = 0, sl = first, ph = 1;
    bool ok = true;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    while (ok && first < turns && next_of_warp()) {
      const Piece c = walk.c;
      for (int ks = c.ks0; ks < c.ks1; ks += kSpc<KIND>, ++chunk) {
        if ((chunk & (turns - 1)) != first) continue;
        // a lane has rows lane, lane + 32, .. (past the end of b: the last row, for columns that nobody stores)
        const uint32_t* from = p.sfb + (long long)(ks * kSb / 4) * p.T;
        int row[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) row[r] = min(c.row0 + lane + 32 * r, p.T - 1);
        uint4 v[2][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (128 * h >= c.neff) break;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const uint32_t* w = from + (long long)k * p.T;
            v[h][k].x = __ldcg(w + row[4 * h]);
            if (128 * h + 32 < c.neff) v[h][k].y = __ldcg(w + row[4 * h + 1]);
            if (128 * h + 64 < c.neff) v[h][k].z = __ldcg(w + row[4 * h + 2]);
            if (128 * h + 96 < c.neff) v[h][k].w = __ldcg(w + row[4 * h + 3]);
          }
        }
        // read before the slot is free, stored after
        ok = __all_sync(0xFFFFFFFFu, wait_local(sf_empty + sl * 8, ph, abort_flag));
        if (!ok) break;
        const uint32_t at = smem_u32(ring_sf) + sl * sf_bytes + 4096;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (128 * h >= c.neff) break;
#pragma unroll
          for (int k = 0; k < 8; ++k) sts128(at + (k * blocks + h) * 512 + lane * 16, v[h][k]);
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(lsf + sl * 8);
        sl += turns;
        if (sl >= (uint32_t)p.sf_slots) { sl -= p.sf_slots; ph ^= 1; }
      }
    }
  } else if (warp >= kEpiWarp0 && warp < kEpiWarp0 + kEpiWarps) {
    // ------------------------------------------------------------ epilogue
    const int w = warp - kEpiWarp0, quad = warp & 3, chalf = w >> 2;
    const uint32_t stg = smem_u32(staging) + w * kStageOut<KIND>;
    const uint32_t lane_field = (uint32_t)(quad * 32) << 16;
    if (!kSum && bars->rows < p.T) {   // rows that belong to no group
      T* z = static_cast<T*>(p.out) + (long long)bars->rows * p.I;
      const long long n = (long long)(p.T - bars->rows) * p.I, step = (long long)gridDim.x * kEpiWarps * 32;
      for (long long i = ((long long)blockIdx.x * kEpiWarps + w) * 32 + lane; i < n; i += step) z[i] = Elem<T>::from_float(0.0f);
    }
    // One thread finds the pieces, the next one while a tile is stored.
    auto find = [&](uint32_t n) {
      const bool more = walk_next<KIND>(p, *bars, tab, walk);
      if (more) bars->piece[n & 1] = walk.c;
      bars->more[n & 1] = more;
    };
    if (w == 0 && lane == 0) find(0);
    for (uint32_t n_piece = 0;; ++n_piece) {
      const uint32_t ab = nacc == 2 ? n_piece & 1 : 0, an = nacc == 2 ? n_piece >> 1 : n_piece;
      // One warp looks and all go by what it found: the abort flag may be raised between two warps' looks.
      if (w == 0) {
        __syncwarp();
        const bool seen = bars->more[n_piece & 1] && __all_sync(0xFFFFFFFFu, wait_tile(smem_u32(&bars->acc_full[ab]), an & 1, abort_flag, p.wait_times));
        if (lane == 0) bars->seen[n_piece & 1] = seen;
        __syncwarp();
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
      if (!bars->seen[n_piece & 1]) break;
      const Piece c = bars->piece[n_piece & 1];
      tcgen05_fence_after();
      float alpha = 1.0f;
      if constexpr (kSf) {
        if (p.ga) alpha = __ldg(p.ga + (p.ga_each ? c.e : 0));
        if (p.gb) alpha *= __ldg(p.gb);
      }
      const bool far = KIND == Kind::Nv && !fp4::one_factor(alpha);
      const uint32_t acc = tmem + ab * p.NT + lane_field;
      const int i_warp = c.i0 + rank * kLanes + quad * 32;
      auto release = [&]() {
        tcgen05_fence_before();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive_cluster(leader_addr(smem_u32(&bars->acc_empty[ab])));
          if (w == 0) find(n_piece + 1);
        }
        __syncwarp();
      };
      // this warp's columns: half of them, in pieces of 32
      const int pieces = (c.neff + 31) / 32, p0 = chalf ? (pieces + 1) / 2 : 0, p1 = chalf ? pieces : (pieces + 1) / 2;
      if (c.parts > 1) {
        const int slot = c.part == 0 ? 2 * c.j0 + 1 : 2 * (c.j0 + c.part);
        float* part = p.partial + ((size_t)slot * 2 + rank) * ((size_t)p.NT * kLanes) + quad * 32 + lane;
        for (int q = p0; q < p1; ++q) {
          uint32_t v[32];
          tcgen05_ld_x32(acc + 32 * q, v);
          tcgen05_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (32 * q + j < c.rows) __stcg(part + (size_t)(32 * q + j) * kLanes, __uint_as_float(v[j]));
        }
        release();
        __threadfence();
        asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
        if (w == 0 && lane == 0) {
          uint32_t* ctr = p.counters + c.j0 * 2 + rank;
          const bool last = atomicAdd(ctr, 1u) == (uint32_t)c.parts - 1;
          if (last) *ctr = 0;
          bars->last = last;
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");
        if (bars->last) {
          __threadfence();
          const size_t pitch = 2 * (size_t)p.NT * kLanes / 4;   // slot to slot
          const float4* base = reinterpret_cast<const float4*>(p.partial + (size_t)rank * ((size_t)p.NT * kLanes)) + lane;
          const int i = c.i0 + rank * kLanes + 4 * lane;
          const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          // two rows and up to eight parts of each in flight
          for (int r = w; r < c.rows; r += 2 * kEpiWarps) {
            const int rows = r + kEpiWarps < c.rows ? 2 : 1;
            const float4* at = base + (size_t)r * (kLanes / 4);
            float4 sum[2] = {zero, zero};
            for (int s = 0; s < c.parts; s += 8) {
              float4 v[2][8];
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                  const int q = s + k;
                  v[h][k] = h < rows && q < c.parts
                                ? __ldcg(at + h * (kEpiWarps * kLanes / 4) + (size_t)(q == 0 ? 2 * c.j0 + 1 : 2 * (c.j0 + q)) * pitch) : zero;
                }
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 8; ++k) { sum[h].x += v[h][k].x; sum[h].y += v[h][k].y; sum[h].z += v[h][k].z; sum[h].w += v[h][k].w; }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
              if (h < rows && i < p.I) {
                T* dst = out_row<T, KIND>(p, c, r + h * kEpiWarps) + i;
                if (far) store4_far(p, c.e, dst, p.I - i, sum[h].x, sum[h].y, sum[h].z, sum[h].w);
                else store4(dst, p.I - i, p.vec != 0, sum[h].x * alpha, sum[h].y * alpha, sum[h].z * alpha, sum[h].w * alpha);
              }
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory");   // `last` may be written again
        continue;
      }
      if (far) {
        store_far<T>(p, bars->piece[n_piece & 1], acc, i_warp + lane, p0, p1);
        release();
        continue;
      }
      if constexpr (sizeof(T) == 2) {
        if (p.vec) {
          const uint32_t row = lane & 7, put = stg + row * 64 + ((((uint32_t)lane >> 3) ^ (row >> 1)) << 4);
          const uint32_t get = stg + (lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4);
          const int i = i_warp + (lane & 3) * 8;
          T* dst = out_row<T, KIND>(p, c, 32 * p0 + (lane >> 2)) + i;
          // Rounded and packed first, so that the accumulator is free for another tile's MMAs before (most of) it is stored.
          // (4 bits: half at a time, for lack of registers)
          constexpr int kBatch = kSf ? 2 : 4;
          if (p0 == p1) release();
          for (int b0 = p0; b0 < p1; b0 += kBatch) {
            uint32_t packed[kBatch][2][8];
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
              if (b0 + q >= p1) break;
              const int col = 32 * (b0 + q);
              const bool two = col + 16 < c.neff;
              uint32_t v[2][16];
              load_16(acc + col, v[0]);
              if (two) load_16(acc + col + 16, v[1]);
              tcgen05_wait_ld16(v[0]);
              tcgen05_wait_ld16(v[1]);
#pragma unroll
              for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int k = 0; k < 8; ++k)
                  packed[q][h][k] = pack2<T>(__uint_as_float(v[h][2 * k]) * alpha, __uint_as_float(v[h][2 * k + 1]) * alpha);
            }
            if (b0 + kBatch >= p1) release();
            if constexpr (kSum) {
              // Two warps (64 i) share rows of 128 bytes, 32 at a time in two buffers.  Whoever issues the stores comes to the
              // pair's barrier when the store before has left its buffer, which then is the next to be written.  (16 rows at a
              // time: 1700 of a tile's 4900 cycles were spent waiting for that, 1400 issuing.)
              const uint32_t both = stg - (w & 1) * kStageOut<KIND>, chunk0 = (w & 1) * 4 + (lane >> 3);
              const bool issues = (w & 1) == 0 && lane == 0;
              const int i64 = i_warp & ~63;
#pragma unroll
              for (int q = 0; q < kBatch; ++q) {
                if (b0 + q >= p1) break;
                const uint32_t buf = both + (q & 1) * 4096;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const uint32_t row = 8 * x + (lane & 7);
                  const uint32_t (&v)[8] = packed[q][x >> 1];
                  const int k = 2 * (x & 1);
                  stmatrix_x4_trans(buf + row * 128 + ((chunk0 ^ (row & 7)) << 4), v[k], v[k + 1], v[4 + k], v[5 + k]);
                }
                if (issues) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                fence_async_smem();
                asm volatile("bar.sync %0, 64;" ::"r"(3 + (w >> 1)) : "memory");
                if (issues && i64 < p.I) tma_store_3d(&maps.out, buf, i64, c.row0 + 32 * (b0 + q), c.e);
              }
              continue;
            }
#pragma unroll
            for (int q = 0; q < kBatch; ++q) {
              if (b0 + q >= p1) break;
              const int col = 32 * (b0 + q);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                if (h == 1 && col + 16 >= c.neff) break;
                // 16 rows of 64 bytes, 16-byte chunks xor-ed with row / 2
#pragma unroll
                for (int x = 0; x < 2; ++x)
                  stmatrix_x4_trans(put + h * 1024 + x * 512, packed[q][h][2 * x], packed[q][h][2 * x + 1], packed[q][h][4 + 2 * x], packed[q][h][5 + 2 * x]);
              }
              __syncwarp();
              if (i < p.I) {   // (whole chunks: rows on 16-byte boundaries are whole eights long)
                const int n = c.rows - col - (lane >> 2);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  uint4 o;
                  lds128(get + k * 512, o);
                  if (8 * k < n) *reinterpret_cast<uint4*>(dst + (long long)(8 * k) * p.I) = o;
                }
              }
              dst += (long long)32 * p.I;
              __syncwarp();
            }
          }
          continue;
        }
      }
      // f32, or rows of any alignment: a lane per i, the warp stores 64 (f32: 128) contiguous bytes per row
      const int i = i_warp + lane;
      for (int q = p0; q < p1; ++q) {
        uint32_t v[32];
        tcgen05_ld_x32(acc + 32 * q, v);
        tcgen05_wait_ld();
        if (q + 1 == p1) release();
        if (i < p.I) {
          T* y = out_row<T, KIND>(p, c, 32 * q) + i;
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (32 * q + j < c.rows) y[(long long)j * p.I] = Elem<T>::from_float(__uint_as_float(v[j]) * alpha);
        }
        __syncwarp();
      }
      if (p0 == p1) release();
    }
  }

  if (kSum) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  __syncwarp();
  tcgen05_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort_flag) atomicMax(p.status, 8u);
  __syncwarp();
  cluster_sync();
  if (warp == 1) {
    tcgen05_fence_after();
    tcgen05_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- host side
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encode_fn() {
  static EncodeFn fn = [] {
    void* sym = nullptr;
    cudaDriverEntryPointQueryResult qres;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &qres) == cudaSuccess &&
                    qres == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeFn>(sym) : nullptr;
  }();
  return fn;
}
int sm_pairs() {
  static int cached[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 74;
  if (!cached[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 2) n = 148;
    cached[dev] = n / 2;
  }
  return cached[dev];
}

// Rows of `cols` elements (bytes where esize is 1), `mid` of them per matrix; boxes of `box0` x `box1`.  `blocks`: columns as
// two dimensions, blocks of 64 and their number, of which a box has `blocks`.
int encode(CUtensorMap* m, int dtype, int esize, const void* base, int64_t cols, int64_t pitch, int64_t mid, int64_t outer, int box0, int box1,
           int blocks = 0) {
  const cuuint64_t dims[4] = {(cuuint64_t)(blocks ? 64 : cols), (cuuint64_t)mid, (cuuint64_t)(blocks ? cols / 64 : outer), (cuuint64_t)outer};
  const cuuint64_t strides[3] = {(cuuint64_t)pitch, (cuuint64_t)(blocks ? 128 : pitch * mid), (cuuint64_t)pitch * mid};
  const cuuint32_t box[4] = {(cuuint32_t)box0, (cuuint32_t)box1, (cuuint32_t)(blocks ? blocks : 1), 1}, one[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t = esize == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                : dtype == B200Q_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = encode_fn()(m, t, blocks ? 4 : 3, const_cast<void*>(base), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? B200Q_OK : fail(B200Q_ERR_CUDA, "[grouped product] a tensor map could not be encoded (%d)", (int)r);
}

// Once per kernel, device and thread.
int allow_smem(const void* kernel) {
  constexpr int kMost = 16;   // instantiations: 12
  static thread_local const void* done[64][kMost];
  static thread_local int count[64];
  int dev = 0;
  B200Q_CUDA_OK(cudaGetDevice(&dev));
  const bool known = dev >= 0 && dev < 64;
  for (int i = 0; known && i < count[dev]; ++i)
    if (done[dev][i] == kernel) return B200Q_OK;
  B200Q_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemMax));
  if (known && count[dev] < kMost) done[dev][count[dev]++] = kernel;
  return B200Q_OK;
}

template <typename T, Kind KIND>
int launch(const Maps& m, Params& p, cudaStream_t st) {
  const size_t stage = kStageA + (size_t)p.b_bytes;
  const size_t other = 1024 + (sizeof(T) == 2 ? kEpiWarps * kStageOut<KIND> : 0) + sizeof(Bars) + (size_t)(p.E + 1) * sizeof(Group);
  size_t fixed;
  for (;; p.sf_slots /= 2) {   // (thousands of groups leave room for fewer scales)
    fixed = other + (kFp4<KIND> ? p.sf_slots * (4096 + (size_t)p.sfb_chunk) : 0);
    p.stages = fixed < kSmemMax ? (int)((kSmemMax - fixed) / stage) : 0;
    if (!kFp4<KIND> || p.stages >= 3 || p.sf_slots == 2) break;
  }
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  if (p.stages < 3) return fail(B200Q_ERR_UNSUPPORTED, "[grouped product] No implementation for problem shape: the table of %d groups leaves no shared memory", p.E);
  size_t smem = fixed + p.stages * stage;
  // One block per SM: the allocation of all of tensor memory never waits for another block of this kernel.
  if (smem < 120 * 1024) smem = 120 * 1024;
  auto kernel = grouped_tc_kernel<T, KIND>;
  if (int rc = allow_smem((const void*)kernel)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * sm_pairs());
  cfg.blockDim = dim3(kThreads<KIND>);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  // 4 bits: starts beside the kernel that quantizes b, which is always the one before it on the stream
  cudaLaunchAttribute early{};
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &early;
  cfg.numAttrs = kFp4<KIND> ? 1 : 0;
  B200Q_CUDA_OK(cudaLaunchKernelEx(&cfg, kernel, m, p));
  B200Q_LAUNCH_OK("grouped_tc_kernel");
  return B200Q_OK;
}

template <Kind KIND>
int launch_t(int dtype, const Maps& m, Params& p, cudaStream_t st) {
  if (dtype == B200Q_BF16) return launch<__nv_bfloat16, KIND>(m, p, st);
  if (dtype == B200Q_F16) return launch<__half, KIND>(m, p, st);
  if constexpr (kFp4<KIND>) return launch<float, KIND>(m, p, st);
  return fail(B200Q_ERR_UNSUPPORTED, "[grouped product] only bfloat16 and float16 are supported");
}

int tile_columns(int64_t rows) { return (int)(rows >= kMaxNT ? kMaxNT : (rows + 15) / 16 * 16); }
constexpr size_t kCounterBytes = 2048;   // [pairs][2] words, 148 SMs and more

}  // namespace

// The product's own part of the workspace: counters, then partial sums.
size_t grouped_tc_bytes(int64_t rows, bool sum) {
  return kCounterBytes + 2 * (size_t)sm_pairs() * 2 * (size_t)(sum ? kMaxNT : tile_columns(rows)) * kLanes * 4;
}

int grouped_tc(const GroupedTcArgs& a, cudaStream_t st) {
  if (!encode_fn()) return fail(B200Q_ERR_CUDA, "[grouped product] cuTensorMapEncodeTiled is not available");
  if (int rc = bind_context()) return rc;
  Maps m;
  Params p{};
  p.sizes = a.sizes; p.size_bytes = a.size_bytes;
  p.E = (int)a.E; p.T = (int)a.T; p.I = (int)a.I; p.J = (int)a.J; p.K = (int)a.K;
  p.i_tiles = (p.I + kTileI - 1) / kTileI;
  const bool sum = a.form == GroupedForm::Sum, fp4 = a.form == GroupedForm::Mx || a.form == GroupedForm::Nv;
  p.NT = sum ? (a.J > 128 ? 256 : 128) : tile_columns(a.T);
  const int es = a.dtype == B200Q_F32 ? 4 : 2;
  p.out = a.out;
  p.vec = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.I * es)) & 15) == 0;
  p.counters = static_cast<uint32_t*>(a.ws);
  p.partial = reinterpret_cast<float*>(static_cast<char*>(a.ws) + kCounterBytes);
  p.status = a.status;
  p.wait_times = wait_times(sum ? a.T / 64 + 1 : (a.K + (fp4 ? 255 : 63)) / (fp4 ? 256 : 64));
  p.sfb_chunk = p.NT > 128 ? 8192 : 4096;
  p.sf_slots = p.NT > 128 ? 4 : 8;
  p.sfb = a.sfb; p.sf_words = (int)a.sf_words;
  p.i_blocks = (p.I + kLanes - 1) / kLanes;
  p.ga = a.ga; p.gb = a.gb; p.ga_each = a.ga_each;
  // number of tiles and steps in 32 bits
  const int64_t tiles = ((sum ? (a.J + p.NT - 1) / p.NT * a.E : a.T / p.NT + a.E + 1)) * p.i_tiles;
  const int64_t steps = sum ? (a.T / 64 + 2 * a.E) * ((a.J + p.NT - 1) / p.NT) * p.i_tiles : tiles * ((a.K + 63) / 64);
  if (tiles >= INT32_MAX || steps >= INT32_MAX)
    return fail(B200Q_ERR_UNSUPPORTED, "[grouped product] No implementation for problem shape: too many tiles");
  const int es_a = fp4 ? 1 : 2;
  const int64_t ka = fp4 ? a.K / 2 : a.K;
  int box0 = 0, rc = B200Q_OK;
  p.b_bytes = (sum ? p.NT / 2 : box_rows(p.NT / 2, &box0)) * 128;
  p.blocks = (a.form != GroupedForm::KK && !fp4 && a.I % 64 == 0 ? 1 : 0) | (sum && a.J % 256 == 0 ? 2 : 0);
  if (sum) {
    rc = encode(&m.a, a.dtype, 2, a.a, a.I, a.a_pitch, a.T, 1, 64, 64, p.blocks & 1 ? 2 : 0);
    if (!rc) rc = encode(&m.b[0], a.dtype, 2, a.b, a.J, a.b_pitch, a.T, 1, 64, 64, p.blocks & 2 ? 2 : 0);
    if (!rc && p.vec) rc = encode(&m.out, a.dtype, 2, a.out, a.I, a.I * 2, a.J, a.E, 64, 32);
  } else {
    const int box = fp4 ? 128 : 64;
    if (a.form == GroupedForm::MK) rc = encode(&m.a, a.dtype, 2, a.a, a.I, a.a_pitch, a.K, a.E, 64, 64, p.blocks & 1 ? 2 : 0);
    else rc = encode(&m.a, a.dtype, es_a, a.a, ka, a.a_pitch, a.I, a.E, box, kLanes);
    for (int i = 0; i < 5 && !rc; ++i)
      if ((128 >> i) <= p.b_bytes / 128) rc = encode(&m.b[i], a.dtype, es_a, a.b, ka, a.b_pitch, a.T, 1, box, 128 >> i);
  }
  if (fp4 && !rc) {
    const int64_t rows = a.E * p.i_blocks * (a.sf_words / 2);
    const cuuint64_t dims[2] = {256, (cuuint64_t)rows}, strides[1] = {1024};
    const cuuint32_t sbox[2] = {256, 4}, one[2] = {1, 1};
    if (rows >= INT32_MAX) return fail(B200Q_ERR_UNSUPPORTED, "[grouped product] No implementation for problem shape: too many scales");
    const CUresult r = encode_fn()(&m.sfa, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint32_t*>(a.sfa), dims, strides, sbox, one,
                                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(B200Q_ERR_CUDA, "[grouped product] a tensor map could not be encoded (%d)", (int)r);
  }
  if (rc) return rc;
  switch (a.form) {
    case GroupedForm::KK: return launch_t<Kind::KK>(a.dtype, m, p, st);
    case GroupedForm::MK: return launch_t<Kind::MK>(a.dtype, m, p, st);
    case GroupedForm::Sum: return launch_t<Kind::MM>(a.dtype, m, p, st);
    case GroupedForm::Mx: return launch_t<Kind::Mx>(a.dtype, m, p, st);
    default: return launch_t<Kind::Nv>(a.dtype, m, p, st);
  }
}

}  // namespace b200q
