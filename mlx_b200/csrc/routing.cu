// Routing to experts (route, its gradient) and the order of rows by group (group_rows).
//
// Of every token's logits l [E]: scores s = softmax(l) or sigmoid(l); keys l, or s + bias where there is a bias.  Groups of
// consecutive experts are ranked by the sum of their best one or two keys (of their scores without a bias) and the first top_groups of
// them stay; of what is left the `top` largest keys are taken, ties to the lowest index.  Weights are the scores of the experts taken,
// divided by their sum if asked for, times `scale`.  An expert whose key is -inf is off: it is never taken, and where too few are on,
// a pair has expert -1, weight 0 and place -1.
//
// A warp has a token, a lane every 32nd expert.  Keys are compared as 32-bit integers of the same order (NaN above everything, 0:
// not to be taken).  The chain of dependent steps is what costs time, so nothing is chosen one by one: of the lanes' best keys the top-th is a bound that
// what is taken has to reach; the few keys that do are put side by side, and each counts those before it.  Which experts a token gets is decided in 64 bits: keys that
// are logits need no rounding, and sums of rounded scores are taken in 32 bits only where neighbours are further apart than the
// rounding can be; else the token's keys are computed again in 64 bits (choose64), for about a token in a thousand.
//
// The pairs (token, choice) are then counting-sorted by expert, stably: every warp has a contiguous range of tokens and counts into a
// histogram of its own, so that a pair's rank among its warp's is known as it is chosen; sums over warps and blocks follow, the latter
// in a second launch where there is more than one block.  No atomics: the order is the same every time.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace b200q {
namespace {

constexpr int kMaxWarps = 32;
constexpr uint32_t kFull = 0xffffffffu;
// Bins of a histogram in memory: whole pieces of 16 bytes.
constexpr __host__ __device__ int pitch(int64_t bins) { return (int)(bins + 3) / 4 * 4; }

// Integers in the order of the numbers; NaN above all, -0 as 0 (the sum with 0 makes them the one NaN and 0 that arithmetic gives).  0 is below every number.
__device__ __forceinline__ uint32_t code32(float f) {
  const int b = __float_as_int(f + 0.0f);
  return (uint32_t)(b ^ (b >> 31 | (int)0x80000000));
}
__device__ __forceinline__ float value32(uint32_t c) { return __uint_as_float(c & 0x80000000u ? c ^ 0x80000000u : ~c); }
__device__ __forceinline__ unsigned long long code64(double f) {
  if (f != f) return ~0ull;
  const unsigned long long b = (unsigned long long)__double_as_longlong(f + 0.0);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double value64(unsigned long long c) {
  if (c == ~0ull) return __longlong_as_double(0x7fffffffffffffffll);
  return __longlong_as_double((long long)(c >> 63 ? c ^ 0x8000000000000000ull : ~c));
}
__device__ __forceinline__ float warp_max(float v) {
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ F warp_sum(F v) {
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// Over the first `lanes` lanes (a power of two), each of which gets the result.
__device__ __forceinline__ float first_max(float v, int lanes) {
  for (int o = 1; o < lanes; o *= 2) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
  return v;
}
__device__ __forceinline__ float first_sum(float v, int lanes) {
  for (int o = 1; o < lanes; o *= 2) v += __shfl_xor_sync(kFull, v, o);
  return v;
}
// How many of n codes (in shared memory; zeros up to a multiple of 4) are before the lane's own, which is the lane-th: larger ones, and equal ones of
// lower lanes.
__device__ __forceinline__ int place_among(const uint32_t* codes, int n, uint32_t own, int lane) {
  int before = 0;
  for (int j = 0; j < n; j += 4) {
    const uint4 c = *reinterpret_cast<const uint4*>(codes + j);
    before += c.x > own || (c.x == own && j < lane);
    before += c.y > own || (c.y == own && j + 1 < lane);
    before += c.z > own || (c.z == own && j + 2 < lane);
    before += c.w > own || (c.w == own && j + 3 < lane);
  }
  return before;
}
// Of the lanes' (code, index) the largest code's, at the lowest index.
__device__ __forceinline__ void warp_best64(unsigned long long& c, int& i) {
  for (int o = 16; o; o >>= 1) {
    const unsigned long long c2 = __shfl_xor_sync(kFull, c, o);
    const int i2 = __shfl_xor_sync(kFull, i, o);
    if (c2 > c || (c2 == c && i2 < i)) { c = c2; i = i2; }
  }
}
__device__ __forceinline__ float sigmoid(float l) { return 1.0f / (1.0f + expf(-l)); }
// sigmoid(l) exp(-far) for far <= 0 and l <= far, or far = 0: scores that would underflow, relative to the largest.
__device__ __forceinline__ float sigmoid_over(float l, float far) {
  const float e = expf(-fabsf(l));
  return (l > 0.0f ? 1.0f : (far < 0.0f ? expf(l - far) : e)) / (1.0f + e);
}
// For keys, whose roundings have room: off by less than a unit of the largest score (the exponential by 2 + 1.2 |x| units, times s (1 - s)).
__device__ __forceinline__ float sigmoid_near(float l) { return __fdividef(1.0f, 1.0f + __expf(-l)); }

struct RouteParams {
  const void* logits;
  const float* bias;
  float* weights;
  int *experts, *sizes, *places, *order;
  uint32_t* hist;      // [blocks][pitch(E + 1)]; one block: not used
  int64_t T, per_block, per_warp;
  int E, top, top2, groups, log_groups, top_groups, best, sigmoid, renormalize;   // top2: top as a power of two, log_groups: both rounded up
  float scale;
};

// One token's experts, in 64 bits: lane j gets the j-th (-1: none).  `row` holds E numbers in shared memory, `few` 96 words.  (The other tokens' warps wait
// for this one at the end of the block, so it has to be quick, too.)
template <typename T, int V>
__device__ __noinline__ int choose64(const RouteParams& p, const T* logits, unsigned long long* row, uint32_t* few, int lane) {
  const int E = p.E;
  double m = -INFINITY, z = 1.0;
  if (!p.sigmoid) {
    for (int i = lane; i < E; i += 32) m = fmax(m, (double)Elem<T>::to_float(logits[i]));
    for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(kFull, m, o));
    z = 0.0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (v * 32 + lane < E) z += exp((double)Elem<T>::to_float(logits[v * 32 + lane]) - m);
    z = warp_sum(z);
  }
  constexpr int U = V < 8 ? V : 8;   // at once: an exponential and a division are chains of some 40 steps each
  for (int v0 = 0; v0 < V; v0 += U) {
    double key[U];
#pragma unroll
    for (int v = 0; v < U; ++v) {
      const int i = (v0 + v) * 32 + lane;
      const double l = i < E ? (double)Elem<T>::to_float(logits[i]) : -INFINITY;
      const double e = exp(p.sigmoid ? -l : l - m);
      key[v] = (p.sigmoid ? 1.0 : e) / (p.sigmoid ? 1.0 + e : z) + (p.bias && i < E ? (double)p.bias[i] : 0.0);
      if (l == -INFINITY) key[v] = -INFINITY;
    }
#pragma unroll
    for (int v = 0; v < U; ++v)
      if ((v0 + v) * 32 + lane < E) row[(v0 + v) * 32 + lane] = key[v] == -INFINITY ? 0 : code64(key[v]);
  }
  __syncwarp();
  uint32_t on = kFull;
  const int size = E / p.groups;
  if (p.groups > 1) {
    const int lanes = 32 >> p.log_groups, group = lane >> (5 - p.log_groups);
    unsigned long long a = 0, b = 0;   // the best two
    if (group < p.groups)
      for (int i = lane & (lanes - 1); i < size; i += lanes) {
        const unsigned long long c = row[group * size + i];
        b = max(b, min(a, c));
        a = max(a, c);
      }
    for (int o = 1; o < lanes; o *= 2) {
      const unsigned long long c = __shfl_xor_sync(kFull, a, o), c2 = __shfl_xor_sync(kFull, b, o);
      b = max(max(b, c2), min(a, c));
      a = max(a, c);
    }
    const unsigned long long rank = p.best == 2 && b != 0 ? code64(value64(a) + value64(b)) : a;
    int before = 0;
    for (int g = 0; g < p.groups; ++g) {
      const unsigned long long c = __shfl_sync(kFull, rank, g * lanes);
      before += c > rank || (c == rank && g < group);
    }
    uint32_t taken = __ballot_sync(kFull, group < p.groups && (lane & (lanes - 1)) == 0 && rank != 0 && before < p.top_groups);
    on = 0;
    for (; taken; taken &= taken - 1) on |= 1u << ((__ffs(taken) - 1) / lanes);
  }
  uint32_t best = 0;   // upper words, which are in the same order
  for (int i = lane; i < E; i += 32) {
    if (!p.bias) {   // among experts the logits decide
      const double l = (double)Elem<T>::to_float(logits[i]);
      row[i] = l == -INFINITY ? 0 : code64(l);
    }
    if (p.groups > 1 && !(on >> (i / size) & 1)) row[i] = 0;
    best = max(best, (uint32_t)(row[i] >> 32));
  }
  uint32_t bound = 1;
  for (int j = 0; j < p.top; ++j) {
    const uint32_t c = __reduce_max_sync(kFull, best);
    if (c == 0) { bound = 1; break; }
    bound = c;
    if (best == c) best = 0;
  }
  unsigned long long* codes = reinterpret_cast<unsigned long long*>(few);
  int n = 0;
  __syncwarp();
  for (int i0 = 0; i0 < E; i0 += 32) {
    const unsigned long long c = i0 + lane < E ? row[i0 + lane] : 0;
    const uint32_t has = __ballot_sync(kFull, (uint32_t)(c >> 32) >= bound);   // (a code's upper word is 0 for no number)
    const int to = n + __popc(has & ((1u << lane) - 1));
    if ((has >> lane & 1) && to < 32) {
      codes[to] = c;
      few[64 + to] = i0 + lane;
    }
    n += __popc(has);
  }
  __syncwarp();
  int mine = -1;
  if (n <= 32) {
    const unsigned long long own = lane < n ? codes[lane] : 0;
    const int index = lane < n ? (int)few[64 + lane] : -1;
    int before = 0;
    for (int j = 0; j < n; ++j) before += codes[j] > own || (codes[j] == own && j < lane);
    __syncwarp();
    if (lane < n) few[before] = index;
    __syncwarp();
    if (lane < min(n, p.top)) mine = (int)few[lane];
    __syncwarp();
    return mine;
  }
  for (int j = 0; j < p.top; ++j) {
    unsigned long long c = 0;
    int at = E;
    for (int i = lane; i < E; i += 32)
      if (row[i] > c) { c = row[i]; at = i; }
    warp_best64(c, at);
    if (c == 0) break;
    if (lane == j) mine = at;
    if (lane == (at & 31)) row[at] = 0;
    __syncwarp();
  }
  return mine;
}

// The same for n candidates, the j-th in lane j, in the order of their indices, among which the experts are (a token in a thousand: 2 us instead of 9, for which
// a call of many tokens waits).
template <typename T>
__device__ __noinline__ int order64(const RouteParams& p, const T* logits, int candidate, int n, uint32_t* few, int lane) {
  double m = 0.0, z = 1.0;
  if (!p.sigmoid) {
    m = -INFINITY;
    for (int i = lane; i < p.E; i += 32) m = fmax(m, (double)Elem<T>::to_float(logits[i]));
    for (int o = 16; o; o >>= 1) m = fmax(m, __shfl_xor_sync(kFull, m, o));
    z = 0.0;
    for (int i = lane; i < p.E; i += 32) z += exp((double)Elem<T>::to_float(logits[i]) - m);
    z = warp_sum(z);
  }
  unsigned long long* codes = reinterpret_cast<unsigned long long*>(few);
  unsigned long long own = 0;
  if (candidate >= 0) {
    const double l = (double)Elem<T>::to_float(logits[candidate]), e = exp(p.sigmoid ? -l : l - m);
    own = code64((p.sigmoid ? 1.0 : e) / (p.sigmoid ? 1.0 + e : z) + (double)p.bias[candidate]);
  }
  codes[lane] = own;
  __syncwarp();
  int before = 0;
  for (int j = 0; j < n; ++j) {
    const unsigned long long c = codes[j];
    before += c > own || (c == own && j < lane);
  }
  if (candidate >= 0) few[64 + before] = candidate;
  __syncwarp();
  const int mine = lane < min(n, p.top) ? (int)few[64 + lane] : -1;
  __syncwarp();
  return mine;
}

// One token: lane j < top gets its j-th expert (-1: none) and the weight.  V = experts per lane; few: 96 words in shared memory.
template <typename T, int V>
__device__ __forceinline__ void route_token(const RouteParams& p, const T* logits, unsigned long long* row, uint32_t* few, int lane, int* expert, float* weight) {
  const int E = p.E;
  float l[V];
  uint32_t u[V];
#pragma unroll
  for (int v = 0; v < V; ++v) l[v] = v * 32 + lane < E ? Elem<T>::to_float(logits[v * 32 + lane]) : -INFINITY;
  float bias[V];   // (before anything is stored: the loads then wait together)
#pragma unroll
  for (int v = 0; v < V; ++v) bias[v] = p.bias && v * 32 + lane < E ? p.bias[v * 32 + lane] : 0.0f;
  const bool sums = p.groups > 1 && p.best == 2;
  const bool scores = p.bias != nullptr || sums;
  float m = -INFINITY, rz = 0.0f;   // softmax: the largest logit, 1 over the sum of exp(l - m)
  if (!p.sigmoid && (scores || !p.renormalize)) {
#pragma unroll
    for (int v = 0; v < V; ++v) m = fmaxf(m, l[v]);
    m = warp_max(m);
    if (m > -INFINITY) {
      float z = 0.0f;
#pragma unroll
      for (int v = 0; v < V; ++v) z += p.renormalize ? __expf(l[v] - m) : expf(l[v] - m);   // (then only keys need it)
      rz = 1.0f / warp_sum(z);
    }
  }
  uint32_t* row32 = reinterpret_cast<uint32_t*>(row);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int i = v * 32 + lane;
    float key = l[v];
    if (scores) {
      const float s = p.sigmoid ? sigmoid_near(l[v]) : __expf(l[v] - m) * rz;
      if (p.bias && i < E) key = l[v] == -INFINITY ? -INFINITY : s + bias[v];
      if (sums && i < E) {
        const float k = p.bias ? key : s;
        row32[i] = key == -INFINITY ? 0 : code32(k);
      }
    }
    u[v] = i >= E || key == -INFINITY ? 0 : code32(key);
    if (p.groups > 1 && !sums && i < E) row32[i] = u[v];
  }
  // how far two keys have to be apart for their rounded forms to be in the right order.  Softmax: 90 half units of the largest score (a sum of up to 37
  // terms, exp, the argument's rounding, a division; 2^-17).  Sigmoid: off by 2^-23 (s (1 - s) (2 + 1.2 |l|) + 2.5 s), at most 3.3 2^-23 (2^-20 for two).
  // And one half unit of each sum with the bias, rounded up.
  const float room = p.sigmoid ? 0x1p-20f : 0x1p-17f * rz;
  bool unsure = false, unsure_group = false;
  if (p.groups > 1) {
    __syncwarp();
    // several lanes scan a group, each from another place on, so that no bank is asked twice; then they put their best two together
    const int size = E / p.groups, lanes = 32 >> p.log_groups, group = lane >> (5 - p.log_groups), each = (size + lanes - 1) / lanes;
    uint32_t rank = 0, b = 0;   // the group's best, the second
    if (group < p.groups) {
      const uint32_t* at = row32 + group * size + (lane & (lanes - 1));
      int k = group % each;
      for (int n = 0; n < each; ++n) {
        const uint32_t c = (k + 1) * lanes <= size || k * lanes + (lane & (lanes - 1)) < size ? at[k * lanes] : 0;
        if (sums) b = max(b, min(rank, c));
        rank = max(rank, c);
        k = k + 1 == each ? 0 : k + 1;
      }
    }
    for (int o = 1; o < lanes; o *= 2) {
      const uint32_t c = __shfl_xor_sync(kFull, rank, o);
      if (sums) b = max(max(b, __shfl_xor_sync(kFull, b, o)), min(rank, c));
      rank = max(rank, c);
    }
    float size_of = fabsf(value32(rank));   // the larger of the two, whose rounding the sum has, however small it is itself
    if (sums && b != 0) {
      size_of = fmaxf(size_of, fabsf(value32(b)));
      rank = code32(value32(rank) + value32(b));
    }
    if (lane < 32) few[lane] = 0;
    __syncwarp();
    if (group < p.groups) {
      few[group] = rank;
      few[32 + group] = __float_as_uint(size_of);
    }
    __syncwarp();
    // lane g looks after group g
    rank = few[lane];
    const int before = place_among(few, p.groups, rank, lane);
    const uint32_t on = __ballot_sync(kFull, rank != 0 && before < p.top_groups);
    if (scores && __popc(on) == p.top_groups) {
      // Where the ranks lie, with their errors, of those that stay and of those that do not: off by `room` and 2^-22 of the larger key (two keys' half units and
      // their sum's, rounded up).  (An infinite sum of finite keys is no answer: its bounds are infinite, too.)
      const float off = rank != 0 ? room + 0x1.2p-22f * __uint_as_float(few[32 + lane]) : 0.0f, r = value32(rank);
      const uint32_t least = __reduce_min_sync(kFull, on >> lane & 1 ? code32(r - off) : kFull);
      const uint32_t most = __reduce_max_sync(kFull, rank != 0 && !(on >> lane & 1) ? code32(r + off) : 0);
      unsure_group = least <= most;
    }
    __syncwarp();
    const uint32_t inv = ((1u << 20) + size - 1) / size;   // i / size for i < 1024
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (!(on >> (((v * 32 + lane) * inv >> 20) & 31) & 1)) u[v] = 0;
  }
  uint32_t best = 0;
  int at = 0;
  auto find = [&] {
    best = 0;
#pragma unroll
    for (int v = 0; v < V; ++v)
      if (u[v] > best) { best = u[v]; at = v; }
  };
  find();
  int mine = -1;
  uint32_t code = 0;   // lane j: the j-th key's
  const int count = p.top + (p.bias ? 1 : 0);   // with a bias the first one left out has to be far enough away, too (lane `top`, if there is one)
  int n = 33, candidate = -1;   // keys that reach the bound; lane j < n: the j-th of them
  if (count <= 32) {
    uint32_t bound = 1, left = best;
    for (int j = 0; j < count; ++j) {   // (equal ones go together: the bound may then be lower than it could)
      const uint32_t c = __reduce_max_sync(kFull, left);
      if (c == 0) { bound = 1; break; }
      bound = c;
      if (left == c) left = 0;
    }
    if (p.bias && bound != 1) {   // with all that could reach it, in 64 bits
      const float b = value32(bound);
      bound = max(1u, min(bound, code32(b - 2 * (room + 0x1p-22f * fabsf(b)))));
    }
    few[lane] = 0;
    __syncwarp();
    n = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {   // in the order of their indices
      const uint32_t has = __ballot_sync(kFull, u[v] >= bound);
      const int to = n + __popc(has & ((1u << lane) - 1));
      if (u[v] >= bound && to < 32) {
        few[to] = u[v];
        few[32 + to] = v * 32 + lane;
      }
      n += __popc(has);
    }
    __syncwarp();
  }
  if (n <= 32) {
    const uint32_t own = few[lane];
    const int before = place_among(few, n, own, lane);
    candidate = lane < n ? (int)few[32 + lane] : -1;
    __syncwarp();
    if (lane < n) {
      few[before] = own;
      few[32 + before] = candidate;
    }
    __syncwarp();
    if (lane < min(n, count)) {
      code = few[lane];
      mine = (int)few[32 + lane];
    }
    __syncwarp();
  } else {   // many of them, or many to take: one by one
    for (int j = 0; j < count; ++j) {
      const uint32_t c = __reduce_max_sync(kFull, best);
      if (c == 0) break;
      const int i = __reduce_min_sync(kFull, best == c ? at * 32 + lane : INT32_MAX);
      if (lane == j) { mine = i; code = c; }
      if (j == 32 && lane == 31) {   // (the 33rd has no lane)
        const float a = value32(code), b = value32(c);
        unsure |= a - b <= room + 0x1p-22f * fmaxf(fabsf(a), fabsf(b));
      }
      if (lane == (i & 31)) {
#pragma unroll
        for (int v = 0; v < V; ++v)
          if (v == i >> 5) u[v] = 0;
        find();
      }
    }
  }
  float lj = mine >= 0 ? Elem<T>::to_float(logits[mine]) : -INFINITY;
  if (p.bias) {
    const float bj = mine >= 0 ? p.bias[mine] : 0.0f;
    const uint32_t c2 = __shfl_down_sync(kFull, code, 1);
    const float l2 = __shfl_down_sync(kFull, lj, 1), b2 = __shfl_down_sync(kFull, bj, 1);
    if (lane < 31 && code != 0 && c2 != 0 && !(lj == l2 && bj == b2)) {   // (the same numbers make the same key)
      const float a = value32(code), b = value32(c2);
      unsure |= a - b <= room + 0x1p-22f * fmaxf(fabsf(a), fabsf(b));
    }
  }
  if (scores && __any_sync(kFull, unsure || unsure_group)) {
    if (n <= 32 && !unsure_group) mine = order64<T>(p, logits, candidate, n, few, lane);
    else mine = choose64<T, V>(p, logits, row, few, lane);
    lj = mine >= 0 ? Elem<T>::to_float(logits[mine]) : -INFINITY;
  }
  if (lane >= p.top) { mine = -1; lj = -INFINITY; }
  float w;
  if (p.renormalize) {   // ratios, which neither the other experts nor small scores touch
    const float top = first_max(lj, p.top2);
    if (p.sigmoid) {
      w = sigmoid_over(lj, fminf(top, 0.0f));
    } else {
      w = expf(lj - top);
    }
    if (mine < 0) w = 0.0f;
    else if (lj != lj) w = lj;
    const float sum = first_sum(w, p.top2);
    w = mine < 0 ? 0.0f : w / sum;
  } else {
    w = p.sigmoid ? sigmoid(lj) : expf(lj - m) * rz;
    if (mine < 0) w = 0.0f;
  }
  *expert = mine;
  *weight = w * p.scale;
}

// Exclusive sums of a[0, n) in shared memory, by the whole block.
__device__ void block_scan(uint32_t* a, int n, uint32_t* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const int each = (n + blockDim.x - 1) / blockDim.x, lo = min(tid * each, n), hi = min(lo + each, n);
  uint32_t sum = 0;
  for (int i = lo; i < hi; ++i) sum += a[i];
  uint32_t before = sum;
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t v = __shfl_up_sync(kFull, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) warp_sums[warp] = before;
  __syncthreads();
  if (warp == 0) {
    uint32_t v = lane < warps ? warp_sums[lane] : 0;
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t q = __shfl_up_sync(kFull, v, o);
      if (lane >= o) v += q;
    }
    warp_sums[lane] = v;
  }
  __syncthreads();
  uint32_t run = before - sum + (warp ? warp_sums[warp - 1] : 0);
  for (int i = lo; i < hi; ++i) {
    const uint32_t v = a[i];
    a[i] = run;
    run += v;
  }
  __syncthreads();
}

// What the sort reads and writes; the last bin, n, is that of pairs without a group.
struct SortParams {
  const void* ids;     // of `bytes` each
  int bytes;
  uint32_t* rank;      // of every pair among its block's of the same group
  uint32_t* hist;      // [blocks][pitch(n + 1)]
  int *sizes, *starts, *places, *order;   // starts and places may be null
  int4* tiles;         // may be null
  int64_t max_tiles, P, per_block;        // pairs
  int n, blocks;
};
__device__ __forceinline__ int bin_of(const SortParams& p, int64_t i) {
  const int64_t e = p.bytes == 8 ? static_cast<const int64_t*>(p.ids)[i] : static_cast<const int*>(p.ids)[i];
  return e >= 0 && e < p.n ? (int)e : p.n;
}
// The bins' sizes, starts and tiles, by one block.  base: the bins' starts; total: their sizes
__device__ void sort_tables(const SortParams& p, const uint32_t* base, uint32_t* total, uint32_t* warp_sums) {
  for (int e = threadIdx.x; e <= p.n; e += blockDim.x) {
    if (e < p.n) p.sizes[e] = (int)total[e];
    if (p.starts) p.starts[e] = (int)base[e];
  }
  if (p.tiles == nullptr) return;
  const int bins = p.n + 1;
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += blockDim.x) total[e] = (total[e] + kAdapterRows - 1) / kAdapterRows;
  __syncthreads();
  block_scan(total, bins, warp_sums);
  const uint32_t starts_of_none = base[p.n], rows = (uint32_t)p.P;
  for (int64_t k = threadIdx.x; k < p.max_tiles; k += blockDim.x) {
    int a = 0, b = bins;   // the last bin whose first tile is at or before k
    while (b - a > 1) {
      const int c = (a + b) / 2;
      if (total[c] <= k) a = c; else b = c;
    }
    const uint32_t end = a < p.n ? base[a + 1] : rows, first = base[a] + (uint32_t)(k - total[a]) * kAdapterRows;
    const int have = first < end ? (int)min(end - first, (uint32_t)kAdapterRows) : 0;
    p.tiles[k] = make_int4(a < p.n ? a : -1, (int)first, have, (int)starts_of_none);
  }
}

// base: where the block's first pair of every bin goes; total: the bins' sizes (block 0 alone needs them, its own base being the bins' starts)
__device__ void sort_finish(const SortParams& p, int block, const uint32_t* base, uint32_t* total, uint32_t* warp_sums) {
  const int64_t lo = block * p.per_block, hi = min(lo + p.per_block, p.P);
  for (int64_t i = lo + threadIdx.x; i < hi; i += blockDim.x) {
    const int e = bin_of(p, i);
    const uint32_t at = p.rank[i] + base[e];
    if (p.places) p.places[i] = e < p.n ? (int)at : -1;
    p.order[at] = e < p.n ? (int)i : (int)(-1 - i);
  }
  if (block == 0) sort_tables(p, base, total, warp_sums);
}

// hist: of every warp of the block [warps][bins].  Becomes the sums before every warp; the block's own sums go to `sums`.
__device__ void sum_over_warps(uint32_t* hist, int bins, uint32_t* sums) {
  const int warps = blockDim.x >> 5;
  for (int e = threadIdx.x; e < bins; e += blockDim.x) {
    uint32_t run = 0;
    for (int w = 0; w < warps; ++w) {
      const uint32_t v = hist[w * bins + e];
      hist[w * bins + e] = run;
      run += v;
    }
    sums[e] = run;
  }
}

// A block has consecutive tokens, a warp a range of them.  Bound by the instructions of a token's dependent steps, HBM is idle: 8192 tokens, 8 of 256 experts in
// groups with a bias, f32, 26 us with cold caches (320 GB/s; bytes would take 1.4) and 13 for the second launch, which begins beside it: 33 together in graph replay, inputs not in L2;
// 16384 tokens, 8 of 128, bf16: 21 and 10, 26 together.  4 tokens: 4 us of latencies.
template <typename T, int V>
__global__ void __launch_bounds__(V > 16 ? 512 : 1024) route_kernel(const RouteParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint32_t warp_sums[32];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, bins = p.E + 1;
  const bool rows = p.bias != nullptr || p.groups > 1;
  unsigned long long* row = reinterpret_cast<unsigned long long*>(smem) + (size_t)warp * (p.E + p.E % 2);
  uint32_t* few = reinterpret_cast<uint32_t*>(smem + (rows ? (size_t)warps * (p.E + p.E % 2) * 8 : 0)) + warp * 96;
  uint32_t* hist = few - warp * 96 + warps * 96;
  uint32_t* mine = hist + (size_t)warp * bins;
  for (int e = lane; e < bins; e += 32) mine[e] = 0;
  __syncwarp();
  const int64_t block_lo = blockIdx.x * p.per_block, block_hi = min(block_lo + p.per_block, p.T);
  const int64_t lo = min(block_lo + warp * p.per_warp, block_hi), hi = min(lo + p.per_warp, block_hi);
  uint32_t* rank = reinterpret_cast<uint32_t*>(p.places);
  for (int64_t t = lo; t < hi; ++t) {
    int e;
    float w;
    route_token<T, V>(p, static_cast<const T*>(p.logits) + t * p.E, row, few, lane, &e, &w);
    const uint32_t none = __ballot_sync(kFull, lane < p.top && e < 0);
    if (lane < p.top) {
      const int bin = e < 0 ? p.E : e;
      const uint32_t r = mine[bin] + (e < 0 ? __popc(none & ((1u << lane) - 1)) : 0);
      p.weights[t * p.top + lane] = w;
      p.experts[t * p.top + lane] = e;
      rank[t * p.top + lane] = r;
    }
    __syncwarp();
    if (lane < p.top) {   // a token's experts are different ones
      if (e >= 0) mine[e] += 1;
      else if (lane == __ffs(none) - 1) mine[p.E] += __popc(none);
    }
    __syncwarp();
  }
  __syncthreads();
  uint32_t* sums = hist + (size_t)warps * bins;
  sum_over_warps(hist, bins, sums);
  __syncthreads();
  for (int64_t i = lo * p.top + lane; i < hi * p.top; i += 32) {
    const int e = p.experts[i];
    rank[i] += mine[e < 0 ? p.E : e];
  }
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < bins; e += blockDim.x) p.hist[(size_t)blockIdx.x * pitch(bins) + e] = sums[e];
    return;
  }
  uint32_t* total = sums + bins;
  for (int e = threadIdx.x; e < bins; e += blockDim.x) total[e] = sums[e];
  __syncthreads();
  block_scan(sums, bins, warp_sums);
  const SortParams s{p.experts, 4, rank, nullptr, p.sizes, nullptr, p.places, p.order, nullptr, 0, p.T * p.top, p.T * p.top, p.E, 1};
  sort_finish(s, 0, sums, total, warp_sums);
}

// More rows: as route_kernel counts its pairs, 32 rows of a warp at a time.  Bound by the latency of ids, ranks and the second launch: 16384 rows of 40 groups 11 us.
__global__ void __launch_bounds__(1024) group_kernel(const SortParams p, int64_t per_warp) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint32_t warp_sums[32];
  asm volatile("griddepcontrol.launch_dependents;");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, bins = p.n + 1;
  uint32_t* hist = reinterpret_cast<uint32_t*>(smem);
  uint32_t* mine = hist + (size_t)warp * bins;
  for (int e = lane; e < bins; e += 32) mine[e] = 0;
  __syncwarp();
  const int64_t block_lo = blockIdx.x * p.per_block, block_hi = min(block_lo + p.per_block, p.P);
  const int64_t lo = min(block_lo + warp * per_warp, block_hi), hi = min(lo + per_warp, block_hi);
  for (int64_t i0 = lo; i0 < hi; i0 += 32) {
    const int64_t i = i0 + lane;
    const int e = i < hi ? bin_of(p, i) : -1;
    const uint32_t same = __match_any_sync(kFull, e);
    if (e >= 0) p.rank[i] = mine[e] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  uint32_t* sums = hist + (size_t)warps * bins;
  sum_over_warps(hist, bins, sums);
  __syncthreads();
  for (int64_t i = lo + lane; i < hi; i += 32) p.rank[i] += mine[bin_of(p, i)];
  if (gridDim.x > 1) {
    for (int e = threadIdx.x; e < bins; e += blockDim.x) p.hist[(size_t)blockIdx.x * pitch(bins) + e] = sums[e];
    return;
  }
  uint32_t* total = sums + bins;
  for (int e = threadIdx.x; e < bins; e += blockDim.x) total[e] = sums[e];
  __syncthreads();
  block_scan(sums, bins, warp_sums);
  sort_finish(p, 0, sums, total, warp_sums);
}

// Up to 128 rows per warp in one block: ids and ranks stay in registers.  (57 rows of 40 groups 3.9 us instead of 4.1, 1024 5.8 instead of 6.4, 4096 9.6 instead of 10.9.)
__global__ void __launch_bounds__(1024) group_few_kernel(const SortParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint32_t warp_sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, bins = p.n + 1, rows = (int)p.P;
  uint32_t* hist = reinterpret_cast<uint32_t*>(smem);
  uint32_t* mine = hist + (size_t)warp * bins;
  const int each = ((rows + warps - 1) / warps + 31) / 32, lo = warp * each * 32 + lane;
  int e[4];
  uint32_t rank[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) e[k] = k < each && lo + k * 32 < rows ? bin_of(p, lo + k * 32) : -1;
  for (int i = lane; i < bins; i += 32) mine[i] = 0;
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (k >= each) break;
    const uint32_t same = __match_any_sync(kFull, e[k]);
    if (e[k] >= 0) rank[k] = mine[e[k]] + __popc(same & ((1u << lane) - 1));
    __syncwarp();
    if (e[k] >= 0 && lane == __ffs(same) - 1) mine[e[k]] += __popc(same);
    __syncwarp();
  }
  __syncthreads();
  uint32_t *base = hist + (size_t)warps * bins, *total = base + bins;
  sum_over_warps(hist, bins, base);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += blockDim.x) total[i] = base[i];
  __syncthreads();
  block_scan(base, bins, warp_sums);
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (e[k] >= 0) {
      const int i = lo + k * 32;
      p.order[rank[k] + mine[e[k]] + base[e[k]]] = e[k] < p.n ? i : -1 - i;
    }
  sort_tables(p, base, total, warp_sums);
}

// The second launch: every block adds up the histograms of those before it, four bins at a time, by threads that share the blocks (148 KB from L2 for 256 bins), and
// places its own pairs.  Bound by these two latencies: 10 to 13 us with cold caches, of which its start lies beside the first launch.
__global__ void __launch_bounds__(1024) place_kernel(const SortParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ uint32_t warp_sums[32];
  const int bins = p.n + 1, quads = pitch(bins) / 4;
  // threads by (part of the blocks, four bins), then by bins
  const int parts = max(1, (int)blockDim.x / quads);
  uint32_t *base = reinterpret_cast<uint32_t*>(smem), *total = base + 4 * quads, *before = total + 4 * quads;
  uint4 *alls = reinterpret_cast<uint4*>(before + 4 * quads), *mines = alls + parts * quads;
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the first launch's results
  for (int i = threadIdx.x; i < parts * quads; i += blockDim.x) {
    const int part = i / quads, e = i % quads;
    uint4 all = make_uint4(0, 0, 0, 0), mine = all;
#pragma unroll 10
    for (int b = part; b < p.blocks; b += parts) {
      const uint4 v = reinterpret_cast<const uint4*>(p.hist)[(size_t)b * quads + e];
      all.x += v.x; all.y += v.y; all.z += v.z; all.w += v.w;
      if (b < (int)blockIdx.x) { mine.x += v.x; mine.y += v.y; mine.z += v.z; mine.w += v.w; }
    }
    alls[i] = all;
    mines[i] = mine;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < bins; e += blockDim.x) {
    uint32_t all = 0, mine = 0;
    for (int k = 0; k < parts; ++k) {
      all += reinterpret_cast<const uint32_t*>(alls)[k * 4 * quads + e];
      mine += reinterpret_cast<const uint32_t*>(mines)[k * 4 * quads + e];
    }
    total[e] = base[e] = all;
    before[e] = mine;
  }
  __syncthreads();
  block_scan(base, bins, warp_sums);
  for (int e = threadIdx.x; e < bins; e += blockDim.x) base[e] += before[e];
  __syncthreads();
  sort_finish(p, blockIdx.x, base, total, warp_sums);
}

// Launched while the first kernel runs, whose last blocks it waits for.
int place(const SortParams& s, cudaStream_t st) {
  const int quads = pitch(s.n + 1) / 4;
  const size_t smem = (size_t)quads * 16 * (3 + 2 * std::max(1, 1024 / quads));
  if (int rc = allow_smem(reinterpret_cast<const void*>(place_kernel), smem)) return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(s.blocks);
  cfg.blockDim = dim3(1024);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  B200Q_CUDA_OK(cudaLaunchKernelEx(&cfg, place_kernel, s));
  B200Q_LAUNCH_OK("place_kernel");
  return B200Q_OK;
}

// ---- the gradient of the weights with respect to the logits: d l = p (g - <g, p>) over all experts, or (renormalized) over those taken, where g = scale dw; sigmoid:
// s (1 - s) g.  A warp has a token and reads its row again for each of three passes, from L1.  16384 tokens, 128 experts, bf16: 8 us in graph replay (1 TB/s of
// logits and gradients; bytes would take 1.4): the chain of three sums over the warp.
struct DlogitsParams {
  const float* dw;
  const void* logits;
  const int* experts;
  void* dlogits;
  int64_t T;
  int E, top, sigmoid, renormalize;
  float scale;
};

template <typename T>
__global__ void __launch_bounds__(256) dlogits_kernel(const DlogitsParams p) {
  const int lane = threadIdx.x & 31;
  const int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (t >= p.T) return;
  const T* l = static_cast<const T*>(p.logits) + t * p.E;
  T* d = static_cast<T*>(p.dlogits) + t * p.E;
  int e = lane < p.top ? p.experts[t * p.top + lane] : -1;
  if (e >= p.E) e = -1;
  const float lj = e >= 0 ? Elem<T>::to_float(l[e]) : -INFINITY;
  const float g = e >= 0 ? p.dw[t * p.top + lane] * p.scale : 0.0f;
  float dj;   // of lane j's expert
  if (!p.sigmoid && !p.renormalize) {
    float m = -INFINITY, z = 0.0f;
    for (int i = lane; i < p.E; i += 32) m = fmaxf(m, Elem<T>::to_float(l[i]));
    m = warp_max(m);
    for (int i = lane; i < p.E; i += 32) z += m > -INFINITY ? expf(Elem<T>::to_float(l[i]) - m) : 0.0f;
    z = warp_sum(z);
    const float rz = z > 0.0f || z != z ? 1.0f / z : 0.0f;
    const float pj = e >= 0 ? expf(lj - m) * rz : 0.0f;
    const float mean = warp_sum(g * pj);
    dj = pj * (g - mean);
    for (int i = lane; i < p.E; i += 32) {
      const float li = Elem<T>::to_float(l[i]);
      d[i] = Elem<T>::from_float(li > -INFINITY || li != li ? -expf(li - m) * rz * mean : 0.0f);
    }
  } else {
    float q = 0.0f;
    if (p.renormalize) {
      const float top = warp_max(lj);
      if (p.sigmoid) q = sigmoid_over(lj, fminf(top, 0.0f));
      else q = expf(lj - top);
      if (e < 0) q = 0.0f;
      else if (lj != lj) q = lj;
      const float sum = warp_sum(q);
      q = e < 0 ? 0.0f : q / sum;
      dj = q * (g - warp_sum(g * q));
    } else {
      dj = sigmoid(lj) * g;
    }
    if (p.sigmoid) dj *= sigmoid(-lj);
    for (int i = lane; i < p.E; i += 32) d[i] = Elem<T>::from_float(0.0f);
  }
  __syncwarp();   // the row's stores before those of its experts
  if (e >= 0) d[e] = Elem<T>::from_float(dj);
}

template <typename T>
int launch_route(const RouteParams& p, int blocks, int warps, cudaStream_t st) {
  const bool rows = p.bias != nullptr || p.groups > 1;
  const size_t smem = (rows ? (size_t)warps * (p.E + p.E % 2) * 8 : 0) + warps * 384 + (size_t)(warps + 2) * (p.E + 1) * 4;
  auto go = [&](auto kern) {
    if (int rc = allow_smem(reinterpret_cast<const void*>(kern), smem)) return rc;
    kern<<<blocks, warps * 32, smem, st>>>(p);
    B200Q_LAUNCH_OK("route_kernel");
    return (int)B200Q_OK;
  };
  if (p.E <= 32) return go(route_kernel<T, 1>);
  if (p.E <= 64) return go(route_kernel<T, 2>);
  if (p.E <= 128) return go(route_kernel<T, 4>);
  if (p.E <= 256) return go(route_kernel<T, 8>);
  if (p.E <= 512) return go(route_kernel<T, 16>);
  return go(route_kernel<T, 32>);
}

// Blocks and warps: up to 16 tokens in one block, one launch (to 24 of up to 128 experts, to 48 of up to 32); else 8 tokens or more per block, one block of up to 32 warps per SM,
// whose histograms the second launch reads.  (One block / several, us: 2 of 8 experts, 16 tokens 5.8 / 9.3, 48 8.4 / 9.6, 64 9.8 / 9.7; 8 of 128, 24 tokens 7.7 / 8.0, 32 9.3 / 8.1;
// 8 of 256 in groups, 16 tokens 9.4 / 10.4, 24 11.6 / 10.5: many experts share one SM's instructions.)
struct Split { int blocks, warps; int64_t per_block, per_warp; };
Split route_split(int64_t T, int64_t E) {
  Split s{};
  const int most = E > 512 ? 16 : kMaxWarps;
  s.blocks = T <= (E <= 32 ? 48 : (E <= 128 ? 24 : 16)) ? 1 : (int)std::min<int64_t>((T + 7) / 8, 148);
  s.per_block = (T + s.blocks - 1) / s.blocks;
  s.blocks = (int)((T + s.per_block - 1) / s.per_block);
  s.warps = (int)std::min<int64_t>(s.per_block, most);
  s.per_warp = (s.per_block + s.warps - 1) / s.warps;
  s.warps = (int)((s.per_block + s.per_warp - 1) / s.per_warp);
  return s;
}
// Up to 4096 rows in one block.  (40 groups, one block / several, us: 4096 rows 9.6 / 11.0, 8192 16.6 / 10.9.)
Split group_split(int64_t T, int64_t n) {
  Split s{};
  s.warps = n <= 512 ? 32 : (n <= 1024 ? 16 : 8);   // their histograms share 132 KB at most
  s.blocks = T <= 4096 ? 1 : (int)std::min<int64_t>((T + 2047) / 2048, 148);
  if (s.blocks == 1) s.warps = (int)std::max<int64_t>(1, std::min<int64_t>(s.warps, (T + 31) / 32));
  s.per_block = (T + s.blocks - 1) / s.blocks;
  s.per_warp = ((s.per_block + s.warps - 1) / s.warps + 31) / 32 * 32;
  s.blocks = (int)((T + s.per_block - 1) / s.per_block);
  return s;
}

constexpr int64_t kMostPairs = INT32_MAX;   // places are 32-bit integers
constexpr int64_t kMostExperts = 1024, kMostTop = 32, kMostGroups = 32, kMostRowGroups = 4096;

int check_route(const char* tag, int dtype, int64_t T, int64_t E, int64_t top, int scoring) {
  if (dtype != B200Q_F32 && dtype != B200Q_F16 && dtype != B200Q_BF16)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unsupported dtype code %d", tag, dtype);
  if (T < 0 || E < 1) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] no experts, or a negative number of tokens.", tag);
  if (top < 1 || top > E) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] cannot take %lld of %lld experts.", tag, (long long)top, (long long)E);
  if (scoring != B200Q_SOFTMAX && scoring != B200Q_SIGMOID) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] unknown scoring code %d", tag, scoring);
  if (E > kMostExperts || top > kMostTop || T > kMostPairs / top)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than %lld experts, %lld of them per token or 2^31 - 1 pairs.", tag,
                (long long)kMostExperts, (long long)kMostTop);
  return B200Q_OK;
}

}  // namespace
}  // namespace b200q

using namespace b200q;

extern "C" size_t b200q_route_workspace_bytes(int64_t T, int64_t E, int64_t top) {
  if (T <= 0 || E <= 0 || top <= 0) return 0;
  const Split s = route_split(T, E);
  return s.blocks == 1 ? 0 : (size_t)s.blocks * pitch(E + 1) * 4;
}

extern "C" int b200q_route(const void* logits, int dtype, int64_t T, int64_t E, int64_t top, int scoring, const float* bias, int64_t groups,
                           int64_t top_groups, int group_best, int renormalize, float scale, float* weights, int32_t* experts, int32_t* sizes,
                           int32_t* places, int32_t* order, void* ws, size_t ws_bytes, void* stream) {
  const char* tag = "route_experts";
  if (int rc = check_route(tag, dtype, T, E, top, scoring)) return rc;
  if (groups < 1 || E % groups != 0 || top_groups < 1 || top_groups > groups)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] cannot take %lld of %lld groups of %lld experts.", tag, (long long)top_groups, (long long)groups, (long long)E);
  if (top > E / groups * top_groups)
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] cannot take %lld experts out of %lld groups of %lld.", tag, (long long)top, (long long)top_groups, (long long)(E / groups));
  if (group_best != 1 && group_best != 2) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] a group is ranked by its best 1 or 2 experts, not %d.", tag, group_best);
  if (groups > kMostGroups) return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than %lld groups.", tag, (long long)kMostGroups);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!sizes) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (!on_boundaries({logits}, dtype_size(dtype)) || !on_boundaries({bias, weights, experts, sizes, places, order}, 4))
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  if (T == 0) {
    B200Q_CUDA_OK(cudaMemsetAsync(sizes, 0, (size_t)E * 4, st));
    return B200Q_OK;
  }
  if (!logits || !weights || !experts || !places || !order) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  const Split s = route_split(T, E);
  const size_t need = b200q_route_workspace_bytes(T, E, top);
  if (need > 0 && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16 != 0))
    return fail(B200Q_ERR_WORKSPACE, "[%s] an aligned workspace of %zu bytes required, %zu given", tag, need, ws ? ws_bytes : (size_t)0);
  if (top_groups == groups) groups = top_groups = 1;   // nothing to leave out
  int log_groups = 0, top2 = 1;
  while (1 << log_groups < groups) ++log_groups;
  while (top2 < top) top2 *= 2;
  const RouteParams p{logits, bias, weights, experts, sizes, places, order, static_cast<uint32_t*>(ws), T, s.per_block, s.per_warp,
                      (int)E, (int)top, top2, (int)groups, log_groups, (int)top_groups, group_best, scoring == B200Q_SIGMOID, renormalize != 0, scale};
  const ScratchLock lock(ws);
  int rc = dtype == B200Q_F32 ? launch_route<float>(p, s.blocks, s.warps, st)
                              : (dtype == B200Q_F16 ? launch_route<__half>(p, s.blocks, s.warps, st) : launch_route<__nv_bfloat16>(p, s.blocks, s.warps, st));
  if (rc || s.blocks == 1) return rc;
  const SortParams sp{experts, 4, reinterpret_cast<uint32_t*>(places), static_cast<uint32_t*>(ws), sizes, nullptr, places, order, nullptr, 0, T * top, s.per_block * top, (int)E, s.blocks};
  return place(sp, st);
}

extern "C" int b200q_route_dlogits(const float* dw, const void* logits, int dtype, const int32_t* experts, int64_t T, int64_t E, int64_t top, int scoring,
                                   int renormalize, float scale, void* dlogits, void* stream) {
  const char* tag = "route_experts";
  if (int rc = check_route(tag, dtype, T, E, top, scoring)) return rc;
  if (T == 0) return B200Q_OK;
  if (!dw || !logits || !experts || !dlogits) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (!on_boundaries({logits, dlogits}, dtype_size(dtype)) || !on_boundaries({dw, experts}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  const DlogitsParams p{dw, logits, experts, dlogits, T, (int)E, (int)top, scoring == B200Q_SIGMOID, renormalize != 0, scale};
  const unsigned blocks = (unsigned)((T + 7) / 8);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == B200Q_F32) dlogits_kernel<float><<<blocks, 256, 0, st>>>(p);
  else if (dtype == B200Q_F16) dlogits_kernel<__half><<<blocks, 256, 0, st>>>(p);
  else dlogits_kernel<__nv_bfloat16><<<blocks, 256, 0, st>>>(p);
  B200Q_LAUNCH_OK("dlogits_kernel");
  return B200Q_OK;
}

extern "C" int64_t b200q_group_rows_tiles(int64_t T, int64_t n) {
  if (T <= 0 || n < 0) return 0;
  return std::min(T, n + 1) + T / kAdapterRows;
}
namespace {
bool few_rows(int64_t T, const Split& s) { return s.blocks == 1 && T <= 128 * s.warps; }
}  // namespace
extern "C" size_t b200q_group_rows_workspace_bytes(int64_t T, int64_t n) {
  if (T <= 0 || n < 0) return 0;
  const Split s = group_split(T, n);
  if (few_rows(T, s)) return 0;
  return (size_t)pitch(T) * 4 + (s.blocks == 1 ? 0 : (size_t)s.blocks * pitch(n + 1) * 4);
}

extern "C" int b200q_group_rows(const void* ids, int id_bytes, int64_t T, int64_t n, int32_t* sizes, int32_t* starts, int32_t* order, int32_t* tiles,
                                void* ws, size_t ws_bytes, void* stream) {
  const char* tag = "group_rows";
  if (T < 0 || n < 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] negative dimension.", tag);
  if ((id_bytes != 4 && id_bytes != 8) || (ids && reinterpret_cast<uintptr_t>(ids) % id_bytes != 0))
    return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] ids are aligned 4- or 8-byte integers", tag);
  if (T > (1 << 30) || n > kMostRowGroups)
    return fail(B200Q_ERR_UNSUPPORTED, "[%s] No implementation for problem shape: more than 2^30 rows or %lld groups.", tag, (long long)kMostRowGroups);
  if (!starts || (n > 0 && !sizes)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (!on_boundaries({sizes, starts, order}, 4)) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] misaligned pointer", tag);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (T == 0) {
    if (n > 0) B200Q_CUDA_OK(cudaMemsetAsync(sizes, 0, (size_t)n * 4, st));
    B200Q_CUDA_OK(cudaMemsetAsync(starts, 0, (size_t)(n + 1) * 4, st));
    return B200Q_OK;
  }
  if (!ids || !order || !tiles) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] null pointer", tag);
  if (reinterpret_cast<uintptr_t>(tiles) % 16 != 0) return fail(B200Q_ERR_INVALID_ARGUMENT, "[%s] tiles must be 16-byte aligned", tag);
  const size_t need = b200q_group_rows_workspace_bytes(T, n);
  if (need > 0 && (!ws || ws_bytes < need || reinterpret_cast<uintptr_t>(ws) % 16 != 0))
    return fail(B200Q_ERR_WORKSPACE, "[%s] an aligned workspace of %zu bytes required, %zu given", tag, need, ws ? ws_bytes : (size_t)0);
  const Split s = group_split(T, n);
  uint32_t* rank = static_cast<uint32_t*>(ws);
  const SortParams p{ids, id_bytes, rank, need ? rank + pitch(T) : nullptr, sizes, starts, nullptr, order, reinterpret_cast<int4*>(tiles), b200q_group_rows_tiles(T, n), T, s.per_block, (int)n, s.blocks};
  const size_t smem = (size_t)(s.warps + 2) * (n + 1) * 4;
  if (few_rows(T, s)) {
    if (int rc = allow_smem(reinterpret_cast<const void*>(group_few_kernel), smem)) return rc;
    group_few_kernel<<<1, s.warps * 32, smem, st>>>(p);
    B200Q_LAUNCH_OK("group_few_kernel");
    return B200Q_OK;
  }
  const ScratchLock lock(ws);
  if (int rc = allow_smem(reinterpret_cast<const void*>(group_kernel), smem)) return rc;
  group_kernel<<<s.blocks, s.warps * 32, smem, st>>>(p, s.per_warp);
  B200Q_LAUNCH_OK("group_kernel");
  return s.blocks == 1 ? B200Q_OK : place(p, st);
}
