// sequence_probs.hip -- what a policy's logits are asked for. Per row and part of a move, over the
// entries that are allowed (not masked, and not -inf):
//
//   m = max x,  Z = sum exp(x - m),  l_j = x_j - m - log Z,  p_j = exp(l_j)
//   log probability of the choice l_c,  entropy H = -sum p l = log Z - sum exp(x - m) (x - m) / Z
//   the k largest l, ties to the lower index
//   dx_j = dl (1[j = c] - p_j) - dH p_j (l_j + H)
//
// A dozen operations an entry that is read once (and written once in the gradient): bound by
// traffic where there are many, by latency where there are few. One pass: a thread keeps the
// maximum, Z and the entropy's sum of what it has seen, and scales both when the maximum moves.
// Sums are float32; m and log Z are kept apart, so that l is as exact as x is.
//
// Measured (us; a large copy reaches 4.8 TB/s):
//   8,192 rows of 50,000 bf16 entries           forward 175 (4.7 TB/s), gradient 307 (5.3 TB/s)
//   2,000 rows of 32,003 floats                 41 (4.6 TB/s), 88 (5.1 TB/s)
//   81,920 rows of parts of 127, 127, 6, 6      31, 37: half of the vector units' time, and short of wavefronts
//                                               (3.5 a SIMD) to cover the loads' latency with
//   64 rows of parts of 10, 10, 3, 3            4: the launch
//   64 rows of 131,072 bf16 entries, top 20     14 + 6; one row of 65,537 floats, top 5, 8 + 6: two launches and
//                                               the latency inside of them
#include <algorithm>
#include <type_traits>

#include "sequence.h"

#define ASTRA_SRC_NAME "sequence_probs.hip"

namespace astra_seq {
namespace {

constexpr int kParts = ASTRA_SEQ_MAX_PARTS;
static_assert(ASTRA_SEQ_MAX_TOP <= kWave, "a lane for each of the largest");
constexpr int V = 8;             // entries a lane takes at a time
constexpr int kStats = 3;        // m, log Z, H of a row and part

struct ProbArgs {
  const void *logits;
  const uint8_t *mask;
  const void *choice;
  float *log_prob, *entropy, *stats, *top_log_prob;
  int64_t *top_index;
  const float *dlog_prob, *dentropy;
  void *dlogits;
  float *pieces;       // what each piece of a larger part saw,
  uint64_t *lists;     // and its largest entries
  int64_t R, stride, mask_stride;
  int32_t W, parts, top, wide_choice;
  int32_t narrow;              // parts up to here are a group of lanes' work, larger ones workgroups'
  bool cut;                    // whether larger parts go through in pieces,
  int32_t piece;               // of so many entries
  int32_t block_rows;          // rows of a workgroup that has all their parts
  int32_t begin[kParts + 1];   // of each part in a row
  int64_t block[kParts + 1];   // the first workgroup of each part in this launch
};

// The part that a workgroup works on, and its number within that part.
__device__ __forceinline__ int part_of(const ProbArgs &a, int64_t *n) {
  int p = 0;
  while (p + 1 < a.parts && (int64_t)blockIdx.x >= a.block[p + 1]) ++p;
  *n = blockIdx.x - a.block[p];
  return p;
}

// The choice of a row and part: -1 for none, and beyond every part for what is in none.
__device__ __forceinline__ int choice_of(const ProbArgs &a, int64_t unit, int size) {
  if (!a.choice) return 0;
  const int64_t c = a.wide_choice ? ((const int64_t *)a.choice)[unit] : (int64_t)((const int32_t *)a.choice)[unit];
  return c == -1 ? -1 : c >= 0 && c < size ? (int)c : INT32_MAX;
}

// V neighbouring entries from any address.
template <class T>
struct Loose {
  typedef T Raw __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
typedef uint8_t LooseMask __attribute__((ext_vector_type(V), aligned(1)));

// Entries i .. i + V - 1 of a part as they lie in memory, the first of them entry `from` of the part, and a
// byte for each that is not 0 for those of them that are in the part and allowed. `room` is what there
// is to read from the part's begin on, to the end of the row: the last lanes of a row start a little
// before their entries rather than take them one by one.
template <class T>
struct Entries {
  typename Loose<T>::Raw raw;
  uint64_t allowed;
  int from;
  __device__ __forceinline__ void load(const T *x, const uint8_t *mask, int i, int size, int room) {
    from = min(i, room - V);
    allowed = 0;
    if (i < size) {
      raw = *reinterpret_cast<const typename Loose<T>::Raw *>(x + from);
      allowed = ~0ull << 8 * (i - from) & ~0ull >> 8 * (V - min(V, size - from));
      if (mask) allowed &= __builtin_bit_cast(uint64_t, *reinterpret_cast<const LooseMask *>(mask + from));
    }
  }
  // -inf for those that are not allowed
  __device__ __forceinline__ void values(float (&v)[V]) const {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (uint8_t)(allowed >> 8 * j) ? (float)raw[j] : -INFINITY;
  }
};
// The same in rows of less than V entries.
template <class T>
__device__ __forceinline__ void short_entries(const T *x, const uint8_t *mask, int size, float (&v)[V]) {
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = j < size && (!mask || mask[j]) ? (float)x[j] : -INFINITY;
}
template <class T>
__device__ __forceinline__ float entry(const T *x, const uint8_t *mask, int i) {
  return !mask || mask[i] ? (float)x[i] : -INFINITY;
}

// What has been seen of a part: its maximum, and sums of t = exp(x - most) and t (x - most).
struct Seen {
  float most, z, s;
};

// exp(d); d is not positive, or not finite
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// The same sums relative to a larger maximum (what was seen of nothing is zero).
__device__ __forceinline__ Seen moved_to(const Seen &a, float most) {
  const float d = fmaxf(a.most - most, -1000.f), f = exp_of(d);  // (as in see)
  const bool none = a.most == -INFINITY;
  return {most, none ? a.z : a.z * f, none ? a.s : (a.s + a.z * d) * f};
}

// Entries of which none is larger than the maximum seen.
__device__ __forceinline__ void add(Seen &a, const float (&x)[V]) {
  const float base = a.most == -INFINITY ? 0.f : a.most;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float d = x[j] - base, t = exp_of(d);
    a.z += t;
    a.s = fmaf(t, fmaxf(d, -1000.f), a.s);  // (t is zero far before that; -inf times it would be NaN)
  }
}

__device__ __forceinline__ void see(Seen &a, const float (&x)[V]) {
  float most = x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) most = fmaxf(most, x[j]);
  if (most > a.most) a = moved_to(a, most);
  add(a, x);
}

struct Result {
  float most, log_z, entropy;
};
__device__ __forceinline__ Result result_of(const Seen &a) {
  if (a.most == -INFINITY && a.z == 0.f) return {0.f, 0.f, 0.f};  // nothing is allowed
  const float log_z = logf(a.z);
  return {a.most == -INFINITY ? 0.f : a.most, log_z, log_z - a.s / a.z};
}

// The maximum over N neighbouring lanes, in each of them (as lanes_sum).
template <int CTRL>
__device__ __forceinline__ float swapped(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
template <int N>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (N >= 2) v = fmaxf(v, swapped<kSwap1>(v));
  if constexpr (N >= 4) v = fmaxf(v, swapped<kSwap2>(v));
  if constexpr (N >= 8) v = fmaxf(v, swapped<kMirror8>(v));
  if constexpr (N >= 16) v = fmaxf(v, swapped<kMirror16>(v));
  if constexpr (N >= 32) {
    const Pair p = rows_of_half(v);
    v = fmaxf(p.first, p.second);
  }
  if constexpr (N >= 64) {
    const Pair p = halves(v);
    v = fmaxf(p.first, p.second);
  }
  return v;
}

// ------------------------------------------------------------------------ the largest

// Entries in order: a larger key is a larger entry, or an equal one before it; 0 is none.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  x += 0.f;  // (-0 is as large as 0)
  const uint32_t b = __builtin_bit_cast(uint32_t, x);
  const uint32_t up = b >> 31 ? ~b : b | 0x80000000u;
  return x > -INFINITY ? (uint64_t)up << 32 | (uint32_t)~i : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t up = (uint32_t)(key >> 32);
  return __builtin_bit_cast(float, up >> 31 ? up & 0x7fffffffu : ~up);
}
__device__ __forceinline__ int64_t index_of(uint64_t key) { return (int64_t)(uint32_t)~(uint32_t)key; }

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)v, lane), hi = __builtin_amdgcn_readlane((uint32_t)(v >> 32), lane);
  return (uint64_t)hi << 32 | lo;
}

// v of lane ^ X, by data-parallel moves and row swaps.
template <int X>
__device__ __forceinline__ uint32_t across(uint32_t v, int lane) {
  constexpr int kReverse4 = 0x1B, kTurn8 = 0x128;  // quad_perm 3,2,1,0; row_ror:8
  const auto dpp = [](uint32_t u, auto ctrl) __attribute__((always_inline)) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)u, decltype(ctrl)::value, 0xf, 0xf, false);
  };
  if constexpr ((X & 3) == 3) v = dpp(v, std::integral_constant<int, kReverse4>());
  if constexpr ((X & 3) == 1) v = dpp(v, std::integral_constant<int, kSwap1>());
  if constexpr ((X & 3) == 2) v = dpp(v, std::integral_constant<int, kSwap2>());
  if constexpr (X & 4) v = dpp(dpp(v, std::integral_constant<int, kMirror8>()), std::integral_constant<int, kReverse4>());
  if constexpr (X & 8) v = dpp(v, std::integral_constant<int, kTurn8>());
  if constexpr (X & 16) {
    const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t even = p[0], odd = p[1];
    v = lane & 16 ? even : odd;
  }
  if constexpr (X & 32) {
    const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    const uint32_t low = p[0], high = p[1];
    v = lane & 32 ? low : high;
  }
  return v;
}
template <int X>
__device__ __forceinline__ uint64_t across(uint64_t v, int lane) {
  return (uint64_t)across<X>((uint32_t)(v >> 32), lane) << 32 | across<X>((uint32_t)v, lane);
}

__device__ __forceinline__ uint64_t larger(uint64_t v, uint64_t w) { return v > w ? v : w; }

// One round of a sorting network: lanes i and i ^ X, of which the lower one gets the larger value.
// The partners differ in X's highest bit.
template <int X, class K>
__device__ __forceinline__ void exchange(K &v, int lane) {
  constexpr int kHigh = X >= 32 ? 32 : X >= 16 ? 16 : X >= 8 ? 8 : X >= 4 ? 4 : X >= 2 ? 2 : 1;
  const K o = across<X>(v, lane);
  const bool more = v > o, lower = !(lane & kHigh);
  v = more == lower ? v : o;
}
// Rounds that sort (falling) what rises and falls once within S lanes: halves, quarters, ...
template <int S, class K>
__device__ __forceinline__ void settle(K &v, int lane) {
  if constexpr (S >= 64) exchange<32>(v, lane);
  if constexpr (S >= 32) exchange<16>(v, lane);
  if constexpr (S >= 16) exchange<8>(v, lane);
  if constexpr (S >= 8) exchange<4>(v, lane);
  if constexpr (S >= 4) exchange<2>(v, lane);
  exchange<1>(v, lane);
}
// A bitonic sort of the wavefront's values (Batcher's), falling: sorted groups of lanes are joined
// by comparing one with the other's mirror image.
template <class K>
__device__ __forceinline__ void sort(K &v, int lane) {
  exchange<1>(v, lane);
  exchange<3>(v, lane);
  settle<2>(v, lane);
  exchange<7>(v, lane);
  settle<4>(v, lane);
  exchange<15>(v, lane);
  settle<8>(v, lane);
  exchange<31>(v, lane);
  settle<16>(v, lane);
  exchange<63>(v, lane);
  settle<32>(v, lane);
}
// The 64 largest of two sorted lists, sorted.
__device__ __forceinline__ uint64_t joined(uint64_t v, uint64_t w, int lane) {
  w = across<63>(w, lane);
  v = larger(v, w);
  settle<64>(v, lane);
  return v;
}

// LDS that only this wavefront uses: what was written before is there to be read.
__device__ __forceinline__ void in_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A wavefront's largest entries, sorted, of those in its lanes' registers. The top-th largest of
// the lanes' maxima is a bound below them all: what reaches it (some 25 of 2,048 entries for the top
// 20, if they are in no order) is gathered in LDS and sorted 64 at a time.
// `from`: the indices of a lane's vectors.
template <int C>
__device__ __forceinline__ uint64_t largest_of(const float (&v)[C][V], const int (&from)[C], float lane_max, int top, uint64_t *gather, int lane) {
  uint32_t bound = (uint32_t)(key_of(lane_max, 0) >> 32);
  sort(bound, lane);
  bound = __builtin_amdgcn_readlane(bound, top - 1);
  const float least = bound ? value_of((uint64_t)bound << 32) : -INFINITY;
  uint64_t best = 0, last = 0;
  int have = 0;
  const auto take = [&](int n) __attribute__((always_inline)) {
    in_order();
    uint64_t k = lane < n ? gather[lane] : 0;
    const uint64_t rest = gather[64 + lane];
    in_order();
    gather[lane] = rest;
    if (!__ballot(k > last)) return;
    sort(k, lane);
    best = joined(best, k, lane);
    last = lane_of(best, top - 1);
  };
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if (!__ballot(v[c][j] >= least)) continue;
      const uint64_t key = key_of(v[c][j], from[c] + j);
      const bool in = key > last && v[c][j] >= least;
      const uint64_t who = __ballot(in);
      if (!who) continue;
      if (in) gather[have + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0))] = key;
      have += __popcll(who);
      if (have >= 64) {
        take(64);
        have -= 64;
      }
    }
  if (have) take(have);
  return best;
}

__device__ __forceinline__ void store_top(const ProbArgs &a, int64_t at, bool some, float x, int64_t index, const Result &r) {
  a.top_log_prob[at] = some ? x - r.most - r.log_z : -INFINITY;
  a.top_index[at] = some ? index : -1;
}
__device__ __forceinline__ void store_top(const ProbArgs &a, int64_t at, uint64_t key, const Result &r) {
  store_top(a, at, key != 0, value_of(key), index_of(key), r);
}

// The log probability of choice c, entry x.
__device__ __forceinline__ float log_prob_of(int c, float x, const Result &r) {
  return c == -1 ? 0.f : c == INT32_MAX ? NAN : x - r.most - r.log_z;
}

// ------------------------------------------------------------------------- smaller parts

// A group of lanes has one part of one row in registers; results go to LDS, from where whole rows
// of them are written.
constexpr int kUnits = 1024;  // rows by parts of a workgroup
struct Out {
  float log_prob[kUnits], entropy[kUnits], stats[kUnits * kStats];
};
// One part of the workgroup's rows: G lanes a row, V entries each, C times.
template <class T, int G, int C, bool TOP>
__device__ void narrow_part(const ProbArgs &a, Out &out, uint64_t *gather, int part, int64_t first, int rows, int turn) {
  constexpr int kEach = kWave / G;
  const int begin = a.begin[part], size = a.begin[part + 1] - begin, lane = threadIdx.x % kWave, j = lane % G;
  const T *logits = (const T *)a.logits + first * a.stride + begin;
  const uint8_t *masks = a.mask ? a.mask + first * a.mask_stride + begin : nullptr;
  for (int task = turn; task * kEach < rows; task += 4) {
    const int local = task * kEach + lane / G;
    const bool in = local < rows;
    const int64_t unit = (first + local) * a.parts + part;
    const T *x = logits + (in ? local : 0) * a.stride;
    const uint8_t *mask = masks ? masks + (in ? local : 0) * a.mask_stride : nullptr;
    Entries<T> e[C];
    const bool tiny = G == 1 && a.W < V;
    if (!tiny) {
#pragma unroll
      for (int k = 0; k < C; ++k) e[k].load(x, mask, (k * G + j) * V, in ? size : 0, a.W - begin);
    }
    // (all on their way before the first is waited for)
    const int c = in ? choice_of(a, unit, size) : -1;
    const float x_c = c >= 0 && c < size ? entry(x, mask, c) : -INFINITY;
    float v[C][V], most = -INFINITY;
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (tiny) {
        short_entries(x, mask, c == -1 ? 0 : size, v[k]);
        e[k].from = 0;
      } else {
        if (c == -1) e[k].allowed = 0;
        e[k].values(v[k]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) most = fmaxf(most, v[k][i]);
    }
    Seen s{lanes_max<G>(most), 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < C; ++k) add(s, v[k]);
    s.z = lanes_sum<G>(s.z);
    s.s = lanes_sum<G>(s.s);
    const Result r = result_of(s);
    if (in && j == 0) {
      const int n = local * a.parts + part;
      out.log_prob[n] = log_prob_of(c, x_c, r);
      out.entropy[n] = c == -1 ? 0.f : r.entropy;
      out.stats[n * kStats] = r.most;
      out.stats[n * kStats + 1] = r.log_z;
      out.stats[n * kStats + 2] = r.entropy;
    }
    // the largest one after the other, or by sorting (20,000 rows of 1,000, us: 3 of them 34 / 42, 7 49 / 43, 20
    // 99 / 48, 64 273 / 80; of 400 5 of them 27 / 32, 7 32 / 32; of 2,000 3 of them 50 / 54, 7 72 / 54)
    if (TOP && G == kWave && a.top > 6) {
      int from[C];
#pragma unroll
      for (int k = 0; k < C; ++k) from[k] = e[k].from;
      const uint64_t best = largest_of(v, from, most, a.top, gather, lane);
      if (in && lane < a.top) store_top(a, unit * a.top + lane, best, r);
    } else if constexpr (TOP) {
      for (int t = 0; t < a.top; ++t) {
        float large = -INFINITY;
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) large = fmaxf(large, v[k][i]);
        large = lanes_max<G>(large);
        uint32_t index = ~0u;  // the first of them
#pragma unroll
        for (int k = C - 1; k >= 0; --k)
#pragma unroll
          for (int i = V - 1; i >= 0; --i) index = v[k][i] == large ? e[k].from + i : index;
        if constexpr (G >= 2) index = min(index, across<1>(index, lane));
        if constexpr (G >= 4) index = min(index, across<2>(index, lane));
        if constexpr (G >= 8) index = min(index, across<4>(index, lane));
        if constexpr (G >= 16) index = min(index, across<8>(index, lane));
        if constexpr (G >= 32) index = min(index, across<16>(index, lane));
        if constexpr (G >= 64) index = min(index, across<32>(index, lane));
#pragma unroll
        for (int k = 0; k < C; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) v[k][i] = e[k].from + i == (int)index ? -INFINITY : v[k][i];
        if (in && j == 0) store_top(a, unit * a.top + t, large > -INFINITY, large, index, r);
      }
    }
  }
}

// A workgroup has block_rows rows, its wavefronts take turns with them. BIG: with parts of more than 512
// entries, whose registers the others do without (168 and 72 with the largest: 81,920 rows of 400, the
// likeliest, 71 and 43 us); three workgroups a CU, or four and 11 to 77 spilled (2,000 entries 113 and 128 us).
template <class T, bool TOP, bool BIG>
__global__ __launch_bounds__(256, BIG && TOP ? 3 : 1) void narrow_forward_kernel(ProbArgs a) {
  __shared__ Out out;
  __shared__ uint64_t gather[TOP ? 4 : 1][128];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t first = (int64_t)blockIdx.x * a.block_rows;
  const int rows = (int)min((int64_t)a.block_rows, a.R - first);
  for (int part = 0; part < a.parts; ++part) {
    const int size = a.begin[part + 1] - a.begin[part], turn = (wave + part) & 3;
    if (size > a.narrow) continue;
    if (size <= V)
      narrow_part<T, 1, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (size <= 2 * V)
      narrow_part<T, 2, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (size <= 4 * V)
      narrow_part<T, 4, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (size <= 8 * V)
      narrow_part<T, 8, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (size <= 16 * V)
      narrow_part<T, 16, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (size <= 32 * V)
      narrow_part<T, 32, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if (!BIG || size <= 64 * V)
      narrow_part<T, 64, 1, TOP>(a, out, gather[wave], part, first, rows, turn);
    else if constexpr (BIG) {
      if (size <= 128 * V)
        narrow_part<T, 64, 2, TOP>(a, out, gather[wave], part, first, rows, turn);
      else
        narrow_part<T, 64, 4, TOP>(a, out, gather[wave], part, first, rows, turn);
    }
  }
  __syncthreads();
  const int64_t at = first * a.parts;
  for (int n = threadIdx.x; n < rows * a.parts * kStats; n += 256) {
    const int unit = n / kStats, part_n = unit % a.parts;
    if (a.begin[part_n + 1] - a.begin[part_n] > a.narrow) continue;
    if (a.stats) a.stats[at * kStats + n] = out.stats[n];
    if (n == unit * kStats) {
      a.entropy[at + unit] = out.entropy[unit];
      if (a.log_prob) a.log_prob[at + unit] = out.log_prob[unit];
    }
  }
}

// What the gradient of a row and part needs besides its entries.
struct Slopes {
  float most, log_z, entropy, dl, dh;
  int c;
};
template <class T>
__device__ __forceinline__ Slopes slopes_of(const ProbArgs &a, int64_t unit, int size, const T *x, const uint8_t *mask) {
  Slopes s;
  s.c = choice_of(a, unit, size);
  s.most = a.stats[unit * kStats];
  s.log_z = a.stats[unit * kStats + 1];
  s.entropy = a.stats[unit * kStats + 2];
  s.dl = a.dlog_prob && a.choice ? a.dlog_prob[unit] : 0.f;
  s.dh = a.dentropy ? a.dentropy[unit] : 0.f;
  if (s.c == INT32_MAX)
    s.dl = NAN;
  else if (a.choice && s.c >= 0 && entry(x, mask, s.c) == -INFINITY)
    s.dl = 0.f;  // its log probability is -inf whatever the others are
  if (!a.choice) s.c = INT32_MAX;
  return s;
}
// dl (1[c = i] - p) - dh p (l + H). (Far below the maximum p is zero before l + H is -1000, and l may
// be -inf, which times zero would be NaN.)
__device__ __forceinline__ float slope(const Slopes &s, float x, int i) {
  const float l = x - s.most - s.log_z, p = exp_of(l);
  const float d = (i == s.c ? s.dl : 0.f) - p * fmaf(s.dh, fmaxf(l + s.entropy, -1000.f), s.dl);
  return x == -INFINITY || s.c == -1 ? 0.f : d;
}

// Entries i .. i + V - 1 of `size`, -inf for those left out.
template <class T>
__device__ __forceinline__ void load_entries(const T *x, const uint8_t *mask, int i, int size, float (&v)[V]) {
  if (i + V <= size) {
    const auto r = *reinterpret_cast<const typename Loose<T>::Raw *>(x + i);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)r[j];
    if (mask) {
      const LooseMask u = *reinterpret_cast<const LooseMask *>(mask + i);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = u[j] ? v[j] : -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = i + j < size && (!mask || mask[i + j]) ? (float)x[i + j] : -INFINITY;
  }
}
template <class T>
__device__ __forceinline__ void store_entries(T *d, int i, int size, const float (&g)[V]) {
  if (i + V <= size) {
    typename Loose<T>::Raw r;
#pragma unroll
    for (int j = 0; j < V; ++j) r[j] = (T)g[j];
    *reinterpret_cast<typename Loose<T>::Raw *>(d + i) = r;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i + j < size) d[i + j] = (T)g[j];
  }
}

// n / d for quotients of up to 64 and d of up to 2^12: (n + 0.5) / d is at least 2^-13 away from every
// whole number, and three roundings of 64 are 2^-16.
__device__ __forceinline__ int quotient(int n, float inv_d) { return (int)(((float)n + 0.5f) * inv_d); }

// A workgroup has block_rows rows, and what their parts' gradients need in LDS: first V entries of a part
// to a lane, then the last size % V entries of the parts, one to a lane: neighbours in memory are
// neighbours among the lanes.
template <class T>
__global__ __launch_bounds__(256) void narrow_backward_kernel(ProbArgs a) {
  __shared__ Slopes of_unit[kUnits];
  const int64_t first = (int64_t)blockIdx.x * a.block_rows;
  const int rows = (int)min((int64_t)a.block_rows, a.R - first);
  const T *logits = (const T *)a.logits + first * a.stride;
  const uint8_t *masks = a.mask ? a.mask + first * a.mask_stride : nullptr;
  T *out = (T *)a.dlogits + first * a.W;
  int full = 0, rest = 0;  // of a row
  for (int p = 0; p < a.parts; ++p) {
    full += (a.begin[p + 1] - a.begin[p]) / V;
    rest += (a.begin[p + 1] - a.begin[p]) % V;
  }
  const float inv_parts = 1.f / a.parts, inv_full = full ? 1.f / full : 0.f, inv_rest = rest ? 1.f / rest : 0.f;
  for (int n = threadIdx.x; n < rows * a.parts; n += 256) {
    const int local = quotient(n, inv_parts), part = n - local * a.parts, begin = a.begin[part];
    of_unit[n] = slopes_of(a, first * a.parts + n, a.begin[part + 1] - begin, logits + local * a.stride + begin,
                           masks ? masks + local * a.mask_stride + begin : nullptr);
  }
  __syncthreads();
  for (int n = threadIdx.x; n < rows * full; n += 256) {
    const int local = quotient(n, inv_full), v = n - local * full;
    int part = 0, begin = 0, i = 0;  // entry i of the part is entry `begin` of the row
    for (int p = 0, seen = 0; p < a.parts; ++p) {  // the part that has vector v of the row
      const int here = (a.begin[p + 1] - a.begin[p]) / V;
      if (v >= seen && here) part = p, i = (v - seen) * V, begin = a.begin[p] + i;
      seen += here;
    }
    const Slopes s = of_unit[local * a.parts + part];
    float x[V];
    load_entries(logits + local * a.stride + begin, masks ? masks + local * a.mask_stride + begin : nullptr, 0, V, x);
#pragma unroll
    for (int j = 0; j < V; ++j) x[j] = slope(s, x[j], i + j);
    store_entries(out + (int64_t)local * a.W + begin, 0, V, x);
  }
  for (int n = threadIdx.x; n < rows * rest; n += 256) {
    const int local = quotient(n, inv_rest), v = n - local * rest;
    int part = 0, at = 0, i = 0;
    for (int p = 0, seen = 0; p < a.parts; ++p) {
      const int size = a.begin[p + 1] - a.begin[p], here = size % V;
      if (v >= seen && here) part = p, i = size - here + v - seen, at = a.begin[p] + i;
      seen += here;
    }
    const Slopes s = of_unit[local * a.parts + part];
    const float x = entry(logits + local * a.stride, masks ? masks + local * a.mask_stride : nullptr, at);
    out[(int64_t)local * a.W + at] = (T)slope(s, x, i);
  }
}

// ------------------------------------------------------------------------- larger parts

// The sum or maximum over a workgroup of WAVES wavefronts.
template <int WAVES>
__device__ __forceinline__ float block_sum(float v, float *lds) {
  v = wave_sum(v);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v += lds[w];
  return v;
}
template <int WAVES>
__device__ __forceinline__ float block_max(float v, float *lds) {
  v = lanes_max<kWave>(v);
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) v = fmaxf(v, lds[w]);
  return v;
}

template <class T>
__device__ __forceinline__ void store_result(const ProbArgs &a, int64_t unit, int c, const T *x, const uint8_t *mask, const Result &r) {
  a.entropy[unit] = c == -1 ? 0.f : r.entropy;
  if (a.log_prob) a.log_prob[unit] = log_prob_of(c, c >= 0 && c < INT32_MAX ? entry(x, mask, c) : 0.f, r);
  if (a.stats) {
    a.stats[unit * kStats] = r.most;
    a.stats[unit * kStats + 1] = r.log_z;
    a.stats[unit * kStats + 2] = r.entropy;
  }
}

// Many rows: a workgroup goes through one part of one row.
template <class T>
__global__ __launch_bounds__(256) void wide_forward_kernel(ProbArgs a) {
  __shared__ float lds[3][4];
  int64_t row;
  const int part = part_of(a, &row);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin;
  const int64_t unit = row * a.parts + part;
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  const int c = choice_of(a, unit, size);
  Seen s{-INFINITY, 0.f, 0.f};
  if (c != -1) {
    for (int i = threadIdx.x * V; i < size; i += 256 * V) {
      float v[V];
      load_entries(x, mask, i, size, v);
      see(s, v);
    }
  }
  s = moved_to(s, block_max<4>(s.most, lds[0]));
  s.z = block_sum<4>(s.z, lds[1]);
  s.s = block_sum<4>(s.s, lds[2]);
  if (threadIdx.x == 0) store_result(a, unit, c, x, mask, result_of(s));
}

// Few rows of many entries, or the largest entries wanted: a workgroup has a piece of 256 x 8 x N entries in
// registers. N is 4, and 2 where that leaves CUs without one (one row of 65,537 floats, the 5 likeliest, 9.7 / 7.6 us,
// but 64 rows of 131,072 14.9 / 18.5).
// In pieces and joined, or a workgroup a row, us: one row of 130,000 bf16 entries 6.9 / 25.9, of 50,000
// 6.6 / 11.5, of 20,000 6.7 / 6.2, of 1,500 4.5 / 3.5; 256 rows 26 / 49, 15 / 22, 10.6 / 9.0, 5.0 / 4.0;
// 511 rows of 50,000 22 / 24, 1,024 rows 37 / 27.
constexpr int kPiece = 256 * V * 4, kCut = 4 * kPiece;
__host__ __device__ inline int pieces_of(const ProbArgs &a, int size) { return (size + a.piece - 1) / a.piece; }

// The lists of WAVES wavefronts, joined in pairs; the first wavefront has the result.
template <int WAVES>
__device__ __forceinline__ uint64_t join_lists(uint64_t best, uint64_t (*lists)[64], int wave, int lane) {
  lists[wave][lane] = best;
  for (int step = 1; step < WAVES; step *= 2) {
    __syncthreads();
    if (wave % (2 * step) == 0) {
      best = joined(best, lists[wave + step][lane], lane);
      lists[wave][lane] = best;
    }
  }
  return best;
}

template <class T, bool TOP, int N>
__global__ __launch_bounds__(256) void piece_kernel(ProbArgs a) {
  __shared__ float lds[3][4];
  __shared__ uint64_t gather[TOP ? 4 : 1][128], lists[TOP ? 4 : 1][64];
  int64_t n;
  const int part = part_of(a, &n);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin, pieces = pieces_of(a, size);
  const int64_t row = n / pieces, unit = row * a.parts + part;
  const int first = (int)(n - row * pieces) * (256 * V * N);
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int c = choice_of(a, unit, size);
  float v[N][V];
#pragma unroll
  for (int k = 0; k < N; ++k) load_entries(x, mask, first + (k * 256 + (int)threadIdx.x) * V, c == -1 ? 0 : size, v[k]);
  float lane_max = -INFINITY;
#pragma unroll
  for (int k = 0; k < N; ++k)
#pragma unroll
    for (int j = 0; j < V; ++j) lane_max = fmaxf(lane_max, v[k][j]);
  Seen s{block_max<4>(lane_max, lds[0]), 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < N; ++k) add(s, v[k]);
  s.z = block_sum<4>(s.z, lds[1]);
  s.s = block_sum<4>(s.s, lds[2]);
  const Result r = result_of(s);
  if (pieces == 1) {
    if (threadIdx.x == 0) store_result(a, unit, c, x, mask, r);
  } else if (threadIdx.x == 0) {
    float *out = a.pieces + (int64_t)blockIdx.x * 3;
    out[0] = s.most;
    out[1] = s.z;
    out[2] = s.s;
  }
  if constexpr (TOP) {
    int from[N];
#pragma unroll
    for (int k = 0; k < N; ++k) from[k] = first + (k * 256 + (int)threadIdx.x) * V;
    uint64_t best = largest_of(v, from, lane_max, a.top, gather[wave], lane);
    best = join_lists<4>(best, lists, wave, lane);
    if (wave == 0 && lane < a.top) {
      if (pieces == 1)
        store_top(a, unit * a.top + lane, best, r);
      else
        a.lists[(int64_t)blockIdx.x * a.top + lane] = best;
    }
  }
}

// The pieces of a part of a row, one workgroup each.
constexpr int kJoinWaves = 16;
template <class T, bool TOP>
__global__ __launch_bounds__(64 * kJoinWaves) void join_pieces_kernel(ProbArgs a) {
  __shared__ float lds[3][kJoinWaves];
  __shared__ uint64_t lists[TOP ? kJoinWaves : 1][64];
  const int part = blockIdx.y;
  const int begin = a.begin[part], size = a.begin[part + 1] - begin, pieces = pieces_of(a, size);
  if (pieces == 1) return;
  const int64_t row = blockIdx.x, unit = row * a.parts + part, at = a.block[part] + row * pieces;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  Seen s{-INFINITY, 0.f, 0.f};
  for (int i = threadIdx.x; i < pieces; i += 64 * kJoinWaves) {
    const float *p = a.pieces + (at + i) * 3;
    const Seen o{p[0], p[1], p[2]};
    const float most = fmaxf(s.most, o.most);
    const Seen x = moved_to(s, most), y = moved_to(o, most);
    s = {most, x.z + y.z, x.s + y.s};
  }
  s = moved_to(s, block_max<kJoinWaves>(s.most, lds[0]));
  s.z = block_sum<kJoinWaves>(s.z, lds[1]);
  s.s = block_sum<kJoinWaves>(s.s, lds[2]);
  const Result r = result_of(s);
  if (threadIdx.x == 0)
    store_result(a, unit, choice_of(a, unit, size), (const T *)a.logits + row * a.stride + begin,
                 a.mask ? a.mask + row * a.mask_stride + begin : nullptr, r);
  if constexpr (TOP) {
    uint64_t best = 0;
    for (int i = wave; i < pieces; i += kJoinWaves) {
      const uint64_t k = lane < a.top ? a.lists[(at + i) * a.top + lane] : 0;
      if (__ballot(k > lane_of(best, a.top - 1))) best = joined(best, k, lane);
    }
    best = join_lists<kJoinWaves>(best, lists, wave, lane);
    if (wave == 0 && lane < a.top) store_top(a, unit * a.top + lane, best, r);
  }
}

// Every workgroup has kSpan entries of a part of a row, from the last to the first: what the forward
// call read last may still be in the caches (256 MB of floats 87.2 us, 88.4 from the first to the last; of
// 819 MB nothing is).
constexpr int kSpan = 256 * V * 2;
template <class T>
__global__ __launch_bounds__(256) void wide_backward_kernel(ProbArgs a) {
  int64_t n;
  const int part = part_of(a, &n);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin;
  const int64_t spans = cdiv(size, kSpan);
  n = a.R * spans - 1 - n;
  const int64_t row = n / spans;
  const int first = (int)(n - row * spans) * kSpan;
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  T *d = (T *)a.dlogits + row * a.W + begin;
  const Slopes s = slopes_of(a, row * a.parts + part, size, x, mask);
  const int last = min(first + kSpan, size);
  for (int i = first + threadIdx.x * V; i < last; i += 256 * V) {
    float v[V];
    load_entries(x, mask, i, s.c == -1 ? 0 : size, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = slope(s, v[j], i + j);
    store_entries(d, i, size, v);
  }
}

// ----------------------------------------------------------------------------- launches

int check(const astra_log_probs *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_ABI_CHECK(f->rows, >=, 0);
  ASTRA_ABI_CHECK(f->rows, <=, kMostRows);
  ASTRA_ABI_CHECK(f->parts, >=, 1);
  ASTRA_ABI_CHECK(f->parts, <=, ASTRA_SEQ_MAX_PARTS);
  ASTRA_ABI_CHECK(f->top, >=, 0);
  ASTRA_ABI_CHECK(f->top, <=, ASTRA_SEQ_MAX_TOP);
  int64_t all = 0;
  for (int i = 0; i < f->parts; ++i) {
    ASTRA_ABI_CHECK(f->sizes[i], >=, 1);
    ASTRA_ABI_CHECK(f->sizes[i], >=, f->top);
    all += f->sizes[i];
  }
  ASTRA_ABI_CHECK(all, <=, ASTRA_SEQ_MAX_ENTRIES);
  ASTRA_ABI_CHECK(f->stride, >=, 0);
  ASTRA_ABI_CHECK(f->mask_stride, >=, 0);
  ASTRA_ABI_CHECK(f->choice_bytes == 4 || f->choice_bytes == 8 || !f->choice, ==, true);
  return ASTRA_OK;
}

ProbArgs args_of(const astra_log_probs &f) {
  ProbArgs a{};
  a.logits = f.logits;
  a.mask = f.mask;
  a.choice = f.choice;
  a.log_prob = f.log_prob;
  a.entropy = f.entropy;
  a.stats = f.stats;
  a.top_log_prob = f.top_log_prob;
  a.top_index = f.top_index;
  a.R = f.rows;
  a.stride = f.stride;
  a.mask_stride = f.mask_stride;
  a.parts = f.parts;
  a.top = f.top;
  a.wide_choice = f.choice_bytes == 8;
  int largest = 0;
  for (int i = 0; i < f.parts; ++i) {
    a.begin[i + 1] = a.begin[i] + f.sizes[i];
    largest = std::max(largest, f.sizes[i]);
  }
  // Lanes' work ends with its loads, a workgroup's with two barriers. Both, us, the former first: 81,920
  // rows of 1,000 bf16 entries 51 / 95, of 1,500 73 / 136, of 2,048 81 / 106; of 1,000 floats 73 / 100, of
  // 1,500 107 / 133, but with the gradient 338 / 312. 4,096 rows of 1,000 bf16 entries with the gradient 15 / 19, 512
  // alike. The 20 largest: 20,000 rows of 1,000 48 / 159, of 2,000 61 / 161.
  a.narrow = f.rows < 512 && !f.top ? 512 : f.type == ASTRA_SEQ_F32 && !f.top ? 1024 : 2048;
  a.cut = f.top > 0 || (f.rows * f.parts < 512 && largest > kCut);
  a.W = a.begin[f.parts];
  a.piece = f.rows < 256 && f.rows * cdiv(a.W, kPiece) < 256 ? kPiece / 2 : kPiece;
  return a;
}

// Gives the workgroups of a launch to the larger parts, `each(size)` for one; how many there are.
template <class Each>
int64_t share(ProbArgs &a, Each &&each) {
  int64_t n = 0;
  for (int i = 0; i < a.parts; ++i) {
    const int size = a.begin[i + 1] - a.begin[i];
    a.block[i] = n;
    if (size > a.narrow) n += each(size);
  }
  for (int i = a.parts; i <= kParts; ++i) a.block[i] = n;
  return n;
}

// Rows of a workgroup that has all their smaller parts: enough for its four wavefronts where there are 512
// such workgroups, and more of them, up to what LDS has room for, where there are many. One / eight / these,
// us, with the gradient: parts of 127, 127, 6, 6, 81,920 rows 381 / 77 / 56, 16,384 rows 83 / 25 / 25; one of 64, 81,920
// rows 233 / 41 / 20. More only with 4,096 workgroups / these: 7,235 rows of 64 18 / 9, of four parts 25 / 18, the
// likeliest of 64 39 / 8.
int rows_together(const ProbArgs &a) {
  int n = 1, lanes = 1;  // lanes: of the largest part
  for (int i = 0; i < a.parts; ++i)
    if (a.begin[i + 1] - a.begin[i] <= a.narrow)
      while (lanes < kWave && lanes * V < a.begin[i + 1] - a.begin[i]) lanes *= 2;
  const int busy = std::max(1, 4 * kWave / lanes / a.parts);
  while (2 * n * a.parts <= kUnits && 2 * n <= 64 && a.R >= (n < busy ? 512 : 4096) * n) n *= 2;
  return n;
}
bool some_narrow(const ProbArgs &a) {
  for (int i = 0; i < a.parts; ++i)
    if (a.begin[i + 1] - a.begin[i] <= a.narrow) return true;
  return false;
}
bool some_wide(const ProbArgs &a) {
  for (int i = 0; i < a.parts; ++i)
    if (a.begin[i + 1] - a.begin[i] > a.narrow) return true;
  return false;
}

int64_t all_pieces(ProbArgs &a) {  // (of the rows of a launch)
  return share(a, [&](int size) { return a.R * pieces_of(a, size); });
}
bool joins(const ProbArgs &a) {
  for (int i = 0; i < a.parts; ++i)
    if (pieces_of(a, a.begin[i + 1] - a.begin[i]) > 1) return true;
  return false;
}
// Rows that one launch of each kernel has room for: at most 1,024 threads a row, and 256 a span or piece.
int64_t most_rows(const ProbArgs &a) {
  int64_t blocks = 4;
  for (int i = 0; i < a.parts; ++i) blocks += cdiv(a.begin[i + 1] - a.begin[i], kSpan);
  return kMostThreads / (256 * blocks);
}
// `n` of the rows, from `first` on
ProbArgs rows_of(ProbArgs a, int32_t type, int64_t first, int64_t n) {
  const auto on = [&](auto &p, int64_t bytes_a_row) {
    if (p) p = (std::decay_t<decltype(p)>)((uintptr_t)p + (uintptr_t)(first * bytes_a_row));
  };
  const int64_t e = (int64_t)elem_size(type), each = a.parts * (int64_t)sizeof(float);
  on(a.logits, a.stride * e);
  on(a.mask, a.mask_stride);
  on(a.choice, a.parts * (a.wide_choice ? 8 : 4));
  on(a.log_prob, each);
  on(a.entropy, each);
  on(a.stats, each * kStats);
  on(a.top_log_prob, each * a.top);
  on(a.top_index, a.parts * a.top * (int64_t)sizeof(int64_t));
  on(a.dlog_prob, each);
  on(a.dentropy, each);
  on(a.dlogits, a.W * e);
  a.R = n;
  return a;
}

// the lists first, which are of 8 bytes
size_t piece_bytes(ProbArgs a) {
  a.R = std::min(a.R, most_rows(a));
  return a.cut && joins(a) ? (size_t)all_pieces(a) * (3 * sizeof(float) + a.top * sizeof(uint64_t)) : 0;
}

#define PROBS_LAUNCH(kernel, blocks, threads)                                                          \
  do {                                                                                                 \
    const int64_t blocks_ = (blocks);                                                                  \
    ASTRA_ABI_CHECK(blocks_ * threads, <=, kMostThreads);                                              \
    hipLaunchKernelGGL((kernel), dim3((unsigned)blocks_), dim3(threads), 0, st, a);                    \
    ASTRA_HIP_CHECK(rt_last_error(), #kernel " launch");                                               \
  } while (false)

template <class T, bool TOP>
int forward_in_pieces(ProbArgs &a, hipStream_t st) {
  const int64_t pieces = all_pieces(a);
  if (a.piece == kPiece) {
    PROBS_LAUNCH((piece_kernel<T, TOP, 4>), pieces, 256);
  } else {
    PROBS_LAUNCH((piece_kernel<T, TOP, 2>), pieces, 256);
  }
  if (!joins(a)) return ASTRA_OK;
  ASTRA_ABI_CHECK(a.R * 64 * kJoinWaves, <=, kMostThreads);
  hipLaunchKernelGGL((join_pieces_kernel<T, TOP>), dim3((unsigned)a.R, (unsigned)a.parts), dim3(64 * kJoinWaves), 0, st, a);
  ASTRA_HIP_CHECK(rt_last_error(), "join_pieces_kernel launch");
  return ASTRA_OK;
}

template <class T>
int forward(ProbArgs a, hipStream_t st) {
  if (a.lists) a.pieces = (float *)(a.lists + all_pieces(a) * a.top);
  if (some_narrow(a)) {
    a.block_rows = rows_together(a);
    bool big = false;
    for (int i = 0; i < a.parts; ++i) {
      const int size = a.begin[i + 1] - a.begin[i];
      big |= size > 64 * V && size <= a.narrow;
    }
    const int64_t blocks = cdiv(a.R, a.block_rows);
    if (a.top && big) {
      PROBS_LAUNCH((narrow_forward_kernel<T, true, true>), blocks, 256);
    } else if (a.top) {
      PROBS_LAUNCH((narrow_forward_kernel<T, true, false>), blocks, 256);
    } else if (big) {
      PROBS_LAUNCH((narrow_forward_kernel<T, false, true>), blocks, 256);
    } else {
      PROBS_LAUNCH((narrow_forward_kernel<T, false, false>), blocks, 256);
    }
  }
  if (!some_wide(a)) return ASTRA_OK;
  if (a.cut) return a.top ? forward_in_pieces<T, true>(a, st) : forward_in_pieces<T, false>(a, st);
  PROBS_LAUNCH(wide_forward_kernel<T>, share(a, [&](int) { return a.R; }), 256);
  return ASTRA_OK;
}

// Rows of which every part is small go through as a whole, others part by part.
template <class T>
int backward(ProbArgs a, hipStream_t st) {
  if (!some_wide(a)) {
    a.block_rows = rows_together(a);
    PROBS_LAUNCH(narrow_backward_kernel<T>, cdiv(a.R, a.block_rows), 256);
    return ASTRA_OK;
  }
  int64_t n = 0;
  for (int i = 0; i < a.parts; ++i) {
    a.block[i] = n;
    n += a.R * cdiv(a.begin[i + 1] - a.begin[i], kSpan);
  }
  for (int i = a.parts; i <= kParts; ++i) a.block[i] = n;
  PROBS_LAUNCH(wide_backward_kernel<T>, n, 256);
  return ASTRA_OK;
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_log_probs_workspace_size(const astra_log_probs *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  *bytes = f->rows ? piece_bytes(args_of(*f)) : 0;
  return ASTRA_OK;
}

int astra_log_probs_forward(const astra_log_probs *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->rows == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(f->logits);
  ASTRA_SEQ_POINTER(f->entropy);
  ProbArgs a = args_of(*f);
  if (const size_t need = piece_bytes(a)) {
    ASTRA_SEQ_POINTER(f->workspace);
    ASTRA_ABI_CHECK(f->workspace_bytes, >=, need);
    if (!aligned(f->workspace, 8)) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_log_probs_forward: the workspace starts on 8 bytes");
    a.lists = (uint64_t *)f->workspace;
  }
  if (f->choice) ASTRA_SEQ_POINTER(f->log_prob);
  if (f->log_prob) ASTRA_SEQ_POINTER(f->choice);
  if (f->top) {
    ASTRA_SEQ_POINTER(f->top_log_prob);
    ASTRA_SEQ_POINTER(f->top_index);
  }
  for (int64_t r = 0, most = most_rows(a); r < f->rows; r += most) {
    const ProbArgs some = rows_of(a, f->type, r, std::min(most, f->rows - r));
    if (int rc = f->type == ASTRA_SEQ_F32 ? forward<float>(some, as_stream(stream)) : forward<bf16>(some, as_stream(stream))) return rc;
  }
  return ASTRA_OK;
}

int astra_log_probs_backward(const astra_log_probs_grad *g, void *stream) {
  ASTRA_SEQ_POINTER(g);
  const astra_log_probs &f = g->f;
  if (int rc = check(&f)) return rc;
  if (f.rows == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(f.logits);
  ASTRA_SEQ_POINTER(f.stats);
  ASTRA_SEQ_POINTER(g->dlogits);
  ProbArgs a = args_of(f);
  a.dlog_prob = g->dlog_prob;
  a.dentropy = g->dentropy;
  a.dlogits = g->dlogits;
  for (int64_t r = 0, most = most_rows(a); r < f.rows; r += most) {
    const ProbArgs some = rows_of(a, f.type, r, std::min(most, f.rows - r));
    if (int rc = f.type == ASTRA_SEQ_F32 ? backward<float>(some, as_stream(stream)) : backward<bf16>(some, as_stream(stream))) return rc;
  }
  return ASTRA_OK;
}

}  // extern "C"
