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
#include "sequence.h"

#define ASTRA_SRC_NAME "sequence_probs.hip"

namespace astra_seq {
namespace {

constexpr int kParts = ASTRA_SEQ_MAX_PARTS, kTop = ASTRA_SEQ_MAX_TOP;
constexpr int V = 8;             // entries a lane takes at a time
constexpr int kNarrow = 1024;    // parts up to here are a group of lanes' work, larger ones a workgroup's
constexpr int kStats = 3;        // m, log Z, H of a row and part

struct ProbArgs {
  const void *logits;
  const uint8_t *mask;
  const void *choice;
  float *log_prob, *entropy, *stats, *top_log_prob;
  int64_t *top_index;
  const float *dlog_prob, *dentropy;
  void *dlogits;
  int64_t R, stride, mask_stride;
  int32_t W, parts, top, wide_choice;
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

// Entries i .. i + V - 1 of a part, -inf for those beyond it or left out.
template <class T>
__device__ __forceinline__ void entries(const T *x, const uint8_t *mask, int i, int size, float (&v)[V]) {
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

__device__ __forceinline__ void see(Seen &a, const float (&x)[V]) {
  float most = x[0];
#pragma unroll
  for (int j = 1; j < V; ++j) most = fmaxf(most, x[j]);
  if (most > a.most) a = moved_to(a, most);
  const float base = a.most == -INFINITY ? 0.f : a.most;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float d = x[j] - base, t = exp_of(d);
    a.z += t;
    a.s = fmaf(t, fmaxf(d, -1000.f), a.s);  // (t is zero far before that; -inf times it would be NaN)
  }
}

struct Result {
  float most, log_z, entropy;
};
__device__ __forceinline__ Result result_of(const Seen &a) {
  if (a.most == -INFINITY && a.z == 0.f) return {0.f, 0.f, 0.f};  // nothing is allowed
  const float log_z = logf(a.z);
  return {a.most == -INFINITY ? 0.f : a.most, log_z, log_z - a.s / a.z};
}

// Sum and maximum over `G` neighbouring lanes (a power of two, the same in the whole wavefront).
template <int CTRL>
__device__ __forceinline__ float swapped(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float group_max(float v, int G) {
  if (G >= 2) v = fmaxf(v, swapped<kSwap1>(v));
  if (G >= 4) v = fmaxf(v, swapped<kSwap2>(v));
  if (G >= 8) v = fmaxf(v, swapped<kMirror8>(v));
  if (G >= 16) v = fmaxf(v, swapped<kMirror16>(v));
  if (G >= 32) {
    const Pair p = rows_of_half(v);
    v = fmaxf(p.first, p.second);
  }
  if (G >= 64) {
    const Pair p = halves(v);
    v = fmaxf(p.first, p.second);
  }
  return v;
}
__device__ __forceinline__ float group_sum(float v, int G) {
  if (G >= 2) v += swapped<kSwap1>(v);
  if (G >= 4) v += swapped<kSwap2>(v);
  if (G >= 8) v += swapped<kMirror8>(v);
  if (G >= 16) v += swapped<kMirror16>(v);
  if (G >= 32) {
    const Pair p = rows_of_half(v);
    v = p.first + p.second;
  }
  if (G >= 64) {
    const Pair p = halves(v);
    v = p.first + p.second;
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

// A wavefront's list of the largest keys, one a lane, falling; `last` is the top-th.
struct Largest {
  uint64_t key = 0, last = 0;

  __device__ __forceinline__ void put(uint64_t k, int lane, int top) {
    const int at = __popcll(__ballot(key > k));
    const uint32_t lo = __shfl_up((uint32_t)key, 1), hi = __shfl_up((uint32_t)(key >> 32), 1);
    key = lane < at ? key : lane == at ? k : (uint64_t)hi << 32 | lo;
    last = lane_of(key, top - 1);
  }
  // a key of each lane (called by the whole wavefront)
  __device__ __forceinline__ void see(uint64_t k, int lane, int top) {
    for (uint64_t more = __ballot(k > last); more; more = __ballot(k > last)) {
      const int from = __builtin_ctzll(more);
      put(lane_of(k, from), lane, top);
      if (lane == from) k = 0;
    }
  }
};

__device__ __forceinline__ void store_top(const ProbArgs &a, int64_t at, uint64_t key, const Result &r) {
  a.top_log_prob[at] = key ? value_of(key) - r.most - r.log_z : -INFINITY;
  a.top_index[at] = key ? index_of(key) : -1;
}

template <class T>
__device__ __forceinline__ void store_result(const ProbArgs &a, int64_t unit, int c, const T *x, const uint8_t *mask, const Result &r) {
  a.entropy[unit] = c == -1 ? 0.f : r.entropy;
  if (a.log_prob)
    a.log_prob[unit] = c == -1 ? 0.f : c == INT32_MAX ? NAN : entry(x, mask, c) - r.most - r.log_z;
  if (a.stats) {
    a.stats[unit * kStats] = r.most;
    a.stats[unit * kStats + 1] = r.log_z;
    a.stats[unit * kStats + 2] = r.entropy;
  }
}

// ------------------------------------------------------------- parts of up to 1,024 entries

// Lanes of a part: V entries each, or 2 V of the largest parts.
__host__ __device__ inline int lanes_of(int size) {
  int G = 1;
  while (G < 64 && G * V < size) G *= 2;
  return G;
}

// A group of lanes has one part of one row in registers.
template <class T, int C, bool TOP>
__device__ __forceinline__ void narrow_forward(const ProbArgs &a, int part, int64_t n) {
  const int begin = a.begin[part], size = a.begin[part + 1] - begin, G = lanes_of(size);
  const int j = threadIdx.x & (G - 1);
  const int64_t row = n * (256 / G) + threadIdx.x / G, unit = row * a.parts + part;
  const bool in = row < a.R;
  const T *x = (const T *)a.logits + (in ? row : 0) * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + (in ? row : 0) * a.mask_stride + begin : nullptr;
  const int c = in ? choice_of(a, unit, size) : -1;
  float v[C][V];
  Seen s{-INFINITY, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < C; ++k) {
    if (c != -1)
      entries(x, mask, (k * G + j) * V, size, v[k]);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) v[k][i] = -INFINITY;
    see(s, v[k]);
  }
  const float most = group_max(s.most, G);
  s = moved_to(s, most);
  s.z = group_sum(s.z, G);
  s.s = group_sum(s.s, G);
  const Result r = result_of(s);
  if (in && j == 0) store_result(a, unit, c, x, mask, r);
  // the largest one after the other
  if constexpr (!TOP) return;
  uint32_t gone = 0;
  for (int t = 0; t < a.top; ++t) {
    uint64_t best = 0;
    int which = 0;
#pragma unroll
    for (int k = 0; k < C; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const uint64_t key = gone >> (k * V + i) & 1 ? 0 : key_of(v[k][i], (k * G + j) * V + i);
        which = key > best ? k * V + i : which;
        best = key > best ? key : best;
      }
    uint64_t all = best;
    for (int d = 1; d < G; d *= 2) {
      const uint64_t o = (uint64_t)__shfl_xor((uint32_t)(all >> 32), d) << 32 | (uint32_t)__shfl_xor((uint32_t)all, d);
      all = o > all ? o : all;
    }
    if (best == all) gone |= 1u << which;
    if (in && j == 0) store_top(a, unit * a.top + t, all, r);
  }
}

template <class T, bool TOP>
__global__ __launch_bounds__(256) void narrow_forward_kernel(ProbArgs a) {
  int64_t n;
  const int part = part_of(a, &n);
  if (a.begin[part + 1] - a.begin[part] <= 64 * V)
    narrow_forward<T, 1, TOP>(a, part, n);
  else
    narrow_forward<T, 2, TOP>(a, part, n);
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
__device__ __forceinline__ float slope(const Slopes &s, float x, int i) {
  const float l = x - s.most - s.log_z, p = exp_of(l);
  const float d = s.dl * ((i == s.c ? 1.f : 0.f) - p) - s.dh * (p > 0.f ? p * (l + s.entropy) : 0.f);
  return x == -INFINITY ? 0.f : d;
}

// V entries of a gradient.
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

template <class T>
__device__ __forceinline__ void entries_backward(const Slopes &s, const T *x, const uint8_t *mask, T *d, int i, int size) {
  float v[V];
  if (s.c != -1) {
    entries(x, mask, i, size, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = slope(s, v[j], i + j);
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.f;
  }
  store_entries(d, i, size, v);
}

template <class T>
__global__ __launch_bounds__(256) void narrow_backward_kernel(ProbArgs a) {
  int64_t n;
  const int part = part_of(a, &n);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin, G = lanes_of(size);
  const int64_t row = n * (256 / G) + threadIdx.x / G;
  if (row >= a.R) return;
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  T *d = (T *)a.dlogits + row * a.W + begin;
  const Slopes s = slopes_of(a, row * a.parts + part, size, x, mask);
  for (int i = (threadIdx.x & (G - 1)) * V; i < size; i += G * V) entries_backward(s, x, mask, d, i, size);
}

// ------------------------------------------------------------------------- larger parts

// A workgroup has one part of one row.
template <class T, int N, bool TOP>
__global__ __launch_bounds__(N) void wide_forward_kernel(ProbArgs a) {
  constexpr int kWaves = N / kWave;
  __shared__ float lds[3][kWaves];
  __shared__ uint64_t lists[TOP ? kWaves : 1][kTop];
  int64_t row;
  const int part = part_of(a, &row);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin;
  const int64_t unit = row * a.parts + part;
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int c = choice_of(a, unit, size);
  Seen s{-INFINITY, 0.f, 0.f};
  Largest best;
  if (c != -1) {
    for (int i = threadIdx.x * V; i - lane * V < size; i += N * V) {
      float v[V];
      entries(x, mask, i, size, v);
      see(s, v);
      if constexpr (TOP) {
#pragma unroll
        for (int j = 0; j < V; ++j) best.see(key_of(v[j], i + j), lane, a.top);
      }
    }
  }
  const auto over_all = [&](float v, float *p, bool sum) __attribute__((always_inline)) {
    v = sum ? group_sum(v, 64) : group_max(v, 64);
    if (lane == 0) p[wave] = v;
    __syncthreads();
    v = p[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) v = sum ? v + p[w] : fmaxf(v, p[w]);
    return v;
  };
  s = moved_to(s, over_all(s.most, lds[0], false));
  s.z = over_all(s.z, lds[1], true);
  s.s = over_all(s.s, lds[2], true);
  const Result r = result_of(s);
  if (threadIdx.x == 0) store_result(a, unit, c, x, mask, r);
  if constexpr (TOP) {
    lists[wave][lane] = best.key;
    __syncthreads();
    if (wave == 0) {
      for (int w = 1; w < kWaves; ++w) best.see(lane < a.top ? lists[w][lane] : 0, lane, a.top);
      if (lane < a.top) store_top(a, unit * a.top + lane, best.key, r);
    }
  }
}

// Every workgroup has kPiece entries of a part of a row.
constexpr int kPiece = 256 * V * 2;
template <class T>
__global__ __launch_bounds__(256) void wide_backward_kernel(ProbArgs a) {
  int64_t n;
  const int part = part_of(a, &n);
  const int begin = a.begin[part], size = a.begin[part + 1] - begin;
  const int64_t pieces = cdiv(size, kPiece), row = n / pieces;
  const int first = (int)(n - row * pieces) * kPiece;
  const T *x = (const T *)a.logits + row * a.stride + begin;
  const uint8_t *mask = a.mask ? a.mask + row * a.mask_stride + begin : nullptr;
  T *d = (T *)a.dlogits + row * a.W + begin;
  const Slopes s = slopes_of(a, row * a.parts + part, size, x, mask);
  const int last = min(first + kPiece, size);
  for (int i = first + threadIdx.x * V; i < last; i += 256 * V) entries_backward(s, x, mask, d, i, size);
}

// ----------------------------------------------------------------------------- launches

int check(const astra_log_probs *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_ABI_CHECK(f->rows, >=, 0);
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
  for (int i = 0; i < f.parts; ++i) a.begin[i + 1] = a.begin[i] + f.sizes[i];
  a.W = a.begin[f.parts];
  return a;
}

// Gives the workgroups of a launch to the parts of one kind; how many there are.
template <class Blocks>
int64_t share(ProbArgs &a, bool narrow, Blocks &&blocks) {
  int64_t n = 0;
  for (int i = 0; i < a.parts; ++i) {
    const int size = a.begin[i + 1] - a.begin[i];
    a.block[i] = n;
    if ((size <= kNarrow) == narrow) n += blocks(size);
  }
  for (int i = a.parts; i <= kParts; ++i) a.block[i] = n;
  return n;
}

#define PROBS_LAUNCH(kernel, blocks, threads)                                                          \
  do {                                                                                                 \
    const int64_t blocks_ = (blocks);                                                                  \
    if (blocks_ == 0) break;                                                                           \
    ASTRA_ABI_CHECK(blocks_, <, 2147483648ll);                                                         \
    hipLaunchKernelGGL((kernel), dim3((unsigned)blocks_), dim3(threads), 0, st, a);                    \
    ASTRA_HIP_CHECK(rt_last_error(), #kernel " launch");                                               \
  } while (false)

template <class T>
int forward(ProbArgs a, hipStream_t st) {
  const int64_t narrow = share(a, true, [&](int size) { return cdiv(a.R, 256 / lanes_of(size)); });
  if (a.top) {
    PROBS_LAUNCH((narrow_forward_kernel<T, true>), narrow, 256);
  } else {
    PROBS_LAUNCH((narrow_forward_kernel<T, false>), narrow, 256);
  }
  const int64_t wide = share(a, false, [&](int) { return a.R; });
  if (wide >= 512 && a.top) {
    PROBS_LAUNCH((wide_forward_kernel<T, 256, true>), wide, 256);
  } else if (wide >= 512) {
    PROBS_LAUNCH((wide_forward_kernel<T, 256, false>), wide, 256);
  } else if (a.top) {
    PROBS_LAUNCH((wide_forward_kernel<T, 1024, true>), wide, 1024);
  } else {
    PROBS_LAUNCH((wide_forward_kernel<T, 1024, false>), wide, 1024);
  }
  return ASTRA_OK;
}

template <class T>
int backward(ProbArgs a, hipStream_t st) {
  PROBS_LAUNCH(narrow_backward_kernel<T>, share(a, true, [&](int size) { return cdiv(a.R, 256 / lanes_of(size)); }), 256);
  PROBS_LAUNCH(wide_backward_kernel<T>, share(a, false, [&](int size) { return a.R * cdiv(size, kPiece); }), 256);
  return ASTRA_OK;
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_log_probs_forward(const astra_log_probs *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->rows == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(f->logits);
  ASTRA_SEQ_POINTER(f->entropy);
  if (f->choice) ASTRA_SEQ_POINTER(f->log_prob);
  if (f->log_prob) ASTRA_SEQ_POINTER(f->choice);
  if (f->top) {
    ASTRA_SEQ_POINTER(f->top_log_prob);
    ASTRA_SEQ_POINTER(f->top_index);
  }
  return f->type == ASTRA_SEQ_F32 ? forward<float>(args_of(*f), as_stream(stream)) : forward<bf16>(args_of(*f), as_stream(stream));
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
  return f.type == ASTRA_SEQ_F32 ? backward<float>(a, as_stream(stream)) : backward<bf16>(a, as_stream(stream));
}

}  // extern "C"
