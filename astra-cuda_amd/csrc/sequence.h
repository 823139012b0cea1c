// sequence.h -- shared by the sequence operators' translation units: element types, wide
// loads and stores, sums over a wavefront or workgroup, and the sum over partial rows that
// ends every gradient of a parameter.
#pragma once

#include "sequence/astra_sequence.h"
#include "runtime.h"

namespace astra_seq {

using astra_rt::as_stream;
using astra_rt::fail;
using astra_rt::rt_last_error;

using bf16 = __bf16;
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr float kLog2e = 1.4426950408889634f;

// V consecutive elements as floats: one load of 16 bytes or less each. V = 1 is the form
// for rows whose width, stride or address does not allow a wide access.
template <class T, int V>
struct Vec {
  typedef T Raw __attribute__((ext_vector_type(V)));
  static __device__ __forceinline__ void load(const T *p, float (&out)[V]) {
    const Raw r = *reinterpret_cast<const Raw *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)r[i];
  }
  static __device__ __forceinline__ void store(T *p, const float (&v)[V]) {
    Raw r;
#pragma unroll
    for (int i = 0; i < V; ++i) r[i] = (T)v[i];
    *reinterpret_cast<Raw *>(p) = r;
  }
};
template <class T>
struct Vec<T, 1> {
  static __device__ __forceinline__ void load(const T *p, float (&out)[1]) { out[0] = (float)*p; }
  static __device__ __forceinline__ void store(T *p, const float (&v)[1]) { *p = (T)v[0]; }
};

// v of another lane by a data-parallel move, which costs a vector operation where a general
// shuffle goes through LDS; lanes that are given none get 0.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float moved(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
}
constexpr int kSwap1 = 0xB1, kSwap2 = 0x4E;                // lane ^ 1, lane ^ 2 (quad_perm)
constexpr int kMirror8 = 0x141, kMirror16 = 0x140;         // reversed within 8, within 16 lanes
constexpr int kUp = 0x110, kBcast15 = 0x142, kBcast31 = 0x143;  // row_shr:n, and the last lane of the rows before

// v of the even and of the odd row of 16 lanes of this lane's half, and of the lower and the
// upper half, at this lane's place in them.
struct Pair {
  float first, second;
};
__device__ __forceinline__ Pair rows_of_half(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const unsigned first = p[0], second = p[1];  // (a bit_cast of p[1] itself reads p[0])
  return {__builtin_bit_cast(float, first), __builtin_bit_cast(float, second)};
}
__device__ __forceinline__ Pair halves(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned first = p[0], second = p[1];  // (a bit_cast of p[1] itself reads p[0])
  return {__builtin_bit_cast(float, first), __builtin_bit_cast(float, second)};
}

// The sum over the lanes with this lane's place in their rows of 16.
__device__ __forceinline__ float rows_sum(float v) {
  Pair p = rows_of_half(v);
  p = halves(p.first + p.second);
  return p.first + p.second;
}

// The sum over N neighbouring lanes, in each of them.
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (N >= 2) v += moved<kSwap1>(v);
  if constexpr (N >= 4) v += moved<kSwap2>(v);
  if constexpr (N >= 8) v += moved<kMirror8>(v);  // the other four lanes, which are alike by now
  if constexpr (N >= 16) v += moved<kMirror16>(v);
  if constexpr (N == 64) return rows_sum(v);
  if constexpr (N == 32) {
    const Pair p = rows_of_half(v);
    return p.first + p.second;
  }
  return v;
}
__device__ __forceinline__ float wave_sum(float v) { return lanes_sum<kWave>(v); }

// The sum over TPR threads (part of a wavefront, or a whole workgroup through `lds`,
// TPR / 64 words that nothing else uses; two calls in a row need two such areas).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
  v = lanes_sum<(TPR < kWave ? TPR : kWave)>(v);
  if constexpr (TPR > kWave) {
    constexpr int W = TPR / kWave;
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) v += lds[i];
  }
  return v;
}

// 1 / (1 + exp(-v)) for results of type T. The hardware's exp2 and reciprocal are each good to
// 1 ulp, but its argument -log2(e) v is rounded, which is up to |v| 2^-24 of the result: 3.6e-6
// at v = -60. That is nothing beside a bf16's 2^-9; for floats, exp2 is multiplied by
// exp(-v - t ln 2) for the rounded argument t, as 1 plus a first-order term.
template <class T>
__device__ __forceinline__ float sigmoid(float v) {
  const float t = -kLog2e * v;
  float e = __builtin_amdgcn_exp2f(t);
  if constexpr (sizeof(T) == 4) {
    const float rest = fmaf(-t, -1.9046543e-9f, fmaf(-t, 0.693147182f, -v));
    e = fabsf(t) < 126.f ? fmaf(e, rest, e) : e;  // (beyond that the result is 0 or 1, and e may be infinite)
  }
  return __builtin_amdgcn_rcpf(1.f + e);
}

__device__ __forceinline__ int row_length(const int32_t *lengths, int64_t b, int64_t T) {
  if (!lengths) return (int)T;
  const int n = lengths[b];
  return n < 0 ? 0 : n > T ? (int)T : n;
}

// The sum of part[r, j] over the rows r, in a fixed order: called by a workgroup of
// kSumThreads for the kSumCols columns from kSumCols * blockIdx.x on. 64 threads a column,
// so that a thousand rows are 16 loads a thread. True in the one thread that has the sum
// of column j.
constexpr int kSumCols = 16, kSumThreads = 1024;
__device__ __forceinline__ bool sum_rows(const float *part, int64_t rows, int64_t cols, int64_t *col, float *sum) {
  constexpr int kSlots = kSumThreads / kSumCols;
  __shared__ float lds[kSlots][kSumCols];
  const int c = threadIdx.x % kSumCols, slot = threadIdx.x / kSumCols;
  const int64_t j = (int64_t)blockIdx.x * kSumCols + c;
  float s[8] = {};
  if (j < cols) {
    int64_t r = slot;
    for (; r + 7 * kSlots < rows; r += 8 * kSlots)
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += part[(r + i * kSlots) * cols + j];
    for (; r < rows; r += kSlots) s[0] += part[r * cols + j];
  }
  lds[slot][c] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
#pragma unroll
  for (int h = kSlots / 2; h; h /= 2) {
    if (slot < h) lds[slot][c] += lds[slot + h][c];
    __syncthreads();
  }
  *col = j;
  *sum = lds[0][c];
  return slot == 0 && j < cols;
}

inline bool aligned(const void *p, int64_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

inline size_t elem_size(int32_t type) { return type == ASTRA_SEQ_BF16 ? 2 : 4; }

}  // namespace astra_seq

#define ASTRA_SEQ_TYPE_CHECK(t)                      \
  do {                                               \
    ASTRA_ABI_CHECK(t, >=, ASTRA_SEQ_F32);           \
    ASTRA_ABI_CHECK(t, <=, ASTRA_SEQ_BF16);          \
  } while (false)

#define ASTRA_SEQ_POINTER(p)                                                                      \
  do {                                                                                            \
    if ((p) == nullptr)                                                                           \
      return astra_rt::fail(ASTRA_ERR_INVALID_ARGUMENT, std::string(__func__) + ": " #p " is NULL"); \
  } while (false)
