// sequence.h -- shared by the sequence operators' translation units: element types, wide
// loads and stores, sums over a wavefront or workgroup, and the sum over partial rows that
// ends every gradient of a parameter.
#pragma once

#include "astra_sequence.h"
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

// The sum over the 64 lanes, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

// The sum over TPR threads (a wavefront, or a whole workgroup through `lds`, TPR / 64
// words that nothing else uses; two calls in a row need two such areas).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float *lds) {
  v = wave_sum(v);
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

__device__ __forceinline__ float sigmoid(float v) { return 1.f / (1.f + __expf(-v)); }

__device__ __forceinline__ int row_length(const int32_t *lengths, int64_t b, int64_t T) {
  if (!lengths) return (int)T;
  const int n = lengths[b];
  return n < 0 ? 0 : n > T ? (int)T : n;
}

// The sum of part[r, j] over the rows r, in a fixed order: called by a workgroup of four
// wavefronts for the 64 columns from 64 * blockIdx.x on, each taking a quarter of the rows.
// True in the one thread that has the sum of column j.
__device__ __forceinline__ bool sum_rows(const float *part, int64_t rows, int64_t cols, int64_t *col, float *sum) {
  __shared__ float lds[4][kWave];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int64_t j = (int64_t)blockIdx.x * kWave + lane;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (j < cols) {
    int64_t r = w;
    for (; r + 12 < rows; r += 16) {
      s0 += part[r * cols + j];
      s1 += part[(r + 4) * cols + j];
      s2 += part[(r + 8) * cols + j];
      s3 += part[(r + 12) * cols + j];
    }
    for (; r < rows; r += 4) s0 += part[r * cols + j];
  }
  lds[w][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  *col = j;
  *sum = (lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane]);
  return w == 0 && j < cols;
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
