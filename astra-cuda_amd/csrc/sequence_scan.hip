// sequence_scan.hip -- the selective state space scan: per head a state h [P, N] that decays
// by exp(dt_t A) at every position and takes in dt_t x_t (x) B_t; read out as h_t C_t.
//
// Done position by position this is 5 P N vector operations a head and position, twenty
// times what moving x and y costs. Over a chunk of Q = 64 positions it is matrix products:
// with s the running sum of dt A from the chunk's start, h0 the state there,
//
//   M[i,j] = (C_i . B_j) exp(s_i - s_j) dt_j for j <= i,  + D on the diagonal
//   Y  = M X + exp(s) (C h0^T)                       (Q x Q) (Q x P) and (Q x N) (N x P)
//   h1 = exp(s_Q) h0 + X^T (w B), w_j = exp(s_Q - s_j) dt_j          (P x Q) (Q x N)
//
// and backwards, with dh1 the gradient of the state after the chunk,
//
//   dX = M^T dY + w (B dh1^T)
//   dC = Q B + exp(s) (dY h0),  Q[i,j] = (dY_i . x_j) exp(s_i - s_j) dt_j
//   dB = Q^T C + w (X dh1)
//   dh0 = exp(s_Q) dh1 + dY^T (exp(s) C)
//   d(dt A)_t = exp(s_Q) <dh1, h0> + sum_{j < t} w_j B_j . (dh1^T x_j)
//               + sum_{i >= t} exp(s_i) C_i . (h0^T dY_i) + sum_{j < t <= i} Q[i,j] (C_i . B_j)
//
// (the last of these is what crosses position t: summed as it stands, and not as differences
// of the shorter sums C.dC and B.dB, whose terms cancel)
// which run on the matrix cores. Every exponent is a difference s_i - s_j with j <= i, so
// nothing overflows where A <= 0; s is summed in 64 bits and kept as two floats, because a
// difference of two long sums would otherwise lose the digits that a short one has.
//
// Types. x, B, C and dY enter the products as they are; sums and states are in 32 bits. For
// bf16 inputs, what is computed in between enters a product as
//   - the sum of two (2^-18): the scores M and Q (with one, results of bf16 type were up to
//     1.1e-3 of their term further from 64 bits than their own rounding; the second part
//     costs 2 to 13% of a pass), and the states in y and dX. With one, the error of y goes with
//     |h| |C| and not with |h C|: a state whose values have a mean 16 times their spread, read
//     out by a C of zero mean, left 2.8e-2 of y where bf16's rounding is 1.7e-3;
//   - the sum of three (2^-26) in those that end in float results: w B and exp(s) C in states,
//     and the states in U = h0^T dY and V = dh1^T x, which are part of d(dt A).
// For float inputs the products use the float matrix instructions, at 1/16 of the bf16
// ones' rate.
// Against 64 bits, two records of 8,192: bf16 results 1.7e-3 (their own rounding), states'
// gradients 1e-7, dA 4e-7 to 7e-7, ddt_bias 2e-7 (the same in 32-bit torch operations: 2e-7,
// 4e-7 to 8e-7, 1.0e-6 to 1.3e-6).
//
// A chunk is handled by wavefronts that each own 16 of its positions. A product's result
// has its column in lane % 16 and four consecutive rows in its registers, which is the
// layout of an operand whose contracted index is those rows: scores are computed
// transposed, so that they enter the next product from registers.
#include "sequence.h"

#include <atomic>

#define ASTRA_SRC_NAME "sequence_scan.hip"

namespace astra_seq {
namespace {

constexpr int Q = 64;  // positions of a chunk

struct ScanArgs {
  const void *x, *dt, *b, *c, *dy;
  const float *A, *D, *bias, *initial, *dfinal;
  const int32_t *lengths;
  void *y, *dx, *ddt, *db, *dc;
  float *final_state, *dinitial;
  float *cs;        // [B, H, chunks, P, N]: the state before each chunk
  float *ds;        // likewise: the gradient of the state after each chunk
  float *seg;       // [B, H, segs, P, N]: what a segment of chunks adds, then what it starts from
  float *seg_log2;  // [B, H, segs]: log2 of a segment's decay
  float *part;      // [B * chunks, H, 3]: parts of dA, ddt_bias, dD
  float *dbc;       // [slices, 2, B, T, G, N]: parts of db and dc, where heads are split
  int64_t B, T;
  int64_t xsb, xst, xsh, dsb, dst, dsh, bsb, bst, bsg, csb, cst, csg;
  int32_t H, P, G, N, ptiles, chunks, seg_chunks, segs;
  int32_t parts;   // forward: workgroups that share a group's heads (and their tiles of P)
  int32_t slices;  // backward: likewise
  bool vec;  // 4 elements of every row can be accessed at once
};

// A kernel's arguments where they were passed, and the same for one more round of a loop:
// what the loop takes from them is loaded again (from the scalar cache) instead of being
// kept for all rounds, for which there are not enough scalar registers: they would be moved
// to and from lanes of vector registers, one instruction a word.
template <class A>
__device__ __forceinline__ const A *arguments() {
  return (const A *)__builtin_amdgcn_kernarg_segment_ptr();
}
template <class A>
__device__ __forceinline__ const A *again(const A *p) {
  typedef const __attribute__((address_space(4))) A *Constant;
  Constant c = (Constant)p;
  asm volatile("" : "+s"(c));
  return (const A *)c;
}

// ---------------------------------------------------------------- operands of the products

// One operand of a product over 32 values of the contracted index k, for lane (q = lane / 16,
// r = lane % 16): row (or column) r and 8 values of k. Which 8 is free as long as both
// operands agree: 8q..8q+7 ("near"), or 4q..4q+3 and 16+4q..16+4q+3 ("far"), which is how
// two results of 16 rows each hold them. Features of floats are near in the far order, so
// that a block with 16 or fewer of them is half the instructions.
struct FragF {
  float v[8];
};
template <class T>
struct Ops;

template <>
struct Ops<bf16> {
  using Frag = bf16x8;
  struct Split {
    bf16x8 hi, lo;
  };
  static __device__ __forceinline__ Frag near(const bf16 *row, int k0, int q) {
    return *reinterpret_cast<const bf16x8 *>(row + k0 + 8 * q);
  }
  static __device__ __forceinline__ Frag far(const bf16 *row, int k0, int q) {
    const bf16x4 a = *reinterpret_cast<const bf16x4 *>(row + k0 + 4 * q);
    const bf16x4 b = *reinterpret_cast<const bf16x4 *>(row + k0 + 16 + 4 * q);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
  struct Split3 {
    bf16x8 hi, mid, lo;
  };
  static __device__ __forceinline__ Split split(const float (&v)[8]) {
    Split s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s.hi[i] = (bf16)v[i];
      s.lo[i] = (bf16)(v[i] - (float)s.hi[i]);
    }
    return s;
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Split &b) {
    mma(acc, a, b.lo);
    mma(acc, a, b.hi);
  }
  static __device__ __forceinline__ Split3 split3(const float (&v)[8]) {
    Split3 s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s.hi[i] = (bf16)v[i];
      const float rest = v[i] - (float)s.hi[i];
      s.mid[i] = (bf16)rest;
      s.lo[i] = (bf16)(rest - (float)s.mid[i]);
    }
    return s;
  }
  static __device__ __forceinline__ void expand(const Frag &f, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)f[i];
  }
  // zeros in the place of what is not finite
  static __device__ __forceinline__ void finite(Frag &f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)f[i] - (float)f[i] == 0.f ? f[i] : (bf16)0.f;
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Split &a, const Frag &b) {
    mma(acc, a.lo, b);
    mma(acc, a.hi, b);
  }
  // a product over features of which `left` are left: nothing is saved within a block
  template <class A, class B>
  static __device__ __forceinline__ void mma_left(f32x4 &acc, const A &a, const B &b, int) {
    mma(acc, a, b);
  }
  // The small parts are added up by themselves, and to the result by the caller: a sum that is
  // much smaller or larger than the products that it is added to is rounded down, by 0.13 or
  // 0.04 2^-24 of the result on average (measured; 0.01 where they are alike), and sums over
  // many positions drift.
  static __device__ __forceinline__ void mma_apart(f32x4 &acc, f32x4 &small, const Split3 &a, const Frag &b) {
    mma(small, a.lo, b);
    mma(small, a.mid, b);
    mma(acc, a.hi, b);
  }
};

template <>
struct Ops<float> {
  using Frag = FragF;
  using Split = FragF;
  using Split3 = FragF;
  static __device__ __forceinline__ Frag near(const float *row, int k0, int q) {
    Frag f;
    const f32x4 a = *reinterpret_cast<const f32x4 *>(row + k0 + 4 * q);
    const f32x4 b = *reinterpret_cast<const f32x4 *>(row + k0 + 16 + 4 * q);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f.v[i] = a[i];
      f.v[4 + i] = b[i];
    }
    return f;
  }
  static __device__ __forceinline__ Split split(const float (&v)[8]) {
    Split s;
#pragma unroll
    for (int i = 0; i < 8; ++i) s.v[i] = v[i];
    return s;
  }
  static __device__ __forceinline__ Split3 split3(const float (&v)[8]) { return split(v); }
  static __device__ __forceinline__ void finite(Frag &f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = f.v[i] - f.v[i] == 0.f ? f.v[i] : 0.f;
  }
  static __device__ __forceinline__ void expand(const Frag &f, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f.v[i];
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Frag &b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma_apart(f32x4 &acc, f32x4 &, const Frag &a, const Frag &b) { mma(acc, a, b); }
  // a product over two tiles of positions with the own one last: the second, before which the
  // first one is zero, or the first
  static __device__ __forceinline__ void mma_own(f32x4 &acc, const Frag &a, const Frag &b, int second) {
#pragma unroll
    for (int i = 4; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
    if (second) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma_left(f32x4 &acc, const Frag &a, const Frag &b, int left) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
    if (left <= 16) return;
#pragma unroll
    for (int i = 4; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
  }
};

template <class T>
struct V4 {
  typedef T type __attribute__((ext_vector_type(4)));
};

// Whether the 16 (or 32) rows, columns or contracted values from `at` on hold any of the `n`
// that count, and how many are left of them. Looked at for floats with up to 32 states only,
// where a state of 16 halves the products: in the larger tiles, and for bf16, the branches
// cost more registers than the skipped instructions are worth.
template <class T, int NT>
__device__ __forceinline__ bool on(int at, int n) {
  return !(sizeof(T) == 4 && NT == 32) || at < n;
}
template <class T, int NT>
__device__ __forceinline__ int rest(int n) {
  return sizeof(T) == 4 && NT == 32 ? n : 32;
}

// A tile of F features by Q positions in LDS, read along its features (`rows`: position
// major) or along its positions. bf16 operands are read 16 bytes at a time, so each order
// that is read needs a copy of its own (`cols`: feature major); floats are read one by one
// along the positions, 16 neighbouring features at once.
template <class T, int F>
struct Tile {
  static constexpr bool kTwo = sizeof(T) == 2;
  static constexpr int kRow = F + 16 / (int)sizeof(T);  // padded pitch of a position's features
  static constexpr int kCol = Q + 8;                    // padded pitch of a feature's positions
  static constexpr size_t kRowsBytes = Q * kRow * sizeof(T);
  static constexpr size_t kColsBytes = kTwo ? F * kCol * sizeof(T) : 0;
};
template <class T, int F>
struct Along {  // operands contracted over positions
  const T *rows, *cols;
  __device__ __forceinline__ float one(int f, int t) const {
    if constexpr (sizeof(T) == 2) return (float)cols[f * Tile<T, F>::kCol + t];
    return (float)rows[t * Tile<T, F>::kRow + f];
  }
  __device__ __forceinline__ typename Ops<T>::Frag near(int f, int t0, int q) const {
    if constexpr (sizeof(T) == 2) {
      return Ops<T>::near(cols + f * Tile<T, F>::kCol, t0, q);
    } else {
      FragF r;
#pragma unroll
      for (int i = 0; i < 8; ++i) r.v[i] = rows[(t0 + 8 * q + i) * Tile<T, F>::kRow + f];
      return r;
    }
  }
  __device__ __forceinline__ typename Ops<T>::Frag far(int f, int t0, int q) const {
    if constexpr (sizeof(T) == 2) {
      return Ops<T>::far(cols + f * Tile<T, F>::kCol, t0, q);
    } else {
      FragF r;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        r.v[i] = rows[(t0 + 4 * q + (i & 3) + 16 * (i >> 2)) * Tile<T, F>::kRow + f];
      return r;
    }
  }
};

// A state tile [R, K] (K contracted) in LDS: the bf16 parts whose sum it is, or floats. bf16 rows
// of 64 and of 256 bytes, of which every fourth or each starts on the same bank, are not padded:
// their 16-byte blocks change places by row (so that two workgroups of the forward kernel, and
// one of the gradient's, with 128 states fit a CU's LDS).
template <class T, int R, int K, int PARTS>
struct StateTile {
  static constexpr int kParts = sizeof(T) == 2 ? PARTS : 1;
  static constexpr int kSwapped = sizeof(T) == 2 && (K == 128 || K == 32) ? K : 0;
  static constexpr int kRow = kSwapped ? K : K + 16 / (int)sizeof(T);
  static constexpr int kPart = R * kRow;
  static constexpr size_t kBytes = kParts * kPart * sizeof(T);
  T *p;
  static __device__ __forceinline__ int at(int r, int k) {
    if constexpr (kSwapped == 128) return r * kRow + (k ^ (r & 15) << 3);
    if constexpr (kSwapped == 32) return r * kRow + (k ^ (r >> 2 & 3) << 3);
    return r * kRow + k;
  }
  __device__ __forceinline__ auto near(int r, int k0, int q) const {
    if constexpr (kParts == 1) {
      return Ops<T>::near(p + r * kRow, k0, q);
    } else {
      const T *const o = p + at(r, k0 + 8 * q);
      if constexpr (kParts == 2) {
        return typename Ops<T>::Split{Ops<T>::near(o, 0, 0), Ops<T>::near(o + kPart, 0, 0)};
      } else {
        return typename Ops<T>::Split3{Ops<T>::near(o, 0, 0), Ops<T>::near(o + kPart, 0, 0), Ops<T>::near(o + 2 * kPart, 0, 0)};
      }
    }
  }
  // contracted over the rows instead (floats only)
  __device__ __forceinline__ FragF across(int k, int r0, int q) const {
    FragF s;
#pragma unroll
    for (int i = 0; i < 8; ++i) s.v[i] = p[(r0 + 4 * q + (i & 3) + 16 * (i >> 2)) * kRow + k];
    return s;
  }
  __device__ __forceinline__ void put4(int r, int k, const float (&v)[4]) const {
    T *const o = p + at(r, k);
    float left[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
    for (int j = 0; j < kParts; ++j) {
      typename V4<T>::type part;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        part[i] = (T)left[i];
        left[i] -= (float)part[i];
      }
      *reinterpret_cast<typename V4<T>::type *>(o + j * kPart) = part;
    }
  }
  // the first N parts of 4 values, as floats
  template <int N>
  __device__ __forceinline__ void get4(int r, int k, float (&v)[4]) const {
    const T *const o = p + at(r, k);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = 0.f;
#pragma unroll
    for (int j = 0; j < (N < kParts ? N : kParts); ++j) {
      const typename V4<T>::type part = *reinterpret_cast<const typename V4<T>::type *>(o + j * kPart);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += (float)part[i];
    }
  }
};

// ---------------------------------------------------------------------- global memory

// A matrix of rows in memory, `n` elements of each counting. VEC: four neighbouring elements
// are one access through a buffer descriptor, whose bounds check (a byte offset of this
// descriptor's size or more reads zeros and writes nothing) stands in for a branch per row;
// needs n, the stride and the address to be multiples of four, and n <= stride < 2^23.
// Otherwise elements go one by one.
constexpr unsigned kOutside = 0x80000000u;  // beyond any descriptor, also after some rows are added
template <class T, bool VEC>
struct Matrix {
  T *base;
  int64_t stride;
  int rows, n;
  __amdgpu_buffer_rsrc_t rsrc;
  __device__ __forceinline__ Matrix(const T *p, int64_t stride_, int64_t rows_, int n_)
      : base(const_cast<T *>(p)), stride(stride_), rows(rows_ < 0 ? 0 : rows_ > Q ? Q : (int)rows_), n(n_) {
    if constexpr (VEC) {
      // (the clamps are done by vector operations, although they are the same in every lane)
      rows = __builtin_amdgcn_readfirstlane(rows);
      const int bytes = rows ? ((rows - 1) * (int)stride + n) * (int)sizeof(T) : 0;
      rsrc = __builtin_amdgcn_make_buffer_rsrc(base, 0, bytes, 0x00020000);
    }
  }
  // the offset of four elements from (row, f) on, for load and store
  __device__ __forceinline__ unsigned at(int row, int f) const {
    return f < n ? (unsigned)(row * (int)stride + f) * (unsigned)sizeof(T) : kOutside;
  }
  __device__ __forceinline__ typename V4<T>::type load(int row, int f, unsigned off) const {
    typename V4<T>::type r = {};
    if constexpr (VEC && sizeof(T) == 2) {
      r = __builtin_bit_cast(typename V4<T>::type, __builtin_amdgcn_raw_buffer_load_b64(rsrc, off, 0, 0));
    } else if constexpr (VEC) {
      r = __builtin_bit_cast(typename V4<T>::type, __builtin_amdgcn_raw_buffer_load_b128(rsrc, off, 0, 0));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row < rows && f + i < n) r[i] = base[row * stride + f + i];
    }
    return r;
  }
  __device__ __forceinline__ typename V4<T>::type load(int row, int f) const { return load(row, f, at(row, f)); }
  // the first element of a row
  __device__ __forceinline__ T load1(int row) const {
    const unsigned off = (unsigned)(row * (int)stride) * (unsigned)sizeof(T);
    if constexpr (VEC && sizeof(T) == 2)
      return __builtin_bit_cast(T, (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rsrc, off, 0, 0));
    else if constexpr (VEC)
      return __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(rsrc, off, 0, 0));
    else
      return row < rows ? base[row * stride] : (T)0.f;
  }
  __device__ __forceinline__ void store(int row, int f, const float (&v)[4]) const {
    typename V4<T>::type r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
    if constexpr (VEC && sizeof(T) == 2) {
      typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, r), rsrc, at(row, f), 0, 0);
    } else if constexpr (VEC) {
      typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
      __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, r), rsrc, at(row, f), 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (row < rows && f + i < n) base[row * stride + f + i] = r[i];
    }
  }
};

// F features by Q positions on their way from memory to LDS: THREADS threads hold blocks of
// 4 positions by 4 features. What lies beyond the matrix is zero, whatever memory holds there.
// Eight neighbouring lanes have neighbouring features, the next eight the next positions:
// 64 bytes of a row at once, and writes along the positions that meet two to a bank instead
// of the four that whole rows of 64 features would.
template <class T, int F, int THREADS, bool VEC>
struct Stage {
  static_assert(F % 32 == 0 && Q == 64, "eight groups of features by sixteen of positions");
  static constexpr int kBlocks = (F / 4) * (Q / 4), kEach = (kBlocks + THREADS - 1) / THREADS;
  static __device__ __forceinline__ int f_of(int blk) { return ((blk & 7) | (blk >> 7) << 3) * 4; }
  static __device__ __forceinline__ int t_of(int blk) { return ((blk >> 3) & 15) * 4; }
  typename V4<T>::type v[kEach][4];
  __device__ __forceinline__ void load(const Matrix<T, VEC> &m, int tid) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS;
      const int f = f_of(blk), t = t_of(blk);
      unsigned off = blk < kBlocks ? m.at(t, f) : kOutside;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[e][k] = {};
        if (VEC || blk < kBlocks) v[e][k] = m.load(t + k, f, off);
        off += (unsigned)m.stride * (unsigned)sizeof(T);
      }
    }
  }
  __device__ __forceinline__ void put(T *rows, T *cols, int tid) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS;
      if (kBlocks % THREADS && blk >= kBlocks) continue;
      const int f = f_of(blk), t = t_of(blk);
      if (rows) {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<typename V4<T>::type *>(rows + (t + k) * Tile<T, F>::kRow + f) = v[e][k];
      }
      if (Tile<T, F>::kTwo && cols) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          typename V4<T>::type w;
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = v[e][k][i];
          *reinterpret_cast<typename V4<T>::type *>(cols + (f + i) * Tile<T, F>::kCol + t) = w;
        }
      }
    }
  }
};

// A row's 8 elements of a near operand from feature f on, read from memory as they are.
template <class T, bool VEC>
__device__ __forceinline__ typename Ops<T>::Frag load_near(const Matrix<T, VEC> &m, int row, int f, int q) {
  const bool far = sizeof(T) == 4;
  const typename V4<T>::type a = m.load(row, f + (far ? 4 : 8) * q), b = m.load(row, f + (far ? 16 + 4 * q : 8 * q + 4));
  typename Ops<T>::Frag r;
  if constexpr (sizeof(T) == 2) {
    r = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r.v[i] = a[i];
      r.v[4 + i] = b[i];
    }
  }
  return r;
}

// ------------------------------------------------------------------------- step sizes

// What one wavefront, a lane a position, works out of a head's dt over a chunk.
struct Times {
  float dt[Q], hi[Q], lo[Q];  // the step; log2 of the decay from the chunk's start, in two parts
  float from[Q];              // exp(s_t)
  float into[Q];              // dt exp(s_Q - s_t): what a position's input counts after the chunk
  // Between tiles of 16 positions exp(s_i - s_j) is a product by way of the end e of j's
  // tile (both factors are at most 1 where A <= 0, and small only where the product is):
  float after[48 + 32 + 16];  // exp(s_i - s_e) for the i after tile 0, 1, 2
  float till[Q];              // exp(s_e - s_j) dt_j for j's own tile
  float total;                // exp(s_Q)
  float nowhere[3];
  // `after` of a tile, such that position i's is at [i] (i >= 16 (tile + 1))
  static __device__ __forceinline__ int past_at(int tile) { return tile == 0 ? -16 : tile == 1 ? 48 - 32 : 80 - 48; }
  __device__ __forceinline__ float past(int tile, int i) const { return after[past_at(tile) + i]; }
};
struct GradTimes : Times {
  float left[Q];   // exp(s_Q - s_t)
  float slope[Q];  // the step's derivative by dt_raw, 0 where no position counts
};

__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

// dt of a head's positions from t0 on, a lane a position, before its bias.
template <class T, bool VEC>
__device__ __forceinline__ T raw_step(const ScanArgs &a, int64_t b, int h, int64_t t0, int len, int lane) {
  return Matrix<T, VEC>((const T *)a.dt + b * a.dsb + t0 * a.dst + h * a.dsh, a.dst, len - t0, 1).load1(lane);
}

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ double moved64(double v) {
  const int64_t i = __builtin_bit_cast(int64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)i, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(i >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// v of one lane, in all of them.
__device__ __forceinline__ double lane64(double v, int lane) {
  const int64_t i = __builtin_bit_cast(int64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)i, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(i >> 32), lane);
  return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// Fills `o` from this lane's dt and the head's bias and A; returns log2 of the chunk's decay.
template <class O>
__device__ __forceinline__ double make_times(O &o, float dt_raw, float bias, bool live, float A, int lane) {
  const float raw = dt_raw + bias, dt = live ? softplus(raw) : 0.f;
  // No position lets less through than nothing: 2^-2000 is 0 in 32 bits, and a bound keeps sums
  // and differences of these finite where A is not (a head without memory).
  double s = dt > 0.f ? (double)dt * (double)A * 1.4426950408889634 : 0.;
  s = s < -2000. ? -2000. : s;
  s += moved64<kUp + 1>(s);
  s += moved64<kUp + 2>(s);
  s += moved64<kUp + 4>(s);
  s += moved64<kUp + 8>(s);
  s += moved64<kBcast15, 0xa>(s);
  s += moved64<kBcast31, 0xc>(s);
  double ends[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    ends[i] = lane64(s, 16 * i + 15);
    // (the other lanes' go nowhere: a place to put them costs less than a branch around them)
    if (i < 3) *(lane >= 16 * (i + 1) ? o.after + Times::past_at(i) + lane : o.nowhere) = __builtin_amdgcn_exp2f((float)(s - ends[i]));
  }
  const double total = ends[3];
  const float left = __builtin_amdgcn_exp2f((float)(total - s));
  const double end = lane < 32 ? (lane < 16 ? ends[0] : ends[1]) : (lane < 48 ? ends[2] : ends[3]);
  o.till[lane] = dt * __builtin_amdgcn_exp2f((float)(end - s));
  o.dt[lane] = dt;
  o.hi[lane] = (float)s;
  o.lo[lane] = (float)(s - (double)(float)s);
  o.from[lane] = __builtin_amdgcn_exp2f((float)s);
  o.into[lane] = dt * left;
  if constexpr (sizeof(O) == sizeof(GradTimes)) {
    o.left[lane] = left;
    o.slope[lane] = live ? sigmoid<float>(raw) : 0.f;
  }
  if (lane == 0) o.total = __builtin_amdgcn_exp2f((float)total);
  return total;
}

// Workgroups go to the eight XCDs in turn: neighbours in this order share an XCD, and with it
// the L2 that holds the B and C that they share.
__device__ __forceinline__ int64_t workgroup_id() {
  const unsigned n = gridDim.x, id = blockIdx.x;
  return n % 8 ? id : (id % 8) * (n / 8) + id / 8;
}

// --------------------------------------------------------- the states' update over a chunk

// A wavefront's part of a state [PT, NT] in registers, WAVES of them sharing it: 16 x 16 tiles
// wave, wave + WAVES, ... of [p tile, n tile]; lane (q, r) of tile (pt, nt) has
// n = 16 nt + 4 q + 0..3 and p = 16 pt + r.
template <int PT, int NT, int WAVES>
struct Mine {
  static constexpr int kN = NT / 16, kTiles = (PT / 16) * kN, kEach = kTiles / WAVES;
  static constexpr bool kOneN = WAVES % kN == 0;  // one tile of n for all of a wavefront's tiles
  static_assert(kTiles % WAVES == 0, "the wavefronts share the tiles evenly");
  static __device__ __forceinline__ int nt_of(int wave, int i) { return (wave + WAVES * i) % kN; }
  static __device__ __forceinline__ int n_of(int wave, int i, int q) { return nt_of(wave, i) * 16 + 4 * q; }
  static __device__ __forceinline__ int p_of(int wave, int i, int r) { return ((wave + WAVES * i) / kN) * 16 + r; }
};

// S = total S + X^T (weight K): X over PT features of which `np` count, K over NT of which
// `nn` count, weight a position's. What the small parts of K give is added to S at the end, or
// (TWICE) after each half of the positions, for kernels that have no registers to keep it in.
template <class T, int PT, int NT, int WAVES, bool TWICE>
__device__ __forceinline__ void update_state(f32x4 *S, float total, const float *weight, const Along<T, PT> &X,
                                             const Along<T, NT> &K, int wave, int q, int r, int np, int nn) {
  using M = Mine<PT, NT, WAVES>;
  constexpr bool kSmall = sizeof(T) == 2;
  f32x4 small[M::kEach];
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) {
    S[i] *= total;
    small[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
#pragma unroll
  for (int t0 = 0; t0 < Q; t0 += 32) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = weight[t0 + 8 * q + e];
    typename Ops<T>::Split3 kf;
#pragma unroll
    for (int i = 0; i < M::kEach; ++i) {
      if (!on<T, NT>(16 * M::nt_of(wave, i), nn) || !on<T, NT>(M::p_of(wave, i, 0), np)) continue;
      if (i == 0 || !M::kOneN) {
        float v[8];
        Ops<T>::expand(K.near(16 * M::nt_of(wave, i) + r, t0, q), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= w[e];
        kf = Ops<T>::split3(v);
      }
      if (TWICE) small[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      Ops<T>::mma_apart(S[i], small[i], kf, X.near(M::p_of(wave, i, r), t0, q));
      if (kSmall && TWICE) S[i] += small[i];
    }
  }
  if (kSmall && !TWICE) {
#pragma unroll
    for (int i = 0; i < M::kEach; ++i) S[i] += small[i];
  }
}

// The PT features from p0 on of a state [P, N], nothing where there is none.
template <bool VEC>
__device__ __forceinline__ Matrix<float, VEC> state_rows(const float *base, const ScanArgs &a, int p0) {
  return Matrix<float, VEC>(base ? base + (int64_t)p0 * a.N : nullptr, a.N, base ? a.P - p0 : 0, a.N);
}
template <int PT, int NT, int WAVES, bool VEC>
__device__ __forceinline__ void load_state(f32x4 *S, const float *base, const ScanArgs &a, int p0, int wave, int q, int r) {
  using M = Mine<PT, NT, WAVES>;
  const Matrix<float, VEC> m = state_rows<VEC>(base, a, p0);
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) S[i] = m.load(M::p_of(wave, i, r), M::n_of(wave, i, q));
}
template <int PT, int NT, int WAVES, bool VEC>
__device__ __forceinline__ void store_state(const f32x4 *S, float *base, const ScanArgs &a, int p0, int wave, int q, int r) {
  using M = Mine<PT, NT, WAVES>;
  const Matrix<float, VEC> m = state_rows<VEC>(base, a, p0);
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) {
    const float v[4] = {S[i][0], S[i][1], S[i][2], S[i][3]};
    m.store(M::p_of(wave, i, r), M::n_of(wave, i, q), v);
  }
}

// ------------------------------------------------------------------------ forward

template <class T, int PT, int NT, bool ST>
struct ForwardLds {
  static constexpr size_t x = 0;  // along positions only
  static constexpr size_t bn = x + (sizeof(T) == 2 ? Tile<T, PT>::kColsBytes : Tile<T, PT>::kRowsBytes);
  static constexpr size_t bt = bn + Tile<T, NT>::kRowsBytes;
  static constexpr size_t h = bt + Tile<T, NT>::kColsBytes;
  static constexpr size_t times = h + (ST ? StateTile<T, PT, NT, 2>::kBytes : 0);
  static constexpr size_t bytes = times + 2 * sizeof(Times);
};

// Wavefronts a SIMD that the kernel's registers leave room for. Measured both ways for every
// tile, with four heads and 40 positions (no states) or 200 (states):
//   floats  4 with up to 32 states (64 x 32: 55 us against 62 with 2; rows that allow single
//           elements only: 133 against 181), else 2 (64 x 64 with states 65 against 90 with 4)
//   bf16    4 (64 x 128 with states 66 us against 73 with 3), but 3 where 4 would spill within
//           an item: 32 x 128 (44 against 73), and 64 x 64 without states, whose scores stay in
//           registers over a workgroup's heads (2,048 games with eight heads, forward and
//           gradient: 336 us against 338; a workgroup with one head is better with 4, 22
//           against 28)
template <class T, int PT, int NT, bool ST>
constexpr int forward_waves() {
  if (sizeof(T) == 4) return NT == 32 ? 4 : 2;
  return (PT == 32 && NT == 128) || (PT == 64 && NT == 64 && !ST) ? 3 : 4;
}

// A workgroup of 4 PW wavefronts: a segment of chunks of one row, for some of a group's heads
// (and tiles of PT features) in turn. Wavefront w has positions 16 (w % 4) + 0..15 and the
// (w / 4)th part of the features. While an item (a head's chunk) is computed, the next one's
// inputs are on their way to registers, and the first wavefront, which has the fewest pairs
// of positions, works out its step sizes. Where the segment is a single chunk, B, C and their
// scores are loaded and computed once for all heads. ST: whether there are states before a chunk.
// Positions that do not exist are worked on like others, up to the chunk's 64. A segment of
// several chunks is one head's, which stages B and C and computes the scores for itself.
// Bound by latency and issue between the two barriers of an item, not by traffic: 2,048 games
// of 40 positions (8 heads of 64, 64 states) 154 us where their bytes, final states among them,
// take 97 at a large copy's 4.7 TB/s; a record of 65,536 (16 heads of 64, 128 states) 300 after
// 119 for the segments' states, where its bytes take 64 and the products of both, some 160
// GFLOP, 133. Counters of the two: vector units busy 39 and 45% of the time, matrix units 10 and
// 17, LDS 22 and 38 (nearly half of it conflicts), 2.3 and 3.4 wavefronts a SIMD.
template <class T, int PT, int NT, int PW, bool ST, bool VEC>
__global__ __launch_bounds__(256 * PW, (forward_waves<T, PT, NT, ST>())) void scan_forward_kernel(ScanArgs args) {
  (void)args;
  const ScanArgs *ap = arguments<ScanArgs>();
  using L = ForwardLds<T, PT, NT, ST>;
  constexpr int kThreads = 256 * PW, kWaves = 4 * PW, PP = PT / PW;
  using M = Mine<PT, NT, kWaves>;
  extern __shared__ __align__(16) char lds[];
  T *xl = (T *)(lds + L::x), *bn = (T *)(lds + L::bn), *bt = (T *)(lds + L::bt);
  const StateTile<T, PT, NT, 2> hl{(T *)(lds + L::h)};
  Times *times = (Times *)(lds + L::times);
  const Along<T, PT> xa{xl, xl};
  const Along<T, NT> ba{bn, bt};

  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wi = wave & 3, f0 = (wave >> 2) * PP;
  const int ti = 16 * wi + r;  // this lane's position
  int64_t id = workgroup_id();
  const int per = ap->H / ap->G, heads = per * ap->ptiles;  // a group's heads and tiles of features
  const int part = (int)(id % ap->parts);
  id /= ap->parts;
  const int g = (int)(id % ap->G);
  id /= ap->G;
  const int seg = (int)(id % ap->segs);
  const int64_t b = id / ap->segs;
  const int len = row_length(ap->lengths, b, ap->T);
  const int c0 = seg * ap->seg_chunks, c1 = min(c0 + ap->seg_chunks, ap->chunks);
  const int last = (int)((int64_t)heads * (part + 1) / ap->parts);
  const int64_t pn = (int64_t)ap->P * ap->N;
  const T *bg = (const T *)ap->b + b * ap->bsb + g * ap->bsg;
  const T *cg = (const T *)ap->c + b * ap->csb + g * ap->csg;

  Stage<T, PT, kThreads, VEC> xs;
  Stage<T, NT, kThreads, VEC> bs;
  typename Ops<T>::Frag cf[NT / 32];  // this position's C, read as it is used
  T raw = (T)0.f;
  // the item that is loaded next: a head, its tile of features and a chunk
  int hp = (int)((int64_t)heads * part / ap->parts), c = c0;
  int h = g * per + hp / ap->ptiles, pt = hp % ap->ptiles;
  const T *xg = (const T *)ap->x + b * ap->xsb + (int64_t)c0 * Q * ap->xst;
  auto load = [&](bool with_bc) __attribute__((always_inline)) {
    const int64_t t0 = (int64_t)c * Q;
    xs.load(Matrix<T, VEC>(xg + (t0 - (int64_t)c0 * Q) * ap->xst + h * ap->xsh + pt * PT, ap->xst, len - t0, ap->P - pt * PT), tid);
    if (with_bc) bs.load(Matrix<T, VEC>(bg + t0 * ap->bst, ap->bst, len - t0, ap->N), tid);
    if (wave == 0) raw = raw_step<T, VEC>(*ap, b, h, t0, len, lane);
  };
  auto load_c = [&]() __attribute__((always_inline)) {
    const int64_t t0 = (int64_t)c * Q;
    const Matrix<T, VEC> cm(cg + t0 * ap->cst, ap->cst, len - t0, ap->N);
#pragma unroll
    for (int n = 0; n < NT / 32; ++n) cf[n] = load_near(cm, ti, 32 * n, q);
  };
  auto step = [&](int k) __attribute__((always_inline)) {
    make_times(times[k & 1], (float)raw, ap->bias ? ap->bias[h] : 0.f, (int64_t)c * Q + lane < len, ap->A[h], lane);
  };
  if (hp >= last) return;
  load(true);
  load_c();
  if (wave == 0) step(0);

  f32x4 S[M::kEach], sc[4];
  bool fresh = true, any = false;
  for (int k = 0;; ++k) {
    ap = again(ap);
    const int p0 = pt * PT, cc = c, h_now = h;
    const int64_t t0 = (int64_t)c * Q, bh = b * ap->H + h;
    const bool new_bc = fresh || c1 - c0 > 1;
    const Times &tm = times[k & 1];
    if (k) __syncthreads();  // nobody reads the last item's tiles any more
    if constexpr (sizeof(T) == 2)
      xs.put(nullptr, xl, tid);
    else
      xs.put(xl, nullptr, tid);
    if (new_bc) bs.put(bn, bt, tid);
    if (c == c0) {
      const float *start = !ST ? nullptr : ap->segs > 1 ? ap->seg + (bh * ap->segs + seg) * pn : ap->initial ? ap->initial + bh * pn : nullptr;
      any = start != nullptr;
      if (any) {
        load_state<PT, NT, kWaves, VEC>(S, start, *ap, p0, wave, q, r);
      } else {
#pragma unroll
        for (int i = 0; i < M::kEach; ++i) S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
    }
    if constexpr (ST) {
      if (any) {
#pragma unroll
        for (int i = 0; i < M::kEach; ++i) {
          const float v[4] = {S[i][0], S[i][1], S[i][2], S[i][3]};
          hl.put4(M::p_of(wave, i, r), M::n_of(wave, i, q), v);
        }
      }
      if (ap->cs) store_state<PT, NT, kWaves, VEC>(S, ap->cs + (bh * ap->chunks + c) * pn, *ap, p0, wave, q, r);
    }
    __syncthreads();
    if (++c == c1) {
      c = c0;
      ++hp;
      if (++pt == ap->ptiles) {
        pt = 0;
        ++h;
      }
    }
    const bool more = hp < last;
    if (more) load(c1 - c0 > 1);

    // this wavefront's 16 positions i = 16 wi + r: first M^T, two tiles of j to an operand
    auto scores = [&](int jt) __attribute__((always_inline)) {
      f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int n = 0; n < NT / 32; ++n)
        if (on<T, NT>(32 * n, ap->N))
          Ops<T>::mma_left(v, Ops<T>::near(bn + (16 * jt + r) * Tile<T, NT>::kRow, 32 * n, q), cf[n], rest<T, NT>(ap->N - 32 * n));
      return v;
    };
    if constexpr (!ST) {
      if (new_bc) {
#pragma unroll
        for (int jt = 0; jt < 4; ++jt)
          if (jt <= wi) sc[jt] = scores(jt);
      }
    }
    fresh = false;
    const float hi = tm.hi[ti], lo = tm.lo[ti], D = ap->D ? ap->D[h_now] : 0.f;
    typename Ops<T>::Split mf[2];
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
      if (2 * jp > wi) break;
      float m[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int jt = 2 * jp + half;
        if (jt > wi) {
#pragma unroll
          for (int e = 0; e < 4; ++e) m[4 * half + e] = 0.f;
          continue;
        }
        const f32x4 g = ST ? scores(jt) : sc[jt];
        if (jt < wi) {
          const float past = tm.past(jt, ti);
          const f32x4 till = *reinterpret_cast<const f32x4 *>(tm.till + 16 * jt + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) m[4 * half + e] = g[e] * (past * till[e]);
          continue;
        }
        // the only tile with pairs j > i, and the diagonal
        const f32x4 thi = *reinterpret_cast<const f32x4 *>(tm.hi + 16 * jt + 4 * q);
        const f32x4 tlo = *reinterpret_cast<const f32x4 *>(tm.lo + 16 * jt + 4 * q);
        const f32x4 tdt = *reinterpret_cast<const f32x4 *>(tm.dt + 16 * jt + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int ahead = 4 * q + e - r;
          const float v = g[e] * (__builtin_amdgcn_exp2f((hi - thi[e]) + (lo - tlo[e])) * tdt[e]);
          m[4 * half + e] = ahead > 0 ? 0.f : ahead == 0 ? v + D : v;
        }
      }
      mf[jp] = Ops<T>::split(m);
    }
    // then Y^T, 16 features at a time. A product over positions has a factor of 0 for those that
    // come later, which 0 * inf makes a NaN of: where a result is not finite, the tiles are done
    // once more with what is not finite in X left out where it does not count, and zeros after
    // the row's end (where C is 0, but the state may not be finite).
    const Matrix<T, VEC> ym((const T *)ap->y + ((b * ap->T + t0) * ap->H + h_now) * ap->P + p0, (int64_t)ap->H * ap->P, ap->T - t0, ap->P - p0);
    const float from = tm.from[ti];
    auto before = [&](int i) __attribute__((always_inline)) {  // what the state before the chunk gives
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      if constexpr (ST) {
        if (any) {
#pragma unroll
          for (int n = 0; n < NT / 32; ++n)
            if (on<T, NT>(32 * n, ap->N)) Ops<T>::mma_left(y, hl.near(f0 + 16 * i + r, 32 * n, q), cf[n], rest<T, NT>(ap->N - 32 * n));
          y *= from;
        }
      }
      return y;
    };
    float odd = 0.f;  // 0, or NaN where a result is not finite
#pragma unroll
    for (int i = 0; i < PP / 16; ++i) {
      if (!on<T, NT>(f0 + 16 * i, ap->P - p0)) continue;
      f32x4 y = before(i);
      Ops<T>::mma(y, xa.far(f0 + 16 * i + r, 0, q), mf[0]);
      if (wi > 1) Ops<T>::mma(y, xa.far(f0 + 16 * i + r, 32, q), mf[1]);
      const float v[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
      for (int e = 0; e < 4; ++e) odd += v[e] - v[e];
      ym.store(ti, f0 + 16 * i + 4 * q, v);
    }
    if (__builtin_expect(__any(!(odd == 0.f)), 0)) {
#pragma unroll 1
      for (int i = 0; i < PP / 16; ++i) {
        if (!on<T, NT>(f0 + 16 * i, ap->P - p0)) continue;
        f32x4 all = before(i), kept = all;
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
          if (2 * jp > wi) break;
          typename Ops<T>::Frag x = xa.far(f0 + 16 * i + r, 32 * jp, q);
          Ops<T>::mma(all, x, mf[jp]);
          Ops<T>::finite(x);
          Ops<T>::mma(kept, x, mf[jp]);
        }
        float v[4] = {kept[0], kept[1], kept[2], kept[3]};
#pragma unroll 1
        for (int j = 0; j <= ti; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = xa.one(f0 + 16 * i + 4 * q + e, j);
            if (!(x - x == 0.f)) v[e] = all[e];
          }
        if (t0 + ti >= len) v[0] = v[1] = v[2] = v[3] = 0.f;
        ym.store(ti, f0 + 16 * i + 4 * q, v);
      }
    }
    if (more && c1 - c0 > 1) load_c();  // this item's is done with
    if (cc + 1 < c1 || ap->final_state) {
      update_state<T, PT, NT, kWaves, true>(S, tm.total, tm.into, xa, ba, wave, q, r, ap->P - p0, ap->N);
      any = true;
      if (ap->final_state && cc + 1 == ap->chunks) store_state<PT, NT, kWaves, VEC>(S, ap->final_state + bh * pn, *ap, p0, wave, q, r);
    }
    if (!more) break;
    if (wave == 0) step(k + 1);
  }
}

// ----------------------------------------------------------------- states of segments

template <class T, int PT, int NT>
struct StatesLds {
  static constexpr size_t x = 0;
  static constexpr size_t k = x + (sizeof(T) == 2 ? Tile<T, PT>::kColsBytes : Tile<T, PT>::kRowsBytes);
  static constexpr size_t times = k + (sizeof(T) == 2 ? Tile<T, NT>::kColsBytes : Tile<T, NT>::kRowsBytes);
  static constexpr size_t bytes = times + 2 * sizeof(Times);
};

// A segment's chunks of one head and PT features without their outputs. Forwards: the state
// that the segment's inputs leave (x, w B). Backwards (REV): the gradient of the state before
// it that its outputs leave (dY, exp(s) C). KEEP: from what the segment starts from, writing
// what comes into each chunk (ds); otherwise from zero, writing what comes out and the
// segment's decay. Pipelined like the forward kernel. Taken where rows are few, because the
// chunks of a row are a chain: the inputs are read twice for it. Bound like the forward kernel:
// two records of 8,192 34 to 35 us without the states between and 46 with them.
template <class T, int PT, int NT, int PW, bool REV, bool KEEP, bool VEC>
__global__ __launch_bounds__(256 * PW, 4) void scan_states_kernel(ScanArgs args) {
  (void)args;
  const ScanArgs *ap = arguments<ScanArgs>();
  using L = StatesLds<T, PT, NT>;
  constexpr int kThreads = 256 * PW, kWaves = 4 * PW;
  using M = Mine<PT, NT, kWaves>;
  extern __shared__ __align__(16) char lds[];
  T *xl = (T *)(lds + L::x), *kl = (T *)(lds + L::k);
  Times *times = (Times *)(lds + L::times);
  const Along<T, PT> xa{xl, xl};
  const Along<T, NT> ka{kl, kl};
  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t id = workgroup_id();
  const int pt = (int)(id % ap->ptiles);
  id /= ap->ptiles;
  const int h = (int)(id % ap->H);
  id /= ap->H;
  const int seg = (int)(id % ap->segs);
  const int64_t b = id / ap->segs;
  const int g = h / (ap->H / ap->G), p0 = pt * PT, len = row_length(ap->lengths, b, ap->T);
  const int c0 = seg * ap->seg_chunks, c1 = min(c0 + ap->seg_chunks, ap->chunks);
  const float A = ap->A[h], bias = ap->bias ? ap->bias[h] : 0.f;
  const T *xg = REV ? (const T *)ap->dy + (b * ap->T * ap->H + h) * ap->P + p0 : (const T *)ap->x + b * ap->xsb + h * ap->xsh + p0;
  const int64_t xstride = REV ? (int64_t)ap->H * ap->P : ap->xst;
  const T *kg = REV ? (const T *)ap->c + b * ap->csb + g * ap->csg : (const T *)ap->b + b * ap->bsb + g * ap->bsg;
  const int64_t kstride = REV ? ap->cst : ap->bst;
  const int64_t bh = b * ap->H + h, pn = (int64_t)ap->P * ap->N;
  // the last chunk that is walked: backwards, what comes out of the first one is not always wanted
  const int n_chunks = c1 - c0 - (REV && KEEP && c0 == 0 && !ap->dinitial ? 1 : 0);
  f32x4 S[M::kEach];
  const float *start = !KEEP ? nullptr : ap->segs > 1 ? ap->seg + (bh * ap->segs + seg) * pn : ap->dfinal ? ap->dfinal + bh * pn : nullptr;
  load_state<PT, NT, kWaves, VEC>(S, start, *ap, p0, wave, q, r);
  double decay = 0.;
  T raw = (T)0.f;
  Stage<T, PT, kThreads, VEC> xs;
  Stage<T, NT, kThreads, VEC> ks;
  auto chunk_of = [&](int n) __attribute__((always_inline)) { return REV ? c1 - 1 - n : c0 + n; };
  auto load = [&](int n) __attribute__((always_inline)) {
    const int64_t t0 = (int64_t)chunk_of(n) * Q;
    xs.load(Matrix<T, VEC>(xg + t0 * xstride, xstride, len - t0, ap->P - p0), tid);
    ks.load(Matrix<T, VEC>(kg + t0 * kstride, kstride, len - t0, ap->N), tid);
    if (wave == 0) raw = raw_step<T, VEC>(*ap, b, h, t0, len, lane);
  };
  auto step = [&](int n) __attribute__((always_inline)) {
    decay += make_times(times[n & 1], (float)raw, bias, (int64_t)chunk_of(n) * Q + lane < len, A, lane);
  };
  if (n_chunks > 0) {
    load(0);
    if (wave == 0) step(0);
  }
  for (int n = 0; n < n_chunks; ++n) {
    const Times &tm = times[n & 1];
    ap = again(ap);
    if (n) __syncthreads();
    if constexpr (sizeof(T) == 2) {
      xs.put(nullptr, xl, tid);
      ks.put(nullptr, kl, tid);
    } else {
      xs.put(xl, nullptr, tid);
      ks.put(kl, nullptr, tid);
    }
    __syncthreads();
    if (n + 1 < n_chunks) load(n + 1);
    if (KEEP && ap->chunks > 1) store_state<PT, NT, kWaves, VEC>(S, ap->ds + (bh * ap->chunks + chunk_of(n)) * pn, *ap, p0, wave, q, r);
    update_state<T, PT, NT, kWaves, false>(S, tm.total, REV ? tm.from : tm.into, xa, ka, wave, q, r, ap->P - p0, ap->N);
    if (wave == 0 && n + 1 < n_chunks) step(n + 1);
  }
  if (!KEEP) {
    store_state<PT, NT, kWaves, VEC>(S, ap->seg + (bh * ap->segs + seg) * pn, *ap, p0, wave, q, r);
    if (tid == 0 && pt == 0) ap->seg_log2[bh * ap->segs + seg] = (float)decay;
  } else if (c0 == 0) {
    if (ap->dinitial)
      store_state<PT, NT, kWaves, VEC>(S, ap->dinitial + bh * pn, *ap, p0, wave, q, r);
    else if (ap->chunks > 1)
      store_state<PT, NT, kWaves, VEC>(S, ap->ds + bh * ap->chunks * pn, *ap, p0, wave, q, r);
  }
}

// Joins segments: seg[s] becomes what segment s starts from. One thread: one state element.
template <bool REV>
__global__ __launch_bounds__(256) void scan_carry_kernel(ScanArgs a) {
  const int64_t pn = (int64_t)a.P * a.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.B * a.H * pn) return;
  const int64_t bh = i / pn, e = i - bh * pn;
  const float *from = REV ? a.dfinal : a.initial;
  float carry = from ? from[i] : 0.f;
  float *p = a.seg + bh * a.segs * pn + e;
  const float *log2 = a.seg_log2 + bh * a.segs;
  for (int n0 = 0; n0 < a.segs; n0 += 8) {  // eight loads in flight at a time
    float own[8], decay[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int s = REV ? a.segs - 1 - n0 - k : n0 + k;
      own[k] = n0 + k < a.segs ? p[s * pn] : 0.f;
      decay[k] = n0 + k < a.segs ? log2[s] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (n0 + k >= a.segs) break;
      p[(REV ? a.segs - 1 - n0 - k : n0 + k) * pn] = carry;
      carry = __builtin_amdgcn_exp2f(decay[k]) * carry + own[k];
    }
  }
}

// ----------------------------------------------------------------------- backward

// What the wavefronts of the backward kernel leave of a head for its gradient of dt.
struct HeadSums {
  float uc[Q];        // exp(s_i) C_i . (h0^T dY_i)
  float vb[Q];        // exp(s_Q - s_j) B_j . (dh1^T x_j)
  float col[Q];       // sum over i >= j of the pairs (i, j), without dt_j
  float cross[4][Q];  // sum of the pairs (i, j) with j < t <= i, over the j of each wavefront
  float dot[32];      // parts of <dh1, h0>, of the rows of 16 lanes
  float diag[4];      // parts of the sum of dY x
};

template <class T, int PT, int NT, bool ST>
struct GradLds {
  static constexpr bool two = sizeof(T) == 2;
  static constexpr size_t bn = 0;
  static constexpr size_t bt = bn + Tile<T, NT>::kRowsBytes;
  static constexpr size_t cn = bt + Tile<T, NT>::kColsBytes;
  static constexpr size_t ct = cn + Tile<T, NT>::kRowsBytes;
  static constexpr size_t xn = ct + Tile<T, NT>::kColsBytes;
  static constexpr size_t yn = xn + Tile<T, PT>::kRowsBytes;
  static constexpr size_t yt = yn + Tile<T, PT>::kRowsBytes;
  static constexpr size_t dh = yt + Tile<T, PT>::kColsBytes;                               // [p][n]
  static constexpr size_t dht = dh + (ST ? StateTile<T, PT, NT, 2>::kBytes : 0);           // [n][p]
  static constexpr size_t h0 = dht + (ST && two ? StateTile<T, NT, PT, 3>::kBytes : 0);    // [n][p], floats [p][n]
  static constexpr size_t times = h0 + (!ST ? 0 : two ? StateTile<T, NT, PT, 3>::kBytes : StateTile<T, PT, NT, 2>::kBytes);
  static constexpr size_t sums = times + 3 * sizeof(GradTimes);
  static constexpr size_t bytes = sums + 2 * sizeof(HeadSums);
  static_assert(bytes <= 160 * 1024, "more LDS than a CU has");
};

// 4 x 4 blocks of a state [P, N] on their way from memory to LDS, of THREADS threads.
template <int PT, int NT, int THREADS, bool VEC>
struct StageState {
  static constexpr int kBlocks = (PT / 4) * (NT / 4), kEach = (kBlocks + THREADS - 1) / THREADS;
  f32x4 v[kEach][4];
  __device__ __forceinline__ void load(const float *base, const ScanArgs &a, int p0, int tid) {
    const Matrix<float, VEC> m = state_rows<VEC>(base, a, p0);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS, n = (blk % (NT / 4)) * 4, p = (blk / (NT / 4)) * 4;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[e][k] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (kBlocks % THREADS == 0 || blk < kBlocks) v[e][k] = m.load(p + k, n);
      }
    }
  }
  template <class Rows, class Cols>
  __device__ __forceinline__ void put(const Rows *rows, const Cols *cols, int tid) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS, n = (blk % (NT / 4)) * 4, p = (blk / (NT / 4)) * 4;
      if (kBlocks % THREADS && blk >= kBlocks) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float along[4] = {v[e][k][0], v[e][k][1], v[e][k][2], v[e][k][3]};
        const float across[4] = {v[e][0][k], v[e][1][k], v[e][2][k], v[e][3][k]};
        if (rows) rows->put4(p + k, n, along);
        if (cols) cols->put4(n + k, p, across);
      }
    }
  }
  // Adds to `sum` this thread's part of the product with the other state in LDS: of h0, all of it
  // with the other's two parts; of the other, what its two parts leave with h0's first.
  template <bool TWO, class Rows, class Cols>
  __device__ __forceinline__ void dot(bool all, const Rows &rows, const Cols &cols, float &sum, int tid) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS, n = (blk % (NT / 4)) * 4, p = (blk / (NT / 4)) * 4;
      if (kBlocks % THREADS && blk >= kBlocks) continue;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float o[4], four = 0.f;
        if (all) {
          rows.template get4<2>(p + k, n, o);
#pragma unroll
          for (int i = 0; i < 4; ++i) four += v[e][k][i] * o[i];
        } else if constexpr (TWO) {
          cols.template get4<1>(n + k, p, o);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = v[e][i][k], rest = x - (float)(bf16)x;
            four += (rest - (float)(bf16)rest) * o[i];
          }
        }
        sum += four;
      }
    }
  }
};

// Wavefronts a SIMD that the kernel's registers leave room for: with 4, two workgroups share a
// CU. Measured both ways for every tile like the forward kernel's: 4 for 32 x 32 tiles (with
// states 225 us against 258 in bf16, 325 against 382 in floats, although 43 and 58 vector registers
// spill) and without states (64 x 32: 90 against 137 in bf16, 248 against 255 in floats), but for
// 128 states (32 x 128: 88 with 2, 142 with 4) and floats of 64 x 64 (152, 158); with states
// otherwise 2 (64 x 32: 156 against 211).
template <class T, int PT, int NT, bool ST>
constexpr int grad_waves() {
  if (PT * NT == 1024) return 4;
  if (ST || NT == 128) return 2;
  return sizeof(T) == 4 && NT == 64 && PT == 64 ? 2 : 4;
}

// One workgroup of eight wavefronts: a chunk of one row and one group's B and C, its heads
// (and their tiles of PT features) one after the other, so that dB and dC are sums in
// registers. The first four wavefronts own 16 positions j each (dX, dB), the other four 16
// positions i each (dC). While an item is computed the next one's inputs are on their way,
// its step sizes are worked out by the wavefront of the first 16 i, and what the last head's
// sums give for dt by the wavefront of the last 16 j: those have the fewest pairs. ST:
// whether there are states before or after the chunk.
// Bound by the vector operations on pairs and the LDS reads of operands, with two barriers an
// item: 2,048 games of 40 positions 203 us (vector units 49% busy, LDS 37, matrix units 11, 3.5
// wavefronts a SIMD); two records of 8,192 with 128 states 239 us (41, 39, 12; one workgroup a CU
// for its 160 KB of LDS as for its 236 registers, and C B^T again for every head); 300 float
// games of up to 100 positions 120 us (26, 12, 24; of 217 MB written, 39 are results, the rest
// spilled registers).
template <class T, int PT, int NT, bool ST, bool VEC>
__global__ __launch_bounds__(512, (grad_waves<T, PT, NT, ST>())) void scan_grad_kernel(ScanArgs args) {
  (void)args;
  const ScanArgs *ap = arguments<ScanArgs>();
  using L = GradLds<T, PT, NT, ST>;
  using O = Ops<T>;
  using BC = Tile<T, NT>;
  using XY = Tile<T, PT>;
  extern __shared__ __align__(16) char lds[];
  T *bn = (T *)(lds + L::bn), *bt = (T *)(lds + L::bt), *cn = (T *)(lds + L::cn), *ct = (T *)(lds + L::ct);
  T *xn = (T *)(lds + L::xn), *yn = (T *)(lds + L::yn), *yt = (T *)(lds + L::yt);
  const StateTile<T, PT, NT, 2> dhl{(T *)(lds + L::dh)}, h0f{(T *)(lds + L::h0)};
  const StateTile<T, NT, PT, 3> dhtl{(T *)(lds + L::dht)}, h0l{(T *)(lds + L::h0)};
  // Times of three heads: the next one's are written while one wavefront may still read the last
  // one's in finish(); HeadSums of two, whose writers are a barrier behind that.
  GradTimes *times = (GradTimes *)(lds + L::times);
  HeadSums *sums = (HeadSums *)(lds + L::sums);
  const Along<T, NT> ba{bn, bt}, ca{cn, ct};
  const Along<T, PT> ya{yn, yt};
  constexpr int kTimesWave = 4, kStepWave = 3;

  const int tid = threadIdx.x, lane = tid & 63, q = lane >> 4, r = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int64_t id = workgroup_id();
  const int slice = (int)(id % ap->slices);
  id /= ap->slices;
  const int g = (int)(id % ap->G);
  id /= ap->G;
  const int c = (int)(id % ap->chunks);
  const int64_t b = id / ap->chunks;
  const int len = row_length(ap->lengths, b, ap->T), per = ap->H / ap->G;
  const int64_t t0 = (int64_t)c * Q, pn = (int64_t)ap->P * ap->N;
  const int h_lo = g * per + (int)((int64_t)per * slice / ap->slices);
  const int h_hi = g * per + (int)((int64_t)per * (slice + 1) / ap->slices);
  const bool own_j = wave < 4;
  const int mine = wave & 3, tw = 16 * mine + r;  // this lane's position
  const bool live = t0 + lane < len, own_live = t0 + tw < len;

  // one half of the workgroup brings x and the state, the other dY and the state's gradient
  const bool lower = wave < 4;
  const int ht = tid & 255;
  Stage<T, PT, 256, VEC> xy;
  StageState<PT, NT, 256, VEC> hd;
  T raw = (T)0.f;
  const float *dh_next = nullptr, *h0_next = nullptr;
  auto load = [&](int h, int pt) __attribute__((always_inline)) {
    const int p0 = pt * PT;
    const T *row = lower ? (const T *)ap->x + b * ap->xsb + t0 * ap->xst + h * ap->xsh + p0
                         : (const T *)ap->dy + ((b * ap->T + t0) * ap->H + h) * ap->P + p0;
    xy.load(Matrix<T, VEC>(row, lower ? ap->xst : (int64_t)ap->H * ap->P, len - t0, ap->P - p0), ht);
    if (pt == 0 && wave == kTimesWave) raw = raw_step<T, VEC>(*ap, b, h, t0, len, lane);
  };
  auto load_states = [&](int h, int pt) __attribute__((always_inline)) {
    if constexpr (ST) {
      const int64_t bh = b * ap->H + h;
      h0_next = ap->chunks > 1 ? ap->cs + (bh * ap->chunks + c) * pn : ap->initial ? ap->initial + bh * pn : nullptr;
      dh_next = ap->chunks > 1 ? ap->ds + (bh * ap->chunks + c) * pn : ap->dfinal ? ap->dfinal + bh * pn : nullptr;
      hd.load(lower ? h0_next : dh_next, *ap, pt * PT, ht);
    }
  };
  auto step = [&](int h) __attribute__((always_inline)) {
    make_times(times[(unsigned)h % 3], (float)raw, ap->bias ? ap->bias[h] : 0.f, live, ap->A[h], lane);
  };
  // dt's gradient of head h from its sums, and the chunk's part of those of A, dt_bias and D
  auto finish = [&](int h) __attribute__((always_inline)) {
    const GradTimes &tm = times[(unsigned)h % 3];
    const HeadSums &s = sums[h & 1];
    double dot = 0.;
    float diag = 0.f, cross = 0.f;
    if constexpr (ST) {
      dot = s.dot[lane & 31];
      dot += moved64<kUp + 1>(dot);
      dot += moved64<kUp + 2>(dot);
      dot += moved64<kUp + 4>(dot);
      dot += moved64<kUp + 8>(dot);
      dot = lane64(dot, 15) + lane64(dot, 31);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      diag += s.diag[i];
      cross += 16 * i <= lane ? s.cross[i][lane] : 0.f;
    }
    const float dt = tm.dt[lane];
    float before = 0.f, bdv = s.col[lane], after = 0.f;
    if constexpr (ST) {
      const float vb = s.vb[lane];
      before = dt * vb;
      bdv += vb;
      after = s.uc[lane];
#pragma unroll
      for (int m = 1; m < Q; m *= 2) {
        const float upper = __shfl_down(after, m, kWave);
        if (lane + m < Q) after += upper;
      }
      before += moved<kUp + 1>(before);
      before += moved<kUp + 2>(before);
      before += moved<kUp + 4>(before);
      before += moved<kUp + 8>(before);
      before += moved<kBcast15, 0xa>(before);
      before += moved<kBcast31, 0xc>(before);
      before = __shfl_up(before, 1, kWave);
      if (lane == 0) before = 0.f;
    }
    const float da = (before + after) + (cross + (float)(tm.total * dot));
    const float ddt = live ? (ap->A[h] * da + bdv) * tm.slope[lane] : 0.f;
    if (t0 + lane < ap->T) ((T *)ap->ddt)[(b * ap->T + t0 + lane) * ap->H + h] = (T)ddt;
    const float dA = wave_sum(da * dt), dbias = wave_sum(ddt);
    if (lane == 0) {
      float *o = ap->part + ((b * ap->chunks + c) * ap->H + h) * 3;
      o[0] = dA;
      o[1] = dbias;
      o[2] = diag;
    }
  };

  {
    Stage<T, NT, 512, VEC> s, u;
    s.load(Matrix<T, VEC>((const T *)ap->b + b * ap->bsb + t0 * ap->bst + g * ap->bsg, ap->bst, len - t0, ap->N), tid);
    u.load(Matrix<T, VEC>((const T *)ap->c + b * ap->csb + t0 * ap->cst + g * ap->csg, ap->cst, len - t0, ap->N), tid);
    load(h_lo, 0);
    load_states(h_lo, 0);
    s.put(bn, bt, tid);
    u.put(cn, ct, tid);
  }
  if (wave == kTimesWave) step(h_lo);
  f32x4 acc[NT / 16];  // dB^T (rows n, columns j), or dC^T, over the heads
#pragma unroll
  for (int i = 0; i < NT / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float diag = 0.f, inter = 0.f, col = 0.f, dot = 0.f;

  int h = h_lo, pt = 0;
  for (bool first = true;; first = false) {
    ap = again(ap);
    const int p0 = pt * PT, np = ap->P - p0, h_now = h, pt_now = pt;
    const GradTimes &tm = times[(unsigned)h % 3];
    HeadSums &sum = sums[h & 1];
    const bool dh = ST && dh_next, h0 = ST && h0_next;
    const float D = ap->D ? ap->D[h] : 0.f;
    if (!first) __syncthreads();
    if (lower)
      xy.put(xn, nullptr, ht);
    else
      xy.put(yn, yt, ht);
    if constexpr (ST) {
      using Rows = const StateTile<T, PT, NT, 2> *;
      using Cols = const StateTile<T, NT, PT, 3> *;
      if (lower)
        hd.put(L::two ? (Rows) nullptr : &h0f, L::two ? &h0l : (Cols) nullptr, ht);
      else
        hd.put(&dhl, L::two ? &dhtl : (Cols) nullptr, ht);
    }
    __syncthreads();
    if (++pt == ap->ptiles) {
      pt = 0;
      ++h;
    }
    const bool more = h < h_hi;
    if (more) load(h, pt);
    if (wave == kStepWave && pt_now == 0 && !first) finish(h_now - 1);
    if (pt_now == 0) diag = inter = col = dot = 0.f;
    // <dh1, h0> = <h0, dh1 in two parts> + <what those leave of dh1, h0's first part>, from the
    // float32 values that each half of the workgroup still holds (products of parts on both
    // sides were 2e-6 of dA off); the sums of 16 threads are added up in 64 bits: thousands of
    // terms that may cancel
    if (dh && h0) hd.template dot<L::two>(lower, dhl, h0l, dot, ht);
    if (more) load_states(h, pt);

    const float hi = tm.hi[tw], lo = tm.lo[tw];
    if (own_j) {
      typename O::Frag bf[NT / 32], xf[PT / 32];
#pragma unroll
      for (int k = 0; k < NT / 32; ++k) bf[k] = O::near(bn + tw * BC::kRow, 32 * k, q);
#pragma unroll
      for (int k = 0; k < PT / 32; ++k) xf[k] = O::near(xn + tw * XY::kRow, 32 * k, q);
      const float left = tm.left[tw], dt = tm.dt[tw];
      float later = 0.f;  // the pairs (i, j) of the tiles of i after this one
      const float till = tm.till[tw];
      typename O::Split mf[2], sf[2];  // M and Q, two tiles of i to an operand
#pragma unroll
      for (int ip = 1; ip >= 0; --ip) {
        if (2 * ip + 1 < mine) break;
        float m[8], s[8];
#pragma unroll
        for (int half = 1; half >= 0; --half) {
          const int it = 2 * ip + half;
          if (it < mine) {
#pragma unroll
            for (int e = 0; e < 4; ++e) m[4 * half + e] = s[4 * half + e] = 0.f;
            continue;
          }
          f32x4 gs = {0.f, 0.f, 0.f, 0.f}, ms = gs;
#pragma unroll
          for (int k = 0; k < NT / 32; ++k)
            if (on<T, NT>(32 * k, ap->N)) O::mma_left(gs, O::near(cn + (16 * it + r) * BC::kRow, 32 * k, q), bf[k], rest<T, NT>(ap->N - 32 * k));
#pragma unroll
          for (int k = 0; k < PT / 32; ++k)
            if (on<T, NT>(32 * k, np)) O::mma_left(ms, O::near(yn + (16 * it + r) * XY::kRow, 32 * k, q), xf[k], rest<T, NT>(np - 32 * k));
          float pair[4];  // with dt_j
          if (it > mine) {
            const f32x4 past = *reinterpret_cast<const f32x4 *>(tm.after + Times::past_at(mine) + 16 * it + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float f = past[e] * till;
              m[4 * half + e] = gs[e] * f;
              s[4 * half + e] = ms[e] * f;
              pair[e] = s[4 * half + e] * gs[e];
            }
          } else {  // the only tile with pairs j > i, and the diagonal
            const f32x4 thi = *reinterpret_cast<const f32x4 *>(tm.hi + 16 * it + 4 * q);
            const f32x4 tlo = *reinterpret_cast<const f32x4 *>(tm.lo + 16 * it + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int ahead = r - 4 * q - e;
              const float f = __builtin_amdgcn_exp2f((thi[e] - hi) + (tlo[e] - lo)) * dt;
              const float v = gs[e] * f, u = ms[e] * f;
              m[4 * half + e] = ahead > 0 ? 0.f : ahead == 0 ? v + D : v;
              s[4 * half + e] = ahead > 0 ? 0.f : u;
              pair[e] = s[4 * half + e] * gs[e];
              diag += ahead == 0 ? ms[e] : 0.f;
            }
          }
          // from each i to the chunk's end, then over the j before i
          pair[2] += pair[3];
          pair[1] += pair[2];
          pair[0] += pair[1];
          const Pair rows = rows_of_half(pair[0]), both = halves(rows.first + rows.second);
          const float after = later + (q & 1 ? 0.f : rows.second) + (q < 2 ? both.second : 0.f);
          f32x4 over;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = pair[e] + after;
            over[e] = lanes_sum<16>(it > mine || r < 4 * q + e ? v : 0.f);
          }
          if (r == 0) {
            f32x4 *o = reinterpret_cast<f32x4 *>(sum.cross[mine] + 16 * it + 4 * q);
            *o = pt_now ? *o + over : over;
          }
          later += both.first + both.second;
        }
        mf[ip] = O::split(m);
        sf[ip] = O::split(s);
      }
      col += dt > 0.f ? later / dt : 0.f;  // (a step of 0 has a slope of 0)
      const float into = left * dt;
      const Matrix<T, VEC> xm((const T *)ap->dx + ((b * ap->T + t0) * ap->H + h_now) * ap->P + p0, (int64_t)ap->H * ap->P, ap->T - t0, ap->P - p0);
#pragma unroll
      for (int i = 0; i < PT / 16; ++i) {
        if (!on<T, NT>(16 * i, np)) continue;
        f32x4 dx = {0.f, 0.f, 0.f, 0.f};
        if (dh) {
#pragma unroll
          for (int k = 0; k < NT / 32; ++k)
            if (on<T, NT>(32 * k, ap->N)) O::mma_left(dx, dhl.near(16 * i + r, 32 * k, q), bf[k], rest<T, NT>(ap->N - 32 * k));
          dx *= into;
        }
        if (i & 1) __builtin_amdgcn_sched_barrier(0);  // (reads further ahead cost more registers than there are)
        if constexpr (L::two) {
          if (mine < 2) O::mma(dx, ya.far(16 * i + r, 0, q), mf[0]);
          O::mma(dx, ya.far(16 * i + r, 32, q), mf[1]);
        } else {
          // the own tile last: what D dY is rounded to is not rounded again with every later term
          // (dX 7e-8 off instead of 1.2e-7)
          if (mine < 2) O::mma(dx, ya.far(16 * i + r, 32, q), mf[1]);
          const typename O::Frag y = ya.far(16 * i + r, mine < 2 ? 0 : 32, q);
          if (mine < 2)
            O::mma_own(dx, y, mf[0], mine & 1);
          else
            O::mma_own(dx, y, mf[1], mine & 1);
        }
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = own_live ? dx[e] : 0.f;
        xm.store(tw, 16 * i + 4 * q, v);
      }
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) {
        if (!on<T, NT>(16 * i, ap->N)) continue;
        if (dh) {
          f32x4 u = {0.f, 0.f, 0.f, 0.f}, small = u;
#pragma unroll
          for (int k = 0; k < PT / 32; ++k) {
            if (!on<T, NT>(32 * k, np)) continue;
            if constexpr (L::two)
              O::mma_apart(u, small, dhtl.near(16 * i + r, 32 * k, q), xf[k]);
            else
              O::mma_left(u, dhl.across(16 * i + r, 32 * k, q), xf[k], rest<T, NT>(np - 32 * k));
          }
          if constexpr (L::two) u += small;
          float four = 0.f;
          const typename V4<T>::type bv = *reinterpret_cast<const typename V4<T>::type *>(bn + tw * BC::kRow + 16 * i + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) four += u[e] * (float)bv[e];
          inter += left * four;
          acc[i] += u * into;
        }
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
        if (mine < 2) O::mma(acc[i], ca.far(16 * i + r, 0, q), sf[0]);
        O::mma(acc[i], ca.far(16 * i + r, 32, q), sf[1]);
      }
    } else {
      typename O::Frag yf[PT / 32];
#pragma unroll
      for (int k = 0; k < PT / 32; ++k) yf[k] = O::near(yn + tw * XY::kRow, 32 * k, q);
      typename O::Split sf[2];
#pragma unroll
      for (int jp = 0; jp < 2; ++jp) {
        if (2 * jp > mine) break;
        float s[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int jt = 2 * jp + half;
          if (jt > mine) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * half + e] = 0.f;
            continue;
          }
          f32x4 ms = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < PT / 32; ++k)
            if (on<T, NT>(32 * k, np)) O::mma_left(ms, O::near(xn + (16 * jt + r) * XY::kRow, 32 * k, q), yf[k], rest<T, NT>(np - 32 * k));
          if (jt < mine) {
            const float past = tm.past(jt, tw);
            const f32x4 till = *reinterpret_cast<const f32x4 *>(tm.till + 16 * jt + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * half + e] = ms[e] * (past * till[e]);
            continue;
          }
          const f32x4 thi = *reinterpret_cast<const f32x4 *>(tm.hi + 16 * jt + 4 * q);
          const f32x4 tlo = *reinterpret_cast<const f32x4 *>(tm.lo + 16 * jt + 4 * q);
          const f32x4 tdt = *reinterpret_cast<const f32x4 *>(tm.dt + 16 * jt + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = ms[e] * (__builtin_amdgcn_exp2f((hi - thi[e]) + (lo - tlo[e])) * tdt[e]);
            s[4 * half + e] = 4 * q + e <= r ? v : 0.f;
          }
        }
        sf[jp] = O::split(s);
      }
      const float from = tm.from[tw];
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) {
        if (!on<T, NT>(16 * i, ap->N)) continue;
        if (h0) {
          f32x4 u = {0.f, 0.f, 0.f, 0.f}, small = u;
#pragma unroll
          for (int k = 0; k < PT / 32; ++k) {
            if (!on<T, NT>(32 * k, np)) continue;
            if constexpr (L::two)
              O::mma_apart(u, small, h0l.near(16 * i + r, 32 * k, q), yf[k]);
            else
              O::mma_left(u, h0f.across(16 * i + r, 32 * k, q), yf[k], rest<T, NT>(np - 32 * k));
          }
          if constexpr (L::two) u += small;
          u *= from;
          float four = 0.f;
          const typename V4<T>::type cv = *reinterpret_cast<const typename V4<T>::type *>(cn + tw * BC::kRow + 16 * i + 4 * q);
#pragma unroll
          for (int e = 0; e < 4; ++e) four += u[e] * (float)cv[e];
          inter += four;
          acc[i] += u;
        }
        if (i & 1) __builtin_amdgcn_sched_barrier(0);
        O::mma(acc[i], ba.far(16 * i + r, 0, q), sf[0]);
        if (mine > 1) O::mma(acc[i], ba.far(16 * i + r, 32, q), sf[1]);
      }
    }
    if (pt_now + 1 == ap->ptiles) {
      // a position's n are spread over the four lanes of one r
      if constexpr (ST) {
        inter = rows_sum(inter);
        if (q == 0) (own_j ? sum.vb : sum.uc)[tw] = inter;
        const float row = lanes_sum<16>(dot);
        if (r == 0) sum.dot[4 * wave + q] = row;
      }
      if (own_j) {
        diag = wave_sum(diag);
        if (q == 0) sum.col[tw] = col;
        if (lane == 0) sum.diag[mine] = diag;
      }
    }
    if (!more) break;
    if (wave == kTimesWave && pt == 0) step(h);
  }
  __syncthreads();
  if (wave == kStepWave) finish(h_hi - 1);
  // after a row's end the factors are 0, but a state's gradient, say, may not be finite
  if (!own_live)
#pragma unroll
    for (int i = 0; i < NT / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int64_t first_row = ((b * ap->T + t0) * ap->G + g) * ap->N;
  if (ap->slices == 1) {
    const Matrix<T, VEC> m((const T *)(own_j ? ap->db : ap->dc) + first_row, (int64_t)ap->G * ap->N, ap->T - t0, ap->N);
#pragma unroll
    for (int i = 0; i < NT / 16; ++i) {
      const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
      m.store(tw, 16 * i + 4 * q, v);
    }
  } else {
    const Matrix<float, VEC> m(ap->dbc + (int64_t)(slice * 2 + !own_j) * ap->B * ap->T * ap->G * ap->N + first_row, (int64_t)ap->G * ap->N,
                               ap->T - t0, ap->N);
#pragma unroll
    for (int i = 0; i < NT / 16; ++i) {
      const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
      m.store(tw, 16 * i + 4 * q, v);
    }
  }
}

// db and dc from the parts of the head slices.
template <class T>
__global__ __launch_bounds__(256) void scan_join_slices_kernel(ScanArgs a) {
  const int64_t n = a.B * a.T * a.G * a.N, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= 2 * n) return;
  float s = 0.f;
  for (int k = 0; k < a.slices; ++k) s += a.dbc[(int64_t)k * 2 * n + i];
  if (i < n)
    ((T *)a.db)[i] = (T)s;
  else
    ((T *)a.dc)[i - n] = (T)s;
}

// dA, ddt_bias and dD from the parts of the chunks, [rows, H, 3]: a first pass leaves at
// most kSumRows rows (grid.y of them), the second ends in the gradients.
constexpr int kSumRows = 128;
__global__ __launch_bounds__(kSumThreads) void scan_sum_rows_kernel(const float *part, int64_t rows, int64_t cols, float *out) {
  const int64_t each = (rows + gridDim.y - 1) / gridDim.y, r0 = each * blockIdx.y;
  const int64_t n = rows - r0 < each ? rows - r0 : each;
  int64_t j;
  float s;
  if (sum_rows(part + r0 * cols, n, cols, &j, &s)) out[(int64_t)blockIdx.y * cols + j] = s;
}
__global__ __launch_bounds__(kSumThreads) void scan_sum_heads_kernel(const float *part, int64_t rows, int32_t H, float *dA,
                                                             float *dbias, float *dD) {
  int64_t j;
  float s;
  if (!sum_rows(part, rows, 3 * (int64_t)H, &j, &s)) return;
  float *o = j % 3 == 0 ? dA : j % 3 == 1 ? dbias : dD;
  if (o) o[j / 3] = s;
}

// --------------------------------------------------------------------- one position

struct StepArgs {
  const void *x, *dt, *b, *c;
  const float *A, *D, *bias;
  float *h;
  void *y;
  int64_t B, xsb, xsh, dsb, dsh, bsb, bsg, csb, csg;
  int32_t H, P, G, N;
};

// A state is read and written once, 8 bytes an element for 5 operations. LPR lanes hold a
// row of N (V * NJ values each); a wavefront has kStepRows / LPR rows of one head, as many
// of them in flight at once as it has, and does the head's step size once for them. 10,000
// envs (8 heads of 32, 32 states): 135 us, 5.0 TB/s, which is a large copy's rate; one env 5 us,
// a launch's latency.
constexpr int kStepRows = 256;  // 4 passes of 64 / LPR rows
template <class T, int V, int LPR, int NJ>
__global__ __launch_bounds__(256) void scan_step_kernel(StepArgs a) {
  constexpr int kRows = 64 / LPR, U = kStepRows / 64;
  const int lane = threadIdx.x & 63, ln = lane % LPR, row = lane / LPR;
  const int parts = (a.P + kRows * U - 1) / (kRows * U);
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), bh = id / parts, b = bh / a.H;
  if (b >= a.B) return;
  const int h = (int)(bh - b * a.H), g = h / (a.H / a.G), p0 = (int)(id - bh * parts) * kRows * U + row;
  float *hp = a.h + (bh * a.P + p0) * a.N;
  float v[U][NJ][V], x[U], bv[NJ][V], cv[NJ][V];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    x[u] = 0.f;
    if (p0 + u * kRows >= a.P) continue;
    x[u] = (float)((const T *)a.x)[b * a.xsb + h * a.xsh + p0 + u * kRows];
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      if ((j * LPR + ln) * V < a.N) Vec<float, V>::load(hp + (int64_t)u * kRows * a.N + (j * LPR + ln) * V, v[u][j]);
  }
  const T *bp = (const T *)a.b + b * a.bsb + g * a.bsg, *cp = (const T *)a.c + b * a.csb + g * a.csg;
  const float raw = (float)((const T *)a.dt)[b * a.dsb + h * a.dsh] + (a.bias ? a.bias[h] : 0.f);
  const float dt = softplus(raw), decay = expf(dt * a.A[h]), D = a.D ? a.D[h] : 0.f;
#pragma unroll
  for (int j = 0; j < NJ; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int n = (j * LPR + ln) * V + i;
      bv[j][i] = n < a.N ? dt * (float)bp[n] : 0.f;
      cv[j][i] = n < a.N ? (float)cp[n] : 0.f;
    }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (p0 + u * kRows >= a.P) continue;
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      if ((j * LPR + ln) * V >= a.N) continue;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        v[u][j][i] = decay * v[u][j][i] + x[u] * bv[j][i];
        s += v[u][j][i] * cv[j][i];
      }
      Vec<float, V>::store(hp + (int64_t)u * kRows * a.N + (j * LPR + ln) * V, v[u][j]);
    }
    s = lanes_sum<LPR>(s);
    if (ln == 0) ((T *)a.y)[bh * a.P + p0 + u * kRows] = (T)(s + D * x[u]);
  }
}

// ------------------------------------------------------------------------ host side

int check(const astra_state_scan *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_ABI_CHECK(f->batch, >=, 0);
  ASTRA_ABI_CHECK(f->length, >=, 0);
  ASTRA_ABI_CHECK(f->length, <, 2147483647 - Q);
  ASTRA_ABI_CHECK(f->heads, >=, 1);
  ASTRA_ABI_CHECK(f->dim, >=, 1);
  ASTRA_ABI_CHECK(f->groups, >=, 1);
  ASTRA_ABI_CHECK(f->heads % f->groups, ==, 0);
  ASTRA_ABI_CHECK(f->state, >=, 1);
  ASTRA_ABI_CHECK(f->state, <=, ASTRA_SEQ_MAX_STATE);
  return ASTRA_OK;
}

// The tiles of features and of states that a call is padded to, and for the forward and
// states kernels the parts of the features that wavefronts share. With states over 64 the
// backward kernel's tiles fit a CU's LDS for 32 features only.
struct Tiles {
  int p, n, pw;
};
Tiles tiles_of(const astra_state_scan &f, bool grad) {
  Tiles t;
  t.n = f.state <= 32 ? 32 : f.state <= 64 ? 64 : 128;
  t.p = f.dim <= 32 || (grad && t.n == 128) ? 32 : 64;
  t.pw = t.n == 128 && t.p == 64 ? 2 : 1;
  return t;
}

ScanArgs args_of(const astra_state_scan &f) {
  ScanArgs a{};
  a.x = f.x;
  a.dt = f.dt;
  a.b = f.b;
  a.c = f.c;
  a.A = f.A;
  a.D = f.D;
  a.bias = f.dt_bias;
  a.initial = f.initial;
  a.lengths = f.lengths;
  a.y = f.y;
  a.final_state = f.final_state;
  a.B = f.batch;
  a.T = f.length;
  a.xsb = f.x_stride_b;
  a.xst = f.x_stride_t;
  a.xsh = f.x_stride_h;
  a.dsb = f.dt_stride_b;
  a.dst = f.dt_stride_t;
  a.dsh = f.dt_stride_h;
  a.bsb = f.b_stride_b;
  a.bst = f.b_stride_t;
  a.bsg = f.b_stride_g;
  a.csb = f.c_stride_b;
  a.cst = f.c_stride_t;
  a.csg = f.c_stride_g;
  a.H = f.heads;
  a.P = f.dim;
  a.G = f.groups;
  a.N = f.state;
  const Tiles tiles = tiles_of(f, false);
  a.ptiles = (int32_t)cdiv(f.dim, tiles.p);
  a.chunks = (int32_t)cdiv(f.length, Q);
  // few rows: the length is split into segments, joined by their states; as many workgroups
  // as are resident at once (two a CU)
  const int64_t resident = 512;
  const int64_t rows = a.B * a.H * a.ptiles;
  int64_t segs = 1;
  if (rows > 0 && rows < resident) segs = cdiv(resident, rows);
  if (segs > a.chunks / 2) segs = a.chunks / 2;
  if (segs < 1) segs = 1;
  a.seg_chunks = (int32_t)cdiv(a.chunks, segs);
  a.segs = a.seg_chunks ? (int32_t)cdiv(a.chunks, a.seg_chunks) : 1;
  // a workgroup walks as many of a group's heads as leave twice that many workgroups
  const int per = a.H / a.G;
  const int64_t shared = a.B * a.G * a.segs;
  a.parts = shared > 0 ? (int32_t)std::min<int64_t>((int64_t)per * a.ptiles, cdiv(2 * resident, shared)) : 1;
  // few chunks: the heads of a group are split, and their parts of db and dc added up
  const int64_t items = a.B * a.chunks * a.G;
  a.slices = items > 0 && items < 256 ? (int32_t)std::min<int64_t>(per, cdiv(256, items)) : 1;
  const int64_t e = 4 * (int64_t)elem_size(f.type);
  a.vec = a.P % 4 == 0 && a.N % 4 == 0 && aligned(a.x, e) && aligned(a.b, e) && aligned(a.c, e) && aligned(a.y, e) &&
          aligned(a.initial, 16) && aligned(a.final_state, 16);
  for (int64_t stride : {a.xsb, a.xst, a.xsh, a.bsb, a.bst, a.bsg, a.csb, a.cst, a.csg}) a.vec = a.vec && stride % 4 == 0;
  const int64_t most = int64_t(1) << 23;  // 64 rows' bytes stay below 2^31
  a.vec = a.vec && a.xst >= a.P && a.xst < most && a.bst >= a.N && a.bst < most && a.cst >= a.N && a.cst < most && a.dst >= 1 && a.dst < most &&
          (int64_t)a.H * a.P < most && (int64_t)a.G * a.N < most && a.P * (int64_t)a.N < most;
  return a;
}

size_t seg_floats(const ScanArgs &a) {
  return a.segs > 1 ? (size_t)a.B * a.H * a.segs * ((size_t)a.P * a.N + 1) : 0;
}
size_t chunk_floats(const ScanArgs &a) {
  return a.chunks > 1 ? (size_t)a.B * a.H * a.chunks * (size_t)a.P * a.N : 0;
}
size_t part_floats(const ScanArgs &a) { return ((size_t)a.B * a.chunks + kSumRows) * a.H * 3; }
size_t slice_floats(const ScanArgs &a) {
  return a.slices > 1 ? (size_t)a.slices * 2 * a.B * a.T * a.G * a.N : 0;
}
// parts of a workspace start on 16 bytes
size_t round4(size_t floats) { return (floats + 3) / 4 * 4; }

// More than 64 KB of LDS has to be asked for, once per kernel and device (a kernel is always
// launched with the same number of bytes).
template <auto kernel>
int allow_lds(size_t bytes) {
  if (bytes <= 64 * 1024) return ASTRA_OK;
  static std::atomic<uint64_t> asked{0};  // a bit a device; devices from 64 on ask every time
  int device = 0;
  ASTRA_HIP_CHECK(hipGetDevice(&device), "hipGetDevice");
  const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
  if (asked.load(std::memory_order_relaxed) & bit) return ASTRA_OK;
  ASTRA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                      hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
                  "hipFuncSetAttribute");
  asked.fetch_or(bit, std::memory_order_relaxed);
  return ASTRA_OK;
}

#define SCAN_LAUNCH(kernel, blocks, threads, bytes)                                                    \
  do {                                                                                                 \
    ASTRA_SEQ_LAUNCH_CHECK(blocks, threads);                                                           \
    if (int rc = allow_lds<&kernel>(bytes)) return rc;                                                 \
    hipLaunchKernelGGL((kernel), dim3((unsigned)(blocks)), dim3(threads), bytes, st, a);               \
    ASTRA_HIP_CHECK(rt_last_error(), #kernel " launch");                                               \
  } while (false)

template <class T, int PT, int NT, int PW, bool REV, bool KEEP>
int states(ScanArgs &a, hipStream_t st) {
  const int64_t blocks = a.B * a.H * a.ptiles * a.segs;
  if (a.vec)
    SCAN_LAUNCH((scan_states_kernel<T, PT, NT, PW, REV, KEEP, true>), blocks, 256 * PW, (StatesLds<T, PT, NT>::bytes));
  else
    SCAN_LAUNCH((scan_states_kernel<T, PT, NT, PW, REV, KEEP, false>), blocks, 256 * PW, (StatesLds<T, PT, NT>::bytes));
  if (KEEP) return ASTRA_OK;
  const int64_t carries = cdiv(a.B * a.H * a.P * a.N, 256);
  ASTRA_SEQ_LAUNCH_CHECK(carries, 256);
  hipLaunchKernelGGL(scan_carry_kernel<REV>, dim3((unsigned)carries), dim3(256), 0, st, a);
  ASTRA_HIP_CHECK(rt_last_error(), "scan_carry_kernel launch");
  return ASTRA_OK;
}

template <class T, int PT, int NT, int PW>
int forward(ScanArgs &a, hipStream_t st) {
  if (a.segs > 1)
    if (int rc = states<T, PT, NT, PW, false, false>(a, st)) return rc;
  const int64_t blocks = a.B * a.G * a.segs * a.parts;
  constexpr size_t bytes = ForwardLds<T, PT, NT, true>::bytes;
  if (!a.vec)
    SCAN_LAUNCH((scan_forward_kernel<T, PT, NT, PW, true, false>), blocks, 256 * PW, bytes);
  else if (a.chunks > 1 || a.initial)
    SCAN_LAUNCH((scan_forward_kernel<T, PT, NT, PW, true, true>), blocks, 256 * PW, bytes);
  else
    SCAN_LAUNCH((scan_forward_kernel<T, PT, NT, PW, false, true>), blocks, 256 * PW, (ForwardLds<T, PT, NT, false>::bytes));
  return ASTRA_OK;
}

// The gradients of the states after the chunks.
template <class T, int PT, int NT, int PW>
int backward_states(ScanArgs &a, hipStream_t st) {
  if (a.segs > 1)
    if (int rc = states<T, PT, NT, PW, true, false>(a, st)) return rc;
  return states<T, PT, NT, PW, true, true>(a, st);
}

template <class T, int PT, int NT>
int backward(ScanArgs &a, hipStream_t st) {
  a.ptiles = (int32_t)cdiv(a.P, PT);
  const int64_t blocks = a.B * a.chunks * a.G * a.slices;
  constexpr size_t bytes = GradLds<T, PT, NT, true>::bytes;
  if (!a.vec)
    SCAN_LAUNCH((scan_grad_kernel<T, PT, NT, true, false>), blocks, 512, bytes);
  else if (a.chunks > 1 || a.initial || a.dfinal)
    SCAN_LAUNCH((scan_grad_kernel<T, PT, NT, true, true>), blocks, 512, bytes);
  else
    SCAN_LAUNCH((scan_grad_kernel<T, PT, NT, false, true>), blocks, 512, (GradLds<T, PT, NT, false>::bytes));
  if (a.slices > 1) {
    const int64_t joins = cdiv(2 * a.B * a.T * a.G * a.N, 256);
    ASTRA_SEQ_LAUNCH_CHECK(joins, 256);
    hipLaunchKernelGGL(scan_join_slices_kernel<T>, dim3((unsigned)joins), dim3(256), 0, st, a);
    ASTRA_HIP_CHECK(rt_last_error(), "scan_join_slices_kernel launch");
  }
  return ASTRA_OK;
}

#define SCAN_BOTH(FN, ...) (h ? FN<bf16, __VA_ARGS__>(a, st) : FN<float, __VA_ARGS__>(a, st))
#define SCAN_TILES(FN)                                              \
  do {                                                              \
    const Tiles t = tiles_of(f, false);                             \
    const bool h = f.type == ASTRA_SEQ_BF16;                        \
    if (t.n == 128 && t.p == 64) return SCAN_BOTH(FN, 64, 128, 2);  \
    if (t.n == 128) return SCAN_BOTH(FN, 32, 128, 1);               \
    if (t.n == 64 && t.p == 64) return SCAN_BOTH(FN, 64, 64, 1);    \
    if (t.n == 64) return SCAN_BOTH(FN, 32, 64, 1);                 \
    if (t.p == 64) return SCAN_BOTH(FN, 64, 32, 1);                 \
    return SCAN_BOTH(FN, 32, 32, 1);                                \
  } while (false)

int run_forward(const astra_state_scan &f, ScanArgs &a, hipStream_t st) { SCAN_TILES(forward); }
int run_backward_states(const astra_state_scan &f, ScanArgs &a, hipStream_t st) { SCAN_TILES(backward_states); }
int run_backward(const astra_state_scan &f, ScanArgs &a, hipStream_t st) {
  if (a.chunks > 1 || a.dinitial)
    if (int rc = run_backward_states(f, a, st)) return rc;
  const Tiles t = tiles_of(f, true);
  const bool h = f.type == ASTRA_SEQ_BF16;
  if (t.n == 128) return SCAN_BOTH(backward, 32, 128);
  if (t.n == 64 && t.p == 64) return SCAN_BOTH(backward, 64, 64);
  if (t.n == 64) return SCAN_BOTH(backward, 32, 64);
  if (t.p == 64) return SCAN_BOTH(backward, 64, 32);
  return SCAN_BOTH(backward, 32, 32);
}

template <class T>
int step(const StepArgs &a, bool wide, hipStream_t st) {
#define STEP_LAUNCH(V, LPR, NJ)                                                                       \
  do {                                                                                                \
    const int64_t blocks = cdiv(a.B * a.H * cdiv(a.P, kStepRows / LPR), 4);                           \
    ASTRA_SEQ_LAUNCH_CHECK(blocks, 256);                                                              \
    hipLaunchKernelGGL((scan_step_kernel<T, V, LPR, NJ>), dim3((unsigned)blocks), dim3(256), 0, st, a); \
  } while (false)
  if (wide) {
    if (a.N <= 16) STEP_LAUNCH(4, 4, 1);
    else if (a.N <= 32) STEP_LAUNCH(4, 8, 1);
    else if (a.N <= 64) STEP_LAUNCH(4, 16, 1);
    else STEP_LAUNCH(4, 32, 1);
  } else {
    if (a.N <= 16) STEP_LAUNCH(1, 16, 1);
    else if (a.N <= 64) STEP_LAUNCH(1, 64, 1);
    else STEP_LAUNCH(1, 64, 2);
  }
  ASTRA_HIP_CHECK(rt_last_error(), "scan_step_kernel launch");
  return ASTRA_OK;
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_state_scan_chunk_states(const astra_state_scan *f, size_t *floats) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(floats);
  *floats = chunk_floats(args_of(*f));
  return ASTRA_OK;
}

int astra_state_scan_workspace_size(const astra_state_scan *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  *bytes = seg_floats(args_of(*f)) * sizeof(float);
  return ASTRA_OK;
}

int astra_state_scan_forward(const astra_state_scan *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->batch == 0) return ASTRA_OK;
  const hipStream_t st = as_stream(stream);
  ScanArgs a = args_of(*f);
  if (f->length == 0) {
    // no position: the state stays what it was
    if (!f->final_state) return ASTRA_OK;
    const int64_t n = a.B * a.H * a.P * a.N;
    if (f->initial) {
      ASTRA_HIP_CHECK(astra_rt::rt_memcpy(f->final_state, f->initial, n * sizeof(float), st), "state copy");
      return ASTRA_OK;
    }
    return astra_fill_i32((int32_t *)f->final_state, n, 0, stream);
  }
  ASTRA_SEQ_POINTER(f->x);
  ASTRA_SEQ_POINTER(f->dt);
  ASTRA_SEQ_POINTER(f->b);
  ASTRA_SEQ_POINTER(f->c);
  ASTRA_SEQ_POINTER(f->A);
  ASTRA_SEQ_POINTER(f->y);
  if (a.chunks > 1) a.cs = f->chunk_states;
  if (a.cs && !aligned(a.cs, 16)) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_state_scan_forward: chunk_states is not aligned to 16 bytes");
  if (a.segs > 1) {
    ASTRA_SEQ_POINTER(f->workspace);
    ASTRA_ABI_CHECK((int64_t)f->workspace_bytes, >=, (int64_t)(seg_floats(a) * sizeof(float)));
    if (!aligned(f->workspace, 16)) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_state_scan_forward: the workspace is not aligned to 16 bytes");
    a.seg = (float *)f->workspace;
    a.seg_log2 = a.seg + (size_t)a.B * a.H * a.segs * a.P * a.N;
  }
  return run_forward(*f, a, st);
}

int astra_state_scan_grad_workspace_size(const astra_state_scan *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  const ScanArgs a = args_of(*f);
  *bytes = (round4(chunk_floats(a)) + round4(seg_floats(a)) + round4(slice_floats(a)) + part_floats(a)) * sizeof(float);
  return ASTRA_OK;
}

int astra_state_scan_backward(const astra_state_scan_grad *g, void *stream) {
  ASTRA_SEQ_POINTER(g);
  const astra_state_scan &f = g->f;
  if (int rc = check(&f)) return rc;
  const hipStream_t st = as_stream(stream);
  ScanArgs a = args_of(f);
  a.dy = g->dy;
  a.dfinal = g->dfinal;
  a.dx = g->dx;
  a.ddt = g->ddt;
  a.db = g->db;
  a.dc = g->dc;
  a.dinitial = g->dinitial;
  if (f.batch == 0 || f.length == 0) {
    for (float *p : {g->dA, g->dD, g->ddt_bias})
      if (p)
        if (int rc = astra_fill_i32((int32_t *)p, a.H, 0, stream)) return rc;
    const int64_t n = a.B * a.H * a.P * a.N;
    if (!g->dinitial || n == 0) return ASTRA_OK;
    if (!g->dfinal) return astra_fill_i32((int32_t *)g->dinitial, n, 0, stream);
    ASTRA_HIP_CHECK(astra_rt::rt_memcpy(g->dinitial, g->dfinal, n * sizeof(float), st), "state copy");
    return ASTRA_OK;
  }
  for (const void *p : {f.x, f.dt, f.b, f.c, (const void *)f.A, g->dy, (const void *)g->dx, (const void *)g->ddt,
                        (const void *)g->db, (const void *)g->dc, (const void *)g->workspace})
    if (!p) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_state_scan_backward: a pointer is NULL");
  if (a.chunks > 1) {
    ASTRA_SEQ_POINTER(f.chunk_states);
    a.cs = f.chunk_states;
  }
  const size_t need = (round4(chunk_floats(a)) + round4(seg_floats(a)) + round4(slice_floats(a)) + part_floats(a)) * sizeof(float);
  ASTRA_ABI_CHECK((int64_t)g->workspace_bytes, >=, (int64_t)need);
  if (!aligned(g->workspace, 16) || !aligned(a.cs, 16))
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_state_scan_backward: the workspace or chunk_states is not aligned to 16 bytes");
  a.ds = (float *)g->workspace;
  a.seg = a.ds + round4(chunk_floats(a));
  a.seg_log2 = a.seg + (size_t)a.B * a.H * a.segs * a.P * a.N;
  a.dbc = a.seg + round4(seg_floats(a));
  a.part = a.dbc + round4(slice_floats(a));
  const int64_t e = 4 * (int64_t)elem_size(f.type);
  for (const void *p : {g->dy, (const void *)a.dx, (const void *)a.db, (const void *)a.dc}) a.vec = a.vec && aligned(p, e);
  a.vec = a.vec && aligned(a.dfinal, 16) && aligned(a.dinitial, 16);
  if (int rc = run_backward(f, a, st)) return rc;
  if (!g->dA && !g->dD && !g->ddt_bias) return ASTRA_OK;
  int64_t rows = a.B * a.chunks;
  const float *part = a.part;
  const unsigned cols = (unsigned)cdiv(3 * (int64_t)a.H, kSumCols);
  if (rows > 4 * kSumRows) {
    float *sums = a.part + (size_t)rows * a.H * 3;
    hipLaunchKernelGGL(scan_sum_rows_kernel, dim3(cols, kSumRows), dim3(kSumThreads), 0, st, part, rows, 3 * (int64_t)a.H, sums);
    ASTRA_HIP_CHECK(rt_last_error(), "scan_sum_rows_kernel launch");
    part = sums;
    rows = kSumRows;
  }
  hipLaunchKernelGGL(scan_sum_heads_kernel, dim3(cols), dim3(kSumThreads), 0, st, part, rows, a.H, g->dA, g->ddt_bias, g->dD);
  ASTRA_HIP_CHECK(rt_last_error(), "scan_sum_heads_kernel launch");
  return ASTRA_OK;
}

int astra_state_scan_step(const astra_state_scan_one *o, void *stream) {
  ASTRA_SEQ_POINTER(o);
  ASTRA_SEQ_TYPE_CHECK(o->type);
  ASTRA_ABI_CHECK(o->batch, >=, 0);
  ASTRA_ABI_CHECK(o->heads, >=, 1);
  ASTRA_ABI_CHECK(o->dim, >=, 1);
  ASTRA_ABI_CHECK(o->groups, >=, 1);
  ASTRA_ABI_CHECK(o->heads % o->groups, ==, 0);
  ASTRA_ABI_CHECK(o->state, >=, 1);
  ASTRA_ABI_CHECK(o->state, <=, ASTRA_SEQ_MAX_STATE);
  if (o->batch == 0) return ASTRA_OK;
  for (const void *p : {o->x, o->dt, o->b, o->c, (const void *)o->A, (const void *)o->h, (const void *)o->y})
    if (!p) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_state_scan_step: a pointer is NULL");
  StepArgs a{o->x, o->dt, o->b, o->c, o->A, o->D, o->dt_bias, o->h, o->y, o->batch, o->x_stride_b, o->x_stride_h,
             o->dt_stride_b, o->dt_stride_h, o->b_stride_b, o->b_stride_g, o->c_stride_b, o->c_stride_g, o->heads,
             o->dim, o->groups, o->state};
  const bool wide = a.N % 4 == 0 && aligned(a.h, 16);
  return o->type == ASTRA_SEQ_BF16 ? step<bf16>(a, wide, as_stream(stream)) : step<float>(a, wide, as_stream(stream));
}

}  // extern "C"
