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
// Types. x, B, C and dY enter the products as they are. What is computed in between (M, Q,
// the states, and the weighted B and C of the states' update) is in 32 bits; for bf16 inputs it
// enters a product as the sum of two bf16 values (16 bits of significand, an error of 4e-6
// at most), so each such product is two matrix instructions. For float inputs the
// products use the float matrix instructions, at 1/16 of the bf16 ones' rate.
//
// A chunk is handled by wavefronts that each own 16 of its positions. A product's result
// has its column in lane % 16 and four consecutive rows in its registers, which is the
// layout of an operand whose contracted index is those rows: scores are computed
// transposed, so that they enter the next product from registers.
#include "sequence.h"

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
  int32_t H, P, G, N, ptiles, chunks, seg_chunks, segs, slices;
  int32_t xv, bv, cv, yv, nv;  // whether 4 elements of a row can be accessed at once
};

// ---------------------------------------------------------------- operands of the products

// One operand of a product over 32 values of the contracted index k, for lane (q = lane / 16,
// r = lane % 16): row (or column) r and 8 values of k. Which 8 is free as long as both
// operands agree: 8q..8q+7 ("near"), or 4q..4q+3 and 16+4q..16+4q+3 ("far"), which is how
// two results of 16 rows each hold them.
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
  static __device__ __forceinline__ Split split(const float (&v)[8]) {
    Split s;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      s.hi[i] = (bf16)v[i];
      s.lo[i] = (bf16)(v[i] - (float)s.hi[i]);
    }
    return s;
  }
  static __device__ __forceinline__ void expand(const Frag &f, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)f[i];
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Frag &b) {
    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Split &a, const Frag &b) {
    mma(acc, a.lo, b);
    mma(acc, a.hi, b);
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Split &b) {
    mma(acc, a, b.lo);
    mma(acc, a, b.hi);
  }
};

template <>
struct Ops<float> {
  using Frag = FragF;
  using Split = FragF;
  static __device__ __forceinline__ Frag near(const float *row, int k0, int q) {
    Frag f;
    const f32x4 a = *reinterpret_cast<const f32x4 *>(row + k0 + 8 * q);
    const f32x4 b = *reinterpret_cast<const f32x4 *>(row + k0 + 8 * q + 4);
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
  static __device__ __forceinline__ void expand(const Frag &f, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = f.v[i];
  }
  static __device__ __forceinline__ void mma(f32x4 &acc, const Frag &a, const Frag &b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], acc, 0, 0, 0);
  }
};

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

// A state tile [R, K] (K contracted) in LDS: two bf16 parts, or floats.
template <class T, int R, int K>
struct StateTile {
  static constexpr int kRow = K + 16 / (int)sizeof(T);
  static constexpr size_t kPart = R * kRow * sizeof(T);
  static constexpr size_t kBytes = (sizeof(T) == 2 ? 2 : 1) * kPart;
  T *p;
  __device__ __forceinline__ typename Ops<T>::Split near(int r, int k0, int q) const {
    if constexpr (sizeof(T) == 2) {
      typename Ops<T>::Split s;
      s.hi = Ops<T>::near(p + r * kRow, k0, q);
      s.lo = Ops<T>::near(p + R * kRow + r * kRow, k0, q);
      return s;
    } else {
      return Ops<T>::near(p + r * kRow, k0, q);
    }
  }
  // contracted over the rows instead (floats only)
  __device__ __forceinline__ typename Ops<T>::Split across(int k, int r0, int q) const {
    FragF s;
#pragma unroll
    for (int i = 0; i < 8; ++i) s.v[i] = p[(r0 + 8 * q + i) * kRow + k];
    return s;
  }
  __device__ __forceinline__ void put4(int r, int k, const float (&v)[4]) const {
    if constexpr (sizeof(T) == 2) {
      bf16x4 hi, lo;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        hi[i] = (bf16)v[i];
        lo[i] = (bf16)(v[i] - (float)hi[i]);
      }
      *reinterpret_cast<bf16x4 *>(p + r * kRow + k) = hi;
      *reinterpret_cast<bf16x4 *>(p + R * kRow + r * kRow + k) = lo;
    } else {
      f32x4 f;
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = v[i];
      *reinterpret_cast<f32x4 *>(p + r * kRow + k) = f;
    }
  }
};

// ---------------------------------------------------------------------- global memory

template <class T>
struct V4 {
  typedef T type __attribute__((ext_vector_type(4)));
};

// 4 elements of a row from element f on, zeros from `n` on.
template <class T>
__device__ __forceinline__ typename V4<T>::type load4(const T *p, int f, int n, bool vec) {
  typename V4<T>::type r = {};
  if (vec) {
    if (f < n) r = *reinterpret_cast<const typename V4<T>::type *>(p + f);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f + i < n) r[i] = p[f + i];
  }
  return r;
}

template <class T>
__device__ __forceinline__ void store4(T *p, int f, int n, bool vec, const float (&v)[4]) {
  if (vec) {
    typename V4<T>::type r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
    if (f < n) *reinterpret_cast<typename V4<T>::type *>(p + f) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (f + i < n) p[f + i] = (T)v[i];
  }
}

// F features by Q positions on their way from memory to LDS: THREADS threads hold blocks of
// 4 positions by 4 features. Positions at and after `len` and features at and after `n`
// are zero, whatever memory holds there.
template <class T, int F, int THREADS>
struct Stage {
  static constexpr int kGroups = F / 4, kBlocks = kGroups * (Q / 4), kEach = (kBlocks + THREADS - 1) / THREADS;
  typename V4<T>::type v[kEach][4];
  __device__ __forceinline__ void load(const T *base, int64_t stride, int64_t t0, int len, int n, bool vec, int tid) {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS;
      const int f = (blk % kGroups) * 4, t = (blk / kGroups) * 4;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v[e][k] = {};
        if (blk < kBlocks && t0 + t + k < len) v[e][k] = load4<T>(base + (t0 + t + k) * stride, f, n, vec);
      }
    }
  }
  __device__ __forceinline__ void put(T *rows, T *cols, int tid) const {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const int blk = tid + e * THREADS;
      if (blk >= kBlocks) continue;
      const int f = (blk % kGroups) * 4, t = (blk / kGroups) * 4;
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

// ------------------------------------------------------------------------- step sizes

// What one wavefront, a lane a position, works out of a head's dt over a chunk.
struct Times {
  float dt[Q], hi[Q], lo[Q];  // the step; log2 of the decay from the chunk's start, in two parts
  float from[Q], left[Q];     // exp(s_t), exp(s_Q - s_t)
  float into[Q];              // dt exp(s_Q - s_t): what a position's input counts after the chunk
  float total;                // exp(s_Q)
};

__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

template <class T>
__device__ __forceinline__ float raw_step(const ScanArgs &a, int64_t b, int h, int64_t t, int len) {
  if (t >= len) return 0.f;
  return (float)((const T *)a.dt)[b * a.dsb + t * a.dst + h * a.dsh] + (a.bias ? a.bias[h] : 0.f);
}

// Fills `o` from this lane's raw step; returns log2 of the chunk's decay.
__device__ __forceinline__ double make_times(Times &o, float raw, bool live, float A, int lane) {
  const float dt = live ? softplus(raw) : 0.f;
  double s = (double)dt * (double)A * 1.4426950408889634;
#pragma unroll
  for (int m = 1; m < Q; m *= 2) {
    const double up = __shfl_up(s, m, kWave);
    if (lane >= m) s += up;
  }
  const double total = __shfl(s, Q - 1, kWave);
  o.dt[lane] = dt;
  o.hi[lane] = (float)s;
  o.lo[lane] = (float)(s - (double)(float)s);
  o.from[lane] = exp2f((float)s);
  o.left[lane] = exp2f((float)(total - s));
  o.into[lane] = dt * o.left[lane];
  if (lane == 0) o.total = exp2f((float)total);
  return total;
}

// --------------------------------------------------------- the states' update over a chunk

// This wavefront's part of a state [PT, NT] in registers: 16 x 16 tiles wave, wave + 4, ...
// of [n tile, p tile]; lane (q, r) of tile (nt, pt) has n = 16 nt + 4 q + 0..3, p = 16 pt + r.
template <int PT, int NT>
struct Mine {
  static constexpr int kN = NT / 16, kTiles = (PT / 16) * kN, kEach = kTiles / 4;
  static_assert(kTiles % 4 == 0, "four wavefronts share the tiles evenly");
  static __device__ __forceinline__ int n_of(int wave, int i, int q) { return ((wave + 4 * i) % kN) * 16 + 4 * q; }
  static __device__ __forceinline__ int p_of(int wave, int i, int r) { return ((wave + 4 * i) / kN) * 16 + r; }
};

// S = total S + X^T (weight K): X over PT features, K over NT, weight a position's.
template <class T, int PT, int NT>
__device__ __forceinline__ void update_state(f32x4 *S, float total, const float *weight,
                                             const Along<T, PT> &X, const Along<T, NT> &K, int wave, int q, int r) {
  using M = Mine<PT, NT>;
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) S[i] *= total;
#pragma unroll
  for (int t0 = 0; t0 < Q; t0 += 32) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = weight[t0 + 8 * q + e];
    typename Ops<T>::Split kf;
#pragma unroll
    for (int i = 0; i < M::kEach; ++i) {
      const int nt = (wave + 4 * i) % M::kN;
      if (i == 0 || M::kN > 4) {  // with up to 4 tiles of n a wavefront has only one of them
        float v[8];
        Ops<T>::expand(K.near(16 * nt + r, t0, q), v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= w[e];
        kf = Ops<T>::split(v);
      }
      Ops<T>::mma(S[i], kf, X.near(M::p_of(wave, i, r), t0, q));
    }
  }
}

template <int PT, int NT>
__device__ __forceinline__ void load_state(f32x4 *S, const float *base, const ScanArgs &a, int p0,
                                           int wave, int q, int r) {
  using M = Mine<PT, NT>;
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) {
    const int p = p0 + M::p_of(wave, i, r), n = M::n_of(wave, i, q);
    S[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (base && p < a.P) S[i] = load4<float>(base + (int64_t)p * a.N, n, a.N, a.nv);
  }
}

template <int PT, int NT>
__device__ __forceinline__ void store_state(const f32x4 *S, float *base, const ScanArgs &a, int p0,
                                            int wave, int q, int r) {
  using M = Mine<PT, NT>;
#pragma unroll
  for (int i = 0; i < M::kEach; ++i) {
    const int p = p0 + M::p_of(wave, i, r), n = M::n_of(wave, i, q);
    const float v[4] = {S[i][0], S[i][1], S[i][2], S[i][3]};
    if (p < a.P) store4<float>(base + (int64_t)p * a.N, n, a.N, a.nv, v);
  }
}

// ------------------------------------------------------------------------ forward

template <class T, int PT, int NT>
struct ForwardLds {
  static constexpr size_t x = 0;  // along positions only
  static constexpr size_t bn = x + (sizeof(T) == 2 ? Tile<T, PT>::kColsBytes : Tile<T, PT>::kRowsBytes);
  static constexpr size_t bt = bn + Tile<T, NT>::kRowsBytes;
  static constexpr size_t cn = bt + Tile<T, NT>::kColsBytes;
  static constexpr size_t h = cn + Tile<T, NT>::kRowsBytes;
  static constexpr size_t times = h + StateTile<T, PT, NT>::kBytes;
  static constexpr size_t bytes = times + sizeof(Times);
};

// One workgroup of four wavefronts: a head's PT features over a segment of chunks, one
// after the other, the state in registers between them.
template <class T, int PT, int NT>
__global__ __launch_bounds__(256) void scan_forward_kernel(ScanArgs a) {
  using L = ForwardLds<T, PT, NT>;
  using M = Mine<PT, NT>;
  extern __shared__ __align__(16) char lds[];
  T *xl = (T *)(lds + L::x), *bn = (T *)(lds + L::bn), *bt = (T *)(lds + L::bt), *cn = (T *)(lds + L::cn);
  const StateTile<T, PT, NT> hl{(T *)(lds + L::h)};
  Times &tm = *(Times *)(lds + L::times);
  const Along<T, PT> xa{xl, xl};
  const Along<T, NT> ba{bn, bt};

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, r = lane & 15;
  int64_t id = blockIdx.x;
  const int pt = (int)(id % a.ptiles);
  id /= a.ptiles;
  const int h = (int)(id % a.H);
  id /= a.H;
  const int64_t b = id % a.B;
  const int seg = (int)(id / a.B);
  const int g = h / (a.H / a.G), p0 = pt * PT, len = row_length(a.lengths, b, a.T);
  const int c0 = seg * a.seg_chunks, c1 = min(c0 + a.seg_chunks, a.chunks);
  const float A = a.A[h], D = a.D ? a.D[h] : 0.f;
  const T *xg = (const T *)a.x + b * a.xsb + h * a.xsh + p0;
  const T *bg = (const T *)a.b + b * a.bsb + g * a.bsg;
  const T *cg = (const T *)a.c + b * a.csb + g * a.csg;
  const int64_t bh = b * a.H + h, pn = (int64_t)a.P * a.N;

  f32x4 S[M::kEach];
  const float *start = a.segs > 1 ? a.seg + (bh * a.segs + seg) * pn : a.initial ? a.initial + bh * pn : nullptr;
  load_state<PT, NT>(S, start, a, p0, wave, q, r);
  bool any = start != nullptr;  // whether the state is more than zeros

  Stage<T, PT, 256> xs;
  Stage<T, NT, 256> bs, cs;
  for (int c = c0; c < c1; ++c) {
    const int64_t t0 = (int64_t)c * Q;
    xs.load(xg, a.xst, t0, len, a.P - p0, a.xv, tid);
    bs.load(bg, a.bst, t0, len, a.N, a.bv, tid);
    cs.load(cg, a.cst, t0, len, a.N, a.cv, tid);
    if constexpr (sizeof(T) == 2)
      xs.put(nullptr, xl, tid);
    else
      xs.put(xl, nullptr, tid);
    bs.put(bn, bt, tid);
    cs.put(cn, nullptr, tid);
    if (wave == 0) make_times(tm, raw_step<T>(a, b, h, t0 + lane, len), t0 + lane < len, A, lane);
    if (any) {
#pragma unroll
      for (int i = 0; i < M::kEach; ++i) {
        const float v[4] = {S[i][0], S[i][1], S[i][2], S[i][3]};
        hl.put4(M::p_of(wave, i, r), M::n_of(wave, i, q), v);
      }
    }
    if (a.cs) store_state<PT, NT>(S, a.cs + (bh * a.chunks + c) * pn, a, p0, wave, q, r);
    __syncthreads();

    // this wavefront's 16 positions i = 16 wave + r: Y^T, rows the features
    f32x4 y[PT / 16];
#pragma unroll
    for (int i = 0; i < PT / 16; ++i) y[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int ti = 16 * wave + r;
    typename Ops<T>::Frag cf[NT / 32];
#pragma unroll
    for (int k = 0; k < NT / 32; ++k) cf[k] = Ops<T>::near(cn + ti * Tile<T, NT>::kRow, 32 * k, q);
    if (any) {
      const float e = tm.from[ti];
#pragma unroll
      for (int i = 0; i < PT / 16; ++i) {
#pragma unroll
        for (int k = 0; k < NT / 32; ++k) Ops<T>::mma(y[i], hl.near(16 * i + r, 32 * k, q), cf[k]);
        y[i] *= e;
      }
    }
    const float hi = tm.hi[ti], lo = tm.lo[ti];
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {  // two tiles of 16 positions j at a time
      if (2 * jp > wave) break;
      float m[8];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int jt = 2 * jp + half;
        f32x4 s = {0.f, 0.f, 0.f, 0.f};
        if (jt <= wave) {
#pragma unroll
          for (int k = 0; k < NT / 32; ++k)
            Ops<T>::mma(s, Ops<T>::near(bn + (16 * jt + r) * Tile<T, NT>::kRow, 32 * k, q), cf[k]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int tj = 16 * jt + 4 * q + e;
          const float f = __builtin_amdgcn_exp2f((hi - tm.hi[tj]) + (lo - tm.lo[tj])) * tm.dt[tj];
          m[4 * half + e] = (tj <= ti ? s[e] * f : 0.f) + (tj == ti ? D : 0.f);
        }
      }
      const typename Ops<T>::Split mf = Ops<T>::split(m);
#pragma unroll
      for (int i = 0; i < PT / 16; ++i) Ops<T>::mma(y[i], xa.far(16 * i + r, 32 * jp, q), mf);
    }
    if (t0 + ti < a.T) {
      T *yp = (T *)a.y + ((b * a.T + t0 + ti) * a.H + h) * a.P + p0;
#pragma unroll
      for (int i = 0; i < PT / 16; ++i) {
        const float v[4] = {y[i][0], y[i][1], y[i][2], y[i][3]};
        store4<T>(yp, 16 * i + 4 * q, a.P - p0, a.yv, v);
      }
    }
    if (c + 1 < c1 || a.final_state) update_state<T, PT, NT>(S, tm.total, tm.into, xa, ba, wave, q, r);
    any = true;
    __syncthreads();
  }
  if (a.final_state && c1 == a.chunks) store_state<PT, NT>(S, a.final_state + bh * pn, a, p0, wave, q, r);
}

// ----------------------------------------------------------------- states of segments

template <class T, int PT, int NT>
struct StatesLds {
  static constexpr size_t x = 0;
  static constexpr size_t k = x + (sizeof(T) == 2 ? Tile<T, PT>::kColsBytes : Tile<T, PT>::kRowsBytes);
  static constexpr size_t times = k + (sizeof(T) == 2 ? Tile<T, NT>::kColsBytes : Tile<T, NT>::kRowsBytes);
  static constexpr size_t bytes = times + sizeof(Times);
};

// A segment's chunks without their outputs. Forwards: the state that the segment's inputs
// leave (x, w B). Backwards (REV): the gradient of the state before it that its outputs
// leave (dY, exp(s) C). KEEP: from what the segment starts from, writing what comes into
// each chunk (ds); otherwise from zero, writing what comes out and the segment's decay.
template <class T, int PT, int NT, bool REV, bool KEEP>
__global__ __launch_bounds__(256) void scan_states_kernel(ScanArgs a) {
  using L = StatesLds<T, PT, NT>;
  using M = Mine<PT, NT>;
  extern __shared__ __align__(16) char lds[];
  T *xl = (T *)(lds + L::x), *kl = (T *)(lds + L::k);
  Times &tm = *(Times *)(lds + L::times);
  const Along<T, PT> xa{xl, xl};
  const Along<T, NT> ka{kl, kl};
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, r = lane & 15;
  int64_t id = blockIdx.x;
  const int pt = (int)(id % a.ptiles);
  id /= a.ptiles;
  const int h = (int)(id % a.H);
  id /= a.H;
  const int64_t b = id % a.B;
  const int seg = (int)(id / a.B);
  const int g = h / (a.H / a.G), p0 = pt * PT, len = row_length(a.lengths, b, a.T);
  const int c0 = seg * a.seg_chunks, c1 = min(c0 + a.seg_chunks, a.chunks);
  const float A = a.A[h];
  const T *xg = REV ? (const T *)a.dy + (b * a.T * a.H + h) * a.P + p0 : (const T *)a.x + b * a.xsb + h * a.xsh + p0;
  const int64_t xstride = REV ? (int64_t)a.H * a.P : a.xst;
  const T *kg = REV ? (const T *)a.c + b * a.csb + g * a.csg : (const T *)a.b + b * a.bsb + g * a.bsg;
  const int64_t kstride = REV ? a.cst : a.bst;
  const int64_t bh = b * a.H + h, pn = (int64_t)a.P * a.N;
  f32x4 S[M::kEach];
  const float *start = !KEEP ? nullptr : a.segs > 1 ? a.seg + (bh * a.segs + seg) * pn : a.dfinal ? a.dfinal + bh * pn : nullptr;
  load_state<PT, NT>(S, start, a, p0, wave, q, r);
  double decay = 0.;
  Stage<T, PT, 256> xs;
  Stage<T, NT, 256> ks;
  for (int n = c0; n < c1; ++n) {
    const int c = REV ? c1 - 1 - (n - c0) : n;
    const int64_t t0 = (int64_t)c * Q;
    if (KEEP) {
      if (a.chunks > 1) store_state<PT, NT>(S, a.ds + (bh * a.chunks + c) * pn, a, p0, wave, q, r);
      if (c == 0 && !a.dinitial) break;
    }
    xs.load(xg, xstride, t0, len, a.P - p0, REV ? a.yv : a.xv, tid);
    ks.load(kg, kstride, t0, len, a.N, REV ? a.cv : a.bv, tid);
    if constexpr (sizeof(T) == 2) {
      xs.put(nullptr, xl, tid);
      ks.put(nullptr, kl, tid);
    } else {
      xs.put(xl, nullptr, tid);
      ks.put(kl, nullptr, tid);
    }
    if (wave == 0) decay += make_times(tm, raw_step<T>(a, b, h, t0 + lane, len), t0 + lane < len, A, lane);
    __syncthreads();
    update_state<T, PT, NT>(S, tm.total, REV ? tm.from : tm.into, xa, ka, wave, q, r);
    __syncthreads();
  }
  if (!KEEP) {
    store_state<PT, NT>(S, a.seg + (bh * a.segs + seg) * pn, a, p0, wave, q, r);
    if (tid == 0 && pt == 0) a.seg_log2[bh * a.segs + seg] = (float)decay;
  } else if (a.dinitial && c0 == 0) {
    store_state<PT, NT>(S, a.dinitial + bh * pn, a, p0, wave, q, r);
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
  for (int n = 0; n < a.segs; ++n) {
    const int s = REV ? a.segs - 1 - n : n;
    float *p = a.seg + (bh * a.segs + s) * pn + e;
    const float own = *p;
    *p = carry;
    carry = __builtin_amdgcn_exp2f(a.seg_log2[bh * a.segs + s]) * carry + own;
  }
}

// ----------------------------------------------------------------------- backward

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
  static constexpr size_t dht = dh + (ST ? StateTile<T, PT, NT>::kBytes : 0);              // [n][p]
  static constexpr size_t h0 = dht + (ST && two ? StateTile<T, NT, PT>::kBytes : 0);       // [n][p], floats [p][n]
  static constexpr size_t times = h0 + (!ST ? 0 : two ? StateTile<T, NT, PT>::kBytes : StateTile<T, PT, NT>::kBytes);
  static constexpr size_t sums = times + sizeof(Times);
  static constexpr size_t bytes = sums + (7 * Q + 2 * 8) * sizeof(float);
};

// One workgroup of eight wavefronts: a chunk of one row and one group's B and C, its heads
// one after the other, so that dB and dC are sums in registers. The first four wavefronts
// own 16 positions j each (dX, dB), the other four 16 positions i each (dC). ST: whether
// there are states before or after the chunk.
template <class T, int PT, int NT, bool ST>
__global__ __launch_bounds__(512) void scan_grad_kernel(ScanArgs a) {
  using L = GradLds<T, PT, NT, ST>;
  using O = Ops<T>;
  using BC = Tile<T, NT>;
  using XY = Tile<T, PT>;
  extern __shared__ __align__(16) char lds[];
  T *bn = (T *)(lds + L::bn), *bt = (T *)(lds + L::bt), *cn = (T *)(lds + L::cn), *ct = (T *)(lds + L::ct);
  T *xn = (T *)(lds + L::xn), *yn = (T *)(lds + L::yn), *yt = (T *)(lds + L::yt);
  const StateTile<T, PT, NT> dhl{(T *)(lds + L::dh)}, h0f{(T *)(lds + L::h0)};
  const StateTile<T, NT, PT> dhtl{(T *)(lds + L::dht)}, h0l{(T *)(lds + L::h0)};
  Times &tm = *(Times *)(lds + L::times);
  // of a head: C.(h0^T dY) and B.(dh1^T x) with their decays, sum_i of the pairs (i, j), for
  // each wavefront's j the pairs across a position, and two sums of each wavefront
  float *uc = (float *)(lds + L::sums), *vb = uc + Q, *col = vb + Q, *cross = col + Q, *red = cross + 4 * Q;
  const Along<T, NT> ba{bn, bt}, ca{cn, ct};
  const Along<T, PT> ya{yn, yt};

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane >> 4, r = lane & 15;
  int64_t id = blockIdx.x;
  const int slice = (int)(id % a.slices);
  id /= a.slices;
  const int g = (int)(id % a.G);
  id /= a.G;
  const int c = (int)(id % a.chunks);
  const int64_t b = id / a.chunks;
  const int len = row_length(a.lengths, b, a.T), per = a.H / a.G;
  const int64_t t0 = (int64_t)c * Q, pn = (int64_t)a.P * a.N;
  const int h_lo = g * per + (int)((int64_t)per * slice / a.slices);
  const int h_hi = g * per + (int)((int64_t)per * (slice + 1) / a.slices);
  const bool own_j = wave < 4;
  const int mine = wave & 3, tw = 16 * mine + r;  // this lane's position

  {
    Stage<T, NT, 512> s;
    s.load((const T *)a.b + b * a.bsb + g * a.bsg, a.bst, t0, len, a.N, a.bv, tid);
    s.put(bn, bt, tid);
    s.load((const T *)a.c + b * a.csb + g * a.csg, a.cst, t0, len, a.N, a.cv, tid);
    s.put(cn, ct, tid);
  }
  f32x4 acc[NT / 16];  // dB^T (rows n, columns j), or dC^T, over the heads
#pragma unroll
  for (int i = 0; i < NT / 16; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int h = h_lo; h < h_hi; ++h) {
    const int64_t bh = b * a.H + h;
    const float *h0 = !ST ? nullptr : a.chunks > 1 ? a.cs + (bh * a.chunks + c) * pn : a.initial ? a.initial + bh * pn : nullptr;
    const float *dh = !ST ? nullptr : a.chunks > 1 ? a.ds + (bh * a.chunks + c) * pn : a.dfinal ? a.dfinal + bh * pn : nullptr;
    const float A = a.A[h], D = a.D ? a.D[h] : 0.f;
    const bool live = t0 + lane < len;
    float raw = 0.f;
    float dot = 0.f, diag = 0.f, inter = 0.f, cols = 0.f;
    for (int pt = 0; pt < a.ptiles; ++pt) {
      const int p0 = pt * PT;
      if (pt == 0 && wave == 0) {
        raw = raw_step<T>(a, b, h, t0 + lane, len);
        make_times(tm, raw, live, A, lane);
      }
      {
        Stage<T, PT, 512> s, u;
        s.load((const T *)a.x + b * a.xsb + h * a.xsh + p0, a.xst, t0, len, a.P - p0, a.xv, tid);
        u.load((const T *)a.dy + (b * a.T * a.H + h) * a.P + p0, (int64_t)a.H * a.P, t0, len, a.P - p0, a.yv, tid);
        s.put(xn, nullptr, tid);
        u.put(yn, yt, tid);
      }
      if constexpr (ST) {
        constexpr int kBlocks = (PT / 4) * (NT / 4);
        for (int blk = tid; blk < kBlocks; blk += 512) {
          const int n = (blk % (NT / 4)) * 4, p = (blk / (NT / 4)) * 4;
          float u[4][4], v[4][4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f}, w = s;
            if (p0 + p + k < a.P) {
              if (h0) s = load4<float>(h0 + (int64_t)(p0 + p + k) * a.N, n, a.N, a.nv);
              if (dh) w = load4<float>(dh + (int64_t)(p0 + p + k) * a.N, n, a.N, a.nv);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              u[k][i] = s[i];
              v[k][i] = w[i];
              dot += s[i] * w[i];
            }
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float ut[4] = {u[0][k], u[1][k], u[2][k], u[3][k]}, vt[4] = {v[0][k], v[1][k], v[2][k], v[3][k]};
            dhl.put4(p + k, n, v[k]);
            if constexpr (L::two) {
              dhtl.put4(n + k, p, vt);
              h0l.put4(n + k, p, ut);
            } else {
              h0f.put4(p + k, n, u[k]);
            }
          }
        }
      }
      __syncthreads();

      f32x4 own[NT / 16];  // this head's dB^T / dt or dC^T
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) own[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      const float hi = tm.hi[tw], lo = tm.lo[tw];
      if (own_j) {
        f32x4 dx[PT / 16];
#pragma unroll
        for (int i = 0; i < PT / 16; ++i) dx[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        typename O::Frag bf[NT / 32], xf[PT / 32];
#pragma unroll
        for (int k = 0; k < NT / 32; ++k) bf[k] = O::near(bn + tw * BC::kRow, 32 * k, q);
#pragma unroll
        for (int k = 0; k < PT / 32; ++k) xf[k] = O::near(xn + tw * XY::kRow, 32 * k, q);
        const float left = tm.left[tw], dt = tm.dt[tw];
        if (ST && dh) {
#pragma unroll
          for (int i = 0; i < PT / 16; ++i) {
#pragma unroll
            for (int k = 0; k < NT / 32; ++k) O::mma(dx[i], dhl.near(16 * i + r, 32 * k, q), bf[k]);
            dx[i] *= left * dt;
          }
#pragma unroll
          for (int i = 0; i < NT / 16; ++i) {
#pragma unroll
            for (int k = 0; k < PT / 32; ++k) {
              if constexpr (L::two)
                O::mma(own[i], dhtl.near(16 * i + r, 32 * k, q), xf[k]);
              else
                O::mma(own[i], dhl.across(16 * i + r, 32 * k, q), xf[k]);
            }
            own[i] *= left;
          }
#pragma unroll
          for (int i = 0; i < NT / 16; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              inter += own[i][e] * (float)bn[tw * BC::kRow + 16 * i + 4 * q + e];
        }
        float later = 0.f;  // the pairs (i, j) of the tiles of i after this one
#pragma unroll
        for (int ip = 1; ip >= 0; --ip) {
          if (2 * ip + 1 < mine) continue;
          float m[8], s[8];
#pragma unroll
          for (int half = 1; half >= 0; --half) {
            const int it = 2 * ip + half;
            f32x4 gs = {0.f, 0.f, 0.f, 0.f}, ms = gs;
            if (it >= mine) {
#pragma unroll
              for (int k = 0; k < NT / 32; ++k) O::mma(gs, O::near(cn + (16 * it + r) * BC::kRow, 32 * k, q), bf[k]);
#pragma unroll
              for (int k = 0; k < PT / 32; ++k) O::mma(ms, O::near(yn + (16 * it + r) * XY::kRow, 32 * k, q), xf[k]);
            }
            float pair[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int ti = 16 * it + 4 * q + e;
              const float f = __builtin_amdgcn_exp2f((tm.hi[ti] - hi) + (tm.lo[ti] - lo));
              const float d = ti >= tw ? ms[e] * f : 0.f;
              m[4 * half + e] = (ti >= tw ? gs[e] * f * dt : 0.f) + (ti == tw ? D : 0.f);
              s[4 * half + e] = d;
              pair[e] = d * gs[e];
              diag += ti == tw ? ms[e] : 0.f;
            }
            if (it >= mine) {
              // from each i to the chunk's end, then over the j before i
              pair[2] += pair[3];
              pair[1] += pair[2];
              pair[0] += pair[1];
              float from = pair[0], up = __shfl_down(from, 16, kWave);
              from += q < 3 ? up : 0.f;
              up = __shfl_down(from, 32, kWave);
              from += q < 2 ? up : 0.f;
              up = __shfl_down(from, 16, kWave);
              const float after = later + (q < 3 ? up : 0.f);
              f32x4 over;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float v = tw < 16 * it + 4 * q + e ? (pair[e] + after) * dt : 0.f;
#pragma unroll
                for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d, kWave);
                over[e] = v;
              }
              if (r == 0) {
                f32x4 *o = reinterpret_cast<f32x4 *>(cross + mine * Q + 16 * it + 4 * q);
                *o = pt ? *o + over : over;
              }
              later += __shfl(from, r, kWave);
            }
          }
          const typename O::Split mf = O::split(m), sf = O::split(s);
#pragma unroll
          for (int i = 0; i < PT / 16; ++i) O::mma(dx[i], ya.far(16 * i + r, 32 * ip, q), mf);
#pragma unroll
          for (int i = 0; i < NT / 16; ++i) O::mma(own[i], ca.far(16 * i + r, 32 * ip, q), sf);
        }
        cols += later;
        if (t0 + tw < a.T) {
          T *xp = (T *)a.dx + ((b * a.T + t0 + tw) * a.H + h) * a.P + p0;
#pragma unroll
          for (int i = 0; i < PT / 16; ++i) {
            const float v[4] = {dx[i][0], dx[i][1], dx[i][2], dx[i][3]};
            store4<T>(xp, 16 * i + 4 * q, a.P - p0, a.yv, v);
          }
        }
#pragma unroll
        for (int i = 0; i < NT / 16; ++i) acc[i] += own[i] * dt;
      } else {
        typename O::Frag yf[PT / 32];
#pragma unroll
        for (int k = 0; k < PT / 32; ++k) yf[k] = O::near(yn + tw * XY::kRow, 32 * k, q);
        if (ST && h0) {
          const float from = tm.from[tw];
#pragma unroll
          for (int i = 0; i < NT / 16; ++i) {
#pragma unroll
            for (int k = 0; k < PT / 32; ++k) {
              if constexpr (L::two)
                O::mma(own[i], h0l.near(16 * i + r, 32 * k, q), yf[k]);
              else
                O::mma(own[i], h0f.across(16 * i + r, 32 * k, q), yf[k]);
            }
            own[i] *= from;
#pragma unroll
            for (int e = 0; e < 4; ++e) inter += own[i][e] * (float)cn[tw * BC::kRow + 16 * i + 4 * q + e];
          }
        }
#pragma unroll
        for (int jp = 0; jp < 2; ++jp) {
          if (2 * jp > mine) break;
          float s[8];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int jt = 2 * jp + half;
            f32x4 ms = {0.f, 0.f, 0.f, 0.f};
            if (jt <= mine) {
#pragma unroll
              for (int k = 0; k < PT / 32; ++k) O::mma(ms, O::near(xn + (16 * jt + r) * XY::kRow, 32 * k, q), yf[k]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int tj = 16 * jt + 4 * q + e;
              const float f = __builtin_amdgcn_exp2f((hi - tm.hi[tj]) + (lo - tm.lo[tj])) * tm.dt[tj];
              s[4 * half + e] = tj <= tw ? ms[e] * f : 0.f;
            }
          }
          const typename O::Split sf = O::split(s);
#pragma unroll
          for (int i = 0; i < NT / 16; ++i) O::mma(own[i], ba.far(16 * i + r, 32 * jp, q), sf);
        }
#pragma unroll
        for (int i = 0; i < NT / 16; ++i) acc[i] += own[i];
      }
      if (pt + 1 == a.ptiles) {
        // a position's n are spread over the four lanes of one r
        inter += __shfl_xor(inter, 16, kWave);
        inter += __shfl_xor(inter, 32, kWave);
        if (q == 0) {
          (own_j ? vb : uc)[tw] = inter;
          if (own_j) col[tw] = cols;
        }
        dot = wave_sum(dot);
        diag = wave_sum(diag);
        if (lane == 0) {
          red[wave] = dot;
          red[8 + wave] = diag;
        }
      }
      __syncthreads();
    }
    if (wave == 0) {
      float dot_all = 0.f, diag_all = 0.f, over = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        dot_all += red[i];
        diag_all += red[8 + i];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) over += 16 * i <= lane ? cross[i * Q + lane] : 0.f;
      const float dt = tm.dt[lane], bdv = col[lane] + vb[lane], into = dt * vb[lane];
      float before = into, after = uc[lane];  // sums over j <= t, i >= t
#pragma unroll
      for (int m = 1; m < Q; m *= 2) {
        const float lower = __shfl_up(before, m, kWave), upper = __shfl_down(after, m, kWave);
        if (lane >= m) before += lower;
        if (lane + m < Q) after += upper;
      }
      before = __shfl_up(before, 1, kWave);
      if (lane == 0) before = 0.f;
      const float da = (before + after) + (over + tm.total * dot_all);
      const float ddt = live ? (A * da + bdv) / (1.f + expf(-raw)) : 0.f;
      if (t0 + lane < a.T) ((T *)a.ddt)[(b * a.T + t0 + lane) * a.H + h] = (T)ddt;
      const float dA = wave_sum(da * dt), dbias = wave_sum(ddt);
      if (lane == 0) {
        float *o = a.part + ((b * a.chunks + c) * a.H + h) * 3;
        o[0] = dA;
        o[1] = dbias;
        o[2] = diag_all;
      }
    }
  }
  if (t0 + tw < a.T) {
    const int64_t row = (b * a.T + t0 + tw) * a.G + g;
    if (a.slices == 1) {
      T *o = (T *)(own_j ? a.db : a.dc) + row * a.N;
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) {
        const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
        store4<T>(o, 16 * i + 4 * q, a.N, a.nv, v);
      }
    } else {
      float *o = a.dbc + ((int64_t)(slice * 2 + !own_j) * a.B * a.T * a.G + row) * a.N;
#pragma unroll
      for (int i = 0; i < NT / 16; ++i) {
        const float v[4] = {acc[i][0], acc[i][1], acc[i][2], acc[i][3]};
        store4<float>(o, 16 * i + 4 * q, a.N, a.nv, v);
      }
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
// of them in flight at once as it has, and does the head's step size once for them.
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

// The tile of features and of states that a call is padded to. With states over 64 the
// backward kernel's tiles fit a CU's LDS for 32 features only.
struct Tiles {
  int p, n;
};
Tiles tiles_of(const astra_state_scan &f) {
  Tiles t;
  t.n = f.state <= 32 ? 32 : f.state <= 64 ? 64 : 128;
  t.p = t.n == 128 || f.dim <= 32 ? 32 : 64;
  return t;
}

constexpr int64_t kFull = 512;  // workgroups that fill the card

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
  a.ptiles = (int32_t)cdiv(f.dim, tiles_of(f).p);
  a.chunks = (int32_t)cdiv(f.length, Q);
  // few rows: the length is split into segments, joined by their states
  const int64_t rows = a.B * a.H * a.ptiles;
  int64_t segs = 1;
  if (rows > 0 && rows < kFull) segs = cdiv(kFull, rows);
  if (segs > a.chunks / 2) segs = a.chunks / 2;
  if (segs < 1) segs = 1;
  a.seg_chunks = (int32_t)cdiv(a.chunks, segs);
  a.segs = a.seg_chunks ? (int32_t)cdiv(a.chunks, a.seg_chunks) : 1;
  // few chunks: the heads of a group are split, and their parts of db and dc added up
  const int64_t items = a.B * a.chunks * a.G;
  const int per = a.H / a.G;
  a.slices = items > 0 && items < kFull / 2 ? (int32_t)std::min<int64_t>(per, cdiv(kFull / 2, items)) : 1;
  const int64_t e = 4 * (int64_t)elem_size(f.type);
  a.xv = a.P % 4 == 0 && a.xsb % 4 == 0 && a.xst % 4 == 0 && a.xsh % 4 == 0 && aligned(a.x, e);
  a.bv = a.N % 4 == 0 && a.bsb % 4 == 0 && a.bst % 4 == 0 && a.bsg % 4 == 0 && aligned(a.b, e);
  a.cv = a.N % 4 == 0 && a.csb % 4 == 0 && a.cst % 4 == 0 && a.csg % 4 == 0 && aligned(a.c, e);
  a.yv = a.P % 4 == 0 && aligned(a.y, e);
  a.nv = a.N % 4 == 0 && aligned(a.initial, 16) && aligned(a.final_state, 16);
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

// More than 64 KB of LDS has to be asked for, once per kernel and device.
template <class K>
int allow_lds(K *kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    ASTRA_HIP_CHECK(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                        hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
                    "hipFuncSetAttribute");
  return ASTRA_OK;
}

#define SCAN_LAUNCH(kernel, blocks, threads, bytes)                                                    \
  do {                                                                                                 \
    ASTRA_ABI_CHECK(blocks, <, 2147483648ll);                                                          \
    if (int rc = allow_lds(&kernel, bytes)) return rc;                                                 \
    hipLaunchKernelGGL((kernel), dim3((unsigned)(blocks)), dim3(threads), bytes, st, a);               \
    ASTRA_HIP_CHECK(rt_last_error(), #kernel " launch");                                               \
  } while (false)

template <class T, int PT, int NT>
int forward(ScanArgs &a, hipStream_t st) {
  const int64_t blocks = a.B * a.H * a.ptiles * a.segs;
  if (a.segs > 1) {
    SCAN_LAUNCH((scan_states_kernel<T, PT, NT, false, false>), blocks, 256, (StatesLds<T, PT, NT>::bytes));
    hipLaunchKernelGGL(scan_carry_kernel<false>, dim3((unsigned)cdiv(a.B * a.H * a.P * a.N, 256)), dim3(256), 0, st, a);
    ASTRA_HIP_CHECK(rt_last_error(), "scan_carry_kernel launch");
  }
  SCAN_LAUNCH((scan_forward_kernel<T, PT, NT>), blocks, 256, (ForwardLds<T, PT, NT>::bytes));
  return ASTRA_OK;
}

template <class T, int PT, int NT>
int backward(ScanArgs &a, hipStream_t st) {
  if (a.chunks > 1 || a.dinitial) {
    const int64_t blocks = a.B * a.H * a.ptiles * a.segs;
    if (a.segs > 1) {
      SCAN_LAUNCH((scan_states_kernel<T, PT, NT, true, false>), blocks, 256, (StatesLds<T, PT, NT>::bytes));
      hipLaunchKernelGGL(scan_carry_kernel<true>, dim3((unsigned)cdiv(a.B * a.H * a.P * a.N, 256)), dim3(256), 0, st, a);
      ASTRA_HIP_CHECK(rt_last_error(), "scan_carry_kernel launch");
    }
    SCAN_LAUNCH((scan_states_kernel<T, PT, NT, true, true>), blocks, 256, (StatesLds<T, PT, NT>::bytes));
  }
  const int64_t blocks = a.B * a.chunks * a.G * a.slices;
  if (a.chunks > 1 || a.initial || a.dfinal)
    SCAN_LAUNCH((scan_grad_kernel<T, PT, NT, true>), blocks, 512, (GradLds<T, PT, NT, true>::bytes));
  else
    SCAN_LAUNCH((scan_grad_kernel<T, PT, NT, false>), blocks, 512, (GradLds<T, PT, NT, false>::bytes));
  if (a.slices > 1) {
    hipLaunchKernelGGL(scan_join_slices_kernel<T>, dim3((unsigned)cdiv(2 * a.B * a.T * a.G * a.N, 256)), dim3(256), 0, st, a);
    ASTRA_HIP_CHECK(rt_last_error(), "scan_join_slices_kernel launch");
  }
  return ASTRA_OK;
}

#define SCAN_TILES(FN)                                                    \
  do {                                                                    \
    const bool h = f.type == ASTRA_SEQ_BF16;                              \
    if (t.n == 128) return h ? FN<bf16, 32, 128>(a, st) : FN<float, 32, 128>(a, st); \
    if (t.n == 64 && t.p == 32) return h ? FN<bf16, 32, 64>(a, st) : FN<float, 32, 64>(a, st); \
    if (t.n == 64) return h ? FN<bf16, 64, 64>(a, st) : FN<float, 64, 64>(a, st); \
    if (t.p == 32) return h ? FN<bf16, 32, 32>(a, st) : FN<float, 32, 32>(a, st); \
    return h ? FN<bf16, 64, 32>(a, st) : FN<float, 64, 32>(a, st);        \
  } while (false)

int run_forward(const astra_state_scan &f, ScanArgs &a, hipStream_t st) {
  const Tiles t = tiles_of(f);
  SCAN_TILES(forward);
}
int run_backward(const astra_state_scan &f, ScanArgs &a, hipStream_t st) {
  const Tiles t = tiles_of(f);
  SCAN_TILES(backward);
}

template <class T>
int step(const StepArgs &a, bool wide, hipStream_t st) {
#define STEP_LAUNCH(V, LPR, NJ)                                                                       \
  do {                                                                                                \
    const int64_t blocks = cdiv(a.B * a.H * cdiv(a.P, kStepRows / LPR), 4);                           \
    ASTRA_ABI_CHECK(blocks, <, 2147483648ll);                                                         \
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
  a.yv = a.P % 4 == 0 && aligned(a.dy, e) && aligned(a.dx, e);
  a.nv = a.N % 4 == 0 && aligned(a.initial, 16) && aligned(a.dfinal, 16) && aligned(a.dinitial, 16) && aligned(a.db, e) && aligned(a.dc, e);
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
