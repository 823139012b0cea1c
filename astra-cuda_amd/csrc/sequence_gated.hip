// sequence_gated.hip -- the gated feed-forward block before its way back:
//
//   a = x Wg^T,  b = x Wu^T,  h = act(a) * b          x [M,D]; Wg, Wu [F,D]; h [M,F]
//   da = dh b act'(a),  db = dh act(a)
//   dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x
//
// All are matrix products out[r, l] = sum_k left[l, k] right[r, k] on the matrix cores, with
// what surrounds them done on the accumulators: 4 M D F operations forwards, 8 M D F backwards, and 4 M D F
// again where a and b are computed a second time. Sums are float32; h is rounded once, da and db are
// rounded to x's type before their products, as the matrix cores take them (2^-8 of bf16 each, which
// makes the gradients' error 1.4 times that of h), or to two bf16 numbers each where the caller asks
// for exact gradients: 8 M D F operations more, whole passes of 81,920 rows of 256 to 1,024 850 us and
// not 580, of 16,384 rows of 4,096 to 8,192 9,800 and not 6,030.
//
// Measured (us; the card's large bf16 library product reaches 1,390 TFLOP/s, its float product 154,
// its copies 4.8 TB/s):
//   16,384 rows of 4,096 to 8,192, bf16   h 1,890 (1,160 TFLOP/s), da and db 345 (5.4 TB/s), weights turned 52, dx 1,849
//                                         (1,190), dWg and dWu 1,805 (1,220)
//   81,920 rows of 256 to 1,024, bf16     h 133, da and db 204 (a and b again), dx 145, dWg and dWu 113 + 14
//   30,000 rows of 256 to 683, float      h 225, da and db 74, dx 189, dWg and dWu 209 + 18
//   one row of 256 to 1,024               3.5; of 4,096 to 8,192 33 (4.1 TB/s), 64 such rows 46 to 51
// The matrix cores are busy 60% of the wide bf16 products' time at some 2.1 GHz, and their power holds the
// clock there; 75% of the float products'. Rows of 256 have 4 steps: bound by the results' traffic (h alone is
// 168 MB) and by how little of it overlaps with the products. Few rows are bound by the weights' traffic.
#include <algorithm>

#include "sequence.h"

#define ASTRA_SRC_NAME "sequence_gated.hip"

namespace astra_seq {
namespace {

// ------------------------------------------------------------------ tiles of a product
//
// A workgroup of WL x WR wavefronts has a tile of BL x BR results, a wavefront NL x NR of 16 x 16.
// 128 bytes of the contraction at a time (64 bf16 or 32 floats) are brought straight into LDS, which the
// products read as fragments: lane i has 16 bytes of line i % 16, the (i / 16)-th of its four. (Products
// of 32 x 32 are no faster: 1,710-1,780 TFLOP/s alone to 1,620-1,940.)
//
// An operand lies along the contraction (a line of the tile is 128 contiguous bytes) or across it
// (TR: the tile is 64 or 32 rows of memory, a line is a column). Its memory starts on 16 bytes, as
// does every row of it, and what lies outside of it is never read: accesses are checked against the
// buffer's size, and bring zeros from outside.
//
// The 16-byte pieces of a row in LDS are permuted (by an exclusive or with a number of the row) so
// that the lanes of a fragment fall on all banks.
typedef uint32_t Piece __attribute__((ext_vector_type(4)));
constexpr int kStep = 128;           // bytes of the contraction in a step
constexpr uint32_t kOutside = 0x7ffffff0u;

template <class T>
constexpr int kStepOf = kStep / (int)sizeof(T);

template <class T>
struct Fragment;
template <>
struct Fragment<bf16> {
  typedef bf16x8 type;
};
template <>
struct Fragment<float> {
  typedef f32x4 type;
};
template <class T>
using Frag = typename Fragment<T>::type;

__device__ __forceinline__ void multiply(f32x4 &acc, const bf16x8 &l, const bf16x8 &r) {
  acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(l, r, acc, 0, 0, 0);
}
__device__ __forceinline__ void multiply(f32x4 &acc, const f32x4 &l, const f32x4 &r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(l[i], r[i], acc, 0, 0, 0);
}

template <class T>
constexpr int kProducts = sizeof(T) == 2 ? 1 : 4;  // instructions

// An operand: `lines` lines of `len` elements of the contraction, rows `ld` elements apart.
struct Operand {
  const void *p;
  int64_t ld, lines, len;
};

// The part of an operand that one wavefront of NW brings into LDS: B lines from `line0` on.
template <class T, bool TR, int B, int NW, bool PAIRED>
struct Loader {
  static constexpr int N = B * kStep / 1024 / NW;               // loads of 1024 bytes
  static constexpr int kRow = TR ? B * (int)sizeof(T) : kStep;  // bytes of a row in LDS
  static constexpr int kPieces = kRow / 16, kRows = 64 / kPieces;  // (rows of one load)
  static constexpr int kReads = !TR ? 1 : sizeof(T) == 2 ? 2 : 4;  // LDS accesses of a fragment
  static_assert(!TR || kRow >= 256, "rows of a tile across the contraction cover all banks");
  static_assert(TR || NW % 2 == 0, "along the contraction a lane has the same piece of all its rows");
  const char *base;
  int32_t ld, lines;  // bytes from row to row; lines of the tile inside the operand (TR: their bytes)
  int64_t left;       // bytes (TR: rows) of the contraction from base on
  uint32_t off[N];
  int32_t piece;

  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!TR) return PAIRED ? 2 * ((row >> 3) & 3) + ((row >> 1) & 1) : (row >> 1) & 7;
    if constexpr (sizeof(T) == 2) return 2 * ((row & 3) + 4 * ((row >> 3) & 1));
    return 4 * ((row >> 2) & 3);
  }

  __device__ __forceinline__ void init(const Operand &o, int64_t line0, int wave, int lane) {
    ld = (int32_t)(o.ld * (int64_t)sizeof(T));
    lines = (int32_t)max((int64_t)0, min((int64_t)B, o.lines - line0)) * (TR ? (int)sizeof(T) : 1);
    base = (const char *)o.p + line0 * (TR ? (int64_t)sizeof(T) : (int64_t)ld);
    left = o.len * (TR ? 1 : (int64_t)sizeof(T));
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int row = (wave + NW * j) * kRows + lane / kPieces;
      piece = ((lane % kPieces) ^ swizzle(row)) * 16;
      off[j] = (TR ? piece : row) < lines ? (uint32_t)(row * ld + piece) : kOutside;
    }
  }

  // The operand's contraction from k0 on, `len` at most.
  static __device__ __forceinline__ void cut(Operand &o, int64_t k0, int64_t len) {
    o.p = (const T *)o.p + (TR ? k0 * o.ld : k0);
    o.len = max((int64_t)0, min(len, o.len - k0));
  }

  // Brings the next step into `lds` and moves on; zeros after the last.
  __device__ __forceinline__ void load(char *lds, int wave) {
    constexpr int kMost = TR ? kStepOf<T> : kStep;
    const int most = (int)min(left, (int64_t)kMost);
    int bytes = TR ? (most - 1) * ld + lines : (lines - 1) * ld + most;
    bytes = ((most > 0) & (lines > 0)) ? bytes : 0;
    const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, bytes, 0x00020000);
    const bool out = !TR && piece >= most;
#pragma unroll
    for (int j = 0; j < N; ++j)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void *)(lds + (wave + NW * j) * 1024), 16,
          out ? kOutside : off[j], 0, 0, 0);
    base += TR ? (int64_t)kMost * ld : kMost;
    left -= kMost;
  }
};

// A lane's fragments of an operand's tile in LDS, from its tile `first` of 16 lines on: tile `t` of a
// wavefront, half `s` of the step. With PAIRED, lines 4 q .. 4 q + 3 of two neighbouring tiles are 8
// neighbouring lines of the operand, so that a lane has 8 neighbouring results.
template <class T, bool TR, int B, bool PAIRED>
struct Reader {
  static constexpr int kRow = TR ? B * (int)sizeof(T) : kStep;
  uint32_t at;

  __device__ __forceinline__ void init(int first, int lane) {
    const int i = lane % 16, g = lane / 16;
    if constexpr (!TR) {
      const int row = PAIRED ? 8 * (i / 4) + i % 4 : i, swz = PAIRED ? 2 * (i / 4) + (i % 4) / 2 : i / 2;
      at = (16 * first + row) * kStep + ((g ^ swz) * 16);
    } else if constexpr (sizeof(T) == 2) {
      const int x = 2 * ((i / 4) + 4 * (g & 1));
      at = (8 * g + i / 4) * kRow + (((2 * first + (i % 4) / 2) ^ x) * 16) + (i % 2) * 8;
    } else {
      at = 4 * g * kRow + (((4 * first + i / 4) ^ (4 * g)) * 16) + (i % 4) * 4;
    }
  }
  // Takes the addresses of the tiles anew from here on: an operation each, where the compiler would
  // keep them all in registers that are not there.
  __device__ __forceinline__ void again() { asm volatile("" : "+v"(at)); }

  __device__ __forceinline__ Frag<T> read(const char *lds, int t, int s) const {
    if constexpr (!TR) {
      const int row = PAIRED ? 32 * (t / 2) + 4 * (t % 2) : 16 * t;
      return *reinterpret_cast<const Frag<T> *>(lds + (at ^ (64 * s)) + row * kStep);
    } else if constexpr (sizeof(T) == 2) {
      // rows 32 s + 8 g + 0..3 and + 4..7: 4 lanes bring 16 lines of a row, each lane gets a line
      const char *p = lds + (at ^ (32 * t)) + 32 * s * kRow;
      typedef short s16x4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s16x4 *Lds;
      const bf16x4 a = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p));
      const bf16x4 b = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)(p + 4 * kRow)));
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      Frag<T> f;
      const char *p = lds + (at ^ (64 * t)) + 16 * s * kRow;
#pragma unroll
      for (int n = 0; n < 4; ++n) f[n] = *reinterpret_cast<const float *>(p + n * kRow);
      return f;
    }
  }
};

// A workgroup's tile: WL x WR wavefronts of NL x NR times 16 x 16 results. HALVES: the left tile is
// two operands of BL / 2 lines each, of which a wavefront has the same lines, PAIRED as above. GROUPS
// workgroups share a CU.
template <class T, bool LTR, bool RTR, int NL_, int NR_, bool HALVES_, int GROUPS_, int WL_ = 2, int WR_ = 2>
struct Product {
  static constexpr int NL = NL_, NR = NR_, WL = WL_, WR = WR_, GROUPS = GROUPS_;
  static constexpr bool HALVES = HALVES_;
  static constexpr int NW = WL * WR, BL = 16 * NL * WL, BR = 16 * NR * WR;
  static constexpr int kBytes = (BL + BR) * kStep, kThreads = 64 * NW;
  static constexpr int BLL = HALVES ? BL / 2 : BL;  // lines of a left operand
  static constexpr int NLL = HALVES ? NL / 2 : NL;  // tiles of it to a wavefront
  static_assert(kBytes * (GROUPS == 1 ? 2 : GROUPS) <= 160 * 1024, "the LDS of a CU");
  typedef T type;
  typedef Loader<T, LTR, BLL, NW, HALVES> Left;
  typedef Loader<T, RTR, BR, NW, false> Right;
  typedef Reader<T, LTR, BLL, HALVES> LeftReader;
  typedef Reader<T, RTR, BR, false> RightReader;

  // The fragments of half a step.
  struct Half {
    Frag<T> l[NL], r[NR];
  };
  static __device__ __forceinline__ void read(Half &h, const char *lds, int s, const LeftReader &left, const RightReader &right) {
#pragma unroll
    for (int r = 0; r < NR; ++r) h.r[r] = right.read(lds + BL * kStep, r, s);
#pragma unroll
    for (int l = 0; l < NL; ++l) h.l[l] = left.read(lds + (l / NLL) * BLL * kStep, l % NLL, s);
  }
  static __device__ __forceinline__ void products(f32x4 (&acc)[NL][NR], const Half &h) {
#pragma unroll
    for (int l = 0; l < NL; ++l)
#pragma unroll
      for (int r = 0; r < NR; ++r) multiply(acc[l][r], h.l[l], h.r[r]);
  }

  // What this wavefront has asked for of LDS, or sent to it, has come, and all others are as far. (The
  // compiler's own barrier may not wait for loads to LDS.)
  static __device__ __forceinline__ void everybody_has_read() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
  static __device__ __forceinline__ void everything_has_come() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }

  // One step of a workgroup that has its CU to itself: the step after comes into a tile of its own
  // meanwhile (they do not overlap). Its loads go out between products: one after the other, they
  // would keep every wavefront from multiplying until the last is taken.
  template <class Load>
  static __device__ __forceinline__ void step(f32x4 (&acc)[NL][NR], char *__restrict next, const char *__restrict now,
                                              const Load &load, LeftReader &left, RightReader &right) {
    constexpr int kReads = NL * Left::kReads + NR * Right::kReads, kLoads = (HALVES ? 2 : 1) * Left::N + Right::N;
    constexpr int kHalf = NL * NR * kProducts<T>;
    if (LTR) left.again();
    if (RTR) right.again();
    Half h;
    read(h, now, 0, left, right);
    load(next);
    products(acc, h);
    read(h, now, 1, left, right);
    products(acc, h);
    __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, kHalf / kLoads, 0);
      __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, kReads, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, kHalf, 0);
    everything_has_come();
  }

  // acc[l][r] += the products of `steps` steps, each brought into a tile by load(lds). Where several
  // workgroups share a CU the others multiply while one waits, and one tile is enough: the step
  // after is sent for as soon as everybody has read it.
  template <class Load>
  static __device__ __forceinline__ void run(f32x4 (&acc)[NL][NR], int steps, const Load &load, int wave, int lane) {
    LeftReader left;
    RightReader right;
    left.init(wave % WL * NLL, lane);
    right.init(wave / WL * NR, lane);
    if constexpr (GROUPS == 1) {
      __shared__ __attribute__((aligned(1024))) char one[kBytes], two[kBytes];
      load(one);
      everything_has_come();
      for (int k = 0; k < steps; k += 2) {
        step(acc, two, one, load, left, right);
        if (k + 1 >= steps) break;
        step(acc, one, two, load, left, right);
      }
    } else {
      __shared__ __attribute__((aligned(1024))) char lds[kBytes];
      load(lds);
      for (int k = 0; k < steps; ++k) {
        everything_has_come();
        if (LTR) left.again();
        if (RTR) right.again();
        Half h;
        read(h, lds, 0, left, right);
        products(acc, h);
        read(h, lds, 1, left, right);
        everybody_has_read();
        load(lds);
        __builtin_amdgcn_sched_barrier(0);
        products(acc, h);
      }
      everything_has_come();  // (the tile may be used again)
    }
  }
};

// Tile `n` of nl x nr, spread so that an XCD (workgroups are given to the eight in turn) works on
// neighbouring tiles, kBand right tiles by all left ones: what they share stays in its L2. (Of a product in slices
// these are the tiles of one slice, all of which read the same part of the contraction. Where a slice has few tiles
// they are on different XCDs, and each of those reads that part: the weights' gradients of 81,920 rows of 256 to
// 1,024, 8 tiles a slice, read 671 MB where 378 would do.) Bands of 2, 4, 8 and
// 12, us: a training pass of 16,384 rows of 4,096 to 8,192 5,940, 5,990, 6,100 and 6,650, of 8,192 of 8,192 5,980,
// 6,020, 6,360, of 16,384 of 2,048 to 4,096 1,730, 1,670, 1,660.
constexpr int kXcds = 8, kBand = 4;
__device__ __forceinline__ void tile_of(uint32_t n, uint32_t nl, uint32_t nr, int *l, int *r) {
  const uint32_t total = nl * nr, each = total / kXcds, rest = total % kXcds;
  const uint32_t xcd = n % kXcds;
  n = xcd * each + min(xcd, rest) + n / kXcds;
  const uint32_t band = n / (kBand * nl), in = n - band * (kBand * nl);
  const uint32_t high = min((uint32_t)kBand, nr - band * kBand);
  *l = (int)(in / high);
  *r = (int)(band * kBand + in % high);
}

// ------------------------------------------------------------------------ activations

// act(a) and its derivative
template <class T>
__device__ __forceinline__ float act(float a, int kind) {
  if (kind == ASTRA_SEQ_SILU) return a * sigmoid<T>(a);
  return a * 0.5f * erfcf(a * -0.70710678f);
}
template <class T>
__device__ __forceinline__ void act_slope(float a, int kind, float *value, float *slope) {
  if (kind == ASTRA_SEQ_SILU) {
    const float s = sigmoid<T>(a);
    *value = a * s;
    *slope = s * (1.f + a * (1.f - s));
  } else {
    const float phi = 0.5f * erfcf(a * -0.70710678f);
    *value = a * phi;
    *slope = phi + a * (0.39894228f * __builtin_amdgcn_exp2f(-0.5f * kLog2e * a * a));
  }
}

// ---------------------------------------------------------------- results and their rows

// N neighbouring elements from any address, n of them inside.
template <class T, int N>
struct Loose {
  typedef T Raw __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  static __device__ __forceinline__ void load(const T *p, float (&v)[N], int n) {
    if (n >= N) {
      const Raw r = *reinterpret_cast<const Raw *>(p);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = (float)r[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < n ? (float)p[i] : 0.f;
    }
  }
  static __device__ __forceinline__ void store(T *p, const float (&v)[N], int n) {
    if (n >= N) {
      Raw r;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = (T)v[i];
      *reinterpret_cast<Raw *>(p) = r;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < n) p[i] = (T)v[i];
    }
  }
};

struct GatedArgs {
  Operand x, gate, up;       // as left or right operands of the first products
  const void *dh;            // [M, F]
  void *h;                   // [M, F]
  float *ab;                 // [2, M, F] (may be NULL): a and b, for the gradients
  void *dab;                 // [M, 2 Fp]: da, db, zero from F to Fp
  void *rest;                // [M, 2 Fp] (may be NULL): what they lose when they are rounded to bf16
  int64_t M, F, Fp;
  int32_t kind;
  float *part;  // [slices, 2, M, F] or NULL: partial sums of a and b instead of results
  int32_t slices, tiles_l, tiles_r, steps;  // steps: of a slice
};

// da and db of 8 elements, n of them inside (zero beyond).
template <class T>
__device__ __forceinline__ void slopes(const GatedArgs &g, const float (&a)[8], const float (&b)[8], const float (&dh)[8],
                                       float (&da)[8], float (&db)[8], int n) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float v, s;
    act_slope<T>(a[i], g.kind, &v, &s);
    da[i] = i < n ? dh[i] * b[i] * s : 0.f;
    db[i] = i < n ? dh[i] * v : 0.f;
  }
}

// da and db of 8 elements of a row, n of them inside, and with REST what they lose if it is wanted.
template <class T, bool REST>
__device__ __forceinline__ void store_slopes(const GatedArgs &g, int64_t at, float (&da)[8], float (&db)[8], int n) {
  T *p = (T *)g.dab + at;
  Loose<T, 8>::store(p, da, n);
  Loose<T, 8>::store(p + g.Fp, db, n);
  if constexpr (REST && sizeof(T) == 2) {
    if (!g.rest) return;
    const auto lost = [](float v) __attribute__((always_inline)) {
      const float kept = (float)(bf16)v;
      return fabsf(kept) < INFINITY ? v - kept : 0.f;  // (an infinity is whole, and so is a NaN)
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) da[i] = lost(da[i]), db[i] = lost(db[i]);
    p = (T *)g.rest + at;
    Loose<T, 8>::store(p, da, n);
    Loose<T, 8>::store(p + g.Fp, db, n);
  }
}

template <class P>
struct LoadHalves {
  typename P::Left &first, &second;
  typename P::Right &right;
  int wave;
  __device__ __forceinline__ void operator()(char *lds) const {
    first.load(lds, wave);
    second.load(lds + P::BLL * kStep, wave);
    right.load(lds + P::BL * kStep, wave);
  }
};

// h (and a, b), or with GRAD da and db from dh: the left tile is half gate, half up, so that a lane
// has a and b of the same elements.
template <class P, bool GRAD>
__global__ __launch_bounds__(P::kThreads, P::GROUPS * P::NW / 4) void gated_kernel(GatedArgs g) {
  typedef typename P::type T;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t tiles = (uint32_t)g.tiles_l * g.tiles_r, slice = blockIdx.x / tiles;
  int tl, tr;
  tile_of(blockIdx.x - slice * tiles, g.tiles_l, g.tiles_r, &tl, &tr);
  const int64_t m0 = (int64_t)tr * P::BR, f0 = (int64_t)tl * P::BLL;
  if (g.slices > 1) {
    const int64_t len = (int64_t)g.steps * kStepOf<T>, k0 = slice * len;
    P::Left::cut(g.gate, k0, len);
    P::Left::cut(g.up, k0, len);
    P::Right::cut(g.x, k0, len);
  }
  typename P::Left gate, up;
  typename P::Right x;
  gate.init(g.gate, f0, wave, lane);
  up.init(g.up, f0, wave, lane);
  x.init(g.x, m0, wave, lane);
  f32x4 acc[P::NL][P::NR] = {};
  P::run(acc, (int)((g.x.len + kStepOf<T> - 1) / kStepOf<T>), LoadHalves<P>{gate, up, x, wave}, wave, lane);
  // results from here on are rows and columns of the tile (less than 2^31 bytes of memory)
  const int rows = (int)min((int64_t)P::BR, g.M - m0), cols = (int)min((int64_t)P::BLL, g.F - f0);
  const int wl = wave % P::WL, wr = wave / P::WL, F = (int)g.F, Fp = (int)g.Fp, zeros = (int)min((int64_t)P::BLL, g.Fp - f0);
  const int64_t start = m0 * g.F + f0;
  // dh: all on its way before the first is waited for (223 to 208 us at 81,920 rows of 256 to 1,024 wide;
  // floats have no registers for it)
  constexpr bool kAhead = GRAD && sizeof(T) == 2;
  typename Loose<T, 8>::Raw dhs[kAhead ? P::NR : 1][kAhead ? P::NLL / 2 : 1];
  if constexpr (kAhead) {
#pragma unroll
    for (int r = 0; r < P::NR; ++r)
#pragma unroll
      for (int l = 0; l < P::NLL; l += 2) {
        const int m = (wr * P::NR + r) * 16 + lane % 16, f = (wl * P::NLL + l) * 16 + 8 * (lane / 16);
        if (!g.part && m < rows && f + 8 <= cols)
          dhs[r][l / 2] = *reinterpret_cast<const typename Loose<T, 8>::Raw *>((const T *)g.dh + start + (m * F + f));
      }
  }
#pragma unroll
  for (int r = 0; r < P::NR; ++r) {
    const int m = (wr * P::NR + r) * 16 + lane % 16;
    if (m >= rows) continue;
#pragma unroll
    for (int l = 0; l < P::NLL; l += 2) {
      const int f = (wl * P::NLL + l) * 16 + 8 * (lane / 16), n = cols - f;
      float a[8], b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        a[i] = acc[l + i / 4][r][i % 4];
        b[i] = acc[P::NLL + l + i / 4][r][i % 4];
      }
      const int at = m * F + f;
      if (g.part) {
        if (n <= 0) continue;
        float *part = g.part + (int64_t)slice * 2 * g.M * g.F + start + at;
        Loose<float, 8>::store(part, a, n);
        Loose<float, 8>::store(part + g.M * g.F, b, n);
        continue;
      }
      if constexpr (GRAD) {
        if (f >= zeros) continue;
        float dh[8], da[8], db[8];
        if (kAhead && n >= 8) {
#pragma unroll
          for (int i = 0; i < 8; ++i) dh[i] = (float)dhs[kAhead ? r : 0][kAhead ? l / 2 : 0][i];
        } else {
          Loose<T, 8>::load((const T *)g.dh + start + at, dh, n);
        }
        slopes<T>(g, a, b, dh, da, db, n);
        store_slopes<T, true>(g, m0 * 2 * g.Fp + f0 + (m * 2 * Fp + f), da, db, zeros - f);
      } else {
        if (n <= 0) continue;
        float h[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) h[i] = act<T>(a[i], g.kind) * b[i];
        Loose<T, 8>::store((T *)g.h + start + at, h, n);
        if (g.ab) {
          Loose<float, 8>::store(g.ab + start + at, a, n);
          Loose<float, 8>::store(g.ab + g.M * g.F + start + at, b, n);
        }
      }
    }
  }
}

// The results from a and b that are in memory: sums of slices, or what the forward call kept for the
// gradient (one slice). 2^shift threads a row; a launch has room for some of very many rows.
// (REST has registers of its own: with them the other bf16 gradients would have 7 wavefronts a SIMD and not 8.)
template <class T, bool GRAD, bool REST>
__device__ __forceinline__ void gated_join_row(const GatedArgs &g, const float *ab, int shift, int64_t m) {
  const int64_t size = g.M * g.F, row = m * g.F;
  const int F = (int)g.F, Fp = (int)g.Fp;
  for (int f = (threadIdx.x & ((1 << shift) - 1)) * 8; f < (GRAD ? Fp : F); f += 8 << shift) {
    float a[8], b[8];
    Loose<float, 8>::load(ab + row + f, a, F - f);
    Loose<float, 8>::load(ab + size + row + f, b, F - f);
    for (int k = 1; k < g.slices; ++k) {
      float x[8], y[8];
      Loose<float, 8>::load(ab + 2 * k * size + row + f, x, F - f);
      Loose<float, 8>::load(ab + (2 * k + 1) * size + row + f, y, F - f);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] += x[i], b[i] += y[i];
    }
    if constexpr (GRAD) {
      float dh[8], da[8], db[8];
      Loose<T, 8>::load((const T *)g.dh + row + f, dh, F - f);
      slopes<T>(g, a, b, dh, da, db, F - f);
      store_slopes<T, REST>(g, m * 2 * g.Fp + f, da, db, Fp - f);
    } else {
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] = act<T>(a[i], g.kind) * b[i];
      Loose<T, 8>::store((T *)g.h + row + f, h, F - f);
      if (g.ab) {
        Loose<float, 8>::store(g.ab + row + f, a, F - f);
        Loose<float, 8>::store(g.ab + size + row + f, b, F - f);
      }
    }
  }
}
template <class T, bool GRAD, bool REST>
__global__ __launch_bounds__(256) void gated_join_kernel(GatedArgs g, const float *ab, int shift) {
  const int each = 256 >> shift;
  for (int64_t m = (int64_t)blockIdx.x * each + (threadIdx.x >> shift); m < g.M; m += (int64_t)gridDim.x * each)
    gated_join_row<T, GRAD, REST>(g, ab, shift, m);
}

// ------------------------------------------------------------------- gradients' products

struct ProductArgs {
  Operand left[4], right[4];  // summed over the pairs
  int32_t pairs;
  // results [r, l]: rows from `split` on are the second output's
  void *out[2];
  int64_t out_ld, nl, nr, split, rows;  // rows: of each output
  float *part;                          // [slices, nr, nl] or NULL: partial sums instead of results
  int32_t slices;
  int32_t tiles_l, tiles_r, steps;  // steps: of a slice
};

template <class P>
struct LoadBoth {
  typename P::Left &left;
  typename P::Right &right;
  int wave;
  __device__ __forceinline__ void operator()(char *lds) const {
    left.load(lds, wave);
    right.load(lds + P::BL * kStep, wave);
  }
};

template <class P>
__global__ __launch_bounds__(P::kThreads, P::GROUPS * P::NW / 4) void product_kernel(ProductArgs g) {
  typedef typename P::type T;
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t tiles = (uint32_t)g.tiles_l * g.tiles_r, slice = blockIdx.x / tiles;
  int tl, tr;
  tile_of(blockIdx.x - slice * tiles, g.tiles_l, g.tiles_r, &tl, &tr);
  f32x4 acc[P::NL][P::NR] = {};
  for (int pair = 0; pair < g.pairs; ++pair) {
    Operand lo = g.left[pair], ro = g.right[pair];
    if (g.slices > 1) {
      P::Left::cut(lo, (int64_t)slice * g.steps * kStepOf<T>, (int64_t)g.steps * kStepOf<T>);
      P::Right::cut(ro, (int64_t)slice * g.steps * kStepOf<T>, (int64_t)g.steps * kStepOf<T>);
    }
    const int steps = (int)((lo.len + kStepOf<T> - 1) / kStepOf<T>);
    typename P::Left left;
    typename P::Right right;
    left.init(lo, (int64_t)tl * P::BL, wave, lane);
    right.init(ro, (int64_t)tr * P::BR, wave, lane);
    P::run(acc, steps, LoadBoth<P>{left, right, wave}, wave, lane);
  }
  const int wl = wave % P::WL, wr = wave / P::WL;
#pragma unroll
  for (int r = 0; r < P::NR; ++r) {
    const int64_t row = (int64_t)tr * P::BR + (wr * P::NR + r) * 16 + lane % 16;
    if (row >= g.nr) continue;
    const bool second = row >= g.split;
    const int64_t at = second ? row - g.split : row;
    if (!g.part && at >= g.rows) continue;
#pragma unroll
    for (int l = 0; l < P::NL; ++l) {
      const int64_t col = (int64_t)tl * P::BL + (wl * P::NL + l) * 16 + 4 * (lane / 16);
      const int n = (int)min((int64_t)4, g.nl - col);
      if (n <= 0) continue;
      const float v[4] = {acc[l][r][0], acc[l][r][1], acc[l][r][2], acc[l][r][3]};
      if (g.part)
        Loose<float, 4>::store(g.part + ((int64_t)slice * g.nr + row) * g.nl + col, v, n);
      else
        Loose<T, 4>::store((T *)g.out[second] + at * g.out_ld + col, v, n);
    }
  }
}

// The results from the slices' partial sums, in order.
template <class T>
__global__ __launch_bounds__(256) void join_slices_kernel(ProductArgs g) {
  const int64_t per = cdiv(g.nl, 4), i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / per;
  if (row >= g.nr) return;
  const int64_t col = (i - row * per) * 4, total = g.nr * g.nl;
  const bool second = row >= g.split;
  const int64_t at = second ? row - g.split : row;
  if (at >= g.rows) return;
  const int n = (int)min((int64_t)4, g.nl - col);
  float s[4] = {};
  for (int k = 0; k < g.slices; ++k) {
    float v[4];
    Loose<float, 4>::load(g.part + k * total + row * g.nl + col, v, n);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] += v[j];
  }
  Loose<T, 4>::store((T *)g.out[second] + at * g.out_ld + col, s, n);
}

// ---------------------------------------------------------------------- aligned copies

// Operands [rows, width] with rows of `ld` elements, any alignment, as rows of `pitch` elements filled up
// with zeros. 2^shift threads a row.
struct AlignArgs {
  const void *in[3];
  void *out[3];
  int64_t rows[3], ld[3];
  int32_t width, pitch;
};
template <class T>
__global__ __launch_bounds__(256) void align_kernel(AlignArgs a, int shift) {
  constexpr int V = 16 / sizeof(T);
  const int which = blockIdx.y, each = 256 >> shift;
  const T *in = (const T *)a.in[which];
  T *out = (T *)a.out[which];
  for (int64_t row = (int64_t)blockIdx.x * each + (threadIdx.x >> shift); row < a.rows[which]; row += (int64_t)gridDim.x * each)
    for (int c = (threadIdx.x & ((1 << shift) - 1)) * V; c < a.pitch; c += V << shift) {
      float v[V];
      Loose<T, V>::load(in + row * a.ld[which] + c, v, a.width - c);
      Vec<T, V>::store(out + row * a.pitch + c, v);
    }
}

// [D, 2 Fp] from the weights [F, D]: row d is column d of gate, zeros up to Fp, and column d of up.
constexpr int kTurn = 64;
__global__ __launch_bounds__(256) void turn_kernel(Operand gate, Operand up, bf16 *out, int64_t D, int64_t F, int64_t Fp) {
  __shared__ bf16 tile[kTurn][kTurn + 4];
  const Operand &w = blockIdx.z ? up : gate;
  const int64_t f0 = (int64_t)blockIdx.x * kTurn, d0 = (int64_t)blockIdx.y * kTurn;
  const int i = threadIdx.x / 16, j = threadIdx.x % 16 * 4;
#pragma unroll
  for (int n = 0; n < kTurn; n += 16) {
    float v[4];
    const int64_t f = f0 + i + n;
    Loose<bf16, 4>::load((const bf16 *)w.p + f * w.ld + d0 + j, v, f < F ? (int)min((int64_t)4, D - d0 - j) : 0);
#pragma unroll
    for (int k = 0; k < 4; ++k) tile[i + n][j + k] = (bf16)v[k];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < kTurn; n += 16) {
    const int64_t d = d0 + i + n;
    float v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = (float)tile[j + k][i + n];
    if (d < D) Loose<bf16, 4>::store(out + d * 2 * Fp + blockIdx.z * Fp + f0 + j, v, (int)min((int64_t)4, Fp - f0 - j));
  }
}

// --------------------------------------------------------------------------- few rows

// One fragment straight from memory, from any address: 16 bytes from element `k` of the contraction on
// (zeros beyond).
template <class T>
__device__ __forceinline__ Frag<T> fragment(const T *row, int k, int len) {
  constexpr int V = 16 / sizeof(T);
  if (k + V <= len) return *reinterpret_cast<const typename Loose<T, V>::Raw *>(row + k);
  Frag<T> f = {};
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (k + i < len) f[i] = row[k + i];
  return f;
}

template <class T>
__device__ __forceinline__ void store4(T *p, const f32x4 &x, int n) {
  const float v[4] = {x[0], x[1], x[2], x[3]};
  Loose<T, 4>::store(p, v, n);
}

// Up to 16 MT rows of x: the weights are read once, each by the lanes that multiply with it, and
// nothing is staged. A workgroup has NT tiles of 16 columns of the result, its wavefronts share the
// contraction; what the next step needs is on its way while the last is multiplied.
template <class T, int MT, int NT>
__global__ __launch_bounds__(256) void gated_few_kernel(GatedArgs g) {
  constexpr int V = 16 / sizeof(T), kStepE = kStepOf<T>, NW = 4;
  __shared__ f32x4 sums[NW][NT * 2 * MT][64];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int i = lane % 16, q = lane / 16, K = (int)g.x.len;
  const int64_t f0 = (int64_t)blockIdx.x * 16 * NT;
  const T *w[2 * NT], *x[MT];  // gate and up of each tile; rows
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t line = min(f0 + 16 * t + i, g.F - 1);
    w[2 * t] = (const T *)g.gate.p + line * g.gate.ld;
    w[2 * t + 1] = (const T *)g.up.p + line * g.up.ld;
  }
#pragma unroll
  for (int r = 0; r < MT; ++r) x[r] = (const T *)g.x.p + min((int64_t)(16 * r + i), g.M - 1) * g.x.ld;
  struct Step {
    Frag<T> w[2][2 * NT], x[2][MT];
  };
  const auto load = [&](Step &s, int k) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int at = k + h * (kStepE / 2);
#pragma unroll
      for (int t = 0; t < 2 * NT; ++t) s.w[h][t] = fragment<T>(w[t], at, K);
#pragma unroll
      for (int r = 0; r < MT; ++r) s.x[h][r] = fragment<T>(x[r], at, K);
    }
  };
  f32x4 acc[2 * NT][MT] = {};
  const auto multiply_all = [&](const Step &s) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
        for (int r = 0; r < MT; ++r) multiply(acc[t][r], s.w[h][t], s.x[h][r]);
  };
  Step one, two;
  int k = wave * kStepE + q * V;  // (beyond K there are zeros)
  load(one, k);
  for (int n = (K + NW * kStepE - 1) / (NW * kStepE); n > 0; n -= 2) {
    load(two, k + NW * kStepE);
    multiply_all(one);
    load(one, k + 2 * NW * kStepE);
    multiply_all(two);
    k += 2 * NW * kStepE;
  }
#pragma unroll
  for (int t = 0; t < 2 * NT; ++t)
#pragma unroll
    for (int r = 0; r < MT; ++r) sums[wave][t * MT + r][lane] = acc[t][r];
  __syncthreads();
  for (int n = wave; n < NT * MT; n += NW) {
    const int t = n / MT, r = n % MT;
    const int64_t m = 16 * r + i, f = f0 + 16 * t + 4 * q;
    const int left = (int)min((int64_t)4, g.F - f);
    if (m >= g.M || left <= 0) continue;
    f32x4 a = sums[0][2 * t * MT + r][lane], b = sums[0][(2 * t + 1) * MT + r][lane], h;
#pragma unroll
    for (int v = 1; v < NW; ++v) {
      a += sums[v][2 * t * MT + r][lane];
      b += sums[v][(2 * t + 1) * MT + r][lane];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = act<T>(a[j], g.kind) * b[j];
    store4((T *)g.h + m * g.F + f, h, left);
    if (g.ab) {
      store4(g.ab + m * g.F + f, a, left);
      store4(g.ab + (g.M + m) * g.F + f, b, left);
    }
  }
}

// ----------------------------------------------------------------------------- launches

int check(const astra_gated_linear *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_ABI_CHECK(f->rows, >=, 0);
  ASTRA_ABI_CHECK(f->rows, <=, kMostRows);
  ASTRA_ABI_CHECK(f->width, >=, 1);
  ASTRA_ABI_CHECK(f->width, <=, ASTRA_SEQ_MAX_LINEAR_WIDTH);
  ASTRA_ABI_CHECK(f->hidden, >=, 1);
  ASTRA_ABI_CHECK(f->hidden, <=, ASTRA_SEQ_MAX_LINEAR_WIDTH);
  ASTRA_ABI_CHECK(f->x_stride, >=, 0);
  ASTRA_ABI_CHECK(f->gate_stride, >=, 0);
  ASTRA_ABI_CHECK(f->up_stride, >=, 0);
  const int32_t kind = f->activation & ~ASTRA_SEQ_EXACT_GRADIENTS;
  if (kind != ASTRA_SEQ_SILU && kind != ASTRA_SEQ_GELU)
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_gated_linear: the activation is ASTRA_SEQ_SILU or ASTRA_SEQ_GELU");
  return ASTRA_OK;
}

// Whether da and db enter their products as two bf16 numbers each, the second of which is what the first lost:
// 2^-17 of them at most is left out, and not 2^-8. Twice the products.
bool exact(const astra_gated_linear &f) { return f.type == ASTRA_SEQ_BF16 && (f.activation & ASTRA_SEQ_EXACT_GRADIENTS); }

int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }
int64_t per16(int32_t type) { return 16 / (int64_t)elem_size(type); }
// Rows in a workspace start on the caches' lines of 128 bytes.
int64_t pitch_of(int64_t width, int32_t type) { return round_up(width, kStep / (int64_t)elem_size(type)); }
int64_t padded_hidden(const astra_gated_linear &f) { return pitch_of(f.hidden, f.type); }

// Whether the backward call gets a and b, 16 bytes an element written and read, or computes them
// again, 4 D operations (and always if the caller has no projections). Again / kept, us, a training pass of 8,192
// rows to four times the width: bf16 of 256 112 / 115, of 512 228 / 250, of 1,024 565 / 564, of 1,280 901 / 861, of
// 1,536 1,271 / 1,153, of 2,048 1,920 / 1,694; 1,000 rows of 1,024 124 / 118, of 1,280 207 / 187; float of 64
// 104 / 104, of 128 139 / 130, of 256 333 / 281.
bool keeps(const astra_gated_linear &f) { return f.width >= (f.type == ASTRA_SEQ_BF16 ? 1024 : 128); }

float *kept(const astra_gated_linear &f) { return keeps(f) ? f.projections : nullptr; }

// Rows that are read straight from memory rather than as tiles. Few rows' kernel / tiles, us: 64 bf16 rows of 256
// to 1,024 10.5 / 8.8, of 1,024 to 4,096 13.5 / 18.3, of 4,096 to 8,192 51 / 58, 17 of them 41 / 49; float 10 / 23,
// 22 / 32, 105 / 150, 77 / 146. Its registers hold 64 rows.
bool few(const astra_gated_linear &f) { return f.rows <= 64; }

// Whether bf16 rows that do not start on the caches' lines are copied to where they do: a step of such a row
// is in two lines. As they lie / copied, us: 20,000 rows of 4,088 to 2,048 948 / 632, with the gradients
// 2,182 / 1,972, of 1,000 to 2,731 293 / 257 and 1,188 / 1,097, to 1,100 126 / 114 and 524 / 496; 4,097 rows to
// 2,731 70 / 70 and 320 / 313; but 20,000 rows to 520 65 / 70 and 292 / 297, 2,048 to 2,731 41 / 41 and 185 / 186,
// 300 to 1,100 21 / 26. (Float products take longer than either.)
bool lined(const astra_gated_linear &f) {
  return f.type == ASTRA_SEQ_BF16 && f.rows >= 1024 && f.hidden >= 1024 && f.rows * f.hidden >= (int64_t(1) << 24);
}

// Whether an operand is read as it lies, or copied to a workspace first. (256 rows of a tile have to be
// within the 2 GB that one access can reach, and what lies behind the last row in no row before it: rows
// that overlap, or one for all, are copied.)
bool direct(const astra_gated_linear &f, const void *p, int64_t stride) {
  const int64_t v = per16(f.type);
  if (lined(f) && (!aligned(p, kStep) || stride * (int64_t)elem_size(f.type) % kStep)) return false;
  return aligned(p, 16) && stride % v == 0 && f.width % v == 0 && stride >= f.width && stride <= ASTRA_SEQ_MAX_LINEAR_WIDTH;
}
struct Operands {
  Operand x, gate, up;
};
// The operands, and what has to be copied first; the copies' bytes.
size_t operands_of(const astra_gated_linear &f, char *ws, Operands *o, AlignArgs *a) {
  const void *p[3] = {f.x, f.gate, f.up};
  const int64_t ld[3] = {f.x_stride, f.gate_stride, f.up_stride}, rows[3] = {f.rows, f.hidden, f.hidden};
  Operand *out[3] = {&o->x, &o->gate, &o->up};
  *a = {};
  a->width = f.width;
  a->pitch = (int32_t)pitch_of(f.width, f.type);
  size_t bytes = 0;
  for (int i = 0; i < 3; ++i) {
    *out[i] = {p[i], ld[i], rows[i], round_up(f.width, per16(f.type))};
    if (direct(f, p[i], ld[i])) continue;
    a->in[i] = p[i];
    a->ld[i] = ld[i];
    a->rows[i] = rows[i];
    a->out[i] = ws + bytes;
    out[i]->p = ws + bytes;
    out[i]->ld = a->pitch;
    bytes += (size_t)(rows[i] * a->pitch) * elem_size(f.type);
  }
  return bytes;
}
size_t copies_bytes(const astra_gated_linear &f) {
  Operands o;
  AlignArgs a;
  return operands_of(f, nullptr, &o, &a);
}

GatedArgs args_of(const astra_gated_linear &f) {
  GatedArgs g{};
  g.h = f.h;
  g.ab = kept(f);
  g.M = f.rows;
  g.F = f.hidden;
  g.Fp = padded_hidden(f);
  g.kind = f.activation & ~ASTRA_SEQ_EXACT_GRADIENTS;
  return g;
}

// Tiles of 128 x 192 results, three workgroups to a CU, or 128 x 128, four; or 256 x 256 with a CU to
// themselves. Along the contraction several workgroups a CU are faster (us: 16,384 rows of 4,096 to 8,192 1,680,
// 1,840, 1,740; 81,920 of 256 to 1,024 136, 123, 150). Across it (both operands of the weights' gradients), where
// every fragment is two transposing reads, bf16 tiles are better large: 256 x 256 alone 1,690 and 113 us, 256 x 128
// twice a CU 1,860 and 130, 128 x 128 four times 3,160 and 153; with floats 128 x 128 takes 209, 256 x 256 296.
template <class T, bool LTR, bool RTR, bool HALVES>
using Large = Product<T, LTR, RTR, 4, 6, HALVES, 3>;
template <class T, bool LTR, bool RTR, bool HALVES>
using Small = Product<T, LTR, RTR, 4, 4, HALVES, 4>;
using Alone = Product<bf16, true, true, 8, 4, false, 1, 2, 4>;

constexpr int64_t kCus = 256;
// Workgroups of 256 threads that go on to further rows where there are more than these have.
constexpr int64_t kMostLoopBlocks = int64_t(1) << 20;
template <class P>
int64_t tiles(int64_t nl, int64_t nr) {
  return cdiv(nl, P::BLL) * cdiv(nr, P::BR);
}
// The results that the CUs have room for until the last tile is done: in the first rounds they all
// wait for it, later their ends have spread.
template <class P>
int64_t room(int64_t nl, int64_t nr) {
  const int64_t n = tiles<P>(nl, nr), each = kCus * P::GROUPS;
  return (n < 3 * each ? round_up(n, each) : n) * P::BL * P::BR;
}
// Large tiles read less for each product, small ones overlap more of what is not products. Large / small, us, 8,192
// rows: of 256 to 4,096 59 / 58, of 512 to 4,096 82.8 / 82.1, of 1,024 134 / 137, of 2,048 248 / 255, of 4,096 to
// 8,192 946 / 984; 3,000 of 1,024 to 5,000 70 / 74.
template <class L, class S>
bool larger(int64_t nl, int64_t nr, int64_t len) {
  return len >= 1024 && 9 * room<L>(nl, nr) <= 10 * room<S>(nl, nr);
}

#define GATED_LAUNCH(kernel, blocks, threads, ...)                                                   \
  do {                                                                                               \
    const int64_t blocks_ = (blocks);                                                                \
    ASTRA_ABI_CHECK(blocks_ * (threads), <=, kMostThreads);                                          \
    hipLaunchKernelGGL((kernel), dim3((unsigned)blocks_), dim3(threads), 0, st, __VA_ARGS__);        \
    ASTRA_HIP_CHECK(rt_last_error(), #kernel " launch");                                             \
  } while (false)

// Slices of a contraction of `steps` steps for `n` tiles of which the CUs hold `room` at a time: more of
// them where there are less tiles than CUs, with 8 steps at least. (Training passes without and with
// slices, us: 183 float rows of 2,083 to 10,203 1,876 / 770, 237 of 224 to 6,808 943 / 130; one bf16 row of
// 536 to 7,336 240 / 101.)
int64_t slices_for(int64_t n, int64_t room, int64_t steps) {
  if (n < 1 || n >= kCus) return 1;
  const int64_t want = cdiv(room, n), most = steps / 8;
  return want < most ? want : most > 1 ? most : 1;
}

template <class T>
int operands(const astra_gated_linear &f, char **ws, Operands *o, hipStream_t st) {
  AlignArgs a;
  *ws += operands_of(f, *ws, o, &a);
  const int64_t rows = std::max(std::max(a.rows[0], a.rows[1]), a.rows[2]);
  if (!rows) return ASTRA_OK;
  int shift = 0;
  while (shift < 8 && ((int64_t)per16(f.type) << shift) < a.pitch) ++shift;
  const dim3 grid((unsigned)std::min(cdiv(rows, 256 >> shift), kMostLoopBlocks), 3);
  hipLaunchKernelGGL(align_kernel<T>, grid, dim3(256), 0, st, a, shift);
  ASTRA_HIP_CHECK(rt_last_error(), "align_kernel launch");
  return ASTRA_OK;
}

template <class T, bool GRAD>
int launch_join(GatedArgs g, const float *ab, hipStream_t st) {
  int shift = 4;
  while (shift < 8 && (int64_t(8) << shift) < g.F) ++shift;
  const int64_t blocks = std::min(cdiv(g.M, 256 >> shift), kMostLoopBlocks);
  if constexpr (GRAD && sizeof(T) == 2) {
    if (g.rest) {
      GATED_LAUNCH((gated_join_kernel<T, GRAD, true>), blocks, 256, g, ab, shift);
      return ASTRA_OK;
    }
  }
  GATED_LAUNCH((gated_join_kernel<T, GRAD, false>), blocks, 256, g, ab, shift);
  return ASTRA_OK;
}

template <class P, bool GRAD>
int launch_gated_tiles(GatedArgs g, hipStream_t st) {
  const int64_t F = GRAD ? g.Fp : g.F;
  const int64_t n = tiles<P>(F, g.M) * g.slices;
  ASTRA_ABI_CHECK(n * P::kThreads, <=, kMostThreads);
  g.tiles_l = (int32_t)cdiv(F, P::BLL);
  g.tiles_r = (int32_t)cdiv(g.M, P::BR);
  g.steps = (int32_t)cdiv(cdiv(g.x.len, kStepOf<typename P::type>), g.slices);
  if (g.slices == 1) g.part = nullptr;
  GATED_LAUNCH((gated_kernel<P, GRAD>), n, P::kThreads, g);
  return g.slices > 1 ? launch_join<typename P::type, GRAD>(g, g.part, st) : ASTRA_OK;
}
template <class T>
int64_t gated_slices(int64_t M, int64_t F, int64_t D) {
  typedef Small<T, false, false, true> S;
  return slices_for(tiles<S>(F, M), kCus * S::GROUPS, cdiv(D, kStepOf<T>));
}
// `part` has room for the slices
template <class T, bool GRAD>
int launch_gated(GatedArgs &g, void *part, hipStream_t st) {
  typedef Large<T, false, false, true> L;
  typedef Small<T, false, false, true> S;
  g.slices = (int32_t)gated_slices<T>(g.M, g.F, g.x.len);
  g.part = (float *)part;
  return g.slices == 1 && larger<L, S>(GRAD ? g.Fp : g.F, g.M, g.x.len) ? launch_gated_tiles<L, GRAD>(g, st)
                                                                       : launch_gated_tiles<S, GRAD>(g, st);
}
template <class T>
size_t gated_part_bytes(const astra_gated_linear &f) {
  const int64_t s = gated_slices<T>(f.rows, f.hidden, round_up(f.width, per16(f.type)));
  return s > 1 ? (size_t)(s * 2 * f.rows * f.hidden) * sizeof(float) : 0;
}

// More than 16 rows are read half as often by two tiles a workgroup, which is worth it where the weights
// are large enough to keep all CUs busy all the same. One / two, us, 64 rows: of 4,096 to 8,192 61 / 50, of 2,048 to
// 8,192 32 / 27, of 2,048 to 4,096 20 / 24, of 256 to 1,024 11 / 13. (16 rows of 4,096 to 8,192: 35 / 42.)
template <class T>
int launch_few(const GatedArgs &g, hipStream_t st) {
  const bool two = g.F >= 32 * kCus && g.x.len >= 2048;
  if (g.M <= 16)
    GATED_LAUNCH((gated_few_kernel<T, 1, 1>), cdiv(g.F, 16), 256, g);
  else if (g.M <= 32 && two)
    GATED_LAUNCH((gated_few_kernel<T, 2, 2>), cdiv(g.F, 32), 256, g);
  else if (g.M <= 32)
    GATED_LAUNCH((gated_few_kernel<T, 2, 1>), cdiv(g.F, 16), 256, g);
  else if (two)
    GATED_LAUNCH((gated_few_kernel<T, 4, 2>), cdiv(g.F, 32), 256, g);
  else
    GATED_LAUNCH((gated_few_kernel<T, 4, 1>), cdiv(g.F, 16), 256, g);
  return ASTRA_OK;
}

template <class T>
int forward(const astra_gated_linear &f, hipStream_t st) {
  GatedArgs g = args_of(f);
  if (few(f)) {
    g.x = {f.x, f.x_stride, f.rows, f.width};
    g.gate = {f.gate, f.gate_stride, f.hidden, f.width};
    g.up = {f.up, f.up_stride, f.hidden, f.width};
    return launch_few<T>(g, st);
  }
  const size_t need = copies_bytes(f) + gated_part_bytes<T>(f);
  if (need) ASTRA_SEQ_POINTER(f.workspace);
  ASTRA_ABI_CHECK(f.workspace_bytes, >=, need);
  if (need && !aligned(f.workspace, 16)) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_gated_linear_forward: the workspace starts on 16 bytes");
  char *ws = (char *)f.workspace;
  Operands o;
  if (int rc = operands<T>(f, &ws, &o, st)) return rc;
  g.x = o.x;
  g.gate = o.gate;
  g.up = o.up;
  return launch_gated<T, false>(g, ws, st);
}

template <class P>
int launch_product(ProductArgs &g, void *part, hipStream_t st) {
  typedef typename P::type T;
  const int64_t n = tiles<P>(g.nl, g.nr) * g.slices;
  ASTRA_ABI_CHECK(n * P::kThreads, <=, kMostThreads);
  g.tiles_l = (int32_t)cdiv(g.nl, P::BL);
  g.tiles_r = (int32_t)cdiv(g.nr, P::BR);
  g.steps = (int32_t)cdiv(cdiv(g.left[0].len, kStepOf<T>), g.slices);
  g.part = g.slices > 1 ? (float *)part : nullptr;
  GATED_LAUNCH(product_kernel<P>, n, P::kThreads, g);
  if (g.part) GATED_LAUNCH(join_slices_kernel<T>, cdiv(g.nr * cdiv(g.nl, 4), 256), 256, g);
  return ASTRA_OK;
}

// The weights' gradients are sums over the rows, which are cut into slices: enough workgroups for all
// CUs, and 8 steps at least to a slice.
struct Slices {
  bool alone;
  int64_t n;
};
template <class T>
Slices slices_of(const astra_gated_linear &f) {
  const int64_t D = f.width, F2 = 2 * padded_hidden(f);
  typedef Small<T, true, true, false> S;
  // of bf16, tiles of 128 x 128 take 1.4 to 1.9 times as long for as many results, floats less (as above)
  const bool alone = f.type == ASTRA_SEQ_BF16 && 10 * tiles<Alone>(D, F2) * Alone::BL * Alone::BR <= 14 * tiles<S>(D, F2) * S::BL * S::BR;
  const int64_t want = alone ? cdiv(kCus, tiles<Alone>(D, F2)) : cdiv(kCus * S::GROUPS, tiles<S>(D, F2));
  const int64_t most = cdiv(f.rows, kStepOf<T>) / 8;
  return {alone, want < most ? want : most > 1 ? most : 1};
}
// With many rows, wide bf16 weights are turned for the inputs' gradient: lines along the contraction are
// read from memory in fewer, longer pieces. Whole passes without and with it, us: 16,384 rows of 4,096
// to 8,192 wide 5,296 / 4,429, 8,192 of 8,192 to 8,192 5,552 / 4,276, 8,192 of 2,048 to 8,192
// 1,317 / 1,306, 8,192 of 1,024 to 4,096 447 / 441; but 4,096 of 2,048 to 8,192 739 / 770, 16,384 of
// 256 to 1,024 101 / 106, and float 16,384 of 4,096 to 4,096 15,580 / 16,010.
bool turned(const astra_gated_linear &f) { return f.type == ASTRA_SEQ_BF16 && f.rows >= 8192 && f.width >= 1024; }
size_t turned_bytes(const astra_gated_linear &f) {
  return turned(f) ? (size_t)round_up(f.width * 2 * padded_hidden(f), 16) * sizeof(bf16) : 0;
}

// Slices of each half of the inputs' gradient's contraction. (Turned, there are tiles enough.)
template <class T>
int64_t dx_slices(const astra_gated_linear &f) {
  typedef Small<T, true, false, false> S;
  return slices_for(tiles<S>(f.width, f.rows), kCus * S::GROUPS, cdiv(padded_hidden(f), kStepOf<T>));
}
// What the slices of one product after the other need.
template <class T>
size_t part_bytes(const astra_gated_linear &f) {
  const int64_t w = slices_of<T>(f).n, x = dx_slices<T>(f);
  const size_t of_w = w > 1 ? (size_t)(w * 2 * padded_hidden(f) * f.width) * sizeof(float) : 0;
  const size_t of_x = x > 1 ? (size_t)(x * f.rows * f.width) * sizeof(float) : 0;
  const size_t of_h = kept(f) ? 0 : gated_part_bytes<T>(f);
  return std::max(std::max(of_w, of_x), of_h);
}

template <class T>
size_t dab_bytes(const astra_gated_linear &f) {
  return (size_t)(f.rows * 2 * padded_hidden(f)) * sizeof(T);
}
template <class T>
size_t grad_bytes(const astra_gated_linear &f) {
  return (exact(f) ? 2 : 1) * dab_bytes<T>(f) + copies_bytes(f) + turned_bytes(f) + part_bytes<T>(f);
}

template <class T>
int backward(const astra_gated_linear_grad &b, hipStream_t st) {
  const astra_gated_linear &f = b.f;
  GatedArgs g = args_of(f);
  const size_t need = grad_bytes<T>(f);
  if (need) ASTRA_SEQ_POINTER(b.workspace);
  ASTRA_ABI_CHECK(b.workspace_bytes, >=, need);
  if (need && !aligned(b.workspace, 16)) return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_gated_linear_backward: the workspace starts on 16 bytes");
  char *ws = (char *)b.workspace;
  const int64_t Fp = g.Fp, Dp = round_up(f.width, per16(f.type));
  g.dab = ws;
  g.dh = b.dh;
  ws += dab_bytes<T>(f);
  if (exact(f)) {
    g.rest = ws;
    ws += dab_bytes<T>(f);
  }
  const T *const parts[2] = {(const T *)g.dab, (const T *)g.rest};  // of da and db
  const int each = exact(f) ? 2 : 1;
  Operands o;
  if (int rc = operands<T>(f, &ws, &o, st)) return rc;
  g.x = o.x;
  g.gate = o.gate;
  g.up = o.up;
  char *const turn = ws, *const part = ws + turned_bytes(f);
  if (f.rows) {
    g.slices = 1;
    if (int rc = kept(f) ? launch_join<T, true>(g, kept(f), st) : launch_gated<T, true>(g, part, st)) return rc;
  }
  if (b.dx && f.rows) {  // da Wg + db Wu
    ProductArgs p{};
    p.out[0] = b.dx;
    p.out_ld = p.nl = f.width;
    p.nr = p.split = p.rows = f.rows;
    p.slices = (int32_t)dx_slices<T>(f);
    if (turned(f)) {
      if constexpr (sizeof(T) == 2) {
        const dim3 grid((unsigned)cdiv(Fp, kTurn), (unsigned)cdiv(f.width, kTurn), 2);
        hipLaunchKernelGGL(turn_kernel, grid, dim3(256), 0, st, o.gate, o.up, (T *)turn, (int64_t)f.width, (int64_t)f.hidden, Fp);
        ASTRA_HIP_CHECK(rt_last_error(), "turn_kernel launch");
        p.pairs = each;
        for (int i = 0; i < each; ++i) {
          p.left[i] = {turn, 2 * Fp, f.width, 2 * Fp};
          p.right[i] = {parts[i], 2 * Fp, f.rows, 2 * Fp};
        }
        typedef Large<T, false, false, false> L;
        typedef Small<T, false, false, false> S;
        if (int rc = larger<L, S>(p.nl, p.nr, 2 * Fp) ? launch_product<L>(p, part, st) : launch_product<S>(p, part, st)) return rc;
      }
    } else {
      p.pairs = 2 * each;
      for (int i = 0; i < p.pairs; ++i) {
        const Operand &w = i % 2 ? o.up : o.gate;
        p.left[i] = {w.p, w.ld, Dp, f.hidden};  // lines: columns of the weight
        p.right[i] = {parts[i / 2] + i % 2 * Fp, 2 * Fp, f.rows, Fp};
      }
      if (int rc = launch_product<Small<T, true, false, false>>(p, part, st)) return rc;
    }
  }
  if (b.dgate || b.dup) {
    const Slices s = slices_of<T>(f);
    ProductArgs p{};
    p.pairs = each;
    // (one weight's gradient alone is the product with its half of the columns)
    p.nr = b.dgate && b.dup ? 2 * Fp : Fp;
    for (int i = 0; i < each; ++i) {
      p.left[i] = {o.x.p, o.x.ld, Dp, f.rows};
      p.right[i] = {parts[i] + (b.dgate ? 0 : Fp), 2 * Fp, p.nr, f.rows};
    }
    p.out[0] = b.dgate ? b.dgate : b.dup;
    p.out[1] = b.dup;
    p.out_ld = p.nl = f.width;
    p.split = Fp;
    p.rows = f.hidden;
    p.slices = (int32_t)s.n;
    int rc = ASTRA_OK;
    if constexpr (sizeof(T) == 2) {
      rc = s.alone ? launch_product<Alone>(p, part, st) : launch_product<Small<T, true, true, false>>(p, part, st);
    } else {
      rc = launch_product<Small<T, true, true, false>>(p, part, st);
    }
    if (rc) return rc;
  }
  return ASTRA_OK;
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_gated_linear_workspace_size(const astra_gated_linear *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  *bytes = few(*f) ? 0 : copies_bytes(*f) + (f->type == ASTRA_SEQ_F32 ? gated_part_bytes<float>(*f) : gated_part_bytes<bf16>(*f));
  return ASTRA_OK;
}

int astra_gated_linear_projections(const astra_gated_linear *f, size_t *floats) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(floats);
  *floats = keeps(*f) ? (size_t)2 * f->rows * f->hidden : 0;
  return ASTRA_OK;
}

int astra_gated_linear_forward(const astra_gated_linear *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->rows == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(f->x);
  ASTRA_SEQ_POINTER(f->gate);
  ASTRA_SEQ_POINTER(f->up);
  ASTRA_SEQ_POINTER(f->h);
  return f->type == ASTRA_SEQ_F32 ? forward<float>(*f, as_stream(stream)) : forward<bf16>(*f, as_stream(stream));
}

int astra_gated_linear_grad_workspace_size(const astra_gated_linear *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  *bytes = f->type == ASTRA_SEQ_F32 ? grad_bytes<float>(*f) : grad_bytes<bf16>(*f);
  return ASTRA_OK;
}

int astra_gated_linear_backward(const astra_gated_linear_grad *g, void *stream) {
  ASTRA_SEQ_POINTER(g);
  if (int rc = check(&g->f)) return rc;
  if (g->f.rows) {
    ASTRA_SEQ_POINTER(g->f.x);
    ASTRA_SEQ_POINTER(g->dh);
  }
  ASTRA_SEQ_POINTER(g->f.gate);
  ASTRA_SEQ_POINTER(g->f.up);
  return g->f.type == ASTRA_SEQ_F32 ? backward<float>(*g, as_stream(stream)) : backward<bf16>(*g, as_stream(stream));
}

}  // extern "C"
