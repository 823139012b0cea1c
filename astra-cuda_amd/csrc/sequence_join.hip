// sequence_join.hip -- what stands between two blocks of a policy, as one pass: the norm
// after a block, its gate and residual scale, the residual sum, and the norm before the
// next block.
//
//   i1 = rsqrt(mean(u^2) + eps)         u the block's output, sg = sigmoid(gate)
//   r' = r + sg * scale * post * u * i1
//   i2 = rsqrt(mean(r'^2) + eps),  n = r' * i2 * next
//
// Some 12 operations an element (45 in the gradient): bound by memory traffic, so a row is
// read once into registers, both sums are taken there, and each thread keeps the weights
// of its columns over all the rows that it works on. Times: 81,920 rows of 256 in bf16
// forwards 52 us (4.1 TB/s), backwards 86 (3.9); 16,384 rows of 4,096 with a residual in
// 32 bits 172 (4.7, a large copy's rate) and 277 (4.4).
// That holds up to two vectors a thread. With four of 8 bf16 columns (widths 1,025 to 2,048 and
// 4,097 to 8,192) a thread needs 207 registers forwards and 256 with 70 to 120 more in the
// accumulation file backwards, one or two wavefronts a SIMD: 2.5 and 1.8 to 2.0 TB/s with a gate
// of full width; backwards beyond 8,192 columns 118 to 170 registers spill: 1.8 (bf16) to 3.3.
#include "sequence.h"

#define ASTRA_SRC_NAME "sequence_join.hip"

namespace astra_seq {
namespace {

struct JoinArgs {
  const void *r, *u, *gate, *dr1, *dn;
  const float *post, *next, *scale;
  void *r1, *n, *dr, *du, *dgate;
  float *rstd, *part;
  int64_t rows, rs, us, gs;
  int32_t D, gate_row, scale_one;
  float eps, inv_d;
};

// A row is TPR threads (256 / TPR rows to a workgroup, or one of 1024 threads), each with
// NV vectors of V columns: column (j * TPR + t) * V + i.
template <int TPR>
constexpr int block_of = TPR > 256 ? TPR : 256;

template <class T, int V, int NV, int TPR>
__device__ __forceinline__ void load_row(const T *p, int t, int D, float (&v)[NV][V]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * V;
    if (c < D)
      Vec<T, V>::load(p + c, v[j]);
    else
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = 0.f;
  }
}

template <class T, int V, int NV, int TPR>
__device__ __forceinline__ void store_row(T *p, int t, int D, const float (&v)[NV][V]) {
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * TPR + t) * V;
    if (c < D) Vec<T, V>::store(p + c, v[j]);
  }
}

// post * scale of this thread's columns (zero beyond the row).
template <int V, int NV, int TPR>
__device__ __forceinline__ void load_weights(const JoinArgs &a, int t, float (&cw)[NV][V], float (&nw)[NV][V]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = (j * TPR + t) * V + i;
      cw[j][i] = 0.f;
      nw[j][i] = 0.f;
      if (c < a.D) {
        if (a.u) cw[j][i] = a.post[c] * (a.scale ? a.scale[a.scale_one ? 0 : c] : 1.f);
        if (a.next) nw[j][i] = a.next[c];
      }
    }
}

template <class TR, class T, int V, int NV, int TPR>
__global__ __launch_bounds__(block_of<TPR>) void join_forward_kernel(JoinArgs a) {
  constexpr int RPB = block_of<TPR> / TPR;
  __shared__ float lds[2][TPR > kWave ? TPR / kWave : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float cw[NV][V], nw[NV][V];
  load_weights<V, NV, TPR>(a, t, cw, nw);
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    float r[NV][V];
    load_row<TR, V, NV, TPR>((const TR *)a.r + row * a.rs, t, a.D, r);
    if (a.u) {
      float u[NV][V];
      load_row<T, V, NV, TPR>((const T *)a.u + row * a.us, t, a.D, u);
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) s += u[j][i] * u[j][i];
      const float i1 = rsqrtf(row_sum<TPR>(s, lds[0]) * a.inv_d + a.eps);
      if (a.rstd && t == 0) a.rstd[row * 2] = i1;
      if (!a.gate) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] += cw[j][i] * (u[j][i] * i1);
      } else if (a.gate_row) {
        const float sg = sigmoid<TR>((float)((const T *)a.gate)[row * a.gs]);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] += sg * cw[j][i] * (u[j][i] * i1);
      } else {
        float g[NV][V];
        load_row<T, V, NV, TPR>((const T *)a.gate + row * a.gs, t, a.D, g);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i) r[j][i] += sigmoid<TR>(g[j][i]) * cw[j][i] * (u[j][i] * i1);
      }
      store_row<TR, V, NV, TPR>((TR *)a.r1 + row * a.D, t, a.D, r);
    }
    if (a.next) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) s += (j * TPR + t) * V + i < a.D ? r[j][i] * r[j][i] : 0.f;
      const float i2 = rsqrtf(row_sum<TPR>(s, lds[1]) * a.inv_d + a.eps);
      if (a.rstd && t == 0) a.rstd[row * 2 + 1] = i2;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) r[j][i] = r[j][i] * i2 * nw[j][i];
      store_row<T, V, NV, TPR>((T *)a.n + row * a.D, t, a.D, r);
    }
    if constexpr (TPR > kWave) __syncthreads();  // before the next row's sums
  }
}

// With z = dn next, hat = u i1 and c = post scale:
//   dr  = dr' + i2 z - r' i2^3 mean(z r')
//   dsg = dr c hat,  dhat = dr sg c,  du = i1 dhat - u i1^3 mean(dhat u)
//   q   = sum over rows of dr sg hat: dpost = q scale, dscale = q post;  dnext = sum dn r' i2
// With a single column the two terms of a norm's gradient cancel but for eps i^3.
// A thread keeps q and dnext of its columns over its rows; a workgroup's are row blockIdx.x
// of part [gridDim.x, 2, D].
template <class TR, class T, int V, int NV, int TPR>
__global__ __launch_bounds__(block_of<TPR>) void join_backward_kernel(JoinArgs a) {
  constexpr int RPB = block_of<TPR> / TPR;
  __shared__ float lds[3][TPR > kWave ? TPR / kWave : 1];
  const int t = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float cw[NV][V], nw[NV][V], q[NV][V], dnw[NV][V];
  load_weights<V, NV, TPR>(a, t, cw, nw);
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) q[j][i] = dnw[j][i] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * RPB + sub; row < a.rows; row += (int64_t)gridDim.x * RPB) {
    float r[NV][V], u[NV][V], g[NV][V], dr[NV][V];
    load_row<TR, V, NV, TPR>((const TR *)a.r + row * a.rs, t, a.D, r);
    float i1 = 0.f;
    if (a.u) {
      load_row<T, V, NV, TPR>((const T *)a.u + row * a.us, t, a.D, u);
      i1 = a.rstd[row * 2];
    }
    if (a.gate && !a.gate_row) {
      load_row<T, V, NV, TPR>((const T *)a.gate + row * a.gs, t, a.D, g);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) g[j][i] = sigmoid<TR>(g[j][i]);
    } else {
      const float sg = a.gate ? sigmoid<TR>((float)((const T *)a.gate)[row * a.gs]) : 1.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) g[j][i] = sg;
    }
    if (a.dr1) {
      load_row<TR, V, NV, TPR>((const TR *)a.dr1 + row * a.D, t, a.D, dr);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) dr[j][i] = 0.f;
    }
    if (a.dn) {
      float z[NV][V], s = 0.f;
      load_row<T, V, NV, TPR>((const T *)a.dn + row * a.D, t, a.D, z);
      const float i2 = a.rstd[row * 2 + 1];
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if (a.u) r[j][i] += g[j][i] * cw[j][i] * (u[j][i] * i1);
          dnw[j][i] += z[j][i] * (r[j][i] * i2);
          z[j][i] *= nw[j][i];
          s += z[j][i] * r[j][i];
        }
      const float m = row_sum<TPR>(s, lds[0]) * a.inv_d * i2 * i2 * i2;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i)
          dr[j][i] += a.D > 1 ? i2 * z[j][i] - m * r[j][i] : a.eps * i2 * i2 * i2 * z[j][i];
    }
    if (a.dr) store_row<TR, V, NV, TPR>((TR *)a.dr + row * a.D, t, a.D, dr);
    if (a.u) {
      float s = 0.f, gsum = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float hat = u[j][i] * i1, e = dr[j][i] * cw[j][i];
          q[j][i] += dr[j][i] * g[j][i] * hat;
          s += e * g[j][i] * u[j][i];
          // from here on dr holds the gradient of the norm's output, and g the gate's
          dr[j][i] = e * g[j][i];
          g[j][i] = e * hat * g[j][i] * (1.f - g[j][i]);
          gsum += g[j][i];
        }
      const float m = row_sum<TPR>(s, lds[1]) * a.inv_d * i1 * i1 * i1;
      if (a.du) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < V; ++i)
            dr[j][i] = a.D > 1 ? i1 * dr[j][i] - m * u[j][i] : a.eps * i1 * i1 * i1 * dr[j][i];
        store_row<T, V, NV, TPR>((T *)a.du + row * a.D, t, a.D, dr);
      }
      if (a.dgate) {
        if (a.gate_row) {
          gsum = row_sum<TPR>(gsum, lds[2]);
          if (t == 0) ((T *)a.dgate)[row] = (T)gsum;
        } else {
          store_row<T, V, NV, TPR>((T *)a.dgate + row * a.D, t, a.D, g);
        }
      }
    }
    if constexpr (TPR > kWave) __syncthreads();
  }
  if (!a.part) return;
  float *part = a.part + (int64_t)blockIdx.x * a.D * 2;
  if constexpr (RPB == 1) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int c = (j * TPR + t) * V + i;
        if (c < a.D) {
          part[c] = q[j][i];
          part[a.D + c] = dnw[j][i];
        }
      }
  } else {
    // one vector of columns of the RPB rows of threads at a time
    __shared__ float sums[2][RPB][TPR * V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < V; ++i) {
        sums[0][sub][t * V + i] = q[j][i];
        sums[1][sub][t * V + i] = dnw[j][i];
      }
      __syncthreads();
      for (int e = threadIdx.x; e < 2 * TPR * V; e += block_of<TPR>) {
        const int k = e / (TPR * V), c = e % (TPR * V);
        if (j * TPR * V + c >= a.D) continue;
        float v = 0.f;
#pragma unroll
        for (int n = 0; n < RPB; ++n) v += sums[k][n][c];
        part[k * a.D + j * TPR * V + c] = v;
      }
    }
  }
}

// dpost, dnext, dscale [D] from the partial rows [parts, 2, D].
__global__ __launch_bounds__(kSumThreads) void join_weights_kernel(const float *part, int64_t parts, JoinArgs a, float *dpost,
                                                           float *dnext, float *dscale) {
  int64_t j;
  float s;
  if (!sum_rows(part, parts, 2 * (int64_t)a.D, &j, &s)) return;
  if (j >= a.D) {
    if (dnext) dnext[j - a.D] = s;
    return;
  }
  if (dpost) dpost[j] = s * (a.scale ? a.scale[a.scale_one ? 0 : j] : 1.f);
  if (dscale) dscale[j] = s * a.post[j];
}

// The gradient of one scale for all columns: the sum of what dscale would be.
__global__ __launch_bounds__(256) void join_scale_kernel(const float *v, int32_t D, float *out) {
  __shared__ float lds[4];
  float s = 0.f;
  for (int c = threadIdx.x; c < D; c += 256) s += v[c];
  s = row_sum<256>(s, lds);
  if (threadIdx.x == 0) *out = s;
}

int check(const astra_join_norm *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_SEQ_TYPE_CHECK(f->residual_type);
  if (f->residual_type != f->type && f->residual_type != ASTRA_SEQ_F32)
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_join_norm: the residual is float, or of the block's type");
  ASTRA_ABI_CHECK(f->rows, >=, 0);
  ASTRA_ABI_CHECK(f->width, >=, 1);
  ASTRA_ABI_CHECK(f->width, <=, ASTRA_SEQ_MAX_NORM_WIDTH);
  if (f->gate && f->gate_width != 1) ASTRA_ABI_CHECK(f->gate_width, ==, f->width);
  if (f->scale && f->scale_width != 1) ASTRA_ABI_CHECK(f->scale_width, ==, f->width);
  if (f->block) {
    ASTRA_SEQ_POINTER(f->post);
  } else if (f->gate || f->scale || !f->next) {
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_join_norm: without a block there is only the norm (next) to take");
  }
  return ASTRA_OK;
}

JoinArgs args_of(const astra_join_norm &f) {
  JoinArgs a{};
  a.r = f.residual;
  a.u = f.block;
  a.gate = f.gate;
  a.post = f.post;
  a.next = f.next;
  a.scale = f.scale;
  a.r1 = f.joined;
  a.n = f.normed;
  a.rstd = f.rstd;
  a.rows = f.rows;
  a.rs = f.residual_stride;
  a.us = f.block_stride;
  a.gs = f.gate_stride;
  a.D = f.width;
  a.gate_row = f.gate && f.gate_width == 1 && f.width != 1;
  a.scale_one = f.scale && f.scale_width == 1;
  a.eps = f.eps;
  a.inv_d = 1.f / (float)f.width;
  return a;
}

// How a row is laid over threads.
struct Shape {
  int v, nv, tpr;
  int rows_per_block() const { return tpr > 256 ? 1 : 256 / tpr; }
};

// 16-byte accesses of the block's type where every row allows it. Threads a row: 16 or 32
// lanes where that is one vector each, a wavefront as long as each lane has at most 4
// vectors, then 256 threads, then 1024.
Shape shape_of(const astra_join_norm &f, std::initializer_list<const void *> ptrs) {
  const int V = f.type == ASTRA_SEQ_BF16 ? 8 : 4;
  bool wide = f.width % V == 0 && f.residual_stride % V == 0 && f.block_stride % V == 0 &&
              (!f.gate || f.gate_width == 1 || f.gate_stride % V == 0);
  for (const void *p : ptrs) wide = wide && aligned(p, 16);
  Shape s{wide ? V : 1, 1, 64};
  for (s.tpr = 16; s.tpr < 64 && s.tpr * s.v < f.width;) s.tpr *= 2;
  if (s.tpr < 64) return s;
  for (s.tpr = 64; s.tpr < 1024 && (int64_t)s.tpr * s.v * 4 < f.width; s.tpr *= 4) {
  }
  while ((int64_t)s.tpr * s.v * s.nv < f.width) s.nv *= 2;
  return s;
}

#define JOIN_ONE(V, NV, TPR)                                                                              \
  if (s.v == V && s.nv == NV && s.tpr == TPR) {                                                           \
    if (backward)                                                                                         \
      hipLaunchKernelGGL((join_backward_kernel<TR, T, V, NV, TPR>), grid, dim3(block_of<TPR>), 0, st, a); \
    else                                                                                                  \
      hipLaunchKernelGGL((join_forward_kernel<TR, T, V, NV, TPR>), grid, dim3(block_of<TPR>), 0, st, a);  \
    return;                                                                                               \
  }

template <class TR, class T>
void launch(bool backward, const Shape &s, dim3 grid, hipStream_t st, const JoinArgs &a) {
  constexpr int VW = 16 / sizeof(T);
  JOIN_ONE(VW, 1, 16)
  JOIN_ONE(VW, 1, 32)
  JOIN_ONE(VW, 1, 64)
  JOIN_ONE(VW, 2, 64)
  JOIN_ONE(VW, 4, 64)
  JOIN_ONE(VW, 2, 256)
  JOIN_ONE(VW, 4, 256)
  JOIN_ONE(VW, 2, 1024)
  if constexpr (VW == 4) {
    JOIN_ONE(VW, 4, 1024)
  }
  JOIN_ONE(1, 1, 16)
  JOIN_ONE(1, 1, 32)
  JOIN_ONE(1, 1, 64)
  JOIN_ONE(1, 2, 64)
  JOIN_ONE(1, 4, 64)
  JOIN_ONE(1, 2, 256)
  JOIN_ONE(1, 4, 256)
  JOIN_ONE(1, 2, 1024)
  JOIN_ONE(1, 4, 1024)
  JOIN_ONE(1, 8, 1024)
  JOIN_ONE(1, 16, 1024)
}

// Workgroups: enough to fill the CUs (8 wavefronts a SIMD forwards, 4 backwards, whose
// threads hold more), few enough that the weights and the partial sums are little beside
// the rows.
int64_t blocks_of(const astra_join_norm &f, const Shape &s, bool backward) {
  const int64_t need = cdiv(f.rows, s.rows_per_block());
  const int64_t most = s.tpr > 256 ? 512 : backward ? 1024 : 2048;
  return need < most ? (need > 0 ? need : 1) : most;
}

void dispatch(const astra_join_norm &f, bool backward, const Shape &s, hipStream_t st, const JoinArgs &a) {
  const dim3 grid((unsigned)blocks_of(f, s, backward));
  if (f.type == ASTRA_SEQ_F32)
    launch<float, float>(backward, s, grid, st, a);
  else if (f.residual_type == ASTRA_SEQ_F32)
    launch<float, bf16>(backward, s, grid, st, a);
  else
    launch<bf16, bf16>(backward, s, grid, st, a);
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_join_norm_forward(const astra_join_norm *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->rows == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(f->residual);
  if (f->block) ASTRA_SEQ_POINTER(f->joined);
  if (f->next) ASTRA_SEQ_POINTER(f->normed);
  const Shape s = shape_of(*f, {f->residual, f->block, f->gate_width == 1 ? nullptr : f->gate, f->joined, f->normed});
  dispatch(*f, false, s, as_stream(stream), args_of(*f));
  ASTRA_HIP_CHECK(rt_last_error(), "join_forward_kernel launch");
  return ASTRA_OK;
}

int astra_join_norm_workspace_size(const astra_join_norm *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  // as many partial rows as any layout has, and the sum for a single scale
  const int64_t rows = f->rows < 1024 ? (f->rows > 0 ? f->rows : 1) : 1024;
  *bytes = (size_t)(rows * 2 + 1) * f->width * sizeof(float);
  return ASTRA_OK;
}

int astra_join_norm_backward(const astra_join_norm_grad *g, void *stream) {
  ASTRA_SEQ_POINTER(g);
  const astra_join_norm &f = g->f;
  if (int rc = check(&f)) return rc;
  JoinArgs a = args_of(f);
  a.dr1 = g->djoined;
  a.dn = g->dnormed;
  a.dr = g->dresidual;
  a.du = g->dblock;
  a.dgate = g->dgate;
  if (f.rows) {
    ASTRA_SEQ_POINTER(f.residual);
    ASTRA_SEQ_POINTER(f.rstd);
  }
  if (a.dn) ASTRA_SEQ_POINTER(f.next);
  if ((g->dblock || g->dpost || g->dscale) && !f.block)
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_join_norm_backward: gradients of an absent block");
  if ((g->dgate && !f.gate) || (g->dscale && !f.scale))
    return fail(ASTRA_ERR_INVALID_ARGUMENT, "astra_join_norm_backward: the gradient of an absent gate or scale");
  const Shape s = shape_of(f, {f.residual, f.block, f.gate_width == 1 ? nullptr : f.gate, g->djoined, g->dnormed,
                               g->dresidual, g->dblock, f.gate_width == 1 ? nullptr : g->dgate});
  const int64_t parts = blocks_of(f, s, true);
  const bool sums = g->dpost || g->dnext || g->dscale;
  const hipStream_t st = as_stream(stream);
  float *single = nullptr;
  if (sums) {
    const int64_t need = (parts * 2 + 1) * f.width * (int64_t)sizeof(float);
    ASTRA_SEQ_POINTER(g->workspace);
    ASTRA_ABI_CHECK((int64_t)g->workspace_bytes, >=, need);
    a.part = (float *)g->workspace;
    single = a.part + parts * 2 * f.width;
  }
  if (f.rows || sums) {
    dispatch(f, true, s, st, a);
    ASTRA_HIP_CHECK(rt_last_error(), "join_backward_kernel launch");
  }
  if (sums) {
    float *dscale = g->dscale && a.scale_one ? single : g->dscale;
    hipLaunchKernelGGL(join_weights_kernel, dim3((unsigned)cdiv(2 * (int64_t)f.width, kSumCols)), dim3(kSumThreads), 0, st,
                       a.part, parts, a, g->dpost, g->dnext, dscale);
    ASTRA_HIP_CHECK(rt_last_error(), "join_weights_kernel launch");
    if (g->dscale && a.scale_one) {
      hipLaunchKernelGGL(join_scale_kernel, dim3(1), dim3(256), 0, st, single, f.width, g->dscale);
      ASTRA_HIP_CHECK(rt_last_error(), "join_scale_kernel launch");
    }
  }
  return ASTRA_OK;
}

}  // extern "C"
