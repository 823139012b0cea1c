// sequence_conv.hip -- the short causal convolution: every channel of a sequence is
// filtered by its own K taps (2 to 4), followed by x * sigmoid(x) if asked for.
//
//   p[t] = bias + sum_k w[k] x[t-K+1+k],  y[t] = act(p[t])
//
// K + 1 multiply-adds and one exp per element that is read and written once: the kernels
// are bound by memory traffic.
#include "sequence.h"

#define ASTRA_SRC_NAME "sequence_conv.hip"

namespace astra_seq {
namespace {

struct ConvArgs {
  const void *x, *window, *dy, *dlast;
  const float *weight, *bias;
  const int32_t *lengths;
  void *y, *last, *dx, *dwindow;
  float *part;
  int64_t B, T, xsb, xst;
  int32_t D, silu, run, runs;  // a thread walks `run` positions; `runs` such runs to a row
};

// The taps of V channels: w[k][i], bias in b.
template <int K, int V>
__device__ __forceinline__ void load_taps(const ConvArgs &a, int d, float (&w)[K][V], float (&b)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) {
    b[i] = a.bias ? a.bias[d + i] : 0.f;
    float taps[K];
    __builtin_memcpy(taps, a.weight + (int64_t)(d + i) * K, sizeof(taps));
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = taps[k];
  }
}

// The input at position t (from the window before the start, zeros at and after `len`).
template <class T, int K, int V>
__device__ __forceinline__ void load_input(const ConvArgs &a, int64_t b, int64_t t, int len, int d, float (&v)[V]) {
  if (t >= 0 && t < len) {
    Vec<T, V>::load((const T *)a.x + b * a.xsb + t * a.xst + d, v);
  } else if (t < 0 && a.window) {
    Vec<T, V>::load((const T *)a.window + (b * (K - 1) + t + K - 1) * a.D + d, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.f;
  }
}

// One thread: V channels, `run` positions, the last K-1 inputs in registers. U positions at
// a time, so that their loads are in flight together; where all of them count, without a
// check each. Bound by traffic: 65,537 positions of 1,280 float channels 138 us, 4.9 TB/s (a
// large copy 4.7); 2,048 games of 40 positions and 640 bf16 channels 45 us.
template <class T, int K, int V>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs a) {
  constexpr int U = 4;
  const int groups = a.D / V;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = item / groups;
  const int d = (int)(item - row * groups) * V;
  const int64_t b = row / a.runs;
  if (b >= a.B) return;
  const int t0 = (int)(row - b * a.runs) * a.run;
  const int t1 = (int)min((int64_t)t0 + a.run, a.T);
  const int len = row_length(a.lengths, b, a.T);
  float w[K][V], bias[V], in[K - 1 + U][V];  // entry K-1+u is position t+u
  load_taps<K, V>(a, d, w, bias);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load_input<T, K, V>(a, b, t0 - (K - 1) + k, len, d, in[k]);
  const T *x = (const T *)a.x + b * a.xsb + (int64_t)t0 * a.xst + d;
  T *y = (T *)a.y + (b * a.T + t0) * a.D + d;
  const int64_t xst = a.xst, yst = a.D;
  auto outputs = [&](int t, bool all) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!all && t + u >= t1) break;
      float out[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float p = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) p += w[k][i] * in[u + k][i];
        out[i] = a.silu ? p * sigmoid<T>(p) : p;
        if (!all) out[i] = t + u < len ? out[i] : 0.f;
      }
      Vec<T, V>::store(y + u * yst, out);
    }
#pragma unroll
    for (int k = 0; k < K - 1; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) in[k][i] = in[k + U][i];
    x += U * xst;
    y += U * yst;
  };
  int t = t0;
  for (const int full = min(t1, len); t + U <= full; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T, V>::load(x + u * xst, in[K - 1 + u]);
    outputs(t, true);
  }
  for (; t < t1; t += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) load_input<T, K, V>(a, b, t + u, len, d, in[K - 1 + u]);
    outputs(t, false);
  }
  if (a.last && t0 == 0) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      float v[V];
      load_input<T, K, V>(a, b, (int64_t)len - (K - 1) + k, len, d, v);
      Vec<T, V>::store((T *)a.last + (b * (K - 1) + k) * a.D + d, v);
    }
  }
}

// g[t] = dy[t] act'(p[t]); dx[t] = sum_k w[k] g[t+K-1-k]; dw[k] = sum_t g[t] x[t-K+1+k].
// A workgroup: CX groups of V channels by 256 / CX rows; a row of threads walks runs of
// positions, `gridDim.y` rows of workgroups apart, and keeps its part of dw and dbias in
// registers. A run recomputes the K-1 values of g after its end. U positions at a time, so
// that their loads are in flight together and the windows of x and g need few moves; inside
// a run without a check each. 2,048 games of 40 positions and 640 bf16 channels: 104 us, 3.0
// TB/s, where its bytes take 67; in floats 150 us, 4.2 TB/s. Neither traffic nor vector work
// (43% busy) is the limit, but what is in flight: 188 registers leave room for two wavefronts
// a SIMD, and 1.5 are there on average. Channel by channel (odd widths) 220 and 258 us.
constexpr int kConvCols = 16;
template <class T, int K, int V>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs a) {
  constexpr int CX = kConvCols, IY = 256 / CX, U = 4;
  const int cx = threadIdx.x % CX, iy = threadIdx.x / CX;
  const int groups = a.D / V;
  const int cg = blockIdx.x * CX + cx;
  const bool live = cg < groups;
  const int d = (live ? cg : 0) * V;
  float w[K][V], bias[V], dw[K][V], db[V];
  load_taps<K, V>(a, d, w, bias);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][i] = 0.f;
  }
  const int64_t rows = a.B * a.runs;
  for (int64_t row = (int64_t)blockIdx.y * IY + iy; row < rows && live; row += (int64_t)gridDim.y * IY) {
    const int64_t b = row / a.runs;
    const int t0 = (int)(row - b * a.runs) * a.run;
    const int t1 = (int)min((int64_t)t0 + a.run, a.T);
    const int len = row_length(a.lengths, b, a.T);
    float in[K - 1 + U][V], g[K - 1 + U][V];  // entry K-1+u is position t+u
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      load_input<T, K, V>(a, b, t0 - (K - 1) + k, len, d, in[k]);
      // the g before a run are another run's, but no output of this one takes them: it
      // writes dx[t - (K-1)] for t in [t0 + K-1, t1 + K-1), and the window
#pragma unroll
      for (int i = 0; i < V; ++i) g[k][i] = 0.f;
    }
    const T *x = (const T *)a.x + b * a.xsb + (int64_t)t0 * a.xst + d;
    const T *dyp = (const T *)a.dy + (b * a.T + t0) * a.D + d;
    T *dx = (T *)a.dx + (b * a.T + t0 - (K - 1)) * a.D + d;
    float dy[U][V];
    auto gradients = [&](int t, bool all) __attribute__((always_inline)) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float v = dy[u][i];
          if (a.silu) {
            float p = bias[i];
#pragma unroll
            for (int k = 0; k < K; ++k) p += w[k][i] * in[u + k][i];
            const float s = sigmoid<T>(p);
            v *= s + p * (s - s * s);
          }
          if (!all) v = t + u < len ? v : 0.f;
          g[K - 1 + u][i] = v;
          if (!all) v = t + u < t1 ? v : 0.f;
          db[i] += v;
#pragma unroll
          for (int k = 0; k < K; ++k) dw[k][i] += v * in[u + k][i];
        }
        // the gradient of the input at t + u - (K-1); before 0 it is the window's
        const int at = t + u - (K - 1);
        if (!all && (t + u >= t1 + K - 1 || (at < t0 && t0 > 0))) continue;
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          o[i] = 0.f;
#pragma unroll
          for (int k = 0; k < K; ++k) o[i] += w[k][i] * g[K - 1 + u - k][i];
        }
        if (all) {
          if (a.dx) Vec<T, V>::store(dx + (int64_t)u * a.D, o);
          continue;
        }
        // position len - (K-1) + k is row k of `last`
        if (a.dlast && at < len && t + u >= len) {
          float e[V];
          Vec<T, V>::load((const T *)a.dlast + (b * (K - 1) + (t + u - len)) * a.D + d, e);
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] += e[i];
        }
        if (at >= 0) {
          if (a.dx) {
            if (at >= len)
#pragma unroll
              for (int i = 0; i < V; ++i) o[i] = 0.f;
            Vec<T, V>::store(dx + (int64_t)u * a.D, o);
          }
        } else if (a.dwindow) {
          Vec<T, V>::store((T *)a.dwindow + (b * (K - 1) + t + u) * a.D + d, o);
        }
      }
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          in[k][i] = in[k + U][i];
          g[k][i] = g[k + U][i];
        }
      x += U * a.xst;
      dyp += (int64_t)U * a.D;
      dx += (int64_t)U * a.D;
    };
    // the first U positions write the window, or nothing; from the last ones on, some do
    // not count
    int t = t0;
    for (const int full = min(t1, len); t < t1 + K - 1; t += U) {
      if (t > t0 && t + U <= full) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Vec<T, V>::load(x + u * a.xst, in[K - 1 + u]);
          Vec<T, V>::load(dyp + (int64_t)u * a.D, dy[u]);
        }
        gradients(t, true);
        continue;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        load_input<T, K, V>(a, b, t + u, len, d, in[K - 1 + u]);
        if (t + u < len)
          Vec<T, V>::load(dyp + (int64_t)u * a.D, dy[u]);
        else
#pragma unroll
          for (int i = 0; i < V; ++i) dy[u][i] = 0.f;
      }
      gradients(t, false);
    }
  }
  if (!a.part) return;
  // the workgroup's sums: row blockIdx.y of part [gridDim.y, D, K + 1]
  __shared__ float lds[IY][CX][V + 1];
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float v = db[i];
#pragma unroll
      for (int q = 0; q < K; ++q) v = k == q ? dw[q][i] : v;
      lds[iy][cx][i] = v;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < CX * V; e += 256) {
      const int c = e / V, i = e % V;
      if (blockIdx.x * CX + c >= groups) continue;
      float s = 0.f;
      for (int r = 0; r < IY; ++r) s += lds[r][c][i];
      const int64_t dd = (int64_t)(blockIdx.x * CX + c) * V + i;
      a.part[((int64_t)blockIdx.y * a.D + dd) * (K + 1) + k] = s;
    }
  }
}

// dweight and dbias from the partial rows [parts, D, K + 1].
template <int K>
__global__ __launch_bounds__(kSumThreads) void conv_weights_kernel(const float *part, int64_t parts, int32_t D, float *dw,
                                                           float *db) {
  int64_t j;
  float s;
  if (!sum_rows(part, parts, (int64_t)D * (K + 1), &j, &s)) return;
  const int64_t d = j / (K + 1);
  const int k = (int)(j - d * (K + 1));
  if (k < K) {
    if (dw) dw[d * K + k] = s;
  } else if (db) {
    db[d] = s;
  }
}

template <class T, int K, int V>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs a) {
  const int groups = a.D / V;
  const int64_t item = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t b = item / groups;
  if (b >= a.B) return;
  const int d = (int)(item - b * groups) * V;
  float w[K][V], bias[V], in[K][V], out[V];
  load_taps<K, V>(a, d, w, bias);
  T *win = (T *)a.dwindow + b * (K - 1) * a.D + d;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) Vec<T, V>::load(win + (int64_t)k * a.D, in[k]);
  Vec<T, V>::load((const T *)a.x + b * a.xsb + d, in[K - 1]);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float p = bias[i];
#pragma unroll
    for (int k = 0; k < K; ++k) p += w[k][i] * in[k][i];
    out[i] = a.silu ? p * sigmoid<T>(p) : p;
  }
  Vec<T, V>::store((T *)a.y + b * a.D + d, out);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) Vec<T, V>::store(win + (int64_t)k * a.D, in[k + 1]);
}

int check(const astra_short_conv *f) {
  ASTRA_SEQ_POINTER(f);
  ASTRA_SEQ_TYPE_CHECK(f->type);
  ASTRA_ABI_CHECK(f->batch, >=, 0);
  ASTRA_ABI_CHECK(f->length, >=, 0);
  ASTRA_ABI_CHECK(f->length, <, 2147483647 - 64);
  ASTRA_ABI_CHECK(f->width, >=, 1);
  ASTRA_ABI_CHECK(f->taps, >=, 2);
  ASTRA_ABI_CHECK(f->taps, <=, ASTRA_SEQ_MAX_TAPS);
  ASTRA_ABI_CHECK(f->activation, >=, ASTRA_SEQ_LINEAR);
  ASTRA_ABI_CHECK(f->activation, <=, ASTRA_SEQ_SILU);
  return ASTRA_OK;
}

ConvArgs args_of(const astra_short_conv &f) {
  ConvArgs a{};
  a.x = f.x;
  a.window = f.window;
  a.weight = f.weight;
  a.bias = f.bias;
  a.lengths = f.lengths;
  a.y = f.y;
  a.last = f.last;
  a.B = f.batch;
  a.T = f.length;
  a.xsb = f.x_stride_b;
  a.xst = f.x_stride_t;
  a.D = f.width;
  a.silu = f.activation == ASTRA_SEQ_SILU;
  return a;
}

// Positions a thread walks: long runs reread less of their neighbours (K-1 inputs each),
// short ones give every CU work where the batch is small. Runs of a row are alike, and of
// whole groups of four positions.
void set_runs(ConvArgs &a, int64_t threads_per_position) {
  int64_t run = 64;
  while (run > 8 && a.B * cdiv(a.T, run) * threads_per_position < 256 * 1024) run /= 2;
  const int64_t runs = a.T > 0 ? cdiv(a.T, run) : 1;
  a.run = (int32_t)(a.T > 0 ? cdiv(cdiv(a.T, runs), 4) * 4 : 1);
  a.runs = (int32_t)(a.T > 0 ? cdiv(a.T, a.run) : 1);
}

// Accesses of V elements where every row starts on one.
template <class T, int V>
int wide(const ConvArgs &a, std::initializer_list<const void *> ptrs) {
  if (a.D % V || a.xsb % V || a.xst % V) return 1;
  for (const void *p : ptrs)
    if (!aligned(p, V * sizeof(T))) return 1;
  return V;
}

// Channels of a thread: 16 bytes forwards; backwards, where 11 values of each are in
// registers, 4.
template <class T>
constexpr int kForward = 16 / sizeof(T);
constexpr int kBackward = 4;

#define CONV_DISPATCH(T, KERNEL, VW, grid)                                                    \
  do {                                                                                        \
    if (v == 1) {                                                                             \
      if (taps == 2) hipLaunchKernelGGL((KERNEL<T, 2, 1>), grid, dim3(256), 0, st, a);        \
      if (taps == 3) hipLaunchKernelGGL((KERNEL<T, 3, 1>), grid, dim3(256), 0, st, a);        \
      if (taps == 4) hipLaunchKernelGGL((KERNEL<T, 4, 1>), grid, dim3(256), 0, st, a);        \
    } else {                                                                                  \
      if (taps == 2) hipLaunchKernelGGL((KERNEL<T, 2, VW>), grid, dim3(256), 0, st, a);       \
      if (taps == 3) hipLaunchKernelGGL((KERNEL<T, 3, VW>), grid, dim3(256), 0, st, a);       \
      if (taps == 4) hipLaunchKernelGGL((KERNEL<T, 4, VW>), grid, dim3(256), 0, st, a);       \
    }                                                                                         \
  } while (false)

template <class T>
int forward(const astra_short_conv &f, hipStream_t st) {
  ConvArgs a = args_of(f);
  const int v = wide<T, kForward<T>>(a, {a.x, a.window, a.y, a.last}), taps = f.taps;
  set_runs(a, a.D / v);
  const int64_t blocks = cdiv(a.B * a.runs * (a.D / v), 256);
  ASTRA_SEQ_LAUNCH_CHECK(blocks, 256);
  CONV_DISPATCH(T, conv_forward_kernel, kForward<T>, dim3((unsigned)blocks));
  ASTRA_HIP_CHECK(rt_last_error(), "conv_forward_kernel launch");
  return ASTRA_OK;
}

// Rows of workgroups of the backward kernel, which is how many partial sums there are.
int64_t backward_rows(const ConvArgs &a, int v) {
  const int64_t cols = cdiv(a.D / v, kConvCols);
  const int64_t most = cdiv(a.B * a.runs, 256 / kConvCols);
  int64_t rows = cdiv(2048, cols);
  if (rows > 512) rows = 512;
  return rows < most ? rows : (most > 0 ? most : 1);
}

template <class T>
int backward(const astra_short_conv_grad &g, hipStream_t st) {
  ConvArgs a = args_of(g.f);
  a.dy = g.dy;
  a.dlast = g.dlast;
  a.dx = g.dx;
  a.dwindow = g.dwindow;
  const int v = wide<T, kBackward>(a, {a.x, a.window, a.dy, a.dlast, a.dx, a.dwindow}), taps = g.f.taps;
  set_runs(a, a.D / v);
  const int64_t rows = backward_rows(a, v);
  const bool sums = g.dweight || g.dbias;
  if (sums) {
    ASTRA_SEQ_POINTER(g.workspace);
    ASTRA_ABI_CHECK((int64_t)g.workspace_bytes, >=, (int64_t)(rows * a.D * (taps + 1) * sizeof(float)));
    a.part = (float *)g.workspace;
  }
  CONV_DISPATCH(T, conv_backward_kernel, kBackward, dim3((unsigned)cdiv(a.D / v, kConvCols), (unsigned)rows));
  ASTRA_HIP_CHECK(rt_last_error(), "conv_backward_kernel launch");
  if (sums) {
    const dim3 grid((unsigned)cdiv((int64_t)a.D * (taps + 1), kSumCols));
    if (taps == 2) hipLaunchKernelGGL(conv_weights_kernel<2>, grid, dim3(kSumThreads), 0, st, a.part, rows, a.D, g.dweight, g.dbias);
    if (taps == 3) hipLaunchKernelGGL(conv_weights_kernel<3>, grid, dim3(kSumThreads), 0, st, a.part, rows, a.D, g.dweight, g.dbias);
    if (taps == 4) hipLaunchKernelGGL(conv_weights_kernel<4>, grid, dim3(kSumThreads), 0, st, a.part, rows, a.D, g.dweight, g.dbias);
    ASTRA_HIP_CHECK(rt_last_error(), "conv_weights_kernel launch");
  }
  return ASTRA_OK;
}

template <class T>
int step(const astra_short_conv_one &o, hipStream_t st) {
  ConvArgs a{};
  a.x = o.x;
  a.weight = o.weight;
  a.bias = o.bias;
  a.dwindow = o.window;
  a.y = o.y;
  a.B = o.batch;
  a.xsb = o.x_stride_b;
  a.D = o.width;
  a.silu = o.activation == ASTRA_SEQ_SILU;
  const int v = wide<T, kForward<T>>(a, {a.x, a.dwindow, a.y}), taps = o.taps;
  const int64_t blocks = cdiv(a.B * (a.D / v), 256);
  ASTRA_SEQ_LAUNCH_CHECK(blocks, 256);
  CONV_DISPATCH(T, conv_step_kernel, kForward<T>, dim3((unsigned)blocks));
  ASTRA_HIP_CHECK(rt_last_error(), "conv_step_kernel launch");
  return ASTRA_OK;
}

}  // namespace
}  // namespace astra_seq

using namespace astra_seq;

extern "C" {

int astra_short_conv_forward(const astra_short_conv *f, void *stream) {
  if (int rc = check(f)) return rc;
  if (f->batch == 0) return ASTRA_OK;
  if (f->length) {
    ASTRA_SEQ_POINTER(f->x);
    ASTRA_SEQ_POINTER(f->y);
  } else if (!f->last) {
    return ASTRA_OK;
  }
  ASTRA_SEQ_POINTER(f->weight);
  return f->type == ASTRA_SEQ_BF16 ? forward<bf16>(*f, as_stream(stream)) : forward<float>(*f, as_stream(stream));
}

int astra_short_conv_workspace_size(const astra_short_conv *f, size_t *bytes) {
  if (int rc = check(f)) return rc;
  ASTRA_SEQ_POINTER(bytes);
  // the most partial rows that any alignment leads to
  ConvArgs a = args_of(*f);
  int64_t rows = 1;
  for (int v : {1, kBackward}) {
    if (a.D % v) continue;
    set_runs(a, a.D / v);
    const int64_t r = backward_rows(a, v);
    rows = r > rows ? r : rows;
  }
  *bytes = (size_t)rows * f->width * (f->taps + 1) * sizeof(float);
  return ASTRA_OK;
}

int astra_short_conv_backward(const astra_short_conv_grad *g, void *stream) {
  ASTRA_SEQ_POINTER(g);
  if (int rc = check(&g->f)) return rc;
  const astra_short_conv &f = g->f;
  if (f.batch && f.length) {
    ASTRA_SEQ_POINTER(f.x);
    ASTRA_SEQ_POINTER(g->dy);
  }
  ASTRA_SEQ_POINTER(f.weight);
  if (f.batch == 0 && !g->dweight && !g->dbias) return ASTRA_OK;
  return f.type == ASTRA_SEQ_BF16 ? backward<bf16>(*g, as_stream(stream)) : backward<float>(*g, as_stream(stream));
}

int astra_short_conv_step(const astra_short_conv_one *o, void *stream) {
  ASTRA_SEQ_POINTER(o);
  ASTRA_SEQ_TYPE_CHECK(o->type);
  ASTRA_ABI_CHECK(o->batch, >=, 0);
  ASTRA_ABI_CHECK(o->width, >=, 1);
  ASTRA_ABI_CHECK(o->taps, >=, 2);
  ASTRA_ABI_CHECK(o->taps, <=, ASTRA_SEQ_MAX_TAPS);
  ASTRA_ABI_CHECK(o->activation, >=, ASTRA_SEQ_LINEAR);
  ASTRA_ABI_CHECK(o->activation, <=, ASTRA_SEQ_SILU);
  if (o->batch == 0) return ASTRA_OK;
  ASTRA_SEQ_POINTER(o->x);
  ASTRA_SEQ_POINTER(o->weight);
  ASTRA_SEQ_POINTER(o->window);
  ASTRA_SEQ_POINTER(o->y);
  return o->type == ASTRA_SEQ_BF16 ? step<bf16>(*o, as_stream(stream)) : step<float>(*o, as_stream(stream));
}

}  // extern "C"
