// Layer norm over the last dimension, forward and backward, and the sum of partial rows that the backward passes of the
// layer operators share.
//   y = (x - mean) rstd w + b,   rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   dx = rstd (g - mean(g) - xh mean(g xh)),  g = dy w,  xh = (x - mean) rstd;  dw = sum_rows dy xh;  db = sum_rows dy
// HBM-bound: one read and one write of the row forward (2 e bytes an element), two reads and one write backward (3 e).
// A row lives in registers (E elements a thread), so the variance is the centred one at no extra traffic; a wave owns a
// row up to 2048 elements (no barrier at all), a workgroup beyond.  The backward's threads keep their columns over all
// the rows they visit, so the sums over rows stay in registers until one partial row a workgroup is written; a second
// launch adds the partial rows in a fixed order.  Statistics and sums are float32.
// Measured at 16384 x 2048 bf16: forward 23 us (5.8 TB/s), backward 40 + 4 us (4.6 TB/s; without the prefetch of the next
// row 64); 4099 x 1537 f16, rows at odd addresses: 8.4 us (14.7 with one element an access).
#include "bkcore_types.h"

namespace {
using namespace bk;

constexpr int MAX_PARTS = 512;  // partial rows of the backward: two workgroups of 256 threads per CU

// Sum over the TPR threads of a row.  TPR == 64: inside the wave; otherwise through LDS (every thread of the workgroup
// calls it).  `slot` alternates between calls so that one barrier per call is enough.
template <int TPR>
__device__ __forceinline__ float row_sum(float x, float *lds, int slot) {
  x = wave_sum(x);
  if constexpr (TPR == 64) return x;
  constexpr int W = TPR / 64;
  if ((threadIdx.x & 63) == 0) lds[slot * W + (threadIdx.x >> 6)] = x;
  __syncthreads();
  float s = 0.0f;
#pragma unroll
  for (int w = 0; w < W; ++w) s += lds[slot * W + w];
  return s;
}

// A row over TPR threads: thread t's E elements, V = 16 bytes at a time, are columns ((i / V) * TPR + t) * V + i % V of the
// whole pieces.  ALIGNED: rows start at 16-byte addresses and hold whole pieces only.  Otherwise pieces are read at any
// address and the D % V columns behind them belong to the first threads, one each (element E).
template <typename T, int TPR, int E, bool ALIGNED>
struct Row {
  static constexpr int V = 16 / (int)sizeof(T), EX = ALIGNED ? E : E + 1;
  typedef Piece<T, V, ALIGNED> P;
  P r[E / V];
  T last;
  static __device__ __forceinline__ int whole(int D) { return ALIGNED ? D : D / V * V; }
  static __device__ __forceinline__ int column(int e, int t, int D) {
    return e < E ? ((e / V) * TPR + t) * V + e % V : whole(D) + t;
  }
  static __device__ __forceinline__ bool holds(int e, int t, int D) {
    return e < E ? ((e / V) * TPR + t) * V < whole(D) : t < D - whole(D);
  }
  __device__ __forceinline__ void load(const T *__restrict__ p, int t, int D) {
    const int Dv = whole(D);
    if (ALIGNED || Dv > 0) {
#pragma unroll
      for (int c = 0; c < E / V; ++c) {
        const int col = (c * TPR + t) * V;
        r[c].load(p + (col < Dv ? col : 0));
      }
    }
    if constexpr (!ALIGNED) last = p[t < D - Dv ? Dv + t : 0];
  }
  __device__ __forceinline__ void get(int t, int D, float (&v)[EX]) const {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
      float w[V];
      r[c].get(holds(c * V, t, D), w);
#pragma unroll
      for (int i = 0; i < V; ++i) v[c * V + i] = w[i];
    }
    if constexpr (!ALIGNED) v[E] = holds(E, t, D) ? (float)last : 0.0f;
  }
  // o[e] to the thread's columns of row p
  static __device__ __forceinline__ void store(T *__restrict__ p, int t, int D, const float (&o)[EX]) {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
      const int col = (c * TPR + t) * V;
      if (col < whole(D)) {
        float w[V];
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = o[c * V + i];
        P::store(p + col, w);
      }
    }
    if constexpr (!ALIGNED) {
      if (holds(E, t, D)) p[whole(D) + t] = (T)o[E];
    }
  }
  // a parameter vector at the thread's columns
  static __device__ __forceinline__ void param(const void *w, bool f32, int t, int D, float (&v)[EX]) {
#pragma unroll
    for (int c = 0; c < E / V; ++c) {
      const int col = (c * TPR + t) * V;
      float x[V];
      if (col < whole(D)) {
        load_param<T, V>(w, f32, col, x);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = 0.0f;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) v[c * V + i] = x[i];
    }
    if constexpr (!ALIGNED) {
      float x[1] = {0.0f};
      if (holds(E, t, D)) load_param<T, 1>(w, f32, whole(D) + t, x);
      v[E] = x[0];
    }
  }
};

template <typename T, int TPR, int E, bool ALIGNED>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void bk_layer_norm_kernel(
    const T *__restrict__ x, long ldx, const void *__restrict__ w, const void *__restrict__ b, int param_f32, float eps,
    long rows, int D, T *__restrict__ y, float *__restrict__ stats) {
  typedef Row<T, TPR, E, ALIGNED> R;
  constexpr int RPB = TPR == 64 ? 4 : 1;  // rows per workgroup
  __shared__ float lds[2 * (TPR / 64)];
  const int t = TPR == 64 ? threadIdx.x & 63 : threadIdx.x;
  const long row = (long)blockIdx.x * RPB + (TPR == 64 ? threadIdx.x >> 6 : 0);
  if (row >= rows) return;  // uniform in the wave (TPR 64) or in the workgroup
  float v[R::EX], p[R::EX];
  R raw;
  raw.load(x + row * ldx, t, D);
  raw.get(t, D, v);
  float s = 0.0f;
#pragma unroll
  for (int e = 0; e < R::EX; ++e) s += v[e];
  const float mean = row_sum<TPR>(s, lds, 0) / (float)D;
  float q = 0.0f;
#pragma unroll
  for (int e = 0; e < R::EX; ++e) {
    const float d = v[e] - mean;
    if (R::holds(e, t, D)) q = fmaf(d, d, q);
    v[e] = d;
  }
  const float rstd = 1.0f / sqrtf(row_sum<TPR>(q, lds, 1) / (float)D + eps);
#pragma unroll
  for (int e = 0; e < R::EX; ++e) v[e] *= rstd;
  if (w) {
    R::param(w, param_f32, t, D, p);
#pragma unroll
    for (int e = 0; e < R::EX; ++e) v[e] *= p[e];
  }
  if (b) {
    R::param(b, param_f32, t, D, p);
#pragma unroll
    for (int e = 0; e < R::EX; ++e) v[e] += p[e];
  }
  R::store(y + row * (long)D, t, D, v);
  if (stats && t == 0) {
    stats[row] = mean;
    stats[rows + row] = rstd;
  }
}

// part: gridDim.x rows of 2 D floats (weight gradient, bias gradient), or NULL when neither is wanted.
template <typename T, int TPR, int E, bool ALIGNED>
__global__ __launch_bounds__(TPR == 64 ? 256 : TPR) void bk_layer_norm_backward_kernel(
    const T *__restrict__ dy, long lddy, const T *__restrict__ x, long ldx, const void *__restrict__ w, int param_f32,
    const float *__restrict__ stats, long rows, int D, T *__restrict__ dx, float *__restrict__ part) {
  typedef Row<T, TPR, E, ALIGNED> R;
  constexpr int RPB = TPR == 64 ? 4 : 1;
  constexpr int JOIN = TPR == 64 ? 64 * 4 * 8 : 1;
  __shared__ float lds[4 * (TPR / 64)];
  __shared__ float join[JOIN];
  const int t = TPR == 64 ? threadIdx.x & 63 : threadIdx.x;
  const int sub = TPR == 64 ? threadIdx.x >> 6 : 0;
  float dw[R::EX], db[R::EX];
#pragma unroll
  for (int e = 0; e < R::EX; ++e) dw[e] = db[e] = 0.0f;
  int slot = 0;
  R rg, rx;  // the next row is under way while this one is worked on
  float rmean, rrstd;
  auto fetch = [&](long row) {
    rg.load(dy + row * lddy, t, D);
    rx.load(x + row * ldx, t, D);
    rmean = stats[row];
    rrstd = stats[rows + row];
  };
  const long first = (long)blockIdx.x * RPB + sub;
  if (first < rows) fetch(first);
  for (long row = first; row < rows; row += (long)gridDim.x * RPB) {
    float g[R::EX], h[R::EX];
    rg.get(t, D, g);
    rx.get(t, D, h);
    const float mean = rmean, rstd = rrstd;
    const long next = row + (long)gridDim.x * RPB;
    if (next < rows) fetch(next);
    float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
    for (int e = 0; e < R::EX; ++e) {
      h[e] = R::holds(e, t, D) ? (h[e] - mean) * rstd : 0.0f;
      dw[e] = fmaf(g[e], h[e], dw[e]);
      db[e] += g[e];
    }
    if (w) {
      float p[R::EX];
      R::param(w, param_f32, t, D, p);
#pragma unroll
      for (int e = 0; e < R::EX; ++e) g[e] *= p[e];
    }
#pragma unroll
    for (int e = 0; e < R::EX; ++e) {
      s0 += g[e];
      s1 = fmaf(g[e], h[e], s1);
    }
    s0 = row_sum<TPR>(s0, lds, 2 * slot) / (float)D;
    s1 = row_sum<TPR>(s1, lds, 2 * slot + 1) / (float)D;
    slot ^= 1;
#pragma unroll
    for (int e = 0; e < R::EX; ++e) g[e] = rstd * (g[e] - s0 - h[e] * s1);
    R::store(dx + row * (long)D, t, D, g);
  }
  if (!part) return;
  float *pw = part + (long)blockIdx.x * 2 * D, *pb = pw + D;
  if constexpr (TPR == 64) {  // the four waves of the workgroup hold the same columns: join them, 8 at a time
    constexpr int G = 8, N = (R::EX + G - 1) / G;
#pragma unroll
    for (int k = 0; k < 2 * N; ++k) {
      const int e0 = (k % N) * G;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < G; ++i)
        if (e0 + i < R::EX) join[(sub * G + i) * 64 + t] = k < N ? dw[e0 + i < R::EX ? e0 + i : 0] : db[e0 + i < R::EX ? e0 + i : 0];
      __syncthreads();
      for (int j = threadIdx.x; j < G * 64; j += 256) {
        const int i = j >> 6, l = j & 63, e = e0 + i;
        if (e < R::EX && R::holds(e, l, D))
          (k < N ? pw : pb)[R::column(e, l, D)] = join[i * 64 + l] + join[(G + i) * 64 + l] + join[(2 * G + i) * 64 + l] +
                                                  join[(3 * G + i) * 64 + l];
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < R::EX; ++e)
      if (R::holds(e, t, D)) {
        pw[R::column(e, t, D)] = dw[e];
        pb[R::column(e, t, D)] = db[e];
      }
  }
}

// 16 columns x 16 groups of partial rows per workgroup.
__global__ __launch_bounds__(256) void bk_sum_parts_kernel(const float *__restrict__ part, long parts, long cols,
                                                           float *__restrict__ out) {
  __shared__ float acc[16][17];
  const int cx = threadIdx.x & 15, gy = threadIdx.x >> 4;
  const long col = (long)blockIdx.x * 16 + cx;
  float s = 0.0f;
  if (col < cols) {
#pragma unroll 4
    for (long p = gy; p < parts; p += 16) s += part[p * cols + col];
  }
  acc[gy][cx] = s;
  __syncthreads();
  if (gy == 0 && col < cols) {
    float r = 0.0f;
#pragma unroll
    for (int k = 0; k < 16; ++k) r += acc[k][cx];
    out[col] = r;
  }
}

// Rows of the backward a workgroup takes at least: partial rows are written and read once more, so few rows must not
// leave as many partial rows as there are rows.
inline int64_t norm_parts(int64_t rows, int64_t D) {
  const int64_t rpb = D <= 2048 ? 4 : 1;
  int64_t n = (rows + 4 * rpb - 1) / (4 * rpb);
  return n < 1 ? 1 : n > MAX_PARTS ? MAX_PARTS : n;
}

}  // namespace

extern "C" void bkcore_internal_sum_parts(const float *part, int64_t parts, int64_t cols, float *out, void *stream) {
  hipLaunchKernelGGL(bk_sum_parts_kernel, dim3((unsigned)((cols + 15) / 16)), dim3(256), 0, (hipStream_t)stream, part,
                     (long)parts, (long)cols, out);
}

// The variant by width alone: threads a row x elements a thread.
#define BK_NORM_SHAPES(LAUNCH)                  \
  do {                                          \
    if (D <= 512) LAUNCH(64, 8);                \
    else if (D <= 1024) LAUNCH(64, 16);         \
    else if (D <= 2048) LAUNCH(64, 32);         \
    else if (D <= 4096) LAUNCH(256, 16);        \
    else if (D <= 8192) LAUNCH(256, 32);        \
    else LAUNCH(512, 32);                      \
  } while (0)

extern "C" int bkcore_layer_norm(const void *x, int64_t ldx, int dtype, const void *weight, const void *bias,
                                 int param_dtype, float eps, int64_t rows, int64_t D, void *y, float *stats,
                                 void *stream) {
  const int es = elem_size(dtype);
  if (rows < 0 || D < 1 || D > BKCORE_LAYER_NORM_MAX_DIM || !es || !(eps >= 0.0f)) return BKCORE_EINVAL;
  if ((weight || bias) && param_dtype != BKCORE_F32 && param_dtype != dtype) return BKCORE_EINVAL;
  if (rows == 0) return BKCORE_OK;
  if (!x || !y || rows > 2147483647LL) return BKCORE_EINVAL;
  hipStream_t s = (hipStream_t)stream;
  const int v = 16 / es, pf = param_dtype == BKCORE_F32;
  const bool vec = D % v == 0 && ldx % v == 0 && aligned16(x) && aligned16(y);
#define BK_LN_V(TPR, E, V)                                                                                             \
  hipLaunchKernelGGL((bk_layer_norm_kernel<T, TPR, E, V>), dim3((unsigned)((rows + (TPR == 64 ? 3 : 0)) / (TPR == 64 ? 4 : 1))), \
                     dim3(TPR == 64 ? 256 : TPR), 0, s, (const T *)x, (long)ldx, weight, bias, pf, eps, (long)rows,    \
                     (int)D, (T *)y, stats)
#define BK_LN(TPR, E)                                           \
  do {                                                          \
    if (vec) BK_LN_V(TPR, E, true);                             \
    else BK_LN_V(TPR, E, false);                                \
  } while (0)
  BK_WITH_TYPE(dtype, BK_NORM_SHAPES(BK_LN));
#undef BK_LN
#undef BK_LN_V
  return launch_status();
}

extern "C" size_t bkcore_layer_norm_backward_workspace_bytes(int64_t rows, int64_t D) {
  if (rows <= 0 || D <= 0) return 0;
  return (size_t)norm_parts(rows, D) * 2 * (size_t)D * sizeof(float);
}

extern "C" int bkcore_layer_norm_backward(const void *dy, int64_t lddy, const void *x, int64_t ldx, int dtype,
                                          const void *weight, int param_dtype, const float *stats, int64_t rows,
                                          int64_t D, void *dx, float *grad_params, void *workspace,
                                          size_t workspace_bytes, void *stream) {
  const int es = elem_size(dtype);
  if (rows < 0 || D < 1 || D > BKCORE_LAYER_NORM_MAX_DIM || !es) return BKCORE_EINVAL;
  if (weight && param_dtype != BKCORE_F32 && param_dtype != dtype) return BKCORE_EINVAL;
  if (rows == 0) return BKCORE_OK;  // the caller's gradients of the parameters are zero
  if (!dy || !x || !stats || !dx || rows > 2147483647LL) return BKCORE_EINVAL;
  if (grad_params && (!workspace || workspace_bytes < bkcore_layer_norm_backward_workspace_bytes(rows, D)))
    return BKCORE_EWORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const int v = 16 / es, pf = param_dtype == BKCORE_F32;
  const bool vec = D % v == 0 && ldx % v == 0 && lddy % v == 0 && aligned16(x) && aligned16(dy) && aligned16(dx);
  const int64_t parts = norm_parts(rows, D);
  float *part = grad_params ? (float *)workspace : nullptr;
#define BK_LN_V(TPR, E, V)                                                                                             \
  hipLaunchKernelGGL((bk_layer_norm_backward_kernel<T, TPR, E, V>), dim3((unsigned)parts), dim3(TPR == 64 ? 256 : TPR), 0, s, \
                     (const T *)dy, (long)lddy, (const T *)x, (long)ldx, weight, pf, stats, (long)rows, (int)D, (T *)dx, part)
#define BK_LN(TPR, E)                                           \
  do {                                                          \
    if (vec) BK_LN_V(TPR, E, true);                             \
    else BK_LN_V(TPR, E, false);                                \
  } while (0)
  BK_WITH_TYPE(dtype, BK_NORM_SHAPES(BK_LN));
#undef BK_LN
#undef BK_LN_V
  if (grad_params) bkcore_internal_sum_parts(part, parts, 2 * D, grad_params, stream);
  return launch_status();
}
