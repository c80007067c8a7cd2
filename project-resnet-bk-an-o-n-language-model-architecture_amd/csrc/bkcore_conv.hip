// The short causal convolution of a selective mixer (depthwise, K = 2..4 taps, channels innermost), forward, backward and
// for single tokens.
//   pre_t = bias + sum_k w_k x_{t-K+1+k},  y_t = pre_t or silu(pre_t);  x at t < 0 is the carried state, or zero
//   g_t = dy_t act'(pre_t);  dx_t = sum_k w_k g_{t+K-1-k};  dw_k = sum g_t x_{t-K+1+k};  db = sum g_t
// Positions at or behind a sequence's length are padding: what is loaded there is dropped, y and dx there are zero.
// HBM-bound: 2 e bytes an element forward, 3 e backward (8 x 2048 x 1024 bf16: 18.5 us = 3.6 TB/s, and 31.9 + 4 us =
// 2.8 TB/s; the forward's vector unit is busy 32 % of the time, the backward's 66 %).  A thread holds V neighbouring channels (16 bytes a position forward, 4 channels backward, where five sums and
// two windows a channel take the registers) and walks a stretch of positions with the last K - 1 inputs in registers; only
// the K - 1 positions in front of its stretch are read twice, from cache.  Arithmetic and sums are float32.
#include "bkcore_types.h"

namespace {
using namespace bk;

constexpr int FWD_TL = 9;   // positions a thread walks forward; stretches a power of two apart meet on the same memory channels
                            // (8 x 2048 x 1024 bf16: 18.5 us at 9, 20.4 at 8, 19.7 at 16)
constexpr int BWD_TL = 16;  // ... and backward (31.9 us there and 12.8 at 2 x 300 x 256; 32: 30.0 and 22.1)
constexpr int BWD_SEGS = 8; // stretches of one workgroup, joined before the partial sums are written
constexpr int BWD_CH = 32;  // channel vectors of one workgroup

struct ConvArgs {
  const void *x, *w, *bias, *init, *dy, *dfinal;
  void *y, *final_state, *dx, *dinit;
  float *part;
  const int *lengths;
  long xb, xt, dyb, dyt;  // strides of x and dy in elements
  int B, L, C, param_f32, param_vec, silu;
};

__device__ __forceinline__ int row_length(const int *lengths, int b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

template <typename T, int V, bool AL>
__device__ __forceinline__ void load_piece(const T *__restrict__ p, float (&v)[V]) {
  Piece<T, V, AL> r;
  r.load(p);
  r.get(true, v);
}

// First channel of the i-th piece: the last one reaches back into its neighbour where V does not divide the channels (both
// compute and write the same values there).
template <int V>
__device__ __forceinline__ int piece_channel(int i, int C) {
  return V == 1 || (i + 1) * V <= C ? i * V : C - V;
}

// x_t of sequence b for V channels from c: the carried state for t < 0, zero where there is none or behind the length.
template <typename T, int K, int V, bool AL>
__device__ __forceinline__ void input_at(const ConvArgs &a, int b, long t, int len, int c, float (&v)[V]) {
  if (t >= 0 && t < len) {
    load_piece<T, V, AL>((const T *)a.x + b * a.xb + t * a.xt + c, v);
  } else if (t < 0 && a.init) {
    load_piece<T, V, AL>((const T *)a.init + ((long)b * (K - 1) + (t + K - 1)) * a.C + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = 0.0f;
  }
}

// The K - 1 inputs in front of position t0, all under way together: positions, or the carried state in front of the first.
template <typename T, int K, int V, bool AL>
struct Halo {
  Piece<T, V, AL> r[K - 1];
  __device__ __forceinline__ void load(const T *__restrict__ x, long step, long t0, int L) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const long t = t0 - (K - 1) + k;
      r[k].load(x + (t < 0 ? 0 : t < L ? t : L - 1) * step);
    }
  }
  __device__ __forceinline__ void get(const ConvArgs &a, int b, long t0, int len, int c, float (&h)[K][V]) const {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const long t = t0 - (K - 1) + k;
      r[k].get(t >= 0 && t < len, h[k]);
    }
    if (t0 == 0 && a.init) {  // stretches are longer than the window: only the first one reaches in front of the sequence
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
        load_piece<T, V, AL>((const T *)a.init + ((long)b * (K - 1) + k) * a.C + c, h[k]);
    }
  }
};

// The taps of V channels are V K neighbouring values; in float32 and aligned they come as 16-byte loads.
template <typename T, int K, int V, bool AL>
__device__ __forceinline__ void load_taps(const ConvArgs &a, int c, float (&w)[K][V], float (&bias)[V]) {
  float flat[V * K];
  if (V > 1 && AL && a.param_vec) {
    const f32x4 *p = reinterpret_cast<const f32x4 *>((const float *)a.w + (long)c * K);
#pragma unroll
    for (int j = 0; j < V * K / 4; ++j) {
      const f32x4 v = p[j];
#pragma unroll
      for (int i = 0; i < 4; ++i) flat[4 * j + i] = v[i];
    }
  } else {
    load_param<T, V * K>(a.w, a.param_f32, (long)c * K, flat);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    bias[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][i] = flat[i * K + k];
  }
  if (a.bias) load_param<T, V>(a.bias, a.param_f32, c, bias);
}

template <typename T, int K, int V, bool AL>
__global__ __launch_bounds__(256) void bk_conv_kernel(ConvArgs a, int nseg, int nvec) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * nseg * nvec) return;
  const int c = piece_channel<V>((int)(id % nvec), a.C);
  const long r = id / nvec;
  const int seg = (int)(r % nseg), b = (int)(r / nseg);
  const int len = row_length(a.lengths, b, a.L);
  const int t0 = seg * FWD_TL, t1 = t0 + FWD_TL < a.L ? t0 + FWD_TL : a.L;
  if (t0 < a.L) {
    const T *x = (const T *)a.x + b * a.xb + c;
    Piece<T, V, AL> raw[FWD_TL];  // all of the stretch is under way before its first position is worked on
#pragma unroll
    for (int j = 0; j < FWD_TL; ++j) raw[j].load(x + (long)(t0 + j < a.L ? t0 + j : a.L - 1) * a.xt);
    Halo<T, K, V, AL> halo;
    halo.load(x, a.xt, t0, a.L);
    float w[K][V], bias[V], h[K][V];
    load_taps<T, K, V, AL>(a, c, w, bias);
    halo.get(a, b, t0, len, c, h);
    T *y = (T *)a.y + ((long)b * a.L) * a.C + c;
#pragma unroll
    for (int j = 0; j < FWD_TL; ++j) {
      const int t = t0 + j;
      raw[j].get(t < len, h[K - 1]);
      float o[V];
#pragma unroll
      for (int i = 0; i < V; ++i) {
        float s = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) s = fmaf(w[k][i], h[k][i], s);
        if (a.silu) s = s * sigmoid(s);
        o[i] = t < len ? s : 0.0f;
      }
      if (t < t1) Piece<T, V, AL>::store(y + (long)t * a.C, o);
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) h[k][i] = h[k + 1][i];
    }
  }
  if (a.final_state && seg == 0) {  // the last K - 1 inputs, the carried ones among them for a short sequence
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
      float v[V];
      input_at<T, K, V, AL>(a, b, (long)len - (K - 1) + j, len, c, v);
      Piece<T, V, AL>::store((T *)a.final_state + ((long)b * (K - 1) + j) * a.C + c, v);
    }
  }
}

// One workgroup: 32 pieces of channels x 8 stretches of positions of one sequence.  part: one row of (K + 1) C floats
// per (sequence, workgroup along time): the weights' sums (C, K), then the bias'.
template <typename T, int K, int V, bool AL>
__global__ __launch_bounds__(BWD_CH *BWD_SEGS) void bk_conv_backward_kernel(ConvArgs a, int nblk, int cblk, int nvec) {
  __shared__ float join[BWD_SEGS][BWD_CH][V + 1];
  const int cv = threadIdx.x % BWD_CH, sg = threadIdx.x / BWD_CH;
  const int cb = blockIdx.x % cblk;
  const long stretch = blockIdx.x / cblk;  // sequence and workgroup along time
  const int b = (int)(stretch / nblk), tb = (int)(stretch % nblk);
  const bool live = cb * BWD_CH + cv < nvec;
  const int c = piece_channel<V>(cb * BWD_CH + cv, a.C);
  const int len = row_length(a.lengths, b, a.L);
  float dw[K][V], db[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    db[i] = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) dw[k][i] = 0.0f;
  }
  const long t0 = ((long)tb * BWD_SEGS + sg) * BWD_TL;
  const long t1 = t0 + BWD_TL < a.L ? t0 + BWD_TL : a.L;
  if (live && t0 < a.L) {
    float w[K][V], bias[V], h[K][V], g[K][V];  // h: x_{t-K+1..t};  g: g_{t-K+1..t}
    Halo<T, K, V, AL> halo;
    halo.load((const T *)a.x + b * a.xb + c, a.xt, t0, a.L);
    const T *dy = (const T *)a.dy + b * a.dyb + c;
    T *dx = (T *)a.dx + (long)b * a.L * a.C + c;
    // dx of position t - K + 1 is complete once g_t is known; the first stretch also gives the carried state's gradient
    const T *x = (const T *)a.x + b * a.xb + c;
    // Positions of a block, the next one under way while this one is worked on; a multiple of K, so that the windows h and g
    // are back in the same registers behind it.
    constexpr int UNDER = K == 3 ? 6 : 4;
    struct Block {
      Piece<T, V, AL> x[UNDER], g[UNDER];
    } cur, next;
    auto fetch = [&](long from) {
#pragma unroll
      for (int j = 0; j < UNDER; ++j) {
        const long t = from + j < a.L ? from + j : a.L - 1;
        next.x[j].load(x + t * a.xt);
        next.g[j].load(dy + t * a.dyt);
      }
    };
    fetch(t0);
    load_taps<T, K, V, AL>(a, c, w, bias);
    halo.get(a, b, t0, len, c, h);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int i = 0; i < V; ++i) g[k][i] = 0.0f;
    for (long tb0 = t0; tb0 < t1 + K - 1; tb0 += UNDER) {
      cur = next;
      if (tb0 + UNDER < t1 + K - 1) fetch(tb0 + UNDER);
#pragma unroll
      for (int j = 0; j < UNDER; ++j) {
        const long t = tb0 + j;
        if (t >= t1 + K - 1) break;
        if (t < len) {
          float d[V];
          cur.x[j].get(true, h[K - 1]);
          cur.g[j].get(true, d);
#pragma unroll
          for (int i = 0; i < V; ++i) {
            if (a.silu) {
              float s = bias[i];
#pragma unroll
              for (int k = 0; k < K; ++k) s = fmaf(w[k][i], h[k][i], s);
              const float sg1 = sigmoid(s);
              d[i] *= sg1 * fmaf(s, 1.0f - sg1, 1.0f);
            }
            g[K - 1][i] = d[i];
            if (t < t1) {
              db[i] += d[i];
#pragma unroll
              for (int k = 0; k < K; ++k) dw[k][i] = fmaf(d[i], h[k][i], dw[k][i]);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) h[K - 1][i] = g[K - 1][i] = 0.0f;
        }
        const long p = t - (K - 1);  // the position that is complete now
        if (p >= t0 || (t0 == 0 && a.dinit)) {
          float o[V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            float s = 0.0f;
#pragma unroll
            for (int k = 0; k < K; ++k) s = fmaf(w[k][i], g[K - 1 - k][i], s);
            o[i] = s;
          }
          const long j = p - ((long)len - (K - 1));  // its place in the final state
          if (a.dfinal && j >= 0 && p < len) {
            float f[V];
            load_piece<T, V, AL>((const T *)a.dfinal + ((long)b * (K - 1) + j) * a.C + c, f);
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] += f[i];
          }
          if (p >= t0)
            Piece<T, V, AL>::store(dx + p * a.C, o);
          else
            Piece<T, V, AL>::store((T *)a.dinit + ((long)b * (K - 1) + (p + K - 1)) * a.C + c, o);
        }
#pragma unroll
        for (int k = 0; k < K - 1; ++k)
#pragma unroll
          for (int i = 0; i < V; ++i) {
            h[k][i] = h[k + 1][i];
            g[k][i] = g[k + 1][i];
          }
      }
    }
  }
  if (!a.part) return;
  float *out = a.part + stretch * (K + 1) * a.C;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; ++i) join[sg][cv][i] = k < K ? dw[k < K ? k : 0][i] : db[i];
    __syncthreads();
    for (int j = threadIdx.x; j < BWD_CH * V; j += BWD_CH * BWD_SEGS) {
      if (cb * BWD_CH + j / V < nvec) {
        const int col = piece_channel<V>(cb * BWD_CH + j / V, a.C) + j % V;
        float s = 0.0f;
#pragma unroll
        for (int q = 0; q < BWD_SEGS; ++q) s += join[q][j / V][j % V];
        out[k < K ? (long)col * K + k : (long)K * a.C + col] = s;
      }
    }
  }
}

// One token: the window is the state and the new input; the state moves on by one position in place.
template <typename T, int K, int V, bool AL>
__global__ __launch_bounds__(256) void bk_conv_step_kernel(ConvArgs a, T *__restrict__ state, int nvec) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)a.B * nvec) return;
  const int c = piece_channel<V>((int)(id % nvec), a.C), b = (int)(id / nvec);
  float w[K][V], bias[V], h[K][V];
  load_taps<T, K, V, AL>(a, c, w, bias);
  T *st = state + (long)b * (K - 1) * a.C + c;
#pragma unroll
  for (int k = 0; k < K - 1; ++k) load_piece<T, V, AL>(st + (long)k * a.C, h[k]);
  load_piece<T, V, AL>((const T *)a.x + b * a.xb + c, h[K - 1]);
  float o[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    float s = bias[i];
#pragma unroll
    for (int k = 0; k < K; ++k) s = fmaf(w[k][i], h[k][i], s);
    o[i] = a.silu ? s * sigmoid(s) : s;
  }
#pragma unroll
  for (int k = 0; k < K - 1; ++k) Piece<T, V, AL>::store(st + (long)k * a.C, h[k + 1]);
  Piece<T, V, AL>::store((T *)a.y + (long)b * a.C + c, o);
}

int check(int dtype, int param_dtype, int64_t B, int64_t L, int64_t C, int64_t K) {
  if (!elem_size(dtype) || (param_dtype != BKCORE_F32 && param_dtype != dtype)) return BKCORE_EINVAL;
  if (B < 0 || L < 0 || C < 0 || K < BKCORE_CONV_MIN_WIDTH || K > BKCORE_CONV_MAX_WIDTH) return BKCORE_EINVAL;
  if (B > (1 << 24) || L > (1 << 30) || C > (1 << 24)) return BKCORE_EINVAL;
  return BKCORE_OK;
}

inline int64_t backward_blocks(int64_t L) { return (L + BWD_TL * BWD_SEGS - 1) / (BWD_TL * BWD_SEGS); }

}  // namespace

#define BK_CONV_K(K, LAUNCH, V, AL)         \
  do {                                      \
    if ((K) == 2) LAUNCH(2, V, AL);         \
    else if ((K) == 3) LAUNCH(3, V, AL);    \
    else LAUNCH(4, V, AL);                  \
  } while (0)
// 16-byte pieces at 16-byte addresses, at any addresses, or single channels where there are fewer than a piece
#define BK_CONV_ANY(K, LAUNCH, V, PIECES)                             \
  do {                                                                \
    if (vec) BK_WITH_TYPE(dtype, BK_CONV_K(K, LAUNCH, V, true));      \
    else if (PIECES) BK_WITH_TYPE(dtype, BK_CONV_K(K, LAUNCH, V, false)); \
    else BK_WITH_TYPE(dtype, BK_CONV_K(K, LAUNCH, 1, false));         \
  } while (0)

extern "C" int bkcore_causal_conv(const void *x, int64_t x_batch, int64_t x_time, int dtype, const void *weight,
                                  const void *bias, int param_dtype, const void *initial_state, const int *lengths,
                                  int64_t B, int64_t L, int64_t C, int64_t K, int silu, void *y, void *final_state,
                                  void *stream) {
  const int rc = check(dtype, param_dtype, B, L, C, K);
  if (rc) return rc;
  if (B == 0 || C == 0 || (L == 0 && !final_state)) return BKCORE_OK;
  if ((L > 0 && (!x || !y)) || !weight) return BKCORE_EINVAL;
  const int v = 16 / elem_size(dtype);
  const bool vec = C % v == 0 && x_batch % v == 0 && x_time % v == 0 && aligned16(x) && aligned16(y) &&
                   aligned16(initial_state) && aligned16(final_state);
  ConvArgs a{};
  a.x = x; a.w = weight; a.bias = bias; a.init = initial_state; a.y = y; a.final_state = final_state;
  a.lengths = lengths; a.xb = x_batch; a.xt = x_time; a.B = (int)B; a.L = (int)L; a.C = (int)C;
  a.param_f32 = param_dtype == BKCORE_F32; a.param_vec = a.param_f32 && aligned16(weight); a.silu = silu != 0;
  const int64_t nseg = L > 0 ? (L + FWD_TL - 1) / FWD_TL : 1, nvec = C >= v ? (C + v - 1) / v : C;
  const int64_t blocks = (B * nseg * nvec + 255) / 256;
  if (blocks > 2147483647LL) return BKCORE_EINVAL;
#define BK_CONV(K_, V_, AL_)                                                                                            \
  hipLaunchKernelGGL((bk_conv_kernel<T, K_, V_, AL_>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, (int)nseg, \
                     (int)nvec)
  BK_CONV_ANY(K, BK_CONV, (int)(16 / sizeof(T)), C >= v);
#undef BK_CONV
  return launch_status();
}

extern "C" size_t bkcore_causal_conv_backward_workspace_bytes(int64_t B, int64_t L, int64_t C, int64_t K) {
  if (B <= 0 || L <= 0 || C <= 0 || K <= 0) return 0;
  return (size_t)B * (size_t)backward_blocks(L) * (size_t)(K + 1) * (size_t)C * sizeof(float);
}

extern "C" int bkcore_causal_conv_backward(const void *dy, int64_t dy_batch, int64_t dy_time, const void *x,
                                           int64_t x_batch, int64_t x_time, int dtype, const void *weight,
                                           const void *bias, int param_dtype, const void *initial_state,
                                           const void *grad_final_state, const int *lengths, int64_t B, int64_t L,
                                           int64_t C, int64_t K, int silu, void *dx, float *grad_params,
                                           void *grad_initial_state, void *workspace, size_t workspace_bytes,
                                           void *stream) {
  const int rc = check(dtype, param_dtype, B, L, C, K);
  if (rc) return rc;
  if (B == 0 || L == 0 || C == 0) return BKCORE_OK;
  if (!dy || !x || !weight || !dx || (grad_initial_state && !initial_state)) return BKCORE_EINVAL;
  if (grad_params && (!workspace || workspace_bytes < bkcore_causal_conv_backward_workspace_bytes(B, L, C, K)))
    return BKCORE_EWORKSPACE;
  constexpr int v = 4;  // channels a thread: eight would leave room for one wave a SIMD only
  const bool vec = C % v == 0 && x_batch % v == 0 && x_time % v == 0 && dy_batch % v == 0 && dy_time % v == 0 &&
                   aligned16(x) && aligned16(dy) && aligned16(dx) && aligned16(initial_state) &&
                   aligned16(grad_initial_state) && aligned16(grad_final_state);
  ConvArgs a{};
  a.x = x; a.w = weight; a.bias = bias; a.init = initial_state; a.dy = dy; a.dfinal = grad_final_state;
  a.dx = dx; a.dinit = grad_initial_state; a.part = grad_params ? (float *)workspace : nullptr; a.lengths = lengths;
  a.xb = x_batch; a.xt = x_time; a.dyb = dy_batch; a.dyt = dy_time; a.B = (int)B; a.L = (int)L; a.C = (int)C;
  a.param_f32 = param_dtype == BKCORE_F32; a.param_vec = a.param_f32 && aligned16(weight); a.silu = silu != 0;
  const int64_t nblk = backward_blocks(L), nvec = C >= v ? (C + v - 1) / v : C, cblk = (nvec + BWD_CH - 1) / BWD_CH;
  if (B * nblk * cblk > 2147483647LL) return BKCORE_EINVAL;
#define BK_CONV(K_, V_, AL_)                                                                                              \
  hipLaunchKernelGGL((bk_conv_backward_kernel<T, K_, V_, AL_>), dim3((unsigned)(B * nblk * cblk)), dim3(BWD_CH * BWD_SEGS), \
                     0, (hipStream_t)stream, a, (int)nblk, (int)cblk, (int)nvec)
  BK_CONV_ANY(K, BK_CONV, v, C >= v);
#undef BK_CONV
  if (grad_params) bkcore_internal_sum_parts((const float *)workspace, B * nblk, (K + 1) * C, grad_params, stream);
  return launch_status();
}

extern "C" int bkcore_causal_conv_step(const void *x, int64_t x_batch, int dtype, void *state, const void *weight,
                                       const void *bias, int param_dtype, int64_t B, int64_t C, int64_t K, int silu,
                                       void *y, void *stream) {
  const int rc = check(dtype, param_dtype, B, 1, C, K);
  if (rc) return rc;
  if (B == 0 || C == 0) return BKCORE_OK;
  if (!x || !state || !weight || !y) return BKCORE_EINVAL;
  const int v = 16 / elem_size(dtype);
  const bool vec = C % v == 0 && x_batch % v == 0 && aligned16(x) && aligned16(y) && aligned16(state);
  ConvArgs a{};
  a.x = x; a.w = weight; a.bias = bias; a.y = y; a.xb = x_batch; a.B = (int)B; a.L = 1; a.C = (int)C;
  a.param_f32 = param_dtype == BKCORE_F32; a.param_vec = a.param_f32 && aligned16(weight); a.silu = silu != 0;
  // whole pieces only: two threads on one channel would race on the state
  const int64_t nvec = C % v == 0 ? C / v : C, blocks = (B * nvec + 255) / 256;
  if (blocks > 2147483647LL) return BKCORE_EINVAL;
#define BK_CONV(K_, V_, AL_)                                                                                              \
  hipLaunchKernelGGL((bk_conv_step_kernel<T, K_, V_, AL_>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, \
                     (T *)state, (int)nvec)
  BK_CONV_ANY(K, BK_CONV, (int)(16 / sizeof(T)), C % v == 0);
#undef BK_CONV
  return launch_status();
}
