// The selective state space scan of a mixer (diagonal transition, N states a channel, channels innermost): forward,
// backward and one token.
//   d_t = softplus(delta_t + bias) (or delta_t + bias);  h_t = exp(d_t A) h_{t-1} + d_t x_t B_t
//   y_t = (C_t . h_t + D x_t) silu(z_t)
//   backward, u_t = dy_t silu(z_t):  g_t = C_t u_t + exp(d_{t+1} A) g_{t+1}   (the adjoint of h_t, from behind)
//   dx = d (g.B) + D u;   dd = x (g.B) + sum_n g h_{t-1} exp(d A) A;   dA = sum g h_{t-1} exp(d A) d;
//   dB = sum_c g d x;  dC = sum_c u h;  dD = sum u x;  dz = dy y_pre silu'(z)
// Positions at or behind a sequence's length are padding: nothing is read there, the state passes through, outputs and
// gradients are zero.
//
// What bounds it: the exponentials and the multiply-adds of the state, N a position and channel -- one v_exp_f32 (8.3
// cycles a wave) and five multiply-adds (2.4 each) -- not the 4 e (7 e backward) bytes.  A channel's states are spread over
// LPC lanes, four a lane in registers (LPC = 4 up to 16 states, 8 up to 32, 16 up to 64), so that 16 times fewer channels
// than lanes still fill the GPU; the lanes of a quad each load and prepare one of four neighbouring positions (softplus
// once, not four times) and hand it round by DPP.  B_t and C_t, shared by all channels, are staged in LDS as float32.
// When the channels of all sequences are too few to fill the GPU the time axis is cut into chunks: one launch forms
// every chunk's end state from a zero start with the sum of its d (the chunk's decay is exp(A sum d)), the next one folds
// those in front of its chunk and runs the chunk from there.
// The backward needs h at every position: the forward keeps it at every 16th (e.g. 4 bytes a position and channel for 16
// states), and a tile of 16 positions recomputes the rest into registers (the transitions twice: kept
// beside the states they would not fit: 313 us with 94 registers spilled, 158 so).
// The sums over channels (dB, dC) are folded across the wave by lane exchanges, across the workgroup's waves in LDS and
// across workgroups by a second launch; every order is fixed, results do not change from run to run.
// States, statistics and sums are float32 whatever the operands' type.
//
// Measured at 4 x 2048 positions x 1024 channels x 16 states, bf16: chunks' ends 34 us, forward 53, adjoint's ends 38,
// backward 160 (four waves a SIMD of 128 positions each: 28, 43, 31 and 123 vector instructions a position; the vector unit
// is busy 65, 76, 69 and 77 % of the time), both sums 10.  8191 positions x 512 channels f32: 20 + 37.  256 tokens x 2048
// channels: 17 us (4.2 TB/s).
#include "bkcore_types.h"

namespace {
using namespace bk;

constexpr int TILE = 16;       // positions of a tile; a checkpoint in front of each
constexpr int WAVES = 4;       // waves of a workgroup
constexpr int THREADS = 64 * WAVES;
constexpr int MAX_CHUNKS = 64; // a chunk folds all chunks in front of it by itself: 512 channels x 8191 positions 70 us
                               // with at most 32, 56 with 64, 64 with 128

struct ScanArgs {
  const void *x, *delta, *z, *Bm, *Cm, *dy;
  long xb, xt, db, dt, zb, zt, Bb, Bt, Cb, Ct, yb, yt;
  const float *A, *D, *bias, *h0, *dhT;
  const int *lengths;
  void *y, *dx, *ddelta, *dz;
  float *hT, *dh0, *ckpt, *agg, *aggd, *part_bc, *part_par;
  int B, L, C, N, softplus, chunk, S, nct;
};

__device__ __forceinline__ int row_length(const int *lengths, int b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

// Sum over the LPC lanes of a channel, in each of them.
template <int LPC>
__device__ __forceinline__ float sum_states(float v) {
  v += dpp_mov<DPP_XOR1>(v);
  v += dpp_mov<DPP_XOR2>(v);
  if constexpr (LPC >= 8) v += dpp_mov<DPP_HALF_MIRROR>(v);
  if constexpr (LPC >= 16) v += dpp_mov<DPP_MIRROR>(v);
  return v;
}

// A state behind a chunk: a h + e.  Where d A is positive a chunk's factor may be beyond float32 although no position's is; a
// state that is still zero stays zero then, as it does position by position.
__device__ __forceinline__ float decayed(float a, float h, float e) { return h == 0.0f ? e : fmaf(a, h, e); }

// The value of lane Q of each quad.
// (The empty asm keeps the move a move: folded into its eight users it would make each of them a DPP instruction at 4.3
// cycles instead of 2.4.)
template <int Q>
__device__ __forceinline__ float quad_get(float v) {
  float r = dpp_mov<Q * 0x55>(v);
  asm("" : "+v"(r));
  return r;
}

// log(1 + e^p): with u = 1 + e^p the correction e^p / (u - 1) keeps the relative accuracy where e^p is small; from 20 on
// it is p to the last bit.
__device__ __forceinline__ float softplus(float p) {
  const float e = exp2_fast(p * LOG2E), u = 1.0f + e;
  const float l = __builtin_amdgcn_logf(u) * (1.0f / LOG2E);
  const float s = u == 1.0f ? e : l * (e * __builtin_amdgcn_rcpf(u - 1.0f));
  return p > 20.0f ? p : s;
}

template <typename T>
__device__ __forceinline__ float at(const void *p, long i) {
  return (float)((const T *)p)[i];
}

// Which workgroup does what: channel tile fastest, so that neighbouring workgroups read neighbouring channels.
struct Place {
  int ct, b, s;
  __device__ __forceinline__ Place(const ScanArgs &a) {
    ct = blockIdx.x % a.nct;
    const unsigned r = blockIdx.x / a.nct;
    b = r % a.B;
    s = r / a.B;
  }
};

// B_t, C_t of a tile on their way to LDS: N padded to NP = 4 LPC states with zeros.  Loads are unconditional (from the
// nearest valid place) and stay in the operands' type until they are used: a load under a condition, or converted where it
// is issued, would be waited for at once.
template <typename T, int LPC>
struct StateRows {
  static constexpr int NP = 4 * LPC;
  static constexpr int PER = TILE * NP / THREADS;
  T b[PER], c[PER];
  __device__ __forceinline__ void load(const ScanArgs &a, int bi, long t0, long stop, bool want_b, bool want_c) {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = threadIdx.x + k * THREADS, n = i % NP;
      const unsigned t = min((unsigned)(i / NP), (unsigned)(stop - 1 - t0 < TILE ? stop - 1 - t0 : TILE));
      const unsigned nn = n < a.N ? n : 0;
      if (want_b) b[k] = ((const T *)a.Bm + bi * a.Bb + t0 * a.Bt)[t * (unsigned)a.Bt + nn];
      if (want_c) c[k] = ((const T *)a.Cm + bi * a.Cb + t0 * a.Ct)[t * (unsigned)a.Ct + nn];
    }
  }
  __device__ __forceinline__ void store(const ScanArgs &a, long t0, long stop, float *sb, float *sc) const {
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = threadIdx.x + k * THREADS;
      const bool in = t0 + i / NP < stop && i % NP < a.N;
      if (sb) sb[i] = in ? (float)b[k] : 0.0f;
      if (sc) sc[i] = in ? (float)c[k] : 0.0f;
    }
  }
};

// Four positions of a lane's quad (t0 + 4 i + q) of a (B, L, C) operand, in its own type.  The address is a uniform
// 64-bit base of the tile and a 32-bit offset inside it (the host keeps 16 strides below 2^31), which saves the register
// pairs that full addresses would take.
template <typename T>
struct Column {
  const T *p;
  long step;
  T v[4];
  __device__ __forceinline__ Column(const void *base, long off, long step_) : p((const T *)base + off), step(step_) {}
  __device__ __forceinline__ void load(long t0, int q, int c, long stop) {
    const T *tile = p + t0 * step;
    const unsigned most = (unsigned)(stop - 1 - t0 < TILE ? stop - 1 - t0 : TILE), st = (unsigned)step;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned t = min((unsigned)(4 * i + q), most);
      v[i] = tile[t * st + (unsigned)c];
    }
  }
};

// AGG: the chunk's end state from a zero start and the sum of its d, for all chunks but the last.
template <typename T, int LPC, bool AGG>
__global__ __launch_bounds__(THREADS) void bk_scan_kernel(ScanArgs a) {
  constexpr int NP = 4 * LPC, CPW = 64 / LPC;
  __shared__ float sB[2][TILE * NP], sC[2][TILE * NP];
  const Place at_(a);
  const int b = at_.b, s = at_.s, lane = threadIdx.x & 63, sub = lane % LPC, q = lane & 3;
  const int c = (at_.ct * WAVES + (threadIdx.x >> 6)) * CPW + lane / LPC;
  const bool live = c < a.C;
  const int len = row_length(a.lengths, b, a.L);
  const long begin = (long)s * a.chunk, end = begin + a.chunk < a.L ? begin + a.chunk : a.L;
  const long stop = end < len ? end : len;  // positions from here to `end` are padding
  float A2[4], h[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int k = sub * 4 + n;
    A2[n] = live && k < a.N ? a.A[(long)c * a.N + k] * LOG2E : 0.0f;
    h[n] = !AGG && live && k < a.N && a.h0 ? a.h0[((long)b * a.C + c) * a.N + k] : 0.0f;
  }
  const float skip = live && a.D ? a.D[c] : 0.0f, bias = live && a.bias ? a.bias[c] : 0.0f;
  if (!AGG && live) {
#pragma unroll 8
    for (int j = 0; j < s; ++j) {
      const long at0 = ((long)j * a.B + b) * a.C + c;
      const float sd = a.aggd[at0];
      const f32x4 e = *reinterpret_cast<const f32x4 *>(a.agg + at0 * NP + sub * 4);
#pragma unroll
      for (int n = 0; n < 4; ++n) h[n] = decayed(exp2_fast(A2[n] * sd), h[n], e[n]);
    }
  }
  float sum_d = 0.0f;
  const int cc = live ? c : a.C - 1;
  Column<T> xr(a.x, b * a.xb, a.xt), dr(a.delta, b * a.db, a.dt), zr(a.z, b * a.zb, a.zt);
  StateRows<T, LPC> rows;
  auto prefetch = [&](long t0) {
    xr.load(t0, q, cc, stop);
    dr.load(t0, q, cc, stop);
    if (!AGG && a.z) zr.load(t0, q, cc, stop);
    rows.load(a, b, t0, stop, true, !AGG);
  };
  if (begin < stop) prefetch(begin);
  int buf = 0;
  for (long t0 = begin; t0 < stop; t0 += TILE, buf ^= 1) {
    float xv[4], dv[4], zv[4], ux[4], yv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = live && t0 + 4 * i + q < stop;
      xv[i] = in ? (float)xr.v[i] : 0.0f;
      if (!AGG) zv[i] = in && a.z ? (float)zr.v[i] : 0.0f;
      const float p = (float)dr.v[i] + bias;
      dv[i] = in ? (a.softplus ? softplus(p) : p) : 0.0f;
      ux[i] = dv[i] * xv[i];
      if (AGG) sum_d += dv[i];
      yv[i] = 0.0f;
    }
    rows.store(a, t0, stop, sB[buf], AGG ? nullptr : sC[buf]);
    __syncthreads();
    if (t0 + TILE < stop) prefetch(t0 + TILE);
    if (!AGG && a.ckpt && live) {
      f32x4 k;
#pragma unroll
      for (int n = 0; n < 4; ++n) k[n] = h[n];
      const long tile = t0 / TILE, ntiles = (a.L + TILE - 1) / TILE;
      *reinterpret_cast<f32x4 *>(a.ckpt + (b * ntiles + tile) * a.C * NP + (unsigned)(c * NP + sub * 4)) = k;
    }
#define BK_STEP(i, Q)                                                                            \
  do {                                                                                           \
    const float d = quad_get<Q>(dv[i]), u = quad_get<Q>(ux[i]);                                  \
    const f32x4 Bv = *reinterpret_cast<const f32x4 *>(&sB[buf][(4 * i + Q) * NP + sub * 4]);     \
    _Pragma("unroll") for (int n = 0; n < 4; ++n)                                                \
        h[n] = fmaf(exp2_fast(d * A2[n]), h[n], u * Bv[n]);                                      \
    if (!AGG) {                                                                                  \
      const f32x4 Cv = *reinterpret_cast<const f32x4 *>(&sC[buf][(4 * i + Q) * NP + sub * 4]);   \
      float y = h[0] * Cv[0];                                                                    \
      _Pragma("unroll") for (int n = 1; n < 4; ++n) y = fmaf(h[n], Cv[n], y);                    \
      y = sum_states<LPC>(y);                                                                    \
      if (q == Q) yv[i] = y;                                                                     \
    }                                                                                            \
  } while (0)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      BK_STEP(i, 0);
      BK_STEP(i, 1);
      BK_STEP(i, 2);
      BK_STEP(i, 3);
    }
#undef BK_STEP
    if (!AGG && live && sub < 4) {
      T *out = (T *)a.y + ((long)b * a.L + t0) * a.C;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long t = t0 + 4 * i + q;
        if (t < end) {
          float y = fmaf(skip, xv[i], yv[i]);
          if (a.z) y *= zv[i] * sigmoid(zv[i]);
          out[(unsigned)((4 * i + q) * a.C + c)] = (T)(t < stop ? y : 0.0f);
        }
      }
    }
  }
  if (AGG) {
    if (live) {
      const long at0 = ((long)s * a.B + b) * a.C + c;
      f32x4 k;
#pragma unroll
      for (int n = 0; n < 4; ++n) k[n] = h[n];
      *reinterpret_cast<f32x4 *>(a.agg + at0 * NP + sub * 4) = k;
      sum_d += dpp_mov<DPP_XOR1>(sum_d);  // the quad's lanes hold a position each; every quad of a channel holds them all
      sum_d += dpp_mov<DPP_XOR2>(sum_d);
      if (sub == 0) a.aggd[at0] = sum_d;
    }
    return;
  }
  // whole tiles behind the length (the last tile that holds a position of the sequence zeroed its own padding)
  const long done = stop > begin ? begin + (stop - begin + TILE - 1) / TILE * TILE : begin;
  if (live && sub < 4)
    for (long t = done + q; t < end; t += 4) ((T *)a.y)[((long)b * a.L + t) * a.C + c] = (T)0.0f;
  if (a.hT && live && s == a.S - 1) {
#pragma unroll
    for (int n = 0; n < 4; ++n)
      if (sub * 4 + n < a.N) a.hT[((long)b * a.C + c) * a.N + sub * 4 + n] = h[n];
  }
}

// The adjoint's end of a chunk from a zero start behind it, and the sum of the chunk's d, for all chunks but the first.
template <typename T, int LPC>
__global__ __launch_bounds__(THREADS) void bk_scan_adjoint_agg_kernel(ScanArgs a) {
  constexpr int NP = 4 * LPC, CPW = 64 / LPC;
  __shared__ float sC[2][TILE * NP];
  const Place at_(a);
  const int b = at_.b, s = at_.s + 1, lane = threadIdx.x & 63, sub = lane % LPC, q = lane & 3;
  const int c = (at_.ct * WAVES + (threadIdx.x >> 6)) * CPW + lane / LPC;
  const bool live = c < a.C;
  const int len = row_length(a.lengths, b, a.L);
  const long begin = (long)s * a.chunk, end = begin + a.chunk < a.L ? begin + a.chunk : a.L;
  const long stop = end < len ? end : len;
  float A2[4], carry[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int k = sub * 4 + n;
    A2[n] = live && k < a.N ? a.A[(long)c * a.N + k] * LOG2E : 0.0f;
    carry[n] = 0.0f;
  }
  const float bias = live && a.bias ? a.bias[c] : 0.0f;
  float sum_d = 0.0f;
  const int cc = live ? c : a.C - 1;
  Column<T> dr(a.delta, b * a.db, a.dt), gr(a.dy, b * a.yb, a.yt), zr(a.z, b * a.zb, a.zt);
  StateRows<T, LPC> rows;
  auto prefetch = [&](long t0) {
    dr.load(t0, q, cc, stop);
    gr.load(t0, q, cc, stop);
    if (a.z) zr.load(t0, q, cc, stop);
    rows.load(a, b, t0, stop, false, true);
  };
  const long last = begin + (stop - begin + TILE - 1) / TILE * TILE - TILE;
  if (begin < stop) prefetch(last);
  int buf = 0;
  for (long t0 = last; begin < stop && t0 >= begin; t0 -= TILE, buf ^= 1) {
    float dv[4], uv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = live && t0 + 4 * i + q < stop;
      const float p = (float)dr.v[i] + bias, g = in ? (float)gr.v[i] : 0.0f, z = in && a.z ? (float)zr.v[i] : 0.0f;
      dv[i] = in ? (a.softplus ? softplus(p) : p) : 0.0f;
      uv[i] = a.z ? g * (z * sigmoid(z)) : g;
      sum_d += dv[i];
    }
    rows.store(a, t0, stop, nullptr, sC[buf]);
    __syncthreads();
    if (t0 - TILE >= begin) prefetch(t0 - TILE);
#define BK_STEP(i, Q)                                                                            \
  do {                                                                                           \
    const float d = quad_get<Q>(dv[i]), u = quad_get<Q>(uv[i]);                                  \
    const f32x4 Cv = *reinterpret_cast<const f32x4 *>(&sC[buf][(4 * i + Q) * NP + sub * 4]);     \
    _Pragma("unroll") for (int n = 0; n < 4; ++n)                                                \
        carry[n] = fmaf(u, Cv[n], carry[n]) * exp2_fast(d * A2[n]);                              \
  } while (0)
#pragma unroll
    for (int i = 3; i >= 0; --i) {
      BK_STEP(i, 3);
      BK_STEP(i, 2);
      BK_STEP(i, 1);
      BK_STEP(i, 0);
    }
#undef BK_STEP
  }
  if (live) {
    const long at0 = ((long)s * a.B + b) * a.C + c;
    f32x4 k;
#pragma unroll
    for (int n = 0; n < 4; ++n) k[n] = carry[n];
    *reinterpret_cast<f32x4 *>(a.agg + at0 * NP + sub * 4) = k;
    sum_d += dpp_mov<DPP_XOR1>(sum_d);
    sum_d += dpp_mov<DPP_XOR2>(sum_d);
    if (sub == 0) a.aggd[at0] = sum_d;
  }
}

// part_bc: (channel tile, sequence, position, 2 NP) sums of dB then dC over the tile's channels.
// part_par: (chunk, sequence) rows of C N + 2 C floats: dA, dD, d bias.
template <typename T, int LPC>
__global__ __launch_bounds__(THREADS, 2) void bk_scan_backward_kernel(ScanArgs a) {
  constexpr int NP = 4 * LPC, CPW = 64 / LPC, GRP = 16 / LPC;
  __shared__ float sB[2][TILE * NP], sC[2][TILE * NP], red[WAVES][TILE * 2 * NP];
  const Place at_(a);
  const int b = at_.b, s = at_.s, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPC, q = lane & 3;
  const int c = (at_.ct * WAVES + wave) * CPW + lane / LPC;
  const bool live = c < a.C;
  const int len = row_length(a.lengths, b, a.L);
  const long begin = (long)s * a.chunk, end = begin + a.chunk < a.L ? begin + a.chunk : a.L;
  const long stop = end < len ? end : len;
  const int row = lane >> 4, grp = (lane & 15) / LPC;
  const int fold_state = sub * 4 + (((row & 1) << 1) | (row >> 1));  // the state whose sum the folds leave in this lane
  float A2[4], carry[4], dA[4], dD = 0.0f, dbias = 0.0f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int k = sub * 4 + n;
    A2[n] = live && k < a.N ? a.A[(long)c * a.N + k] * LOG2E : 0.0f;
    carry[n] = live && k < a.N && a.dhT ? a.dhT[((long)b * a.C + c) * a.N + k] : 0.0f;
    dA[n] = 0.0f;
  }
  const float skip = live && a.D ? a.D[c] : 0.0f, bias = live && a.bias ? a.bias[c] : 0.0f;
  if (live) {
#pragma unroll 8
    for (int j = a.S - 1; j > s; --j) {
      const long at0 = ((long)j * a.B + b) * a.C + c;
      const float sd = a.aggd[at0];
      const f32x4 e = *reinterpret_cast<const f32x4 *>(a.agg + at0 * NP + sub * 4);
#pragma unroll
      for (int n = 0; n < 4; ++n) carry[n] = decayed(exp2_fast(A2[n] * sd), carry[n], e[n]);
    }
  }
  const long ntiles = (a.L + TILE - 1) / TILE;
  const int cc = live ? c : a.C - 1;
  Column<T> xr(a.x, b * a.xb, a.xt), dr(a.delta, b * a.db, a.dt), gr(a.dy, b * a.yb, a.yt), zr(a.z, b * a.zb, a.zt);
  f32x4 hr;
  StateRows<T, LPC> rows;
  auto prefetch = [&](long t0) {
    xr.load(t0, q, cc, stop);
    dr.load(t0, q, cc, stop);
    gr.load(t0, q, cc, stop);
    if (a.z) zr.load(t0, q, cc, stop);
    hr = *reinterpret_cast<const f32x4 *>(a.ckpt + (b * ntiles + t0 / TILE) * a.C * NP + (unsigned)(cc * NP + sub * 4));
    rows.load(a, b, t0, stop, true, true);
  };
  const long last = begin + (stop - begin + TILE - 1) / TILE * TILE - TILE;
  if (begin < stop) prefetch(last);
  int buf = 0;
  for (long t0 = last; begin < stop && t0 >= begin; t0 -= TILE, buf ^= 1) {
    float xv[4], dv[4], pv[4], uv[4], gv[4], ux[4], yv[4], gb[4], sa[4], zv[4];
    float h0[4], h[TILE][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) h0[n] = live ? hr[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool in = live && t0 + 4 * i + q < stop;
      xv[i] = in ? (float)xr.v[i] : 0.0f;
      zv[i] = in && a.z ? (float)zr.v[i] : 0.0f;
      gv[i] = in ? (float)gr.v[i] : 0.0f;
      pv[i] = (float)dr.v[i] + bias;
      dv[i] = in ? (a.softplus ? softplus(pv[i]) : pv[i]) : 0.0f;
      ux[i] = dv[i] * xv[i];
      uv[i] = a.z ? gv[i] * (zv[i] * sigmoid(zv[i])) : gv[i];
      yv[i] = gb[i] = sa[i] = 0.0f;
    }
    rows.store(a, t0, stop, sB[buf], sC[buf]);
    __syncthreads();
    if (t0 - TILE >= begin) prefetch(t0 - TILE);
#define BK_STEP(i, Q)                                                                            \
  do {                                                                                           \
    constexpr int t_ = 4 * (i) + Q;                                                              \
    const float d = quad_get<Q>(dv[i]), u = quad_get<Q>(ux[i]);                                  \
    const f32x4 Bv = *reinterpret_cast<const f32x4 *>(&sB[buf][t_ * NP + sub * 4]);              \
    float y = 0.0f;                                                                              \
    const f32x4 Cv = *reinterpret_cast<const f32x4 *>(&sC[buf][t_ * NP + sub * 4]);              \
    _Pragma("unroll") for (int n = 0; n < 4; ++n) {                                              \
      h[t_][n] = fmaf(exp2_fast(d * A2[n]), t_ ? h[t_ ? t_ - 1 : 0][n] : h0[n], u * Bv[n]);      \
      y = fmaf(h[t_][n], Cv[n], y);                                                              \
    }                                                                                            \
    if (a.z) {                                                                                   \
      y = sum_states<LPC>(y);                                                                    \
      if (q == Q) yv[i] = y;                                                                     \
    }                                                                                            \
  } while (0)
// The barriers keep the scheduler from raising the LDS reads of all sixteen positions to the top, which spills.
#define BK_STEPS(i) BK_STEP(i, 0); BK_STEP(i, 1); BK_STEP(i, 2); BK_STEP(i, 3); __builtin_amdgcn_sched_barrier(0)
    BK_STEPS(0);
    BK_STEPS(1);
    BK_STEPS(2);
    BK_STEPS(3);
#undef BK_STEPS
#undef BK_STEP
    // The transitions are formed again in the way back: the compiler would keep the first ones (64 registers) and spill.
    float A2r[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      A2r[n] = A2[n];
      asm volatile("" : "+v"(A2r[n]));
    }
    float pair[4];  // (position, dB or dC) sums of two positions, waiting to be written together
#define BK_STEP(i, Q)                                                                            \
  do {                                                                                           \
    constexpr int t_ = 4 * (i) + Q;                                                              \
    const float d = quad_get<Q>(dv[i]), ud = quad_get<Q>(ux[i]), u = quad_get<Q>(uv[i]);         \
    const f32x4 Bv = *reinterpret_cast<const f32x4 *>(&sB[buf][t_ * NP + sub * 4]);              \
    const f32x4 Cv = *reinterpret_cast<const f32x4 *>(&sC[buf][t_ * NP + sub * 4]);              \
    float vB[4], vC[4], gB = 0.0f, sA = 0.0f;                                                    \
    _Pragma("unroll") for (int n = 0; n < 4; ++n) {                                              \
      const float g = fmaf(u, Cv[n], carry[n]);                                                  \
      vC[n] = u * h[t_][n];                                                                      \
      vB[n] = g * ud;                                                                            \
      gB = fmaf(g, Bv[n], gB);                                                                   \
      carry[n] = g * exp2_fast(d * A2r[n]);                                                      \
      const float eh = carry[n] * (t_ ? h[t_ ? t_ - 1 : 0][n] : h0[n]);                          \
      sA = fmaf(eh, A2[n], sA);                                                                  \
      dA[n] = fmaf(eh, d, dA[n]);                                                                \
    }                                                                                            \
    gB = sum_states<LPC>(gB);                                                                    \
    sA = sum_states<LPC>(sA);                                                                    \
    if (q == Q) {                                                                                \
      gb[i] = gB;                                                                                \
      sa[i] = sA;                                                                                \
    }                                                                                            \
    constexpr int k_ = 2 * (t_ & 1);                                                             \
    pair[k_] = fold16(fold32(vB[0], vB[1]), fold32(vB[2], vB[3]));                               \
    pair[k_ + 1] = fold16(fold32(vC[0], vC[1]), fold32(vC[2], vC[3]));                           \
    _Pragma("unroll") for (int k = k_; k < k_ + 2; ++k) {                                        \
      if (LPC <= 4) pair[k] += dpp_mov<DPP_ROR4>(pair[k]);                                       \
      if (LPC <= 8) pair[k] += dpp_mov<DPP_ROR8>(pair[k]);                                       \
    }                                                                                            \
    if (k_ == 0) {                                                                               \
      _Pragma("unroll") for (int k = 0; k < 4; k += GRP) {                                       \
        float v = pair[k];                                                                       \
        _Pragma("unroll") for (int m = 1; m < GRP; ++m) v = grp == m ? pair[k + m] : v;          \
        const int kk = k + grp;                                                                  \
        red[wave][(t_ + (kk >> 1)) * 2 * NP + (kk & 1) * NP + fold_state] = v;                   \
      }                                                                                          \
    }                                                                                            \
  } while (0)
// The sums over positions are pinned to their place: sunk behind the tile they would keep all 64 of their terms alive.
#define BK_STEPS(i)                                                                              \
  BK_STEP(i, 3); BK_STEP(i, 2); BK_STEP(i, 1); BK_STEP(i, 0);                                    \
  asm volatile("" : "+v"(dA[0]), "+v"(dA[1]), "+v"(dA[2]), "+v"(dA[3]));                        \
  __builtin_amdgcn_sched_barrier(0)
    BK_STEPS(3);
    BK_STEPS(2);
    BK_STEPS(1);
    BK_STEPS(0);
#undef BK_STEPS
#undef BK_STEP
    if (live && sub < 4) {
      const long tile = ((long)b * a.L + t0) * a.C;
      T *dx = (T *)a.dx + tile, *ddl = (T *)a.ddelta + tile, *dzo = a.z ? (T *)a.dz + tile : nullptr;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const long t = t0 + 4 * i + q;
        if (t < end) {
          const bool in = t < stop;
          const unsigned o = (unsigned)((4 * i + q) * a.C + c);
          const float dxo = fmaf(dv[i], gb[i], skip * uv[i]);
          float dd = fmaf(xv[i], gb[i], sa[i] * (1.0f / LOG2E));
          if (a.softplus) dd *= pv[i] > 20.0f ? 1.0f : sigmoid(pv[i]);
          dx[o] = (T)(in ? dxo : 0.0f);
          ddl[o] = (T)(in ? dd : 0.0f);
          if (a.z) {
            const float sg = sigmoid(zv[i]);
            const float dz = gv[i] * fmaf(skip, xv[i], yv[i]) * (sg * fmaf(zv[i], 1.0f - sg, 1.0f));
            dzo[o] = (T)(in ? dz : 0.0f);
          }
          if (in) {
            dD = fmaf(uv[i], xv[i], dD);
            dbias += dd;
          }
        }
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < TILE * 2 * NP; i += THREADS) {
      const long t = t0 + i / (2 * NP);
      if (t < stop)
        a.part_bc[(((long)at_.ct * a.B + b) * a.L + t) * (2 * NP) + i % (2 * NP)] =
            red[0][i] + red[1][i] + red[2][i] + red[3][i];
    }
  }
  const long done = stop > begin ? begin + (stop - begin + TILE - 1) / TILE * TILE : begin;
  if (live && sub < 4)
    for (long t = done + q; t < end; t += 4) {
      const long o = ((long)b * a.L + t) * a.C + c;
      ((T *)a.dx)[o] = (T)0.0f;
      ((T *)a.ddelta)[o] = (T)0.0f;
      if (a.z) ((T *)a.dz)[o] = (T)0.0f;
    }
  dD += dpp_mov<DPP_XOR1>(dD);
  dD += dpp_mov<DPP_XOR2>(dD);
  dbias += dpp_mov<DPP_XOR1>(dbias);
  dbias += dpp_mov<DPP_XOR2>(dbias);
  if (live) {
    float *p = a.part_par + ((long)s * a.B + b) * ((long)a.C * a.N + 2 * a.C);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int k = sub * 4 + n;
      if (k < a.N) {
        p[(long)c * a.N + k] = dA[n];
        if (a.dh0 && s == 0) a.dh0[((long)b * a.C + c) * a.N + k] = carry[n];
      }
    }
    if (sub == 0) {
      p[(long)a.C * a.N + c] = dD;
      p[(long)a.C * a.N + a.C + c] = dbias;
    }
  }
}

// dB, dC from the channel tiles' sums, rounded to the operands' type; zero behind the length.
template <typename T>
__global__ __launch_bounds__(256) void bk_scan_sum_bc_kernel(const float *__restrict__ part, const int *lengths, int nct,
                                                             int B, int L, int N, int NP, T *__restrict__ dB,
                                                             T *__restrict__ dC) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x, per = (long)B * L * 2 * NP;
  if (id >= per) return;
  const int k = (int)(id % (2 * NP)), n = k % NP;
  const long bt = id / (2 * NP);
  if (n >= N) return;
  float s = 0.0f;
  if (bt % L < row_length(lengths, (int)(bt / L), L)) {
#pragma unroll 4
    for (int p = 0; p < nct; ++p) s += part[p * per + id];
  }
  (k < NP ? dB : dC)[bt * N + n] = (T)s;
}

// One token: four states a thread; the state is read and written once.
template <typename T>
__global__ __launch_bounds__(256) void bk_scan_step_kernel(ScanArgs a, float *__restrict__ state, int lpc) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  const int sub = (int)(id % lpc);
  const long bc = id / lpc;
  const bool live = bc < (long)a.B * a.C;
  const int b = live ? (int)(bc / a.C) : 0, c = live ? (int)(bc % a.C) : 0;
  float y = 0.0f, x = 0.0f;
  if (live) {
    x = at<T>(a.x, b * a.xb + c);
    float d = at<T>(a.delta, b * a.db + c) + (a.bias ? a.bias[c] : 0.0f);
    if (a.softplus) d = softplus(d);
    const float u = d * x;
    float *h = state + bc * a.N + sub * 4;
    const float *A = a.A + (long)c * a.N + sub * 4;
    if (a.N % 4 == 0) {
      if (sub * 4 < a.N) {
        f32x4 v = *reinterpret_cast<const f32x4 *>(h);
        const f32x4 Av = *reinterpret_cast<const f32x4 *>(A);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int k = sub * 4 + n;
          v[n] = fmaf(exp2_fast(d * (Av[n] * LOG2E)), v[n], u * at<T>(a.Bm, b * a.Bb + k));
          y = fmaf(v[n], at<T>(a.Cm, b * a.Cb + k), y);
        }
        *reinterpret_cast<f32x4 *>(h) = v;
      }
    } else {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int k = sub * 4 + n;
        if (k < a.N) {
          const float v = fmaf(exp2_fast(d * (A[n] * LOG2E)), h[n], u * at<T>(a.Bm, b * a.Bb + k));
          y = fmaf(v, at<T>(a.Cm, b * a.Cb + k), y);
          h[n] = v;
        }
      }
    }
  }
  // lpc is 4, 8 or 16: a channel's lanes are neighbours inside a row of 16
  y = sum_states<4>(y);
  if (lpc >= 8) y += dpp_mov<DPP_HALF_MIRROR>(y);
  if (lpc >= 16) y += dpp_mov<DPP_MIRROR>(y);
  if (live && sub == 0) {
    if (a.D) y = fmaf(a.D[c], x, y);
    if (a.z) {
      const float z = at<T>(a.z, b * a.zb + c);
      y *= z * sigmoid(z);
    }
    ((T *)a.y)[bc] = (T)y;
  }
}

inline int lanes_per_channel(int64_t N) { return N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Chunks of the time axis: one while the channels alone give every SIMD a wave (cutting adds a pass over the inputs),
// else enough for four waves a SIMD, of at least four tiles each (4 x 2048 positions x 1024 channels, 256 waves uncut, both
// launches of the forward: 97 us at two waves a SIMD, 86 at four, 95 at six; other numbers of channels are not measured).
struct Plan {
  int lpc, nct, S, chunk;
};
inline Plan plan(int64_t B, int64_t L, int64_t C, int64_t N) {
  Plan p;
  p.lpc = lanes_per_channel(N);
  const int64_t per = 64 / p.lpc * WAVES;  // channels of a workgroup
  p.nct = (int)((C + per - 1) / per);
  const int64_t waves = B * p.nct * WAVES;
  int64_t S = 1;
  if (waves < 1024) {
    S = 4096 / (waves > 0 ? waves : 1);
    const int64_t most = L / (4 * TILE);
    if (S > most) S = most;
    if (S > MAX_CHUNKS) S = MAX_CHUNKS;
    if (S < 1) S = 1;
  }
  int64_t chunk = (L + S - 1) / S;
  chunk = (chunk + TILE - 1) / TILE * TILE;
  if (chunk < TILE) chunk = TILE;
  p.chunk = (int)chunk;
  p.S = (int)((L + chunk - 1) / chunk);
  if (p.S < 1) p.S = 1;
  return p;
}

int check(int dtype, int64_t B, int64_t L, int64_t C, int64_t N) {
  if (!elem_size(dtype)) return BKCORE_EINVAL;
  if (B < 0 || L < 0 || C < 0 || N < 1 || N > BKCORE_SCAN_MAX_STATE) return BKCORE_EINVAL;
  if (B > (1 << 24) || L > (1 << 30) || C > (1 << 24)) return BKCORE_EINVAL;
  return BKCORE_OK;
}

// 16 positions of an operand within 32-bit offsets
inline bool near(int64_t time_stride) { return time_stride >= 0 && time_stride < (1LL << 26); }

inline size_t agg_floats(const Plan &p, int64_t B, int64_t C) {
  return p.S > 1 ? (size_t)p.S * B * C * (4 * p.lpc + 1) : 0;
}
inline size_t round4(size_t n) { return (n + 3) & ~(size_t)3; }

#define BK_SCAN_LPC(lpc, LAUNCH)     \
  do {                               \
    if ((lpc) == 4) LAUNCH(4);       \
    else if ((lpc) == 8) LAUNCH(8);  \
    else LAUNCH(16);                 \
  } while (0)

}  // namespace

extern "C" size_t bkcore_selective_scan_workspace_bytes(int64_t B, int64_t L, int64_t C, int64_t N) {
  if (B <= 0 || L <= 0 || C <= 0 || N < 1 || N > BKCORE_SCAN_MAX_STATE) return 0;
  return agg_floats(plan(B, L, C, N), B, C) * sizeof(float);
}

extern "C" size_t bkcore_selective_scan_checkpoint_bytes(int64_t B, int64_t L, int64_t C, int64_t N) {
  if (B <= 0 || L <= 0 || C <= 0 || N < 1 || N > BKCORE_SCAN_MAX_STATE) return 0;
  return (size_t)B * ((L + TILE - 1) / TILE) * C * (4 * lanes_per_channel(N)) * sizeof(float);
}

extern "C" int bkcore_selective_scan(const void *x, int64_t x_batch, int64_t x_time, const void *delta,
                                     int64_t delta_batch, int64_t delta_time, const float *A, const void *Bm,
                                     int64_t B_batch, int64_t B_time, const void *Cm, int64_t C_batch, int64_t C_time,
                                     const float *D, const void *z, int64_t z_batch, int64_t z_time,
                                     const float *delta_bias, int softplus_delta, int dtype, const int *lengths,
                                     const float *initial_state, int64_t B, int64_t L, int64_t C, int64_t N, void *y,
                                     float *final_state, float *checkpoints, void *workspace, size_t workspace_bytes,
                                     void *stream) {
  const int rc = check(dtype, B, L, C, N);
  if (rc) return rc;
  if (B == 0 || C == 0 || L == 0) return BKCORE_OK;
  if (!x || !delta || !A || !Bm || !Cm || !y) return BKCORE_EINVAL;
  if (!near(x_time) || !near(delta_time) || !near(B_time) || !near(C_time) || (z && !near(z_time))) return BKCORE_EINVAL;
  const Plan p = plan(B, L, C, N);
  if (p.S > 1 && (!workspace || workspace_bytes < bkcore_selective_scan_workspace_bytes(B, L, C, N)))
    return BKCORE_EWORKSPACE;
  if ((int64_t)p.nct * B * p.S > 2147483647LL) return BKCORE_EINVAL;
  ScanArgs a{};
  a.x = x; a.xb = x_batch; a.xt = x_time; a.delta = delta; a.db = delta_batch; a.dt = delta_time; a.A = A;
  a.Bm = Bm; a.Bb = B_batch; a.Bt = B_time; a.Cm = Cm; a.Cb = C_batch; a.Ct = C_time; a.D = D;
  a.z = z; a.zb = z_batch; a.zt = z_time; a.bias = delta_bias; a.softplus = softplus_delta != 0; a.lengths = lengths;
  a.h0 = initial_state; a.y = y; a.hT = final_state; a.ckpt = checkpoints;
  a.agg = (float *)workspace;
  a.aggd = a.agg ? a.agg + (size_t)p.S * B * C * (4 * p.lpc) : nullptr;
  a.B = (int)B; a.L = (int)L; a.C = (int)C; a.N = (int)N; a.chunk = p.chunk; a.S = p.S; a.nct = p.nct;
  const unsigned grid = (unsigned)(p.nct * B * p.S), grid_agg = (unsigned)(p.nct * B * (p.S - 1));
  hipStream_t s = (hipStream_t)stream;
#define BK_AGG(LPC) hipLaunchKernelGGL((bk_scan_kernel<T, LPC, true>), dim3(grid_agg), dim3(THREADS), 0, s, a)
#define BK_MAIN(LPC) hipLaunchKernelGGL((bk_scan_kernel<T, LPC, false>), dim3(grid), dim3(THREADS), 0, s, a)
  if (p.S > 1) BK_WITH_TYPE(dtype, BK_SCAN_LPC(p.lpc, BK_AGG));
  BK_WITH_TYPE(dtype, BK_SCAN_LPC(p.lpc, BK_MAIN));
#undef BK_AGG
#undef BK_MAIN
  return launch_status();
}

extern "C" size_t bkcore_selective_scan_backward_workspace_bytes(int64_t B, int64_t L, int64_t C, int64_t N) {
  if (B <= 0 || L <= 0 || C <= 0 || N < 1 || N > BKCORE_SCAN_MAX_STATE) return 0;
  const Plan p = plan(B, L, C, N);
  const size_t bc = (size_t)p.nct * B * L * 2 * (4 * p.lpc);
  const size_t par = (size_t)p.S * B * ((size_t)C * N + 2 * C);
  return (round4(agg_floats(p, B, C)) + round4(bc) + par) * sizeof(float);
}

extern "C" int bkcore_selective_scan_backward(
    const void *dy, int64_t dy_batch, int64_t dy_time, const float *grad_final_state, const void *x, int64_t x_batch,
    int64_t x_time, const void *delta, int64_t delta_batch, int64_t delta_time, const float *A, const void *Bm,
    int64_t B_batch, int64_t B_time, const void *Cm, int64_t C_batch, int64_t C_time, const float *D, const void *z,
    int64_t z_batch, int64_t z_time, const float *delta_bias, int softplus_delta, int dtype, const int *lengths,
    const float *checkpoints, int64_t B, int64_t L, int64_t C, int64_t N, void *dx, void *grad_delta, float *grad_params,
    void *dB, void *dC, void *dz, float *grad_initial_state, void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = check(dtype, B, L, C, N);
  if (rc) return rc;
  if (B == 0 || C == 0 || L == 0) return BKCORE_OK;
  if (!dy || !x || !delta || !A || !Bm || !Cm || !checkpoints || !dx || !grad_delta || !grad_params || !dB || !dC ||
      (z && !dz))
    return BKCORE_EINVAL;
  if (!near(x_time) || !near(delta_time) || !near(B_time) || !near(C_time) || !near(dy_time) || (z && !near(z_time)))
    return BKCORE_EINVAL;
  if (!workspace || workspace_bytes < bkcore_selective_scan_backward_workspace_bytes(B, L, C, N))
    return BKCORE_EWORKSPACE;
  const Plan p = plan(B, L, C, N);
  const int NP = 4 * p.lpc;
  const int64_t bc = B * L * 2 * NP;
  if ((int64_t)p.nct * B * p.S > 2147483647LL || (bc + 255) / 256 > 2147483647LL) return BKCORE_EINVAL;
  ScanArgs a{};
  a.x = x; a.xb = x_batch; a.xt = x_time; a.delta = delta; a.db = delta_batch; a.dt = delta_time; a.A = A;
  a.Bm = Bm; a.Bb = B_batch; a.Bt = B_time; a.Cm = Cm; a.Cb = C_batch; a.Ct = C_time; a.D = D;
  a.z = z; a.zb = z_batch; a.zt = z_time; a.bias = delta_bias; a.softplus = softplus_delta != 0; a.lengths = lengths;
  a.dy = dy; a.yb = dy_batch; a.yt = dy_time; a.dhT = grad_final_state; a.dx = dx; a.ddelta = grad_delta; a.dz = dz;
  a.dh0 = grad_initial_state; a.ckpt = const_cast<float *>(checkpoints);
  a.agg = (float *)workspace;
  a.aggd = a.agg + (p.S > 1 ? (size_t)p.S * B * C * NP : 0);
  a.part_bc = a.agg + round4(agg_floats(p, B, C));
  a.part_par = a.part_bc + round4((size_t)p.nct * bc);
  a.B = (int)B; a.L = (int)L; a.C = (int)C; a.N = (int)N; a.chunk = p.chunk; a.S = p.S; a.nct = p.nct;
  const unsigned grid = (unsigned)(p.nct * B * p.S), grid_agg = (unsigned)(p.nct * B * (p.S - 1));
  hipStream_t s = (hipStream_t)stream;
#define BK_AGG(LPC) hipLaunchKernelGGL((bk_scan_adjoint_agg_kernel<T, LPC>), dim3(grid_agg), dim3(THREADS), 0, s, a)
#define BK_MAIN(LPC) hipLaunchKernelGGL((bk_scan_backward_kernel<T, LPC>), dim3(grid), dim3(THREADS), 0, s, a)
  if (p.S > 1) BK_WITH_TYPE(dtype, BK_SCAN_LPC(p.lpc, BK_AGG));
  BK_WITH_TYPE(dtype, BK_SCAN_LPC(p.lpc, BK_MAIN));
#undef BK_AGG
#undef BK_MAIN
  BK_WITH_TYPE(dtype, hipLaunchKernelGGL((bk_scan_sum_bc_kernel<T>), dim3((unsigned)((bc + 255) / 256)), dim3(256), 0, s,
                                         a.part_bc, lengths, p.nct, (int)B, (int)L, (int)N, NP, (T *)dB, (T *)dC));
  bkcore_internal_sum_parts(a.part_par, (int64_t)p.S * B, C * N + 2 * C, grad_params, stream);
  return launch_status();
}

extern "C" int bkcore_selective_scan_step(const void *x, int64_t x_batch, float *state, const void *delta,
                                          int64_t delta_batch, const float *A, const void *Bm, int64_t B_batch,
                                          const void *Cm, int64_t C_batch, const float *D, const void *z,
                                          int64_t z_batch, const float *delta_bias, int softplus_delta, int dtype,
                                          int64_t B, int64_t C, int64_t N, void *y, void *stream) {
  const int rc = check(dtype, B, 1, C, N);
  if (rc) return rc;
  if (B == 0 || C == 0) return BKCORE_OK;
  if (!x || !state || !delta || !A || !Bm || !Cm || !y) return BKCORE_EINVAL;
  if (N % 4 == 0 && (!aligned16(state) || !aligned16(A))) return BKCORE_EINVAL;
  ScanArgs a{};
  a.x = x; a.xb = x_batch; a.delta = delta; a.db = delta_batch; a.A = A; a.Bm = Bm; a.Bb = B_batch; a.Cm = Cm;
  a.Cb = C_batch; a.D = D; a.z = z; a.zb = z_batch; a.bias = delta_bias; a.softplus = softplus_delta != 0; a.y = y;
  a.B = (int)B; a.C = (int)C; a.N = (int)N;
  const int lpc = lanes_per_channel(N);
  const int64_t blocks = (B * C * lpc + 255) / 256;
  if (blocks > 2147483647LL) return BKCORE_EINVAL;
  BK_WITH_TYPE(dtype, hipLaunchKernelGGL((bk_scan_step_kernel<T>), dim3((unsigned)blocks), dim3(256), 0,
                                         (hipStream_t)stream, a, state, lpc));
  return launch_status();
}
