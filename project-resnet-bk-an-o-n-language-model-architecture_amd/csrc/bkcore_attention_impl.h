// Kernels of sliding-window attention with sinks, instantiated for one operand type by the file that includes this one.
//   s_ij = scale q_i . k_j for j <= i with i - j < W or j < S;  o_i = sum_j p_ij v_j,  p_ij = exp(s_ij) / sum_j exp(s_ij)
//   backward, delta_i = do_i . o_i:  ds_ij = p_ij (do_i . v_j - delta_i);  dq_i = scale sum_j ds_ij k_j;
//   dk_j = scale sum_i ds_ij q_i;  dv_j = sum_i p_ij do_i   (sums over the query heads that share the key's head)
//
// All products go to the 16 x 16 matrix instructions.  A fragment is eight elements a lane: for 16-bit operands one
// instruction of depth 32, for float32 eight of depth 4 on the same registers (the order of the contracted index is free as
// long as both operands agree), so one body serves all types.  Scores are formed transposed (keys x queries): a lane then
// holds four neighbouring keys of one query, which is the layout the next product wants its second operand in -- the
// probabilities go from accumulators to operands without leaving the lane, and the row's maximum and sum are a lane's own
// plus two exchanges.  The other operand of that product (V, or K, Q, dO in the backward) is contracted over its rows: it
// is read from LDS through the transposing read (16-bit) or element by element (float32).
//
// What bounds it: in the prompts and in training the vector unit (17 instructions a visible score in the forward), the
// matrix unit and LDS, of which two waves a SIMD hide only part behind one another.
// Measured at 2 x 16 heads x 8192 x 128 bf16 over 4 key heads, window 1024, 4 sinks (share of the time that the vector unit,
// the matrix unit and LDS are busy): forward 288 us (56, 33, 17 %), dq with delta 332 (44, 39, 20 %), dk and dv 465 (37, 38,
// 27 %) + 44 + 5 (the sinks' part and its join).  Products of 65 GFLOP: the forward does three for two (the second half of
// the probabilities), the backward ten for five (both its kernels form the scores again, and three are second halves).
// 4 x 8 heads x 3001 ragged x 64 f16, window 500: 37.  The single-token step is bound by the cache's bytes: 64 sequences x
// 32 heads over 8 x 4100 slots x 128 bf16 in 171 + 5 us = 5.7 TB/s.
#include "bkcore_attention.h"

namespace bk {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T>
struct Frag {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec v;
};

template <typename T>
__device__ __forceinline__ void mma(const Frag<T> &a, const Frag<T> &b, f32x4 &c) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.v[i], b.v[i], c, 0, 0, 0);
  } else if constexpr (__is_same(T, bf16_t)) {
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
  } else {
    c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v, b.v, c, 0, 0, 0);
  }
}

// float16 has no exponents to spare: score gradients enter their products times a power of two, chosen so that the largest
// one possible is just below 2^15, and the accumulators are brought to a smaller power when a tile with larger ones comes.
// Unscaled, gradients below 6e-5 lose bits (dout of 1e-4: dk off by 0.004 of its size) and those above 65504 are lost.
template <typename T>
constexpr bool SCALED = __is_same(T, f16_t);
constexpr int TOP_POWER = 15, MOST_POWER = 60, LEAST_POWER = -40;  // 2^-40: the largest f16 operands at 128 elements
// The power for values below `bound` (not a number or infinite: such a tile has no finite results).
__device__ __forceinline__ int power_for(float bound) {
  const int k = (int)((__float_as_uint(bound) >> 23) & 255) - 126;  // bound < 2^k
  return max(LEAST_POWER, min(MOST_POWER, TOP_POWER - k));
}
__device__ __forceinline__ float pow2(int n) { return __builtin_amdgcn_ldexpf(1.0f, n); }
// What rounding took from the output is kept times 2^11 in float16: it starts 11 bits below the output itself.
template <typename T>
constexpr float LO_SCALE = SCALED<T> ? 2048.0f : 1.0f;

template <typename T>
constexpr int pad() { return sizeof(T) == 2 ? 16 : 4; }

// Eight elements of row `row` (clamped by the caller to one that exists) from column c: raw, zeroed where not wanted.
template <typename T, bool VEC>
__device__ __forceinline__ Frag<T> load8(const T *row, int c, int D) {
  Frag<T> f;
  if constexpr (VEC) {
    f.v = *reinterpret_cast<const typename Frag<T>::vec *>(row + (c < D ? c : 0));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = row[c + i < D ? c + i : 0];
  }
  return f;
}
// (VEC: D is a multiple of 8, so the piece is inside or outside as a whole and is selected in 32-bit words.)
template <typename T, bool VEC>
__device__ __forceinline__ Frag<T> zero_unless(const Frag<T> &f, bool row_ok, int c, int D) {
  Frag<T> r;
  if constexpr (VEC) {
    constexpr int N = 8 * (int)sizeof(T) / 4;
    union {
      typename Frag<T>::vec v;
      unsigned w[N];
    } a, b;
    a.v = f.v;
    const bool in = row_ok & (c < D);
#pragma unroll
    for (int i = 0; i < N; ++i) b.w[i] = in ? a.w[i] : 0u;
    r.v = b.v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = row_ok && c + i < D ? f.v[i] : (T)0.0f;
  }
  return r;
}

// The largest magnitude among eight float16 values and `so_far`, as its bits (their order is that of the magnitudes).
__device__ __forceinline__ unsigned top_bits(const Frag<f16_t> &f, unsigned so_far) {
  typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
  union {
    Frag<f16_t>::vec v;
    u16x8 u;
  } a;
  a.v = f.v;
  a.u &= (unsigned short)0x7fff;
#pragma unroll
  for (int i = 0; i < 8; ++i) so_far = max(so_far, (unsigned)a.u[i]);
  return so_far;
}
__device__ __forceinline__ float from_bits(unsigned u) {
  union {
    unsigned short u;
    f16_t h;
  } a;
  a.u = (unsigned short)u;
  return (float)a.h;
}
// Maximum over the four lanes that hold one column (l, l + 16, l + 32, l + 48), in each of them.
__device__ __forceinline__ float col_max(float x) {
  u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Maximum over the wave, in every lane.
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp_mov<DPP_XOR1>(x));
  x = fmaxf(x, dpp_mov<DPP_XOR2>(x));
  x = fmaxf(x, dpp_mov<DPP_HALF_MIRROR>(x));
  x = fmaxf(x, dpp_mov<DPP_MIRROR>(x));
  return col_max(x);
}

// ROWS x DP elements on their way from memory to LDS (row stride DP + pad), THREADS threads.
template <typename T, int ROWS, int DP, int THREADS, bool VEC>
struct Tile {
  static constexpr int CH = DP / 8, N = (ROWS * CH + THREADS - 1) / THREADS;
  static constexpr bool WHOLE = ROWS * CH % THREADS == 0;  // else the last pass is for some of the threads
  Frag<T> r[N];
  // A uniform 64-bit base and a 32-bit offset (the host keeps ROWS strides below 2^31); rows behind the last one repeat it.
  __device__ __forceinline__ void load(const T *base, long stride, long row0, long rows, int D, int tid) {
    const T *tile = base + row0 * stride;
    const unsigned most = (unsigned)(rows - 1 - row0 < ROWS ? rows - 1 - row0 : ROWS);
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * THREADS;
      const unsigned row = min((unsigned)(i / CH), most);
      r[k] = load8<T, VEC>(tile + row * (unsigned)stride, (i % CH) * 8, D);
    }
  }
  // top: the largest magnitude of what this thread stores (float16; as its bits)
  template <bool TOP = false>
  __device__ __forceinline__ void store(T *lds, long row0, long rows, int D, int tid, unsigned *top = nullptr) const {
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int i = tid + k * THREADS, row = i / CH, c = (i % CH) * 8;
      if (!WHOLE && i >= ROWS * CH) break;
      const Frag<T> f = zero_unless<T, VEC>(r[k], row0 + row < rows, c, D);
      *reinterpret_cast<typename Frag<T>::vec *>(lds + row * (DP + pad<T>()) + c) = f.v;
      if constexpr (TOP) *top = top_bits(f, *top);
    }
  }
};

// Operand whose contracted index runs along the row: element i of lane l is row l % 16, column 8 (l / 16) + i.
template <typename T, int DP>
__device__ __forceinline__ Frag<T> along(const T *lds, int row0, int col0, int lane) {
  Frag<T> f;
  f.v = *reinterpret_cast<const typename Frag<T>::vec *>(lds + (row0 + (lane & 15)) * (DP + pad<T>()) + col0 + (lane >> 4) * 8);
  return f;
}

// Operand contracted over rows: lane l holds column col0 + l % 16 of rows row0 + 4 g + (0..3) and row0 + 16 + 4 g + (0..3),
// g = l / 16 -- the order in which two 16-row score blocks leave their accumulators.
template <typename T, int DP>
__device__ __forceinline__ Frag<T> across(const T *lds, int row0, int col0, int lane) {
  constexpr int LD = DP + pad<T>();
  const int g = lane >> 4, m = lane & 15;
  Frag<T> f;
  if constexpr (sizeof(T) == 2) {
    typedef __attribute__((address_space(3))) s16x4 lds_vec;
    const T *p = lds + (row0 + 4 * g + (m >> 2)) * LD + col0 + 4 * (m & 3);
    union {
      s16x4 s[2];
      typename Frag<T>::vec v;
    } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)p);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_vec *)(p + 16 * LD));
    f.v = u.v;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = lds[(row0 + 4 * g + (i & 3) + 16 * (i >> 2)) * LD + col0 + m];
  }
  return f;
}

// Four neighbouring values of a lane as elements i0 .. i0 + 3 of two operands, what rounding takes from the first in the
// second.  Score gradients: those of a row sum to zero, so their products with K and Q cancel, and one rounding of half a
// step each would be half as much again as the rounding of the result (0.0026 of dq's size against 0.0017 in bfloat16).
// Probabilities: rounded once they would leave the output and dv 1.3 times as far from the formula as the rounding of the
// result does (0.0022 against 0.0017).  The second products cost 10 % of a training pass and 20 % of a prompt.
// (float16 goes through the packed conversion, which cuts instead of rounding: the second value takes that up too.)
template <typename T>
__device__ __forceinline__ void put_split(const f32x4 &x, int i0, Frag<T> &hi, Frag<T> &lo) {
  if constexpr (__is_same(T, f16_t)) {
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
      const auto h = __builtin_amdgcn_cvt_pkrtz(x[i], x[i + 1]);
      const auto l = __builtin_amdgcn_cvt_pkrtz(x[i] - (float)h[0], x[i + 1] - (float)h[1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        hi.v[i0 + i + k] = (T)h[k];
        lo.v[i0 + i + k] = (T)l[k];
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T h = (T)x[i];
      hi.v[i0 + i] = h;
      lo.v[i0 + i] = (T)(x[i] - (float)h);
    }
  }
}

// Their sum.
__device__ __forceinline__ float col_sum(float x) {
  x = fold16(x, x);
  return fold32(x, x);
}

__device__ __forceinline__ int row_length(const int *lengths, int b, int L) {
  if (!lengths) return L;
  const int n = lengths[b];
  return n < 0 ? 0 : n > L ? L : n;
}

constexpr float INF = __builtin_inff();

// Work item of a workgroup: neighbouring items share keys and values, so each of the eight dies gets a contiguous run of
// them (workgroups go to the dies in turn).  -1: none left.
__device__ __forceinline__ long work_item(long total) {
  const long per = (total + 7) / 8, w = (long)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
  return (long)(blockIdx.x >> 3) < per && w < total ? w : -1;
}
// The (batch, key head) of a run's g-th group: every eighth one after the other, so that sequences of unequal lengths (which
// lie batch by batch) spread over the dies.
__device__ __forceinline__ int work_group(int g, int groups) {
  const int q = groups / 8, more = groups % 8, split = more * (q + 1);
  if (g < split) return g % (q + 1) * 8 + g / (q + 1);
  return (g - split) % q * 8 + more + (g - split) / q;
}
inline unsigned work_grid(long total) { return (unsigned)((total + 7) / 8 * 8); }

template <typename T>
__device__ __forceinline__ const T *head(const Heads &x, int b, int h) {
  return (const T *)x.p + b * x.b + h * x.h;
}

// Four neighbouring d of a row (of a (B, L, heads, D) result), rounded to T.
template <typename T, bool VEC>
__device__ __forceinline__ void store4(T *row, int d, int D, const f32x4 &v) {
  if constexpr (VEC) {
    if (d < D) {
      typedef T vec4 __attribute__((ext_vector_type(4)));
      vec4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = (T)v[i];
      *reinterpret_cast<vec4 *>(row + d) = w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (d + i < D) row[d + i] = (T)v[i];
  }
}

// Keys of a tile: 64 for 16-bit operands, 32 for float32 (registers on the way to LDS).
template <typename T>
constexpr int key_tile() { return sizeof(T) == 2 ? 64 : 32; }

// The tiles of keys that queries [q0, q1] see: first those that hold only sinks, then the window's.
struct KeyTiles {
  int nsink, first, n;
  __device__ __forceinline__ KeyTiles(int q0, int q1, int W, int S, int BN) {
    const int lo = q0 - W + 1 > 0 ? q0 - W + 1 : 0;
    first = lo / BN;
    const int s = (S + BN - 1) / BN;
    nsink = s < first ? s : first;
    n = q1 >= q0 ? nsink + q1 / BN - first + 1 : 0;
  }
  __device__ __forceinline__ int key0(int i, int BN) const { return (i < nsink ? i : first + i - nsink) * BN; }
};

// What queries [q0, q1] see of keys [j0, j1]: 0 nothing, 1 some, 2 everything.
__device__ __forceinline__ int tile_view(int q0, int q1, int j0, int j1, int W, int S) {
  if (j0 > q1 || (q0 - j1 >= W && j0 >= S)) return 0;
  return j1 <= q0 && (q1 - j0 < W || j1 < S) ? 2 : 1;
}
// One unsigned comparison holds both ends of the window (a later key gives a huge distance); the sinks only where the tile
// has some.
template <bool SINKS>
__device__ __forceinline__ bool sees(int i, int j, int W, int S) {
  const unsigned gap = (unsigned)(i - j);
  return SINKS ? (gap < (unsigned)W) | ((j < S) & (j <= i)) : gap < (unsigned)W;
}

// ---- forward: 4 waves x 16 QB queries; keys and values through LDS, the next tile on its way in registers.
template <typename T, int DP, bool VEC, int QB>
__global__ __launch_bounds__(256, 2) void bk_attn_kernel(AttnArgs a) {
  constexpr int BN = key_tile<T>(), LD = DP + pad<T>(), NK = BN / 16, ND = DP / 16, NC = DP / 32, WQ = 16 * QB, BM = 4 * WQ;
  __shared__ __attribute__((aligned(16))) T sK[BN * LD], sV[BN * LD];
  const int nq = (a.L + BM - 1) / BM;
  long w = work_item((long)a.B * a.H * nq);
  if (w < 0) return;
  const int G = a.H / a.Hk;
  const int g_ = (int)(w % G);
  w /= G;
  const int qt = (int)(w % nq);
  w /= nq;
  const int group = work_group((int)w, a.B * a.Hk), hk = group % a.Hk, b = group / a.Hk, h = hk * G + g_;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
  const int len = row_length(a.lengths, b, a.L);
  const int q0 = qt * BM, q1 = min(q0 + BM, len) - 1;
  const int w0 = q0 + wave * WQ, w1 = min(w0 + WQ, len) - 1;  // the wave's own queries
  const T *qp = head<T>(a.q, b, h), *kp = head<T>(a.k, b, hk), *vp = head<T>(a.v, b, hk);
  const float sc = a.scale * LOG2E;

  Frag<T> q[QB][NC];
  if (q1 >= q0) {
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int row = w0 + 16 * i + m;
#pragma unroll
      for (int c = 0; c < NC; ++c)
        q[i][c] = load8<T, VEC>(qp + (long)min(row, len - 1) * a.q.t, c * 32 + g * 8, a.D);
#pragma unroll
      for (int c = 0; c < NC; ++c) q[i][c] = zero_unless<T, VEC>(q[i][c], row < len, c * 32 + g * 8, a.D);
    }
  }
  f32x4 o[ND][QB];
  float mx[QB], sum[QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    mx[i] = -INF;
    sum[i] = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d][i] = {0.0f, 0.0f, 0.0f, 0.0f};
  }
  const KeyTiles kt(q0, q1, a.W, a.S, BN);
  Tile<T, BN, DP, 256, VEC> tk, tv;
  if (kt.n) {
    tk.load(kp, a.k.t, kt.key0(0, BN), len, a.D, tid);
    tv.load(vp, a.v.t, kt.key0(0, BN), len, a.D, tid);
  }
  for (int it = 0; it < kt.n; ++it) {
    const int j0 = kt.key0(it, BN);
    __syncthreads();
    tk.store(sK, j0, len, a.D, tid);
    tv.store(sV, j0, len, a.D, tid);
    __syncthreads();
    if (it + 1 < kt.n) {
      const int j = kt.key0(it + 1, BN);
      tk.load(kp, a.k.t, j, len, a.D, tid);
      tv.load(vp, a.v.t, j, len, a.D, tid);
    }
    const int view = w1 >= w0 ? tile_view(w0, w1, j0, j0 + BN - 1, a.W, a.S) : 0;
    if (!view) continue;
    f32x4 s[NK][QB];
#pragma unroll
    for (int k = 0; k < NK; ++k) {
#pragma unroll
      for (int i = 0; i < QB; ++i) s[k][i] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const Frag<T> kf = along<T, DP>(sK, 16 * k, 32 * c, lane);
#pragma unroll
        for (int i = 0; i < QB; ++i) mma(kf, q[i][c], s[k][i]);
      }
    }
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int qi = w0 + 16 * i + m;
      float top = -INF;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[k][i][r] *= sc;
      if (view == 1) {
        if (j0 < a.S) {
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[k][i][r] = sees<true>(qi, j0 + 16 * k + 4 * g + r, a.W, a.S) ? s[k][i][r] : -INF;
        } else {
#pragma unroll
          for (int k = 0; k < NK; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              s[k][i][r] = sees<false>(qi, j0 + 16 * k + 4 * g + r, a.W, a.S) ? s[k][i][r] : -INF;
        }
      }
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[k][i][r]);
      top = fmaxf(mx[i], col_max(top));
      const float ref = top == -INF ? 0.0f : top, alpha = exp2_fast(mx[i] - ref);
      mx[i] = top;
      float part = 0.0f;
#pragma unroll
      for (int k = 0; k < NK; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[k][i][r] = exp2_fast(s[k][i][r] - ref);
          part += s[k][i][r];
        }
      sum[i] = fmaf(sum[i], alpha, part);
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][i][r] *= alpha;
    }
#pragma unroll
    for (int k = 0; k < NK; k += 2) {
      Frag<T> p[QB], pl[QB];
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        put_split(s[k][i], 0, p[i], pl[i]);
        put_split(s[k + 1][i], 4, p[i], pl[i]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const Frag<T> vf = across<T, DP>(sV, 16 * k, 16 * d, lane);
#pragma unroll
        for (int i = 0; i < QB; ++i) mma(vf, p[i], o[d][i]);
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < QB; ++i) mma(vf, pl[i], o[d][i]);
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int row = w0 + 16 * i + m;
    const float l = col_sum(sum[i]);
    if (row < a.L) {
      const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // a row that sees nothing: zeros
      T *op = (T *)a.o + (((long)b * a.L + row) * a.H + h) * a.D;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = row < len ? o[d][i][r] * inv : 0.0f;
        store4<T, VEC>(op, 16 * d + 4 * g, a.D, v);
        if (a.lo) {
          f32x4 e;
#pragma unroll
          for (int r = 0; r < 4; ++r) e[r] = (v[r] - (float)(T)v[r]) * LO_SCALE<T>;
          store4<T, VEC>((T *)a.lo + (op - (T *)a.o), 16 * d + 4 * g, a.D, e);
        }
      }
      if (a.lse && g == 0)
        a.lse[((long)b * a.H + h) * a.L + row] =
            row < len && (l > 0.0f || l != l) ? mx[i] + __builtin_amdgcn_logf(l) : INF;
    }
  }
}

// ---- dq: the forward's loop with two score products, dS^T in the lane, and K contracted over its rows.  It runs first and
// leaves delta_i = do_i . o_i for the keys' launch: a row's gradient is in its registers anyway.  A 16-bit output's rounding
// is added back (lo): it would reach every score gradient of the row.  delta is the diagonal of the same matrix product, in
// the same order, that gives do_i . v_j: a row that sees one key has o_i = v_j, and its score gradient do_i . v_j - delta_i
// is zero to the last bit, as it is by the formula (a sum in another order leaves 1e-7 of its terms there).
template <typename T, int DP, bool VEC, int QB>
__global__ __launch_bounds__(256, DP * sizeof(T) > 256 ? 1 : 2) void bk_attn_dq_kernel(AttnArgs a) {
  constexpr int BN = key_tile<T>(), LD = DP + pad<T>(), NK = BN / 16, ND = DP / 16, NC = DP / 32, WQ = 16 * QB, BM = 4 * WQ;
  __shared__ __attribute__((aligned(16))) T sK[BN * LD], sV[BN * LD];
  const int nq = (a.L + BM - 1) / BM;
  long w = work_item((long)a.B * a.H * nq);
  if (w < 0) return;
  const int G = a.H / a.Hk;
  const int g_ = (int)(w % G);
  w /= G;
  const int qt = (int)(w % nq);
  w /= nq;
  const int group = work_group((int)w, a.B * a.Hk), hk = group % a.Hk, b = group / a.Hk, h = hk * G + g_;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
  const int len = row_length(a.lengths, b, a.L);
  const int q0 = qt * BM, q1 = min(q0 + BM, len) - 1;
  const int w0 = q0 + wave * WQ, w1 = min(w0 + WQ, len) - 1;
  const T *qp = head<T>(a.q, b, h), *gp = head<T>(a.dout, b, h), *kp = head<T>(a.k, b, hk), *vp = head<T>(a.v, b, hk);
  const float sc = a.scale * LOG2E;
  Frag<T> q[QB][NC], go[QB][NC];
  float lse[QB], delta[QB];  // lse less the power of two that the row's score gradients carry (SCALED)
  // SCALED: largest |v| of a tile, by wave; by row sum |do_i|, so that |do_i . v_j| <= reach max |v|, and the power.  The rows
  // are the wave's own and its lanes' accesses stay in order.
  __shared__ float sTop[4], sReach[SCALED<T> ? BM : 1];
  __shared__ int sPower[SCALED<T> ? BM : 1];
  float *reach = sReach + (SCALED<T> ? wave * WQ + m : 0);
  int *power = sPower + (SCALED<T> ? wave * WQ + m : 0);
  f32x4 dq[ND][QB];
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int row = w0 + 16 * i + m;
    lse[i] = INF;
    delta[i] = 0.0f;
    if constexpr (SCALED<T>) {
      reach[16 * i] = 0.0f;
      power[16 * i] = MOST_POWER;
    }
    if (q1 >= q0) {
      const long r = min(row, len - 1);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        q[i][c] = load8<T, VEC>(qp + r * a.q.t, c * 32 + g * 8, a.D);
        go[i][c] = load8<T, VEC>(gp + r * a.dout.t, c * 32 + g * 8, a.D);
      }
      const T *orow = (const T *)a.out + (((long)b * a.L + r) * a.H + h) * a.D;
      const T *lrow = (const T *)a.lo + (((long)b * a.L + r) * a.H + h) * a.D;
      Frag<T> oo[NC], ol[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        oo[c] = load8<T, VEC>(orow, c * 32 + g * 8, a.D);
        if (a.lo) ol[c] = load8<T, VEC>(lrow, c * 32 + g * 8, a.D);
      }
      const float l_ = a.lse[((long)b * a.H + h) * a.L + r];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        q[i][c] = zero_unless<T, VEC>(q[i][c], row < len, c * 32 + g * 8, a.D);
        go[i][c] = zero_unless<T, VEC>(go[i][c], row < len, c * 32 + g * 8, a.D);
        oo[c] = zero_unless<T, VEC>(oo[c], row < len, c * 32 + g * 8, a.D);
        if (a.lo) ol[c] = zero_unless<T, VEC>(ol[c], row < len, c * 32 + g * 8, a.D);
      }
      f32x4 od = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) mma(oo[c], go[i][c], od);
      if (a.lo) {
        f32x4 rest = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c) mma(ol[c], go[i][c], rest);
#pragma unroll
        for (int r = 0; r < 4; ++r) od[r] = fmaf(rest[r], 1.0f / LO_SCALE<T>, od[r]);
      }
      if constexpr (SCALED<T>) {
        float l1 = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e) l1 += fabsf((float)go[i][c].v[e]);
        reach[16 * i] = col_sum(l1);
      }
      const float mine = (m & 2) ? ((m & 1) ? od[3] : od[2]) : ((m & 1) ? od[1] : od[0]);
      const float dot = col_sum(g == (m >> 2) ? mine : 0.0f);  // to the four lanes that share the row
      if (row < len) {
        lse[i] = SCALED<T> ? l_ - (float)MOST_POWER : l_;
        delta[i] = dot;
        if (g == 0) a.delta[((long)b * a.H + h) * a.L + row] = dot;
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) dq[d][i] = {0.0f, 0.0f, 0.0f, 0.0f};
  }
  const KeyTiles kt(q0, q1, a.W, a.S, BN);
  Tile<T, BN, DP, 256, VEC> tk, tv;
  if (kt.n) {
    tk.load(kp, a.k.t, kt.key0(0, BN), len, a.D, tid);
    tv.load(vp, a.v.t, kt.key0(0, BN), len, a.D, tid);
  }
  for (int it = 0; it < kt.n; ++it) {
    const int j0 = kt.key0(it, BN);
    __syncthreads();
    tk.store(sK, j0, len, a.D, tid);
    if constexpr (SCALED<T>) {
      unsigned top = 0;
      tv.template store<true>(sV, j0, len, a.D, tid, &top);
      const float w_ = wave_max(from_bits(top));
      if (lane == 0) sTop[wave] = w_;
    } else {
      tv.store(sV, j0, len, a.D, tid);
    }
    __syncthreads();
    if (it + 1 < kt.n) {
      const int j = kt.key0(it + 1, BN);
      tk.load(kp, a.k.t, j, len, a.D, tid);
      tv.load(vp, a.v.t, j, len, a.D, tid);
    }
    const int view = w1 >= w0 ? tile_view(w0, w1, j0, j0 + BN - 1, a.W, a.S) : 0;
    if (!view) continue;
    if constexpr (SCALED<T>) {
      const float top = fmaxf(fmaxf(sTop[0], sTop[1]), fmaxf(sTop[2], sTop[3]));
      int to[QB];
      bool less = false;
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        to[i] = min(power[16 * i], power_for(fmaf(reach[16 * i], top, fabsf(delta[i]))));
        less |= to[i] < power[16 * i];
      }
      if (__any(less)) {
#pragma unroll
        for (int i = 0; i < QB; ++i) {
          const float f = pow2(to[i] - power[16 * i]);
          lse[i] += (float)(power[16 * i] - to[i]);
          power[16 * i] = to[i];
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) dq[d][i][r] *= f;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < NK; k += 2) {
      Frag<T> ds[QB], dl[QB];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        f32x4 s[QB], dp[QB];
#pragma unroll
        for (int i = 0; i < QB; ++i) s[i] = dp[i] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          const Frag<T> kf = along<T, DP>(sK, 16 * (k + kk), 32 * c, lane), vf = along<T, DP>(sV, 16 * (k + kk), 32 * c, lane);
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            mma(kf, q[i][c], s[i]);
            mma(vf, go[i][c], dp[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < QB; ++i) {
          const int qi = w0 + 16 * i + m;
#pragma unroll
          for (int r = 0; r < 4; ++r) s[i][r] = fmaf(s[i][r], sc, -lse[i]);
          if (view == 1) {
            const int j = j0 + 16 * (k + kk) + 4 * g;
            if (j0 < a.S) {
#pragma unroll
              for (int r = 0; r < 4; ++r) s[i][r] = sees<true>(qi, j + r, a.W, a.S) ? s[i][r] : -INF;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r) s[i][r] = sees<false>(qi, j + r, a.W, a.S) ? s[i][r] : -INF;
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) dp[i][r] = exp2_fast(s[i][r]) * (dp[i][r] - delta[i]);
          put_split(dp[i], 4 * kk, ds[i], dl[i]);
        }
      }
#pragma unroll
      for (int d = 0; d < ND; d += 2) {  // two column blocks: four products between two on the same accumulator
        const Frag<T> ka = across<T, DP>(sK, 16 * k, 16 * d, lane), kb = across<T, DP>(sK, 16 * k, 16 * d + 16, lane);
#pragma unroll
        for (int i = 0; i < QB; ++i) {
          mma(ka, ds[i], dq[d][i]);
          mma(kb, ds[i], dq[d + 1][i]);
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
          for (int i = 0; i < QB; ++i) {
            mma(ka, dl[i], dq[d][i]);
            mma(kb, dl[i], dq[d + 1][i]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int i = 0; i < QB; ++i) {
    const int row = w0 + 16 * i + m;
    if (row < a.L) {
      T *op = (T *)a.dq + (((long)b * a.L + row) * a.H + h) * a.D;
      const float back = SCALED<T> ? a.scale * pow2(-power[16 * i]) : a.scale;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = row < len && lse[i] != INF ? dq[d][i][r] * back : 0.0f;
        store4<T, VEC>(op, 16 * d + 4 * g, a.D, v);
      }
    }
  }
}

// ---- dk, dv.  SINK false: 4 waves x 16 KB keys, all of them over the same 32 queries at a time, over the tile's own queries
// (its window) and the heads of the group.  SINK true: the sinks' part behind that -- the first 64 keys see all later
// queries, so their loop is the whole sequence: it is cut into stretches, a wave takes 16 KB of these keys and its own
// 32 of every 128 queries, and leaves float32 sums that the join adds up in a fixed order.
// part: (1 + 4 nsplit, B, Hk, S, 2, D); slot 0 is what the first key tile has from its own queries.
template <typename T, int DP, bool VEC, bool SINK, int KB>
__global__ __launch_bounds__(256, KB == 2 && DP * (SINK ? 2 : 1) * sizeof(T) > 256 ? 1 : 2) void bk_attn_dkv_kernel(AttnArgs a) {
  constexpr int WK = 16 * KB, BK = 4 * WK, BQ = ATTN_BQ, ROWS = SINK ? SINK_TILE : BQ, LD = DP + pad<T>(), ND = DP / 16, NC = DP / 32;
  // At 128 elements of 16 bits the values' fragments and half of the keys' wait in LDS, each lane's as it wants them: in
  // registers they leave no room for two waves a SIMD, and a single spilled word costs more than these reads (its reload
  // waits for the rows under way).
  constexpr bool VLDS = KB == 2 && DP == 128 && sizeof(T) == 2 && !SINK;
  __shared__ __attribute__((aligned(16))) T sQ[ROWS * LD], sG[ROWS * LD];
  __shared__ Frag<T> sF[VLDS ? 4 * 3 * NC * 64 : 1];
  __shared__ __attribute__((aligned(16))) float sL[ROWS], sD[ROWS];
  __shared__ float sTop[4], sFar[4];  // SCALED: largest |do| and |delta| of a tile, by wave
  const int nk = SINK ? (a.S + WK - 1) / WK : (a.L + BK - 1) / BK, ns = SINK ? a.nsplit : 1;
  long w = work_item((long)a.B * a.Hk * nk * ns);
  if (w < 0) return;
  const int tile = (int)(w % nk);
  w /= nk;
  const int split = (int)(w % ns);
  w /= ns;
  const int group = work_group((int)w, a.B * a.Hk), hk = group % a.Hk, b = group / a.Hk, G = a.H / a.Hk;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
  const int len = row_length(a.lengths, b, a.L);
  const int key0 = SINK ? tile * WK : tile * BK + wave * WK;  // the wave's first key
  const int sub = SINK ? wave * BQ : 0;                              // its queries inside the tile
  long q_from, q_to;
  if (SINK) {
    const long rest = a.rest, n = a.L > rest ? a.L - rest : 0;
    const long per = ((n + ns - 1) / ns + ROWS - 1) / ROWS * ROWS;
    q_from = rest + split * per;
    q_to = q_from + per < len ? q_from + per : len;
  } else {
    const int k0 = tile * BK;
    q_from = k0 / BQ * BQ;
    q_to = ((long)k0 + BK - 1 + a.W - 1) / BQ * BQ + BQ;
    q_to = q_to < len ? q_to : len;
  }
  const T *kp = head<T>(a.k, b, hk), *vp = head<T>(a.v, b, hk);
  const float sc = a.scale * LOG2E;
  Frag<T> kf[VLDS ? 1 : KB][NC], vf[VLDS ? 1 : KB][VLDS ? 1 : NC];
  Frag<T> *mine = sF + (VLDS ? wave * 3 * NC * 64 + lane : 0);  // v of both key blocks, then k of the second
  f32x4 dk[ND][KB], dv[ND][KB];
  unsigned vtop = 0;
#pragma unroll
  for (int i = 0; i < KB; ++i) {
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d][i] = dv[d][i] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (len > 0) {
      const int row = key0 + 16 * i + m;
      const long r = min(row, len - 1);
      Frag<T> k_[NC], v_[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        k_[c] = load8<T, VEC>(kp + r * a.k.t, c * 32 + g * 8, a.D);
        v_[c] = load8<T, VEC>(vp + r * a.v.t, c * 32 + g * 8, a.D);
      }
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        k_[c] = zero_unless<T, VEC>(k_[c], row < len, c * 32 + g * 8, a.D);
        v_[c] = zero_unless<T, VEC>(v_[c], row < len, c * 32 + g * 8, a.D);
        if constexpr (SCALED<T>) vtop = top_bits(v_[c], vtop);
        if constexpr (VLDS) {
          mine[(i * NC + c) * 64] = v_[c];
          if (i == 0) kf[0][c] = k_[c];
          else mine[(2 * NC + c) * 64] = k_[c];
        } else {
          kf[i][c] = k_[c];
          vf[i][c] = v_[c];
        }
      }
    }
  }
  const float vmost = SCALED<T> ? wave_max(from_bits(vtop)) * (float)a.D : 0.0f;  // |do . v| <= D max |do| max |v|
  int power = MOST_POWER;
  const int per_head = q_to > q_from ? (int)((q_to - q_from + ROWS - 1) / ROWS) : 0, total = per_head * G;
  Tile<T, ROWS, DP, 256, VEC> tq, tg;
  float rl = INF, rd = 0.0f;
  auto fetch = [&](int it) {
    const int h = hk * G + it / per_head;
    const long qi = q_from + (long)(it % per_head) * ROWS;
    tq.load(head<T>(a.q, b, h), a.q.t, qi, len, a.D, tid);
    tg.load(head<T>(a.dout, b, h), a.dout.t, qi, len, a.D, tid);
    if (tid < ROWS) {
      const long r = ((long)b * a.H + h) * a.L + (qi + tid < len ? qi + tid : len - 1);
      rl = a.lse[r];
      rd = a.delta[r];
    }
  };
  if (total) fetch(0);
  for (int it = 0; it < total; ++it) {
    const long qi = q_from + (long)(it % per_head) * ROWS;
    __syncthreads();
    tq.store(sQ, qi, len, a.D, tid);
    if constexpr (SCALED<T>) {
      unsigned top = 0;
      tg.template store<true>(sG, qi, len, a.D, tid, &top);
      const float w_ = wave_max(from_bits(top));
      if (lane == 0) sTop[wave] = w_;
      if (wave * 64 < ROWS) {
        const float f_ = wave_max(tid < ROWS && qi + tid < len ? fabsf(rd) : 0.0f);
        if (lane == 0) sFar[wave] = f_;
      }
    } else {
      tg.store(sG, qi, len, a.D, tid);
    }
    if (tid < ROWS) {
      sL[tid] = qi + tid < len ? (SCALED<T> ? rl - (float)TOP_POWER : rl) : INF;
      sD[tid] = qi + tid < len ? rd : 0.0f;
    }
    __syncthreads();
    if (it + 1 < total) fetch(it + 1);
    const int i0 = (int)qi + sub;
    const int view = i0 < len && key0 < len ? tile_view(i0, i0 + BQ - 1, key0, key0 + WK - 1, a.W, a.S) : 0;
    if (!view) continue;
    float factor = 1.0f;  // of do . v - delta, beside the 2^15 that the probabilities carry in float16
    if constexpr (SCALED<T>) {
      const float top = fmaxf(fmaxf(sTop[0], sTop[1]), fmaxf(sTop[2], sTop[3]));
      const float far = ROWS > 64 ? fmaxf(sFar[0], sFar[1]) : sFar[0];
      const int to = min(power, __builtin_amdgcn_readfirstlane(power_for(fmaf(vmost, top, far))));
      if (to < power) {
        const float f = pow2(to - power);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int y = 0; y < KB; ++y)
#pragma unroll
            for (int r = 0; r < 4; ++r) dk[d][y][r] *= f;
        power = to;
      }
      factor = pow2(power - TOP_POWER);
    }
    Frag<T> pf[KB], pl[KB], df[KB], dl[KB];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      f32x4 s[KB], dp[KB];  // of the key blocks: a lane holds four queries of one key
#pragma unroll
      for (int y = 0; y < KB; ++y) s[y] = dp[y] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const Frag<T> qf = along<T, DP>(sQ, sub + 16 * x, 32 * c, lane), gf = along<T, DP>(sG, sub + 16 * x, 32 * c, lane);
#pragma unroll
        for (int y = 0; y < KB; ++y) {
          if constexpr (VLDS) {
            mma(qf, y ? mine[(2 * NC + c) * 64] : kf[0][c], s[y]);
            mma(gf, mine[(y * NC + c) * 64], dp[y]);
          } else {
            mma(qf, kf[y][c], s[y]);
            mma(gf, vf[y][c], dp[y]);
          }
        }
      }
      const f32x4 ls = *reinterpret_cast<const f32x4 *>(&sL[sub + 16 * x + 4 * g]);
      f32x4 de = *reinterpret_cast<const f32x4 *>(&sD[sub + 16 * x + 4 * g]);
      if constexpr (SCALED<T>) {
#pragma unroll
        for (int r = 0; r < 4; ++r) de[r] *= factor;
      }
#pragma unroll
      for (int y = 0; y < KB; ++y)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[y][r] = fmaf(s[y][r], sc, -ls[r]);
      if (view == 1) {
#pragma unroll
        for (int y = 0; y < KB; ++y) {
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[y][r] = sees<true>(i0 + 16 * x + 4 * g + r, key0 + 16 * y + m, a.W, a.S) ? s[y][r] : -INF;
        }
      }
#pragma unroll
      for (int y = 0; y < KB; ++y) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          s[y][r] = exp2_fast(s[y][r]);
          dp[y][r] = s[y][r] * (SCALED<T> ? fmaf(dp[y][r], factor, -de[r]) : dp[y][r] - de[r]);
        }
        put_split(s[y], 4 * x, pf[y], pl[y]);
        put_split(dp[y], 4 * x, df[y], dl[y]);
      }
      if constexpr (VLDS) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const Frag<T> gt = across<T, DP>(sG, sub, 16 * d, lane), qt = across<T, DP>(sQ, sub, 16 * d, lane);
#pragma unroll
      for (int y = 0; y < KB; ++y) {
        mma(qt, df[y], dk[d][y]);
        mma(gt, pf[y], dv[d][y]);
      }
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int y = 0; y < KB; ++y) {
          mma(qt, dl[y], dk[d][y]);
          mma(gt, pl[y], dv[d][y]);
        }
      }
      if constexpr (VLDS) {
        if (d & 1) __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  const bool parts = a.nsplit > 0;
  const float kback = SCALED<T> ? a.scale * pow2(-power) : a.scale;
  const float vback = SCALED<T> ? 1.0f / (1 << TOP_POWER) : 1.0f;
#pragma unroll
  for (int y = 0; y < KB; ++y) {
    const int key = key0 + 16 * y + m;
    if (SINK || (parts && key < a.S)) {
      if (key < a.S) {
        const long slot = SINK ? 1 + 4 * split + wave : 0;
        float *p = a.part + ((((slot * a.B + b) * a.Hk + hk) * a.S + key) * 2) * a.D;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (16 * d + 4 * g + r < a.D) {
              p[16 * d + 4 * g + r] = dk[d][y][r] * kback;
              p[a.D + 16 * d + 4 * g + r] = dv[d][y][r] * vback;
            }
      }
    } else if (key < a.L) {
      const long at0 = (((long)b * a.L + key) * a.Hk + hk) * a.D;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x4 v;
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = dk[d][y][r] * kback;
        store4<T, VEC>((T *)a.dk + at0, 16 * d + 4 * g, a.D, v);
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = dv[d][y][r] * vback;
        store4<T, VEC>((T *)a.dv + at0, 16 * d + 4 * g, a.D, v);
      }
    }
  }
}

// ---- the sinks' gradients from their parts
template <typename T>
__global__ __launch_bounds__(256) void bk_attn_sink_join_kernel(AttnArgs a) {
  const int rows = a.S < a.L ? a.S : a.L;
  const long per = (long)a.B * a.Hk * a.S * 2 * a.D, id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= per) return;
  const int d = (int)(id % a.D), which = (int)(id / a.D % 2), key = (int)(id / (2 * a.D) % a.S);
  const long bh = id / (2 * a.D) / a.S;
  if (key >= rows) return;
  float s = 0.0f;
#pragma unroll 8
  for (int p = 0; p < 1 + 4 * a.nsplit; ++p) s += a.part[p * per + id];
  const int b = (int)(bh / a.Hk), hk = (int)(bh % a.Hk);
  ((T *)(which ? a.dv : a.dk))[(((long)b * a.L + key) * a.Hk + hk) * a.D + d] = (T)s;
}

// ---- one token: 4 waves over a stretch of the visible positions, 32 at a time each; up to 16 query heads of a key head
// are the columns of one product.  The new token's key and value come from the call's operands and are written to the
// cache by the first stretch; the slot they go to holds a position that is out of the window, so nobody reads it.
template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256) void bk_attn_step_kernel(StepArgs a) {
  constexpr int LD = DP + pad<T>(), ND = DP / 16, NC = DP / 32, NV = 32 * (DP / 8) / 64;
  constexpr int OUT = 4 * 16 * (DP + 4), TILE_BYTES = 4 * 32 * LD * (int)sizeof(T);
  __shared__ __attribute__((aligned(16))) char mem[TILE_BYTES > OUT * 4 ? TILE_BYTES : OUT * 4];
  __shared__ float sM[4][16], sS[4][16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
  unsigned w = blockIdx.x;
  const int split = w % a.nsplit;
  w /= a.nsplit;
  const int hc = w % a.hchunks;
  w /= a.hchunks;
  const int hk = w % a.Hk, b = w / a.Hk, G = a.H / a.Hk;
  const int pos = a.positions[b];
  const int nh = min(16, G - hc * 16), h0 = hk * G + hc * 16;
  const T *kc = head<T>(a.kc, b, hk), *vc = head<T>(a.vc, b, hk);
  const T *kn = head<T>(a.k, b, hk), *vn = head<T>(a.v, b, hk);
  const int ring = a.cap - a.S;
  const int first = max(a.S, pos - a.W + 1);                     // first position of the window behind the sinks
  const int nsink = pos < 0 ? 0 : min(a.S - 1, pos) + 1, n = pos < 0 ? 0 : nsink + max(0, pos - first + 1);
  auto slot = [&](int t) {  // of the t-th visible position
    return t < nsink ? t : a.S + (first - a.S + t - nsink) % ring;
  };
  if (pos >= 0 && split == 0 && hc == 0) {
    const long at0 = pos < a.S ? pos : a.S + (pos - a.S) % ring;
    T *ko = const_cast<T *>(kc) + at0 * a.kc.t, *vo = const_cast<T *>(vc) + at0 * a.vc.t;
    for (int d = tid; d < a.D; d += 256) {
      ko[d] = kn[d];
      vo[d] = vn[d];
    }
  }
  Frag<T> q[NC];
  {
    const T *qp = head<T>(a.q, b, h0 + min(m, nh - 1));
#pragma unroll
    for (int c = 0; c < NC; ++c) q[c] = load8<T, VEC>(qp, c * 32 + g * 8, a.D);
#pragma unroll
    for (int c = 0; c < NC; ++c) q[c] = zero_unless<T, VEC>(q[c], m < nh, c * 32 + g * 8, a.D);
  }
  f32x4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = {0.0f, 0.0f, 0.0f, 0.0f};
  float mx = -INF, sum = 0.0f;
  const float sc = a.scale * LOG2E;
  const int from = split * a.per, to = min(n, from + a.per);
  T *sV = (T *)mem + wave * 32 * LD;
  Frag<T> kr[2][NC], vr[NV];
  auto row = [&](const T *cache, const T *fresh, long stride, int t) {  // the newest position is not in the cache yet
    return t >= n - 1 ? fresh : cache + (long)slot(t) * stride;
  };
  auto fetch = [&](int t0) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const T *p = row(kc, kn, a.kc.t, t0 + 16 * k + m);
#pragma unroll
      for (int c = 0; c < NC; ++c) kr[k][c] = load8<T, VEC>(p, c * 32 + g * 8, a.D);
    }
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = lane + 64 * k;
      vr[k] = load8<T, VEC>(row(vc, vn, a.vc.t, t0 + i / (DP / 8)), (i % (DP / 8)) * 8, a.D);
    }
  };
  if (from + wave * 32 < to) fetch(from + wave * 32);
  for (int t0 = from + wave * 32; t0 < to; t0 += 128) {
    f32x4 s[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      s[k] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if (!VEC || a.D < DP) kr[k][c] = zero_unless<T, VEC>(kr[k][c], true, c * 32 + g * 8, a.D);
        mma(kr[k][c], q[c], s[k]);
      }
    }
    // the wave's own LDS rows: its accesses stay in order, no other wave touches them
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int i = lane + 64 * k, r = i / (DP / 8), c = (i % (DP / 8)) * 8;
      const Frag<T> f = zero_unless<T, VEC>(vr[k], t0 + r < to, c, a.D);
      *reinterpret_cast<typename Frag<T>::vec *>(sV + r * LD + c) = f.v;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (t0 + 128 < to) fetch(t0 + 128);
    float top = -INF;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[k][r] = t0 + 16 * k + 4 * g + r < to ? s[k][r] * sc : -INF;
        top = fmaxf(top, s[k][r]);
      }
    top = fmaxf(mx, col_max(top));
    const float ref = top == -INF ? 0.0f : top, alpha = exp2_fast(mx - ref);
    mx = top;
    float part = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[k][r] = exp2_fast(s[k][r] - ref);
        part += s[k][r];
      }
    sum = fmaf(sum, alpha, part);
    Frag<T> p, pl;
    put_split(s[0], 0, p, pl);
    put_split(s[1], 4, p, pl);
#pragma unroll
    for (int d = 0; d < ND; ++d) {
#pragma unroll
      for (int r = 0; r < 4; ++r) o[d][r] *= alpha;
      const Frag<T> vf = across<T, DP>(sV, 0, 16 * d, lane);
      mma(vf, p, o[d]);
      if constexpr (sizeof(T) == 2) mma(vf, pl, o[d]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  sum = col_sum(sum);
  __syncthreads();  // the value rows are done with: their memory takes the waves' results
  float *sO = (float *)mem;
  if (g == 0) {
    sM[wave][m] = mx;
    sS[wave][m] = sum;
  }
#pragma unroll
  for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4 *>(&sO[(wave * 16 + m) * (DP + 4) + 16 * d + 4 * g]) = o[d];
  __syncthreads();
  for (int i = tid; i < nh * a.D; i += 256) {
    const int h = i / a.D, d = i % a.D;
    float top = -INF, l = 0.0f, acc = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; ++k) top = fmaxf(top, sM[k][h]);
    const float ref = top == -INF ? 0.0f : top;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float f = exp2_fast(sM[k][h] - ref);
      l = fmaf(sS[k][h], f, l);
      acc = fmaf(sO[(k * 16 + h) * (DP + 4) + d], f, acc);
    }
    const long bh = (long)b * a.H + h0 + h;
    if (a.nsplit == 1) {
      ((T *)a.o)[bh * a.D + d] = (T)(l > 0.0f || l != l ? acc / l : 0.0f);
    } else {
      float *p = a.part + ((long)split * a.B * a.H + bh) * (a.D + 2);
      p[d] = acc;
      if (d == 0) {
        p[a.D] = top;
        p[a.D + 1] = l;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(128) void bk_attn_step_join_kernel(StepArgs a) {
  const long bh = blockIdx.x, stride = (long)a.B * a.H * (a.D + 2);
  const float *p = a.part + bh * (a.D + 2);
  float top = -INF;
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) top = fmaxf(top, p[s * stride + a.D]);
  const float ref = top == -INF ? 0.0f : top;
  const int d = threadIdx.x;
  if (d >= a.D) return;
  float l = 0.0f, acc = 0.0f;
#pragma unroll 4
  for (int s = 0; s < a.nsplit; ++s) {
    const float f = exp2_fast(p[s * stride + a.D] - ref);
    l = fmaf(p[s * stride + a.D + 1], f, l);
    acc = fmaf(p[s * stride + d], f, acc);
  }
  ((T *)a.o)[bh * a.D + d] = (T)(l > 0.0f || l != l ? acc / l : 0.0f);
}

}  // namespace

#define BK_ATTN_DP(LAUNCH)                                            \
  do {                                                                \
    if (dp == 32) { if (vec) LAUNCH(32, true); else LAUNCH(32, false); }        \
    else if (dp == 64) { if (vec) LAUNCH(64, true); else LAUNCH(64, false); }   \
    else { if (vec) LAUNCH(128, true); else LAUNCH(128, false); }     \
  } while (0)

template <typename T>
void attn_forward(const AttnArgs &a, int dp, bool vec, hipStream_t s) {
  const long heads = (long)a.B * a.H;
#define BK_LAUNCH_Q(DP, VEC, QB)                                                                                     \
  hipLaunchKernelGGL((bk_attn_kernel<T, DP, VEC, QB>), dim3(work_grid(heads * ((a.L + 64 * QB - 1) / (64 * QB)))),   \
                     dim3(256), 0, s, a)
#define BK_LAUNCH(DP, VEC)                   \
  do {                                       \
    if (a.wide_q) BK_LAUNCH_Q(DP, VEC, 2);   \
    else BK_LAUNCH_Q(DP, VEC, 1);            \
  } while (0)
  BK_ATTN_DP(BK_LAUNCH);
#undef BK_LAUNCH
#undef BK_LAUNCH_Q
}

template <typename T>
void attn_backward(const AttnArgs &a, int dp, bool vec, hipStream_t s) {
  const long heads = (long)a.B * a.H, kheads = (long)a.B * a.Hk;
#define BK_LAUNCH_Q(DP, VEC, QB)                                                                                      \
  hipLaunchKernelGGL((bk_attn_dq_kernel<T, DP, VEC, QB>), dim3(work_grid(heads * ((a.L + 64 * QB - 1) / (64 * QB)))), \
                     dim3(256), 0, s, a)
#define BK_LAUNCH_K(DP, VEC, KB)                                                                                      \
  hipLaunchKernelGGL((bk_attn_dkv_kernel<T, DP, VEC, false, KB>),                                                     \
                     dim3(work_grid(kheads * ((a.L + 64 * KB - 1) / (64 * KB)))), dim3(256), 0, s, a)
#define BK_LAUNCH_S(DP, VEC, KB)                                                                                      \
  hipLaunchKernelGGL((bk_attn_dkv_kernel<T, DP, VEC, true, KB>),                                                      \
                     dim3(work_grid(kheads * ((a.S + 16 * KB - 1) / (16 * KB)) * a.nsplit)), dim3(256), 0, s, a)
#define BK_LAUNCH(DP, VEC)                                                                        \
  do {                                                                                            \
    if (a.wide_q) BK_LAUNCH_Q(DP, VEC, 2);                                                        \
    else BK_LAUNCH_Q(DP, VEC, 1);                                                                 \
    if (a.wide_k) BK_LAUNCH_K(DP, VEC, 2);                                                        \
    else BK_LAUNCH_K(DP, VEC, 1);                                                                 \
    if (a.nsplit && a.S > 16) BK_LAUNCH_S(DP, VEC, 2);                                            \
    else if (a.nsplit) BK_LAUNCH_S(DP, VEC, 1);                                                   \
  } while (0)
  BK_ATTN_DP(BK_LAUNCH);
#undef BK_LAUNCH
#undef BK_LAUNCH_Q
#undef BK_LAUNCH_K
#undef BK_LAUNCH_S
  if (a.nsplit) {
    const long per = (long)a.B * a.Hk * a.S * 2 * a.D;
    hipLaunchKernelGGL((bk_attn_sink_join_kernel<T>), dim3((unsigned)((per + 255) / 256)), dim3(256), 0, s, a);
  }
}

template <typename T>
void attn_step(const StepArgs &a, int dp, bool vec, hipStream_t s) {
  const unsigned grid = (unsigned)(a.B * a.Hk * a.hchunks * a.nsplit);
#define BK_LAUNCH(DP, VEC) hipLaunchKernelGGL((bk_attn_step_kernel<T, DP, VEC>), dim3(grid), dim3(256), 0, s, a)
  BK_ATTN_DP(BK_LAUNCH);
#undef BK_LAUNCH
  if (a.nsplit > 1)
    hipLaunchKernelGGL((bk_attn_step_join_kernel<T>), dim3((unsigned)(a.B * a.H)), dim3(128), 0, s, a);
}

}  // namespace bk
