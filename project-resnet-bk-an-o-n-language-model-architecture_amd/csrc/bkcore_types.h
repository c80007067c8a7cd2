// Element types and small wave / workgroup helpers shared by the layer operators (norm, convolution, scan, attention).
// Device code only; 64-lane waves.
#ifndef BKCORE_TYPES_H
#define BKCORE_TYPES_H
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/bkcore.h"
#include "bkcore_internal.h"

namespace bk {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef float f32x4 __attribute__((ext_vector_type(4)));

// BKCORE_OK, or BKCORE_ELAUNCH with the HIP code recorded for bkcore_last_hip_error()
inline int launch_status() {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return BKCORE_OK;
  bkcore_internal_set_hip_error((int)e);
  return BKCORE_ELAUNCH;
}

inline int elem_size(int dtype) { return dtype == BKCORE_F32 ? 4 : (dtype == BKCORE_BF16 || dtype == BKCORE_F16) ? 2 : 0; }
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }

// Runs CALL with T bound to the element type of dtype (one of BKCORE_F32 / BF16 / F16; checked by the caller).
#define BK_WITH_TYPE(dtype, ...)                    \
  do {                                              \
    if ((dtype) == BKCORE_F32) {                    \
      using T = float;                              \
      __VA_ARGS__;                                  \
    } else if ((dtype) == BKCORE_BF16) {            \
      using T = bk::bf16_t;                         \
      __VA_ARGS__;                                  \
    } else {                                        \
      using T = bk::f16_t;                          \
      __VA_ARGS__;                                  \
    }                                               \
  } while (0)

// V consecutive elements as floats.  V * sizeof(T) is 16 on the aligned paths (one 16-byte access) and V is 1 elsewhere.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T *__restrict__ p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = (float)p[0];
  } else {
    typedef T vec_t __attribute__((ext_vector_type(V)));
    const vec_t w = *reinterpret_cast<const vec_t *>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = (float)w[i];
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T *__restrict__ p, const float (&v)[V]) {
  if constexpr (V == 1) {
    p[0] = (T)v[0];  // round to nearest even, as the tensor library rounds
  } else {
    typedef T vec_t __attribute__((ext_vector_type(V)));
    vec_t w;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = (T)v[i];
    *reinterpret_cast<vec_t *>(p) = w;
  }
}

// A parameter vector (weight, bias) in float32 or in the operand's type.
template <typename T, int V>
__device__ __forceinline__ void load_param(const void *__restrict__ p, bool is_f32, long i, float (&v)[V]) {
  if (is_f32) {
    const float *q = (const float *)p + i;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = q[k];
  } else {
    const T *q = (const T *)p + i;
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = (float)q[k];
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp_mov(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, true));
}
constexpr int DPP_XOR1 = 0xB1;   // quad_perm:[1,0,3,2]
constexpr int DPP_XOR2 = 0x4E;   // quad_perm:[2,3,0,1]
constexpr int DPP_HALF_MIRROR = 0x141;
constexpr int DPP_MIRROR = 0x140;
constexpr int DPP_ROR4 = 0x124;
constexpr int DPP_ROR8 = 0x128;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
// x in lanes 0-31 becomes {x.lo + x.hi} there, y's sum goes to lanes 32-63 (one exchange reduces two registers to one).
__device__ __forceinline__ float fold32(float x, float y) {
  const u32x2 r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The same between neighbouring rows of 16 lanes: rows 0, 2 hold x's sums of rows (0,1), (2,3), rows 1, 3 hold y's.
__device__ __forceinline__ float fold16(float x, float y) {
  const u32x2 r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(y), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over the 64 lanes of a wave, the result in every lane; the order of the additions is fixed.
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp_mov<DPP_XOR1>(x);
  x += dpp_mov<DPP_XOR2>(x);
  x += dpp_mov<DPP_HALF_MIRROR>(x);
  x += dpp_mov<DPP_MIRROR>(x);
  x = fold16(x, x);
  return fold32(x, x);
}

// exp(x) through the base-2 instruction: one part in 2^21 at |x| <= 4, 2^20 at |x| <= 16, growing with |x| by the rounding
// of the product x log2(e).
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * LOG2E));
}

// V neighbouring elements of a row, at 16-byte (ALIGNED) or at any addresses: held raw until they are
// used, so that several loads are under way before the first is waited for (a load converted where it is issued, or issued
// under a condition, is waited for at once).
template <typename T, int V, bool ALIGNED>
struct Piece {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  typedef vec_t mem_t __attribute__((aligned(ALIGNED ? sizeof(T) * V : sizeof(T))));
  vec_t w;
  __device__ __forceinline__ void load(const T *__restrict__ p) { w = *reinterpret_cast<const mem_t *>(p); }
  __device__ __forceinline__ void get(bool in, float (&v)[V]) const {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = in ? (float)w[i] : 0.0f;
  }
  static __device__ __forceinline__ void store(T *__restrict__ p, const float (&v)[V]) {
    vec_t w;
#pragma unroll
    for (int i = 0; i < V; ++i) w[i] = (T)v[i];
    *reinterpret_cast<mem_t *>(p) = w;
  }
};
template <typename T, bool ALIGNED>
struct Piece<T, 1, ALIGNED> {
  T w;
  __device__ __forceinline__ void load(const T *__restrict__ p) { w = *p; }
  __device__ __forceinline__ void get(bool in, float (&v)[1]) const { v[0] = in ? (float)w : 0.0f; }
  static __device__ __forceinline__ void store(T *__restrict__ p, const float (&v)[1]) { *p = (T)v[0]; }
};

}  // namespace bk

// out[c] = sum over p < parts of part[p * cols + c], written in the order of the parts (bkcore_norm.hip).
extern "C" __attribute__((visibility("hidden"))) void bkcore_internal_sum_parts(const float *part, int64_t parts,
                                                                                int64_t cols, float *out, void *stream);
#endif
