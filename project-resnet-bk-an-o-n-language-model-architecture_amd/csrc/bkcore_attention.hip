// Entry points of sliding-window attention with sinks (kernels: bkcore_attention_impl.h) and the fill of a rolling cache
// from a prompt.
#include "bkcore_attention.h"

namespace {
using namespace bk;

inline int padded(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// 16-byte pieces of every row (8 elements; float32 as two)
inline bool rows_aligned(const Heads &x, int dtype) {
  const int v = 16 / elem_size(dtype);
  return aligned16(x.p) && x.b % v == 0 && x.h % v == 0 && x.t % v == 0;
}

// a tile of 128 rows within 32-bit offsets
inline bool near(const Heads &x) { return x.t >= 0 && x.t < (1 << 24); }

int check(int dtype, int64_t B, int64_t H, int64_t Hk, int64_t L, int64_t D, int64_t window, int64_t sinks, float scale) {
  if (!elem_size(dtype) || B < 0 || H < 1 || Hk < 1 || H % Hk || L < 0 || D < 1 || D > BKCORE_ATTENTION_MAX_HEAD_DIM)
    return BKCORE_EINVAL;
  if (window < 1 || sinks < 0 || sinks > BKCORE_ATTENTION_MAX_SINKS || scale != scale) return BKCORE_EINVAL;
  if (B > (1 << 14) || H > (1 << 14) || L > (1 << 30)) return BKCORE_EINVAL;
  return BKCORE_OK;
}

// 128 queries (keys) a workgroup read a key (query) tile half as often as 64; where that leaves compute units without a
// workgroup (there are 256), twice as many of the short ones are better off (8 x 8 heads x 256 x 32 float32, both passes:
// 69 us on the GPU with 128, 46 with 64).
inline int wide(int64_t heads, int64_t L) { return heads * ((L + 127) / 128) >= 256; }

// First query that only the sinks of the first key tile are left for: behind the tile's own queries.
inline int64_t sink_rest(int64_t W, int wide_k) { return ((64 * (1 + wide_k) - 1 + W - 1) / ATTN_BQ + 1) * ATTN_BQ; }

// Stretches of queries for the sinks' gradient: about two workgroups a CU together, at least 512 queries each.
inline int sink_splits(int64_t B, int64_t Hk, int64_t L, int64_t W, int64_t S) {
  const int64_t rest = L - sink_rest(W, wide(B * Hk, L));
  if (S == 0 || rest <= 0) return 0;
  int64_t n = 512 / (B * Hk * (S > 16 ? (S + 31) / 32 : 1));
  const int64_t most = (rest + 511) / 512;
  if (n > most) n = most;
  return n < 1 ? 1 : (int)n;
}

// Stretches of the visible positions of a step: four workgroups a CU together, at least 128 positions each.
inline int step_splits(int64_t items, int64_t span) {
  int64_t n = 1024 / (items > 0 ? items : 1);
  const int64_t most = (span + 127) / 128;
  if (n > most) n = most;
  if (n > 64) n = 64;
  return n < 1 ? 1 : (int)n;
}

template <typename T>
__global__ __launch_bounds__(256) void bk_attn_fill_kernel(Heads k, Heads v, Heads kc, Heads vc, const int *lengths, int B,
                                                           int Hk, int L, int cap, int D, int S, int rows) {
  const long id = (long)blockIdx.x * 256 + threadIdx.x;
  if (id >= (long)B * Hk * rows * D) return;
  const int d = (int)(id % D);
  long r = id / D;
  const int i = (int)(r % rows);  // of the positions that stay: the sinks, then the last cap - S behind them
  r /= rows;
  const int h = (int)(r % Hk), b = (int)(r / Hk);
  int len = lengths ? lengths[b] : L;
  len = len < 0 ? 0 : len > L ? L : len;
  const int ring = cap - S, first = len - ring > S ? len - ring : S;
  const int p = i < S ? i : first + i - S;
  if (p >= len) return;
  const long slot = p < S ? p : S + (p - S) % ring;
  ((T *)const_cast<void *>(kc.p))[b * kc.b + h * kc.h + slot * kc.t + d] = ((const T *)k.p)[b * k.b + h * k.h + p * k.t + d];
  ((T *)const_cast<void *>(vc.p))[b * vc.b + h * vc.h + slot * vc.t + d] = ((const T *)v.p)[b * v.b + h * v.h + p * v.t + d];
}

}  // namespace

extern "C" int bkcore_sliding_attention(const void *q, int64_t q_batch, int64_t q_head, int64_t q_time, const void *k,
                                        int64_t k_batch, int64_t k_head, int64_t k_time, const void *v, int64_t v_batch,
                                        int64_t v_head, int64_t v_time, int dtype, const int *lengths, int64_t B, int64_t H,
                                        int64_t Hk, int64_t L, int64_t D, int64_t window, int64_t sinks, float scale,
                                        void *out, void *out_lo, float *lse, void *stream) {
  const int rc = check(dtype, B, H, Hk, L, D, window, sinks, scale);
  if (rc) return rc;
  if (B == 0 || L == 0) return BKCORE_OK;
  if (!q || !k || !v || !out) return BKCORE_EINVAL;
  if (B * H * ((L + 63) / 64) > 2147483000LL) return BKCORE_EINVAL;
  AttnArgs a{};
  a.q = {q, q_batch, q_head, q_time};
  a.k = {k, k_batch, k_head, k_time};
  a.v = {v, v_batch, v_head, v_time};
  a.o = out; a.lo = out_lo; a.lse = lse; a.lengths = lengths;
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.L = (int)L; a.D = (int)D; a.S = (int)(sinks < L ? sinks : L);
  a.W = (int)(window < L ? window : L); a.scale = scale;
  a.wide_q = wide(B * H, L);
  if (!near(a.k) || !near(a.v)) return BKCORE_EINVAL;
  const bool vec = D % 8 == 0 && rows_aligned(a.q, dtype) && rows_aligned(a.k, dtype) && rows_aligned(a.v, dtype) &&
                   aligned16(out) && aligned16(out_lo);
  BK_WITH_TYPE(dtype, attn_forward<T>(a, padded(D), vec, (hipStream_t)stream));
  return launch_status();
}

extern "C" size_t bkcore_sliding_attention_backward_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t L, int64_t D,
                                                                    int64_t window, int64_t sinks) {
  if (check(BKCORE_F32, B, H, Hk, L, D, window, sinks, 1.0f) || B == 0 || L == 0) return 0;
  const int64_t W = window < L ? window : L, S = sinks < L ? sinks : L;
  const int ns = sink_splits(B, Hk, L, W, S);
  const size_t delta = ((size_t)B * H * L + 3) & ~(size_t)3;
  return (delta + (ns ? (size_t)(1 + 4 * ns) * B * Hk * S * 2 * D : 0)) * sizeof(float);
}

extern "C" int bkcore_sliding_attention_backward(
    const void *dout, int64_t do_batch, int64_t do_head, int64_t do_time, const void *q, int64_t q_batch, int64_t q_head,
    int64_t q_time, const void *k, int64_t k_batch, int64_t k_head, int64_t k_time, const void *v, int64_t v_batch,
    int64_t v_head, int64_t v_time, const void *out, const void *out_lo, const float *lse, int dtype, const int *lengths, int64_t B, int64_t H,
    int64_t Hk, int64_t L, int64_t D, int64_t window, int64_t sinks, float scale, void *dq, void *dk, void *dv,
    void *workspace, size_t workspace_bytes, void *stream) {
  const int rc = check(dtype, B, H, Hk, L, D, window, sinks, scale);
  if (rc) return rc;
  if (B == 0 || L == 0) return BKCORE_OK;
  if (!dout || !q || !k || !v || !out || !lse || !dq || !dk || !dv) return BKCORE_EINVAL;
  if (B * H * ((L + 63) / 64) > 2147483000LL) return BKCORE_EINVAL;
  if (!workspace || workspace_bytes < bkcore_sliding_attention_backward_workspace_bytes(B, H, Hk, L, D, window, sinks))
    return BKCORE_EWORKSPACE;
  AttnArgs a{};
  a.dout = {dout, do_batch, do_head, do_time};
  a.q = {q, q_batch, q_head, q_time};
  a.k = {k, k_batch, k_head, k_time};
  a.v = {v, v_batch, v_head, v_time};
  a.out = out; a.lo = const_cast<void *>(out_lo); a.lse = const_cast<float *>(lse); a.lengths = lengths; a.dq = dq; a.dk = dk; a.dv = dv;
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.L = (int)L; a.D = (int)D; a.S = (int)(sinks < L ? sinks : L);
  a.W = (int)(window < L ? window : L); a.scale = scale;
  a.wide_q = wide(B * H, L);
  a.wide_k = wide(B * Hk, L);
  a.rest = sink_rest(a.W, a.wide_k);
  a.nsplit = sink_splits(B, Hk, L, a.W, a.S);
  a.delta = (float *)workspace;
  a.part = a.delta + (((size_t)B * H * L + 3) & ~(size_t)3);
  if (!near(a.q) || !near(a.k) || !near(a.v) || !near(a.dout)) return BKCORE_EINVAL;
  const bool vec = D % 8 == 0 && rows_aligned(a.q, dtype) && rows_aligned(a.k, dtype) && rows_aligned(a.v, dtype) &&
                   rows_aligned(a.dout, dtype) && aligned16(out) && aligned16(out_lo) && aligned16(dq) && aligned16(dk) && aligned16(dv);
  BK_WITH_TYPE(dtype, attn_backward<T>(a, padded(D), vec, (hipStream_t)stream));
  return launch_status();
}

static int step_plan(int64_t B, int64_t H, int64_t Hk, int64_t window, int64_t sinks, int *hchunks, int *per) {
  *hchunks = (int)((H / Hk + 15) / 16);
  const int64_t span = window + sinks;
  const int ns = step_splits(B * Hk * *hchunks, span);
  *per = (int)(((span + ns - 1) / ns + 127) / 128 * 128);
  return (int)((span + *per - 1) / *per);
}

extern "C" size_t bkcore_sliding_attention_step_workspace_bytes(int64_t B, int64_t H, int64_t Hk, int64_t cap, int64_t D,
                                                                int64_t window, int64_t sinks) {
  if (check(BKCORE_F32, B, H, Hk, cap, D, window, sinks, 1.0f) || B == 0 || cap < window + sinks) return 0;
  int hc, per;
  const int ns = step_plan(B, H, Hk, window, sinks, &hc, &per);
  return ns > 1 ? (size_t)ns * B * H * (D + 2) * sizeof(float) : 0;
}

extern "C" int bkcore_sliding_attention_step(
    const void *q, int64_t q_batch, int64_t q_head, const void *k, int64_t k_batch, int64_t k_head, const void *v,
    int64_t v_batch, int64_t v_head, void *k_cache, int64_t kc_batch, int64_t kc_head, int64_t kc_slot, void *v_cache,
    int64_t vc_batch, int64_t vc_head, int64_t vc_slot, const int *positions, int dtype, int64_t B, int64_t H, int64_t Hk,
    int64_t cap, int64_t D, int64_t window, int64_t sinks, float scale, void *out, void *workspace, size_t workspace_bytes,
    void *stream) {
  const int rc = check(dtype, B, H, Hk, cap, D, window, sinks, scale);
  if (rc) return rc;
  if (B == 0) return BKCORE_OK;
  if (!q || !k || !v || !k_cache || !v_cache || !positions || !out || cap < window + sinks) return BKCORE_EINVAL;
  const size_t need = bkcore_sliding_attention_step_workspace_bytes(B, H, Hk, cap, D, window, sinks);
  if (need && (!workspace || workspace_bytes < need)) return BKCORE_EWORKSPACE;
  StepArgs a{};
  a.q = {q, q_batch, q_head, 0};
  a.k = {k, k_batch, k_head, 0};
  a.v = {v, v_batch, v_head, 0};
  a.kc = {k_cache, kc_batch, kc_head, kc_slot};
  a.vc = {v_cache, vc_batch, vc_head, vc_slot};
  a.positions = positions; a.o = out; a.part = (float *)workspace;
  a.B = (int)B; a.H = (int)H; a.Hk = (int)Hk; a.cap = (int)cap; a.D = (int)D; a.W = (int)window; a.S = (int)sinks;
  a.scale = scale;
  a.nsplit = step_plan(B, H, Hk, window, sinks, &a.hchunks, &a.per);
  if (B * Hk * a.hchunks * a.nsplit > 2147483000LL || B * H > 2147483000LL) return BKCORE_EINVAL;
  const bool vec = D % 8 == 0 && rows_aligned(a.q, dtype) && rows_aligned(a.k, dtype) && rows_aligned(a.v, dtype) &&
                   rows_aligned(a.kc, dtype) && rows_aligned(a.vc, dtype);
  BK_WITH_TYPE(dtype, attn_step<T>(a, padded(D), vec, (hipStream_t)stream));
  return launch_status();
}

extern "C" int bkcore_sliding_cache_fill(const void *k, int64_t k_batch, int64_t k_head, int64_t k_time, const void *v,
                                         int64_t v_batch, int64_t v_head, int64_t v_time, void *k_cache, int64_t kc_batch,
                                         int64_t kc_head, int64_t kc_slot, void *v_cache, int64_t vc_batch,
                                         int64_t vc_head, int64_t vc_slot, const int *lengths, int dtype, int64_t B,
                                         int64_t Hk, int64_t L, int64_t cap, int64_t D, int64_t sinks, void *stream) {
  const int rc = check(dtype, B, Hk, Hk, L, D, 1, sinks, 1.0f);
  if (rc) return rc;
  if (cap <= sinks || cap > (1 << 30)) return BKCORE_EINVAL;
  if (B == 0 || L == 0) return BKCORE_OK;
  if (!k || !v || !k_cache || !v_cache) return BKCORE_EINVAL;
  const int64_t rows = cap < L + sinks ? cap : L + sinks;  // positions that may stay, counted as the kernel counts them
  const int64_t blocks = (B * Hk * rows * D + 255) / 256;
  if (blocks > 2147483647LL) return BKCORE_EINVAL;
  const Heads hk = {k, k_batch, k_head, k_time}, hv = {v, v_batch, v_head, v_time};
  const Heads ck = {k_cache, kc_batch, kc_head, kc_slot}, cv = {v_cache, vc_batch, vc_head, vc_slot};
  BK_WITH_TYPE(dtype, hipLaunchKernelGGL((bk_attn_fill_kernel<T>), dim3((unsigned)blocks), dim3(256), 0,
                                         (hipStream_t)stream, hk, hv, ck, cv, lengths, (int)B, (int)Hk, (int)L, (int)cap,
                                         (int)D, (int)sinks, (int)rows));
  return launch_status();
}
