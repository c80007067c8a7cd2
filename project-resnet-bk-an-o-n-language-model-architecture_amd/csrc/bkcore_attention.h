// Sliding-window attention with sinks: what the translation units of one operand type each (bkcore_attention_<type>.hip)
// share with the entry points (bkcore_attention.hip).
#ifndef BKCORE_ATTENTION_H
#define BKCORE_ATTENTION_H
#include "bkcore_types.h"

namespace bk {

// A (batch, head, position, d) operand: d has stride 1.
struct Heads {
  const void *p;
  long b, h, t;
};

struct AttnArgs {
  Heads q, k, v, dout;
  const void *out;          // forward's output for the backward, (B, L, H, D) contiguous like o, dq, dk, dv
  void *o, *dq, *dk, *dv;
  void *lo;                 // what rounding took from the output, for delta (16-bit operands; may be null)
  float *lse, *delta, *part;  // log2 of the row's sum, (B, H, L); rows that see nothing hold +inf
  const int *lengths;
  int B, H, Hk, L, D, W, S;
  float scale;
  int nsplit;         // sinks' gradient: stretches of queries behind the first key tile's own ...
  long rest;          // ... which end here
  int wide_q, wide_k; // 128 queries / keys a workgroup, else 64
};

struct StepArgs {
  Heads q, k, v, kc, vc;  // q, k, v: t unused; caches: t is the slot's stride
  const int *positions;
  void *o;
  float *part;  // (split, B, H, D + 2): unnormalised output, maximum, sum
  int B, H, Hk, cap, D, W, S, nsplit, per, hchunks;
  float scale;
};

constexpr int ATTN_BQ = 32;  // queries of one tile of a dk, dv workgroup
constexpr int SINK_TILE = 4 * ATTN_BQ;  // queries a workgroup of the sinks' gradient takes at once: 32 a wave

template <typename T>
void attn_forward(const AttnArgs &a, int dp, bool vec, hipStream_t s);
template <typename T>
void attn_backward(const AttnArgs &a, int dp, bool vec, hipStream_t s);
template <typename T>
void attn_step(const StepArgs &a, int dp, bool vec, hipStream_t s);

}  // namespace bk
#endif
