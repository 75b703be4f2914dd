// What the distillation kernels share
#pragma once

#include "rows.cuh"

namespace adk {

struct DistillP {
  Rows x, g;
  const void* logits;
  void* dlogits;
  float scale, cs;
  uint32_t top;
  int rest;
  const uint32_t* top_class;
  const float *top_logit, *top_lse;
  float ts;              // top_scale * log2(e)
  float* loss;
  const float* dloss;
  int accumulate;
};

// What is known of a row when its list and its classes have been summed
struct Distilled {
  float S, mt, L;      // the row's sum against mt, a maximum, and its log2
  float off, offt;     // roundings of the references of the pass's sum and of S
  float qr, Q;         // q_r, sum q + q_r
  float out, rS;       // gradient outside of the list: dloss * scale * out * 2^u with u as in the pass; p of a listed class: 2^((x - mt) cs) rS
  bool some;
  __device__ float term(float q, float a, float x, float scale) const { return q != 0.f ? __fmul_rn(q, fmaf(kLn2, a + L + offt, -__fmul_rn(x - mt, scale))) : 0.f; }
};
// R: the pass's sum, of all classes or (rest) of those outside of the list, against m * cs + off.  K: the list's share of the
// row (rest), each class once, against mk.
__device__ __forceinline__ Distilled row_sums(const DistillP& p, float m, float off, float R, float mk, float K, float Q, float& rest_loss) {
  Distilled d;
  float to = 0.f;
  if (m == -INFINITY) m = 0.f;
  d.S = R;
  d.mt = m;
  bool by_list = false;
  if (K != 0.f) {
    if (R == 0.f) {
      d.S = K;
      by_list = true;
    } else if (m >= mk) {
      d.S = fmaf(K, exp2_fast(fmaf(mk - m, p.cs, -off)), R);
    } else {
      to = (mk - m) * p.cs - off;
      d.S = K + R * exp2_fast(-to);
      by_list = true;
    }
    if (by_list) d.mt = mk;
  }
  d.off = off;
  d.offt = by_list ? 0.f : off;
  d.some = d.S != 0.f;
  d.L = d.some ? log2f(d.S) : 0.f;
  d.qr = p.rest && R != 0.f ? fmaxf(1.f - Q, 0.f) : 0.f;
  d.Q = Q + d.qr;
  d.rS = d.some ? 1.f / d.S : 0.f;
  d.out = d.some ? d.Q * d.rS * exp2_fast(-to) - (d.qr > 0.f ? d.qr / R : 0.f) : 0.f;
  d.rS *= exp2_fast(-d.offt);
  rest_loss = d.qr > 0.f ? d.qr * (kLn2 * (log2f(d.qr) - log2f(R) + d.L + (d.offt - off)) + (d.mt - m) * p.scale) : 0.f;
  return d;
}

// A thread per position (distill_pos.cu): AD_ERR_UNSUPPORTED where the rows are none for it
template <typename T, bool BWD> int distill_positions(const DistillP& p, cudaStream_t s);

}  // namespace adk
