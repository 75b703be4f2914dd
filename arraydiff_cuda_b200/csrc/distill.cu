// Distillation from a teacher's top classes: the loss and its gradient.
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

// Any layout: a warp per row, an element per lane and step.  The gradient of a class outside of the list is
// dloss * scale * p_c * (Q - q_r / p_r), which the warp writes everywhere; the list's classes are read beforehand and written over it.
template <typename T, bool BWD>
__global__ void __launch_bounds__(256) distill_any(DistillP p) {
  grid_dependency();
  __shared__ uint32_t s_cls[8][kMostTop];
  __shared__ float s_q[8][kMostTop];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const size_t warp = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nw = ((size_t)gridDim.x * blockDim.x) >> 5;
  const uint32_t C = p.x.C, k = p.top;
  uint32_t* cls = s_cls[w];
  float* qs = s_q[w];
  for (size_t r = warp; r < p.x.rows; r += nw) {
    const T* x = (const T*)p.logits + p.x.offset(r);
    const int64_t st = p.x.step;
    // the list: a_j = log2 q_j
    float a[4], xj[4], am = -INFINITY;
    uint32_t cj[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t j = lane + 32 * i;
      cj[i] = j < k ? p.top_class[r * k + j] : kNoClass;
      a[i] = cj[i] < C ? p.top_logit[r * k + j] * p.ts : -INFINITY;
      xj[i] = cj[i] < C ? ld_f(x + cj[i] * st) : 0.f;
      am = fmaxf(am, a[i]);
    }
    float shift;
    if (p.rest) {
      shift = p.top_lse ? (float)(p.top_lse[r] * kLog2e) : 0.f;
    } else {
      am = warp_max(am);
      if (am == -INFINITY) am = 0.f;
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) z += exp2f(a[i] - am);
      z = warp_sum(z);
      shift = z != 0.f ? am + log2f(z) : 0.f;
    }
    float q[4], Q = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] -= shift;
      q[i] = exp2f(a[i]);
      Q += q[i];
      const uint32_t j = lane + 32 * i;
      if (j < k) { cls[j] = cj[i]; qs[j] = q[i]; }
    }
    Q = warp_sum(Q);
    __syncwarp();
    // every class, or with rest the classes outside of the list: reference m, sum R; the list's own beside them
    auto listed = [&](uint32_t c) {
      bool in = false;
      if (p.rest)
        for (uint32_t j = 0; j < k; ++j) in |= cls[j] == c;
      return in;
    };
    float m = -INFINITY, R = 0.f, mk = -INFINITY, K = 0.f;
    for (uint32_t c = lane; c < C; c += 32)
      if (!listed(c)) m = fmaxf(m, ld_f(x + c * st));
    m = warp_max(m);
    if (m == -INFINITY) m = 0.f;
    for (uint32_t c = lane; c < C; c += 32)
      if (!listed(c)) R += exp2_fast((ld_f(x + c * st) - m) * p.cs);
    R = warp_sum(R);
    if (p.rest) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (cj[i] < C) mk = fmaxf(mk, xj[i]);
      mk = warp_max(mk);
      if (mk == -INFINITY) mk = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (cj[i] < C) {   // a class that stands twice has its weight once
          bool first = true;
          for (uint32_t j = 0; j < (uint32_t)(lane + 32 * i); ++j) first &= cls[j] != cj[i];
          if (first) K += exp2_fast((xj[i] - mk) * p.cs);
        }
      K = warp_sum(K);
    }
    float S = R, mt = m, to = 0.f, L = 0.f;   // S against its own reference mt = m + to / cs
    if (K != 0.f) {
      if (R == 0.f) {
        S = K;
        mt = mk;
      } else if (m >= mk) {
        S = R + K * exp2_fast((mk - m) * p.cs);
      } else {
        to = (mk - m) * p.cs;
        S = K + R * exp2_fast(-to);
        mt = mk;
      }
    }
    const bool some = S != 0.f;
    if (some) L = log2f(S);
    const float qr = p.rest && R != 0.f ? fmaxf(1.f - Q, 0.f) : 0.f;
    float loss = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (q[i] != 0.f) loss += q[i] * (kLn2 * (a[i] + L) - (xj[i] - mt) * p.scale);
    loss = warp_sum(loss);
    if (qr > 0.f) loss += qr * (kLn2 * (log2f(qr) - log2f(R) + L) + (mt - m) * p.scale);
    if (lane == 0 && p.loss) p.loss[r] = some ? loss + 0.f * L : 0.f;   // NaN without any entry, too
    if constexpr (BWD) {
      T* g = (T*)p.dlogits + p.g.offset(r);
      const float d = p.dloss[r] * p.scale;
      float old[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) old[i] = p.accumulate && cj[i] < C ? ld_f(g + cj[i] * p.g.step) : 0.f;
      __syncwarp();
      Q += qr;
      const float rS = some ? 1.f / S : 0.f, out = some ? Q * rS * exp2_fast(-to) - (qr > 0.f ? qr / R : 0.f) : 0.f;
      for (uint32_t c = lane; c < C; c += 32) {
        float v = d * (exp2_fast((ld_f(x + c * st) - m) * p.cs) * out);
        if (p.accumulate) v += ld_f(g + c * p.g.step);
        st_f(g + c * p.g.step, v);
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (cj[i] < C) {
          float sum = 0.f;
          for (uint32_t j = 0; j < k; ++j) sum += cls[j] == cj[i] ? qs[j] : 0.f;
          const float v = some ? d * (exp2_fast((xj[i] - mt) * p.cs) * rS * Q - sum) : 0.f;
          st_f(g + cj[i] * p.g.step, p.accumulate ? old[i] + v : v);
        }
    }
    __syncwarp();
  }
}

static int distill_args(const ad_distill_args* a, bool bwd, DistillP& p) {
  if (!a) return AD_ERR_BAD_ARG;
  p = {};
  int rc = rows_of(a->dtype, a->layout, a->N, a->C, a->HW, a->pitch, p.x);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  if (!a->logits || !scale_ok(a->scale) || !scale_ok(a->top_scale)) return AD_ERR_BAD_ARG;
  if (a->top > kMostTop) return AD_ERR_LIMIT;
  if (a->top == 0 || !a->top_class || !a->top_logit) return AD_ERR_BAD_ARG;
  const size_t elem = (size_t)elem_size(a->dtype);
  if (!aligned_to(a->logits, elem)) return AD_ERR_ALIGN;
  p.logits = a->logits;
  p.scale = a->scale;
  p.cs = (float)(a->scale * kLog2e);
  p.top = a->top;
  p.rest = a->rest != 0;
  p.top_class = a->top_class;
  p.top_logit = a->top_logit;
  p.top_lse = a->top_lse;
  p.ts = (float)(a->top_scale * kLog2e);
  p.loss = a->loss;
  if (bwd) {
    rc = rows_of(a->dtype, a->layout, a->N, a->C, a->HW, a->dlogits_pitch, p.g);
    if (rc != AD_OK) return rc;
    if (!a->dlogits || !a->dloss) return AD_ERR_BAD_ARG;
    if (!aligned_to(a->dlogits, elem)) return AD_ERR_ALIGN;
    if (!gradient_clear(p.x, a->logits, p.g, a->dlogits, elem, a->accumulate)) return AD_ERR_BAD_ARG;
    p.dlogits = a->dlogits;
    p.dloss = a->dloss;
    p.accumulate = a->accumulate != 0;
  } else if (!a->loss) {
    return AD_ERR_BAD_ARG;
  }
  return AD_OK;
}

template <typename T, bool BWD>
static int launch_distill(const DistillP& p, cudaStream_t s) {
  launch(distill_any<T, BWD>, grid_for(p.x.rows, 8), 256, 0, s, p);
  count_launch();
  return launch_status();
}

}  // namespace adk

using namespace adk;

extern "C" int ad_distill_fwd(const ad_distill_args* a, void* stream) {
  DistillP p;
  const int rc = distill_args(a, false, p);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  AD_DISPATCH_DTYPE(a->dtype, return (launch_distill<T, false>(p, as_stream(stream))));
}

extern "C" int ad_distill_bwd(const ad_distill_args* a, void* stream) {
  DistillP p;
  const int rc = distill_args(a, true, p);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  AD_DISPATCH_DTYPE(a->dtype, return (launch_distill<T, true>(p, as_stream(stream))));
}
