// Log probabilities of given classes, with entropy, rank and top alternatives, and their gradient.
#include "rows.cuh"

namespace adk {

struct LogprobP {
  Rows x, g;
  const void *logits;
  void* dlogits;
  float scale, cs;
  const uint32_t* label;
  float *lse, *entropy, *logp;
  uint32_t *rank, *top_class;
  float* top_logp;
  uint32_t top;
  const float *dlse, *dentropy, *dlogp;
  int accumulate;
};

// Any layout: a warp per row, an element per lane and step
template <typename T, bool BWD>
__global__ void __launch_bounds__(256) logprob_any(LogprobP p) {
  grid_dependency();
  const int lane = threadIdx.x & 31;
  const size_t warp = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nw = ((size_t)gridDim.x * blockDim.x) >> 5;
  const uint32_t C = p.x.C;
  for (size_t r = warp; r < p.x.rows; r += nw) {
    const T* x = (const T*)p.logits + p.x.offset(r);
    const int64_t st = p.x.step;
    float m = -INFINITY;
    for (uint32_t c = lane; c < C; c += 32) m = fmaxf(m, ld_f(x + c * st));
    m = warp_max(m);
    if (m == -INFINITY) m = 0.f;
    const uint32_t l = p.label ? p.label[r] : kNoClass;
    const float xl = l < C ? ld_f(x + l * st) : 0.f;
    float S = 0.f, E = 0.f;
    uint32_t cnt = 0;
    for (uint32_t c = lane; c < C; c += 32) {
      const float v = ld_f(x + c * st), u = (v - m) * p.cs, e = exp2_fast(u);
      S += e;
      if (e > 0.f) E += e * u;
      cnt += in_front(v, c, xl, l) ? 1u : 0u;
    }
    S = warp_sum(S);
    E = warp_sum(E);
    const bool some = S != 0.f;
    const float L = some ? log2f(S) : 0.f;
    const float H = some ? kLn2 * (L - E / S) : 0.f;
    const float lp = l >= C ? 0.f : (some ? (xl - m) * p.scale - kLn2 * L : -INFINITY);
    if (lane == 0) {
      if (p.lse) p.lse[r] = some ? m * p.scale + kLn2 * L : -INFINITY;
      if (p.entropy) p.entropy[r] = H;
      if (p.logp) p.logp[r] = lp;
    }
    if constexpr (!BWD) {
      if (p.rank) {
        cnt = __reduce_add_sync(0xffffffffu, cnt);
        if (lane == 0) p.rank[r] = l < C ? cnt : kNoClass;
      }
      float lv = 0.f;
      uint32_t lc = kNoClass;
      for (uint32_t k = 0; k < p.top; ++k) {
        float bv = 0.f;
        uint32_t bc = kNoClass;
        for (uint32_t c = lane; c < C; c += 32) {
          const float v = ld_f(x + c * st);
          if (v != v || (k > 0 && !in_front(lv, lc, v, c))) continue;
          if (bc == kNoClass || in_front(v, c, bv, bc)) { bv = v; bc = c; }
        }
        for (int o = 16; o > 0; o >>= 1) {
          const float ov = __shfl_xor_sync(0xffffffffu, bv, o);
          const uint32_t oc = __shfl_xor_sync(0xffffffffu, bc, o);
          if (oc != kNoClass && (bc == kNoClass || in_front(ov, oc, bv, bc))) { bv = ov; bc = oc; }
        }
        if (lane == 0) {
          if (p.top_class) p.top_class[r * p.top + k] = bc;
          if (p.top_logp) p.top_logp[r * p.top + k] = bc == kNoClass || !some ? -INFINITY : (bv - m) * p.scale - kLn2 * L;
        }
        lv = bv;
        lc = bc;
        if (bc == kNoClass) {   // no more classes
          for (uint32_t q = k + 1 + lane; q < p.top; q += 32) {
            if (p.top_class) p.top_class[r * p.top + q] = kNoClass;
            if (p.top_logp) p.top_logp[r * p.top + q] = -INFINITY;
          }
          break;
        }
      }
    } else {
      const float dl = p.dlogp && l < C && some ? p.dlogp[r] : 0.f, dh = p.dentropy ? p.dentropy[r] : 0.f;
      const float A = (p.dlse ? p.dlse[r] : 0.f) - dl, rS = some ? 1.f / S : 0.f;
      T* g = (T*)p.dlogits + p.g.offset(r);
      for (uint32_t c = lane; c < C; c += 32) {
        const float u = (ld_f(x + c * st) - m) * p.cs, pc = exp2_fast(u) * rS;
        float d = pc * A;
        if (p.dentropy && pc != 0.f) d -= dh * pc * (kLn2 * (u - L) + H);
        if (c == l) d += dl;
        d *= p.scale;
        if (p.accumulate) d += ld_f(g + c * p.g.step);
        st_f(g + c * p.g.step, d);
      }
    }
  }
}

static int logprob_args(const ad_logprob_args* a, bool bwd, LogprobP& p) {
  if (!a) return AD_ERR_BAD_ARG;
  p = {};
  int rc = rows_of(a->dtype, a->layout, a->N, a->C, a->HW, a->pitch, p.x);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  if (!a->logits || !scale_ok(a->scale)) return AD_ERR_BAD_ARG;
  const size_t elem = (size_t)elem_size(a->dtype);
  if (!aligned_to(a->logits, elem)) return AD_ERR_ALIGN;
  p.logits = a->logits;
  p.scale = a->scale;
  p.cs = (float)(a->scale * kLog2e);
  p.label = a->label;
  p.lse = a->lse;
  p.entropy = a->entropy;
  p.logp = a->logp;
  if (a->logp && !a->label) return AD_ERR_BAD_ARG;
  if (bwd) {
    rc = rows_of(a->dtype, a->layout, a->N, a->C, a->HW, a->dlogits_pitch, p.g);
    if (rc != AD_OK) return rc;
    if (!a->dlogits || (!a->dlse && !a->dentropy && !a->dlogp) || (a->dlogp && !a->label)) return AD_ERR_BAD_ARG;
    if (!aligned_to(a->dlogits, elem)) return AD_ERR_ALIGN;
    if (!gradient_clear(p.x, a->logits, p.g, a->dlogits, elem, a->accumulate)) return AD_ERR_BAD_ARG;
    p.dlogits = a->dlogits;
    p.dlse = a->dlse;
    p.dentropy = a->dentropy;
    p.dlogp = a->dlogp;
    p.accumulate = a->accumulate != 0;
  } else {
    if (a->rank && !a->label) return AD_ERR_BAD_ARG;
    if (a->top > kMostTop) return AD_ERR_LIMIT;
    if (a->top && !a->top_class && !a->top_logp) return AD_ERR_BAD_ARG;
    if (!a->lse && !a->entropy && !a->logp && !a->rank && !a->top) return AD_ERR_BAD_ARG;
    p.rank = a->rank;
    p.top = a->top;
    p.top_class = a->top_class;
    p.top_logp = a->top_logp;
  }
  return AD_OK;
}

template <typename T, bool BWD>
static int launch_logprob(const LogprobP& p, cudaStream_t s) {
  launch(logprob_any<T, BWD>, grid_for(p.x.rows, 8), 256, 0, s, p);
  count_launch();
  return launch_status();
}

}  // namespace adk

using namespace adk;

extern "C" int ad_logprob_fwd(const ad_logprob_args* a, void* stream) {
  LogprobP p;
  const int rc = logprob_args(a, false, p);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  AD_DISPATCH_DTYPE(a->dtype, return (launch_logprob<T, false>(p, as_stream(stream))));
}

extern "C" int ad_logprob_bwd(const ad_logprob_args* a, void* stream) {
  LogprobP p;
  const int rc = logprob_args(a, true, p);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  AD_DISPATCH_DTYPE(a->dtype, return (launch_logprob<T, true>(p, as_stream(stream))));
}
