// What the log-probability kernels share
#pragma once

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


struct TopMem {
  Key *list, *cand;   // the result, in order; what reaches the bound
  uint32_t cap;       // room in cand
  __host__ __device__ static constexpr uint32_t room(uint32_t k) { return 64 + 9 * k; }   // k vectors of equal elements and the single ones fit
};
// One class after the other, from classes [lo, hi): for rows that the bound does not serve
template <int NT, typename T>
__device__ void rounds(Group<NT>& g, const TopMem& t, const T* x, int64_t st, uint32_t lo, uint32_t hi, uint32_t k) {
  Key last = ~0ull;
  for (uint32_t i = 0; i < k; ++i) {
    Key best = 0;
    if (last)
      for (uint32_t c = lo + g.tid; c < hi; c += NT) {
        const float v = ld_f(x + c * st);
        const Key key = v == v ? key_of(v, c) : 0;
        if (key < last && key > best) best = key;
      }
    best = last = g.max(best);
    if (g.tid == 0) t.list[i] = best;
  }
  g.sync();
}

__device__ __forceinline__ void put_top(const LogprobP& p, const RowSums& s, size_t r, uint32_t at, Key key) {
  if (p.top_class) p.top_class[r * p.top + at] = key ? key_class(key) : kNoClass;
  if (p.top_logp) p.top_logp[r * p.top + at] = key ? s.log_p(key_value((uint32_t)(key >> 32)), p.scale) : -INFINITY;
}
__device__ __forceinline__ void put_row(const LogprobP& p, const RowSums& s, size_t r, float H, uint32_t l, float xl) {
  if (p.lse) p.lse[r] = s.lse(p.scale);
  if (p.entropy) p.entropy[r] = H < 0.f ? 0.f : H;   // by the rounding of log S and of E / S, where a row is nearly certain
  if (p.logp) p.logp[r] = l < p.x.C ? s.log_p(xl, p.scale) : 0.f;
}

// The gradient's factors: e (c0 + c1 u) with e = 2^u is scale p (A - dentropy (log p + H)); dl: what the label's class has besides
struct Factors {
  float c0, c1, dl, dh, dz;
  __device__ void fetch(const LogprobP& p, size_t r, uint32_t l) {
    dl = p.dlogp && l < p.x.C ? p.dlogp[r] : 0.f;
    dh = p.dentropy ? p.dentropy[r] : 0.f;
    dz = p.dlse ? p.dlse[r] : 0.f;
  }
  template <bool ENT> __device__ void set(const LogprobP& p, const RowSums& s, float H) {
    if (!s.some) dl = 0.f;
    const float A = dz - dl, k = s.some ? p.scale / s.S : 0.f;
    c1 = ENT ? -k * dh * kLn2 : 0.f;
    c0 = ENT ? k * (A - dh * (H - kLn2 * s.L)) : k * A;
    dl *= p.scale;
  }
  template <bool ENT> __device__ float grad(float x, float cs, float mc) const {
    float u = fmaf(x, cs, -mc);
    if (ENT) u = above_nothing(u);
    const float e = exp2_fast(u);
    return ENT ? entropy_grad(e, u, c0, c1) : e * c0;
  }
};

// A thread per position (logprob_pos.cu): AD_ERR_UNSUPPORTED where the rows are none for it
template <typename T> int logprob_positions(const LogprobP& p, cudaStream_t s);
template <typename T> int logprob_positions_bwd(const LogprobP& p, cudaStream_t s);

}  // namespace adk
