// Rows of logits: what the log-probability and the distillation kernels share.
//
// A row's numbers are worked out in units of log 2: with m the row's maximum, cs = scale * log2(e) and u_c = (x_c - m) * cs,
//   S = sum 2^u_c,   log2 p_c = u_c - log2 S,   lse = scale * m + ln2 * log2 S,
//   entropy = ln2 * (log2 S - sum 2^u_c u_c / S).
// A row of -inf takes m = 0: every term is 0 and so is S, which is how it is recognised afterwards.
#pragma once

#include "common.cuh"

namespace adk {

constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2e = 1.442695040888963407;
constexpr uint32_t kMostTop = 128;                 // entries of a row's list
constexpr uint32_t kNoClass = 0xffffffffu;

// Where the rows lie: row r's class c is at offset(r) + c * step (elements)
struct Rows {
  size_t rows;
  uint32_t C, HW;      // HW: positions per image where classes lie in planes, else 0
  int64_t pitch, step, image;
  __host__ __device__ size_t offset(size_t r) const { return HW ? (r / HW) * (size_t)image + r % HW : r * (size_t)pitch; }
};

// Checks what both operators' arguments have in common.  AD_OK with r.rows == 0: nothing to do.
inline int rows_of(int32_t dtype, int32_t layout, uint32_t N, uint32_t C, uint32_t HW, int64_t pitch, Rows& r) {
  r = {};
  if (layout != AD_NCHW && layout != AD_NHWC) return AD_ERR_UNSUPPORTED;
  if (dtype != AD_F32 && dtype != AD_BF16) return AD_ERR_UNSUPPORTED;
  if (C == 0 || pitch < 0) return AD_ERR_BAD_ARG;
  if (C > (1u << 30)) return AD_ERR_LIMIT;
  r.rows = (size_t)N * HW;
  r.C = C;
  if (layout == AD_NHWC) {
    if (pitch && pitch < (int64_t)C) return AD_ERR_BAD_ARG;
    r.pitch = pitch ? pitch : C;
    r.step = 1;
  } else {
    if (pitch && pitch < (int64_t)HW) return AD_ERR_BAD_ARG;
    const int64_t plane = pitch ? pitch : HW;
    r.image = plane * C;
    r.step = plane;
    r.HW = HW;
    if (plane == 1) {   // one position per image: the rows of a matrix
      r.HW = 0;
      r.pitch = C;
    }
  }
  return AD_OK;
}
// Elements from the first of row 0 to behind the last one
inline size_t rows_extent(const Rows& r) {
  if (r.rows == 0) return 0;
  return r.offset(r.rows - 1) + (size_t)(r.C - 1) * (size_t)r.step + 1;
}
// A gradient is the logits themselves, element for element, or shares nothing with them
inline bool gradient_clear(const Rows& x, const void* logits, const Rows& g, const void* dlogits, size_t elem, int32_t accumulate) {
  const uintptr_t a = (uintptr_t)logits, b = (uintptr_t)dlogits;
  if (a == b && x.pitch == g.pitch && x.step == g.step) return !accumulate;
  return a + rows_extent(x) * elem <= b || b + rows_extent(g) * elem <= a;
}
inline bool scale_ok(float s) { return s >= 1e-30f && s <= 1e30f; }
inline bool aligned_to(const void* p, size_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));   // 2 ulp; -inf gives 0
  return r;
}

// In front of: the larger value, then the lower class
__device__ __forceinline__ bool in_front(float v, uint32_t c, float w, uint32_t d) { return v > w || (v == w && c < d); }

}  // namespace adk
