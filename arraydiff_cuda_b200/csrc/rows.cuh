// Rows of logits: what the log-probability and the distillation kernels share.
//
// A row's numbers are worked out in units of log 2: with m the row's maximum, cs = scale * log2(e), mc = m * cs as rounded,
//   u_c = x_c * cs - mc (one FMA),   S = sum 2^u_c,   E = sum 2^u_c u_c,   p_c = 2^u_c / S,
//   entropy = ln2 (log2 S - E / S),   log p_c = scale (x_c - m) - ln2 (log2 S + (mc - m * cs)),
// where mc - m * cs, the rounding of mc, is what an FMA gives.  One pass over the row: a thread keeps its own maximum,
// and S and E against it, and rescales them when the maximum of a batch of loads is larger.
// mc is off by up to 2^-24 of itself, and the terms by 2 to that: a row whose maximum is beyond +-kFar in units of log 2, or
// that holds +inf or NaN, is done again by plain loops over x_c - m; a list of the former, and its rank, stand.  A share's
// reference is at least kFloor, so that what is masked (-inf, the type's lowest value, -1e9) adds 2^-4e6 = 0 to the row and never
// inf or inf - inf.
// A row of -inf has S = 0, which is how it is recognised.
#pragma once

#include "cluster_counts.h"
#include "common.cuh"

namespace adk {

constexpr float kLn2 = 0.693147180559945309f;
constexpr double kLog2e = 1.442695040888963407;
constexpr uint32_t kMostTop = 128;                 // entries of a row's list
constexpr uint32_t kNoClass = 0xffffffffu;
constexpr float kFloor = -4e6f, kFar = 1e6f;

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
template <typename... P> inline bool words(P... p) { return ((aligned_to(p, 4)) && ...); }

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));   // 2 ulp; -inf gives 0
  return r;
}
__device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint4 load_shared(uint32_t a) {
  uint4 w;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(a) : "memory");
  return w;
}
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory"); }
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// two fp32 numbers at once
typedef unsigned long long F2;
__device__ __forceinline__ F2 pair(float a, float b) { F2 r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ float2 halves(F2 v) { float2 r; asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v)); return r; }
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) { F2 r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ F2 add2(F2 a, F2 b) { F2 r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) { F2 r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// v, not below -200 (2^-200 is 0 here), and NaN where v is: what may be multiplied by its exponential
__device__ __forceinline__ float above_nothing(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-200.f));
  return r;
}

// v, not above w, and NaN where v is
__device__ __forceinline__ float not_above(float v, float w) {
  float r;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(w));
  return r;
}

// In front of: the larger value, then the lower class
__device__ __forceinline__ bool in_front(float v, uint32_t c, float w, uint32_t d) { return v > w || (v == w && c < d); }
// The same order as whole numbers.  -0 and 0 are one value.
__device__ __forceinline__ uint32_t value_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu)); }
typedef unsigned long long Key;   // value, then the complement of the class; 0: none
__device__ __forceinline__ Key key_of(float v, uint32_t c) { return (Key)value_key(v) << 32 | (uint32_t)~c; }
__device__ __forceinline__ uint32_t key_class(Key k) { return ~(uint32_t)k; }

// ---- threads that work on one row: a warp, or NT threads of a block with `red` (8 bytes for each warp)
template <int NT> struct Group;
template <> struct Group<32> {
  uint32_t tid = threadIdx.x & 31;
  __device__ explicit Group(void*) {}
  __device__ void sync() { __syncwarp(); }
  __device__ float max(float v) { return warp_max(v); }
  __device__ float sum(float v) { return warp_sum(v); }
  __device__ uint32_t sum(uint32_t v) { return __reduce_add_sync(0xffffffffu, v); }
  __device__ Key max(Key v) {
    const uint32_t h = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32));
    const uint32_t l = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32) == h ? (uint32_t)v : 0u);
    return (Key)h << 32 | l;
  }
};
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
template <int NT> struct Group {
  uint32_t tid = threadIdx.x;
  Key* red;   // one per warp
  __device__ explicit Group(void* r) : red((Key*)r) {}
  __device__ void sync() { __syncwarp(); asm volatile("bar.sync 9, %0;" ::"n"(NT) : "memory"); }   // these threads alone: a block may have more
  template <typename V, typename F>
  __device__ V all(V w, F f) {   // of the warps' values, in order
    sync();
    if ((tid & 31) == 0) *(V*)&red[tid >> 5] = w;
    sync();
    V v = *(V*)&red[0];
#pragma unroll
    for (int i = 1; i < NT / 32; ++i) v = f(v, *(V*)&red[i]);
    return v;
  }
  __device__ float max(float v) { return all(warp_max(v), [](float a, float b) { return fmaxf(a, b); }); }
  __device__ float sum(float v) { return all(warp_sum(v), [](float a, float b) { return a + b; }); }
  __device__ uint32_t sum(uint32_t v) { return all(__reduce_add_sync(0xffffffffu, v), [](uint32_t a, uint32_t b) { return a + b; }); }
  __device__ Key max(Key v);
};
template <int NT> __device__ Key Group<NT>::max(Key v) { return all(Group<32>(nullptr).max(v), [](Key a, Key b) { return a > b ? a : b; }); }

// ---- 16 bytes of a row
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int V = 4;
  typedef float Max;
  __device__ static uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  __device__ static void unpack(uint4 w, float* f) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
  __device__ static float element(uint4 w, uint32_t i) { return __uint_as_float(i & 2 ? (i & 1 ? w.w : w.z) : (i & 1 ? w.y : w.x)); }
  __device__ static uint4 pack(const float* f) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  __device__ static Max max(uint4 w) {
    float f[4];
    unpack(w, f);
    return fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3]));
  }
  __device__ static Max max(Max a, Max b) { return fmaxf(a, b); }
  __device__ static float value(Max a) { return a; }
  // not below v, NaN as it is
  __device__ static uint4 above_or(uint4 w, float v) {
    uint32_t* p = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+r"(p[i]) : "r"(__float_as_uint(v)));
    return w;
  }
  __device__ static uint32_t above(uint4 w, float t) {
    return (__uint_as_float(w.x) > t) + (__uint_as_float(w.y) > t) + (__uint_as_float(w.z) > t) + (__uint_as_float(w.w) > t);
  }
  __device__ static float below(float v) {   // the next lower number
    const uint32_t b = __float_as_uint(v);
    return __uint_as_float((b << 1) == 0 ? 0x80000001u : b >> 31 ? b + 1 : b - 1);
  }
  static constexpr int kKeyShift = 0;   // low bits of a value's key that say nothing
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int V = 8;
  typedef __nv_bfloat162 Max;
  __device__ static __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); }
  __device__ static uint4 none() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
  __device__ static void unpack(uint4 w, float* f) {
    const uint32_t* p = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(p[i] << 16); f[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u); }
  }
  __device__ static float element(uint4 w, uint32_t i) {
    const uint32_t q = i & 4 ? (i & 2 ? w.w : w.z) : (i & 2 ? w.y : w.x);
    return __uint_as_float(i & 1 ? q & 0xffff0000u : q << 16);
  }
  __device__ static uint4 pack(const float* f) {
    uint4 w;
    uint32_t* p = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      p[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return w;
  }
  __device__ static Max max(uint4 w) { return __hmax2(__hmax2(two(w.x), two(w.y)), __hmax2(two(w.z), two(w.w))); }
  __device__ static Max max(Max a, Max b) { return __hmax2(a, b); }
  __device__ static uint4 above_or(uint4 w, float v) {
    const __nv_bfloat162 t = __float2bfloat162_rn(v);
    uint32_t* p = &w.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 m = __hmax2_nan(two(p[i]), t);
      p[i] = *reinterpret_cast<const uint32_t*>(&m);
    }
    return w;
  }
  __device__ static float value(Max a) { return fmaxf(__low2float(a), __high2float(a)); }
  __device__ static uint32_t above(uint4 w, float t) {
    const __nv_bfloat162 tt = __float2bfloat162_rn(t);
    // masks of 0xffff: with a set in the low halves and b in the high ones the sum is -a + ((a - b) << 16)
    const uint32_t s = __hgt2_mask(two(w.x), tt) + __hgt2_mask(two(w.y), tt) + __hgt2_mask(two(w.z), tt) + __hgt2_mask(two(w.w), tt);
    const uint32_t a = (0u - s) & 0xffffu;
    return a + ((a - ((s + a) >> 16)) & 0xffffu);
  }
  __device__ static float below(float v) {
    const uint32_t b = __float_as_uint(v);
    return __uint_as_float((b << 1) == 0 ? 0x80010000u : b >> 31 ? b + 0x10000u : b - 0x10000u);
  }
  static constexpr int kKeyShift = 16;
};

// A row as single elements up to a 16-byte boundary, vectors, and single elements behind them; of a row that the blocks of a
// cluster share, the vectors [vb, ve), the elements in front with the first block, those behind with the last.
template <typename T>
struct Strip {
  static constexpr uint32_t V = Vec<T>::V;
  uint32_t head, nv, tail, vb, ve;
  bool first, last;
  __device__ Strip(const T* x, uint32_t C, uint32_t part = 0, uint32_t parts = 1) {
    head = (uint32_t)((0u - (uint32_t)(uintptr_t)x) & 15u) / (uint32_t)sizeof(T);
    if (head > C) head = C;
    nv = (C - head) / V;
    tail = C - head - nv * V;
    vb = (uint32_t)((uint64_t)nv * part / parts);
    ve = (uint32_t)((uint64_t)nv * (part + 1) / parts);
    first = part == 0;
    last = part + 1 == parts;
  }
  __device__ uint32_t class_of(uint32_t v) const { return head + v * V; }
  // the single elements, at most 2 V - 2 of them: thread i has its i-th, or none
  __device__ uint32_t single(uint32_t i) const {
    if (i < V) return first && i < head ? i : kNoClass;
    return last && i - V < tail ? head + nv * V + (i - V) : kNoClass;
  }
  __device__ uint32_t begin() const { return first ? 0u : class_of(vb); }
  __device__ uint32_t end() const { return last ? head + nv * V + tail : class_of(ve); }
};

// What a thread, a group or a block of a cluster knows about its share of a row.  S and E stand against mc, which follows the
// maximum when that is kAhead beyond it (a term is then 2^kAhead at most), and is moved to the maximum when shares are joined.
constexpr float kAhead = 16.f;
struct Part {
  float m, mc, S, E;
  uint32_t cnt;
  __device__ void clear() { m = -INFINITY; mc = kFloor; S = E = 0.f; cnt = 0; }
  __device__ static float reference(float m, float cs) { return fmaxf(m * cs, kFloor); }
  template <bool ENT> __device__ void refer(float mcn) {
    const float d = mc - mcn, f = exp2_fast(d);
    if (ENT) E = __fmul_rn(fmaf(d, S, E), f);   // rounded alike wherever this is inlined: results do not depend on what else is asked for
    S = __fmul_rn(S, f);
    mc = mcn;
  }
  // before elements of which bm is the largest
  template <bool ENT> __device__ void reach(float bm, float cs) {
    m = fmaxf(m, bm);
    if (bm * cs > mc + kAhead) refer<ENT>(bm * cs);
  }
  template <bool ENT> __device__ void add(float x, float cs) {
    reach<ENT>(x, cs);
    const float u = ENT ? above_nothing(fmaf(x, cs, -mc)) : fmaf(x, cs, -mc), e = exp2_fast(u);
    S += e;
    if (ENT) E = fmaf(e, u, E);
  }
  // the sum over lanes that differ in the bits below N, the same in all of them
  template <bool ENT, int N> __device__ void join(float cs) {
    float M = m;
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    m = M;
    refer<ENT>(reference(M, cs));
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
      S += __shfl_xor_sync(0xffffffffu, S, o);
      if (ENT) E += __shfl_xor_sync(0xffffffffu, E, o);
      cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
    }
  }
  // not for the fast pass: beyond the range of its products, or not a number
  __device__ bool strange(float cs) const { return S != S || far(cs); }
  // beyond the range, and no NaN or +inf among the elements (their S is NaN): only the sums are to be done again
  __device__ bool far(float cs) const { return S == S && fabsf(m * cs) > kFar && m != -INFINITY; }
};

// The vectors w[0..U) of a thread, of which bm is the largest element, into its share.  ENT: `nothing`, a number whose product
// with cs is far below every reference and finite, stands for what is lower: 2^u u is then 0 and not 0 * inf.
__device__ __forceinline__ float as_nothing(float cs) { return fmaxf(-1e30f / cs, -3e38f); }
template <bool ENT, int U, typename T>
__device__ __forceinline__ void add_vectors(Part& a, const uint4 (&w)[U], int n, float bm, float cs, float nothing) {
  constexpr int V = Vec<T>::V;
  a.reach<ENT>(bm, cs);
  const F2 c = pair(cs, cs), m = pair(-a.mc, -a.mc);
  F2 S[2] = {0, 0}, E[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u >= n) break;
    float f[V];
    Vec<T>::unpack(ENT ? Vec<T>::above_or(w[u], nothing) : w[u], f);
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const F2 z = fma2(pair(f[i], f[i + 1]), c, m);
      const float2 q = halves(z);
      const F2 e = pair(exp2_fast(q.x), exp2_fast(q.y));
      S[i / 2 & 1] = add2(S[i / 2 & 1], e);
      if (ENT) E[i / 2 & 1] = fma2(e, z, E[i / 2 & 1]);
    }
  }
  const float2 s = halves(add2(S[0], S[1]));
  a.S += s.x + s.y;
  if (ENT) {
    const float2 e = halves(add2(E[0], E[1]));
    a.E += e.x + e.y;
  }
}
// The gradient of an element, e (c0 + c1 u) with e = 2^u: u meets the exponential first, which is 0 where u stands for something
// masked.  c1, the size of the caller's factors, would make it infinite, and 0 times that NaN.
__device__ __forceinline__ float entropy_grad(float e, float u, float c0, float c1) { return fmaf(__fmul_rn(e, u), c1, __fmul_rn(e, c0)); }
__device__ __forceinline__ F2 entropy_grad(F2 e, F2 u, F2 c0, F2 c1) { return fma2(mul2(e, u), c1, mul2(e, c0)); }
// ... of a vector's elements; without ENT c0 e
template <bool ENT, typename T>
__device__ __forceinline__ void grad_vector(uint4 w, float (&h)[Vec<T>::V], float cs, float mc, float c0, float c1, float nothing) {
  float f[Vec<T>::V];
  Vec<T>::unpack(ENT ? Vec<T>::above_or(w, nothing) : w, f);
#pragma unroll
  for (int i = 0; i < Vec<T>::V; i += 2) {
    const F2 z = fma2(pair(f[i], f[i + 1]), pair(cs, cs), pair(-mc, -mc));
    const float2 q = halves(z);
    const F2 e = pair(exp2_fast(q.x), exp2_fast(q.y));
    const float2 g = halves(ENT ? entropy_grad(e, z, pair(c0, c0), pair(c1, c1)) : mul2(e, pair(c0, c0)));
    h[i] = g.x;
    h[i + 1] = g.y;
  }
}
// ... and to where it goes: a vector, or single elements where the gradient's rows lie otherwise than the logits'
template <typename T>
__device__ __forceinline__ void put_vector(T* o, bool even, int accumulate, float (&h)[Vec<T>::V]) {
  if (even) {
    if (accumulate) {
      float d[Vec<T>::V];
      Vec<T>::unpack(*(const uint4*)o, d);
#pragma unroll
      for (int i = 0; i < Vec<T>::V; ++i) h[i] += d[i];
    }
    *(uint4*)o = Vec<T>::pack(h);
  } else {
#pragma unroll
    for (int i = 0; i < Vec<T>::V; ++i) st_f(o + i, accumulate ? h[i] + ld_f(o + i) : h[i]);
  }
}

// What the row's results are made of
struct RowSums {
  float m, mc, S, L, low;   // L = log2 S; low = L + (mc - m * cs)
  bool some;
  __device__ void set(float m_, float mc_, float S_, float cs) {
    m = m_; mc = mc_; S = S_;
    some = S != 0.f;
    L = some ? log2f(S) : 0.f;
    low = some ? L + fmaf(-m, cs, mc) : 0.f;
  }
  // The sum of a nearly certain row may be rounded to less than its largest term: no log probability is above 0 all the same
  __device__ float log_p(float x, float scale) const {
    return not_above(some ? fmaf(-kLn2, low, __fmul_rn(x - m, scale)) : -INFINITY, 0.f);
  }
  __device__ float entropy(float E) const { return some ? __fmul_rn(kLn2, L - __fdiv_rn(E, S)) : 0.f; }
  __device__ float lse(float scale) const { return some ? fmaf(kLn2, low, __fmul_rn(m, scale)) : -INFINITY; }
};

// A row's vectors [vb, ve), batch after batch: f(v0, w) gets the thread's vectors v0 + u * NT + tid, -inf behind the last.
// A block feeds them through shared memory, kAheadBatches copies (cp.async) in front of the one that is worked on; a thread
// reads what it has copied itself, so nothing is waited for together.  Where all of them fit (`slots` batches) they stay, and
// a second pass reads them there, else again from global memory.  A warp loads them into registers.
template <int NT>
struct Feed {
  static constexpr uint32_t U = NT == 32 ? 8 : 4, kBatch = U * NT;
  static constexpr int kAheadBatches = 3;
  const uint4* xv;
  uint32_t vb, ve, tid, slots;
  uint4* mem;
  uint32_t put, get;
  uint4 w[U];
  __device__ Feed(const uint4* xv_, uint32_t vb_, uint32_t ve_, uint32_t tid_, uint32_t slots_, uint4* mem_) : xv(xv_), vb(vb_), ve(ve_), tid(tid_), slots(slots_), mem(mem_) {}
  __device__ uint32_t batches() const { return (ve - vb + kBatch - 1) / kBatch; }
  __device__ __forceinline__ void copy(uint32_t i) {
    if (i < batches()) {
      const uint32_t v0 = vb + i * kBatch + tid;
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
        if (v0 + u * NT < ve) copy_async(shared_address(mem + put * kBatch + u * NT + tid), xv + v0 + u * NT);
      if (++put == slots) put = 0;
    }
    commit_copies();
  }
  template <typename T> __device__ __forceinline__ void load(uint32_t v0) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) {
      const uint32_t v = v0 + u * NT + tid;
      w[u] = v < ve ? xv[v] : Vec<T>::none();
    }
  }
  template <typename T> __device__ __forceinline__ void take(uint32_t v0, const uint4* slot) {
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) w[u] = v0 + u * NT + tid < ve ? load_shared(shared_address(slot + u * NT + tid)) : Vec<T>::none();
  }
  // the first loads of a pass
  template <typename T> __device__ __forceinline__ void start() {
    if constexpr (NT == 32) {
      load<T>(vb);
    } else {
      put = get = 0;
#pragma unroll
      for (int i = 0; i < kAheadBatches; ++i) copy(i);
    }
  }
  template <typename T, bool AGAIN, typename F>
  __device__ __forceinline__ void run(F&& f) {
    if constexpr (NT == 32) {
      if (AGAIN) load<T>(vb);
      for (uint32_t v0 = vb; v0 < ve; v0 += kBatch) {
        if (v0 != vb) load<T>(v0);
        f(v0, w);
      }
    } else {
      const uint32_t n = batches();
      if (AGAIN && n <= slots) {
        for (uint32_t i = 0; i < n; ++i) {
          take<T>(vb + i * kBatch, mem + i * kBatch);
          f(vb + i * kBatch, w);
        }
        return;
      }
      if (AGAIN) start<T>();
      for (uint32_t i = 0; i < n; ++i) {
        wait_copies<kAheadBatches - 1>();
        take<T>(vb + i * kBatch, mem + get * kBatch);
        if (++get == slots) get = 0;
        f(vb + i * kBatch, w);
        copy(i + kAheadBatches);   // into the slot that has just been read, where there are no more
      }
    }
  }
};
// Batches that a block's share of a row has room for: all of them where they fit into `most` bytes, else as many as are ahead
inline uint32_t feed_slots(size_t row_bytes, uint32_t parts, size_t most) {
  constexpr size_t batch = Feed<kRowThreads>::kBatch * 16, ahead = Feed<kRowThreads>::kAheadBatches;
  const size_t n = (row_bytes / 16 / parts + 1 + Feed<kRowThreads>::kBatch - 1) / Feed<kRowThreads>::kBatch;
  return (uint32_t)(n * batch <= most || n < ahead ? n : ahead);
}
constexpr size_t kMostFeed = 96 * 1024;

// ---- many rows: blocks that stay, W warps that stream and one that does what a row needs besides
// The streaming warps take one row's vectors after the other's: their copies (cp.async) go on into the next rows, so that
// loads are in flight while a row is finished.  The last warp prepares a row while the one in front of it is streamed (label,
// lists, masks), and finishes a row while the next one is.
// Three blocks of an SM with eight streaming warps each.  Backward every row is passed over twice: a row (or a block's part
// of it) that fits into the ring stays there for the second pass, each batch of which makes room for one of the next row;
// other rows are copied again, out of the L2.  One block of an SM with sixteen warps and 192 KB of ring was slower (4096 rows
// of 64 KB: 149 us for 122): nothing else fills the SM while a row's sums are joined.
enum { kBarReady = 1, kBarResult = 3, kBarSums = 5, kBarFree = 7 };   // and the row's slot (of four forward, of two backward); 9: Group<W * 32>
// The sums of the blocks of a cluster: whole[parity] is this block's, the one in the same place the others'.  All threads of
// all blocks meet in between, and the next row's meeting comes before whole[parity] is written again.
template <int W> struct Crew {
  static constexpr uint32_t kThreads = W * 32 + 32, kBlocks = 3;   // that meet at a barrier, blocks of an SM
  __device__ static void arrive(uint32_t id) {
    __syncwarp();
    __threadfence_block();
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
  }
  __device__ static void wait(uint32_t id) {
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
  }
};
template <int N> __device__ __forceinline__ void wait_for_copies(uint32_t n) {   // until at most n are on their way
  if constexpr (N == 0) wait_copies<0>();
  else if (n >= N) wait_copies<N>();
  else wait_for_copies<N - 1>(n);
}

template <typename T, int W, bool BWD>
struct Stream {
  static constexpr uint32_t U = 4, NS = W * 32, kBatch = U * NS, kBytes = kBatch * 16, kVec = NS * 16, kMostSlots = 6, kForward = 3;
  const T* x;
  const Rows& at;
  uint32_t r, stride, part, parts;   // the row that is copied; this block's part of it
  const uint4* from;       // this thread's vector to be copied next
  uint32_t left;           // vectors of the row that are left
  uint32_t ring, end, put, get; // this thread's places in shared memory
  uint32_t held;           // batches that are copied or on their way
  bool twice, second;      // rows are copied for each of two passes
  __device__ void row() {
    left = 0;
    if (r < at.rows) {
      const T* p = x + at.offset(r);
      const Strip<T> b(p, at.C, part, parts);
      from = (const uint4*)(p + b.head) + b.vb + threadIdx.x;
      left = b.ve - b.vb;
    }
  }
  __device__ __forceinline__ void copy() {
    if (left == 0) {
      if (!BWD) commit_copies();   // there are always as many groups behind a batch
      return;
    }
    if (left >= kBatch) {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u) copy_async(put + u * kVec, from + u * NS);
      left -= kBatch;
      from += kBatch;
    } else {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
        if (u * NS + threadIdx.x < left) copy_async(put + u * kVec, from + u * NS);
      left = 0;
    }
    commit_copies();
    ++held;
    put = put + kBytes == end ? ring : put + kBytes;
    if (left == 0) {
      if (twice && !second) {
        second = true;
      } else {
        second = false;
        r += stride;
      }
      row();
    }
  }
  __device__ Stream(const T* x_, const Rows& at_, void* mem, uint32_t slots, bool twice_, uint32_t first, uint32_t stride_, uint32_t part_, uint32_t parts_)
      : x(x_), at(at_), r(first), stride(stride_), part(part_), parts(parts_), from(nullptr), left(0), ring(shared_address(mem) + threadIdx.x * 16),
        end(ring + slots * kBytes), put(ring), get(ring), held(0), twice(twice_), second(false) {
    row();
    for (uint32_t i = 0; i < slots; ++i) copy();
  }
  template <typename F> __device__ __forceinline__ void take(uint32_t at, uint32_t v0, uint32_t n, F&& f) {
    uint4 w[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) w[u] = load_shared(at + u * kVec);
    if (v0 + kBatch <= n) {
      f(v0, w, true);
    } else {
#pragma unroll
      for (uint32_t u = 0; u < U; ++u)
        if (v0 + u * NS + threadIdx.x >= n) w[u] = Vec<T>::none();
      f(v0, w, false);
    }
  }
  // f(v0, w, full) for the batches of a row of n vectors; full: all threads have all of theirs.  f may change w.
  // The batches that have been there longest, and their room for further ones
  template <typename F> __device__ __forceinline__ void run(uint32_t n, F&& f) {
    for (uint32_t v0 = 0; v0 < n; v0 += kBatch) {
      if (BWD) wait_for_copies<kMostSlots - 1>(held - 1);
      else wait_copies<kForward - 1>();
      take(get, v0, n, f);
      get = get + kBytes == end ? ring : get + kBytes;
      --held;
      copy();   // into the slot that has just been read, where there are no more
    }
  }
  // ... which stay where they are, for run() to have them once more (all of a row: not where it is copied twice)
  template <typename F> __device__ __forceinline__ void look(uint32_t n, F&& f) {
    uint32_t there = get, newer = held;
    for (uint32_t v0 = 0; v0 < n; v0 += kBatch) {
      wait_for_copies<kMostSlots - 1>(--newer);
      take(there, v0, n, f);
      there = there + kBytes == end ? ring : there + kBytes;
    }
  }
};
// How the blocks of a call are laid out: blocks that share a row (a cluster), batches of a ring, whether rows are copied twice
struct RingPlan {
  uint32_t parts, slots, twice;
  size_t bytes;
};
// besides(parts): bytes of shared memory that a block needs for other things.  Backward: the rows that are in hand together
// have to stay in the L2 for the second pass, or in the ring where they fit.  444 rows of 200 KB did not (1001 of them read 1.7
// times, 107 us), 222 rows shared by two blocks each do (95); of 400 KB four blocks each (2000 rows: 401 -> 352 us).  Sharing costs
// a meeting per row: the log probabilities' gradient of 4096 rows of 131 KB takes 221 us unshared and took 232 by twos.
constexpr size_t kRowsInL2 = 60 << 20;
template <typename T, int W, bool BWD, typename F>
inline RingPlan ring_plan(uint32_t C, F&& besides) {
  typedef Stream<T, W, BWD> Str;
  RingPlan p = {1, Str::kForward, 0, 0};
  if (BWD) {
    constexpr size_t blocks = Crew<W>::kBlocks * kNumSMs;
    while (p.parts < 8 && blocks / p.parts * (size_t)C * sizeof(T) > kRowsInL2) p.parts *= 2;
    const long long room = (227 * 1024 / (long long)Crew<W>::kBlocks - 9 * 1024 - (long long)besides(p.parts)) / (long long)Str::kBytes;
    const size_t need = (C / Vec<T>::V / p.parts + 1 + Str::kBatch - 1) / Str::kBatch;
    p.slots = (uint32_t)(room < 3 ? 3 : room < (long long)Str::kMostSlots ? room : Str::kMostSlots);
    p.twice = need > p.slots;
  }
  p.bytes = (size_t)p.slots * Str::kBytes;
  return p;
}
// What the launches of one kernel share: on which devices (a bit each) its limit is raised, and how many clusters of each shape
// a device holds at a time
struct StreamLaunch {
  unsigned raised;
  ClusterCounts held;
};
constexpr size_t kMostRing = 218 * 1024;   // dynamic shared memory of the blocks that stay
template <typename... P, typename... A>
inline int launch_stream(void (*kernel)(P...), StreamLaunch& l, uint32_t threads, size_t rows, uint32_t parts, size_t smem, cudaStream_t s, A... args) {
  int dev = 0;
  cudaGetDevice(&dev);
  if (!(__atomic_load_n(&l.raised, __ATOMIC_RELAXED) & (1u << (dev & 31)))) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostRing) != cudaSuccess) {
      cudaGetLastError();
      return AD_ERR_CUDA;
    }
    __atomic_fetch_or(&l.raised, 1u << (dev & 31), __ATOMIC_RELAXED);
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  cfg.blockDim = threads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.gridDim = parts;
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  // as many clusters as are resident together, which is less than three blocks per SM: a cluster stays within one group of SMs
  const uint32_t shape = ClusterCounts::key(dev, parts, smem);
  size_t n = l.held.find(shape);
  if (n == 0) {
    int most = 0;
    if (cudaOccupancyMaxActiveClusters(&most, kernel, &cfg) != cudaSuccess || most < 1) {   // part of a GPU: the other kernels serve it
      cudaGetLastError();
      return AD_ERR_UNSUPPORTED;
    }
    n = (uint32_t)most;
    l.held.keep(shape, (uint32_t)most);
  }
  cfg.gridDim = (unsigned)((rows < n ? rows : n) * parts);
  launch_attr(cfg, at);
  cudaLaunchKernelEx(&cfg, kernel, P(args)...);   // an error is what launch_status() returns
  return AD_OK;
}

// Plain loops over a row in any layout: what the fast pass does not serve
template <int NT, typename T, bool ENT>
__device__ void plain_sums(Group<NT>& g, const T* x, int64_t st, uint32_t C, float cs, RowSums& s, float& E) {
  float m = -INFINITY, S = 0.f;
  for (uint32_t c = g.tid; c < C; c += NT) m = fmaxf(m, ld_f(x + c * st));
  m = g.max(m);
  if (m == -INFINITY) m = 0.f;
  E = 0.f;
  for (uint32_t c = g.tid; c < C; c += NT) {
    const float u = (ld_f(x + c * st) - m) * cs, e = exp2_fast(u);
    S += e;
    if (ENT && e > 0.f) E += e * u;
  }
  S = g.sum(S);
  if (ENT) E = g.sum(E);
  s.m = m; s.mc = 0.f; s.S = S;
  s.some = S != 0.f;
  s.low = s.L = s.some ? log2f(S) : 0.f;
}

// ---- a thread per position: few classes, or classes in planes
// MODE 0: from global memory, neighbouring threads on neighbouring positions of a plane.  1, 2: rows that a block has copied
// to shared memory, read by single elements (1: rows of any length, one behind the other) or by vectors (2: rows of whole
// vectors, an odd number of them apart, so that eight lanes' loads fall into different banks).
template <typename T, int MODE>
struct Position {
  const T* x;
  uint32_t step;   // MODE 0: bytes from one class to the next
  uint32_t C;
  __device__ const T* at(uint32_t c) const { return MODE == 0 ? (const T*)((const char*)x + (uint64_t)c * step) : x + c; }
  __device__ float get(uint32_t c) const { return ld_f(at(c)); }
  // classes [c, c + 8), -inf from `hi` on (MODE 2: hi is C, a multiple of the vector)
  __device__ void batch(uint32_t c, uint32_t hi, float (&f)[8]) const {
    constexpr uint32_t V = Vec<T>::V;
    if (MODE == 2) {
      Vec<T>::unpack(*(const uint4*)(x + c), f);
      if (V == 4) Vec<T>::unpack(c + 4 < hi ? *(const uint4*)(x + c + 4) : Vec<T>::none(), f + 8 - V);
    } else if (c + 8 <= hi) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) f[i] = get(c + i);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) f[i] = c + i < hi ? get(c + i) : -INFINITY;
    }
  }
  __device__ void set(uint32_t c, float v) const { st_f(const_cast<T*>(at(c)), v); }
};
constexpr uint32_t kPositions = 128;         // of a block
constexpr uint32_t kFewClasses = 64;         // of rows in shared memory
// MODE 1, 2: elements from one row to the next in shared memory
template <typename T, int MODE> __host__ __device__ inline uint32_t tile_pitch(uint32_t C) { return MODE == 2 ? (C / Vec<T>::V | 1u) * Vec<T>::V : C; }
template <typename T>
__device__ __forceinline__ void copy_tile(bool vec, const T* from, const Rows& g, size_t r0, uint32_t n, T* tile) {
  constexpr uint32_t V = Vec<T>::V;
  const T* src = from + r0 * (size_t)g.pitch;
  if (vec) {
    const uint32_t q = g.C / V, to = tile_pitch<T, 2>(g.C);
    for (uint32_t i = threadIdx.x; i < n * q; i += kPositions) {
      const uint32_t row = i / q, col = i - row * q;
      copy_async(shared_address(tile + row * to + col * V), src + row * (size_t)g.pitch + col * V);
    }
  } else if (g.pitch == (int64_t)g.C) {
    const uint32_t e = n * g.C, v = ((uintptr_t)src & 15u) == 0 ? e / V : 0;
    for (uint32_t i = threadIdx.x; i < v; i += kPositions) copy_async(shared_address(tile + i * V), src + i * V);
    for (uint32_t i = v * V + threadIdx.x; i < e; i += kPositions) tile[i] = src[i];
  } else {
    for (uint32_t i = threadIdx.x; i < n * g.C; i += kPositions) tile[i] = src[i / g.C * (size_t)g.pitch + i % g.C];
  }
  commit_copies();
  wait_copies<0>();
}
template <typename T>
__device__ __forceinline__ void write_tile(bool vec, T* to, const Rows& g, size_t r0, uint32_t n, const T* tile) {
  constexpr uint32_t V = Vec<T>::V;
  T* dst = to + r0 * (size_t)g.pitch;
  if (vec) {
    const uint32_t q = g.C / V, tp = tile_pitch<T, 2>(g.C);
    for (uint32_t i = threadIdx.x; i < n * q; i += kPositions) {
      const uint32_t row = i / q, col = i - row * q;
      *(uint4*)(dst + row * (size_t)g.pitch + col * V) = *(const uint4*)(tile + row * tp + col * V);
    }
  } else if (g.pitch == (int64_t)g.C) {
    const uint32_t e = n * g.C, v = ((uintptr_t)dst & 15u) == 0 ? e / V : 0;
    for (uint32_t i = threadIdx.x; i < v; i += kPositions) ((uint4*)dst)[i] = ((const uint4*)tile)[i];
    for (uint32_t i = v * V + threadIdx.x; i < e; i += kPositions) dst[i] = tile[i];
  } else {
    for (uint32_t i = threadIdx.x; i < n * g.C; i += kPositions) dst[i / g.C * (size_t)g.pitch + i % g.C] = tile[i];
  }
}
// A row of up to CM classes (C rounded up to a multiple of 4) in registers, -inf behind the last
template <typename T, int CM, int MODE>
__device__ __forceinline__ void load_few(const Position<T, MODE>& x, bool vec, float (&v)[CM]) {
  constexpr int V = Vec<T>::V;
  if constexpr (CM % V == 0 && MODE != 0) {
    if (vec) {
#pragma unroll
      for (int c = 0; c < CM; c += V) {
        float f[V];
        Vec<T>::unpack(*(const uint4*)(x.x + c), f);
#pragma unroll
        for (int i = 0; i < V; ++i) v[c + i] = f[i];
      }
      return;
    }
  }
#pragma unroll
  for (uint32_t c = 0; c < CM; ++c) v[c] = c + 4 < CM || c < x.C ? x.get(c) : -INFINITY;
}
template <typename T, int CM, int MODE>
__device__ __forceinline__ void store_few(const Position<T, MODE>& x, bool vec, const float (&v)[CM]) {
  constexpr int V = Vec<T>::V;
  if constexpr (CM % V == 0 && MODE != 0) {
    if (vec) {
#pragma unroll
      for (int c = 0; c < CM; c += V) {
        float f[V];
#pragma unroll
        for (int i = 0; i < V; ++i) f[i] = v[c + i];
        *(uint4*)const_cast<T*>(x.x + c) = Vec<T>::pack(f);
      }
      return;
    }
  }
#pragma unroll
  for (uint32_t c = 0; c < CM; ++c)
    if (c + 4 < CM || c < x.C) x.set(c, v[c]);
}
template <bool ENT, int CM>
__device__ __forceinline__ void sum_few(Part& a, const float (&v)[CM], float cs) {
  a.clear();
#pragma unroll
  for (int c = 0; c < CM; ++c) a.m = fmaxf(a.m, v[c]);
  a.mc = Part::reference(a.m, cs);
  const F2 cs2 = pair(cs, cs), mc2 = pair(-a.mc, -a.mc);
  F2 S[2] = {0, 0}, E[2] = {0, 0};
#pragma unroll
  for (int c = 0; c < CM; c += 2) {
    F2 z = fma2(pair(v[c], v[c + 1]), cs2, mc2);
    float2 q = halves(z);
    if (ENT) {
      q.x = above_nothing(q.x);
      q.y = above_nothing(q.y);
      z = pair(q.x, q.y);
    }
    const F2 e = pair(exp2_fast(q.x), exp2_fast(q.y));
    S[c / 2 & 1] = add2(S[c / 2 & 1], e);
    if (ENT) E[c / 2 & 1] = fma2(e, z, E[c / 2 & 1]);
  }
  const float2 s = halves(add2(S[0], S[1]));
  a.S = s.x + s.y;
  if (ENT) {
    const float2 e = halves(add2(E[0], E[1]));
    a.E = e.x + e.y;
  }
}
// Bytes of such a tile, a multiple of 16
template <typename T, int MODE> inline size_t tile_bytes(uint32_t C) {
  return MODE == 0 ? 0 : (kPositions * (size_t)tile_pitch<T, MODE>(C) * sizeof(T) + 15) / 16 * 16;
}
// The mode that a call's rows are for; -1: none of them
template <typename T>
inline int position_mode(const Rows& g, const void* x) {
  if (g.HW) return g.C <= 0xffffu && (uint64_t)g.step * sizeof(T) <= 0xffffffffu ? 0 : -1;
  if (g.step != 1 || g.C > kFewClasses) return -1;
  return g.C % Vec<T>::V == 0 && g.pitch % Vec<T>::V == 0 && aligned_to(x, 16) ? 2 : 1;
}
inline unsigned position_blocks(size_t rows, uint32_t places = kPositions) {
  const size_t n = (rows + places - 1) / places;
  return (unsigned)(n < (1u << 20) ? n : (1u << 20));
}
// One position by plain loops over x_c - m
template <bool ENT, typename P>
__device__ void plain_position_sums(const P& x, float cs, RowSums& s, float& E) {
  float m = -INFINITY, S = 0.f;
  for (uint32_t c = 0; c < x.C; ++c) m = fmaxf(m, x.get(c));
  if (m == -INFINITY) m = 0.f;
  E = 0.f;
  for (uint32_t c = 0; c < x.C; ++c) {
    const float u = (x.get(c) - m) * cs, e = exp2_fast(u);
    S += e;
    if (ENT && e > 0.f) E += e * u;
  }
  s.m = m; s.mc = 0.f; s.S = S;
  s.some = S != 0.f;
  s.low = s.L = s.some ? log2f(S) : 0.f;
}

// A warp per row: rows of up to 8 KB, and, where there are rows for eight warps of each SM, up to 44 KB forward and 26 KB
// backward.  8192 rows of 18 KB (bf16, all results with 8 alternatives / gradient): 64 / 74 us, by blocks that stay 112 / 101; 26 KB:
// 81 / 108, 120 / 118; 4096 of 40 KB: 65 / 89, 71 / 79; of 64 KB: 95 / 144, 83 / 108.  600 rows of 18 KB: 13.5 / 15.5, 14.4 / 12.5.
inline bool by_warp(size_t rows, size_t row_bytes, bool bwd) {
  return row_bytes <= 8192 || (rows >= 8 * kNumSMs && row_bytes <= (bwd ? 26u : 44u) * 1024);
}
// Rows enough for blocks that stay: at least one for each
template <int W> inline bool stream_worth(size_t rows, uint32_t parts) { return rows * parts >= Crew<W>::kBlocks * kNumSMs && rows < (1u << 31); }
// Blocks of a row: few rows share the machine, a part at least 8 KB
inline uint32_t row_parts(size_t rows, size_t row_bytes) {
  uint32_t n = 1;
  while (n < 8 && rows * n * 2 <= 3 * kNumSMs && row_bytes / (n * 2) >= 8192) n *= 2;
  return n;
}
// `units` blocks, or clusters of n blocks; a kernel's blocks go on to further rows where there are more
template <typename P>
void launch_row_kernel(void (*kernel)(P, uint32_t), const P& p, uint32_t slots, size_t units, uint32_t n, size_t smem, cudaStream_t s) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  cfg.gridDim = (unsigned)((units < (1u << 20) ? units : (1u << 20)) * n);
  cfg.blockDim = kRowThreads;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  if (n > 1) {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = n;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  launch_attr(cfg, at);
  cudaLaunchKernelEx(&cfg, kernel, p, slots);   // an error is what launch_status() returns
}

}  // namespace adk
