// Rows of logits: what the log-probability and the distillation kernels share.
//
// A row's numbers are worked out in units of log 2: with m the row's maximum, cs = scale * log2(e), mc = m * cs as rounded,
//   u_c = x_c * cs - mc (one FMA),   S = sum 2^u_c,   E = sum 2^u_c u_c,   p_c = 2^u_c / S,
//   entropy = ln2 (log2 S - E / S),   log p_c = scale (x_c - m) - ln2 (log2 S + (mc - m * cs)),
// where mc - m * cs, the rounding of mc, is what an FMA gives.  One pass over the row: a thread keeps its own maximum,
// and S and E against it, and rescales them when the maximum of a batch of loads is larger.
// mc is off by up to 2^-24 of itself, and the terms by 2 to that: a row whose maximum is beyond +-kFar in units of log 2, or
// that holds +inf or NaN, is done again by plain loops over x_c - m.  A share's reference is at least kFloor, so that
// what is masked (-inf, the type's lowest value, -1e9) adds 2^-4e6 = 0 to the row and never inf or inf - inf.
// A row of -inf has S = 0, which is how it is recognised.
#pragma once

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

__device__ __forceinline__ float exp2_fast(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));   // 2 ulp; -inf gives 0
  return r;
}
// v, not below -200 (2^-200 is 0 here), and NaN where v is: what may be multiplied by its exponential
__device__ __forceinline__ float above_nothing(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(-200.f));
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

// ---- threads that work on one row: a warp, or a block of 256 with `red` (10 words of shared memory)
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
template <> struct Group<kRowThreads> {
  uint32_t tid = threadIdx.x;
  Key* red;   // one per warp
  __device__ explicit Group(void* r) : red((Key*)r) {}
  __device__ void sync() { __syncthreads(); }
  template <typename V, typename F>
  __device__ V all(V w, F f) {   // of the warps' values, in order
    __syncthreads();
    if ((tid & 31) == 0) *(V*)&red[tid >> 5] = w;
    __syncthreads();
    V v = *(V*)&red[0];
#pragma unroll
    for (int i = 1; i < kRowWarps; ++i) v = f(v, *(V*)&red[i]);
    return v;
  }
  __device__ float max(float v) { return all(warp_max(v), [](float a, float b) { return fmaxf(a, b); }); }
  __device__ float sum(float v) { return all(warp_sum(v), [](float a, float b) { return a + b; }); }
  __device__ uint32_t sum(uint32_t v) { return all(__reduce_add_sync(0xffffffffu, v), [](uint32_t a, uint32_t b) { return a + b; }); }
  __device__ Key max(Key v) { return all(Group<32>(nullptr).max(v), [](Key a, Key b) { return a > b ? a : b; }); }
};

// ---- 16 bytes of a row
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int V = 4;
  typedef float Max;
  __device__ static uint4 none() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
  __device__ static void unpack(uint4 w, float* f) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
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

// What a thread, a group or a block of a cluster knows about its share of a row
struct Part {
  float m, mc, S, E;
  uint32_t cnt;
  __device__ void clear() { m = -INFINITY; mc = kFloor; S = E = 0.f; cnt = 0; }
  __device__ static float reference(float m, float cs) { return fmaxf(m * cs, kFloor); }
  template <bool ENT> __device__ void refer(float mcn) {   // S and E against a larger reference
    const float d = mc - mcn, f = exp2_fast(d);
    if (ENT) E = (E + d * S) * f;
    S *= f;
    mc = mcn;
  }
  template <bool ENT> __device__ void add(float x, float cs) {
    if (x > m) {
      m = x;
      refer<ENT>(reference(m, cs));
    }
    const float u = ENT ? above_nothing(fmaf(x, cs, -mc)) : fmaf(x, cs, -mc), e = exp2_fast(u);
    S += e;
    if (ENT) E = fmaf(e, u, E);
  }
  template <bool ENT> __device__ void join(const Part& o) {   // the same bits whichever of the two is asked
    m = fmaxf(m, o.m);
    cnt += o.cnt;
    const float mcn = fmaxf(mc, o.mc);
    Part q = o;
    refer<ENT>(mcn);
    q.refer<ENT>(mcn);
    S += q.S;
    if (ENT) E += q.E;
  }
  template <bool ENT> __device__ void join_lanes() {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Part q;
      q.m = __shfl_xor_sync(0xffffffffu, m, o);
      q.mc = __shfl_xor_sync(0xffffffffu, mc, o);
      q.S = __shfl_xor_sync(0xffffffffu, S, o);
      q.E = ENT ? __shfl_xor_sync(0xffffffffu, E, o) : 0.f;
      q.cnt = 0;
      join<ENT>(q);
    }
    cnt = __reduce_add_sync(0xffffffffu, cnt);
  }
  // not for the fast pass: beyond the range of its products, or not a number
  __device__ bool strange(float cs) const { return S != S || fabsf(m * cs) > kFar && m != -INFINITY; }
};

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
  __device__ float log_p(float x, float scale) const { return some ? (x - m) * scale - kLn2 * low : -INFINITY; }
  __device__ float lse(float scale) const { return some ? m * scale + kLn2 * low : -INFINITY; }
};

// Plain loops over a row in any layout: what the fast pass does not serve
template <typename G, typename T, bool ENT>
__device__ void plain_sums(G& g, const T* x, int64_t st, uint32_t C, float cs, RowSums& s, float& E) {
  const uint32_t NT = sizeof(G) == sizeof(Group<32>) ? 32 : kRowThreads;
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
  int64_t step;   // MODE 0
  uint32_t C;
  __device__ float get(uint32_t c) const { return ld_f(MODE == 0 ? x + c * step : x + c); }
  // classes [c, c + 8), -inf behind the last one
  __device__ void batch(uint32_t c, float (&f)[8]) const {
    constexpr uint32_t V = Vec<T>::V;
    if (MODE == 2) {
      Vec<T>::unpack(*(const uint4*)(x + c), f);
      if (V == 4) Vec<T>::unpack(c + 4 < C ? *(const uint4*)(x + c + 4) : Vec<T>::none(), f + 8 - V);
    } else if (c + 8 <= C) {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) f[i] = get(c + i);
    } else {
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) f[i] = c + i < C ? get(c + i) : -INFINITY;
    }
  }
  __device__ void set(uint32_t c, float v) const { st_f(const_cast<T*>(MODE == 0 ? x + c * step : x + c), v); }
};
constexpr uint32_t kPositions = 128;         // of a block
constexpr uint32_t kFewClasses = 64;         // of rows in shared memory
// MODE 1, 2: elements from one row to the next in shared memory
template <typename T, int MODE> __host__ __device__ inline uint32_t tile_pitch(uint32_t C) { return MODE == 2 ? (C / Vec<T>::V | 1u) * Vec<T>::V : C; }
template <typename T, int MODE>
__device__ __forceinline__ void copy_tile(const T* from, const Rows& g, size_t r0, uint32_t n, T* tile) {
  constexpr uint32_t V = Vec<T>::V;
  const T* src = from + r0 * (size_t)g.pitch;
  auto async = [](void* d, const void* s) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(d)), "l"(s) : "memory");
  };
  if (MODE == 2) {
    const uint32_t q = g.C / V, to = tile_pitch<T, 2>(g.C);
    for (uint32_t i = threadIdx.x; i < n * q; i += kPositions) {
      const uint32_t row = i / q, col = i - row * q;
      async(tile + row * to + col * V, src + row * (size_t)g.pitch + col * V);
    }
  } else if (g.pitch == (int64_t)g.C) {
    const uint32_t e = n * g.C, v = ((uintptr_t)src & 15u) == 0 ? e / V : 0;
    for (uint32_t i = threadIdx.x; i < v; i += kPositions) async(tile + i * V, src + i * V);
    for (uint32_t i = v * V + threadIdx.x; i < e; i += kPositions) tile[i] = src[i];
  } else {
    for (uint32_t i = threadIdx.x; i < n * g.C; i += kPositions) tile[i] = src[i / g.C * (size_t)g.pitch + i % g.C];
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}
template <typename T, int MODE>
__device__ __forceinline__ void write_tile(T* to, const Rows& g, size_t r0, uint32_t n, const T* tile) {
  constexpr uint32_t V = Vec<T>::V;
  T* dst = to + r0 * (size_t)g.pitch;
  const uint32_t tp = tile_pitch<T, MODE>(g.C);
  if (MODE == 2 && ((uintptr_t)dst & 15u) == 0 && g.pitch % V == 0) {
    const uint32_t q = g.C / V;
    for (uint32_t i = threadIdx.x; i < n * q; i += kPositions) {
      const uint32_t row = i / q, col = i - row * q;
      *(uint4*)(dst + row * (size_t)g.pitch + col * V) = *(const uint4*)(tile + row * tp + col * V);
    }
  } else if (MODE == 1 && g.pitch == (int64_t)g.C) {
    const uint32_t e = n * g.C, v = ((uintptr_t)dst & 15u) == 0 ? e / V : 0;
    for (uint32_t i = threadIdx.x; i < v; i += kPositions) ((uint4*)dst)[i] = ((const uint4*)tile)[i];
    for (uint32_t i = v * V + threadIdx.x; i < e; i += kPositions) dst[i] = tile[i];
  } else {
    for (uint32_t i = threadIdx.x; i < n * g.C; i += kPositions) dst[i / g.C * (size_t)g.pitch + i % g.C] = tile[i / g.C * tp + i % g.C];
  }
}
// Bytes of such a tile, a multiple of 16
template <typename T, int MODE> inline size_t tile_bytes(uint32_t C) {
  return MODE == 0 ? 0 : (kPositions * (size_t)tile_pitch<T, MODE>(C) * sizeof(T) + 15) / 16 * 16;
}
// The mode that a call's rows are for; -1: none of them
template <typename T>
inline int position_mode(const Rows& g, const void* x) {
  if (g.HW) return g.C <= 0xffffu ? 0 : -1;
  if (g.step != 1 || g.C > kFewClasses) return -1;
  return g.C % Vec<T>::V == 0 && g.pitch % Vec<T>::V == 0 && aligned_to(x, 16) ? 2 : 1;
}
inline unsigned position_blocks(size_t rows) {
  const size_t n = (rows + kPositions - 1) / kPositions;
  return (unsigned)(n < (1u << 20) ? n : (1u << 20));
}
// One position by plain loops over x_c - m
template <bool ENT, typename P>
__device__ void plain_position(const P& x, float cs, RowSums& s, float& E) {
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

// Blocks of a row: few rows share the machine, a part at least 8 KB
inline uint32_t row_parts(size_t rows, size_t row_bytes) {
  uint32_t n = 1;
  while (n < 8 && rows * n * 2 <= 4 * kNumSMs && row_bytes / (n * 2) >= 8192) n *= 2;
  return n;
}
// `units` blocks, or clusters of n blocks; a kernel's blocks go on to further rows where there are more
template <typename P>
void launch_row_kernel(void (*kernel)(P), const P& p, size_t units, uint32_t n, size_t smem, cudaStream_t s) {
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
  cudaLaunchKernelEx(&cfg, kernel, p);   // an error is what launch_status() returns
}

}  // namespace adk
