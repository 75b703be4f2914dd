// Log probabilities with a thread per position: few classes in neighbouring elements, or classes in planes.
//
// Few classes: a block copies the rows of 128 positions to shared memory (contiguous bytes, whatever the row length) and a
// thread takes its own row into registers; gradients go back into the tile and out by vectors.  Planes are read as they lie,
// neighbouring threads at neighbouring positions: up to 32 classes into registers, too (1,048,576 positions of 19 fp32 classes, 80
// MB: log-sum-exp 18 us, by four warps as below 66; gradient 32, 100), of more each of four warps takes a quarter.
// 4,194,304 pixels of 19 bf16 classes with three alternatives (344 MB, 53 us at the copy rate): 118 us, by instructions (865
// per 32 pixels: about 20 per class, and as many again for labels, logarithms, lists and stores).  Gradient of 2 x 150 x 256 x 255
// fp32 planes (157 MB, 24): 41, by the latency of eight loads in flight per thread, ten blocks of an SM.
#include "logprob.cuh"

namespace adk {

// The first KT classes of those seen so far (NaN apart: such a row is done again).  16-bit values: value and class in one word, the list sorted by exchanges.
template <typename T, int KT> struct Firsts;
// The word orders values and, among equal ones, classes: of two the larger is in front.
__device__ __forceinline__ uint32_t word_of(float v, uint32_t c) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return b ^ ((uint32_t)((int)b >> 31) & 0x7fff0000u) ^ (0x8000ffffu - c);
}
template <int KT> struct Firsts<__nv_bfloat16, KT> {
  uint32_t k[KT] = {};
  __device__ void add(float v, uint32_t c) { add(word_of(v, c)); }
  __device__ void add(uint32_t t) {
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      const uint32_t hi = max(k[i], t);
      t = min(k[i], t);
      k[i] = hi;
    }
  }
  __device__ Key key(int i) const {
    if (!k[i]) return 0;
    const uint32_t v = k[i] & 0xffff0000u;
    return (Key)(v >> 31 ? v : v | 0xffffu) << 32 | (uint32_t)~(0xffffu - (k[i] & 0xffffu));
  }
};
template <int KT> struct Firsts<float, KT> {   // classes come in ascending order
  uint32_t k[KT] = {}, c[KT] = {};
  __device__ void add(float v, uint32_t cls) {
    uint32_t t = value_key(v);
    bool g = false;   // from the place that it takes on, everything moves by one
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      g |= t > k[i];
      const uint32_t tk = g ? k[i] : t, tc = g ? c[i] : cls;
      k[i] = g ? t : k[i];
      c[i] = g ? cls : c[i];
      t = tk;
      cls = tc;
    }
  }
  __device__ Key key(int i) const { return k[i] ? (Key)k[i] << 32 | (uint32_t)~c[i] : 0; }
};


// Where a block's lists go: to shared memory, from where they leave in one piece (a position's own entries are parts of sectors:
// 4,194,304 positions with three entries each wrote 2.4 times their bytes), or directly where they are too long for that
struct ListOut {
  uint32_t* cls;   // [positions][top], then as many log probabilities; NULL: directly
  float* logp;
  __device__ void put(const LogprobP& p, const RowSums& s, size_t r, uint32_t place, uint32_t at, Key key) const {
    if (!cls) return put_top(p, s, r, at, key);
    cls[place * p.top + at] = key ? key_class(key) : kNoClass;
    logp[place * p.top + at] = key ? s.log_p(key_value((uint32_t)(key >> 32)), p.scale) : -INFINITY;
  }
  __device__ void flush(const LogprobP& p, size_t r0, uint32_t n) const {   // behind a barrier
    if (!cls) return;
    for (uint32_t i = threadIdx.x; i < n * p.top; i += kPositions) {
      if (p.top_class) p.top_class[r0 * p.top + i] = cls[i];
      if (p.top_logp) p.top_logp[r0 * p.top + i] = logp[i];
    }
  }
};

// One position by plain loops: any numbers, any length of list
template <typename P>
__device__ __noinline__ void plain_position(const LogprobP& p, P x, size_t r, uint32_t l, float xl) {
  RowSums s;
  float E;
  plain_position_sums<true>(x, p.cs, s, E);
  put_row(p, s, r, s.entropy(E), l, xl);
  if (p.rank) {
    uint32_t n = 0;
    for (uint32_t c = 0; c < x.C; ++c) n += in_front(x.get(c), c, xl, l);
    p.rank[r] = l < x.C ? n : kNoClass;
  }
}
template <typename P>
__device__ __noinline__ void plain_list(const LogprobP& p, P x, RowSums s, size_t r, ListOut out, uint32_t place) {
  Key last = ~0ull;
  for (uint32_t i = 0; i < p.top; ++i) {
    Key best = 0;
    if (last)
      for (uint32_t c = 0; c < x.C; ++c) {
        const float v = x.get(c);
        const Key key = v == v ? key_of(v, c) : 0;
        if (key < last && key > best) best = key;
      }
    out.put(p, s, r, place, i, best);
    last = best;
  }
}
// Both, as far as they are asked for
template <typename P>
__device__ __noinline__ void plain_all(const LogprobP& p, P x, size_t r, uint32_t l, float xl, ListOut out, uint32_t place) {
  plain_position(p, x, r, l, xl);
  if (p.top) {
    RowSums s;
    float E;
    plain_position_sums<false>(x, p.cs, s, E);
    plain_list(p, x, s, r, out, place);
  }
}
template <bool ENT, typename P>
__device__ __noinline__ void plain_gradient(const LogprobP& p, P x, P o, P old, size_t r, uint32_t l, float xl) {
  RowSums s;
  float E;
  plain_position_sums<ENT>(x, p.cs, s, E);
  const float H = s.entropy(E);
  put_row(p, s, r, H, l, xl);
  Factors f;
  f.fetch(p, r, l);
  f.set<ENT>(p, s, H);
  for (uint32_t c = 0; c < x.C; ++c) {
    float u = (x.get(c) - s.m) * p.cs;
    if (ENT) u = above_nothing(u);
    const float e = exp2_fast(u);
    float g = ENT ? entropy_grad(e, u, f.c0, f.c1) : e * f.c0;
    if (c == l) g += f.dl;
    o.set(c, p.accumulate ? g + old.get(c) : g);
  }
}

// ---------------------------------------------------------------- up to 32 classes: a row in registers
// CM: C rounded up to a multiple of 4.  PLANES: the classes come from planes as they lie; else from rows in shared memory,
// vec: of whole vectors, an odd number of them apart.
template <typename T, int CM, int KT, bool PLANES>
__global__ void __launch_bounds__(kPositions) logprob_few(const __grid_constant__ LogprobP p, int vec) {
  typedef Position<T, PLANES ? 0 : 1> X;
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  __shared__ uint32_t cls[kPositions * KT];
  __shared__ float logps[kPositions * KT];
  T* tile = (T*)tiles;
  const uint32_t C = p.x.C;
  const ListOut out = {p.top <= KT ? cls : nullptr, logps};
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions);
    const uint32_t l = p.label && threadIdx.x < n ? p.label[r] : kNoClass;
    if (!PLANES) copy_tile<T>(vec != 0, (const T*)p.logits, p.x, r0, n, tile);
    __syncthreads();
    if (threadIdx.x < n) {
      const X x = {PLANES ? (const T*)p.logits + p.x.offset(r) : tile + threadIdx.x * (vec ? tile_pitch<T, 2>(C) : C), (uint32_t)(p.x.step * sizeof(T)), C};
      float v[CM];
      load_few<T, CM>(x, vec != 0, v);
      const float xl = l < C ? x.get(l) : 0.f;
      Part a;
      sum_few<true, CM>(a, v, p.cs);
      if (a.strange(p.cs)) {
        plain_all(p, x, r, l, xl, out, threadIdx.x);
      } else {
        RowSums s;
        s.set(a.m, a.mc, a.S, p.cs);
        put_row(p, s, r, s.entropy(a.E), l, xl);
        Firsts<T, KT> top;
        uint32_t k = 0;
        if constexpr (sizeof(T) == 2) {
          if (p.rank || p.top) {
            const uint32_t wl = word_of(xl, l < C ? l : 0xffffu);
#pragma unroll
            for (uint32_t c = 0; c < CM; ++c)
              if (c + 4 < CM || c < C) {
                const uint32_t w = word_of(v[c], c);
                k += w > wl;
                top.add(w);
              }
          }
        } else {
          if (p.rank) {
#pragma unroll
            for (uint32_t c = 0; c < CM; ++c)
              if (c + 4 < CM || c < C) k += in_front(v[c], c, xl, l);
          }
          if (p.top && p.top <= KT) {
#pragma unroll
            for (uint32_t c = 0; c < CM; ++c)
              if (c + 4 < CM || c < C) top.add(v[c], c);
          }
        }
        if (p.rank) p.rank[r] = l < C ? k : kNoClass;
        if (p.top > KT) {
          plain_list(p, x, s, r, out, threadIdx.x);
        } else if (p.top) {
#pragma unroll
          for (int i = 0; i < KT; ++i)
            if ((uint32_t)i < p.top) out.put(p, s, r, threadIdx.x, i, top.key(i));
        }
      }
    }
    __syncthreads();
    out.flush(p, r0, n);
  }
}

template <typename T, int CM, bool ENT, bool PLANES>
__global__ void __launch_bounds__(kPositions) logprob_few_bwd(const __grid_constant__ LogprobP p, int vec) {
  typedef Position<T, PLANES ? 0 : 1> X;
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  const uint32_t C = p.x.C, tp = vec ? tile_pitch<T, 2>(C) : C;
  T *tile = (T*)tiles, *olds = tile + kPositions * tp;   // what the gradient is added to
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions);
    const uint32_t l = p.label && threadIdx.x < n ? p.label[r] : kNoClass;
    Factors f;
    if (threadIdx.x < n) f.fetch(p, r, l);
    if (!PLANES) {
      copy_tile<T>(vec != 0, (const T*)p.logits, p.x, r0, n, tile);
      if (p.accumulate) copy_tile<T>(vec != 0, (const T*)p.dlogits, p.g, r0, n, olds);
      __syncthreads();
    }
    if (threadIdx.x < n) {
      const X x = {PLANES ? (const T*)p.logits + p.x.offset(r) : tile + threadIdx.x * tp, (uint32_t)(p.x.step * sizeof(T)), C};
      const X o = {PLANES ? (T*)p.dlogits + p.g.offset(r) : tile + threadIdx.x * tp, (uint32_t)(p.g.step * sizeof(T)), C};
      const X old = {PLANES ? o.x : olds + threadIdx.x * tp, o.step, C};
      float v[CM];
      load_few<T, CM>(x, vec != 0, v);
      const float xl = l < C ? x.get(l) : 0.f;
      Part a;
      sum_few<ENT, CM>(a, v, p.cs);
      if (a.strange(p.cs)) {
        plain_gradient<ENT>(p, x, o, old, r, l, xl);
      } else {
        RowSums s;
        s.set(a.m, a.mc, a.S, p.cs);
        const float H = s.entropy(a.E);
        put_row(p, s, r, H, l, xl);
        f.set<ENT>(p, s, H);
        float gl = f.grad<ENT>(xl, p.cs, s.mc) + f.dl;   // the label's class, whose value replaces the one that the loop writes
        const F2 cs2 = pair(p.cs, p.cs), mc2 = pair(-s.mc, -s.mc), c0 = pair(f.c0, f.c0), c1 = pair(f.c1, f.c1);
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
          const float2 g = halves(ENT ? entropy_grad(e, z, c0, c1) : mul2(e, c0));
          v[c] = g.x;
          v[c + 1] = g.y;
        }
        if (p.accumulate) {
          if (l < C) gl += old.get(l);
#pragma unroll
          for (uint32_t c = 0; c < CM; ++c)
            if (c + 4 < CM || c < C) v[c] += old.get(c);
        }
        store_few<T, CM>(o, vec != 0, v);
        if (l < C) o.set(l, gl);
      }
    }
    if (!PLANES) {
      __syncthreads();
      write_tile<T>(vec != 0, (T*)p.dlogits, p.g, r0, n, tile);
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- up to 64 classes, and planes: batches of eight classes
// MODE 0: planes, a position per lane, and the classes dealt out to G warps.  1, 2: rows in shared memory (G = 1).
template <int MODE, int G> constexpr uint32_t kPlaces = MODE == 0 && G > 1 ? 32 : kPositions;   // positions of a block
template <bool ENT, typename P, typename F>
__device__ __forceinline__ void sum_classes(const P& x, Part& a, uint32_t lo, uint32_t hi, float cs, F&& also) {
  float next[8];
  x.batch(lo, hi, next);
  for (uint32_t c = lo; c < hi; c += 8) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = next[i];
    if (c + 8 < hi) x.batch(c + 8, hi, next);   // on its way while this one is worked on
    a.reach<ENT>(fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7]))), cs);
    const F2 cs2 = pair(cs, cs), mc2 = pair(-a.mc, -a.mc);
    F2 S[2] = {0, 0}, E[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      F2 z = fma2(pair(f[i], f[i + 1]), cs2, mc2);
      float2 q = halves(z);
      if (ENT) {
        q.x = above_nothing(q.x);
        q.y = above_nothing(q.y);
        z = pair(q.x, q.y);
      }
      const F2 e = pair(exp2_fast(q.x), exp2_fast(q.y));
      S[i / 2 & 1] = add2(S[i / 2 & 1], e);
      if (ENT) E[i / 2 & 1] = fma2(e, z, E[i / 2 & 1]);
    }
    const float2 s = halves(add2(S[0], S[1]));
    a.S += s.x + s.y;
    if (ENT) {
      const float2 e = halves(add2(E[0], E[1]));
      a.E += e.x + e.y;
    }
    also(c, f);
  }
}
// The sum over the warps of a block, lane by lane, in order
template <bool ENT, int G>
__device__ __forceinline__ void join_warps(Part& a, Part (&all)[G][32], float cs) {
  const uint32_t lane = threadIdx.x & 31;
  a.refer<ENT>(Part::reference(a.m, cs));
  all[threadIdx.x >> 5][lane] = a;
  __syncthreads();
  a = all[0][lane];
#pragma unroll
  for (int g = 1; g < G; ++g) {
    Part b = all[g][lane];
    a.m = fmaxf(a.m, b.m);
    const float mc = fmaxf(a.mc, b.mc);
    a.refer<ENT>(mc);
    b.refer<ENT>(mc);
    a.S += b.S;
    if (ENT) a.E += b.E;
    a.cnt += b.cnt;
  }
}

template <typename T, int MODE, int KT, int G>
__global__ void __launch_bounds__(kPositions, 8) logprob_positions_fwd(const __grid_constant__ LogprobP p) {
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  __shared__ Part sums[G][32];
  __shared__ Key lists[G][KT ? KT : 1][32];
  __shared__ uint32_t cls[KT ? kPlaces<MODE, G> * KT : 1];
  __shared__ float logps[KT ? kPlaces<MODE, G> * KT : 1];
  const ListOut out = {KT ? cls : nullptr, logps};
  T* tile = (T*)tiles;
  constexpr uint32_t N = kPlaces<MODE, G>;
  const uint32_t C = p.x.C, at = threadIdx.x % N, part = G > 1 ? threadIdx.x / N : 0;
  const uint32_t lo = (uint32_t)((uint64_t)C * part / G), hi = (uint32_t)((uint64_t)C * (part + 1) / G);
  const size_t blocks = (p.x.rows + N - 1) / N;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * N, r = r0 + at;
    const bool mine = r < p.x.rows;
    if (MODE) {
      copy_tile<T>(MODE == 2, (const T*)p.logits, p.x, r0, (uint32_t)(p.x.rows - r0 < N ? p.x.rows - r0 : N), tile);
      __syncthreads();
    }
    const Position<T, MODE> x = {MODE ? tile + at * tile_pitch<T, MODE ? MODE : 1>(C) : (const T*)p.logits + (mine ? p.x.offset(r) : 0), (uint32_t)(p.x.step * sizeof(T)), C};
    const uint32_t l = p.label && mine ? p.label[r] : kNoClass;
    const float xl = mine && l < C ? x.get(l) : 0.f;
    Part a;
    a.clear();
    Firsts<T, KT ? KT : 1> top;
    if (mine)
      sum_classes<true>(x, a, lo, hi, p.cs, [&](uint32_t c, const float (&f)[8]) {
        if (p.rank) {
#pragma unroll
          for (int i = 0; i < 8; ++i) a.cnt += c + i < hi && in_front(f[i], c + i, xl, l);
        }
        if (KT) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < hi) top.add(f[i], c + i);
        }
      });
    if (G > 1) {
      if (KT)
#pragma unroll
        for (int i = 0; i < KT; ++i) lists[part][i][threadIdx.x & 31] = top.key(i);
      join_warps<true, G>(a, sums, p.cs);
    }
    if (mine && part == 0) {
      if (a.strange(p.cs)) {
        plain_all(p, x, r, l, xl, out, at);
      } else {
        a.refer<true>(Part::reference(a.m, p.cs));
        RowSums s;
        s.set(a.m, a.mc, a.S, p.cs);
        put_row(p, s, r, s.entropy(a.E), l, xl);
        if (p.rank) p.rank[r] = l < C ? a.cnt : kNoClass;
        if constexpr (KT == 0) {
          if (p.top) plain_list(p, x, s, r, out, at);
        } else if constexpr (G == 1) {
#pragma unroll
          for (int i = 0; i < KT; ++i)
            if ((uint32_t)i < p.top) out.put(p, s, r, at, i, top.key(i));
        } else {   // the warps' lists are in order
          uint32_t next[G] = {};
          for (uint32_t i = 0; i < p.top; ++i) {
            Key best = 0;
            uint32_t from = 0;
#pragma unroll
            for (int g = 0; g < G; ++g) {
              const Key key = next[g] < KT ? lists[g][next[g]][at] : 0;
              if (key > best) { best = key; from = g; }
            }
#pragma unroll
            for (int g = 0; g < G; ++g) next[g] += best && from == (uint32_t)g;
            out.put(p, s, r, at, i, best);
          }
        }
      }
    }
    __syncthreads();
    out.flush(p, r0, (uint32_t)(p.x.rows - r0 < N ? p.x.rows - r0 : N));
    if (KT) __syncthreads();
  }
}

template <typename T, int MODE, bool ENT, int G>
__global__ void __launch_bounds__(kPositions, 10) logprob_positions_grad(const __grid_constant__ LogprobP p) {
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  __shared__ Part sums[G][32];
  constexpr uint32_t N = kPlaces<MODE, G>;
  constexpr int TM = MODE ? MODE : 1;
  const uint32_t C = p.x.C, at = threadIdx.x % N, part = G > 1 ? threadIdx.x / N : 0;
  const uint32_t lo = (uint32_t)((uint64_t)C * part / G), hi = (uint32_t)((uint64_t)C * (part + 1) / G);
  T *tile = (T*)tiles, *olds = tile + kPositions * tile_pitch<T, TM>(C);   // what the gradient is added to
  const size_t blocks = (p.x.rows + N - 1) / N;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * N, r = r0 + at;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < N ? p.x.rows - r0 : N);
    const bool mine = at < n;
    if (MODE) {
      copy_tile<T>(MODE == 2, (const T*)p.logits, p.x, r0, n, tile);
      if (p.accumulate) copy_tile<T>(MODE == 2, (const T*)p.dlogits, p.g, r0, n, olds);
      __syncthreads();
    }
    const uint32_t place = at * tile_pitch<T, TM>(C);
    T* out = (T*)p.dlogits + (MODE == 0 && mine ? p.g.offset(r) : 0);
    const Position<T, MODE> x = {MODE ? tile + place : (const T*)p.logits + (mine ? p.x.offset(r) : 0), (uint32_t)(p.x.step * sizeof(T)), C};
    const Position<T, MODE> o = {MODE ? tile + place : out, (uint32_t)(p.g.step * sizeof(T)), C}, old = {MODE ? olds + place : out, (uint32_t)(p.g.step * sizeof(T)), C};
    const uint32_t l = p.label && mine ? p.label[r] : kNoClass;
    const float xl = mine && l < C ? x.get(l) : 0.f;
    Factors f;
    if (mine) f.fetch(p, r, l);
    Part a;
    a.clear();
    if (mine) sum_classes<ENT>(x, a, lo, hi, p.cs, [](uint32_t, const float (&)[8]) {});
    if (G > 1) join_warps<ENT, G>(a, sums, p.cs);
    if (mine) {
      if (a.strange(p.cs)) {
        if (part == 0) plain_gradient<ENT>(p, x, o, old, r, l, xl);
      } else {
        a.refer<ENT>(Part::reference(a.m, p.cs));
        RowSums s;
        s.set(a.m, a.mc, a.S, p.cs);
        const float H = s.entropy(a.E), mc = s.mc;
        if (part == 0) put_row(p, s, r, H, l, xl);
        f.set<ENT>(p, s, H);
        float gl = 0.f;
        if (l >= lo && l < hi) gl = f.grad<ENT>(xl, p.cs, mc) + f.dl + (p.accumulate ? old.get(l) : 0.f);
        float next[8];
        x.batch(lo, hi, next);
        for (uint32_t c = lo; c < hi; c += 8) {
          float h[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) h[i] = next[i];
          if (c + 8 < hi) x.batch(c + 8, hi, next);
          const F2 cs2 = pair(p.cs, p.cs), mc2 = pair(-mc, -mc), c0 = pair(f.c0, f.c0), c1 = pair(f.c1, f.c1);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            F2 z = fma2(pair(h[i], h[i + 1]), cs2, mc2);
            float2 q = halves(z);
            if (ENT) {
              q.x = above_nothing(q.x);
              q.y = above_nothing(q.y);
              z = pair(q.x, q.y);
            }
            const F2 e = pair(exp2_fast(q.x), exp2_fast(q.y));
            const float2 g = halves(ENT ? entropy_grad(e, z, c0, c1) : mul2(e, c0));
            h[i] = g.x;
            h[i + 1] = g.y;
          }
          if (c + 8 <= hi && !p.accumulate) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o.set(c + i, h[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (c + i < hi) o.set(c + i, p.accumulate ? h[i] + old.get(c + i) : h[i]);
          }
        }
        if (l >= lo && l < hi) o.set(l, gl);   // over what the loop wrote
      }
    }
    __syncthreads();
    if (MODE) {
      write_tile<T>(MODE == 2, (T*)p.dlogits, p.g, r0, n, tile);
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- launches
template <typename... K, typename... A>
static int go(void (*kernel)(K...), const LogprobP& p, uint32_t places, size_t smem, cudaStream_t s, A... args) {
  // the limit belongs to the function: the most that it takes
  if (smem > 32 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (kFewClasses * 4 + 16) * kPositions) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch(kernel, position_blocks(p.x.rows, places), kPositions, smem, s, p, args...);
  return AD_OK;
}
// mode: as position_mode() has it
template <typename T, int CM, int KT>
static int go_few(const LogprobP& p, int mode, cudaStream_t s) {
  if constexpr (CM <= 32) {
    if (p.x.C > CM) return go_few<T, CM + 4, KT>(p, mode, s);
    if (mode == 0) return go(logprob_few<T, CM, KT, true>, p, kPositions, 0, s, 0);
    return go(logprob_few<T, CM, KT, false>, p, kPositions, mode == 2 ? tile_bytes<T, 2>(p.x.C) : tile_bytes<T, 1>(p.x.C), s, mode == 2);
  } else return AD_ERR_UNSUPPORTED;
}
template <typename T, int CM, bool ENT>
static int go_few_bwd(const LogprobP& p, int mode, cudaStream_t s) {
  if constexpr (CM <= 32) {
    if (p.x.C > CM) return go_few_bwd<T, CM + 4, ENT>(p, mode, s);
    if (mode == 0) return go(logprob_few_bwd<T, CM, ENT, true>, p, kPositions, 0, s, 0);
    return go(logprob_few_bwd<T, CM, ENT, false>, p, kPositions, (mode == 2 ? tile_bytes<T, 2>(p.x.C) : tile_bytes<T, 1>(p.x.C)) * (p.accumulate ? 2 : 1), s, mode == 2);
  } else return AD_ERR_UNSUPPORTED;
}
template <typename T, int MODE, int G>
static int go_fwd(const LogprobP& p, cudaStream_t s) {
  const size_t smem = tile_bytes<T, MODE>(p.x.C);
  constexpr uint32_t N = kPlaces<MODE, G>;
  if (p.top == 0 || p.top > 8) return go(logprob_positions_fwd<T, MODE, 0, G>, p, N, smem, s);
  if (p.top <= 3) return go(logprob_positions_fwd<T, MODE, 3, G>, p, N, smem, s);
  return go(logprob_positions_fwd<T, MODE, 8, G>, p, N, smem, s);
}
template <typename T, int MODE, int G>
static int go_bwd(const LogprobP& p, cudaStream_t s) {
  const size_t smem = tile_bytes<T, MODE>(p.x.C) * (p.accumulate ? 2 : 1);
  constexpr uint32_t N = kPlaces<MODE, G>;
  return p.entropy || p.dentropy ? go(logprob_positions_grad<T, MODE, true, G>, p, N, smem, s) : go(logprob_positions_grad<T, MODE, false, G>, p, N, smem, s);
}

template <typename T>
int logprob_positions(const LogprobP& p, cudaStream_t s) {
  const int mode = position_mode<T>(p.x, p.logits);
  if (mode < 0) return AD_ERR_UNSUPPORTED;
  if (p.x.C <= 32) {
    if (p.top <= 1 || p.top > 8) return go_few<T, 4, 1>(p, mode, s);
    return p.top <= 3 ? go_few<T, 4, 3>(p, mode, s) : go_few<T, 4, 8>(p, mode, s);
  }
  if (mode == 0) return go_fwd<T, 0, 4>(p, s);
  return mode == 1 ? go_fwd<T, 1, 1>(p, s) : go_fwd<T, 2, 1>(p, s);
}
template <typename T>
int logprob_positions_bwd(const LogprobP& p, cudaStream_t s) {
  int mode = position_mode<T>(p.x, p.logits);
  if (mode == 0 && (p.g.HW == 0 || (uint64_t)p.g.step * sizeof(T) > 0xffffffffu)) mode = -1;   // the gradient of an image of one position, packed
  if (mode > 0 && p.g.step != 1) mode = -1;
  if (mode == 2 && position_mode<T>(p.g, p.dlogits) != 2) mode = 1;
  if (mode < 0) return AD_ERR_UNSUPPORTED;
  if (p.x.C <= 32) return p.entropy || p.dentropy ? go_few_bwd<T, 4, true>(p, mode, s) : go_few_bwd<T, 4, false>(p, mode, s);
  if (mode == 0) return go_bwd<T, 0, 4>(p, s);
  return mode == 1 ? go_bwd<T, 1, 1>(p, s) : go_bwd<T, 2, 1>(p, s);
}
template int logprob_positions<float>(const LogprobP&, cudaStream_t);
template int logprob_positions<__nv_bfloat16>(const LogprobP&, cudaStream_t);
template int logprob_positions_bwd<float>(const LogprobP&, cudaStream_t);
template int logprob_positions_bwd<__nv_bfloat16>(const LogprobP&, cudaStream_t);

}  // namespace adk
