// Log probabilities of given classes, with entropy, rank and top alternatives, and their gradient.
//
// Forward: bytes of the logits, read once.  The top classes come out of the same pass: the row is dealt out in 256 shares
// (a block's threads, or eight per lane of a warp), each share keeps its largest value and the first vector that holds it,
// and the k-th of these 256 pairs bounds the row's k-th class from below, ties by class included: k elements are in front of
// or at it.  Only the shares that reach it, k of them, are read again, for the elements at or in front of the bound.
// Backward: the sums as in the forward pass, then the row once more (out of the L2 or L1) for the gradient.
#include <cooperative_groups.h>

#include "rows.cuh"

namespace cg = cooperative_groups;

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


// ---------------------------------------------------------------- top classes
struct TopMem {
  Key *list, *cand;   // the result, in order; what is at or in front of the bound
  uint32_t cap, *n;   // room in cand, and how many there are (more than cap: not all are there)
  __host__ __device__ static constexpr uint32_t room(uint32_t k) { return 64 + 9 * k; }   // k vectors of equal elements and the single ones fit
  __device__ void push(float v, uint32_t c) {
    const uint32_t at = atomicAdd(n, 1u);
    if (at < cap) cand[at] = key_of(v, c);
  }
};

// Of 256 shares, eight per lane (value key, 0 for none, and class): the k-th by value, then class.  value 0: fewer than k.
template <int SHIFT>
__device__ void kth_share(const uint32_t (&kv)[8], const uint32_t (&kc)[8], uint32_t k, uint32_t& value, uint32_t& cls) {
  uint32_t t = 0;
  for (uint32_t bit = 1u << (31 - SHIFT); bit; bit >>= 1) {
    uint32_t n = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) n += (kv[i] >> SHIFT) >= (t | bit);
    if (__reduce_add_sync(0xffffffffu, n) >= k) t |= bit;
  }
  uint32_t over = 0, same = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) { over += (kv[i] >> SHIFT) > t; same += (kv[i] >> SHIFT) == t; }
  over = __reduce_add_sync(0xffffffffu, over);
  same = __reduce_add_sync(0xffffffffu, same);
  value = t == 0 ? 0u : SHIFT ? t << SHIFT | (t >> (31 - SHIFT) ? 0u : (1u << SHIFT) - 1) : t;   // the bits that a key's sign tells
  cls = kNoClass;
  if (t != 0 && over + same > k) {
    uint32_t u = 0;
    for (uint32_t bit = 1u << 30; bit; bit >>= 1) {
      uint32_t n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += (kv[i] >> SHIFT) == t && kc[i] < (u | bit);
      if (over + __reduce_add_sync(0xffffffffu, n) < k) u |= bit;
    }
    cls = u;
  }
}

// The list out of the candidates: each one's place is the number of those in front of it
template <int NT>
__device__ void sort_candidates(Group<NT>& g, const TopMem& t, uint32_t n, uint32_t k) {
  Key least = 0;
  if (n > 64 + 2 * k) {   // many equal or clustered ones: the k-th first, bit by bit
    for (Key bit = 1ull << 63; bit; bit >>= 1) {
      uint32_t m = 0;
      for (uint32_t i = g.tid; i < n; i += NT) m += t.cand[i] >= (least | bit);
      if (g.sum(m) >= k) least |= bit;
    }
  }
  for (uint32_t i = g.tid; i < n; i += NT) {
    const Key key = t.cand[i];
    if (key < least) continue;
    uint32_t at = 0;
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) at += t.cand[j] > key;
    if (at < k) t.list[at] = key;
  }
  for (uint32_t i = n + g.tid; i < k; i += NT) t.list[i] = 0;
  g.sync();
}

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
  if (p.entropy) p.entropy[r] = H;
  if (p.logp) p.logp[r] = l < p.x.C ? s.log_p(xl, p.scale) : 0.f;
}

// ---------------------------------------------------------------- any layout, any numbers: plain loops over one row
template <int NT, typename T, bool BWD>
__device__ void plain_row(Group<NT>& g, const LogprobP& p, size_t r, const TopMem& t) {
  const T* x = (const T*)p.logits + p.x.offset(r);
  const int64_t st = p.x.step;
  const uint32_t C = p.x.C, l = p.label ? p.label[r] : kNoClass;
  const float xl = l < C ? ld_f(x + l * st) : 0.f;
  RowSums s;
  float E;
  plain_sums<Group<NT>, T, true>(g, x, st, C, p.cs, s, E);
  const float H = s.some ? kLn2 * (s.L - E / s.S) : 0.f;
  if (g.tid == 0) put_row(p, s, r, H, l, xl);
  if constexpr (!BWD) {
    if (p.rank) {
      uint32_t n = 0;
      for (uint32_t c = g.tid; c < C; c += NT) n += in_front(ld_f(x + c * st), c, xl, l);
      n = g.sum(n);
      if (g.tid == 0) p.rank[r] = l < C ? n : kNoClass;
    }
    if (p.top) {
      rounds(g, t, x, st, 0, C, p.top);
      for (uint32_t i = g.tid; i < p.top; i += NT) put_top(p, s, r, i, t.list[i]);
      g.sync();
    }
  } else {
    const float dl = p.dlogp && l < C && s.some ? p.dlogp[r] : 0.f, dh = p.dentropy ? p.dentropy[r] : 0.f;
    const float A = (p.dlse ? p.dlse[r] : 0.f) - dl, rS = s.some ? 1.f / s.S : 0.f;
    T* o = (T*)p.dlogits + p.g.offset(r);
    g.sync();   // the label's logit has been read by all
    for (uint32_t c = g.tid; c < C; c += NT) {
      const float u = (ld_f(x + c * st) - s.m) * p.cs, pc = exp2_fast(u) * rS;
      float d = pc * A;
      if (p.dentropy && pc != 0.f) d -= dh * pc * (kLn2 * (u - s.L) + H);
      if (c == l) d += dl;
      d *= p.scale;
      if (p.accumulate) d += ld_f(o + c * p.g.step);
      st_f(o + c * p.g.step, d);
    }
  }
}

template <typename T, bool BWD>
__global__ void __launch_bounds__(256) logprob_any(LogprobP p) {
  grid_dependency();
  __shared__ Key list[8][kMostTop];
  Group<32> g(nullptr);
  TopMem t = {list[threadIdx.x >> 5], nullptr, 0, nullptr};
  const size_t warp = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nw = ((size_t)gridDim.x * blockDim.x) >> 5;
  for (size_t r = warp; r < p.x.rows; r += nw) plain_row<32, T, BWD>(g, p, r, t);
}

// ---------------------------------------------------------------- rows of many neighbouring classes
// NT 32: a warp per row, eight vectors per lane and batch.  NT 256: a block per row, or a cluster of blocks, four vectors.
// ENT: the entropy is asked for.  RANK: the label's rank.  TOP: top classes.  BWD: the gradient.
template <int NT, typename T, bool ENT, bool RANK, bool TOP, bool BWD>
__global__ void __launch_bounds__(256) logprob_rows(LogprobP p) {
  constexpr int U = NT == 32 ? 8 : 4, SH = NT == 32 ? 8 : 1, V = Vec<T>::V;
  typedef Vec<T> X;
  extern __shared__ Key dyn[];
  __shared__ Key red[kRowWarps];
  __shared__ Part parts[kRowWarps], whole;
  __shared__ uint32_t sv[NT == 32 ? 1 : 256], sc[NT == 32 ? 1 : 256], bound[2], flagged[kMostTop], count[kRowWarps], nflag;
  grid_dependency();
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts_n = NT == 32 ? 1 : cluster.num_blocks(), part = NT == 32 ? 0 : cluster.block_rank();
  Group<NT> g(red);
  const uint32_t C = p.x.C, warp = threadIdx.x >> 5;
  TopMem t = {nullptr, nullptr, TopMem::room(p.top), &count[NT == 32 ? warp : 0]};
  if (TOP) {
    t.list = dyn + (NT == 32 ? (size_t)warp * (p.top + t.cap) : 0);
    t.cand = t.list + p.top;
  }
  const size_t row0 = NT == 32 ? (size_t)blockIdx.x * kRowWarps + warp : blockIdx.x / parts_n;
  const size_t rows_n = NT == 32 ? (size_t)gridDim.x * kRowWarps : gridDim.x / parts_n;
  for (size_t r = row0; r < p.x.rows; r += rows_n) {
    const T* x = (const T*)p.logits + p.x.offset(r);
    const Strip<T> b(x, C, part, parts_n);
    const uint4* xv = (const uint4*)(x + b.head);
    const uint32_t l = p.label ? p.label[r] : kNoClass;
    const float xl = l < C ? ld_f(x + l) : 0.f;
    // vectors in front of the label's count what is at least its logit, the others what is above it
    const bool low = xl == -INFINITY;   // there is nothing below: all classes in front of it count, whatever they hold
    const uint32_t lv = l < b.head ? 0 : (l - b.head) / V;
    const float thr0 = low ? INFINITY : X::below(xl);
    Part a;
    a.clear();
    float km[SH];
    uint32_t kc[SH];
#pragma unroll
    for (int i = 0; i < SH; ++i) { km[i] = -INFINITY; kc[i] = kNoClass; }
    if (g.tid < 2 * V) {
      const uint32_t c = b.single(g.tid);
      if (c != kNoClass) {
        const float v = ld_f(x + c);
        a.add<ENT>(v, p.cs);
        if (RANK) a.cnt += low ? c > l && v > xl : in_front(v, c, xl, l);
      }
    }
    for (uint32_t v0 = b.vb; v0 < b.ve; v0 += U * NT) {
      uint4 w[U];
      typename X::Max mx[U], most;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t v = v0 + u * NT + g.tid;
        w[u] = v < b.ve ? xv[v] : X::none();
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        mx[u] = X::max(w[u]);
        most = u ? X::max(most, mx[u]) : mx[u];
      }
      const float bm = X::value(most);
      if (TOP && SH > 1) {
#pragma unroll
        for (int u = 0; u < SH; ++u) {
          const float m = X::value(mx[u]);
          const uint32_t v = v0 + u * NT + g.tid;
          if (v < b.ve && (m > km[u] || kc[u] == kNoClass)) { km[u] = m; kc[u] = b.class_of(v); }
        }
      }
      if (TOP && SH == 1 && (bm > km[0] || kc[0] == kNoClass)) {
        km[0] = bm;
#pragma unroll
        for (int u = U - 1; u >= 0; --u) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v < b.ve && X::value(mx[u]) == bm) kc[0] = b.class_of(v);
        }
      }
      if (bm > a.m) {
        a.m = bm;
        a.refer<ENT>(fmaxf(a.mc, Part::reference(bm, p.cs)));
      }
      float S[4] = {0.f, 0.f, 0.f, 0.f}, E[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (v0 + u * NT >= b.ve) break;
        float f[V];
        X::unpack(w[u], f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float z = fmaf(f[i], p.cs, -a.mc);
          if (ENT) z = above_nothing(z);
          const float e = exp2_fast(z);
          S[i & 3] += e;
          if (ENT) E[i & 3] = fmaf(e, z, E[i & 3]);
        }
        if (RANK) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v < b.ve) a.cnt += X::above(w[u], v < lv ? thr0 : xl);
        }
      }
      a.S += (S[0] + S[1]) + (S[2] + S[3]);
      if (ENT) a.E += (E[0] + E[1]) + (E[2] + E[3]);
    }
    if (RANK && l < C && l >= b.head && lv >= b.vb && lv < b.ve && g.tid == 0)   // the label's own vector: the elements in front of it
      for (uint32_t c = b.class_of(lv); c < l; ++c) {
        const float v = ld_f(x + c);
        if (low) a.cnt -= v > xl;
        else a.cnt += v == xl;
      }
    a.join_lanes<ENT>();
    if (NT != 32) {
      if ((g.tid & 31) == 0) parts[warp] = a;
      if (TOP) {
        sv[g.tid] = kc[0] == kNoClass ? 0u : value_key(km[0]);
        sc[g.tid] = kc[0];
      }
      __syncthreads();
      a = parts[0];
#pragma unroll
      for (int i = 1; i < kRowWarps; ++i) a.join<ENT>(parts[i]);
      if (parts_n > 1) {
        if (g.tid == 0) whole = a;
        cluster.sync();
        a = *cluster.map_shared_rank(&whole, 0);
        for (uint32_t q = 1; q < parts_n; ++q) a.join<ENT>(*cluster.map_shared_rank(&whole, q));
      }
    }
    if (a.strange(p.cs)) {
      if (part == 0) plain_row<NT, T, BWD>(g, p, r, t);
      if (parts_n > 1) cluster.sync();
      else g.sync();
      continue;
    }
    RowSums s;
    s.set(a.m, a.mc, a.S, p.cs);
    const float H = s.some ? kLn2 * (s.L - a.E / s.S) : 0.f;
    if (g.tid == 0 && part == 0) {
      put_row(p, s, r, H, l, xl);
      if (RANK) p.rank[r] = l < C ? a.cnt + (low ? l : 0u) : kNoClass;
    }
    if constexpr (TOP) {
      const uint32_t k = p.top;
      uint32_t tv, tc;
      if (NT == 32) {
        uint32_t kv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) kv[i] = kc[i % SH] == kNoClass ? 0u : value_key(km[i % SH]);
        uint32_t cc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) cc[i] = kc[i % SH];
        kth_share<X::kKeyShift>(kv, cc, k, tv, tc);
        if (g.tid == 0) *t.n = 0;
        g.sync();
        const float least = tv ? key_value(tv) : -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (kv[i] > tv || (kv[i] == tv && cc[i] <= tc && kv[i])) {
            for (uint32_t v = b.vb + i * 32 + g.tid; v < b.ve; v += 256) {
              float f[V];
              X::unpack(xv[v], f);
              const uint32_t c0 = b.class_of(v);
#pragma unroll
              for (int j = 0; j < V; ++j)
                if (f[j] > least || (f[j] == least && c0 <= tc)) t.push(f[j], c0 + j);
            }
          }
      } else {
        if (warp == 0) {
          uint32_t kv[8], cc[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) { kv[i] = sv[i * 32 + g.tid]; cc[i] = sc[i * 32 + g.tid]; }
          kth_share<X::kKeyShift>(kv, cc, k, tv, tc);
          if (g.tid == 0) { bound[0] = tv; bound[1] = tc; *t.n = 0; nflag = 0; }
        }
        __syncthreads();
        tv = bound[0];
        tc = bound[1];
        const uint32_t mine = sv[g.tid];
        if (mine > tv || (mine == tv && sc[g.tid] <= tc && mine)) flagged[atomicAdd(&nflag, 1u)] = g.tid;
        __syncthreads();
        const float least = tv ? key_value(tv) : -INFINITY;
        const uint32_t per = (b.ve - b.vb + NT - 1) / NT;
        // the shares' vectors, over all threads
        for (uint32_t i = g.tid; i < nflag * per; i += NT) {
          const uint32_t v = b.vb + i % per * NT + flagged[i / per];
          if (v >= b.ve) continue;
          float f[V];
          X::unpack(xv[v], f);
          const uint32_t c0 = b.class_of(v);
#pragma unroll
          for (int j = 0; j < V; ++j)
            if (f[j] > least || (f[j] == least && c0 <= tc)) t.push(f[j], c0 + j);
        }
      }
      if (g.tid < 2 * V) {
        const uint32_t c = b.single(g.tid);
        if (c != kNoClass) {
          const float v = ld_f(x + c), least = tv ? key_value(tv) : -INFINITY;
          if (v > least || (v == least && c <= tc)) t.push(v, c);
        }
      }
      g.sync();
      const uint32_t n = *t.n;
      if (n <= t.cap) sort_candidates<NT>(g, t, n, k);
      else rounds<NT, T>(g, t, x, 1, b.begin(), b.end(), k);
      if (parts_n == 1) {
        for (uint32_t i = g.tid; i < k; i += NT) put_top(p, s, r, i, t.list[i]);
      } else {
        // every block's list is in order: an entry's place in the row's is its own and those in front of it in the others
        cluster.sync();
        Key* all = t.cand + t.cap;
        for (uint32_t i = g.tid; i < parts_n * k; i += NT) all[i] = cluster.map_shared_rank(t.list, i / k)[i % k];
        __syncthreads();
        if (g.tid < k) {
          const Key key = t.list[g.tid];
          uint32_t at = 0;
          for (uint32_t q = 0; q < parts_n; ++q) {
            uint32_t lo = 0, hi = k;
            while (lo < hi) {
              const uint32_t mid = (lo + hi) / 2;
              if (all[q * k + mid] > key) lo = mid + 1;
              else hi = mid;
            }
            at += lo;
          }
          if (key && at < k) put_top(p, s, r, at, key);
        }
      }
    }
    if constexpr (BWD) {
      const float dl = p.dlogp && l < C && s.some ? p.dlogp[r] : 0.f, dh = p.dentropy ? p.dentropy[r] : 0.f;
      const float A = (p.dlse ? p.dlse[r] : 0.f) - dl, k = s.some ? p.scale / s.S : 0.f;
      // e (c0 + c1 u) with e = 2^u: scale p (A - dentropy (log p + H))
      const float c1 = ENT ? -k * dh * kLn2 : 0.f, c0 = ENT ? k * (A - dh * (H - kLn2 * s.L)) : k * A;
      T* o = (T*)p.dlogits + p.g.offset(r);
      const bool even = (((uintptr_t)o ^ (uintptr_t)x) & 15u) == 0;   // both have their vectors at the same classes
      auto grad = [&](float v) {
        float u = fmaf(v, p.cs, -s.mc);
        if (ENT) u = above_nothing(u);
        return exp2_fast(u) * (ENT ? fmaf(c1, u, c0) : c0);
      };
      // the label's class is written last, over what the loop wrote
      const bool mine = l < C && l >= b.begin() && l < b.end() && g.tid == 0;
      float gl = 0.f;
      if (mine) gl = grad(xl) + p.scale * dl + (p.accumulate ? ld_f(o + l) : 0.f);
      if (parts_n == 1) g.sync();   // its logit has been read by all, and what it adds to (a cluster has met already)
      else __syncthreads();
      if (g.tid < 2 * V) {
        const uint32_t c = b.single(g.tid);
        if (c != kNoClass) st_f(o + c, grad(ld_f(x + c)) + (p.accumulate ? ld_f(o + c) : 0.f));
      }
      uint4* ov = (uint4*)(o + b.head);
      for (uint32_t v0 = b.vb; v0 < b.ve; v0 += U * NT) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v < b.ve) w[u] = xv[v];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v >= b.ve) break;
          float f[V];
          X::unpack(w[u], f);
#pragma unroll
          for (int i = 0; i < V; ++i) f[i] = grad(f[i]);
          if (even) {
            if (p.accumulate) {
              float d[V];
              X::unpack(ov[v], d);
#pragma unroll
              for (int i = 0; i < V; ++i) f[i] += d[i];
            }
            ov[v] = X::pack(f);
          } else {
            T* os = o + b.class_of(v);
#pragma unroll
            for (int i = 0; i < V; ++i) st_f(os + i, p.accumulate ? f[i] + ld_f(os + i) : f[i]);
          }
        }
      }
      g.sync();
      if (mine) st_f(o + l, gl);
    }
    if (parts_n > 1) cluster.sync();   // what the others read of this block's
    else g.sync();
  }
}

// ---------------------------------------------------------------- a thread per position
// The first KT classes of those seen so far.  16-bit values: value and class in one word, the list sorted by exchanges.
template <typename T, int KT> struct Firsts;
template <int KT> struct Firsts<__nv_bfloat16, KT> {
  uint32_t k[KT] = {};
  __device__ void add(float v, uint32_t c) {
    uint32_t t = v == v ? (value_key(v) & 0xffff0000u) | (0xffffu - c) : 0u;
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
    uint32_t t = v == v ? value_key(v) : 0u;
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

// KT: room for the top classes in registers (0: none, or more than eight: one round over the classes for each)
template <typename T, int MODE, int KT>
__global__ void __launch_bounds__(kPositions) logprob_positions(LogprobP p) {
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  T* tile = (T*)tiles;
  const uint32_t C = p.x.C;
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    if (MODE) {
      copy_tile<T, MODE>((const T*)p.logits, p.x, r0, (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions), tile);
      __syncthreads();
    }
    if (r < p.x.rows) {
      const Position<T, MODE> x = {MODE ? tile + threadIdx.x * tile_pitch<T, MODE>(C) : (const T*)p.logits + p.x.offset(r), p.x.step, C};
      const uint32_t l = p.label ? p.label[r] : kNoClass;
      const float xl = l < C ? x.get(l) : 0.f;
      Part a;
      a.clear();
      Firsts<T, KT ? KT : 1> top;
      for (uint32_t c = 0; c < C; c += 8) {
        float f[8], bm;
        x.batch(c, f);
        bm = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
        if (bm > a.m) {
          a.m = bm;
          a.refer<true>(fmaxf(a.mc, Part::reference(bm, p.cs)));
        }
        float S[2] = {0.f, 0.f}, E[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float u = above_nothing(fmaf(f[i], p.cs, -a.mc)), e = exp2_fast(u);
          S[i & 1] += e;
          E[i & 1] = fmaf(e, u, E[i & 1]);
        }
        a.S += S[0] + S[1];
        a.E += E[0] + E[1];
        if (p.rank) {
#pragma unroll
          for (int i = 0; i < 8; ++i) a.cnt += c + i < C && in_front(f[i], c + i, xl, l);
        }
        if (KT) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (c + i < C) top.add(f[i], c + i);
        }
      }
      RowSums s;
      if (a.strange(p.cs)) plain_position<true>(x, p.cs, s, a.E);
      else s.set(a.m, a.mc, a.S, p.cs);
      put_row(p, s, r, s.some ? kLn2 * (s.L - a.E / s.S) : 0.f, l, xl);
      if (p.rank) p.rank[r] = l < C ? a.cnt : kNoClass;
      if (KT) {
#pragma unroll
        for (int i = 0; i < KT; ++i)
          if ((uint32_t)i < p.top) put_top(p, s, r, i, top.key(i));
      } else {
        Key last = ~0ull;
        for (uint32_t i = 0; i < p.top; ++i) {
          Key best = 0;
          if (last)
            for (uint32_t c = 0; c < C; ++c) {
              const float v = x.get(c);
              const Key key = v == v ? key_of(v, c) : 0;
              if (key < last && key > best) best = key;
            }
          put_top(p, s, r, i, best);
          last = best;
        }
      }
    }
    if (MODE) __syncthreads();
  }
}

template <typename T, int MODE, bool ENT>
__global__ void __launch_bounds__(kPositions) logprob_positions_bwd(LogprobP p) {
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  const uint32_t C = p.x.C;
  T *tile = (T*)tiles, *olds = tile + kPositions * tile_pitch<T, MODE ? MODE : 1>(C);   // what the gradient is added to
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions);
    if (MODE) {
      copy_tile<T, MODE>((const T*)p.logits, p.x, r0, n, tile);
      if (p.accumulate) copy_tile<T, MODE>((const T*)p.dlogits, p.g, r0, n, olds);
      __syncthreads();
    }
    if (r < p.x.rows) {
      const uint32_t at = threadIdx.x * tile_pitch<T, MODE ? MODE : 1>(C);
      const Position<T, MODE> x = {MODE ? tile + at : (const T*)p.logits + p.x.offset(r), p.x.step, C};
      const Position<T, MODE> o = {MODE ? tile + at : (T*)p.dlogits + p.g.offset(r), p.g.step, C};
      const Position<T, MODE> old = {MODE ? olds + at : (T*)p.dlogits + p.g.offset(r), p.g.step, C};
      const uint32_t l = p.label ? p.label[r] : kNoClass;
      const float xl = l < C ? x.get(l) : 0.f;
      Part a;
      a.clear();
      for (uint32_t c = 0; c < C; c += 8) {
        float f[8], bm;
        x.batch(c, f);
        bm = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
        if (bm > a.m) {
          a.m = bm;
          a.refer<ENT>(fmaxf(a.mc, Part::reference(bm, p.cs)));
        }
        float S[2] = {0.f, 0.f}, E[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float u = fmaf(f[i], p.cs, -a.mc);
          if (ENT) u = above_nothing(u);
          const float e = exp2_fast(u);
          S[i & 1] += e;
          if (ENT) E[i & 1] = fmaf(e, u, E[i & 1]);
        }
        a.S += S[0] + S[1];
        if (ENT) a.E += E[0] + E[1];
      }
      RowSums s;
      const bool strange = a.strange(p.cs);
      if (strange) plain_position<ENT>(x, p.cs, s, a.E);
      else s.set(a.m, a.mc, a.S, p.cs);
      const float H = s.some ? kLn2 * (s.L - a.E / s.S) : 0.f;
      put_row(p, s, r, H, l, xl);
      const float dl = p.dlogp && l < C && s.some ? p.dlogp[r] : 0.f, dh = p.dentropy ? p.dentropy[r] : 0.f;
      const float A = (p.dlse ? p.dlse[r] : 0.f) - dl, k = s.some ? p.scale / s.S : 0.f;
      const float c1 = ENT ? -k * dh * kLn2 : 0.f, c0 = ENT ? k * (A - dh * (H - kLn2 * s.L)) : k * A;
      const float mc = s.mc;
      for (uint32_t c = 0; c < C; c += 8) {
        float f[8];
        x.batch(c, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          float u = strange ? (f[i] - s.m) * p.cs : fmaf(f[i], p.cs, -mc);
          if (ENT) u = above_nothing(u);
          f[i] = exp2_fast(u) * (ENT ? fmaf(c1, u, c0) : c0);
          if (c + i == l) f[i] += p.scale * dl;
          if (c + i < C) o.set(c + i, p.accumulate ? f[i] + old.get(c + i) : f[i]);
        }
      }
    }
    if (MODE) {
      __syncthreads();
      write_tile<T, MODE>((T*)p.dlogits, p.g, r0, n, tile);
      __syncthreads();
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
static int launch_any(const LogprobP& p, cudaStream_t s) {
  launch(logprob_any<T, BWD>, grid_for(p.x.rows, 8), 256, 0, s, p);
  return AD_OK;
}

template <int NT, typename T, bool ENT, bool RANK, bool TOP, bool BWD>
static int launch_rows(const LogprobP& p, cudaStream_t s) {
  auto kernel = logprob_rows<NT, T, ENT, RANK, TOP, BWD>;
  const uint32_t n = NT == 32 ? 1 : row_parts(p.x.rows, (size_t)p.x.C * sizeof(T));
  const size_t keys = TOP ? (NT == 32 ? (size_t)kRowWarps * (p.top + TopMem::room(p.top)) : p.top + TopMem::room(p.top) + (n > 1 ? n * p.top : 0)) : 0;
  constexpr int most = (int)(sizeof(Key) * kRowWarps * (kMostTop + TopMem::room(kMostTop)));   // a warp per row
  // the limit belongs to the function: the most that it takes
  if (keys * sizeof(Key) > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch_row_kernel(kernel, p, NT == 32 ? (p.x.rows + kRowWarps - 1) / kRowWarps : p.x.rows, n, keys * sizeof(Key), s);
  return AD_OK;
}

template <int NT, typename T>
static int launch_fwd(const LogprobP& p, cudaStream_t s) {
  const bool ent = p.entropy != nullptr, rank = p.rank != nullptr, top = p.top != 0;
  if (top) {
    if (ent) return rank ? launch_rows<NT, T, true, true, true, false>(p, s) : launch_rows<NT, T, true, false, true, false>(p, s);
    return rank ? launch_rows<NT, T, false, true, true, false>(p, s) : launch_rows<NT, T, false, false, true, false>(p, s);
  }
  if (ent) return rank ? launch_rows<NT, T, true, true, false, false>(p, s) : launch_rows<NT, T, true, false, false, false>(p, s);
  return rank ? launch_rows<NT, T, false, true, false, false>(p, s) : launch_rows<NT, T, false, false, false, false>(p, s);
}
template <int NT, typename T>
static int launch_bwd(const LogprobP& p, cudaStream_t s) {
  return p.entropy || p.dentropy ? launch_rows<NT, T, true, false, false, true>(p, s) : launch_rows<NT, T, false, false, false, true>(p, s);
}

template <typename P>
static int launch_positions(void (*kernel)(P), const P& p, size_t smem, cudaStream_t s) {
  // the limit belongs to the function: the most that it takes
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * (kFewClasses * 4 + 16) * kPositions) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch(kernel, position_blocks(p.x.rows), kPositions, smem, s, p);
  return AD_OK;
}
template <typename T, int MODE>
static int positions_fwd(const LogprobP& p, cudaStream_t s) {
  const size_t smem = tile_bytes<T, MODE>(p.x.C);
  if (p.top == 0 || p.top > 8) return launch_positions(logprob_positions<T, MODE, 0>, p, smem, s);
  if (p.top == 1) return launch_positions(logprob_positions<T, MODE, 1>, p, smem, s);
  if (p.top <= 3) return launch_positions(logprob_positions<T, MODE, 3>, p, smem, s);
  return launch_positions(logprob_positions<T, MODE, 8>, p, smem, s);
}
template <typename T, int MODE>
static int positions_bwd(const LogprobP& p, cudaStream_t s) {
  const size_t smem = tile_bytes<T, MODE>(p.x.C) * (p.accumulate ? 2 : 1);
  return p.entropy || p.dentropy ? launch_positions(logprob_positions_bwd<T, MODE, true>, p, smem, s) : launch_positions(logprob_positions_bwd<T, MODE, false>, p, smem, s);
}

template <typename T, bool BWD>
static int launch_logprob(const LogprobP& p, cudaStream_t s) {
  int rc, mode = position_mode<T>(p.x, p.logits);
  if (BWD && mode == 0 && p.g.HW == 0) mode = -1;   // the gradient of an image of one position, packed
  if (BWD && mode == 2 && p.accumulate && position_mode<T>(p.g, p.dlogits) != 2) mode = 1;
  if (mode > 0 && BWD && p.g.step != 1) mode = -1;
  if (mode == 0) rc = BWD ? positions_bwd<T, 0>(p, s) : positions_fwd<T, 0>(p, s);
  else if (mode == 1) rc = BWD ? positions_bwd<T, 1>(p, s) : positions_fwd<T, 1>(p, s);
  else if (mode == 2) rc = BWD ? positions_bwd<T, 2>(p, s) : positions_fwd<T, 2>(p, s);
  else if (p.x.step != 1 || (BWD && p.g.step != 1)) rc = launch_any<T, BWD>(p, s);
  else if (p.x.C * sizeof(T) <= 8192) rc = BWD ? launch_bwd<32, T>(p, s) : launch_fwd<32, T>(p, s);
  else rc = BWD ? launch_bwd<256, T>(p, s) : launch_fwd<256, T>(p, s);
  if (rc != AD_OK) return rc;
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
