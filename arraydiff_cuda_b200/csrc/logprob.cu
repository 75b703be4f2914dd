// Log probabilities of given classes, with entropy, rank and top alternatives, and their gradient: rows of neighbouring classes.
//
// Forward: bytes of the logits, read once.  The top classes come out of the same pass: the row is dealt out in 256 shares
// (a block's threads, or eight per lane of a warp), each share keeps its largest value, and the k-th of these 256 bounds
// the row's k-th class from below.  Only the shares that reach it, or the batches of theirs that do, are looked at again.
// Where more reach the bound than there is room for it rises; equal values go by class: those above it and the first equal ones.
// Backward: the sums as in the forward pass, then the row once more (out of shared memory or the L2) for the gradient.
//
// 4001 x 50001 bf16 (400 MB, 62 us at the copy rate): log-sum-exp 70 us, with the entropy 74, the rank 81 (labels
// at random), 8 alternatives 78; all of them 96 where labels are likely, 102 where not, bound by instructions (70 M, 69 % of the issue
// slots).  2000 x 100000 fp32 (124): 123.  Gradient of 4096 x 32000 bf16 (81): 109, with the entropy's 116: two exponentials per
// element (57 us of the special units) and a meeting of the block's warps between the passes.  One row of 32768 with 5
// alternatives: 8, by the latency of label, loads, sums, selection and a cluster's meeting, one behind the other; 64 x 131072 with
// 20: 16, by that and by four blocks a row, 256 of the 444 that the machine holds.
#include <cooperative_groups.h>

#include "logprob.cuh"

namespace cg = cooperative_groups;

namespace adk {

// ---------------------------------------------------------------- top classes
// One warp: places for `mine` things of each lane behind `n` that are there already, which is increased by all of them
__device__ __forceinline__ uint32_t places(uint32_t mine, uint32_t& n) {
  const uint32_t lane = threadIdx.x & 31;
  uint32_t upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t q = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= (uint32_t)o) upto += q;
  }
  const uint32_t at = n + upto - mine;
  n += __shfl_sync(0xffffffffu, upto, 31);
  return at;
}

// One warp: f(bit, place) for every bit that is set in the lanes' words, places one behind the other from n on
template <typename F>
__device__ __forceinline__ void each_bit(uint32_t bits, uint32_t& n, F&& f) {
  const uint32_t below = (1u << (threadIdx.x & 31)) - 1;
  for (uint32_t who; (who = __ballot_sync(0xffffffffu, bits != 0)) != 0; n += __popc(who))
    if (bits) {
      f((uint32_t)__ffs(bits) - 1, n + __popc(who & below));
      bits &= bits - 1;
    }
}

// One warp: of 256 shares' maxima, eight per lane (keys, 0 for none), the k-th, or less; 0: fewer than k
template <int SHIFT>
__device__ uint32_t kth_share(const uint32_t (&kv)[8], uint32_t k) {
  if (k <= (SHIFT ? 10 : 20)) {   // the k-th of the lanes' largest: little less, and sooner found than bit by bit
    uint32_t best = kv[0], t = 0;
#pragma unroll
    for (int i = 1; i < 8; ++i) best = max(best, kv[i]);
    for (uint32_t n = 0; n < k;) {
      t = __reduce_max_sync(0xffffffffu, best);
      if (t == 0) break;
      n += __popc(__ballot_sync(0xffffffffu, best == t));
      if (best == t) best = 0;
    }
    return t;
  }
  uint32_t t = 0;
  if (k <= 32) {   // of the lanes' two largest, bit by bit
    uint32_t a = 0, b = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t q = kv[i] >> SHIFT;
      b = max(b, min(a, q));
      a = max(a, q);
    }
    for (uint32_t bit = 1u << (31 - SHIFT); bit; bit >>= 1) {
      const uint32_t u = t | bit;
      if (__popc(__ballot_sync(0xffffffffu, a >= u)) + __popc(__ballot_sync(0xffffffffu, b >= u)) >= (int)k) t = u;
    }
  } else {
    for (uint32_t bit = 1u << (31 - SHIFT); bit; bit >>= 1) {
      uint32_t n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += (kv[i] >> SHIFT) >= (t | bit);
      if (__reduce_add_sync(0xffffffffu, n) >= k) t |= bit;
    }
  }
  return t == 0 ? 0u : SHIFT ? t << SHIFT | (t >> (31 - SHIFT) ? 0u : (1u << SHIFT) - 1) : t;   // the bits that a key's sign tells
}

// One warp: the list out of n candidates, each one's place being the number of those in front of it.  Q of them per lane and pass.
template <int Q>
__device__ __forceinline__ void sort_candidates(const TopMem& t, uint32_t n, uint32_t k, Key least) {
  const uint32_t lane = threadIdx.x & 31;
  for (uint32_t i0 = 0; i0 < n; i0 += 32 * Q) {
    Key key[Q];
    uint32_t at[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      key[q] = i0 + q * 32 + lane < n ? t.cand[i0 + q * 32 + lane] : 0;
      at[q] = 0;
    }
#pragma unroll 4
    for (uint32_t j = 0; j < n; ++j) {
      const Key other = t.cand[j];
#pragma unroll
      for (int q = 0; q < Q; ++q) at[q] += other > key[q];
    }
#pragma unroll
    for (int q = 0; q < Q; ++q)
      if (key[q] >= least && key[q] && at[q] < k) t.list[at[q]] = key[q];
  }
}
// One warp: the k-th of n candidates, bit by bit; 0: fewer
__device__ __noinline__ Key kth_candidate(const Key* cand, uint32_t n, uint32_t k) {
  Key least = 0;
  for (Key bit = 1ull << 63; bit; bit >>= 1) {
    uint32_t m = 0;
    for (uint32_t i = threadIdx.x & 31; i < n; i += 32) m += cand[i] >= (least | bit);
    if (__reduce_add_sync(0xffffffffu, m) >= k) least |= bit;
  }
  return least;
}
__device__ void sort_candidates(const TopMem& t, uint32_t n, uint32_t k) {
  const uint32_t lane = threadIdx.x & 31;
  __syncwarp();
  Key least = 0;
  if (n <= 32) {
    sort_candidates<1>(t, n, k, 0);
  } else {
    if (n > 64 + 2 * k) {   // many equal or clustered ones: the k-th first, and only those up to it
      least = kth_candidate(t.cand, n, k);
      uint32_t kept = 0;
      for (uint32_t i0 = 0; i0 < n; i0 += 32) {
        const Key key = i0 + lane < n ? t.cand[i0 + lane] : 0;
        __syncwarp();
        const uint32_t at = places(key >= least && key, kept);
        if (key >= least && key) t.cand[at] = key;   // not behind where it was
        __syncwarp();
      }
      n = kept;
    }
    sort_candidates<4>(t, n, k, least);
  }
  for (uint32_t i = n + lane; i < k; i += 32) t.list[i] = 0;
  __syncwarp();
}

// One warp: adds the first r elements of a strip that equal v, in order of their classes, to the n candidates
template <typename T>
__device__ void add_equal(const TopMem& t, const Strip<T>& b, const T* x, float v, uint32_t r, uint32_t& n) {
  constexpr uint32_t V = Vec<T>::V;
  const uint32_t lane = threadIdx.x & 31, most = n + r;
  for (uint32_t c0 = b.begin(); c0 < b.end() && n < most; c0 += 32 * V) {
    uint32_t hits = 0;
    for (uint32_t i = 0; i < V; ++i) {
      const uint32_t c = c0 + lane * V + i;
      if (c < b.end() && ld_f(x + c) == v) hits |= 1u << i;
    }
    uint32_t at = places(__popc(hits), n);
    for (uint32_t i = 0; i < V; ++i)
      if (hits >> i & 1 && at++ < most) t.cand[at - 1] = key_of(v, c0 + lane * V + i);
  }
  if (n > most) n = most;
}

// The maxima of what a thread has taken at a time: batches of four vectors, `1 << shift` of them together, as the upper
// half of the number.  [slot][thread]; none: a share's vectors are looked at one by one.
struct Maxima {
  const uint16_t* m;
  uint32_t shift, slots;
};
constexpr uint32_t kMostSlots = 8;
__device__ __forceinline__ uint32_t half_key(uint32_t h) { return h & 0x8000u ? 0xffffu ^ h : h | 0x8000u; }   // value_key >> 16

constexpr uint32_t kWork = 512;   // words of 16 bits that a selection works with: shares, and slots of 32 of them
template <int N> struct Loads { static constexpr int value = N; };

// One warp: a strip's list out of its 256 shares, of which lane i has number 32 j + i in kv[j]: the key of its largest value, 0
// for none.  Share s is the vectors vb + s + 256 n, xv[0] being vector vb.  `single`: a single element of the strip in this
// lane (class `sc`).  work: 256 words of 16 bits, with maxima kWork.
template <typename T>
__device__ void select_top(const TopMem& t, uint32_t k, const uint32_t (&kv)[8], const Maxima& mx, const Strip<T>& b, const T* x, const uint4* xv, uint32_t sc,
                           float single, uint16_t* work) {
  typedef Vec<T> X;
  constexpr int V = X::V;
  Group<32> g(nullptr);
  const uint32_t lane = g.tid;
  uint32_t lo = kth_share<X::kKeyShift>(kv, k);
  const uint32_t nv = b.ve - b.vb, per = mx.m ? mx.slots : (nv + 255) / 256;
  // All elements of the shares that reach the bound.  Where there is no room for them the bound rises to the k-th of those
  // found so far; where it is that one already, because so many equal it, only those above are taken, and of the equal ones the first.
  bool strict = false;
  for (int tries = 0; tries < 64; ++tries) {
    const float bound = lo ? key_value(lo) : -INFINITY;
    auto reaches = [&](float v) { return v >= bound; };
    uint32_t ns = 0, n = 0, mine = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine |= kv[i] && kv[i] >= lo ? 1u << i : 0u;
    each_bit(mine, ns, [&](uint32_t i, uint32_t at) { work[at] = (uint16_t)(i * 32 + lane); });
    __syncwarp();
    const uint32_t wide = per <= 1 ? 0 : 32 - __clz(per - 1);   // a share's vectors as a power of two
    uint16_t* list = work + 256;
    auto look = [&](auto loads, uint32_t i0, uint32_t vectors) {   // so many loads at a time
      constexpr int Q = decltype(loads)::value;
      uint4 w[Q];
      uint32_t at[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const uint32_t i = i0 + q * 32 + lane;
        at[q] = nv;
        if (i < vectors) {
          if (mx.m) {
            const uint32_t e = list[i >> (2 + mx.shift)], sub = i & ((4u << mx.shift) - 1);
            at[q] = (((e >> 8) << (2 + mx.shift)) + sub) * 256 + (e & 255);
          } else {
            at[q] = (i & ((1u << wide) - 1)) * 256 + work[i >> wide];
          }
        }
        w[q] = at[q] < nv ? xv[at[q]] : X::none();
      }
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        uint32_t hits = 0;
        const uint32_t c0 = b.class_of(b.vb + at[q]);
        if (at[q] < nv && reaches(X::value(X::max(w[q])))) {
          float f[V];
          X::unpack(w[q], f);
#pragma unroll
          for (int j = 0; j < V; ++j) hits |= reaches(f[j]) ? 1u << j : 0u;
        }
        each_bit(hits, n, [&](uint32_t j, uint32_t to) {
          if (to < t.cap) t.cand[to] = key_of(X::element(w[q], j), c0 + j);
        });
      }
    };
    for (uint32_t i0 = 0; i0 < ns && n <= t.cap; i0 += mx.m ? 32 : 256) {
      uint32_t vectors = ns << wide;
      if (mx.m) {   // the slots that reach it, of 32 shares at a time
        uint32_t slots = 0, found = 0;
        const uint32_t share = i0 + lane < ns ? work[i0 + lane] : 0;
        if (i0 + lane < ns)
          for (uint32_t q = 0; q < per; ++q) slots |= half_key(mx.m[q * 256 + share]) >= lo >> 16 ? 1u << q : 0u;
        if (i0) __syncwarp();
        each_bit(slots, found, [&](uint32_t q, uint32_t at) { list[at] = (uint16_t)(q * 256 + share); });
        __syncwarp();
        vectors = found * (4u << mx.shift);
      }
      for (uint32_t j0 = 0; j0 < vectors && n <= t.cap;) {
        if (vectors - j0 <= 32) {
          look(Loads<1>(), j0, vectors);
          j0 += 32;
        } else {
          look(Loads<4>(), j0, vectors);
          j0 += 128;
        }
      }
    }
    each_bit(sc != kNoClass && reaches(single) ? 1u : 0u, n, [&](uint32_t, uint32_t to) {
      if (to < t.cap) t.cand[to] = key_of(single, sc);
    });
    __syncwarp();
    if (n <= t.cap) {
      if (strict && n < k) add_equal<T>(t, b, x, key_value(lo - 1), k - n, n);
      sort_candidates(t, n, k);
      return;
    }
    const uint32_t higher = (uint32_t)(kth_candidate(t.cand, t.cap, k) >> 32);
    strict = higher == lo;
    lo = higher + strict;
    __syncwarp();
  }
  rounds<32, T>(g, t, x, 1, b.begin(), b.end(), k);
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
  plain_sums<NT, T, true>(g, x, st, C, p.cs, s, E);
  const float H = s.entropy(E);
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
  TopMem t = {list[threadIdx.x >> 5], nullptr, 0};
  const size_t warp = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nw = ((size_t)gridDim.x * blockDim.x) >> 5;
  for (size_t r = warp; r < p.x.rows; r += nw) plain_row<32, T, BWD>(g, p, r, t);
}

// ---------------------------------------------------------------- rows of many neighbouring classes
// What a thread finds in its vectors: sums, classes in front of the label, its shares of the row
template <int NT, typename T, bool ENT, bool RANK, bool TOP, int U_ = NT == 32 ? 8 : 4>
struct Scan {
  static constexpr int U = U_, SH = NT == 32 ? 8 : 1;
  typedef Vec<T> X;
  Part a;
  uint32_t km[SH];   // maxima of the eight shares of a lane, as keys; a thread's own share has a.m
  __device__ void clear() {
    a.clear();
#pragma unroll
    for (int i = 0; i < SH; ++i) km[i] = 0;
  }
  // v0: the first vector of the batch, lv: the label's; before that one counts what is above thr0, else what is above xl.
  // The batch's maximum.
  __device__ __forceinline__ float batch(uint32_t v0, const uint4 (&w)[U], bool full, const Strip<T>& b, uint32_t tid, float cs, float nothing, uint32_t lv, float xl, float thr0) {
    typename X::Max mx[U], most;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mx[u] = X::max(w[u]);
      most = u ? X::max(most, mx[u]) : mx[u];
    }
    const float bm = X::value(most);
    if (TOP && SH > 1) {
#pragma unroll
      for (int u = 0; u < SH; ++u)
        if (v0 + u * NT + tid < b.ve) km[u] = max(km[u], value_key(X::value(mx[u])));
    }
    add_vectors<ENT, U, T>(a, w, full ? U : (int)((b.ve - v0 + NT - 1) / NT), bm, cs, nothing);
    if (RANK && bm >= xl) {   // few batches hold something above a likely label
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t v = v0 + u * NT + tid;
        if (full || v < b.ve) a.cnt += X::above(w[u], v < lv ? thr0 : xl);
      }
    }
    return bm;
  }
};
// A label and what the rank's counting needs of it
template <typename T>
struct Label {
  uint32_t l, lv;
  float xl, thr0;
  bool low;   // its logit is -inf, nothing is below: all classes in front of it count, whatever they hold
  __device__ void fetch(const LogprobP& p, size_t r, const T* x, const Strip<T>& b) { fetch(p, p.label ? p.label[r] : kNoClass, x, b, 0); }
  __device__ void fetch(const LogprobP& p, uint32_t l_, const T* x, const Strip<T>& b, int) {
    l = l_;
    xl = l < p.x.C ? ld_f(x + l) : 0.f;
    low = xl == -INFINITY;
    lv = l < b.head ? 0 : (l - b.head) / Vec<T>::V;
    thr0 = low ? INFINITY : Vec<T>::below(xl);
  }
  // what the counting by vectors leaves out: lane i looks at the i-th element of the label's own vector
  __device__ uint32_t own_vector(const Strip<T>& b, const T* x, uint32_t C, uint32_t i) const {
    if (l >= C || l < b.head || lv < b.vb || lv >= b.ve || b.class_of(lv) + i >= l || i >= Vec<T>::V) return 0;
    const float v = ld_f(x + b.class_of(lv) + i);
    return low ? 0u - (v > xl) : (uint32_t)(v == xl);
  }
  __device__ bool single_counts(float v, uint32_t c) const { return low ? c > l && v > xl : in_front(v, c, xl, l); }
  __device__ uint32_t rank(uint32_t cnt, uint32_t C) const { return l < C ? cnt + (low ? l : 0u) : kNoClass; }
};
// NT 32: a warp per row, eight vectors per lane and batch.  NT 256: for few rows, a block or a cluster of blocks per row.
// ENT: the entropy is asked for.  RANK: the label's rank.  TOP: top classes.  BWD: the gradient.
template <int NT, typename T, bool ENT, bool RANK, bool TOP, bool BWD>
__global__ void __launch_bounds__(256, NT == 32 ? (TOP ? 2 : 4) : 3) logprob_rows(LogprobP p, uint32_t slots) {
  typedef Scan<NT, T, ENT, RANK, TOP> S;
  constexpr int U = S::U, V = Vec<T>::V;
  typedef Vec<T> X;
  extern __shared__ __align__(16) Key dyn[];   // batches of vectors, then what the top classes need
  __shared__ Key red[kRowWarps];
  __shared__ Part parts[kRowWarps], whole;
  __shared__ uint32_t sv[NT == 32 ? 1 : 256];
  __shared__ uint16_t work[NT == 32 ? kRowWarps : 1][TOP ? 256 : 1];
  grid_dependency();
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts_n = NT == 32 ? 1 : cluster.num_blocks(), part = NT == 32 ? 0 : cluster.block_rank();
  Group<NT> g(red);
  const uint32_t C = p.x.C, warp = threadIdx.x >> 5;
  const float nothing = as_nothing(p.cs);
  TopMem t = {nullptr, nullptr, TopMem::room(p.top)};
  if (TOP) {
    t.list = dyn + (size_t)slots * Feed<NT>::kBatch * 2 + (NT == 32 ? (size_t)warp * (p.top + t.cap) : 0);
    t.cand = t.list + p.top;
  }
  const size_t row0 = NT == 32 ? (size_t)blockIdx.x * kRowWarps + warp : blockIdx.x / parts_n;
  const size_t rows_n = NT == 32 ? (size_t)gridDim.x * kRowWarps : gridDim.x / parts_n;
  for (size_t r = row0; r < p.x.rows; r += rows_n) {
    const T* x = (const T*)p.logits + p.x.offset(r);
    const Strip<T> b(x, C, part, parts_n);
    const uint4* xv = (const uint4*)(x + b.head);
    Feed<NT> feed(xv, b.vb, b.ve, g.tid, slots, (uint4*)dyn);
    S scan;
    scan.clear();
    Part& a = scan.a;
    const uint32_t cls = g.tid < 2 * V ? b.single(g.tid) : kNoClass;
    const float single = cls != kNoClass ? ld_f(x + cls) : 0.f;
    Label<T> label;
    const uint32_t l = p.label ? p.label[r] : kNoClass;
    feed.template start<T>();
    label.fetch(p, l, x, b, 0);
    feed.template run<T, false>([&](uint32_t v0, const uint4 (&w)[U]) { scan.batch(v0, w, false, b, g.tid, p.cs, nothing, label.lv, label.xl, label.thr0); });
    if (TOP && NT != 32) sv[g.tid] = b.vb + g.tid < b.ve ? value_key(a.m) : 0u;
    if (cls != kNoClass) a.add<ENT>(single, p.cs);
    if (RANK) a.cnt += label.own_vector(b, x, C, g.tid) + (cls != kNoClass && label.single_counts(single, cls));
    a.join<ENT, 32>(p.cs);
    const uint32_t k = p.top;
    if (NT != 32) {
      if ((g.tid & 31) == 0) parts[warp] = a;
      __syncthreads();
      a = parts[g.tid % kRowWarps];
      a.join<ENT, kRowWarps>(p.cs);
    }
    if constexpr (TOP) {   // before the blocks of a cluster meet
      if (NT == 32 || warp == 0) {
        uint32_t kv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) kv[i] = NT == 32 ? scan.km[i % S::SH] : sv[i * 32 + g.tid];
        const Maxima none = {nullptr, 0, 0};
        // a part that is in shared memory as a whole is looked at there
        const uint4* vectors = NT != 32 && feed.batches() <= slots ? (const uint4*)dyn : xv + b.vb;
        select_top<T>(t, k, kv, none, b, x, vectors, cls, single, work[NT == 32 ? warp : 0]);
      }
    }
    if (parts_n > 1) {
      if (g.tid == kRowThreads - 1) whole = a;
      cluster.sync();
      const uint32_t q = g.tid % 8;
      if (q < parts_n) a = *cluster.map_shared_rank(&whole, q);
      else a.clear();
      a.join<ENT, 8>(p.cs);
    } else if (TOP) {
      g.sync();
    }
    const bool far = TOP && a.far(p.cs);   // without a list plain_row() costs one pass more, and its place here registers
    if (a.strange(p.cs) && !far) {
      if (parts_n > 1) cluster.sync();   // the others' sums have been read
      if (part == 0) plain_row<NT, T, BWD>(g, p, r, t);
      if (parts_n > 1) cluster.sync();
      else g.sync();
      continue;
    }
    RowSums s;
    if (far) plain_sums<NT, T, ENT>(g, x, 1, C, p.cs, s, a.E);   // list and rank stand; each block of a cluster for itself
    else s.set(a.m, a.mc, a.S, p.cs);
    const float H = s.entropy(a.E);
    if (g.tid == 0 && part == 0) {
      put_row(p, s, r, H, label.l, label.xl);
      if (RANK) p.rank[r] = label.rank(a.cnt, C);
    }
    if constexpr (TOP) {
      if (parts_n == 1) {
        for (uint32_t i = g.tid; i < k; i += NT) put_top(p, s, r, i, t.list[i]);
      } else {
        // every block's list is in order: an entry's place in the row's is its own and those in front of it in the others
        Key* all = t.cand + t.cap;
        const uint32_t n = parts_n * k;
        for (uint32_t i = g.tid; i < n; i += NT) all[i] = cluster.map_shared_rank(t.list, i / k)[i % k];
        __syncthreads();
        if (g.tid < k) {
          const Key key = t.list[g.tid];
          uint32_t at = 0;
          if (n <= 256) {
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) at += all[i] > key;
          } else {
            for (uint32_t q = 0; q < parts_n; ++q) {
              uint32_t lo = 0, hi = k;
              while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (all[q * k + mid] > key) lo = mid + 1;
                else hi = mid;
              }
              at += lo;
            }
          }
          if (key && at < k) put_top(p, s, r, at, key);
        }
      }
    }
    if constexpr (BWD) {
      Factors f;
      f.fetch(p, r, label.l);
      f.set<ENT>(p, s, H);
      T* o = (T*)p.dlogits + p.g.offset(r);
      const bool even = (((uintptr_t)o ^ (uintptr_t)x) & 15u) == 0;   // both have their vectors at the same classes
      // the label's class is written last, over what the loop wrote
      const bool mine = label.l < C && label.l >= b.begin() && label.l < b.end() && g.tid == 0;
      float gl = 0.f;
      if (mine) gl = f.grad<ENT>(label.xl, p.cs, s.mc) + f.dl + (p.accumulate ? ld_f(o + label.l) : 0.f);
      if (parts_n == 1) g.sync();   // its logit has been read by all, and what it adds to (a cluster has met already)
      else __syncthreads();
      if (cls != kNoClass) st_f(o + cls, f.grad<ENT>(single, p.cs, s.mc) + (p.accumulate ? ld_f(o + cls) : 0.f));
      feed.template run<T, true>([&](uint32_t v0, const uint4 (&w)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v >= b.ve) break;
          float h[V];
          grad_vector<ENT, T>(w[u], h, p.cs, s.mc, f.c0, f.c1, nothing);
          put_vector<T>(o + b.class_of(v), even, p.accumulate, h);
        }
      });
      g.sync();
      if (mine) st_f(o + label.l, gl);
    }
    if (parts_n > 1) cluster.sync();   // what the others read of this block's
    else g.sync();
  }
}

// Batches whose maxima share a slot: at most kMostSlots of them for a row
template <typename T>
__host__ __device__ inline uint32_t slot_shift(uint32_t C) {
  uint32_t s = 0;
  while ((C / Vec<T>::V + (1024u << s) - 1) / (1024u << s) > kMostSlots) ++s;
  return s;
}
// Many rows of many classes: see Stream.  Two rows are in hand, by parity.
template <typename T, int W>
struct LogprobSlot {
  Label<T> label;
  Part parts[W];
  uint32_t sv[256];
  Factors f;
  float mc;
  bool strange;
};
template <typename T, bool ENT, bool RANK, bool TOP, bool BWD>
__global__ void __launch_bounds__(Crew<8>::kThreads + (TOP ? 32 : 0), Crew<8>::kBlocks) logprob_stream(LogprobP p, RingPlan plan) {
  constexpr int W = 8, E = TOP ? 2 : 1, N = 2 * E;   // warps beside the streaming ones, rows in hand
  typedef Crew<W> Team;
  typedef Stream<T, W, BWD> Str;
  constexpr int U = Str::U, V = Vec<T>::V;
  constexpr uint32_t NS = Str::NS;
  typedef Scan<(int)NS, T, ENT, RANK, TOP, U> S;
  extern __shared__ __align__(16) uint4 ring[];   // batches of vectors, then what the top classes need
  __shared__ LogprobSlot<T, W> slot[N];
  __shared__ Key red[W];
  __shared__ Part whole[2];
  __shared__ uint16_t works[E][TOP ? kWork : 1];
  grid_dependency();
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = BWD ? cluster.num_blocks() : 1, part = BWD ? cluster.block_rank() : 0, row0 = blockIdx.x / parts, stride = gridDim.x / parts;
  const uint32_t rows = (uint32_t)p.x.rows;
  const uint32_t shift = slot_shift<T>(p.x.C), slots = (p.x.C / V + (Str::kBatch << shift) - 1) / (Str::kBatch << shift);
  uint16_t* maxima = (uint16_t*)((uint8_t*)ring + plan.bytes);   // [N][slots][256]
  const uint32_t C = p.x.C, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float nothing = as_nothing(p.cs);
  if (warp < W) {
    Str stream((const T*)p.logits, p.x, ring, plan.slots, plan.twice != 0, row0, stride, part, parts);
    uint32_t i = 0;
    for (uint32_t r = row0; r < rows; r += stride, ++i) {
      LogprobSlot<T, W>& q = slot[i % N];
      const T* x = (const T*)p.logits + p.x.offset(r);
      const Strip<T> b(x, C, part, parts);
      Team::wait(kBarReady + (i % N));
      const uint32_t lv = q.label.lv;
      const float xl = q.label.xl, thr0 = q.label.thr0;
      S scan;
      scan.clear();
      uint16_t* mine = maxima + (i % N) * slots * 256 + tid;
      float most = -INFINITY;
      auto sums = [&](uint32_t v0, const uint4 (&w)[U], bool full) {
        const float bm = scan.batch(b.vb + v0, w, full, b, tid, p.cs, nothing, lv, xl, thr0);
        if (TOP) {   // the slot's maximum so far
          const uint32_t n = v0 / Str::kBatch;
          most = (n & ((1u << shift) - 1)) ? fmaxf(most, bm) : bm;
          mine[(n >> shift) * 256] = (uint16_t)(__float_as_uint(most + 0.f) >> 16);
        }
      };
      const uint32_t nv = b.ve - b.vb;
      if (BWD && !plan.twice) stream.look(nv, sums);
      else stream.run(nv, sums);
      if (TOP) q.sv[tid] = tid < nv ? value_key(scan.a.m) : 0u;
      scan.a.template join<ENT, 32>(p.cs);
      if (lane == 0) q.parts[warp] = scan.a;
      Team::arrive(kBarSums + (i % N));
      if constexpr (BWD) {
        __syncwarp();
        if (parts > 1) cluster.sync();
        Team::wait(kBarResult + (i & 1));
        T* o = (T*)p.dlogits + p.g.offset(r);
        const bool even = (((uintptr_t)o ^ (uintptr_t)x) & 15u) == 0, plain = q.strange;
        const float c0 = q.f.c0, c1 = q.f.c1, mc = q.mc;
        // the thread that has the label's vector writes its class once more
        const uint32_t l = q.label.l < C && q.label.l >= b.head && lv >= b.vb && lv < b.ve && (lv - b.vb) % NS == tid ? lv - b.vb : kNoClass;
        float gl = 0.f;
        if (l != kNoClass) gl = q.f.template grad<ENT>(xl, p.cs, mc) + q.f.dl + (p.accumulate ? ld_f(o + q.label.l) : 0.f);
        T* to = o + b.class_of(b.vb) + tid * V;   // this thread's vector of the batch
        stream.run(nv, [&](uint32_t v0, const uint4 (&w)[U], bool full) {
          if (!plain) {
            if (full && even && !p.accumulate) {
#pragma unroll
              for (int u = 0; u < U; ++u) {
                float h[V];
                grad_vector<ENT, T>(w[u], h, p.cs, mc, c0, c1, nothing);
                __stcs((uint4*)(to + u * NS * V), Vec<T>::pack(h));
              }
            } else {
#pragma unroll
              for (int u = 0; u < U; ++u) {
                if (v0 + u * NS + tid >= nv) break;
                float h[V];
                grad_vector<ENT, T>(w[u], h, p.cs, mc, c0, c1, nothing);
                put_vector<T>(to + u * NS * V, even, p.accumulate, h);
              }
            }
            if (l - v0 < Str::kBatch) st_f(o + q.label.l, gl);
          }
          to += Str::kBatch * V;
        });
        if (plain && part == 0) {
          Group<(int)NS> g(red);
          const TopMem none = {};
          plain_row<(int)NS, T, true>(g, p, r, none);
        }
        if (r + 2 * stride < rows) Team::arrive(kBarFree + (i & 1));   // there is a row to come in this slot
      }
    }
  } else {
    TopMem t = {nullptr, nullptr, TopMem::room(p.top)};
    const uint32_t who = warp - W;   // rows who, who + E, ...
    t.list = (Key*)(maxima + (TOP ? N * slots * 256 : 0)) + who * (p.top + t.cap);
    t.cand = t.list + p.top;
    struct Row {   // what this warp keeps of a row between its two turns
      uint32_t cls;
      float single, old;
      Factors f;
      Part sum;   // of the row's single elements
    };
    const uint32_t first = row0 + who * stride, step = E * stride;
    uint32_t coming = p.label && first < rows ? p.label[first] : kNoClass;   // the label of the row to be prepared next
    auto prepare = [&](uint32_t r, uint32_t i) {
      Row w = {kNoClass, 0.f, 0.f, {}, {}};
      w.sum.clear();
      if (r >= rows) return w;
      if (BWD && i >= 2) Team::wait(kBarFree + (i & 1));
      LogprobSlot<T, W>& q = slot[i % N];
      const T* x = (const T*)p.logits + p.x.offset(r);
      const Strip<T> b(x, C, part, parts);
      Label<T> label;
      label.fetch(p, coming, x, b, 0);
      coming = p.label && r + step < rows ? p.label[r + step] : kNoClass;
      w.cls = lane < 2 * V ? b.single(lane) : kNoClass;
      if (w.cls != kNoClass) {
        w.single = ld_f(x + w.cls);
        if (BWD && p.accumulate) w.old = ld_f((const T*)p.dlogits + p.g.offset(r) + w.cls);
      }
      if (w.cls != kNoClass) w.sum.add<ENT>(w.single, p.cs);
      if (RANK) w.sum.cnt = label.own_vector(b, x, C, lane) + (w.cls != kNoClass && label.single_counts(w.single, w.cls));
      w.sum.join<ENT, 32>(p.cs);
      if (BWD) w.f.fetch(p, r, label.l);
      if (lane == 0) q.label = label;
      __syncwarp();
      Team::arrive(kBarReady + (i % N));
      return w;
    };
    uint32_t i = who;
    Row now = prepare(first, i);
    for (uint32_t r = first; r < rows; r += step, i += E) {
      const Row next = prepare(r + step, i + E);
      LogprobSlot<T, W>& q = slot[i % N];
      const T* x = (const T*)p.logits + p.x.offset(r);
      const Strip<T> b(x, C, part, parts);
      const Label<T> label = q.label;
      Team::wait(kBarSums + (i % N));
      Part a;
      a.clear();
      if (lane % 16 < W) a = q.parts[lane % 16];
      else if (lane % 16 == W) a = now.sum;
      a.join<ENT, 16>(p.cs);
      if (parts > 1) {
        if (lane == 0) whole[i & 1] = a;
        __syncwarp();
        cluster.sync();
        a.clear();
        if (lane % 8 < parts) a = *cluster.map_shared_rank(&whole[i & 1], lane % 8);
        a.join<ENT, 8>(p.cs);
      }
      const bool far = TOP && a.far(p.cs), strange = !far && a.strange(p.cs);
      RowSums s;
      if (far) {   // list and rank stand
        Group<32> g(nullptr);
        plain_sums<32, T, ENT>(g, x, 1, p.x.C, p.cs, s, a.E);
      } else {
        s.set(a.m, a.mc, a.S, p.cs);
      }
      const float H = s.entropy(a.E);
      if constexpr (BWD) {
        Factors f = now.f;
        f.set<ENT>(p, s, H);
        if (lane == 0) {
          q.f = f;
          q.mc = s.mc;
          q.strange = strange;
        }
        Team::arrive(kBarResult + (i & 1));
        if (!strange && now.cls != kNoClass)
          st_f((T*)p.dlogits + p.g.offset(r) + now.cls, f.grad<ENT>(now.single, p.cs, s.mc) + (now.cls == label.l ? f.dl : 0.f) + now.old);
      }
      if (strange) {
        Group<32> g(nullptr);
        if (!BWD) plain_row<32, T, false>(g, p, r, t);
      } else {
        if (lane == 0 && part == 0) {
          put_row(p, s, r, H, label.l, label.xl);
          if (RANK) p.rank[r] = label.rank(a.cnt, C);
        }
        if constexpr (TOP) {
          uint32_t kv[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) kv[j] = q.sv[j * 32 + lane];
          const Maxima mx = {maxima + (i % N) * slots * 256, shift, slots};
          select_top<T>(t, p.top, kv, mx, b, x, (const uint4*)(x + b.head), now.cls, now.single, works[who]);
          for (uint32_t j = lane; j < p.top; j += 32) put_top(p, s, r, j, t.list[j]);
          __syncwarp();
        }
      }
      now = next;
    }
  }
  __syncwarp();
  if (parts > 1) cluster.sync();   // nobody leaves while its sums are still read
}

static int logprob_args(const ad_logprob_args* a, bool bwd, LogprobP& p) {
  if (!a) return AD_ERR_BAD_ARG;
  p = {};
  int rc = rows_of(a->dtype, a->layout, a->N, a->C, a->HW, a->pitch, p.x);
  if (rc != AD_OK || p.x.rows == 0) return rc;
  if (!a->logits || !scale_ok(a->scale)) return AD_ERR_BAD_ARG;
  const size_t elem = (size_t)elem_size(a->dtype);
  if (!aligned_to(a->logits, elem) || !words(a->label, a->lse, a->entropy, a->logp)) return AD_ERR_ALIGN;
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
    if (!aligned_to(a->dlogits, elem) || !words(a->dlse, a->dentropy, a->dlogp)) return AD_ERR_ALIGN;
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
    if (!words(a->rank) || (a->top && !words(a->top_class, a->top_logp))) return AD_ERR_ALIGN;
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
  const size_t bytes = (size_t)p.x.C * sizeof(T), list = p.top + TopMem::room(p.top);
  // the limits belong to the functions: the most that they take
  if constexpr (NT != 32) {
    constexpr int W = 8;
    const uint32_t shift = slot_shift<T>(p.x.C), slots = (p.x.C / Vec<T>::V + (1024u << shift) - 1) / (1024u << shift);
    const size_t besides = TOP ? 2 * list * sizeof(Key) + 4 * slots * 256 * 2 : 0;
    const RingPlan plan = ring_plan<T, W, BWD>(p.x.C, [&](uint32_t) { return besides; });
    if (stream_worth<W>(p.x.rows, plan.parts)) {
      static StreamLaunch shared;
      const int rc = launch_stream(logprob_stream<T, ENT, RANK, TOP, BWD>, shared, Crew<W>::kThreads + (TOP ? 32 : 0), p.x.rows, plan.parts, plan.bytes + besides, s, p, plan);
      if (rc != AD_ERR_UNSUPPORTED) return rc;
    }
  }
  auto kernel = logprob_rows<NT, T, ENT, RANK, TOP, BWD>;
  const uint32_t n = NT == 32 ? 1 : row_parts(p.x.rows, bytes), slots = NT == 32 ? 0 : feed_slots(bytes, n, BWD || TOP ? kMostFeed : 0);
  const size_t keys = TOP ? (NT == 32 ? kRowWarps * list : list + (n > 1 ? n * p.top : 0)) : 0;
  const size_t smem = slots * Feed<NT>::kBatch * 16 + keys * sizeof(Key);
  constexpr int most = (int)(NT == 32 ? sizeof(Key) * kRowWarps * (kMostTop + TopMem::room(kMostTop)) : kMostFeed + sizeof(Key) * (9 * kMostTop + TopMem::room(kMostTop)));
  if (smem > 40 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch_row_kernel(kernel, p, slots, NT == 32 ? (p.x.rows + kRowWarps - 1) / kRowWarps : p.x.rows, n, smem, s);
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

template <typename T, bool BWD>
static int launch_logprob(const LogprobP& p, cudaStream_t s) {
  int rc = BWD ? logprob_positions_bwd<T>(p, s) : logprob_positions<T>(p, s);
  if (rc != AD_ERR_UNSUPPORTED) {   // a thread per position
  } else if (p.x.step != 1 || (BWD && p.g.step != 1)) rc = launch_any<T, BWD>(p, s);
  else if (by_warp(p.x.rows, p.x.C * sizeof(T), BWD)) rc = BWD ? launch_bwd<32, T>(p, s) : launch_fwd<32, T>(p, s);
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
