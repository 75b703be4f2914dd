// Distillation from a teacher's top classes, the loss and its gradient: rows of neighbouring classes.
//
// Bytes of the logits, read once (backward: once more out of shared memory or the L2, and the gradient written).  The
// gradient of a class outside of the list is dloss * scale * p_c * (Q - q_r / p_r), which is written everywhere; the list's
// logits are read before, and their gradients written over that.  With rest the pass over the row leaves the list's classes
// out (a byte of mask per vector in shared memory) and sums the others alone, against their own maximum: p_r is then exact
// however little of the row it is, and the row's sum is theirs and that of the list, each class of it once.
//
// 4096 x 65536 bf16 (537 MB, 83 us at the copy rate): loss with the rest 89 to 109 us for lists of 1 to 128 classes.  Gradient (166):
// 221 with one class, 235 to 240 with 64 and the rest; 1001 x 50001 fp32 (62): 96; 2048 x 32000 bf16 (41) with 16 classes: 64, with
// the rest 72.  Two exponentials per element (119 us of the special units for the first) and the second pass's way through
// shared memory beside the copies.
#include <cooperative_groups.h>

#include "distill.cuh"

namespace cg = cooperative_groups;

namespace adk {

constexpr size_t kMostMask = 120 * 1024;   // bytes of mask in shared memory

// A row's list in shared memory
struct __align__(16) List {
  uint32_t cls[kMostTop];
  float a[kMostTop], x[kMostTop];   // log2 q, later q, and the student's logit
  uint8_t first[kMostTop];          // no earlier entry has the class
  bool twice;                       // some class stands twice
};

// One warp: the teacher's weights, the list's share of the row, and the loss
__device__ __forceinline__ Distilled distill_row(const DistillP& p, size_t r, List& list, float m, float off, float R, float& loss) {
  const uint32_t lane = threadIdx.x & 31, k = p.top, C = p.x.C;
  float a[4], x[4], am = -INFINITY;
  bool in[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t j = lane + 32 * i;
    in[i] = j < k && list.cls[j] < C;
    a[i] = in[i] ? list.a[j] : -INFINITY;
    x[i] = in[i] ? list.x[j] : 0.f;
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
  }
  Q = warp_sum(Q);
  float mk = -INFINITY, K = 0.f;
  if (p.rest) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in[i]) mk = fmaxf(mk, x[i]);
    mk = warp_max(mk);
    if (mk == -INFINITY) mk = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (in[i] && list.first[lane + 32 * i]) K += exp2_fast((x[i] - mk) * p.cs);   // a class that stands twice has its weight once
    K = warp_sum(K);
  }
  float rest_loss;
  const Distilled d = row_sums(p, m, off, R, mk, K, Q, rest_loss);
  loss = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    loss += d.term(q[i], a[i], x[i], p.scale);
    if (lane + 32 * i < k) list.a[lane + 32 * i] = q[i];   // for the gradient
  }
  loss = warp_sum(loss) + rest_loss;
  loss = d.some ? loss + 0.f * d.L : 0.f;   // NaN without any entry, too
  return d;
}
// The gradient of entry j's class; q: the entries' weights
__device__ __forceinline__ float listed_grad(const DistillP& p, const Distilled& d, const List& list, const float* q, uint32_t j, float f) {
  const uint32_t c = list.cls[j];
  float sum = q[j];
  if (list.twice) {
    sum = 0.f;
    for (uint32_t i = 0; i < p.top; ++i) sum += list.cls[i] == c ? q[i] : 0.f;
  }
  return d.some ? f * (exp2_fast((list.x[j] - d.mt) * p.cs) * d.rS * d.Q - sum) : 0.f;
}

// Any layout, any numbers: plain loops of a group over one row, whose list is in place
template <int NT, typename T, bool BWD>
__device__ void plain_row(Group<NT>& g, const DistillP& p, size_t r, List& list, Distilled* shared) {
  const T* x = (const T*)p.logits + p.x.offset(r);
  const int64_t st = p.x.step;
  const uint32_t C = p.x.C, k = p.top;
  auto outside = [&](uint32_t c) {
    bool in = false;
    if (p.rest)
      for (uint32_t j = 0; j < k; ++j) in |= list.cls[j] == c;
    return !in;
  };
  float m = -INFINITY, R = 0.f;
  for (uint32_t c = g.tid; c < C; c += NT)
    if (outside(c)) m = fmaxf(m, ld_f(x + c * st));
  m = g.max(m);
  if (m == -INFINITY) m = 0.f;
  for (uint32_t c = g.tid; c < C; c += NT)
    if (outside(c)) R += exp2_fast((ld_f(x + c * st) - m) * p.cs);
  R = g.sum(R);
  if (threadIdx.x % NT < 32) {
    float loss;
    const Distilled d = distill_row(p, r, list, m, 0.f, R, loss);
    if (g.tid == 0) {
      *shared = d;
      if (p.loss) p.loss[r] = loss;
    }
  }
  g.sync();
  if constexpr (BWD) {
    const Distilled d = *shared;
    T* o = (T*)p.dlogits + p.g.offset(r);
    const float f = p.dloss[r] * p.scale;
    float old[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t j = g.tid + i * NT;
      old[i] = p.accumulate && j < k && list.cls[j] < C ? ld_f(o + list.cls[j] * p.g.step) : 0.f;
    }
    g.sync();
    for (uint32_t c = g.tid; c < C; c += NT) {
      float v = f * (exp2_fast((ld_f(x + c * st) - m) * p.cs) * d.out);
      if (p.accumulate) v += ld_f(o + c * p.g.step);
      st_f(o + c * p.g.step, v);
    }
    g.sync();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t j = g.tid + i * NT;
      if (j < k && list.cls[j] < C) {
        const float v = listed_grad(p, d, list, list.a, j, f);
        st_f(o + list.cls[j] * p.g.step, p.accumulate ? old[i] + v : v);
      }
    }
  }
  g.sync();
}

// A row's list into shared memory, entry j by the group's thread j.  Synchronises the group.
template <int NT, typename T>
__device__ __forceinline__ void fetch_list(Group<NT>& g, const DistillP& p, size_t r, const T* x, int64_t st, List& list) {
  if (g.tid == 0) list.twice = false;
  for (uint32_t j = g.tid; j < kMostTop; j += NT) {
    const uint32_t c = j < p.top ? p.top_class[r * p.top + j] : kNoClass;
    list.cls[j] = c;
    if (j < p.top) {
      list.a[j] = p.top_logit[r * p.top + j] * p.ts;
      list.x[j] = c < p.x.C ? ld_f(x + c * st) : 0.f;
    }
  }
  g.sync();
  for (uint32_t j = g.tid; j < p.top; j += NT) {
    const uint32_t c = list.cls[j];
    uint32_t before = 0, all = 0;
    for (uint32_t i = 0; i < p.top; i += 8) {
      const uint4 lo = *(const uint4*)&list.cls[i], hi = *(const uint4*)&list.cls[i + 4];
      const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (uint32_t q = 0; q < 8; ++q) {
        all += v[q] == c;
        before += v[q] == c && i + q < j;
      }
    }
    list.first[j] = before == 0;
    if (all > 1 && c < p.x.C) list.twice = true;
  }
  g.sync();
}

template <typename T, bool BWD>
__global__ void __launch_bounds__(256) distill_any(DistillP p) {
  grid_dependency();
  __shared__ List lists[8];
  __shared__ Distilled shared[8];
  Group<32> g(nullptr);
  const uint32_t w = threadIdx.x >> 5;
  const size_t warp = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5, nw = ((size_t)gridDim.x * blockDim.x) >> 5;
  for (size_t r = warp; r < p.x.rows; r += nw) {
    fetch_list<32, T>(g, p, r, (const T*)p.logits + p.x.offset(r), p.x.step, lists[w]);
    plain_row<32, T, BWD>(g, p, r, lists[w], &shared[w]);
  }
}

// The elements of a vector whose bits are set become -inf
template <typename T>
__device__ __forceinline__ void leave_out(uint4& w, uint32_t bits) {
  constexpr int V = Vec<T>::V;
  uint32_t* q = &w.x;
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (bits >> i & 1) {
      if (V == 4) q[i] = 0xff800000u;
      else q[i / 2] = i & 1 ? (q[i / 2] & 0xffffu) | 0xff800000u : (q[i / 2] & 0xffff0000u) | 0xff80u;
    }
}

// ---------------------------------------------------------------- rows of many neighbouring classes
// NT 32: a warp per row, eight vectors per lane and batch.  NT 256: a block per row, or a cluster of blocks, four vectors.
// REST: the classes of the list are left out of the pass.
template <int NT, typename T, bool REST, bool BWD>
__global__ void __launch_bounds__(256) distill_rows(DistillP p, uint32_t slots) {
  constexpr int U = Feed<NT>::U, V = Vec<T>::V;
  typedef Vec<T> X;
  extern __shared__ __align__(16) uint8_t dyn[];   // batches of vectors, then a byte per vector of the row's share (NT 32: of each warp's row)
  __shared__ Key red[kRowWarps];
  __shared__ Part parts[kRowWarps], whole;
  __shared__ List lists[NT == 32 ? kRowWarps : 1];
  __shared__ Distilled shared[NT == 32 ? kRowWarps : 1];
  grid_dependency();
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts_n = NT == 32 ? 1 : cluster.num_blocks(), part = NT == 32 ? 0 : cluster.block_rank();
  Group<NT> g(red);
  const uint32_t C = p.x.C, warp = threadIdx.x >> 5, k = p.top;
  List& list = lists[NT == 32 ? warp : 0];
  uint8_t* mask = dyn + (size_t)slots * Feed<NT>::kBatch * 16 + (NT == 32 ? (size_t)warp * ((C / V + 15) / 16 * 16) : 0);
  const size_t row0 = NT == 32 ? (size_t)blockIdx.x * kRowWarps + warp : blockIdx.x / parts_n;
  const size_t rows_n = NT == 32 ? (size_t)gridDim.x * kRowWarps : gridDim.x / parts_n;
  for (size_t r = row0; r < p.x.rows; r += rows_n) {
    const T* x = (const T*)p.logits + p.x.offset(r);
    const Strip<T> b(x, C, part, parts_n);
    const uint4* xv = (const uint4*)(x + b.head);
    if (REST)
      for (uint32_t i = g.tid; i < (b.ve - b.vb + 15) / 16; i += NT) ((uint4*)mask)[i] = make_uint4(0, 0, 0, 0);
    fetch_list<NT, T>(g, p, r, x, 1, list);
    bool apart = true;   // this thread's single element is outside of the list
    const uint32_t sc = g.tid < 2 * V ? b.single(g.tid) : kNoClass;
    if (REST) {
      for (uint32_t j = g.tid; j < k; j += NT) {
        const uint32_t c = list.cls[j], v = (c - b.head) / V;
        if (c < C && c >= b.head && v >= b.vb && v < b.ve) {
          const uint32_t at = v - b.vb;
          atomicOr((uint32_t*)mask + at / 4, 1u << (at % 4 * 8 + (c - b.head) % V));
        }
      }
      if (sc != kNoClass)
        for (uint32_t j = 0; j < k; ++j) apart &= list.cls[j] != sc;
      g.sync();
    }
    Part a;
    a.clear();
    if (sc != kNoClass && apart) a.add<false>(ld_f(x + sc), p.cs);
    Feed<NT> feed(xv, b.vb, b.ve, g.tid, slots, (uint4*)dyn);
    feed.template start<T>();
    feed.template run<T, false>([&](uint32_t v0, uint4 (&w)[U]) {
      typename X::Max most;
      if (REST) {
        uint32_t out[U], any = 0;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t v = v0 + u * NT + g.tid;
          out[u] = v < b.ve ? mask[v - b.vb] : 0;
          any |= out[u];
        }
        if (any) {
#pragma unroll
          for (int u = 0; u < U; ++u) leave_out<T>(w[u], out[u]);
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) most = u ? X::max(most, X::max(w[u])) : X::max(w[u]);
      add_vectors<false, U, T>(a, w, (int)((b.ve - v0 + NT - 1) / NT), X::value(most), p.cs, 0.f);
    });
    a.join<false, 32>(p.cs);
    if (NT != 32) {
      if ((g.tid & 31) == 0) parts[warp] = a;
      __syncthreads();
      a = parts[g.tid % kRowWarps];
      a.join<false, kRowWarps>(p.cs);
      if (parts_n > 1) {
        if (g.tid == 0) whole = a;
        cluster.sync();
        const uint32_t q = g.tid % 8;
        if (q < parts_n) a = *cluster.map_shared_rank(&whole, q);
        else a.clear();
        a.join<false, 8>(p.cs);
      }
    }
    if (a.strange(p.cs)) {
      if (part == 0) plain_row<NT, T, BWD>(g, p, r, list, shared + (NT == 32 ? warp : 0));
      if (parts_n > 1) cluster.sync();
      else g.sync();
      continue;
    }
    const float off = a.m == -INFINITY ? 0.f : fmaf(-a.m, p.cs, a.mc);
    Distilled d;
    if (NT == 32 || warp == 0) {
      float loss;
      d = distill_row(p, r, list, a.m, off, a.S, loss);
      if (g.tid == 0 && part == 0 && p.loss) p.loss[r] = loss;
      if (NT != 32 && BWD && g.tid == 0) shared[0] = d;
    }
    g.sync();
    if constexpr (BWD) {
      if (NT != 32) d = shared[0];
      T* o = (T*)p.dlogits + p.g.offset(r);
      const bool even = (((uintptr_t)o ^ (uintptr_t)x) & 15u) == 0;   // both have their vectors at the same classes
      const float f = p.dloss[r] * p.scale, coef = f * d.out, mc = a.mc;
      auto grad = [&](float v) { return coef * exp2_fast(fmaf(v, p.cs, -mc)); };
      float gl[NT == 32 ? 4 : 1];   // the list's gradients, written last
#pragma unroll
      for (int i = 0; i < (NT == 32 ? 4 : 1); ++i) {
        const uint32_t j = g.tid + i * NT;
        if (j < k && list.cls[j] >= b.begin() && list.cls[j] < b.end()) gl[i] = listed_grad(p, d, list, list.a, j, f) + (p.accumulate ? ld_f(o + list.cls[j]) : 0.f);
      }
      if (p.accumulate) g.sync();
      if (sc != kNoClass) st_f(o + sc, grad(ld_f(x + sc)) + (p.accumulate ? ld_f(o + sc) : 0.f));
      feed.template run<T, true>([&](uint32_t v0, const uint4 (&w)[U]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t v = v0 + u * NT + g.tid;
          if (v >= b.ve) break;
          float h[V];
          grad_vector<false, T>(w[u], h, p.cs, mc, coef, 0.f, 0.f);
          put_vector<T>(o + b.class_of(v), even, p.accumulate, h);
        }
      });
      g.sync();
#pragma unroll
      for (int i = 0; i < (NT == 32 ? 4 : 1); ++i) {
        const uint32_t j = g.tid + i * NT;
        if (j < k && list.cls[j] >= b.begin() && list.cls[j] < b.end()) st_f(o + list.cls[j], gl[i]);
      }
    }
    if (parts_n > 1) cluster.sync();   // what the others read of this block's
    else g.sync();
  }
}

// Many rows of many classes: see Stream.  Two rows are in hand, by parity.
template <int W>
struct __align__(16) DistillSlot {
  List list;
  float q[kMostTop], old[kMostTop], grad[kMostTop];   // an entry's weight, what the gradient of its class is added to, and that gradient
  Part parts[W];
  float mc, coef;
  uint32_t singles;                      // which of the row's single elements are listed
  bool strange;
};
template <typename T, bool REST, bool BWD>
__global__ void __launch_bounds__(Crew<8>::kThreads, Crew<8>::kBlocks) distill_stream(DistillP p, RingPlan plan, uint32_t mask_bytes) {
  constexpr int W = 8;
  typedef Crew<W> Team;
  typedef Stream<T, W, BWD> Str;
  constexpr int U = Str::U, V = Vec<T>::V;
  constexpr uint32_t NS = Str::NS;
  typedef Vec<T> X;
  extern __shared__ __align__(16) uint8_t dyn[];   // batches of vectors, then two masks: a byte per vector
  __shared__ DistillSlot<W> slot[2];
  __shared__ Key red[W];
  __shared__ Part whole[2];
  __shared__ Distilled shared;
  grid_dependency();
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = BWD ? cluster.num_blocks() : 1, part = BWD ? cluster.block_rank() : 0, row0 = blockIdx.x / parts, stride = gridDim.x / parts;
  const uint32_t rows = (uint32_t)p.x.rows;
  const uint32_t C = p.x.C, k = p.top, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint8_t* masks = dyn + plan.bytes;
  if (warp < W) {
    Str stream((const T*)p.logits, p.x, dyn, plan.slots, plan.twice != 0, row0, stride, part, parts);
    uint32_t i = 0;
    for (uint32_t r = row0; r < rows; r += stride, ++i) {
      DistillSlot<W>& q = slot[i & 1];
      const T* x = (const T*)p.logits + p.x.offset(r);
      const Strip<T> b(x, C, part, parts);
      const uint32_t nv = b.ve - b.vb;
      const uint8_t* mask = masks + (i & 1) * mask_bytes + tid;
      Team::wait(kBarReady + (i & 1));
      Part a;
      a.clear();
      auto sums = [&](uint32_t v0, uint4 (&w)[U], bool full) {
        if (REST) {
          uint32_t out[U], any = 0;
#pragma unroll
          for (int u = 0; u < U; ++u) {
            out[u] = full || v0 + u * NS + tid < nv ? mask[v0 + u * NS] : 0;
            any |= out[u];
          }
          if (any) {
#pragma unroll
            for (int u = 0; u < U; ++u) leave_out<T>(w[u], out[u]);
          }
        }
        typename X::Max most = X::max(w[0]);
#pragma unroll
        for (int u = 1; u < U; ++u) most = X::max(most, X::max(w[u]));
        add_vectors<false, U, T>(a, w, full ? U : (int)((nv - v0 + NS - 1) / NS), X::value(most), p.cs, 0.f);
      };
      if (BWD && !plan.twice) stream.look(nv, sums);
      else stream.run(nv, sums);
      a.join<false, 32>(p.cs);
      if (lane == 0) q.parts[warp] = a;
      Team::arrive(kBarSums + (i & 1));
      if constexpr (BWD) {
        __syncwarp();
        if (parts > 1) cluster.sync();
        Team::wait(kBarResult + (i & 1));
        T* o = (T*)p.dlogits + p.g.offset(r);
        const bool even = (((uintptr_t)o ^ (uintptr_t)x) & 15u) == 0, plain = q.strange;
        const float mc = q.mc, coef = q.coef;
        T* to = o + b.class_of(b.vb) + tid * V;   // this thread's vector of the batch
        stream.run(nv, [&](uint32_t v0, uint4 (&w)[U], bool full) {
          if (!plain) {
            if (full && even && !p.accumulate) {
#pragma unroll
              for (int u = 0; u < U; ++u) {
                float h[V];
                grad_vector<false, T>(w[u], h, p.cs, mc, coef, 0.f, 0.f);
                __stcs((uint4*)(to + u * NS * V), X::pack(h));
              }
            } else {
#pragma unroll
              for (int u = 0; u < U; ++u) {
                if (v0 + u * NS + tid >= nv) break;
                float h[V];
                grad_vector<false, T>(w[u], h, p.cs, mc, coef, 0.f, 0.f);
                put_vector<T>(to + u * NS * V, even, p.accumulate, h);
              }
            }
          }
          to += Str::kBatch * V;
        });
        Group<(int)NS> g(red);
        if (plain) {
          if (part == 0) plain_row<(int)NS, T, true>(g, p, r, q.list, &shared);
        } else {
          g.sync();   // the list's classes over what the loop wrote
          if (tid < k && q.list.cls[tid] >= b.begin() && q.list.cls[tid] < b.end()) st_f(o + q.list.cls[tid], q.grad[tid]);
        }
        if (r + 2 * stride < rows) Team::arrive(kBarFree + (i & 1));   // there is a row to come in this slot
      }
    }
  } else {
    struct Row {   // what this warp keeps of a row between its two turns
      uint32_t cls;
      float single, old, Q, mk, K, dloss;
      Part sum;   // of the row's single elements that are not listed
    };
    auto prepare = [&](uint32_t r, uint32_t i) {
      Row w = {kNoClass, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, {}};
      w.sum.clear();
      if (r >= rows) return w;
      if (BWD && i >= 2) Team::wait(kBarFree + (i & 1));
      DistillSlot<W>& q = slot[i & 1];
      uint8_t* mask = masks + (i & 1) * mask_bytes;
      const T* x = (const T*)p.logits + p.x.offset(r);
      const T* o = (const T*)p.dlogits + (BWD ? p.g.offset(r) : 0);
      const Strip<T> b(x, C, part, parts);
      uint32_t cls[4];
      float a[4], xs[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t j = lane + 32 * e;
        cls[e] = j < k ? p.top_class[r * k + j] : kNoClass;
        a[e] = j < k ? p.top_logit[r * k + j] * p.ts : 0.f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t j = lane + 32 * e;
        const bool in = cls[e] < C;
        xs[e] = in ? ld_f(x + cls[e]) : 0.f;
        if (!in) a[e] = -INFINITY;
        if (BWD && p.accumulate) q.old[j] = in ? ld_f(o + cls[e]) : 0.f;
        q.list.cls[j] = cls[e];
        q.list.x[j] = xs[e];
      }
      w.cls = lane < 2 * V ? b.single(lane) : kNoClass;
      if (w.cls != kNoClass) {
        w.single = ld_f(x + w.cls);
        if (BWD && p.accumulate) w.old = ld_f(o + w.cls);
      }
      if (BWD) w.dloss = p.dloss[r];
      float shift = 0.f;
      if (p.rest) {
        if (p.top_lse) shift = (float)(p.top_lse[r] * kLog2e);
      } else {
        float am = warp_max(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
        if (am == -INFINITY) am = 0.f;
        const float z = warp_sum((exp2f(a[0] - am) + exp2f(a[1] - am)) + (exp2f(a[2] - am) + exp2f(a[3] - am)));
        shift = z != 0.f ? am + log2f(z) : 0.f;
      }
      // which classes are listed, and whether one of them stands twice
      bool twice = false, apart = true;
      if (REST) {
        for (uint32_t v = lane; v < (b.ve - b.vb + 15) / 16; v += 32) ((uint4*)mask)[v] = make_uint4(0, 0, 0, 0);
        if (lane == 0) q.singles = 0;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t c = cls[e];
          if (c >= C) continue;
          const uint32_t v = (c - b.head) / V;
          if (c >= b.head && v < b.nv) {
            if (v >= b.vb && v < b.ve) {   // this block's part
              const uint32_t at = v - b.vb, bit = 1u << (at % 4 * 8 + (c - b.head) % V);
              twice |= (atomicOr((uint32_t*)mask + at / 4, bit) & bit) != 0;
            }
          } else {
            const uint32_t bit = 1u << (c < b.head ? c : V + (c - b.head - b.nv * V));
            twice |= (atomicOr(&q.singles, bit) & bit) != 0;
          }
        }
        if (parts > 1) twice = true;   // the other parts are not known: looked for below
        twice = __any_sync(0xffffffffu, twice);
        __syncwarp();
        apart = !(q.singles >> lane & 1u);
      }
      if (BWD && !REST) twice = true;   // looked for below
      bool first[4] = {true, true, true, true};
      if (twice) {
        __syncwarp();
        uint32_t more = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (32 * e >= (int)k) break;
          uint32_t before = 0, all = 0;
          for (uint32_t f = 0; f < k; f += 4) {
            const uint4 c = *(const uint4*)&q.list.cls[f];
            const uint32_t j = lane + 32 * e;
            all += (c.x == cls[e]) + (c.y == cls[e]) + (c.z == cls[e]) + (c.w == cls[e]);
            before += (c.x == cls[e] && f < j) + (c.y == cls[e] && f + 1 < j) + (c.z == cls[e] && f + 2 < j) + (c.w == cls[e] && f + 3 < j);
          }
          first[e] = before == 0;
          more += cls[e] < C && all > 1;
        }
        twice = __any_sync(0xffffffffu, more != 0);
      }
      if (REST) {
        float mk = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) mk = cls[e] < C ? fmaxf(mk, xs[e]) : mk;
        mk = warp_max(mk);
        w.mk = mk == -INFINITY ? 0.f : mk;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (cls[e] < C && first[e]) w.K += exp2_fast((xs[e] - w.mk) * p.cs);
        w.K = warp_sum(w.K);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (32 * e >= (int)k) break;
        a[e] -= shift;
        const float weight = exp2f(a[e]);
        q.list.a[lane + 32 * e] = a[e];
        q.q[lane + 32 * e] = weight;
        w.Q += weight;
      }
      w.Q = warp_sum(w.Q);
      if (w.cls != kNoClass && apart) w.sum.add<false>(w.single, p.cs);
      w.sum.join<false, 32>(p.cs);
      if (lane == 0) q.list.twice = twice;
      Team::arrive(kBarReady + (i & 1));
      return w;
    };
    uint32_t i = 0;
    Row now = prepare(row0, 0);
    for (uint32_t r = row0; r < rows; r += stride, ++i) {
      const Row next = prepare(r + stride, i + 1);
      DistillSlot<W>& q = slot[i & 1];
      Team::wait(kBarSums + (i & 1));
      Part a;
      a.clear();
      if (lane % 16 < W) a = q.parts[lane % 16];
      else if (lane % 16 == W) a = now.sum;
      a.join<false, 16>(p.cs);
      if (parts > 1) {
        if (lane == 0) whole[i & 1] = a;
        __syncwarp();
        cluster.sync();
        a.clear();
        if (lane % 8 < parts) a = *cluster.map_shared_rank(&whole[i & 1], lane % 8);
        a.join<false, 8>(p.cs);
      }
      const bool strange = a.strange(p.cs);
      const float off = a.m == -INFINITY ? 0.f : fmaf(-a.m, p.cs, a.mc);
      float loss;
      const Distilled d = row_sums(p, a.m, off, a.S, now.mk, now.K, now.Q, loss);
      const float f = now.dloss * p.scale;
      if (!strange) {
        if (BWD) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t j = lane + 32 * e;
            if (j < k) q.grad[j] = listed_grad(p, d, q.list, q.q, j, f) + (p.accumulate ? q.old[j] : 0.f);
          }
          if (lane == 0) {
            q.mc = a.mc;
            q.coef = f * d.out;
            q.strange = false;
          }
          // before the list's, which the streaming threads write behind this barrier
          if (now.cls != kNoClass) st_f((T*)p.dlogits + p.g.offset(r) + now.cls, f * d.out * exp2_fast(fmaf(now.single, p.cs, -a.mc)) + now.old);
          Team::arrive(kBarResult + (i & 1));
        }
        float terms = 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t j = lane + 32 * e;
          if (j < k) terms += d.term(q.q[j], q.list.a[j], q.list.x[j], p.scale);
        }
        loss += warp_sum(terms);
        if (lane == 0 && part == 0 && p.loss) p.loss[r] = d.some ? loss + 0.f * d.L : 0.f;
      } else {
        // the plain loops want the list as it is fetched
        Group<32> g(nullptr);
        __syncwarp();
        fetch_list<32, T>(g, p, r, (const T*)p.logits + p.x.offset(r), 1, q.list);
        if (BWD) {
          if (lane == 0) q.strange = true;
          Team::arrive(kBarResult + (i & 1));
        } else {
          plain_row<32, T, false>(g, p, r, q.list, &shared);
        }
      }
      now = next;
    }
  }
  __syncwarp();
  if (parts > 1) cluster.sync();   // nobody leaves while its sums are still read
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
  if (!aligned_to(a->logits, elem) || !words(a->top_class, a->top_logit, a->top_lse, a->loss)) return AD_ERR_ALIGN;
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
    if (!aligned_to(a->dlogits, elem) || !words(a->dloss)) return AD_ERR_ALIGN;
    if (!gradient_clear(p.x, a->logits, p.g, a->dlogits, elem, a->accumulate)) return AD_ERR_BAD_ARG;
    p.dlogits = a->dlogits;
    p.dloss = a->dloss;
    p.accumulate = a->accumulate != 0;
  } else if (!a->loss) {
    return AD_ERR_BAD_ARG;
  }
  return AD_OK;
}

template <int NT, typename T, bool REST, bool BWD>
static int launch_rows(const DistillP& p, uint32_t n, size_t mask, cudaStream_t s) {
  if constexpr (NT != 32) {
    constexpr int W = 8;
    auto bytes = [&](uint32_t parts) { return REST ? (p.x.C / Vec<T>::V / parts + 1 + 15) / 16 * 16 : (size_t)0; };   // of a mask
    const RingPlan plan = ring_plan<T, W, BWD>(p.x.C, [&](uint32_t parts) { return 2 * bytes(parts) < kMostMask ? 2 * bytes(parts) : kMostMask; });
    const size_t one = bytes(plan.parts);
    if (one <= kMostMask / 2 && stream_worth<W>(p.x.rows, plan.parts)) {
      static StreamLaunch shared;
      const int rc = launch_stream(distill_stream<T, REST, BWD>, shared, Crew<W>::kThreads, p.x.rows, plan.parts, plan.bytes + 2 * one, s, p, plan, (uint32_t)one);
      if (rc != AD_ERR_UNSUPPORTED) return rc;
    }
  }
  auto kernel = distill_rows<NT, T, REST, BWD>;
  const uint32_t slots = NT == 32 ? 0 : feed_slots((size_t)p.x.C * sizeof(T), n, BWD ? kMostFeed : 0);
  const size_t smem = slots * Feed<NT>::kBatch * 16 + mask;
  // the limit belongs to the function: the most that it takes
  if (smem > 32 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)(kMostFeed + kMostMask)) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch_row_kernel(kernel, p, slots, NT == 32 ? (p.x.rows + kRowWarps - 1) / kRowWarps : p.x.rows, n, smem, s);
  return AD_OK;
}

template <typename T, bool BWD>
static int launch_distill(const DistillP& p, cudaStream_t s) {
  const size_t vectors = p.x.C / Vec<T>::V;
  uint32_t n = row_parts(p.x.rows, (size_t)p.x.C * sizeof(T));
  auto mask_of = [&](uint32_t parts) { return p.rest ? (vectors / parts + 17) / 16 * 16 : (size_t)0; };
  // blocks enough to hold the row's mask: element by element 450 x 600001 fp32 took 23 ms and its gradient 32
  while (n < 8 && mask_of(n) > kMostMask) n *= 2;
  const size_t mask = mask_of(n);
  int rc = distill_positions<T, BWD>(p, s);
  if (rc != AD_ERR_UNSUPPORTED) {   // a thread per position
  } else if (p.x.step != 1 || (BWD && p.g.step != 1) || mask > kMostMask) {
    rc = AD_OK;
    launch(distill_any<T, BWD>, grid_for(p.x.rows, 8), 256, 0, s, p);
  } else if (by_warp(p.x.rows, p.x.C * sizeof(T), BWD)) {
    const size_t all = p.rest ? kRowWarps * ((vectors + 15) / 16 * 16) : 0;
    rc = p.rest ? launch_rows<32, T, true, BWD>(p, 1, all, s) : launch_rows<32, T, false, BWD>(p, 1, all, s);
  } else {
    rc = p.rest ? launch_rows<256, T, true, BWD>(p, n, mask, s) : launch_rows<256, T, false, BWD>(p, n, mask, s);
  }
  if (rc != AD_OK) return rc;
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
