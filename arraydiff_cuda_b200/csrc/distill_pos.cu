// Distillation with a thread per position: few classes in neighbouring elements, or classes in planes.
//
// Up to 32 classes and eight entries: the rows of 128 positions in shared memory, a thread's row and list in registers, the
// gradient back into the tile, where the entries' classes are written over it, and out by vectors; planes as they lie (1,048,576
// positions of 19 fp32 classes: 55 us, from memory class by class 97).  2,097,152 pixels of 19 bf16
// classes with four entries each (243 MB, 38 us at the copy rate): 96 us, 61 of it instructions (1080 per 32 pixels), the rest latency
// at 42 % of the warps; with the lists read from memory wherever they are needed it took 142.  72 registers hold 20 classes and four
// entries; more spill (32 classes and eight entries 316 to 372 bytes: 1,048,576 positions in 104 us, with four entries in 60).
#include "distill.cuh"

namespace adk {

// CM: C rounded up to a multiple of 4.  K: room for the entries.  PLANES: the classes come from planes as they lie; else from rows
// in shared memory, vec: of whole vectors, an odd number of them apart.
template <typename T, int CM, int K, bool BWD, bool PLANES>
__global__ void __launch_bounds__(kPositions, 7) distill_few(DistillP p, int vec) {
  typedef Position<T, PLANES ? 0 : 1> X;
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  __shared__ uint32_t all_cls[kPositions * K];
  __shared__ float all_t[kPositions * K];
  const uint32_t C = p.x.C, k = p.top, tp = vec ? tile_pitch<T, 2>(C) : C;
  T *tile = (T*)tiles, *olds = tile + kPositions * tp;   // what the gradient is added to
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions);
    for (uint32_t i = threadIdx.x; i < n * k; i += kPositions) {
      all_cls[i] = p.top_class[r0 * k + i];
      all_t[i] = p.top_logit[r0 * k + i];
    }
    const float f = BWD && threadIdx.x < n ? p.dloss[r] * p.scale : 0.f;
    float shift = p.rest && p.top_lse && threadIdx.x < n ? (float)(p.top_lse[r] * kLog2e) : 0.f;
    if (!PLANES) {
      copy_tile<T>(vec != 0, (const T*)p.logits, p.x, r0, n, tile);
      if (BWD && p.accumulate) copy_tile<T>(vec != 0, (const T*)p.dlogits, p.g, r0, n, olds);
    }
    __syncthreads();
    if (threadIdx.x < n) {
      const X x = {PLANES ? (const T*)p.logits + p.x.offset(r) : tile + threadIdx.x * tp, (uint32_t)(p.x.step * sizeof(T)), C};
      const X o = {PLANES ? (T*)p.dlogits + (BWD ? p.g.offset(r) : 0) : tile + threadIdx.x * tp, (uint32_t)(p.g.step * sizeof(T)), C};
      const X old = {PLANES ? o.x : olds + threadIdx.x * tp, o.step, C};
      float v[CM];
      load_few<T, CM>(x, vec != 0, v);
      // the list
      uint32_t cls[K], bits = 0, entries = 0;
      float a[K], xs[K], am = -INFINITY, mk = -INFINITY;
#pragma unroll
      for (uint32_t j = 0; j < K; ++j) {
        cls[j] = j < k ? all_cls[threadIdx.x * k + j] : kNoClass;
        const bool in = cls[j] < C;
        a[j] = in ? all_t[threadIdx.x * k + j] * p.ts : -INFINITY;
        xs[j] = in ? x.get(cls[j]) : -INFINITY;
        bits |= in ? 1u << cls[j] : 0u;
        entries += in;
        am = fmaxf(am, a[j]);
        mk = fmaxf(mk, xs[j]);
      }
      const bool twice = __popc(bits) != (int)entries;   // a class stands twice
      float Q = 0.f, z = 0.f;
      if (!p.rest) {
        if (am == -INFINITY) am = 0.f;
#pragma unroll
        for (uint32_t j = 0; j < K; ++j)
          if (j < k) z += exp2_fast(a[j] - am);
        shift = z != 0.f ? am + log2f(z) : 0.f;
      }
      float q[K];
#pragma unroll
      for (uint32_t j = 0; j < K; ++j) {
        q[j] = 0.f;
        if (j < k) {
          a[j] -= shift;
          q[j] = exp2_fast(a[j]);
          Q += q[j];
        }
      }
      // the classes: with rest those outside of the list, and the list's, each once
      float K1 = 0.f;
      Part s;
      if (p.rest) {
        if (mk == -INFINITY) mk = 0.f;
        uint32_t left = bits;
#pragma unroll
        for (uint32_t j = 0; j < K; ++j)
          if (j < k && cls[j] < C && (left >> cls[j] & 1u)) {
            left &= ~(1u << cls[j]);
            K1 += exp2_fast((xs[j] - mk) * p.cs);
          }
        float w[CM];
#pragma unroll
        for (uint32_t c = 0; c < CM; ++c) w[c] = bits >> c & 1u ? -INFINITY : v[c];
        sum_few<false, CM>(s, w, p.cs);
      } else {
        sum_few<false, CM>(s, v, p.cs);
      }
      const bool strange = s.strange(p.cs);
      float off = s.m == -INFINITY ? 0.f : fmaf(-s.m, p.cs, s.mc);
      if (strange) {
        off = s.S = 0.f;
        if (s.m == -INFINITY) s.m = 0.f;
        for (uint32_t c = 0; c < C; ++c)
          if (!p.rest || !(bits >> c & 1u)) s.S += exp2_fast((x.get(c) - s.m) * p.cs);
      }
      float loss;
      const Distilled d = row_sums(p, s.m, off, s.S, mk, K1, Q, loss);
#pragma unroll
      for (uint32_t j = 0; j < K; ++j)
        if (j < k && cls[j] < C) loss += d.term(q[j], a[j], xs[j], p.scale);
      if (p.loss) p.loss[r] = d.some ? loss + 0.f * d.L : 0.f;
      if constexpr (BWD) {
        const float coef = f * d.out;
        // the entries' gradients, which replace what is written for all classes
        float g[K];
#pragma unroll
        for (uint32_t j = 0; j < K; ++j)
          if (j < k && cls[j] < C) {
            float sum = q[j];
            if (twice) {
              sum = 0.f;
#pragma unroll
              for (uint32_t i = 0; i < K; ++i) sum += cls[i] == cls[j] ? q[i] : 0.f;
            }
            g[j] = d.some ? f * (exp2_fast((xs[j] - d.mt) * p.cs) * d.rS * d.Q - sum) : 0.f;
            if (p.accumulate) g[j] += old.get(cls[j]);
          }
        if (strange) {
#pragma unroll
          for (uint32_t c = 0; c < CM; ++c) v[c] = coef * exp2_fast((v[c] - s.m) * p.cs);
        } else {
          const F2 cs2 = pair(p.cs, p.cs), mc2 = pair(-s.mc, -s.mc), k2 = pair(coef, coef);
#pragma unroll
          for (int c = 0; c < CM; c += 2) {
            const float2 u = halves(fma2(pair(v[c], v[c + 1]), cs2, mc2));
            const float2 h = halves(mul2(pair(exp2_fast(u.x), exp2_fast(u.y)), k2));
            v[c] = h.x;
            v[c + 1] = h.y;
          }
        }
        if (p.accumulate) {
#pragma unroll
          for (uint32_t c = 0; c < CM; ++c)
            if (c + 4 < CM || c < C) v[c] += old.get(c);
        }
        store_few<T, CM>(o, vec != 0, v);
#pragma unroll
        for (uint32_t j = 0; j < K; ++j)
          if (j < k && cls[j] < C) o.set(cls[j], g[j]);
      }
    }
    __syncthreads();
    if (BWD && !PLANES) {
      write_tile<T>(vec != 0, (T*)p.dlogits, p.g, r0, n, tile);
      __syncthreads();
    }
  }
}

// ---------------------------------------------------------------- more classes or entries, and planes
// Rows of few classes in shared memory (MODE 1, 2), or classes in planes (MODE 0).  A bit per class tells which are listed.
constexpr uint32_t kMostBits = 4096;   // classes of such a mask: a word of 32 for each thread and 32 classes

template <typename T, int MODE, bool BWD>
__global__ void __launch_bounds__(kPositions) distill_by_position(DistillP p) {
  grid_dependency();
  extern __shared__ __align__(16) uint8_t tiles[];
  const uint32_t C = p.x.C, k = p.top, words = (C + 31) / 32;
  constexpr int TM = MODE ? MODE : 1;
  const uint32_t tile_elems = MODE ? kPositions * tile_pitch<T, TM>(C) : 0;
  uint32_t* bits = (uint32_t*)tiles + threadIdx.x;   // word w at [w * kPositions]
  T *tile = (T*)(tiles + (size_t)words * kPositions * 4), *olds = tile + tile_elems;
  const size_t blocks = (p.x.rows + kPositions - 1) / kPositions;
  for (size_t blk = blockIdx.x; blk < blocks; blk += gridDim.x) {
    const size_t r0 = blk * kPositions, r = r0 + threadIdx.x;
    const uint32_t n = (uint32_t)(p.x.rows - r0 < kPositions ? p.x.rows - r0 : kPositions);
    if (MODE) {
      copy_tile<T>(TM == 2, (const T*)p.logits, p.x, r0, n, tile);
      if (BWD && p.accumulate) copy_tile<T>(TM == 2, (const T*)p.dlogits, p.g, r0, n, olds);
      __syncthreads();
    }
    if (r < p.x.rows) {
      const uint32_t at = threadIdx.x * tile_pitch<T, TM>(C);
      const Position<T, MODE> x = {MODE ? tile + at : (const T*)p.logits + p.x.offset(r), (uint32_t)(p.x.step * sizeof(T)), C};
      const uint32_t* cls = p.top_class + r * k;
      const float* t = p.top_logit + r * k;
      auto listed = [&](uint32_t c) { return bits[(c >> 5) * kPositions] >> (c & 31) & 1u; };
      // the list: its weights' sum, and a bit for each class
      for (uint32_t w = 0; w < words; ++w) bits[w * kPositions] = 0;
      float am = -INFINITY, shift, Q = 0.f, mk = -INFINITY, K = 0.f;
      for (uint32_t j = 0; j < k; ++j)
        if (cls[j] < C) {
          bits[(cls[j] >> 5) * kPositions] |= 1u << (cls[j] & 31);
          am = fmaxf(am, t[j] * p.ts);
          mk = fmaxf(mk, x.get(cls[j]));
        }
      if (mk == -INFINITY) mk = 0.f;
      if (p.rest) {
        shift = p.top_lse ? (float)(p.top_lse[r] * kLog2e) : 0.f;
      } else {
        if (am == -INFINITY) am = 0.f;
        float z = 0.f;
        for (uint32_t j = 0; j < k; ++j)
          if (cls[j] < C) z += exp2f(t[j] * p.ts - am);
        shift = z != 0.f ? am + log2f(z) : 0.f;
      }
      for (uint32_t j = 0; j < k; ++j)
        if (cls[j] < C) Q += exp2f(t[j] * p.ts - shift);
      // the classes: with rest those outside of the list, and the list's, each once
      Part a;
      a.clear();
      for (uint32_t c = 0; c < C; c += 8) {
        float f[8], bm;
        x.batch(c, C, f);
        if (p.rest) {
          const uint32_t w = bits[(c >> 5) * kPositions] >> (c & 31);
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = w >> i & 1u ? -INFINITY : f[i];
        }
        bm = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
        a.reach<false>(bm, p.cs);
        float S[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) S[i & 1] += exp2_fast(fmaf(f[i], p.cs, -a.mc));
        a.S += S[0] + S[1];
      }
      const bool strange = a.strange(p.cs);
      a.refer<false>(Part::reference(a.m, p.cs));
      float off = a.m == -INFINITY ? 0.f : fmaf(-a.m, p.cs, a.mc);
      if (strange) {
        off = a.S = 0.f;
        if (a.m == -INFINITY) a.m = 0.f;
        for (uint32_t c = 0; c < C; ++c)
          if (!p.rest || !listed(c)) a.S += exp2_fast((x.get(c) - a.m) * p.cs);
      }
      if (p.rest)
        for (uint32_t c0 = 0; c0 < C; c0 += 32)
          for (uint32_t w = bits[(c0 >> 5) * kPositions]; w; w &= w - 1) K += exp2_fast((x.get(c0 + __ffs(w) - 1) - mk) * p.cs);
      float loss;
      const Distilled d = row_sums(p, a.m, off, a.S, mk, K, Q, loss);
      for (uint32_t j = 0; j < k; ++j)
        if (cls[j] < C) {
          const float v = t[j] * p.ts - shift;
          loss += d.term(exp2f(v), v, x.get(cls[j]), p.scale);
        }
      if (p.loss) p.loss[r] = d.some ? loss + 0.f * d.L : 0.f;
      if constexpr (BWD) {
        const Position<T, MODE> o = {MODE ? tile + at : (T*)p.dlogits + p.g.offset(r), (uint32_t)(p.g.step * sizeof(T)), C};
        const Position<T, MODE> old = {MODE ? olds + at : (T*)p.dlogits + p.g.offset(r), (uint32_t)(p.g.step * sizeof(T)), C};
        const float f = p.dloss[r] * p.scale, coef = f * d.out;
        // the classes outside of the list; those of the list keep their logits for the loop behind it
        for (uint32_t c = 0; c < C; c += 8) {
          float h[8];
          x.batch(c, C, h);
          const uint32_t w = bits[(c >> 5) * kPositions] >> (c & 31);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float u = strange ? (h[i] - a.m) * p.cs : fmaf(h[i], p.cs, -a.mc);
            h[i] = coef * exp2_fast(u);
            if (c + i < C && !(w >> i & 1u)) o.set(c + i, p.accumulate ? h[i] + old.get(c + i) : h[i]);
          }
        }
        for (uint32_t j = 0; j < k; ++j) {
          const uint32_t c = cls[j];
          if (c >= C || !listed(c)) continue;   // no class, or written already
          bits[(c >> 5) * kPositions] &= ~(1u << (c & 31));
          float sum = 0.f;
          for (uint32_t i = j; i < k; ++i)
            if (cls[i] == c) sum += exp2f(t[i] * p.ts - shift);
          const float v = d.some ? f * (exp2_fast((x.get(c) - d.mt) * p.cs) * d.rS * d.Q - sum) : 0.f;
          o.set(c, p.accumulate ? v + old.get(c) : v);
        }
      }
    }
    if (MODE && BWD) {
      __syncthreads();
      write_tile<T>(TM == 2, (T*)p.dlogits, p.g, r0, n, tile);
    }
    if (MODE) __syncthreads();
  }
}

// mode: as position_mode() has it
template <typename T, int CM, int K, bool BWD>
static int launch_few(const DistillP& p, int mode, cudaStream_t s) {
  if constexpr (CM <= 32) {
    if (p.x.C > CM) return launch_few<T, CM + 4, K, BWD>(p, mode, s);
    const size_t smem = (mode == 0 ? 0 : mode == 2 ? tile_bytes<T, 2>(p.x.C) : tile_bytes<T, 1>(p.x.C)) * (BWD && p.accumulate ? 2 : 1);   // 36 KB at most, beside 8 KB of lists
    if (mode == 0) launch(distill_few<T, CM, K, BWD, true>, position_blocks(p.x.rows), kPositions, smem, s, p, 0);
    else launch(distill_few<T, CM, K, BWD, false>, position_blocks(p.x.rows), kPositions, smem, s, p, mode == 2);
    return AD_OK;
  } else return AD_ERR_UNSUPPORTED;
}
template <typename T, int MODE, bool BWD>
static int launch_positions(const DistillP& p, cudaStream_t s) {
  auto kernel = distill_by_position<T, MODE, BWD>;
  const size_t smem = (p.x.C + 31) / 32 * kPositions * 4 + tile_bytes<T, MODE>(p.x.C) * (BWD && p.accumulate ? 2 : 1);
  // the limit belongs to the function: the most that it takes
  constexpr int most = kPositions * (MODE ? 2 * 4 + 2 * (kFewClasses * 4 + 16) : kMostBits / 8);
  if (smem > 48 * 1024 && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, most) != cudaSuccess) {
    cudaGetLastError();
    return AD_ERR_CUDA;
  }
  launch(kernel, position_blocks(p.x.rows), kPositions, smem, s, p);
  return AD_OK;
}

template <typename T, bool BWD>
int distill_positions(const DistillP& p, cudaStream_t s) {
  int mode = position_mode<T>(p.x, p.logits);
  if (mode == 0 && (p.x.C > kMostBits || (BWD && (p.g.HW == 0 || (uint64_t)p.g.step * sizeof(T) > 0xffffffffu)))) mode = -1;   // the gradient of an image of one position, packed
  if (mode > 0 && BWD && p.g.step != 1) mode = -1;
  if (mode == 2 && BWD && position_mode<T>(p.g, p.dlogits) != 2) mode = 1;
  if (mode < 0) return AD_ERR_UNSUPPORTED;
  if (p.x.C <= 32 && p.top <= 4) return launch_few<T, 4, 4, BWD>(p, mode, s);
  if (p.x.C <= 32 && p.top <= 8) return launch_few<T, 4, 8, BWD>(p, mode, s);
  if (mode == 0) return launch_positions<T, 0, BWD>(p, s);
  return mode == 1 ? launch_positions<T, 1, BWD>(p, s) : launch_positions<T, 2, BWD>(p, s);
}
template int distill_positions<float, false>(const DistillP&, cudaStream_t);
template int distill_positions<float, true>(const DistillP&, cudaStream_t);
template int distill_positions<__nv_bfloat16, false>(const DistillP&, cudaStream_t);
template int distill_positions<__nv_bfloat16, true>(const DistillP&, cudaStream_t);

}  // namespace adk
