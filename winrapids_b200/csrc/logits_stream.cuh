// logits_stream.cuh -- passes over a row of logits that stays in L2, and the collection of its largest
// elements (top_logits.cu, sample.cu).
//
// A cluster of C CTAs takes one row (C = 1 when there are many); CTA c a contiguous slice of its
// 16-byte vectors, warp w of it a contiguous part of the slice, so that "in the order of the index" is
// the order (CTA, warp, step, lane, element).  The first pass brings the row from HBM, later ones find
// it in L2.
#pragma once
#include "logits_row.cuh"

namespace tbgb {
namespace row {

constexpr int STEP = 4;  // vectors of a lane that are loaded together

template <typename T, int NT, bool MASK>
struct Stream {
  static constexpr int EPV = Elem<T>::EPV;
  RowView<T> rv;
  const uint64_t* mask;
  int v0, v1;  // this CTA's vectors
  int a, b;    // this warp's

  __device__ __forceinline__ Stream(const T* p, int vocab, const uint64_t* m, int rank, int C) : rv(p, vocab), mask(m) {
    const int each = (rv.nvec + C - 1) / C;
    v0 = min(rank * each, rv.nvec);
    v1 = min(v0 + each, rv.nvec);
    const int per = ((v1 - v0 + NT - 1) / NT) * 32;
    a = min(v0 + static_cast<int>(threadIdx.x >> 5) * per, v1);
    b = min(a + per, v1);
  }
  __device__ __forceinline__ uint4 load(int v) const {
    uint4 x = rv.whole(v) ? __ldcg(reinterpret_cast<const uint4*>(rv.base) + v) : rv.load_part(v);
    if (MASK) mask_vector<T>(x, rv, v, mask);
    return x;
  }
  // f(x, base): x[i] is vector base + 32 i + lane; steps of the warp from vector `from` to before `to`.
  // The next step's vectors are on their way while f works on this one's.
  // TWO: two steps a turn, which saves handing the next step's vectors on (a move for each register) and holds
  // f twice: top logits 176 -> 167 us for 2048 x 131072 bf16, top-p's longer steps 114 -> 126 for 256 x 131072.
  template <bool TWO = false, typename F>
  __device__ __forceinline__ void each(int from, int to, F f) const {
    const int lane = threadIdx.x & 31;
    uint4 x[STEP];
    auto get = [&](uint4 (&y)[STEP], int base) {
      if (!MASK && base > 0 && base + 32 * STEP <= to && base + 32 * STEP < rv.nvec) {
        const uint4* p = reinterpret_cast<const uint4*>(rv.base) + base + lane;
#pragma unroll
        for (int i = 0; i < STEP; ++i) y[i] = __ldcg(p + 32 * i);
      } else {
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
          y[i] = RowView<T>::none();
          const int v = base + 32 * i + lane;
          if (v < to) y[i] = load(v);
        }
      }
    };
    if (from < to) get(x, from);
#pragma unroll 1
    for (int base = from; base < to; base += (TWO ? 64 : 32) * STEP) {
      uint4 y[STEP];
      if (base + 32 * STEP < to) get(y, base + 32 * STEP);
      f(x, base);
      if (TWO) {
        if (base + 32 * STEP >= to) break;
        if (base + 64 * STEP < to) get(x, base + 64 * STEP);
        f(y, base + 32 * STEP);
      } else {
#pragma unroll
        for (int i = 0; i < STEP; ++i) x[i] = y[i];
      }
    }
  }
  __device__ __forceinline__ int index(int v, int e) const { return rv.first(v) + e; }
};

// ---- a lower bound of the K-th largest of a CTA's values ------------------------------------------------

constexpr int BINS = 512;

struct BoundSmem {
  unsigned hist[BINS];
  float2 ends[32];
  unsigned least;
};

// values(g) calls g(v) for every value (> -inf) of the calling thread.  The result is one of the values
// (or -FLT_MAX when there are fewer than K): at least K of them are not below it, and not many more:
// the values are counted in BINS equal parts of their range.
template <int NT, typename F>
__device__ __forceinline__ float kth_bound(BoundSmem& sm, int K, F values) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float hi = neg_inff(), lo = -neg_inff();
  values([&](float v) {
    hi = fmaxf(hi, v);
    lo = fminf(lo, v);
  });
  hi = warp_max(hi);
  lo = -warp_max(-lo);
  __syncthreads();  // the arrays are free
  for (int b = tid; b < BINS; b += NT) sm.hist[b] = 0;
  if (lane == 0) sm.ends[warp] = make_float2(lo, hi);
  if (tid == 0) sm.least = 0xffffffffu;
  __syncthreads();
  const float2 en = lane < NT / 32 ? sm.ends[lane] : make_float2(-neg_inff(), neg_inff());
  hi = warp_max(en.y);
  lo = -warp_max(-en.x);
  const float scale = hi > lo ? BINS / (hi - lo) : 0.0f;
  // (an infinite range gives 0 or NaN, that is bin 0: a looser bound)
  auto bin = [&](float v) { return min(static_cast<int>((hi - v) * scale), BINS - 1); };
  values([&](float v) { atomicAdd(&sm.hist[bin(v)], 1u); });
  __syncthreads();
  unsigned part = 0, c[BINS / 32];
#pragma unroll
  for (int i = 0; i < BINS / 32; ++i) {
    c[i] = sm.hist[lane * (BINS / 32) + i];
    part += c[i];
  }
  const unsigned upto = warp_inclusive(part);
  const unsigned hit = __ballot_sync(FULL, upto >= static_cast<unsigned>(K));
  if (hit == 0) return -3.402823466e38f;
  const int at = __ffs(hit) - 1;
  int last = 0;
  unsigned run = upto - part;
#pragma unroll
  for (int i = 0; i < BINS / 32; ++i) {
    if (run < static_cast<unsigned>(K)) last = lane * (BINS / 32) + i;
    run += c[i];
  }
  last = __shfl_sync(FULL, last, at);
  unsigned least = 0xffffffffu;
  values([&](float v) {
    if (bin(v) <= last) least = min(least, Elem<float>::key(v));
  });
  least = __reduce_min_sync(FULL, least);
  if (lane == 0) atomicMin(&sm.least, least);
  __syncthreads();
  return Elem<float>::unkey(sm.least);
}

// ---- the largest elements of a row ------------------------------------------------------------------------

// A CTA's lists, in dynamic shared memory: vectors that may hold one of the K largest (key of the
// vector's largest element, vector), and elements (key, ~id): sorted as whole numbers they are in the
// order (logit descending, id ascending).  Keys are those of the logit as a 32-bit number.
struct TopLists {
  unsigned long long* vec;
  unsigned long long* el;
  int vec_cap, el_cap;
};

struct TopSmem {
  BoundSmem bound;
  int n_vec, n_el, spilled;
  float tau;
};

__host__ __device__ inline int top_vec_cap(int k) { return k <= 128 ? 1024 : 8 * k; }
__host__ __device__ inline int top_el_cap(int k) { return k <= 256 ? 1024 : 4096; }

// Fills lists.el (sm.n_el entries) with every element of the CTA's slice that is not below the returned bound;
// the K largest of the slice are among them.  sm.spilled is set when the lists are too short (many equal
// elements).  With `pass` the caller sees every step of the pass over the slice too (x, base).
//   1. a sample (the first 4096 vectors of the warps' parts, a quarter of the row at 131072 16-bit logits): the K-th largest
//      of its lanes' (for many K its vectors') maxima is a first bound
//   2. one pass: vectors whose maximum reaches it are listed
//   3. the K-th largest of the listed maxima is the bound: their elements above it are listed
template <typename T, int NT, bool MASK, typename F>
__device__ __forceinline__ void collect_top(const Stream<T, NT, MASK>& st, int K, TopSmem& sm, const TopLists& li, F pass) {
  constexpr int SAMPLE = 4096 / NT;  // vectors of a lane
  const int tid = threadIdx.x, lane = tid & 31;
  float s[SAMPLE], most = neg_inff();
#pragma unroll
  for (int i = 0; i < SAMPLE; ++i) {
    const int v = st.a + i * 32 + lane;
    s[i] = v < st.b ? Elem<T>::vmax(st.load(v)) : neg_inff();
    most = fmaxf(most, s[i]);
  }
  if (tid == 0) sm.n_vec = sm.n_el = sm.spilled = 0;
  const bool lanes_do = K <= NT / 4;
  const float tau0 = kth_bound<NT>(sm.bound, K, [&](auto g) {
    if (lanes_do) {
      if (most > neg_inff()) g(most);
    } else {
#pragma unroll
      for (int i = 0; i < SAMPLE; ++i)
        if (s[i] > neg_inff()) g(s[i]);
    }
  });
  st.template each<true>(st.a, st.b, [&](const uint4 (&x)[STEP], int base) {
    float m[STEP], top = neg_inff();
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      m[i] = Elem<T>::vmax(x[i]);
      top = fmaxf(top, m[i]);
    }
    if (top >= tau0) {
#pragma unroll
      for (int i = 0; i < STEP; ++i)
        if (m[i] >= tau0) {
          const int at = atomicAdd(&sm.n_vec, 1);
          if (at < li.vec_cap)
            li.vec[at] = (static_cast<unsigned long long>(Elem<float>::key(m[i])) << 32) |
                         static_cast<unsigned>(base + 32 * i + lane);
        }
    }
    pass(x, top);
  });
  __syncthreads();
  const int n = min(sm.n_vec, li.vec_cap);
  const float tau = kth_bound<NT>(sm.bound, K, [&](auto g) {
    for (int i = tid; i < n; i += NT) g(Elem<float>::unkey(static_cast<uint32_t>(li.vec[i] >> 32)));
  });
  if (tid == 0) {
    if (sm.n_vec > li.vec_cap) sm.spilled = 1;
    sm.tau = tau;
  }
  for (int i = tid; i < n; i += NT) {
    const unsigned long long u = li.vec[i];
    if (Elem<float>::unkey(static_cast<uint32_t>(u >> 32)) < tau) continue;
    const int v = static_cast<int>(static_cast<uint32_t>(u));
    const uint4 x = st.load(v);
#pragma unroll
    for (int e = 0; e < Stream<T, NT, MASK>::EPV; ++e) {
      const float z = Elem<T>::get(x, e);
      if (z >= tau) {
        const int at = atomicAdd(&sm.n_el, 1);
        if (at < li.el_cap)
          li.el[at] = (static_cast<unsigned long long>(Elem<float>::key(z)) << 32) | static_cast<uint32_t>(~st.index(v, e));
      }
    }
  }
  __syncthreads();
  if (tid == 0 && sm.n_el > li.el_cap) sm.spilled = 1;
}

// list[0, n) without what lies below a bound of the K-th largest; the new n (all of it where that is not more than
// sort_list takes quickly).
template <int NT>
__device__ __forceinline__ int prune_list(BoundSmem& sm, unsigned long long* list, unsigned long long* spare, int* count,
                                          int n, int K) {
  if (n <= 256 || K > 224) return n;
  const int tid = threadIdx.x;
  if (tid == 0) *count = 0;
  const float tau = kth_bound<NT>(sm, K, [&](auto g) {
    for (int i = tid; i < n; i += NT) g(Elem<float>::unkey(static_cast<uint32_t>(list[i] >> 32)));
  });
  for (int i = tid; i < n; i += NT)
    if (Elem<float>::unkey(static_cast<uint32_t>(list[i] >> 32)) >= tau) spare[atomicAdd(count, 1)] = list[i];
  __syncthreads();
  n = *count;
  for (int i = tid; i < n; i += NT) list[i] = spare[i];
  __syncthreads();
  return n;
}

// Sorts list[0, n), largest first, n <= cap (a power of two).
template <int NT>
__device__ __forceinline__ void sort_list(unsigned long long* list, int n) {
  const int tid = threadIdx.x;
  int n2 = 32;
  while (n2 < n) n2 <<= 1;
  for (int j = n + tid; j < n2; j += NT) list[j] = 0;
  __syncthreads();
  if (n2 <= 256) {
    // the place of an element is the number of larger ones (no two are equal but the zeros behind them)
    unsigned long long mine = 0;
    int place = 0;
    if (tid < n) {
      mine = list[tid];
#pragma unroll 4
      for (int j = 0; j < n2; j += 2) {
        const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(&list[j]);
        place += (two.x > mine) + (two.y > mine);
      }
    }
    __syncthreads();
    if (tid < n) list[place] = mine;
    __syncthreads();
    return;
  }
  for (int size = 2; size <= n2; size <<= 1)
    for (int step = size >> 1; step > 0; step >>= 1) {
      for (int p = tid; p < n2 / 2; p += NT) {
        const int i = (p / step) * step * 2 + p % step, j = i + step;
        const bool down = (i & size) == 0;
        const unsigned long long x = list[i], y = list[j];
        if ((x < y) == down) {
          list[i] = y;
          list[j] = x;
        }
      }
      __syncthreads();
    }
}

}  // namespace row
}  // namespace tbgb
