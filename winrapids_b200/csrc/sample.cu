// sample.cu -- one token per row from its logits, by temperature, top-k, top-p and min-p, from a
// given uniform number.
//
// With zmax the row's largest allowed logit, a token's weight is
//   w = 2^((z - zmax) * (log2(e) / T)),   rounded to a multiple of 2^-30,
// so weights are whole numbers (in units of 2^-30, at most 2^30 each) and every sum of them is
// exact: the token does not depend on the order of summation or on the split over CTAs.  (The power itself is the
// device's ex2.approx, right to about 2 units in the last place of 24 bits.)  The grid is finer than the numbers that pick (a 32-bit uniform number has steps of
// 2^-24) and than the rounding of a 32-bit running sum would be.
//   top-k   the first k by (logit descending, id ascending)
//   top-p   of those, with sum W, the shortest prefix whose sum reaches ceil(p W)
//   min-p   of those, the tokens with 2^(...) >= min_p
// Each cut keeps a prefix of the same order, so all of them together are one threshold: a key tau
// and how many of the tokens equal to it are kept (the lowest ids).  The token is the first, in the
// order of the ids, whose running sum exceeds floor(u W'), W' the sum of what is kept.
#include <algorithm>
#include <climits>

#include "logits_select.cuh"
#include "logits_stream.cuh"

namespace tbgb {

namespace {

using namespace row;

constexpr float kGrid = 1073741824.0f;  // 2^30

struct Weight {
  float zmax, scale;
  __device__ __forceinline__ float power(float z) const { return z == zmax ? 1.0f : power2((z - zmax) * scale); }
  // 0 for -inf (and for the NaN of -inf at an infinite temperature)
  __device__ __forceinline__ unsigned unit(float z) const { return __float2uint_rn(power(z) * kGrid); }
  __device__ __forceinline__ unsigned long long operator()(float z) const { return unit(z); }
};

struct Share {  // one CTA's part of what is kept
  unsigned long long sure;  // weight beyond tau
  unsigned ties;            // tokens at tau
};

struct ExactSmem {
  SelectSmem sel;
  float wm[32], cta_max;
  unsigned long long w_sure[32], cta_sum;
  unsigned w_ties[32];
  Share share;
};

// A row by radix descent and passes over all of it: right for any number of equal logits, NaN, infinities, any
// temperature and any k.  For rows that the quicker ways below do not take.
template <typename T, int NT>
__device__ __noinline__ void exact_row(const SampleArgs& a, long long r, ExactSmem& sm) {
  constexpr int NW = NT / 32;
  constexpr bool RES = false;
  SelectSmem& sel = sm.sel;
  float *wm = sm.wm, &cta_max = sm.cta_max;
  unsigned long long *w_sure = sm.w_sure, &cta_sum = sm.cta_sum;
  unsigned* w_ties = sm.w_ties;
  Share& share = sm.share;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Slice<T, NT, RES> sl(static_cast<const T*>(a.x.logits) + r * a.x.ld, a.x.vocab,
                       a.mask ? a.mask + r * a.mask_ld : nullptr, rank, C);
  const float temperature = a.p.temperature ? a.p.temperature[r] : a.p.temperature_all;
  const int top_k = a.p.top_k ? a.p.top_k[r] : a.p.top_k_all;
  const float top_p = a.p.top_p ? a.p.top_p[r] : a.p.top_p_all;
  const float min_p = fminf(a.p.min_p ? a.p.min_p[r] : a.p.min_p_all, 1.0f);  // the largest logit always stays

  // the largest logit
  float m = neg_inff();
  for (int t = 0; t < sl.tiles; ++t) {
    sl.fetch(t);
    sl.each([&](float z, int, int) { m = fmaxf(m, z); });
  }
  m = warp_max(m);
  if (lane == 0) wm[warp] = m;
  __syncthreads();
  if (warp == 0) {
    m = warp_max(lane < NW ? wm[lane] : neg_inff());
    if (lane == 0) cta_max = m;
  }
  cl.sync();
  m = neg_inff();
  for (int c = 0; c < C; ++c) m = fmaxf(m, *cl.map_shared_rank(&cta_max, c));
  if (m == neg_inff()) {  // nothing is allowed (the same for every CTA of the cluster)
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = neg_inff();
    }
    cl.sync();  // peers may still be reading cta_max
    return;
  }
  const bool greedy = !(temperature > 0.0f);
  const Weight weight{m, greedy ? 1.0f : 1.4426950408889634f / temperature};

  // the threshold
  int flip = 0;
  uint32_t tau = 0;           // below every key
  unsigned long long above = 0;
  unsigned keep_ties = UINT_MAX;
  if (greedy) {
    tau = Elem<T>::key(m);
    keep_ties = 1;
  } else {
    if (top_k > 0 && top_k < a.x.vocab &&
        radix_select(sl, cl, sel, flip, static_cast<unsigned long long>(top_k), CountOne(), tau, above))
      keep_ties = static_cast<unsigned>(top_k - above);
    else
      tau = 0;
    if (top_p < 1.0f) {
      // the sum of what top-k left
      unsigned long long sum = 0;
      for (int t = 0; t < sl.tiles; ++t) {
        sl.fetch(t);
        sl.each([&](float z, int, int) { sum += Elem<T>::key(z) > tau ? weight.unit(z) : 0u; });
      }
      sum = warp_sum(sum);
      if (lane == 0) w_sure[warp] = sum;
      __syncthreads();
      if (tid == 0) {
        unsigned long long s = 0;
        for (int w = 0; w < NW; ++w) s += w_sure[w];
        cta_sum = s;
      }
      cl.sync();
      unsigned long long W = 0;
      for (int c = 0; c < C; ++c) W += *cl.map_shared_rank(&cta_sum, c);
      if (keep_ties != UINT_MAX) W += static_cast<unsigned long long>(keep_ties) * weight.unit(Elem<T>::unkey(tau));
      const double want = ceil(static_cast<double>(top_p) * static_cast<double>(W));
      const unsigned long long target = want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull;
      if (radix_select(sl, cl, sel, flip, target, weight, tau, above)) {
        const unsigned w = weight.unit(Elem<T>::unkey(tau));  // > 0: tau's tokens carry the sum over the target
        keep_ties = static_cast<unsigned>((target - above + w - 1) / w);
      }
    }
  }
  const unsigned w_tau = keep_ties == UINT_MAX ? 0u : weight.unit(Elem<T>::unkey(tau));
  const bool tau_ok = keep_ties != UINT_MAX && (greedy || weight.power(Elem<T>::unkey(tau)) >= min_p);
  auto sure = [&](float z) -> unsigned {  // a token's weight if it is kept whatever the ties
    if (Elem<T>::key(z) <= tau) return 0u;
    const float e = weight.power(z);
    return e >= min_p ? __float2uint_rn(e * kGrid) : 0u;
  };
  auto tie = [&](float z) -> unsigned { return tau_ok && Elem<T>::key(z) == tau; };

  // this CTA's part
  unsigned long long sum = 0;
  unsigned ties = 0;
  for (int t = 0; t < sl.tiles; ++t) {
    sl.fetch(t);
    sl.each([&](float z, int, int) {
      sum += sure(z);
      ties += tie(z);
    });
  }
  sum = warp_sum(sum);
  ties = __reduce_add_sync(FULL, ties);
  if (lane == 0) {
    w_sure[warp] = sum;
    w_ties[warp] = ties;
  }
  __syncthreads();
  if (tid == 0) {
    Share s{0, 0};
    for (int w = 0; w < NW; ++w) {
      s.sure += w_sure[w];
      s.ties += w_ties[w];
    }
    share = s;
  }
  cl.sync();
  unsigned long long total = 0, before = 0, own = 0;
  unsigned ties_before = 0, seen = 0;
  for (int c = 0; c < C; ++c) {
    const Share s = *cl.map_shared_rank(&share, c);
    const unsigned left = keep_ties > seen ? keep_ties - seen : 0u;
    const unsigned long long kept = s.sure + static_cast<unsigned long long>(min(left, s.ties)) * w_tau;
    if (c == rank) {
      before = total;
      own = kept;
      ties_before = seen;
    }
    total += kept;
    seen += s.ties;
  }
  cl.sync();  // the last read of a peer's shared memory
  const float u = a.u[r];
  const double goal = floor(static_cast<double>(u) * static_cast<double>(total));
  unsigned long long target = goal > 0.0 ? static_cast<unsigned long long>(goal) : 0ull;
  if (target >= total) target = total - 1;
  if (target < before || target >= before + own) return;

  // the token is in this CTA: walk its tiles, warps, vector rows, lanes
  unsigned long long run = before;
  unsigned rank_tie = ties_before;
  for (int t = 0; t < sl.tiles; ++t) {
    sl.fetch(t);
    unsigned long long ws = 0;
    unsigned wt = 0;
    sl.each([&](float z, int, int) {
      ws += sure(z);
      wt += tie(z);
    });
    ws = warp_sum(ws);
    wt = __reduce_add_sync(FULL, wt);
    __syncthreads();
    if (lane == 0) {
      w_sure[warp] = ws;
      w_ties[warp] = wt;
    }
    __syncthreads();
    unsigned long long at = run;
    unsigned tr = rank_tie;
    bool mine = false;
    unsigned long long my_at = 0;
    unsigned my_tr = 0;
    for (int w = 0; w < NW; ++w) {
      const unsigned left = keep_ties > tr ? keep_ties - tr : 0u;
      const unsigned long long kept = w_sure[w] + static_cast<unsigned long long>(min(left, w_ties[w])) * w_tau;
      if (w == warp && target >= at && target < at + kept) {
        mine = true;
        my_at = at;
        my_tr = tr;
      }
      at += kept;
      tr += w_ties[w];
    }
    run = at;
    rank_tie = tr;
    if (mine) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i >= sl.per) break;
        unsigned n = 0;
#pragma unroll
        for (int e = 0; e < Elem<T>::EPV; ++e) n += tie(Elem<T>::get(sl.r[i], e));
        const unsigned upto = warp_inclusive(n);
        unsigned rk = my_tr + upto - n;
        unsigned long long v = 0;
#pragma unroll
        for (int e = 0; e < Elem<T>::EPV; ++e) {
          const float z = Elem<T>::get(sl.r[i], e);
          v += sure(z);
          if (tie(z) && rk++ < keep_ties) v += w_tau;
        }
        unsigned long long inc = warp_inclusive(v);
        const unsigned long long all = __shfl_sync(FULL, inc, 31);
        if (target < my_at + all) {
          unsigned long long x = my_at + inc - v;
          if (target >= x && target < x + v) {
            rk = my_tr + upto - n;
#pragma unroll
            for (int e = 0; e < Elem<T>::EPV; ++e) {
              const float z = Elem<T>::get(sl.r[i], e);
              unsigned long long w = sure(z);
              if (tie(z) && rk++ < keep_ties) w = w_tau;
              if (target >= x && target < x + w) {
                a.tokens[r] = sl.index(t, i, e);
                if (a.logprobs)
                  a.logprobs[r] = greedy ? 0.0f
                                         : (z == m ? 0.0f : (z - m) / temperature) -
                                               logf(static_cast<float>(static_cast<double>(total) / kGrid));
              }
              x += w;
            }
          }
          break;
        }
        my_at += all;
        my_tr += __shfl_sync(FULL, upto, 31);
      }
    }
    if (target < run) return;
  }
}

// ---- the quick ways ------------------------------------------------------------------------------------
//
// A kept prefix is all tokens whose (key of the logit, ~id), as one whole number, is at least `cut`: ties need no
// counting.
//   top-k (k <= 1024), greedy   the k largest are collected in one pass (logits_stream.cuh); everything
//                               else happens in that sorted list
//   nothing but min-p           a pass for the largest logit, one for the weights, summed per warp
//   top-p                       a pass for the largest logit, one for the sum W; one that counts the weights into
//                               1024 equal parts of the exponent's range, which finds the part that holds the
//                               prefix's end; one that lists that part and sums what lies above it
// The first pass reads HBM, the others L2.  Weights below 2^-7 are turned into whole numbers by an addition:
// 2^-7 + e has steps of 2^-30, so its bits less those of 2^-7 are e in those units (rounded to nearest,
// ties to even, as the conversion does), and bits are summed.  A conversion would cost a second
// instruction on the special function units, which are busy for most of the pass with the power itself.
// 96 us for 1024 x 100000 bf16 uncut (2.1 TB/s of its first pass's bytes); 149 for top-p 0.95 alone, 29 for top-k with top-p
// and 24 greedy over 256 x 131072 bf16.  512 threads a row: 256 took 1.7 times as long for top-p, 1024 1.1 and 1.5 times for
// top-p and top-k.

constexpr int kParts = 1024;       // of the exponent's range
constexpr int kPartBytes = 9 * 1024;  // two words for each, later the search's arrays
// Tokens of the part that holds the end of the prefix; with more the row takes the exact way.  Equal 16-bit logits between
// 16 and 32 are up to one in 40 of a vocabulary with a spread of 2: 256 rows of 151936 bf16 logits around 20, top-p 0.95,
// 229 us (around 0: 189), of 201088 9.4 ms (246).  A longer list costs the CTAs that an SM holds.
constexpr int kEdgeMost = 4096;
constexpr float kSmall = 0.0078125f;  // 2^-7

static_assert(2 * 4 * (kParts + 2) <= kPartBytes, "counters");

struct SampleSmem {
  TopSmem top;
  float f[32];
  unsigned long long w[32];
  unsigned long long cta_w, above;
  float cta_f;
  int n_edge, part;
  unsigned long long sub[32];
};

template <typename T, int NT, bool MASK>
struct Sampler {
  static constexpr int NW = NT / 32, EPV = Elem<T>::EPV, PAIRS = Elem<T>::PAIRS;
  const SampleArgs& a;
  const Stream<T, NT, MASK>& st;
  SampleSmem& sm;
  cg::cluster_group& cl;
  long long r;
  int C, rank;
  float temperature, min_p;
  Weight weight;

  __device__ __forceinline__ unsigned long long order_key(float z, int id) const {
    return (static_cast<unsigned long long>(Elem<float>::key(z)) << 32) | static_cast<uint32_t>(~id);
  }
  // sum of a u64 over the cluster, the same in every thread; `own_before` the sum over the CTAs in front
  __device__ __forceinline__ unsigned long long cluster_sum(unsigned long long warp_total, unsigned long long* own,
                                                            unsigned long long* before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (lane == 0) sm.w[warp] = warp_total;
    __syncthreads();
    unsigned long long mine = warp_sum(lane < NW ? sm.w[lane] : 0ull);
    *own = mine;
    *before = 0;
    if (C == 1) return mine;
    if (threadIdx.x == 0) sm.cta_w = mine;
    cl.sync();
    unsigned long long all = 0;
    for (int c = 0; c < C; ++c) {
      const unsigned long long v = *cl.map_shared_rank(&sm.cta_w, c);
      if (c < rank) *before += v;
      all += v;
    }
    cl.sync();
    return all;
  }
  // the weights of a vector's elements that pass keep(z, power, id), by conversion
  template <typename K>
  __device__ __forceinline__ unsigned long long exact_weights(const uint4& x, int v, K keep) const {
    unsigned long long s = 0;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      const float z = Elem<T>::get(x, e);
      const float p = z > neg_inff() ? weight.power(z) : 0.0f;
      if (keep(z, p, st.index(v, e))) s += __float2uint_rn(p * kGrid);
    }
    return s;
  }
  // All weights of this warp's part, nothing cut off.
  __device__ __forceinline__ unsigned long long all_weights() const {
    unsigned long long s = 0;
    const int lane = threadIdx.x & 31;
    const float2 minus = make_float2(-weight.zmax, -weight.zmax), scale2 = make_float2(weight.scale, weight.scale),
                 small2 = make_float2(kSmall, kSmall);
    st.each(st.a, st.b, [&](const uint4 (&x)[STEP], int base) {
      unsigned bits = 0;
#pragma unroll
      for (int i = 0; i < STEP; ++i) {
        if ((Elem<T>::vmax(x[i]) - weight.zmax) * weight.scale < -7.0f) {
#pragma unroll
          for (int j = 0; j < PAIRS; ++j) {
            const float2 q = add2(power2(Elem<T>::pair(x[i], j), minus, scale2), small2);
            bits += __float_as_uint(q.x) + __float_as_uint(q.y);
          }
          bits -= static_cast<unsigned>(EPV) * __float_as_uint(kSmall);  // (modulo 2^32: what is left is below it)
        } else {
          s += exact_weights(x[i], base + 32 * i + lane, [](float, float, int) { return true; });
        }
      }
      s += bits;
    });
    return s;
  }
  // Weights of [from, to) that pass keep(z, power, id); vectors whose largest logit is below `least` have none.
  template <typename K>
  __device__ __forceinline__ unsigned long long kept_weights(int from, int to, float least, K keep) const {
    unsigned long long s = 0;
    const int lane = threadIdx.x & 31;
    st.each(from, to, [&](const uint4 (&x)[STEP], int base) {
#pragma unroll 1
      for (int i = 0; i < STEP; ++i) {
        const uint4 y = i == 0 ? x[0] : i == 1 ? x[1] : i == 2 ? x[2] : x[3];
        if (Elem<T>::vmax(y) >= least) s += exact_weights(y, base + 32 * i + lane, keep);
      }
    });
    return s;
  }
  __device__ __forceinline__ float logprob(float z, unsigned long long total) const {
    return (z == weight.zmax ? 0.0f : (z - weight.zmax) / temperature) -
           logf(static_cast<float>(static_cast<double>(total) / kGrid));
  }
  __device__ __forceinline__ unsigned long long target_of(unsigned long long total) const {
    const double goal = floor(static_cast<double>(a.u[r]) * static_cast<double>(total));
    unsigned long long t = goal > 0.0 ? static_cast<unsigned long long>(goal) : 0ull;
    return t >= total ? total - 1 : t;
  }
  // The token, from the warps' sums of kept weights (sm.w, this CTA's from `before` on).
  template <typename K>
  __device__ __forceinline__ void pick(unsigned long long total, unsigned long long own, unsigned long long before,
                                       float least, K keep) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long target = target_of(total);
    if (target < before || target >= before + own) return;
    target -= before;
    const unsigned long long part = lane < NW ? sm.w[lane] : 0;
    const unsigned long long upto = warp_inclusive(part);
    int at = __ffs(__ballot_sync(FULL, upto > target)) - 1;  // the warp whose part holds the token
    target -= __shfl_sync(FULL, upto - part, at);
    // all warps share that part
    const int per = ((st.v1 - st.v0 + NT - 1) / NT) * 32;
    const int from = min(st.v0 + at * per, st.v1), to = min(from + per, st.v1);
    const int each = ((to - from + NT - 1) / NT) * 32;
    const int f = min(from + warp * each, to), t = min(f + each, to);
    const unsigned long long mine = warp_sum(kept_weights(f, t, least, keep));
    if (lane == 0) sm.sub[warp] = mine;
    __syncthreads();
    const unsigned long long p2 = lane < NW ? sm.sub[lane] : 0;
    const unsigned long long u2 = warp_inclusive(p2);
    at = __ffs(__ballot_sync(FULL, u2 > target)) - 1;
    if (warp != at) return;
    target -= __shfl_sync(FULL, u2 - p2, at);
    for (int v0 = f; v0 < t; v0 += 32) {
      const int v = v0 + lane;
      uint4 x = RowView<T>::none();
      if (v < t) x = st.load(v);
      const unsigned long long s = v < t && Elem<T>::vmax(x) >= least ? exact_weights(x, v, keep) : 0;
      const unsigned long long inc = warp_inclusive(s);
      const unsigned long long all = __shfl_sync(FULL, inc, 31);
      if (target >= all) {
        target -= all;
        continue;
      }
      if (target >= inc - s && target < inc) {
        unsigned long long left = target - (inc - s);
#pragma unroll 1
        for (int e = 0; e < EPV; ++e) {
          const int id = st.index(v, e);
          if (id < 0 || id >= a.x.vocab) continue;
          float z = neg_inff();
#pragma unroll
          for (int k = 0; k < EPV; ++k)
            if (k == e) z = Elem<T>::get(x, k);
          const float p = z > neg_inff() ? weight.power(z) : 0.0f;
          const unsigned long long w = keep(z, p, id) ? __float2uint_rn(p * kGrid) : 0u;
          if (left < w) {
            a.tokens[r] = id;
            if (a.logprobs) a.logprobs[r] = logprob(z, total);
            break;
          }
          left -= w;
        }
      }
      break;
    }
  }
};

struct CutSmem {
  unsigned long long mass[512], few[256], most, least, rem;
  unsigned count[512];
  int bin, n;
};

static_assert(sizeof(CutSmem) <= kPartBytes, "the search takes the place of the counters");

// The entry of list[0, n) (in no order) at which the running sum of weight(entry), from the largest entry down, reaches
// `need`; the sum of the list reaches it.  The range of entries that holds it is cut into 512 equal parts
// until no more than 256 entries are left: by their keys first, by their ids where keys are equal.
template <int NT, typename W>
__device__ __forceinline__ unsigned long long cut_of(CutSmem& sm, const unsigned long long* list, int n,
                                                     unsigned long long need, W weight) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) {
    sm.most = 0;
    sm.least = ~0ull;
    sm.n = 0;
  }
  __syncthreads();
  unsigned long long hi = 0, lo = ~0ull;
  for (int i = tid; i < n; i += NT) {
    hi = max(hi, list[i]);
    lo = min(lo, list[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    hi = max(hi, __shfl_xor_sync(FULL, hi, o));
    lo = min(lo, __shfl_xor_sync(FULL, lo, o));
  }
  if (lane == 0) {
    atomicMax(&sm.most, hi);
    atomicMin(&sm.least, lo);
  }
  __syncthreads();
  hi = sm.most;
  lo = sm.least;
  int left = n;
  while (left > 256) {
    const int shift = max(55 - __clzll(static_cast<long long>(hi - lo)), 0);  // (hi - lo) >> shift < 512
    for (int b = tid; b < 512; b += NT) {
      sm.mass[b] = 0;
      sm.count[b] = 0;
    }
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const unsigned long long u = list[i];
      if (u <= hi && u >= lo) {
        const int b = static_cast<int>((hi - u) >> shift);
        atomicAdd(&sm.mass[b], static_cast<unsigned long long>(weight(u)));
        atomicAdd(&sm.count[b], 1u);
      }
    }
    __syncthreads();
    if (warp == 0) {
      unsigned long long part = 0;
      for (int j = 0; j < 16; ++j) part += sm.mass[lane * 16 + j];
      const unsigned long long upto = warp_inclusive(part);
      const int at = __ffs(__ballot_sync(FULL, upto >= need)) - 1;
      if (lane == at) {
        unsigned long long run = upto - part;
        int b = lane * 16;
        while (run + sm.mass[b] < need) run += sm.mass[b++];
        sm.bin = b;
        sm.rem = need - run;
      }
    }
    __syncthreads();
    const unsigned long long b = static_cast<unsigned long long>(sm.bin);
    const unsigned long long top = hi - (b << shift), width = (1ull << shift) - 1;
    lo = top - lo < width ? lo : top - width;
    hi = top;
    need = sm.rem;
    left = static_cast<int>(sm.count[sm.bin]);
    __syncthreads();
  }
  for (int i = tid; i < n; i += NT)
    if (list[i] <= hi && list[i] >= lo) sm.few[atomicAdd(&sm.n, 1)] = list[i];
  __syncthreads();
  sort_list<NT>(sm.few, left);
  if (warp == 0) {
    unsigned long long run = 0;
    for (int j0 = 0; j0 < left; j0 += 32) {
      const int j = j0 + lane;
      const unsigned long long w = j < left ? weight(sm.few[j]) : 0;
      const unsigned long long inc = run + warp_inclusive(w);
      const unsigned hit = __ballot_sync(FULL, j < left && inc >= need);
      if (hit) {
        if (lane == 0) sm.most = sm.few[j0 + __ffs(hit) - 1];
        break;
      }
      run = __shfl_sync(FULL, inc, 31);
    }
  }
  __syncthreads();
  return sm.most;
}

template <typename T, int NT, bool MASK>
__global__ void __launch_bounds__(NT, 1024 / NT) sample_kernel(const SampleArgs a, int list_k) {
  constexpr int NW = NT / 32;
  extern __shared__ __align__(16) char dyn[];
  __shared__ SampleSmem sm;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const long long r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const float temperature = a.p.temperature ? a.p.temperature[r] : a.p.temperature_all;
  const int top_k = a.p.top_k ? a.p.top_k[r] : a.p.top_k_all;
  const float top_p = a.p.top_p ? a.p.top_p[r] : a.p.top_p_all;
  const float min_p = fminf(a.p.min_p ? a.p.min_p[r] : a.p.min_p_all, 1.0f);  // the largest logit always stays
  const Stream<T, NT, MASK> st(static_cast<const T*>(a.x.logits) + r * a.x.ld, a.x.vocab,
                               MASK ? a.mask + r * a.mask_ld : nullptr, rank, C);
  const bool greedy = !(temperature > 0.0f);
  const int k = greedy ? 1 : top_k;
  auto exact = [&]() {
    cl.sync();  // every CTA of the cluster is done with what lies there
    exact_row<T, NT>(a, r, *reinterpret_cast<ExactSmem*>(dyn));
  };

  if (k > 0 && k <= list_k) {
    // ---- the k largest in a list
    TopLists li;
    li.vec_cap = top_vec_cap(list_k);
    li.el_cap = top_el_cap(list_k);
    li.el = reinterpret_cast<unsigned long long*>(dyn);
    li.vec = li.el + li.el_cap;
    collect_top<T, NT, MASK>(st, k, sm.top, li, [](const uint4 (&)[STEP], float) {});
    if (C > 1) cl.sync();
    else __syncthreads();
    bool any = false;
    int n = 0;
    for (int c = 0; c < C; ++c) {
      const TopSmem* peer = cl.map_shared_rank(&sm.top, c);
      any |= peer->spilled != 0;
      n += peer->n_el;
    }
    if (any || n > li.el_cap) {
      exact();
      return;
    }
    if (rank == 0) {
      int at = sm.top.n_el;
      for (int c = 1; c < C; ++c) {
        const int nc = cl.map_shared_rank(&sm.top, c)->n_el;
        const unsigned long long* src = cl.map_shared_rank(li.el, c);
        for (int j = tid; j < nc; j += NT) li.el[at + j] = src[j];
        at += nc;
      }
    }
    if (C > 1) cl.sync();  // the lists have been read
    if (rank != 0) return;
    __syncthreads();
    n = prune_list<NT>(sm.top.bound, li.el, li.vec, &sm.top.n_vec, n, k);
    sort_list<NT>(li.el, n);
    n = min(n, k);
    if (n == 0 || greedy) {
      if (tid == 0) {
        a.tokens[r] = n ? static_cast<int>(~static_cast<uint32_t>(li.el[0])) : -1;
        if (a.logprobs) a.logprobs[r] = n ? 0.0f : neg_inff();
      }
      return;
    }
    const Weight weight{Elem<float>::unkey(static_cast<uint32_t>(li.el[0] >> 32)), 1.4426950408889634f / temperature};
    auto z_of = [&](int j) { return Elem<float>::unkey(static_cast<uint32_t>(li.el[j] >> 32)); };
    // running sums by warp 0, in chunks of 32: top-p, then what min-p leaves, as (~id, weight) for the second sort
    if (warp == 0) {
      unsigned long long W = 0;
      for (int j = lane; j < n; j += 32) W += weight.unit(z_of(j));
      W = warp_sum(W);
      unsigned long long need = ~0ull;
      if (top_p < 1.0f) {
        const double want = ceil(static_cast<double>(top_p) * static_cast<double>(W));
        need = want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull;
      }
      unsigned long long run = 0;
      int kept = 0;
      for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const float z = j < n ? z_of(j) : neg_inff();
        const float e = j < n ? weight.power(z) : 0.0f;
        const unsigned w = j < n ? __float2uint_rn(e * kGrid) : 0u;
        const unsigned long long inc = warp_inclusive(static_cast<unsigned long long>(w));
        const bool keep = j < n && run + inc - w < need && e >= min_p;
        if (keep) li.vec[j] = (li.el[j] << 32) | w;  // ~id in the upper half: larger for lower ids
        kept += __popc(__ballot_sync(FULL, keep));  // a prefix
        run += __shfl_sync(FULL, inc, 31);
      }
      if (lane == 0) sm.n_edge = kept;
    }
    __syncthreads();
    n = sm.n_edge;
    sort_list<NT>(li.vec, n);
    if (warp == 0) {
      unsigned long long W = 0;
      for (int j = lane; j < n; j += 32) W += static_cast<uint32_t>(li.vec[j]);
      W = warp_sum(W);
      const double goal = floor(static_cast<double>(a.u[r]) * static_cast<double>(W));
      unsigned long long target = goal > 0.0 ? static_cast<unsigned long long>(goal) : 0ull;
      if (target >= W) target = W - 1;
      unsigned long long run = 0;
      for (int j0 = 0; j0 < n; j0 += 32) {
        const int j = j0 + lane;
        const unsigned long long w = j < n ? static_cast<uint32_t>(li.vec[j]) : 0;
        const unsigned long long inc = run + warp_inclusive(w);
        if (target < inc && target >= inc - w) {
          const int id = static_cast<int>(~static_cast<uint32_t>(li.vec[j] >> 32));
          a.tokens[r] = id;
          if (a.logprobs) {
            const T* p = static_cast<const T*>(a.x.logits) + r * a.x.ld + id;
            const float z = Elem<T>::from_bits(Elem<T>::load_bits(p));
            a.logprobs[r] = (z == weight.zmax ? 0.0f : (z - weight.zmax) / temperature) -
                            logf(static_cast<float>(static_cast<double>(W) / kGrid));
          }
        }
        run = __shfl_sync(FULL, inc, 31);
      }
    }
    return;
  }

  // ---- the largest logit
  float m = neg_inff();
  st.each(st.a, st.b, [&](const uint4 (&x)[STEP], int) {
#pragma unroll
    for (int i = 0; i < STEP; ++i) m = max_nan(m, Elem<T>::vmax_nan(x[i]));
  });
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(FULL, m, o));
  if (lane == 0) sm.f[warp] = m;
  __syncthreads();
  m = sm.f[0];
  for (int w = 1; w < NW; ++w) m = max_nan(m, sm.f[w]);
  if (C > 1) {
    if (tid == 0) sm.cta_f = m;
    cl.sync();
    for (int c = 0; c < C; ++c) m = max_nan(m, *cl.map_shared_rank(&sm.cta_f, c));
    cl.sync();
  }
  if (m == neg_inff()) {  // nothing is allowed (the same for every CTA of the cluster)
    if (rank == 0 && tid == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = neg_inff();
    }
    return;
  }
  const float scale = 1.4426950408889634f / temperature;
  // NaN, infinite logits, an infinite temperature, a k past the lists: the exact row
  const bool cut_p = top_p < 1.0f;
  if (!(m <= 3.402823466e38f) || !(scale > 0.0f) || (top_k > 0 && top_k < a.x.vocab)) {
    exact();
    return;
  }
  Sampler<T, NT, MASK> sp{a, st, sm, cl, r, C, rank, temperature, min_p, Weight{m, scale}};
  unsigned long long own, before;
  // no vector below this logit has a token with a power of min_p: d < log2(min_p) by more than any rounding
  const float floor_d = min_p > 0.0f ? log2f(min_p) - 0.01f : -40.0f;
  const float reach = floor_d / scale;
  float least = m + (reach - fabsf(reach) * 1e-5f) - fabsf(m) * 1e-6f;
  if (!cut_p) {
    if (min_p > 0.0f) {
      auto keep = [&](float, float p, int) { return p >= min_p; };
      const unsigned long long mine = warp_sum(sp.kept_weights(st.a, st.b, least, keep));
      const unsigned long long total = sp.cluster_sum(mine, &own, &before);
      sp.pick(total, own, before, least, keep);
    } else {
      auto keep = [](float, float, int) { return true; };
      const unsigned long long total = sp.cluster_sum(warp_sum(sp.all_weights()), &own, &before);
      sp.pick(total, own, before, least, keep);
    }
    return;
  }

  // ---- top-p
  const unsigned long long W = sp.cluster_sum(warp_sum(sp.all_weights()), &own, &before);
  const double want = ceil(static_cast<double>(top_p) * static_cast<double>(W));
  const unsigned long long need = want >= 1.0 ? static_cast<unsigned long long>(want) : 1ull;
  // tokens below (W - need) / V together weigh no more than W - need: the prefix ends above them
  const float light = static_cast<float>(static_cast<double>(W - need) / a.x.vocab) * (1.0f / kGrid);
  const float depth = fminf(31.5f, light > 1e-12f ? 0.01f - log2f(light) : 31.5f);
  const float part_scale = kParts / depth;
  auto part_of = [&](float z) {  // of a token; kParts: below them all
    const float d = z == m ? 0.0f : (z - m) * scale;
    return min(static_cast<int>(-d * part_scale), kParts);
  };
  unsigned* lo = reinterpret_cast<unsigned*>(dyn);
  unsigned* hi = lo + kParts + 2;
  unsigned long long* list = reinterpret_cast<unsigned long long*>(dyn + kPartBytes);
  for (int i = tid; i < 2 * (kParts + 2); i += NT) lo[i] = 0;
  if (tid == 0) sm.n_edge = 0;
  __syncthreads();
  float low = m - (depth / scale) * 1.00001f - fabsf(m) * 1e-6f;  // nothing below has a part
  st.each(st.a, st.b, [&](const uint4 (&x)[STEP], int) {
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      if (!(Elem<T>::vmax(x[i]) >= low)) continue;
#pragma unroll
      for (int e = 0; e < Elem<T>::EPV; ++e) {
        const float z = Elem<T>::get(x[i], e);
        if (z >= low) {
          const float d = z == m ? 0.0f : (z - m) * scale;
          const int b = min(static_cast<int>(-d * part_scale), kParts);  // (one more part for what lies below)
          const unsigned w = __float2uint_rn(power2(d) * kGrid);
          // a part's sum in two words, the carry taken from the low one's old value: exact for any number of tokens
          // (a u32 pair of 15 + 16 bits wraps at 131072 tokens of weight 1)
          if (atomicAdd(&lo[b], w) > ~w) atomicAdd(&hi[b], 1u);
        }
      }
    }
  });
  if (C > 1) cl.sync();
  else __syncthreads();
  // the cluster's sums of the parts (where the lists will be)
  for (int b = tid; b < kParts; b += NT) {
    unsigned long long v = 0;
    for (int c = 0; c < C; ++c)
      v += cl.map_shared_rank(lo, c)[b] + (static_cast<unsigned long long>(cl.map_shared_rank(hi, c)[b]) << 32);
    list[b] = v;
  }
  __syncthreads();
  if (warp == 0) {  // lane l takes parts 32 l, 32 l + 1, ...
    unsigned long long sum = 0;
    for (int j = 0; j < kParts / 32; ++j) sum += list[lane * (kParts / 32) + j];
    const unsigned long long upto = warp_inclusive(sum);
    const unsigned hit = __ballot_sync(FULL, upto >= need);
    if (hit == 0) {
      if (lane == 0) sm.part = -1;
    } else if (lane == __ffs(hit) - 1) {
      unsigned long long run = upto - sum;
      int b = lane * (kParts / 32);
      while (run + list[b] < need) run += list[b++];
      sm.part = b;
      sm.above = run;
    }
  }
  if (C > 1) cl.sync();
  else __syncthreads();
  const int part = sm.part;
  const unsigned long long above = sm.above;
  if (part < 0) {
    exact();
    return;
  }
  // what lies above that part, per warp, and the part's own tokens
  float edge = m - ((part + 1) / part_scale / scale) * 1.00001f - fabsf(m) * 1e-6f;
  unsigned long long mine = 0;
  const float sure = m - ((part / part_scale) / scale) * 0.99999f + fabsf(m) * 1e-6f;  // above it no test is needed
  st.each(st.a, st.b, [&](const uint4 (&x)[STEP], int base) {
#pragma unroll
    for (int i = 0; i < STEP; ++i) {
      if (!(Elem<T>::vmax(x[i]) >= edge)) continue;
#pragma unroll
      for (int e = 0; e < Elem<T>::EPV; ++e) {
        const float z = Elem<T>::get(x[i], e);
        if (z < edge) continue;
        const int b = z > sure ? -1 : part_of(z);
        if (b < part) {
          const float p = sp.weight.power(z);
          if (p >= min_p) mine += __float2uint_rn(p * kGrid);
        } else if (b == part) {
          const int at = atomicAdd(&sm.n_edge, 1);
          if (at < kEdgeMost) list[at] = sp.order_key(z, st.index(base + 32 * i + lane, e));
        }
      }
    }
  });
  mine = warp_sum(mine);
  if (C > 1) cl.sync();
  else __syncthreads();
  int n = 0;
  for (int c = 0; c < C; ++c) n += *cl.map_shared_rank(&sm.n_edge, c);
  if (n > kEdgeMost) {
    exact();
    return;
  }
  // the whole part, sorted, in every CTA (behind the CTA's own tokens): where the prefix ends
  unsigned long long* all = C > 1 ? list + kEdgeMost : list;
  int at = 0;
  for (int c = 0; c < C && C > 1; ++c) {
    const int nc = *cl.map_shared_rank(&sm.n_edge, c);
    const unsigned long long* src = cl.map_shared_rank(list, c);
    for (int j = tid; j < nc; j += NT) all[at + j] = src[j];
    at += nc;
  }
  if (C > 1) cl.sync();
  else __syncthreads();
  const unsigned long long cut = cut_of<NT>(*reinterpret_cast<CutSmem*>(lo), all, n, need - above, [&](unsigned long long u) {
    return sp.weight.unit(Elem<float>::unkey(static_cast<uint32_t>(u >> 32)));
  });
  auto keep = [&](float z, float p, int id) {
    if (!(p >= min_p)) return false;
    const int b = part_of(z);
    return b < part || (b == part && sp.order_key(z, id) >= cut);
  };
  // kept tokens of the part go to their warps
  const int per = ((st.v1 - st.v0 + NT - 1) / NT) * 32;
  if (lane == 0) sm.sub[warp] = mine;
  __syncthreads();
  for (int j = tid; j < sm.n_edge; j += NT) {
    const unsigned long long u = list[j];
    const float z = Elem<float>::unkey(static_cast<uint32_t>(u >> 32));
    const float p = sp.weight.power(z);
    if (u >= cut && p >= min_p) {
      const int id = static_cast<int>(~static_cast<uint32_t>(u));
      const int v = (id + st.rv.off) / Elem<T>::EPV - st.v0;
      atomicAdd(&sm.sub[v / per], static_cast<unsigned long long>(__float2uint_rn(p * kGrid)));
    }
  }
  __syncthreads();
  mine = sm.sub[warp];
  const unsigned long long total = sp.cluster_sum(mine, &own, &before);
  sp.pick(total, own, before, edge, keep);
}

template <typename T>
cudaError_t launch(const SampleArgs& a, int num_sms, cudaStream_t s) {
  constexpr int NT = 512;
  const long long nvec = static_cast<long long>(a.x.vocab) * sizeof(T) / 16 + 2;
  // the lists of the k largest: for the k of all rows where it is one, for every k they can hold where rows have their own
  const int list_k = a.p.top_k ? kTopMax : std::min(std::max(a.p.top_k_all, 1), kTopMax);
  // More CTAs for a row while rows leave SMs without work, a lane keeps a step and the lists hold what all the CTAs may
  // collect (a row that spills takes the exact way: 32 x 131072 with rows' own k up to 1024 500 us with four CTAs, 91 with
  // two).  Two CTAs an SM in all: 64 x 150001 f32 top-p 68 us (one: 80, four: 103, always one a row: 125), 100 x 131072
  // uncut 27 (30, 32, 30); top-k alone would do with fewer (64 rows: 24, 19, 46, 18).
  int c = 1;
  auto more = [&] { return c < 8 && nvec / (c * 2) >= NT && c * 2 * list_k * 5 / 4 + 64 < top_el_cap(list_k); };
  while (more() && a.x.rows * c * 2 <= 2 * num_sms) c *= 2;
  size_t smem = (static_cast<size_t>(top_vec_cap(list_k)) + top_el_cap(list_k)) * 8;
  smem = std::max(smem, sizeof(ExactSmem));
  smem = std::max(smem, static_cast<size_t>(kPartBytes) + (c > 1 ? 2 : 1) * kEdgeMost * 8);
  auto kernel = a.mask ? sample_kernel<T, NT, true> : sample_kernel<T, NT, false>;
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_rows(kernel, NT, c, smem, a.x.rows, s, a, list_k);
}

}  // namespace

cudaError_t sample_launch(const SampleArgs& a, int num_sms, cudaStream_t s, uint64_t* launches) {
  if (a.x.rows == 0) return cudaSuccess;
  cudaError_t e = a.x.dtype == TBGB_F32   ? launch<float>(a, num_sms, s)
                  : a.x.dtype == TBGB_F16 ? launch<__half>(a, num_sms, s)
                                          : launch<__nv_bfloat16>(a, num_sms, s);
  if (e == cudaSuccess) (*launches)++;
  return e;
}

}  // namespace tbgb
