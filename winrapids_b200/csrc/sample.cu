// sample.cu -- one token per row from its logits, by temperature, top-k, top-p and min-p, from a
// given uniform number.
//
// With zmax the row's largest allowed logit, a token's weight is
//   w = 2^((z - zmax) * (log2(e) / T)),   rounded to a multiple of 2^-30,
// so weights are whole numbers (in units of 2^-30, at most 2^30 each) and every sum of them is
// exact: the token does not depend on the order of summation, on the split over CTAs or on the
// hardware.  The grid is finer than the numbers that pick (a 32-bit uniform number has steps of
// 2^-24) and than the rounding of a 32-bit running sum would be.
//   top-k   the first k by (logit descending, id ascending)
//   top-p   of those, with sum W, the shortest prefix whose sum reaches ceil(p W)
//   min-p   of those, the tokens with 2^(...) >= min_p
// Each cut keeps a prefix of the same order, so all of them together are one threshold: a key tau
// and how many of the tokens equal to it are kept (the lowest ids).  The token is the first, in the
// order of the ids, whose running sum exceeds floor(u W'), W' the sum of what is kept.
#include <climits>

#include "logits_select.cuh"

namespace tbgb {

namespace {

using namespace row;

constexpr float kGrid = 1073741824.0f;  // 2^30

struct Weight {
  float zmax, scale;
  __device__ __forceinline__ float power(float z) const { return z == zmax ? 1.0f : exp2f((z - zmax) * scale); }
  // 0 for -inf (and for the NaN of -inf at an infinite temperature)
  __device__ __forceinline__ unsigned unit(float z) const { return __float2uint_rn(power(z) * kGrid); }
  __device__ __forceinline__ unsigned long long operator()(float z) const { return unit(z); }
};

struct Share {  // one CTA's part of what is kept
  unsigned long long sure;  // weight beyond tau
  unsigned ties;            // tokens at tau
};

template <typename T, int NT, bool RES>
__global__ void __launch_bounds__(NT) sample_kernel(const SampleArgs a) {
  constexpr int NW = NT / 32;
  __shared__ SelectSmem sel;
  __shared__ float wm[NW], cta_max;
  __shared__ unsigned long long w_sure[NW], cta_sum;
  __shared__ unsigned w_ties[NW];
  __shared__ Share share;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const long long r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Slice<T, NT, RES> sl(static_cast<const T*>(a.x.logits) + r * a.x.ld, a.x.vocab,
                       a.mask ? a.mask + r * a.mask_ld : nullptr, rank, C);
  if (RES) {
    sl.load(0);
    sl.clean(0);
  }
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

template <typename T>
cudaError_t launch(const SampleArgs& a, int num_sms, cudaStream_t s) {
  const long long bytes = static_cast<long long>(a.x.vocab) * sizeof(T);
  constexpr int NT = 512;
  const int c = cluster_size(bytes, NT * NV * 16, a.x.rows, num_sms, NT);
  const bool res = static_cast<long long>(c) * NT * NV * 16 >= bytes + 32;
  if (res) return launch_rows(sample_kernel<T, NT, true>, NT, c, 0, a.x.rows, s, a);
  return launch_rows(sample_kernel<T, NT, false>, NT, c, 0, a.x.rows, s, a);
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
