// top_logits.cu -- the K largest logits of every row with their ids, and the row's log-sum-exp.
//
//   values, ids   the K largest by (logit descending, id ascending); NaN, -inf and ids whose mask bit
//                 is clear are never taken, and a row with fewer ends in (-inf, -1)
//   lse           log sum exp(z / T) over the logits that are neither NaN nor masked
#include <climits>

#include "logits_select.cuh"

namespace tbgb {

namespace {

using namespace row;

template <typename T, int NT, bool RES>
__global__ void __launch_bounds__(NT) top_logits_kernel(const TopArgs a) {
  __shared__ SelectSmem sel;
  __shared__ unsigned long long list[kTopMax];
  __shared__ int n_list;
  __shared__ float wm[NT / 32], ws[NT / 32];
  __shared__ float2 cta_ms;
  __shared__ int warp_ties[NT / 32], cta_ties;
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
  if (tid == 0) n_list = 0;

  // log-sum-exp
  const float scale = 1.4426950408889634f / a.temperature;
  if (a.lse) {
    MaxSum ms{neg_inff(), 0.0f};
    for (int t = 0; t < sl.tiles; ++t) {
      sl.fetch(t);
      float m = neg_inff(), s = 0.0f;
      sl.each([&](float z, int, int) { m = fmaxf(m, z); });
      if (m > neg_inff()) sl.each([&](float z, int, int) { s += z == m ? 1.0f : exp2f((z - m) * scale); });
      ms.merge(m, s, scale);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(FULL, ms.m, o), s2 = __shfl_xor_sync(FULL, ms.s, o);
      ms.merge(m2, s2, scale);
    }
    if (lane == 0) {
      wm[warp] = ms.m;
      ws[warp] = ms.s;
    }
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < NT / 32; ++w) ms.merge(wm[w], ws[w], scale);
      cta_ms = make_float2(ms.m, ms.s);
    }
  }

  // the K-th largest
  int flip = 0;
  uint32_t tau = 0;
  unsigned long long above = 0;
  int ties_wanted = 0;
  if (radix_select(sl, cl, sel, flip, static_cast<unsigned long long>(a.k), CountOne(), tau, above))
    ties_wanted = a.k - static_cast<int>(above);
  else
    tau = Elem<T>::key(neg_inff());  // fewer than K: all of them

  if (a.lse && rank == 0 && tid == 0) {
    MaxSum ms{neg_inff(), 0.0f};
    for (int c = 0; c < C; ++c) {
      const float2 p = *cl.map_shared_rank(&cta_ms, c);
      ms.merge(p.x, p.y, scale);
    }
    a.lse[r] = ms.m == neg_inff() ? neg_inff() : ms.m / a.temperature + logf(ms.s);
  }

  // ties in front of this CTA
  int mine = 0;
  for (int t = 0; t < sl.tiles; ++t) {
    sl.fetch(t);
    sl.each([&](float z, int, int) { mine += z > neg_inff() && Elem<T>::key(z) == tau; });
  }
  mine = warp_sum(mine);
  if (lane == 0) warp_ties[warp] = mine;
  __syncthreads();
  if (tid == 0) {
    int s = 0;
    for (int w = 0; w < NT / 32; ++w) s += warp_ties[w];
    cta_ties = s;
  }
  cl.sync();
  int run = 0;
  for (int c = 0; c < rank; ++c) run += *cl.map_shared_rank(&cta_ties, c);

  unsigned long long* out = cl.map_shared_rank(list, 0);
  int* n_out = cl.map_shared_rank(&n_list, 0);
  auto push = [&](uint32_t k, int j) {
    const int at = atomicAdd(n_out, 1);
    if (at < kTopMax) out[at] = (static_cast<unsigned long long>(k) << 32) | static_cast<uint32_t>(~j);
  };
  for (int t = 0; t < sl.tiles; ++t) {
    sl.fetch(t);
    int n = 0;
    sl.each([&](float z, int, int) { n += z > neg_inff() && Elem<T>::key(z) == tau; });
    n = warp_sum(n);
    __syncthreads();
    if (lane == 0) warp_ties[warp] = n;
    __syncthreads();
    int at = run;
    for (int w = 0; w < warp; ++w) at += warp_ties[w];
    for (int w = 0; w < NT / 32; ++w) run += warp_ties[w];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i >= sl.per) break;
      int have = 0;
#pragma unroll
      for (int e = 0; e < Elem<T>::EPV; ++e) {
        const float z = Elem<T>::get(sl.r[i], e);
        have += z > neg_inff() && Elem<T>::key(z) == tau;
      }
      int before = warp_inclusive(have);
      const int all = __shfl_sync(FULL, before, 31);
      before += at - have;
      at += all;
#pragma unroll
      for (int e = 0; e < Elem<T>::EPV; ++e) {
        const float z = Elem<T>::get(sl.r[i], e);
        if (z > neg_inff()) {
          const uint32_t k = Elem<T>::key(z);
          if (k > tau || (k == tau && before++ < ties_wanted)) push(k, sl.index(t, i, e));
        }
      }
    }
  }
  cl.sync();
  if (rank != 0) return;

  // sort the list (at most K entries), largest first
  const int n = min(n_list, a.k);
  int n2 = 1;
  while (n2 < n) n2 <<= 1;
  for (int j = n + tid; j < n2; j += NT) list[j] = 0;
  __syncthreads();
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
  for (int j = tid; j < a.k; j += NT) {
    const bool have = j < n;
    const long long o = r * a.k + j;
    a.ids[o] = have ? static_cast<int>(~static_cast<uint32_t>(list[j])) : -1;
    const uint32_t bits = have ? Elem<T>::to_bits(Elem<T>::unkey(static_cast<uint32_t>(list[j] >> 32)))
                               : Elem<T>::NEG_INF;
    if (sizeof(T) == 4)
      static_cast<uint32_t*>(a.values)[o] = bits;
    else
      static_cast<unsigned short*>(a.values)[o] = static_cast<unsigned short>(bits);
  }
}

template <typename T>
cudaError_t launch(const TopArgs& a, int num_sms, cudaStream_t s) {
  const long long bytes = static_cast<long long>(a.x.vocab) * sizeof(T);
  constexpr int NT = 512;
  const int c = cluster_size(bytes, NT * NV * 16, a.x.rows, num_sms, NT);
  const bool res = static_cast<long long>(c) * NT * NV * 16 >= bytes + 32;
  if (res) return launch_rows(top_logits_kernel<T, NT, true>, NT, c, 0, a.x.rows, s, a);
  return launch_rows(top_logits_kernel<T, NT, false>, NT, c, 0, a.x.rows, s, a);
}

}  // namespace

cudaError_t top_logits_launch(const TopArgs& a, int num_sms, cudaStream_t s, uint64_t* launches) {
  if (a.x.rows == 0) return cudaSuccess;
  cudaError_t e = a.x.dtype == TBGB_F32   ? launch<float>(a, num_sms, s)
                  : a.x.dtype == TBGB_F16 ? launch<__half>(a, num_sms, s)
                                          : launch<__nv_bfloat16>(a, num_sms, s);
  if (e == cudaSuccess) (*launches)++;
  return e;
}

}  // namespace tbgb
