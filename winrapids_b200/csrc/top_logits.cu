// top_logits.cu -- the K largest logits of every row with their ids, and the row's log-sum-exp.
//
//   values, ids   the K largest by (logit descending, id ascending); NaN, -inf and ids whose mask bit
//                 is clear are never taken, and a row with fewer ends in (-inf, -1)
//   lse           log sum exp(z / T) over the logits that are neither NaN nor masked
//
// 165 us for the 64 largest of 2048 x 131072 bf16 (3.3 TB/s), 39 us for 20 of 509 x 50001 f32 (2.6 TB/s): bound by
// instructions (11.3 an element, 5 of them the softmax) and the fixed work per row, which four CTAs of 256
// threads an SM hide better than two of 512 (210 us).  A mask of its own per row takes the element-wise loads:
// 512 x 131072 bf16 52 us, masked 103.
#include <climits>

#include "logits_select.cuh"
#include "logits_stream.cuh"

namespace tbgb {

namespace {

using namespace row;

struct ExactSmem {
  SelectSmem sel;
  alignas(16) unsigned long long list[kTopMax];
  float wm[32], ws[32];
  float2 cta_ms;
  int warp_ties[32], cta_ties, n_list;
};

// A row by radix descent over the keys and the ids' order: right for any number of equal logits, NaN and
// infinities, at several passes over the row.  For rows that do not fit the lists below.
template <typename T, int NT>
__device__ __noinline__ void exact_row(const TopArgs& a, long long r, ExactSmem& sm) {
  constexpr bool RES = false;
  SelectSmem& sel = sm.sel;
  unsigned long long* list = sm.list;
  int& n_list = sm.n_list;
  float *wm = sm.wm, *ws = sm.ws;
  float2& cta_ms = sm.cta_ms;
  int *warp_ties = sm.warp_ties, &cta_ties = sm.cta_ties;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  Slice<T, NT, RES> sl(static_cast<const T*>(a.x.logits) + r * a.x.ld, a.x.vocab,
                       a.mask ? a.mask + r * a.mask_ld : nullptr, rank, C);
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

  const int n = min(n_list, a.k);
  sort_list<NT>(list, n);
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

// One cluster per row: the pass of collect_top carries the running maximum and sum of the softmax too,
// so the row is read once from HBM.
template <typename T, int NT, bool MASK>
__global__ void __launch_bounds__(NT, 1024 / NT) top_logits_kernel(const TopArgs a) {
  extern __shared__ __align__(16) char dyn[];
  __shared__ TopSmem sm;
  __shared__ float2 w_ms[NT / 32], cta_ms;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const long long r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  TopLists li;
  li.vec_cap = top_vec_cap(a.k);
  li.el_cap = top_el_cap(a.k);
  li.el = reinterpret_cast<unsigned long long*>(dyn);
  li.vec = li.el + li.el_cap;
  const Stream<T, NT, MASK> st(static_cast<const T*>(a.x.logits) + r * a.x.ld, a.x.vocab,
                               MASK ? a.mask + r * a.mask_ld : nullptr, rank, C);
  const float scale = 1.4426950408889634f / a.temperature;
  const float2 scale2 = make_float2(scale, scale);
  const bool with_lse = a.lse != nullptr;
  float m = neg_inff();
  float2 sum = make_float2(0.0f, 0.0f);
  collect_top<T, NT, MASK>(st, a.k, sm, li, [&](const uint4 (&x)[STEP], float top) {
    if (!with_lse) return;
    if (top > m) {  // the sum is scaled when the maximum rises
      const float f = m == neg_inff() ? 1.0f : power2((m - top) * scale);
      sum = mul2(sum, make_float2(f, f));
      m = top;
    }
    const float ref = m == neg_inff() ? 0.0f : m;
    const float2 minus_ref = make_float2(-ref, -ref);
#pragma unroll
    for (int i = 0; i < STEP; ++i)
#pragma unroll
      for (int j = 0; j < Elem<T>::PAIRS; ++j) sum = add2(sum, power2(Elem<T>::pair(x[i], j), minus_ref, scale2));
  });
  if (with_lse) {
    const float m_w = warp_max(m);
    const float s_w = warp_sum(m == neg_inff() || m == m_w ? sum.x + sum.y : (sum.x + sum.y) * power2((m - m_w) * scale));
    if (lane == 0) w_ms[warp] = make_float2(m_w, s_w);
    __syncthreads();
    if (tid == 0) {
      MaxSum ms{neg_inff(), 0.0f};
      for (int w = 0; w < NT / 32; ++w) ms.merge(w_ms[w].x, w_ms[w].y, scale);
      cta_ms = make_float2(ms.m, ms.s);
      if (!(ms.s < -neg_inff())) sm.spilled = 1;  // a NaN or an infinity: the exact row leaves NaN out
    }
  }
  cl.sync();
  bool any = false;
  int n = 0;
  for (int c = 0; c < C; ++c) {
    const TopSmem* peer = cl.map_shared_rank(&sm, c);
    any |= peer->spilled != 0;
    n += peer->n_el;
  }
  any |= n > li.el_cap;
  if (any) {  // the same for every CTA of the cluster
    cl.sync();
    exact_row<T, NT>(a, r, *reinterpret_cast<ExactSmem*>(dyn));
    return;
  }
  if (rank == 0) {
    if (with_lse && tid == 0) {
      MaxSum ms{neg_inff(), 0.0f};
      for (int c = 0; c < C; ++c) {
        const float2 p = *cl.map_shared_rank(&cta_ms, c);
        ms.merge(p.x, p.y, scale);
      }
      a.lse[r] = ms.m == neg_inff() ? neg_inff() : ms.m / a.temperature + logf(ms.s);
    }
    int at = sm.n_el;
    for (int c = 1; c < C; ++c) {
      const int nc = cl.map_shared_rank(&sm, c)->n_el;
      const unsigned long long* src = cl.map_shared_rank(li.el, c);
      for (int j = tid; j < nc; j += NT) li.el[at + j] = src[j];
      at += nc;
    }
  }
  if (C > 1) cl.sync();  // the lists have been read
  if (rank != 0) return;
  __syncthreads();
  n = prune_list<NT>(sm.bound, li.el, li.vec, &sm.n_vec, n, a.k);
  sort_list<NT>(li.el, n);
  for (int j = tid; j < a.k; j += NT) {
    const bool have = j < n;
    const long long o = r * a.k + j;
    const unsigned long long u = have ? li.el[j] : 0;
    a.ids[o] = have ? static_cast<int>(~static_cast<uint32_t>(u)) : -1;
    const uint32_t bits = have ? Elem<T>::to_bits(Elem<float>::unkey(static_cast<uint32_t>(u >> 32))) : Elem<T>::NEG_INF;
    if (sizeof(T) == 4)
      static_cast<uint32_t*>(a.values)[o] = bits;
    else
      static_cast<unsigned short*>(a.values)[o] = static_cast<unsigned short>(bits);
  }
}

template <typename T>
cudaError_t launch(const TopArgs& a, int num_sms, cudaStream_t s) {
  constexpr int NT = 256;
  const long long nvec = static_cast<long long>(a.x.vocab) * sizeof(T) / 16 + 2;
  // More CTAs for a row while rows leave SMs without work, a lane keeps a step and the lists hold them all: 60 x 50001 f32
  // 16 us (always one: 18, up to two or four an SM: 17, 24), 30 x 131072 bf16 with K 200 25 (31, 25, 25); 8 x 32000 bf16,
  // where the clusters' barriers cost as much as the rows, 14 (13).
  int c = 1;
  while (c < 8 && a.x.rows * c * 2 <= num_sms && nvec / (c * 2) >= NT && c * 2 * a.k * 5 / 4 + 64 < top_el_cap(a.k)) c *= 2;
  const size_t lists = (static_cast<size_t>(top_vec_cap(a.k)) + top_el_cap(a.k)) * 8;
  const size_t smem = lists > sizeof(ExactSmem) ? lists : sizeof(ExactSmem);
  auto kernel = a.mask ? top_logits_kernel<T, NT, true> : top_logits_kernel<T, NT, false>;
  const cudaError_t e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  return launch_rows(kernel, NT, c, smem, a.x.rows, s, a);
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
