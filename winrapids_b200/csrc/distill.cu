// distill.cu -- KL divergence of a student's softmax from a teacher known by its top logits, and
// its gradient by the student's logits.
//
// A row has K entries (id_i, t_i) of the teacher; S is the set of its ids (-1: no entry).
//   closed      p = softmax of t / T over the entries
//   with tail   p_i = exp(t_i / T - lse), lse the teacher's log-sum-exp over the whole vocabulary, and
//               one more outcome, "a token outside S", with p_r = 1 - sum p_i
//   q = softmax(z / T), q_r = the sum of q outside S (taken over those logits, not as 1 - q(S), which
//   loses everything when the student has learnt the entries)
//   loss = sum p_i (log p_i - log q_i) + p_r (log p_r - log q_r)
//   T dloss/dz_j = q_j - p_j in S,  q_j (1 - p_r / q_r) = q_j (p(S) - q(S)) / q_r outside
// A row whose student has no weight outside S, and one whose teacher has none there, have no such
// outcome.  stats[r] = (log sum exp(z / T), the factor of q_j outside S) is what the backward pass
// needs of the forward pass.
#include <climits>

#include "logits_row.cuh"

namespace tbgb {

namespace {

using namespace row;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float teacher_logit(const DistillArgs& a, long long i) {
  if (a.teacher_dtype == TBGB_F32) return static_cast<const float*>(a.teacher)[i];
  if (a.teacher_dtype == TBGB_F16) return __half2float(static_cast<const __half*>(a.teacher)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.teacher)[i]);
}

template <typename T>
__device__ __forceinline__ void store_elem(void* grad, long long i, float g) {
  const uint32_t b = Elem<T>::to_bits(g);
  if (sizeof(T) == 4)
    static_cast<uint32_t*>(grad)[i] = b;
  else
    static_cast<unsigned short*>(grad)[i] = static_cast<unsigned short>(b);
}

// g[0 .. EPV) into the gradient's row at the places of vector v: 16 bytes at once where the
// gradient's row starts at the same place between 16-byte boundaries as the logits' row.
template <typename T>
__device__ __forceinline__ void store_vector(const RowView<T>& rv, char* grad_base, bool same, T* grad_row, int v,
                                             const float* g) {
  constexpr int EPV = Elem<T>::EPV;
  if (same && rv.whole(v)) {
    uint4 o = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < EPV; ++e) Elem<T>::set(o, e, Elem<T>::to_bits(g[e]));
    __stcs(reinterpret_cast<uint4*>(grad_base) + v, o);
    return;
  }
  const int j0 = rv.first(v);
#pragma unroll
  for (int e = 0; e < EPV; ++e)
    if (j0 + e >= 0 && j0 + e < rv.vocab) store_elem<T>(grad_row, j0 + e, g[e]);
}

// The row's entries in shared memory: id (-1: none, also an id outside the vocabulary, which is
// reported), student logit (only of ids in [lo, hi), or of all when `all`), teacher probability.
struct Entries {
  int* id;
  float* z;
  float* p;
};

// Called by one warp: p of every entry and the sum of them.  log2p is left in `p` by the loader.
__device__ __forceinline__ float entry_probs(const DistillArgs& a, const Entries& en, long long r) {
  const int lane = threadIdx.x & 31;
  float sum = 0.0f;
  if (a.teacher_lse) {
    const double lse = a.teacher_lse[r];
    for (int k = lane; k < a.k; k += 32) {
      if (en.id[k] < 0) continue;
      const double x = static_cast<double>(en.p[k]) / a.temperature - lse;
      en.p[k] = exp2f(static_cast<float>(x) * kLog2e);
      sum += en.p[k];
    }
    return warp_sum(sum);
  }
  float m = neg_inff();
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) m = fmaxf(m, en.p[k]);
  m = warp_max(m);
  if (m == neg_inff()) {
    for (int k = lane; k < a.k; k += 32) en.p[k] = 0.0f;
    return 0.0f;
  }
  const float scale = kLog2e / a.temperature;
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) sum += exp2f((en.p[k] - m) * scale);
  sum = warp_sum(sum);
  const float l2 = log2f(sum);
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) en.p[k] = exp2f((en.p[k] - m) * scale - l2);
  return 1.0f;
}

struct Part {  // a CTA's part of the student's softmax
  float m;     // largest logit
  float out;   // sum outside S of 2^((z - m) * scale)
  float in;    // sum over S
};

// loss and stats, and with GRAD the gradient; one cluster per row.  GRAD needs RES.
template <typename T, int NT, bool RES, bool GRAD>
__global__ void __launch_bounds__(NT) distill_kernel(const DistillArgs a) {
  constexpr int NW = NT / 32, EPV = Elem<T>::EPV;
  extern __shared__ uint32_t smem[];
  __shared__ float w_m[NW], w_s[NW];
  __shared__ Part parts[8];
  __shared__ float p_sum;
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const long long r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* z_row = static_cast<const T*>(a.x.logits) + r * a.x.ld;
  T* g_row = GRAD ? static_cast<T*>(a.grad) + r * a.grad_ld : nullptr;
  Slice<T, NT, RES> sl(z_row, a.x.vocab, nullptr, rank, C);
  const bool same = GRAD && ((reinterpret_cast<uintptr_t>(g_row) ^ reinterpret_cast<uintptr_t>(z_row)) & 15) == 0;
  char* g_base = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(g_row) & ~static_cast<uintptr_t>(15));
  const float w = a.weight ? a.weight[r] : 1.0f;
  if (w == 0.0f) {  // a padding row: not read
    if (GRAD) {
      float zero[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) zero[e] = 0.0f;
      for (int v = sl.v0 + tid; v < sl.v1; v += NT) store_vector<T>(sl.rv, g_base, same, g_row, v, zero);
    }
    if (rank == 0 && tid == 0) {
      a.loss[r] = 0.0f;
      a.stats[2 * r] = 0.0f;
      a.stats[2 * r + 1] = 1.0f;
    }
    return;
  }
  if (RES) sl.load(0);

  // the entries; bit (vector - v0) * EPV + e marks an element of S in this CTA's slice
  Entries en;
  en.id = reinterpret_cast<int*>(smem);
  en.z = reinterpret_cast<float*>(smem) + a.k;
  en.p = en.z + a.k;
  uint32_t* bits = smem + 3 * a.k;
  const int n_words = ((sl.v1 - sl.v0) * EPV + 31) / 32;
  for (int i = tid; i < n_words; i += NT) bits[i] = 0;
  __syncthreads();
  const int lo = max(sl.rv.first(sl.v0), 0), hi = min(sl.rv.first(sl.v1), a.x.vocab);
  for (int k = tid; k < a.k; k += NT) {
    int id = a.ids[r * a.ids_ld + k];
    if (id < -1 || id >= a.x.vocab) {
      atomicOr(a.err, KERR_TOKEN_ID);
      id = -1;
    }
    en.id[k] = id;
    en.p[k] = id >= 0 ? teacher_logit(a, r * a.teacher_ld + k) : 0.0f;
    if (id >= 0 && (rank == 0 || (id >= lo && id < hi))) en.z[k] = Elem<T>::from_bits(Elem<T>::load_bits(z_row + id));
    if (id >= lo && id < hi) {
      const int b = id - sl.rv.first(sl.v0);
      if (atomicOr(&bits[b >> 5], 1u << (b & 31)) & (1u << (b & 31))) atomicOr(a.err, KERR_TOKEN_TWICE);
    }
  }
  __syncthreads();
  if (warp == 0) {
    const float s = entry_probs(a, en, r);
    if (lane == 0) p_sum = s;
  }

  // this CTA's softmax
  const float scale = kLog2e / a.temperature;
  float m_w = neg_inff(), s_w = 0.0f;
  for (int t = 0; t < sl.tiles; ++t) {
    if (!RES) sl.load(t);
    float m = neg_inff(), s = 0.0f;
    sl.each([&](float z, int, int) { m = fmaxf(m, z); });
    m = warp_max(m);
    const float ref = m == neg_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = sl.vec(t, i);
      if (i < sl.per && v < sl.v1) {
        const int b = (v - sl.v0) * EPV;
        const uint32_t in = bits[b >> 5] >> (b & 31);
#pragma unroll
        for (int e = 0; e < EPV; ++e) {
          const float x = exp2f((Elem<T>::get(sl.r[i], e) - ref) * scale);
          s += (in >> e) & 1u ? 0.0f : x;
        }
      }
    }
    s = warp_sum(s);
    MaxSum ms{m_w, s_w};
    ms.merge(m, s, scale);
    m_w = ms.m;
    s_w = ms.s;
  }
  if (lane == 0) {
    w_m[warp] = m_w;
    w_s[warp] = s_w;
  }
  __syncthreads();
  if (warp == 0) {
    MaxSum ms{lane < NW ? w_m[lane] : neg_inff(), lane < NW ? w_s[lane] : 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(FULL, ms.m, o), s2 = __shfl_xor_sync(FULL, ms.s, o);
      ms.merge(m2, s2, scale);
    }
    float in = 0.0f;
    const float ref = ms.m == neg_inff() ? 0.0f : ms.m;
    for (int k = lane; k < a.k; k += 32)
      if (en.id[k] >= lo && en.id[k] < hi) in += exp2f((en.z[k] - ref) * scale);
    in = warp_sum(in);
    if (lane < C) *cl.map_shared_rank(&parts[rank], lane) = Part{ms.m, ms.s, in};
  }
  cl.sync();
  float m = neg_inff(), s_out = 0.0f, s_in = 0.0f;
  for (int c = 0; c < C; ++c) m = fmaxf(m, parts[c].m);
  const float ref = m == neg_inff() ? 0.0f : m;
  for (int c = 0; c < C; ++c) {
    const Part p = parts[c];
    const float f = p.m == m ? 1.0f : exp2f((p.m - ref) * scale);
    s_out += p.m == neg_inff() ? p.out : p.out * f;  // (a NaN reaches the sums with a maximum of -inf too)
    s_in += p.m == neg_inff() ? p.in : p.in * f;
  }
  const float total = s_out + s_in, ps = p_sum;
  const bool tail = a.teacher_lse && ps < 1.0f && s_out > 0.0f;
  const float q_out = s_out / total;
  const float off = tail ? (ps - s_in / total) / q_out : 1.0f;

  if (rank == 0 && warp == 0) {
    const float l2 = log2f(total);
    float loss = 0.0f;
    for (int k = lane; k < a.k; k += 32) {
      if (en.id[k] < 0 || en.p[k] == 0.0f) continue;
      const float lp = a.teacher_lse ? static_cast<float>(static_cast<double>(teacher_logit(a, r * a.teacher_ld + k)) /
                                                              a.temperature - a.teacher_lse[r])
                                     : logf(en.p[k]);
      loss += en.p[k] * (lp - ((en.z[k] - ref) * scale - l2) * kLn2);
    }
    loss = warp_sum(loss);
    if (tail) {
      const float q_in = s_in / total;
      const float lq = q_in < 0.5f ? log1pf(-q_in) : logf(q_out);
      loss += (1.0f - ps) * (log1pf(-ps) - lq);
    }
    if (lane == 0) {
      a.loss[r] = loss;
      a.stats[2 * r] = m == neg_inff() ? neg_inff() + total : m / a.temperature + l2 * kLn2;
      a.stats[2 * r + 1] = off;
    }
  }
  if (!GRAD) return;

  const float wt = w / a.temperature, f = wt / total;
  const float f_off = f * off;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = sl.vec(0, i);
    if (i < sl.per && v < sl.v1) {
      float g[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) g[e] = exp2f((Elem<T>::get(sl.r[i], e) - ref) * scale) * f_off;
      store_vector<T>(sl.rv, g_base, same, g_row, v, g);
    }
  }
  __syncthreads();  // the entries' gradients go over what was just stored
  for (int k = tid; k < a.k; k += NT)
    if (en.id[k] >= lo && en.id[k] < hi)
      store_elem<T>(g_row, en.id[k], exp2f((en.z[k] - ref) * scale) * f - wt * en.p[k]);
}

// The gradient from a forward pass's stats: one CTA per tile of NT * NV vectors of a row.
template <typename T, int NT>
__global__ void __launch_bounds__(NT) distill_grad_kernel(const DistillArgs a, int tiles) {
  constexpr int EPV = Elem<T>::EPV;
  extern __shared__ uint32_t smem[];
  const long long r = blockIdx.x / tiles;
  const int rank = static_cast<int>(blockIdx.x - r * tiles);
  const int tid = threadIdx.x;
  const T* z_row = static_cast<const T*>(a.x.logits) + r * a.x.ld;
  T* g_row = static_cast<T*>(a.grad) + r * a.grad_ld;
  Slice<T, NT, true> sl(z_row, a.x.vocab, nullptr, rank, tiles);
  const bool same = ((reinterpret_cast<uintptr_t>(g_row) ^ reinterpret_cast<uintptr_t>(z_row)) & 15) == 0;
  char* g_base = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(g_row) & ~static_cast<uintptr_t>(15));
  const float w = a.weight[r];
  if (w == 0.0f) {
    float zero[EPV];
#pragma unroll
    for (int e = 0; e < EPV; ++e) zero[e] = 0.0f;
    for (int v = sl.v0 + tid; v < sl.v1; v += NT) store_vector<T>(sl.rv, g_base, same, g_row, v, zero);
    return;
  }
  sl.load(0);
  Entries en;
  en.id = reinterpret_cast<int*>(smem);
  en.z = reinterpret_cast<float*>(smem) + a.k;
  en.p = en.z + a.k;
  const int lo = max(sl.rv.first(sl.v0), 0), hi = min(sl.rv.first(sl.v1), a.x.vocab);
  for (int k = tid; k < a.k; k += NT) {
    int id = a.ids[r * a.ids_ld + k];
    if (id < -1 || id >= a.x.vocab) {
      atomicOr(a.err, KERR_TOKEN_ID);
      id = -1;
    }
    en.id[k] = id;
    en.p[k] = id >= 0 ? teacher_logit(a, r * a.teacher_ld + k) : 0.0f;
    if (id >= lo && id < hi) en.z[k] = Elem<T>::from_bits(Elem<T>::load_bits(z_row + id));
  }
  __syncthreads();
  if (tid < 32) entry_probs(a, en, r);
  const float inv_t = 1.0f / a.temperature, lse = a.stats[2 * r], off = a.stats[2 * r + 1];
  const float wt = w * inv_t, f_off = wt * off;
  auto q = [&](float z) { return exp2f((z * inv_t - lse) * kLog2e); };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = sl.vec(0, i);
    if (i < sl.per && v < sl.v1) {
      float g[EPV];
#pragma unroll
      for (int e = 0; e < EPV; ++e) g[e] = q(Elem<T>::get(sl.r[i], e)) * f_off;
      store_vector<T>(sl.rv, g_base, same, g_row, v, g);
    }
  }
  __syncthreads();
  for (int k = tid; k < a.k; k += NT)
    if (en.id[k] >= lo && en.id[k] < hi) store_elem<T>(g_row, en.id[k], wt * (q(en.z[k]) - en.p[k]));
}

template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes) {
  return bytes > 48 * 1024
             ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(bytes))
             : cudaSuccess;
}

template <typename T>
cudaError_t launch(const DistillArgs& a, bool with_loss, bool with_grad, int num_sms, cudaStream_t s,
                   uint64_t* launches) {
  constexpr int NT = 512;
  constexpr long long SLICE = NT * NV * 16;
  const long long bytes = static_cast<long long>(a.x.vocab) * sizeof(T);
  const size_t entries = static_cast<size_t>(a.k) * 12;
  cudaError_t e = cudaSuccess;
  if (with_loss) {
    const int c = cluster_size(bytes, SLICE, a.x.rows, num_sms, NT);
    const bool res = c * SLICE >= bytes + 32;
    const long long nvec = bytes / 16 + 2;
    const size_t smem = entries + ((nvec + c - 1) / c * Elem<T>::EPV + 31) / 32 * 4;
    auto kernel = res ? (with_grad ? distill_kernel<T, NT, true, true> : distill_kernel<T, NT, true, false>)
                      : distill_kernel<T, NT, false, false>;
    e = allow_smem(kernel, smem);
    if (e == cudaSuccess) e = launch_rows(kernel, NT, c, smem, a, a.x.rows, s);
    if (e != cudaSuccess) return e;
    (*launches)++;
    if (res || !with_grad) return e;
  }
  if (with_grad) {
    const int tiles = static_cast<int>((bytes + 32 + SLICE - 1) / SLICE);
    distill_grad_kernel<T, NT><<<static_cast<unsigned>(a.x.rows * tiles), NT, entries, s>>>(a, tiles);
    e = cudaGetLastError();
    if (e == cudaSuccess) (*launches)++;
  }
  return e;
}

}  // namespace

cudaError_t distill_launch(const DistillArgs& a, bool with_loss, bool with_grad, int num_sms, cudaStream_t s,
                           uint64_t* launches) {
  if (a.x.rows == 0) return cudaSuccess;
  return a.x.dtype == TBGB_F32   ? launch<float>(a, with_loss, with_grad, num_sms, s, launches)
         : a.x.dtype == TBGB_F16 ? launch<__half>(a, with_loss, with_grad, num_sms, s, launches)
                                 : launch<__nv_bfloat16>(a, with_loss, with_grad, num_sms, s, launches);
}

}  // namespace tbgb
