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
// The sum outside S is carried by its own largest logit: however far below the entries it lies, log q_r and
// q_j / q_r are as exact as any.  A row whose student has no logit above -inf outside S, and one whose teacher
// has nothing there, have no such outcome: their loss is the sum over S alone, whose p sum to P = p(S), and
//   T dloss/dz_j = P q_j - p_j in S,  P q_j outside
// (P = 1 for a closed teacher with an entry, 0 without one).  stats[r] = (log sum exp(z / T), the factor of
// q_j outside S, 1 where the outcome is missing) is what the backward pass needs of the forward pass; P it
// takes from the record.  A log-sum-exp in 32 bits carries 2^-24 of its size into every q_j.  Stats of six add
// (z_in, c_in, z_out, c_out), which do not:
//   T dloss/dz_j = c_in 2^((z - z_in) log2(e) / T) - p_j in S,  c_out 2^((z - z_out) log2(e) / T) outside
#include <algorithm>
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

// log2 of p = exp(t / T - lse): the quotient's own rounding is put back, it would be the error of log p
__device__ __forceinline__ float tail_log2(float t, float lse, float temperature, float inv_t) {
  const float q = t * inv_t;
  const float rest = fabsf(q) < 1e30f ? fmaf(-q, temperature, t) * inv_t : 0.0f;
  return t == neg_inff() ? neg_inff() : (q - lse + rest) * kLog2e;
}

template <typename T>
__device__ __forceinline__ void store_elem(void* grad, long long i, float g) {
  const uint32_t b = Elem<T>::to_bits(g);
  if (sizeof(T) == 4)
    static_cast<uint32_t*>(grad)[i] = b;
  else
    static_cast<unsigned short*>(grad)[i] = static_cast<unsigned short>(b);
}

// The gradient's row.  Vectors go out 16 bytes at once where its first element lies at the same place
// between 16-byte boundaries as that of the logits' row (the usual case: the same strides).
template <typename T>
struct GradRow {
  T* row;
  char* base;
  bool same;

  __device__ __forceinline__ GradRow(T* g, const T* z)
      : row(g),
        base(reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(g) & ~static_cast<uintptr_t>(15))),
        same(((reinterpret_cast<uintptr_t>(g) ^ reinterpret_cast<uintptr_t>(z)) & 15) == 0) {}
  __device__ __forceinline__ void store(const RowView<T>& rv, int v, const uint4& g) const {
    if (same && rv.whole(v)) {
      __stcs(reinterpret_cast<uint4*>(base) + v, g);
      return;
    }
    const int j0 = rv.first(v);
#pragma unroll
    for (int e = 0; e < Elem<T>::EPV; ++e)
      if (j0 + e >= 0 && j0 + e < rv.vocab) store_elem<T>(row, j0 + e, Elem<T>::get(g, e));
  }
};

// ---- loss and stats, and the gradient, in one pass over the logits -----------------------------------
//
// For rows that the stages of a cluster of eight hold (222 KB a CTA for two of them: 227,000 32-bit or 454,000 16-bit
// logits); longer ones below take two passes.
// One cluster per row at a time, persistent over rows; CTA c holds its slice of a row in one of two
// stages of shared memory.  Warp roles:
//   producer   bulk-copies the slice of the next row as soon as its stage is free
//   entries    loads the record of the next row, takes the slice's entries out of the stage (their logits are
//              kept, their places become -inf, so the softmax's loop over the rest needs no test), and
//              when the row is done writes the loss and the entries' gradients
//   others     the running maximum and sum over the stage, the exchange of six numbers per CTA over
//              distributed shared memory, then the gradient from the stage
// The three overlap across rows and across the CTAs of an SM.  Bound by that chain per row (copy, entries, sums,
// exchange, gradient) with three CTAs an SM to hide it: 486 us for 4096 x 131072 bf16 with 64 entries (4.4 TB/s of the
// 2.15 GB that the step reads and writes), 131 us for the loss alone over 2048 x 100003 f16 (3.1 TB/s).

__device__ __forceinline__ float scaled(float m, float s, float top, float scale) {
  return m == neg_inff() || m == top ? s : s * power2((m - top) * scale);
}

// 1 / total and the factors are quotients right to 2 units of the last place: 1.2e-7 of a gradient that the powers of two
// leave with 2.4e-7 and more.
struct RowPart {  // a CTA's part of a row
  float m, s;     // largest logit outside S, sum of 2^((z - m) * scale)
  float ms, ss;   // the same over S
  float loss;     // sum p (log p - (z - ms) / T) over S
  float p;        // sum p over S
};

struct RowSum {
  float ref, total, s_in;  // largest logit of all (0 for none), the whole sum and S's by it
  float m_out, s_out;      // largest logit outside S, the sum there by that
  float loss, p;
};

// The row's sums from its parts, the same in every lane: lane c takes CTA c's part
// (a loop over them is a chain of latencies that stands between the two passes over a row).  LOSS: with the loss, which
// only the warp that writes it needs.
template <bool LOSS>
__device__ __forceinline__ RowSum row_sum(const RowPart* parts, int C, float scale) {
  const int lane = threadIdx.x & 31;
  RowPart p{neg_inff(), 0.0f, neg_inff(), 0.0f, 0.0f, 0.0f};
  if ((lane & 7) < C) p = parts[lane & 7];
  RowSum t;
  t.m_out = p.m;
  float m = p.ms;
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    t.m_out = fmaxf(t.m_out, __shfl_xor_sync(FULL, t.m_out, o));
    m = fmaxf(m, __shfl_xor_sync(FULL, m, o));
  }
  m = fmaxf(m, t.m_out);
  t.ref = m == neg_inff() ? 0.0f : m;
  t.s_out = scaled(p.m, p.s, t.m_out, scale);
  t.s_in = scaled(p.ms, p.ss, m, scale);
  t.p = p.p;
  t.loss = p.loss;
  if (LOSS && p.p > 0.0f && p.ms > neg_inff()) t.loss -= p.p * ((p.ms - t.ref) * scale * kLn2);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) {
    t.s_out += __shfl_xor_sync(FULL, t.s_out, o);
    t.s_in += __shfl_xor_sync(FULL, t.s_in, o);
    t.p += __shfl_xor_sync(FULL, t.p, o);
    if (LOSS) t.loss += __shfl_xor_sync(FULL, t.loss, o);
  }
  t.total = t.s_in + scaled(t.m_out, t.s_out, m, scale);
  if (LOSS) t.loss += t.p * log2f(t.total) * kLn2;
  return t;
}

// Whether "a token outside S" is one of the row's outcomes.
__device__ __forceinline__ bool rest_counts(const RowSum& t, bool with_tail) {
  return with_tail && t.p < 1.0f && t.m_out > neg_inff();
}
// P of a row without it; a closed teacher's p sum to 1 but for their rounding.
__device__ __forceinline__ float whole(const RowSum& t, bool with_tail) { return with_tail || t.p == 0.0f ? t.p : 1.0f; }

// Loss and stats, by one thread.
__device__ __forceinline__ void write_row(const DistillArgs& a, long long r, const RowSum& t, float scale) {
  float loss = t.loss, off = 1.0f;
  if (rest_counts(t, a.teacher_lse != nullptr)) {
    const float inv = __fdividef(1.0f, t.total), q_in = t.s_in * inv;
    const float q_out = scaled(t.m_out, t.s_out, t.ref, scale) * inv;
    // (the logarithms apart lose digits where they are near one another, and the quotient where it underflows)
    const float lq = q_in < 0.5f      ? log1pf(-q_in)
                     : q_out >= 1e-30f ? logf(q_out)
                                       : (t.m_out - t.ref) * scale * kLn2 + logf(t.s_out) - logf(t.total);
    loss += (1.0f - t.p) * (log1pf(-t.p) - lq);
    off = __fdividef(t.p - q_in, q_out);  // (to 2 units; an exact division in this chain costs the step 1 %)
    if (fabsf(off) > 3.402823466e38f) off = copysignf(3.402823466e38f, off);  // q_out below the type's range
    if (t.p == q_in) off = 0.0f;
  }
  a.loss[r] = loss;
  float* stats = a.stats + r * a.stats_ld;
  stats[0] = t.total > 0.0f ? t.ref / a.temperature + logf(t.total) : neg_inff() + t.total;
  stats[1] = off;
  if (a.stats_ld == 6) {
    const bool with_tail = a.teacher_lse != nullptr, rest = rest_counts(t, with_tail);
    const float inv = __fdividef(1.0f, t.total), P = whole(t, with_tail);
    stats[2] = t.ref;
    stats[3] = rest ? inv : P * inv;
    stats[4] = rest ? t.m_out : t.ref;
    stats[5] = rest ? __fdividef(t.p - t.s_in * inv, t.s_out) : P * inv;
  }
}

// The same of a padding row.
__device__ __forceinline__ void write_padding(const DistillArgs& a, long long r) {
  a.loss[r] = 0.0f;
  for (int i = 0; i < a.stats_ld; ++i) a.stats[r * a.stats_ld + i] = i == 1 ? 1.0f : 0.0f;
}

constexpr long long kWaitCycles = 4000000000ll;  // about 2 s

// A bounded wait of a whole warp (KERR_TIMEOUT when it gives up) that also acquires what other CTAs of the
// cluster wrote.  The answer is the same in every lane.
__device__ __forceinline__ bool wait_phase(uint64_t* bar, uint32_t parity, uint32_t* err) {
  const uint32_t at = smem_u32(bar);
  const long long t0 = clock64();  // (the global timer takes long to read)
  for (uint32_t it = 1;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(at), "r"(parity)
        : "memory");
    if (__all_sync(FULL, ok != 0)) return true;
    if ((it & 255u) == 0 && __any_sync(FULL, clock64() - t0 > kWaitCycles)) {
      if ((threadIdx.x & 31) == 0) atomicOr(err, KERR_TIMEOUT);
      return false;
    }
  }
}

// The softmax warps' barrier; true when one of them brings `failed`.
template <int NT>
__device__ __forceinline__ bool any_failed(bool failed) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, 1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(static_cast<uint32_t>(failed)), "n"(NT)
      : "memory");
  return r != 0;
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Six floats to `to` in CTA `cta` of the cluster, then an arrival on its barrier `bar`.
__device__ __forceinline__ void send_part(RowPart* to, uint64_t* bar, int cta, const RowPart& p) {
  uint32_t a, b;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(to)), "r"(cta));
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(smem_u32(bar)), "r"(cta));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(p.m), "f"(p.s) : "memory");
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a + 8), "f"(p.ms), "f"(p.ss) : "memory");
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a + 16), "f"(p.loss), "f"(p.p) : "memory");
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(b) : "memory");
}

// A CTA's slice of a row: vectors v0 .. v0 + nv, those in [w0, w1) of the slice whole.
template <typename T>
struct RowSlice {
  const T* z;
  RowView<T> rv;
  int v0, nv, w0, w1;

  __device__ __forceinline__ RowSlice(const DistillArgs& a, long long r, int rank, int log2c)
      : z(static_cast<const T*>(a.x.logits) + r * a.x.ld), rv(z, a.x.vocab) {
    const int each = (rv.nvec + (1 << log2c) - 1) >> log2c;
    v0 = min(rank * each, rv.nvec);
    nv = min(each, rv.nvec - v0);
    w0 = rv.off && v0 == 0 && nv > 0 ? 1 : 0;
    w1 = nv > 0 && (rv.off + rv.vocab) % Elem<T>::EPV && v0 + nv == rv.nvec ? nv - 1 : nv;
  }
  __device__ __forceinline__ const char* at(int j) const { return rv.base + static_cast<long long>(v0 + j) * 16; }
};

// Warps of the third role: what a warp does once a row (waits, reductions, the cluster's sums) is about 500 instructions,
// so few warps with many elements each do better (4096 x 131072 bf16: 4 warps 496 us, 6 557, 8 568, 12 658).
constexpr int kRingWarps = 4;
constexpr int kRingThreads = 32 * (kRingWarps + 2);  // and the producer's and the entries' warp

// KR: entries of the record per lane of the entries' warp.
template <typename T, int KR, bool GRAD>
__global__ void __launch_bounds__(kRingThreads, KR > 4 ? 1 : 3) distill_kernel(const DistillArgs a, int cap) {
  constexpr int EPV = Elem<T>::EPV, NW = kRingWarps, NT = 32 * NW;
  extern __shared__ __align__(16) char ring[];  // two stages of `cap` bytes
  // row n: index n & 1, phase (n >> 1) & 1
  __shared__ __align__(8) uint64_t full[2], done[2], ready[2], counted[2], heard[2];
  // four rows' parts: a peer may send row n + 1's while this CTA's entries' warp still reads row n - 1's
  __shared__ __align__(8) RowPart parts[4][8];
  __shared__ RowPart entries_part[2];
  __shared__ float2 w_ms[NW];
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank()), log2c = 31 - __clz(C);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const long long stride = gridDim.x >> log2c, rows = a.x.rows;
  const float scale = kLog2e / a.temperature, inv_t = 1.0f / a.temperature;
  const bool with_tail = a.teacher_lse != nullptr;
  if (tid == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&done[s], NW);
      mbar_init(&ready[s], 1);
      mbar_init(&counted[s], 1);
      mbar_init(&heard[s], C);
    }
    mbar_fence_init();
  }
  cl.sync();

  auto weight_of = [&](long long r) { return GRAD && r < rows ? a.weight[r] : 1.0f; };
  int n = 0;  // rows taken so far (padding rows are not counted)
  long long r = blockIdx.x >> log2c;
  float w = weight_of(r);

  if (warp == NW) {  // the producer
    for (; r < rows; r += stride) {
      const float next_w = weight_of(r + stride);
      if (w != 0.0f) {
        const int s = n & 1;
        if (n >= 2 && !wait_phase(&done[s], ((n >> 1) - 1) & 1, a.err)) break;
        const RowSlice<T> sl(a, r, rank, log2c);
        char* stage = ring + s * cap;
        // whole vectors by a bulk copy; the row's first and last vector, where partial, by elements
        if (lane == 0) {
          fence_proxy_async_smem();
          if (sl.w1 > sl.w0) {
            const uint32_t bytes = static_cast<uint32_t>(sl.w1 - sl.w0) * 16;
            asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[s])), "r"(bytes)
                         : "memory");
            bulk_g2s(stage + sl.w0 * 16, sl.at(sl.w0), bytes, &full[s]);
          }
        }
        for (int side = 0; side < 2; ++side) {
          const int j = side ? sl.nv - 1 : 0;
          if ((side ? sl.w1 == sl.nv : sl.w0 == 0) || lane >= EPV) continue;
          const int id = sl.rv.first(sl.v0 + j) + lane;
          const uint32_t bits = id >= 0 && id < sl.rv.vocab ? Elem<T>::load_bits(sl.z + id) : Elem<T>::NEG_INF;
          char* to = stage + j * 16 + lane * sizeof(T);
          if (sizeof(T) == 4)
            *reinterpret_cast<uint32_t*>(to) = bits;
          else
            *reinterpret_cast<unsigned short*>(to) = static_cast<unsigned short>(bits);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[s]);
        ++n;
      }
      w = next_w;
    }
    // no copy may be in flight when the CTA ends
    for (int k = max(n - 2, 0); k < n; ++k) wait_phase(&full[k & 1], (k >> 1) & 1, a.err);
  } else if (warp == NW + 1) {  // the entries
    struct Entry {
      int id;   // -1: none, or not in this CTA's slice
      float z;  // the student's logit
      float p;
      float l;  // log2 p
    };
    Entry now[KR], before[KR];
    int ahead_id[KR];
    float ahead_t[KR], ahead_lse = 0.0f;
    auto fetch = [&](long long row) {  // a row ahead of set(), so that nothing waits for it
      if (row >= rows) return;
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (lane + 32 * i < a.k) {
          ahead_id[i] = a.ids[row * a.ids_ld + lane + 32 * i];
          ahead_t[i] = teacher_logit(a, row * a.teacher_ld + lane + 32 * i);
        }
      if (with_tail) ahead_lse = a.teacher_lse[row];
    };
    auto set = [&](const RowSlice<T>& sl) {  // ids and p of the row that was fetched
      const int lo = max(sl.rv.first(sl.v0), 0), hi = min(sl.rv.first(sl.v0 + sl.nv), a.x.vocab);
      float t[KR], m = neg_inff(), sum = 0.0f;
#pragma unroll
      for (int i = 0; i < KR; ++i) {
        int id = lane + 32 * i < a.k ? ahead_id[i] : -1;
        if (id < -1 || id >= a.x.vocab) {
          if (rank == 0) atomicOr(a.err, KERR_TOKEN_ID);
          id = -1;
        }
        t[i] = id >= 0 ? ahead_t[i] : neg_inff();
        now[i].id = id >= lo && id < hi ? id : -1;
        m = fmaxf(m, t[i]);
      }
      if (with_tail) {
#pragma unroll
        for (int i = 0; i < KR; ++i) now[i].l = tail_log2(t[i], ahead_lse, a.temperature, inv_t);
      } else {
        m = warp_max(m);
        const float ref = m == neg_inff() ? 0.0f : m;
#pragma unroll
        for (int i = 0; i < KR; ++i) sum += power2((t[i] - ref) * scale);
        const float l2 = log2f(warp_sum(sum));
#pragma unroll
        for (int i = 0; i < KR; ++i) now[i].l = m == neg_inff() ? neg_inff() : (t[i] - ref) * scale - l2;
      }
#pragma unroll
      for (int i = 0; i < KR; ++i) now[i].p = power2(now[i].l);
    };
    long long last_r = -1;
    int last_n = 0;
    float last_w = 0.0f;
    auto finish = [&]() {  // loss, stats and the entries' gradients of the row before
      const int s = last_n & 1, phase = (last_n >> 1) & 1;
      if (!wait_phase(&heard[s], phase, a.err)) return false;
      const RowSum t = row_sum<true>(parts[last_n & 3], C, scale);
      if (rank == 0 && lane == 0) write_row(a, last_r, t, scale);
      if (!GRAD) return true;
      if (!wait_phase(&done[s], phase, a.err)) return false;  // over what the others have stored
      T* g = static_cast<T*>(a.grad) + last_r * a.grad_ld;
      const float wt = last_w * inv_t;
      const float q_factor = __fdividef(rest_counts(t, with_tail) ? 1.0f : whole(t, with_tail), t.total);
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (before[i].id >= 0)
          store_elem<T>(g, before[i].id, wt * (power2((before[i].z - t.ref) * scale) * q_factor - before[i].p));
      return true;
    };
    fetch(r);
    if (r < rows && w != 0.0f) set(RowSlice<T>(a, r, rank, log2c));
    fetch(r + stride);
    for (; r < rows; r += stride) {
      const float next_w = weight_of(r + stride);
      if (w != 0.0f) {
        const int s = n & 1, phase = (n >> 1) & 1;
        const RowSlice<T> sl(a, r, rank, log2c);
        const int f0 = sl.rv.first(sl.v0);
        if (!wait_phase(&full[s], phase, a.err)) break;
        T* stage = reinterpret_cast<T*>(ring + s * cap);
        auto put = [&](int j, uint32_t bits) {
          if (sizeof(T) == 4)
            reinterpret_cast<volatile uint32_t*>(stage)[j] = bits;
          else
            reinterpret_cast<volatile unsigned short*>(stage)[j] = static_cast<unsigned short>(bits);
        };
        // z out of the stage; k into its place, to see whether another entry has the same place; then -inf
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) now[i].z = Elem<T>::from_bits(Elem<T>::load_bits(stage + (now[i].id - f0)));
        __syncwarp();
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) put(now[i].id - f0, lane + 32 * i);
        __syncwarp();
        bool twice = false;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) twice |= Elem<T>::load_bits(stage + (now[i].id - f0)) != static_cast<uint32_t>(lane + 32 * i);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) put(now[i].id - f0, Elem<T>::NEG_INF);
        fence_proxy_async_smem();  // before the stage's next bulk copy
        __syncwarp();
        if (lane == 0) mbar_arrive(&ready[s]);
        if (twice) atomicOr(a.err, KERR_TOKEN_TWICE);
        float ms = neg_inff(), ss = 0.0f, loss = 0.0f, ps = 0.0f;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) ms = fmaxf(ms, now[i].z);
        ms = warp_max(ms);
        const float ref = ms == neg_inff() ? 0.0f : ms;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (now[i].id >= 0) {
            const float d = (now[i].z - ref) * scale;
            ss += power2(d);
            if (now[i].p != 0.0f) loss += now[i].p * ((now[i].l - d) * kLn2);
            ps += now[i].p;
          }
        ss = warp_sum(ss);
        loss = warp_sum(loss);
        ps = warp_sum(ps);
        if (lane == 0) {
          entries_part[s] = RowPart{neg_inff(), 0.0f, ms, ss, loss, ps};
          mbar_arrive(&counted[s]);
        }
        if (last_r >= 0 && !finish()) break;
#pragma unroll
        for (int i = 0; i < KR; ++i) before[i] = now[i];
        last_r = r;
        last_n = n;
        last_w = w;
        ++n;
      } else if (rank == 0 && lane == 0) {
        write_padding(a, r);
      }
      if (r + stride < rows && next_w != 0.0f) set(RowSlice<T>(a, r + stride, rank, log2c));
      fetch(r + 2 * stride);
      w = next_w;
    }
    if (last_r >= 0 && r >= rows) finish();
  } else {  // the softmax and the gradient
    const float2 scale2 = make_float2(scale, scale);
    bool ok = true;  // false once a wait of this warp gave up: it then only meets the others at their barrier
    for (; r < rows; r += stride) {
      const float next_w = weight_of(r + stride);
      const RowSlice<T> sl(a, r, rank, log2c);
      const GradRow<T> out(GRAD ? static_cast<T*>(a.grad) + r * a.grad_ld : nullptr, sl.z);
      if (w == 0.0f) {
        for (int j = tid; j < sl.nv; j += NT) out.store(sl.rv, sl.v0 + j, make_uint4(0, 0, 0, 0));
        w = next_w;
        continue;
      }
      const int s = n & 1, phase = (n >> 1) & 1, nv = sl.nv;
      const uint4* stage = reinterpret_cast<const uint4*>(ring + s * cap);
      ok = ok && wait_phase(&full[s], phase, a.err) && wait_phase(&ready[s], phase, a.err);

      // four vectors at a time; the sum is scaled when they raise the maximum
      float m = neg_inff();
      float2 sum = make_float2(0.0f, 0.0f);
      auto take = [&](const uint4 (&x)[4]) {
        float top = m;
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, Elem<T>::vmax(x[i]));
        if (top > m) {
          const float f = m == neg_inff() ? 1.0f : power2((m - top) * scale);
          sum = mul2(sum, make_float2(f, f));
          m = top;
        }
        const float ref = m == neg_inff() ? 0.0f : m;
        const float2 minus_ref = make_float2(-ref, -ref);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < Elem<T>::PAIRS; ++j) sum = add2(sum, power2(Elem<T>::pair(x[i], j), minus_ref, scale2));
      };
      int v = ok ? tid : nv;
      for (; v + 3 * NT < nv; v += 4 * NT) {
        const uint4 x[4] = {stage[v], stage[v + NT], stage[v + 2 * NT], stage[v + 3 * NT]};
        take(x);
      }
      if (v < nv) {
        uint4 x[4] = {stage[v], RowView<T>::none(), RowView<T>::none(), RowView<T>::none()};
#pragma unroll
        for (int i = 1; i < 4; ++i)
          if (v + i * NT < nv) x[i] = stage[v + i * NT];
        take(x);
      }
      __syncwarp();
      if (!GRAD && ok && lane == 0) mbar_arrive(&done[s]);
      const float m_w = warp_max(m);
      const float s_w = warp_sum(scaled(m, sum.x + sum.y, m_w, scale));
      if (lane == 0) w_ms[warp] = make_float2(m_w, s_w);
      if (any_failed<NT>(!ok)) break;  // every one of these warps, or none
      if (warp == 0) {
        const float2 ms = lane < NW ? w_ms[lane] : make_float2(neg_inff(), 0.0f);
        ok = wait_phase(&counted[s], phase, a.err);
        RowPart part = entries_part[s];
        part.m = ms.x;
#pragma unroll
        for (int o = NW > 8 ? 8 : 4; o > 0; o >>= 1) part.m = fmaxf(part.m, __shfl_xor_sync(FULL, part.m, o));
        part.s = scaled(ms.x, ms.y, part.m, scale);
#pragma unroll
        for (int o = NW > 8 ? 8 : 4; o > 0; o >>= 1) part.s += __shfl_xor_sync(FULL, part.s, o);
        if (ok && lane < C) send_part(&parts[n & 3][rank], &heard[s], lane, part);
      }
      ok = ok && wait_phase(&heard[s], phase, a.err);
      if (GRAD && ok) {
        const RowSum t = row_sum<false>(parts[n & 3], C, scale);
        const float inv = __fdividef(1.0f, t.total);
        const bool rest = rest_counts(t, with_tail);
        // outside S: 2^((z - m_out) scale) (p(S) - q(S)) / s_out, or P 2^((z - ref) scale) / total
        const float f = w * inv_t * (rest ? __fdividef(t.p - t.s_in * inv, t.s_out) : whole(t, with_tail) * inv);
        const float ref = rest ? t.m_out : t.ref;
        const float2 minus_ref = make_float2(-ref, -ref), f2 = make_float2(f, f);
        auto give = [&](const uint4& x) {
          uint4 g;
#pragma unroll
          for (int j = 0; j < Elem<T>::PAIRS; ++j)
            Elem<T>::set_pair(g, j, mul2(power2(Elem<T>::pair(x, j), minus_ref, scale2), f2));
          return g;
        };
        if (out.same) {
          // whole vectors at once, the row's partial ends by elements
          uint4* to = reinterpret_cast<uint4*>(out.base) + sl.v0;
          int v = tid + sl.w0;
          for (; v + 3 * NT < sl.w1; v += 4 * NT) {
            const uint4 x[4] = {stage[v], stage[v + NT], stage[v + 2 * NT], stage[v + 3 * NT]};
#pragma unroll
            for (int i = 0; i < 4; ++i) __stcs(to + v + i * NT, give(x[i]));
          }
          for (; v < sl.w1; v += NT) __stcs(to + v, give(stage[v]));
          if (tid == 0 && sl.w0 > 0) out.store(sl.rv, sl.v0, give(stage[0]));
          if (tid == NT - 1 && sl.w1 < nv && sl.w1 >= sl.w0) out.store(sl.rv, sl.v0 + nv - 1, give(stage[nv - 1]));
        } else {
          for (int v = tid; v < nv; v += NT) out.store(sl.rv, sl.v0 + v, give(stage[v]));
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&done[s]);
      }
      ++n;
      w = next_w;
    }
  }
  // peers may still send to this CTA, also after one of its waits gave up
  __syncwarp();
  cl.sync();
}

// The row's entries in shared memory: id (-1: none, also an id outside the vocabulary, which is reported), student
// logit (of ids in this CTA's part [lo, hi)), the teacher's logit, then p or log2 p.
struct Entries {
  int* id;
  float* z;
  float* p;
};

// Called by one warp: log2 p of every entry in the place of the teacher's logit (LOG), or p and, asked for, their sum.
template <bool LOG>
__device__ __forceinline__ float entry_probs(const DistillArgs& a, const Entries& en, long long r, bool with_sum) {
  const int lane = threadIdx.x & 31;
  float sum = 0.0f;
  if (a.teacher_lse) {
    const float lse = a.teacher_lse[r], inv_t = 1.0f / a.temperature;
    for (int k = lane; k < a.k; k += 32) {
      if (en.id[k] < 0) continue;
      const float l = tail_log2(en.p[k], lse, a.temperature, inv_t);
      en.p[k] = LOG ? l : power2(l);
      sum += en.p[k];
    }
    return with_sum ? warp_sum(sum) : 0.0f;
  }
  float m = neg_inff();
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) m = fmaxf(m, en.p[k]);
  m = warp_max(m);
  if (m == neg_inff()) {
    for (int k = lane; k < a.k; k += 32) en.p[k] = LOG ? neg_inff() : 0.0f;
    return 0.0f;
  }
  const float scale = kLog2e / a.temperature;
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) sum += exp2f((en.p[k] - m) * scale);
  sum = warp_sum(sum);
  const float l2 = log2f(sum);
  for (int k = lane; k < a.k; k += 32)
    if (en.id[k] >= 0) {
      const float l = (en.p[k] - m) * scale - l2;
      en.p[k] = LOG ? l : exp2f(l);
    }
  return 1.0f;
}

// Rows too long for the stages above: a cluster per row, the slices read in tiles, a bit per element of the
// slice for the entries; the gradient in a second pass over the slice.  512 x 524288 bf16: loss 356 us (1.5 TB/s), step
// 561 us (1.9 TB/s of what it reads and writes once): one CTA an SM, bound by its latencies.
template <typename T, int NT, bool GRAD>
__global__ void __launch_bounds__(NT) distill_wide_kernel(const DistillArgs a) {
  constexpr int NW = NT / 32, EPV = Elem<T>::EPV;
  extern __shared__ uint32_t smem[];
  __shared__ float w_m[NW], w_s[NW];
  __shared__ __align__(8) RowPart parts[8];
  cg::cluster_group cl = cg::this_cluster();
  const int C = static_cast<int>(cl.num_blocks()), rank = static_cast<int>(cl.block_rank());
  const long long r = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* z_row = static_cast<const T*>(a.x.logits) + r * a.x.ld;
  Slice<T, NT, false> sl(z_row, a.x.vocab, nullptr, rank, C);
  const GradRow<T> out_row(GRAD ? static_cast<T*>(a.grad) + r * a.grad_ld : nullptr, z_row);
  const float w = GRAD ? a.weight[r] : 1.0f;
  if (w == 0.0f) {  // a padding row: not read
    for (int v = sl.v0 + tid; v < sl.v1; v += NT) out_row.store(sl.rv, v, make_uint4(0, 0, 0, 0));
    if (rank == 0 && tid == 0) write_padding(a, r);
    return;
  }
  cl.sync();  // every CTA of the cluster runs: their shared memory is written below

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
    if (id >= lo && id < hi) {
      en.z[k] = Elem<T>::from_bits(Elem<T>::load_bits(z_row + id));
      const int b = id - sl.rv.first(sl.v0);
      if (atomicOr(&bits[b >> 5], 1u << (b & 31)) & (1u << (b & 31))) atomicOr(a.err, KERR_TOKEN_TWICE);
    }
  }
  __syncthreads();
  if (warp == 0) entry_probs<true>(a, en, r, false);

  // this CTA's softmax outside S
  const float scale = kLog2e / a.temperature;
  float m_w = neg_inff(), s_w = 0.0f;
  auto fetch = [&](int t) {  // a tile, S's places -inf
    sl.load(t);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = sl.vec(t, i);
      if (i < sl.per && v < sl.v1) {
        const int b = (v - sl.v0) * EPV;
        const uint32_t in = (bits[b >> 5] >> (b & 31)) & ((1u << EPV) - 1);
        if (in) {
#pragma unroll
          for (int e = 0; e < EPV; ++e)
            if ((in >> e) & 1u) Elem<T>::set(sl.r[i], e, Elem<T>::NEG_INF);
        }
      }
    }
  };
  for (int t = 0; t < sl.tiles; ++t) {
    fetch(t);
    float m = neg_inff(), s = 0.0f;
    sl.each([&](float z, int, int) { m = fmaxf(m, z); });
    m = warp_max(m);
    const float ref = m == neg_inff() ? 0.0f : m;
    sl.each([&](float z, int, int) { s += exp2f((z - ref) * scale); });
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
    MaxSum out{lane < NW ? w_m[lane] : neg_inff(), lane < NW ? w_s[lane] : 0.0f};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float m2 = __shfl_xor_sync(FULL, out.m, o), s2 = __shfl_xor_sync(FULL, out.s, o);
      out.merge(m2, s2, scale);
    }
    float ms = neg_inff(), ss = 0.0f, loss = 0.0f, ps = 0.0f;
    for (int k = lane; k < a.k; k += 32)
      if (en.id[k] >= lo && en.id[k] < hi) ms = fmaxf(ms, en.z[k]);
    ms = warp_max(ms);
    const float ref = ms == neg_inff() ? 0.0f : ms;
    for (int k = lane; k < a.k; k += 32)
      if (en.id[k] >= lo && en.id[k] < hi) {
        const float d = (en.z[k] - ref) * scale, p = power2(en.p[k]);
        ss += power2(d);
        if (p != 0.0f) loss += p * ((en.p[k] - d) * kLn2);
        ps += p;
      }
    ss = warp_sum(ss);
    loss = warp_sum(loss);
    ps = warp_sum(ps);
    if (lane < C) *cl.map_shared_rank(&parts[rank], lane) = RowPart{out.m, out.s, ms, ss, loss, ps};
  }
  cl.sync();
  const RowSum sum = row_sum<true>(parts, C, scale);
  if (rank == 0 && tid == 0) write_row(a, r, sum, scale);
  if (!GRAD) return;
  const bool with_tail = a.teacher_lse != nullptr, rest = rest_counts(sum, with_tail);
  const float wt = w / a.temperature, inv = 1.0f / sum.total, P = whole(sum, with_tail);
  const float f = wt * (rest ? (sum.p - sum.s_in * inv) / sum.s_out : P * inv);
  const float ref = rest ? sum.m_out : sum.ref;
  const float2 minus_ref = make_float2(-ref, -ref), scale2 = make_float2(scale, scale), f2 = make_float2(f, f);
  for (int t = 0; t < sl.tiles; ++t) {
    fetch(t);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = sl.vec(t, i);
      if (i < sl.per && v < sl.v1) {
        uint4 g;
#pragma unroll
        for (int j = 0; j < Elem<T>::PAIRS; ++j)
          Elem<T>::set_pair(g, j, mul2(power2(Elem<T>::pair(sl.r[i], j), minus_ref, scale2), f2));
        out_row.store(sl.rv, v, g);
      }
    }
  }
  __syncthreads();
  const float q_factor = (rest ? 1.0f : P) * inv;
  for (int k = tid; k < a.k; k += NT)
    if (en.id[k] >= lo && en.id[k] < hi)
      store_elem<T>(out_row.row, en.id[k], wt * (power2((en.z[k] - sum.ref) * scale) * q_factor - power2(en.p[k])));
}

// The gradient from a forward pass's stats: one CTA per tile of NT * NV vectors of a row, held in registers.  90 us
// for 1024 x 50001 f32 with 100 entries (4.6 TB/s), 75 with 8: the stores wait behind a barrier for the entries (the barrier is
// the largest stall); 239 us with single-number arithmetic and element-wise stores.  FULL: six stats a row, 85 us.
template <typename T, int NT, bool FULL>
__global__ void __launch_bounds__(NT, 1024 / NT) distill_grad_kernel(const DistillArgs a, int tiles) {
  constexpr int NS = FULL ? 6 : 2;
  extern __shared__ uint32_t smem[];
  __shared__ float p_sum, stat[NS];
  const long long r = blockIdx.x / tiles;
  const int rank = static_cast<int>(blockIdx.x - r * tiles);
  const int tid = threadIdx.x;
  const T* z_row = static_cast<const T*>(a.x.logits) + r * a.x.ld;
  T* g_row = static_cast<T*>(a.grad) + r * a.grad_ld;
  Slice<T, NT, true> sl(z_row, a.x.vocab, nullptr, rank, tiles);
  const GradRow<T> out(g_row, z_row);
  const float w = a.weight[r];
  if (w == 0.0f) {
    for (int v = sl.v0 + tid; v < sl.v1; v += NT) out.store(sl.rv, v, make_uint4(0, 0, 0, 0));
    return;
  }
  if (tid >= NT - NS) stat[tid - (NT - NS)] = a.stats[NS * r + tid - (NT - NS)];  // (the first threads have entries to fetch)
  sl.load(0);
  Entries en;
  en.id = reinterpret_cast<int*>(smem);
  en.z = reinterpret_cast<float*>(smem) + a.k;
  en.p = en.z + a.k;
  const int lo = max(sl.rv.first(sl.v0), 0), hi = min(sl.rv.first(sl.v1), a.x.vocab);
  int some = 0;  // an entry above -inf
  for (int k = tid; k < a.k; k += NT) {
    int id = a.ids[r * a.ids_ld + k];
    if (id < -1 || id >= a.x.vocab) {
      atomicOr(a.err, KERR_TOKEN_ID);
      id = -1;
    }
    en.id[k] = id;
    en.p[k] = id >= 0 ? teacher_logit(a, r * a.teacher_ld + k) : 0.0f;
    some |= id >= 0 && !(en.p[k] == neg_inff());
    if (id >= lo && id < hi) en.z[k] = Elem<T>::from_bits(Elem<T>::load_bits(z_row + id));
  }
  if (FULL || a.teacher_lse)
    __syncthreads();
  else
    some = __syncthreads_or(some);
  const float inv_t = 1.0f / a.temperature, wt = w * inv_t;
  // outside S: f 2^e, e = (z - z_out) log2(e) / T, or (z / T + c) log2(e)
  float c, f, f_in;  // and f_in, the factor of q_j in S
  const float scale = kLog2e / a.temperature;
  if (FULL) {
    if (tid < 32) entry_probs<false>(a, en, r, false);
    c = -stat[NS - 2];
    f = wt * stat[NS - 1];
    f_in = stat[NS - 3];
  } else {
    float off = stat[1];
    const bool missing = off == 1.0f;  // the outcome outside S (where it is there, P is 1 but for its rounding)
    const float P = tid < 32 ? entry_probs<false>(a, en, r, missing) : 0.0f;
    if (missing) {  // the same for the whole CTA; a closed teacher's P is known without the sum
      off = some ? 1.0f : 0.0f;
      if (a.teacher_lse) {
        if (tid == 0) p_sum = P;
        __syncthreads();
        off = p_sum;
      }
    }
    // where the factor is large, q_j underflows before their product does: it is formed in the exponent
    const bool fold = !(fabsf(off) < 1024.0f);
    c = fold ? logf(fabsf(off)) - stat[0] : -stat[0];
    f = fold ? copysignf(wt, off) : wt * off;
    f_in = missing ? off : 1.0f;
  }
  const float2 c2 = make_float2(c, c), f2 = make_float2(f, f), inv2 = make_float2(inv_t, inv_t);
  const float u = FULL ? scale : kLog2e;
  const float2 u2 = make_float2(u, u);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int v = sl.vec(0, i);
    if (i < sl.per && v < sl.v1) {
      uint4 g;
#pragma unroll
      for (int j = 0; j < Elem<T>::PAIRS; ++j) {
        const float2 z = Elem<T>::pair(sl.r[i], j);
        const float2 d = mul2(FULL ? add2(z, c2) : fma2(z, inv2, c2), u2);
        Elem<T>::set_pair(g, j, mul2(make_float2(power2(d.x), power2(d.y)), f2));
      }
      out.store(sl.rv, v, g);
    }
  }
  __syncthreads();
  for (int k = tid; k < a.k; k += NT)
    if (en.id[k] >= lo && en.id[k] < hi) {
      const float e = FULL ? (en.z[k] - stat[NS - 4]) * scale : fmaf(en.z[k], inv_t, -stat[0]) * kLog2e;
      store_elem<T>(g_row, en.id[k], wt * (f_in * power2(e) - en.p[k]));
    }
}

template <typename T>
cudaError_t launch(const DistillArgs& a, bool with_loss, bool with_grad, int num_sms, cudaStream_t s,
                   uint64_t* launches) {
  const long long bytes = static_cast<long long>(a.x.vocab) * sizeof(T);
  if (with_loss) {
    // The fewest CTAs whose two stages leave room for three CTAs on an SM: 4096 x 131072 bf16 step 484 us (as many as fit one
    // CTA: 746), 2048 x 100003 f16 loss 129 (room for two: 150, for one: 170); 600 x 50001 f32 would do with two (54, not 61).
    // More while rows are few, up to two CTAs an SM in all: 64 x 32000 bf16 step 7.7 us (never: 7.9, up to four: 10.4).
    const bool aligned = reinterpret_cast<uintptr_t>(a.x.logits) % 16 == 0 && a.x.ld * sizeof(T) % 16 == 0;
    const long long nvec = aligned ? (bytes + 15) / 16 : bytes / 16 + 2;
    int c = 1;
    while (c < 8 && 2 * ((nvec + c - 1) / c * 16) > 72 * 1024) c *= 2;
    while (c < 8 && a.x.rows * c * 2 <= 2 * num_sms && nvec / (c * 2) >= 128) c *= 2;
    const long long cap = (nvec + c - 1) / c * 16;
    if (2 * cap <= 222 * 1024) {
      const size_t smem = static_cast<size_t>(2 * cap);
      // Entries stay in the registers of their warp, 4 a lane, or 32 for long records, which leaves room for one CTA an SM:
      // 512 x 131072 bf16 step with K 64 69 us (in the kernel for 32: 429), K 128 73 (485), K 129 483, K 1024 978.
      auto kernel = a.k <= 128 ? (with_grad ? distill_kernel<T, 4, true> : distill_kernel<T, 4, false>)
                               : (with_grad ? distill_kernel<T, 32, true> : distill_kernel<T, 32, false>);
      int held = 0;
      cudaError_t e = allow_smem(kernel, smem);
      if (e == cudaSuccess) e = resident_clusters(kernel, kRingThreads, c, smem, &held);
      if (e == cudaSuccess)
        e = launch_rows(kernel, kRingThreads, c, smem, std::min(a.x.rows, static_cast<long long>(std::max(held, 1))), s,
                        a, static_cast<int>(cap));
      if (e == cudaSuccess) (*launches)++;
      return e;
    }
    constexpr int NT = 512;
    const size_t wide = static_cast<size_t>(a.k) * 12 + ((nvec + c - 1) / c * Elem<T>::EPV + 31) / 32 * 4;
    auto kernel = with_grad ? distill_wide_kernel<T, NT, true> : distill_wide_kernel<T, NT, false>;
    cudaError_t e = allow_smem(kernel, wide);
    if (e == cudaSuccess) e = launch_rows(kernel, NT, c, wide, a.x.rows, s, a);
    if (e == cudaSuccess) (*launches)++;
    return e;
  }
  constexpr int NT = 512;
  constexpr long long TILE = NT * NV * 16;
  const int tiles = static_cast<int>((bytes + 32 + TILE - 1) / TILE);
  auto kernel = a.stats_ld == 6 ? distill_grad_kernel<T, NT, true> : distill_grad_kernel<T, NT, false>;
  kernel<<<static_cast<unsigned>(a.x.rows * tiles), NT, static_cast<size_t>(a.k) * 12, s>>>(a, tiles);
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) (*launches)++;
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
