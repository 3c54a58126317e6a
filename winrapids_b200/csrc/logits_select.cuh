// logits_select.cuh -- the K-th largest of a row, by count or by weight, over a cluster of CTAs.
#pragma once
#include "logits_row.cuh"

namespace tbgb {
namespace row {

struct SelectSmem {
  unsigned long long hist[2][256];
  unsigned long long comb[256];
  unsigned long long above;
  int bin;
};

// The largest key `tau` for which the sum over the elements with key >= tau reaches `target`
// (target >= 1); `above` is the sum over the keys beyond tau.  The sum counts elements, or adds
// weight(z).  False when the whole row does not reach the target.  Radix descent, 8 key bits a
// pass: each CTA of the cluster counts its slice into shared memory, every CTA adds the
// cluster's 256 counters and takes the same decision.  `flip` alternates the buffers between
// passes (one that a peer may still be reading is not cleared).
template <typename T, int NT, bool RES, typename W>
__device__ __forceinline__ bool radix_select(Slice<T, NT, RES>& sl, cg::cluster_group& cl, SelectSmem& sm, int& flip,
                                             unsigned long long target, W weight, uint32_t& tau,
                                             unsigned long long& above) {
  constexpr int KB = Elem<T>::KEY_BITS;
  const int tid = threadIdx.x, lane = tid & 31;
  const int C = static_cast<int>(cl.num_blocks());
  unsigned long long prefix = 0, over = 0;
  for (int shift = KB - 8; shift >= 0; shift -= 8) {
    unsigned long long* h = sm.hist[flip];
    flip ^= 1;
    for (int b = tid; b < 256; b += NT) h[b] = 0;
    __syncthreads();
    for (int t = 0; t < sl.tiles; ++t) {
      sl.fetch(t);
      sl.each([&](float z, int, int) {
        if (z > neg_inff()) {
          const unsigned long long k = Elem<T>::key(z);
          if ((k >> (shift + 8)) == prefix) atomicAdd(&h[(k >> shift) & 255], weight(z));
        }
      });
    }
    cl.sync();
    for (int b = tid; b < 256; b += NT) {
      unsigned long long v = 0;
      for (int c = 0; c < C; ++c) v += cl.map_shared_rank(h, c)[b];
      sm.comb[b] = v;
    }
    __syncthreads();
    if (tid < 32) {  // lane l holds bins 255 - 8 l ... 248 - 8 l, in that order
      unsigned long long part = 0;
      for (int j = 0; j < 8; ++j) part += sm.comb[255 - 8 * lane - j];
      const unsigned long long upto = warp_inclusive(part);
      const unsigned hit = __ballot_sync(FULL, over + upto >= target);
      if (hit == 0) {
        if (lane == 0) sm.bin = -1;
      } else if (lane == __ffs(hit) - 1) {
        unsigned long long run = over + upto - part;
        int b = 255 - 8 * lane;
        while (run + sm.comb[b] < target) run += sm.comb[b--];
        sm.bin = b;
        sm.above = run;
      }
    }
    __syncthreads();
    if (sm.bin < 0) return false;
    prefix = (prefix << 8) | static_cast<unsigned>(sm.bin);
    over = sm.above;
    __syncthreads();
  }
  tau = static_cast<uint32_t>(prefix);
  above = over;
  return true;
}

struct CountOne {
  __device__ __forceinline__ unsigned long long operator()(float) const { return 1ull; }
};

}  // namespace row
}  // namespace tbgb
