// logits_row.cuh -- a row of logits held by the threads of a cluster of CTAs, shared by the
// kernels of top_logits.cu, distill.cu and sample.cu.
//
// A row of V elements is cut into 16-byte vectors on 16-byte boundaries of the address space, so
// a row that starts anywhere (an odd vocabulary) is read with wide loads all the same: only its
// first and last vector can be partial, and their elements are read one by one.  A cluster of C
// CTAs takes one row; CTA c takes a contiguous slice of the vectors, warp w of it a contiguous
// part of that, so "in the order of the index" is the order (CTA, warp, vector row, lane, element).
#pragma once
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "common.cuh"
#include "logits.cuh"

namespace tbgb {
namespace row {

namespace cg = cooperative_groups;

constexpr int NV = 8;  // 16-byte vectors a thread holds
constexpr unsigned FULL = 0xffffffffu;

__device__ __forceinline__ float neg_inff() { return __uint_as_float(0xff800000u); }

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// ---- element types -------------------------------------------------------------------------
// KEY_BITS-bit ordered keys: k(a) < k(b) iff a < b, equal zeros, -inf lowest (NaN is replaced
// by -inf before keys are taken).

template <typename T>
struct Elem;

template <>
struct Elem<float> {
  static constexpr int EPV = 4, KEY_BITS = 32;
  static constexpr uint32_t NEG_INF = 0xff800000u;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    return __uint_as_float(e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w);
  }
  static __device__ __forceinline__ void set(uint4& v, int e, uint32_t bits) {
    (e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w) = bits;
  }
  static constexpr int PAIRS = 2;
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                  : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  }
  static __device__ __forceinline__ void set_pair(uint4& v, int i, float2 f) {
    (i == 0 ? v.x : v.z) = __float_as_uint(f.x);
    (i == 0 ? v.y : v.w) = __float_as_uint(f.y);
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ float vmax_nan(const uint4& v) {  // NaN when one is among them
    return max_nan(max_nan(__uint_as_float(v.x), __uint_as_float(v.y)), max_nan(__uint_as_float(v.z), __uint_as_float(v.w)));
  }
  static __device__ __forceinline__ uint32_t load_bits(const float* p) { return __float_as_uint(*p); }
  static __device__ __forceinline__ float from_bits(uint32_t b) { return __uint_as_float(b); }
  static __device__ __forceinline__ uint32_t to_bits(float f) { return __float_as_uint(f); }
  static __device__ __forceinline__ uint32_t no_nan(uint32_t w) {
    return __float_as_uint(fmaxf(__uint_as_float(w), neg_inff()));
  }
  static __device__ __forceinline__ uint32_t key(float z) {
    const uint32_t u = __float_as_uint(z + 0.0f);
    return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
  }
  static __device__ __forceinline__ float unkey(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
  }
};

template <typename T>
struct Elem16 {
  static constexpr int EPV = 8, KEY_BITS = 16, PAIRS = 4;
  static __device__ __forceinline__ uint32_t word(const uint4& v, int i) {
    return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  }
  static __device__ __forceinline__ void set(uint4& v, int e, uint32_t bits) {
    uint32_t& w = (e >> 1) == 0 ? v.x : (e >> 1) == 1 ? v.y : (e >> 1) == 2 ? v.z : v.w;
    w = (e & 1) ? (w & 0xffffu) | (bits << 16) : (w & 0xffff0000u) | bits;
  }
  static __device__ __forceinline__ uint32_t load_bits(const T* p) {
    return *reinterpret_cast<const unsigned short*>(p);
  }
  static __device__ __forceinline__ uint32_t key_of_bits(uint32_t b) {
    if (b == 0x8000u) b = 0;
    return (b & 0x8000u) ? (~b & 0xffffu) : (b | 0x8000u);
  }
  static __device__ __forceinline__ uint32_t bits_of_key(uint32_t k) {
    return (k & 0x8000u) ? (k & 0x7fffu) : (~k & 0xffffu);
  }
};

template <>
struct Elem<__nv_bfloat16> : Elem16<__nv_bfloat16> {
  static constexpr uint32_t NEG_INF = 0xff80u;
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = word(v, e >> 1);
    return __uint_as_float((e & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ void set_pair(uint4& v, int i, float2 f) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
    (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  static __device__ __forceinline__ float vmax_nan(const uint4& v) {
    const uint32_t m = max2_nan(max2_nan(v.x, v.y), max2_nan(v.z, v.w));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  static __device__ __forceinline__ float from_bits(uint32_t b) { return __uint_as_float(b << 16); }
  static __device__ __forceinline__ uint32_t to_bits(float f) {
    return __bfloat16_as_ushort(__float2bfloat16_rn(f));
  }
  static __device__ __forceinline__ uint32_t no_nan(uint32_t w) {
    __nv_bfloat162 x = *reinterpret_cast<__nv_bfloat162*>(&w);
    const uint32_t lo = 0xff80ff80u;
    x = __hmax2(x, *reinterpret_cast<const __nv_bfloat162*>(&lo));
    return *reinterpret_cast<uint32_t*>(&x);
  }
  static __device__ __forceinline__ uint32_t key(float z) { return key_of_bits(__float_as_uint(z) >> 16); }
  static __device__ __forceinline__ float unkey(uint32_t k) { return from_bits(bits_of_key(k)); }
};

template <>
struct Elem<__half> : Elem16<__half> {
  static constexpr uint32_t NEG_INF = 0xfc00u;
  static __device__ __forceinline__ float from_bits(uint32_t b) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(b)));
  }
  static __device__ __forceinline__ float2 pair(const uint4& v, int i) {
    const uint32_t w = word(v, i);
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
  }
  static __device__ __forceinline__ void set_pair(uint4& v, int i, float2 f) {
    const __half2 h = __floats2half2_rn(f.x, f.y);
    (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t max2_nan(uint32_t a, uint32_t b) {
    const __half2 h = __hmax2_nan(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float vmax(const uint4& v) {
    const uint32_t m = max2(max2(v.x, v.y), max2(v.z, v.w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return fmaxf(f.x, f.y);
  }
  static __device__ __forceinline__ float vmax_nan(const uint4& v) {
    const uint32_t m = max2_nan(max2_nan(v.x, v.y), max2_nan(v.z, v.w));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&m));
    return max_nan(f.x, f.y);
  }
  static __device__ __forceinline__ float get(const uint4& v, int e) {
    const uint32_t w = word(v, e >> 1);
    return from_bits((e & 1) ? (w >> 16) : (w & 0xffffu));
  }
  static __device__ __forceinline__ uint32_t to_bits(float f) { return __half_as_ushort(__float2half_rn(f)); }
  static __device__ __forceinline__ uint32_t no_nan(uint32_t w) {
    __half2 x = *reinterpret_cast<__half2*>(&w);
    const uint32_t lo = 0xfc00fc00u;
    x = __hmax2(x, *reinterpret_cast<const __half2*>(&lo));
    return *reinterpret_cast<uint32_t*>(&x);
  }
  static __device__ __forceinline__ uint32_t key(float z) { return key_of_bits(to_bits(z)); }
  static __device__ __forceinline__ float unkey(uint32_t k) { return from_bits(bits_of_key(k)); }
};

// ---- two 32-bit numbers at a time ------------------------------------------------------------
// Blackwell's packed f32 instructions do the softmax's subtraction, scaling and additions on two
// elements per issue slot, rounding each as the single instructions do.

__device__ __forceinline__ uint64_t pack2(float2 a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
  return unpack2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)));
  return unpack2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(a)), "l"(pack2(b)), "l"(pack2(c)));
  return unpack2(r);
}
// 2^x; results below 2^-126 are 0
__device__ __forceinline__ float power2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 2^((z - ref) * scale)
__device__ __forceinline__ float2 power2(float2 z, float2 minus_ref, float2 scale) {
  const float2 d = mul2(add2(z, minus_ref), scale);
  return make_float2(power2(d.x), power2(d.y));
}

// ---- a row's vectors -------------------------------------------------------------------------

template <typename T>
struct RowView {
  const char* base;  // the row's first element, rounded down to 16 bytes
  int off;           // elements between `base` and the row's first element
  int vocab;
  int nvec;  // vectors that hold at least one element of the row

  __device__ __forceinline__ RowView(const T* p, int v) : vocab(v) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(p);
    base = reinterpret_cast<const char*>(a & ~static_cast<uintptr_t>(15));
    off = static_cast<int>((a & 15) / sizeof(T));
    nvec = (off + v + Elem<T>::EPV - 1) / Elem<T>::EPV;
  }
  // index in the row of vector v's first element (negative in front of the row)
  __device__ __forceinline__ int first(int v) const { return v * Elem<T>::EPV - off; }
  __device__ __forceinline__ bool whole(int v) const {
    const int j = first(v);
    return j >= 0 && j + Elem<T>::EPV <= vocab;
  }
  // vector v; elements outside the row are -inf.  v < nvec.
  __device__ __forceinline__ uint4 load_whole(int v) const { return __ldcs(reinterpret_cast<const uint4*>(base) + v); }
  __device__ __forceinline__ uint4 load_part(int v) const {
    uint4 r = none();
    const T* e0 = reinterpret_cast<const T*>(base) + static_cast<long long>(v) * Elem<T>::EPV;
    const int j0 = first(v);
#pragma unroll
    for (int e = 0; e < Elem<T>::EPV; ++e)
      if (j0 + e >= 0 && j0 + e < vocab) Elem<T>::set(r, e, Elem<T>::load_bits(e0 + e));
    return r;
  }
  static __device__ __forceinline__ uint4 none() {
    constexpr uint32_t w = sizeof(T) == 4 ? Elem<T>::NEG_INF : Elem<T>::NEG_INF * 0x10001u;
    return make_uint4(w, w, w, w);
  }
};

// Elements whose mask bit is clear become -inf, NaN too.
template <typename T>
__device__ __forceinline__ void mask_vector(uint4& r, const RowView<T>& rv, int v, const uint64_t* mask) {
  constexpr int EPV = Elem<T>::EPV;
  r.x = Elem<T>::no_nan(r.x);
  r.y = Elem<T>::no_nan(r.y);
  r.z = Elem<T>::no_nan(r.z);
  r.w = Elem<T>::no_nan(r.w);
  if (!mask) return;
  const int j0 = rv.first(v);
  uint32_t bits = 0;
  if (rv.whole(v)) {
    const int sh = j0 & 63;
    uint64_t w = mask[j0 >> 6] >> sh;
    if (sh > 64 - EPV) w |= mask[(j0 >> 6) + 1] << (64 - sh);
    bits = static_cast<uint32_t>(w);
  } else {
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      const int j = j0 + e;
      if (j >= 0 && j < rv.vocab) bits |= static_cast<uint32_t>((mask[j >> 6] >> (j & 63)) & 1u) << e;
    }
  }
#pragma unroll
  for (int e = 0; e < EPV; ++e)
    if (!((bits >> e) & 1u)) Elem<T>::set(r, e, Elem<T>::NEG_INF);
}

// ---- a CTA's slice of a row -------------------------------------------------------------------
// RES: the whole slice is in registers (at most NT * NV vectors), every pass reads it there.
// Otherwise the slice is taken in tiles of NT * NV vectors that every pass loads again.

template <typename T, int NT, bool RES>
struct Slice {
  static constexpr int EPV = Elem<T>::EPV;
  static constexpr int TILE = NT * NV;
  RowView<T> rv;
  const uint64_t* mask;
  int v0, v1;  // the slice's vectors
  int tiles;
  int per;     // vector rows a warp takes of a tile (<= NV)
  uint4 r[NV];

  __device__ __forceinline__ Slice(const T* p, int vocab, const uint64_t* m, int rank, int C) : rv(p, vocab), mask(m) {
    const int each = (rv.nvec + C - 1) / C;
    v0 = min(rank * each, rv.nvec);
    v1 = min(v0 + each, rv.nvec);
    const int n = v1 - v0;
    tiles = RES ? 1 : (n + TILE - 1) / TILE;
    per = min((n + NT - 1) / NT, NV);
  }
  __device__ __forceinline__ int vec(int tile, int i) const {
    const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
    return v0 + tile * TILE + (w * per + i) * 32 + lane;
  }
  __device__ __forceinline__ void load(int tile) {
    // whole vectors lie between the row's first and last; each of those two is one thread's
    const int head = rv.off ? 1 : 0, tail = (rv.off + rv.vocab) % EPV ? rv.nvec - 1 : rv.nvec;
    const int end = min(v1, tail);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      r[i] = RowView<T>::none();
      const int v = vec(tile, i);
      if (i < per && v < end && v >= head) r[i] = rv.load_whole(v);
    }
    if (head && v0 == 0 && tile == 0 && threadIdx.x == 0 && v1 > 0) r[0] = rv.load_part(0);
    if (tail < v1) {  // (after a head that is the whole row: the same vector again)
      const uint4 last = vec(tile, 0) <= tail && vec(tile, per - 1) >= tail ? rv.load_part(tail) : RowView<T>::none();
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (i < per && vec(tile, i) == tail) r[i] = last;
    }
  }
  __device__ __forceinline__ void clean(int tile) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int v = vec(tile, i);
      if (i < per && v < v1) mask_vector<T>(r[i], rv, v, mask);
    }
  }
  __device__ __forceinline__ void fetch(int tile) {
    if (!RES) {
      load(tile);
      clean(tile);
    }
  }
  // f(z, i, e) for every held element of a tile (also those outside the row: z = -inf)
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i < per) {
#pragma unroll
        for (int e = 0; e < EPV; ++e) f(Elem<T>::get(r[i], e), i, e);
      }
    }
  }
  __device__ __forceinline__ int index(int tile, int i, int e) const { return rv.first(vec(tile, i)) + e; }
};

// ---- reductions ---------------------------------------------------------------------------------

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(FULL, v, o);
  return v;
}
__device__ __forceinline__ int warp_sum(int v) { return static_cast<int>(__reduce_add_sync(FULL, static_cast<unsigned>(v))); }

template <typename U>
__device__ __forceinline__ U warp_inclusive(U v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const U t = __shfl_up_sync(FULL, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// ---- the softmax's running maximum and sum, in base 2 -------------------------------------------
// Sums of 2^((z - m) * s) with m the largest z seen and s = log2(e) / T: z - m comes first, so a
// row of the type's lowest values has exponents of 0 and no product overflows.

struct MaxSum {
  float m, s;
  __device__ __forceinline__ void merge(float m2, float s2, float scale) {
    if (m2 == neg_inff() || m == neg_inff()) {  // one side is empty: its sum is 0 (or NaN, which stays)
      m = fmaxf(m, m2);
      s += s2;
      return;
    }
    const float top = fmaxf(m, m2);
    s = s * (m == top ? 1.0f : exp2f((m - top) * scale)) + s2 * (m2 == top ? 1.0f : exp2f((m2 - top) * scale));
    m = top;
  }
};

// ---- launch ----------------------------------------------------------------------------------------

struct ClusterLaunch {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  ClusterLaunch(int threads, int cluster, size_t smem, long long clusters, cudaStream_t s) {
    cfg.gridDim = dim3(static_cast<unsigned>(clusters * cluster));
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cluster;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
  }
};

// `clusters` clusters of `cluster` CTAs.
template <typename... P, typename... A>
cudaError_t launch_rows(void (*kernel)(P...), int threads, int cluster, size_t smem, long long clusters, cudaStream_t s,
                        const A&... args) {
  ClusterLaunch l(threads, cluster, smem, clusters, s);
  return cudaLaunchKernelEx(&l.cfg, kernel, args...);
}

// Lets `kernel` be launched with `smem` bytes of dynamic shared memory.  The limit belongs to the function, not to a
// context or a call: it is only ever set to the most that a CTA can have, so no host thread lowers it under another's
// launch.  (That it is set is kept per thread: setting it costs as long as a launch.)
template <typename... P>
cudaError_t allow_smem(void (*kernel)(P...), size_t smem) {
  if (smem <= 48 * 1024) return cudaSuccess;
  struct Set {
    void (*kernel)(P...);
    int device;
  };
  static thread_local Set last[8] = {};
  static thread_local unsigned next = 0;
  int device = 0, most = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  for (const Set& k : last)
    if (k.kernel == kernel && k.device == device) return cudaSuccess;
  cudaFuncAttributes fixed;
  e = cudaFuncGetAttributes(&fixed, kernel);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&most, cudaDevAttrMaxSharedMemoryPerBlockOptin, device);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             most - static_cast<int>(fixed.sharedSizeBytes));
  if (e == cudaSuccess) last[next++ % 8] = Set{kernel, device};
  return e;
}

// Clusters of a persistent kernel that the device holds at once.  A cluster lies within one GPC, so
// this is less than the SMs' room divided by its size (C = 8: 48 instead of 55), and one cluster
// more than it would run after the others: twice the time.
// (The answer for a kernel, cluster and memory size is kept per thread: asking costs as long as a launch.)
template <typename... P>
cudaError_t resident_clusters(void (*kernel)(P...), int threads, int cluster, size_t smem, int* n) {
  struct Asked {
    void (*kernel)(P...);
    int device, cluster;
    size_t smem;
    int n;
  };
  static thread_local Asked last[8] = {};
  static thread_local unsigned next = 0;
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  for (const Asked& k : last)
    if (k.kernel == kernel && k.device == device && k.cluster == cluster && k.smem == smem && k.n > 0) {
      *n = k.n;
      return cudaSuccess;
    }
  e = allow_smem(kernel, smem);
  if (e != cudaSuccess) return e;
  ClusterLaunch l(threads, cluster, smem, 1, nullptr);
  e = cudaOccupancyMaxActiveClusters(n, kernel, &l.cfg);
  if (e == cudaSuccess) last[next++ % 8] = Asked{kernel, device, cluster, smem, *n};
  return e;
}

}  // namespace row
}  // namespace tbgb
