// chm_likelihood.cuh -- softmax rows over the profile logits of a signal
// group: log probabilities of given entries with entropy and top entries,
// their gradient, and distillation from a teacher's listed entries.
//
// Notation: z the row's logits, x = (z - m) / T * log2(e) <= 0 with m the
// row's maximum, e = 2^x, s = sum e. Entries that are masked or -inf count as
// -inf throughout. z - m is formed before the scaling, so logits near the
// type's largest or lowest value neither overflow nor lose the row.
#pragma once

#include <cstdint>

#include "chm_likelihood.h"

namespace chm {
namespace lk {

__device__ __forceinline__ float neg_inf() { return __int_as_float(0xff800000); }
__device__ __forceinline__ float quiet_nan() { return __int_as_float(0x7fffffff); }

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T to_type(float v);
template <> __device__ __forceinline__ float to_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 to_type<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <> __device__ __forceinline__ __half to_type<__half>(float v) { return __float2half_rn(v); }

// 2^x; subnormal results are 0, which no sum or gradient here notices
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------ 16-byte vectors
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y);
    f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]),
                      __float_as_uint(f[3]));
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)),
                 fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = reinterpret_cast<const uint32_t&>(h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ void unpack(const uint4& r, float (&f)[8]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 v = __half22float2(h[i]);
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = reinterpret_cast<const uint32_t&>(h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  static __device__ __forceinline__ float max(const uint4& r) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};

// Writes -inf over element E of a vector.
template <typename T, int E> __device__ __forceinline__ void drop(uint4& r) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&r);
  if constexpr (sizeof(T) == 4) {
    w[E] = Vec<T>::kNegInf;
  } else if constexpr (E % 2 == 0) {
    w[E / 2] = (w[E / 2] & 0xffff0000u) | (Vec<T>::kNegInf & 0xffffu);
  } else {
    w[E / 2] = (w[E / 2] & 0xffffu) | (Vec<T>::kNegInf & 0xffff0000u);
  }
}
// -inf over the elements whose bit is set
template <typename T, int E = 0> __device__ __forceinline__ void drop_bits(uint4& r, uint32_t b) {
  if constexpr (E < Vec<T>::N) {
    if ((b >> E) & 1u) drop<T, E>(r);
    drop_bits<T, E + 1>(r, b);
  }
}

// One row of the launch. Its entries are seen as 16-byte vectors of the
// aligned granules they lie in: entry v is element (v + ph) % N of vector
// (v + ph) / N, so any start address reads and writes full vectors but for
// the two at the ends, which go element by element and stay inside the row.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* z;
  const uint8_t* mask;
  T* grad;
  int size, ph, nvec;
  long long index;
  bool vec_store;                 // the gradient's rows lie in their granules alike

  __device__ __forceinline__ Row(const Rows& a, unsigned r) {
    const unsigned n = r / (unsigned)a.ng, g = r - n * (unsigned)a.ng;
    z = static_cast<const T*>(a.z) + n * a.row_stride + a.off[g];
    mask = a.mask ? a.mask + n * a.mask_stride + a.moff[g] : nullptr;
    grad = a.grad ? static_cast<T*>(a.grad) + n * a.grad_stride + a.goff[g] : nullptr;
    size = a.size[g];
    index = (long long)n * a.n_groups + a.g0 + g;
    ph = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    nvec = size ? (size + ph + N - 1) / N : 0;
    vec_store = ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  }
  __device__ __forceinline__ float at(int v) const {
    return (mask && !mask[v]) ? neg_inf() : to_float(z[v]);
  }
  // vector j; entries that do not take part, and places outside the row, are -inf
  __device__ __forceinline__ uint4 load(int j) const {
    const int v0 = j * N - ph;
    uint4 r;
    if (v0 >= 0 && v0 + N <= size) {
      asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                   : "l"(z + v0));
    } else {
      uint32_t w[4] = {Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf};
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int v = v0 + e;
        if (v < 0 || v >= size) continue;
        if constexpr (sizeof(T) == 4) {
          w[e] = reinterpret_cast<const uint32_t*>(z)[v];
        } else {
          const uint32_t h = reinterpret_cast<const uint16_t*>(z)[v];
          w[e / 2] = e % 2 ? (w[e / 2] & 0xffffu) | (h << 16) : (w[e / 2] & 0xffff0000u) | h;
        }
      }
      r = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (mask) drop_bits<T>(r, masked(v0));
    return r;
  }
  // bits of the elements that the mask takes out
  __device__ __forceinline__ uint32_t masked(int v0) const {
    uint32_t b = 0;
    if (v0 >= 0 && v0 + N <= size && (reinterpret_cast<uintptr_t>(mask + v0) & (N - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) {
        const uint32_t w = reinterpret_cast<const uint32_t*>(mask + v0)[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) b |= ((w >> (8 * e)) & 0xffu) ? 0u : 1u << (4 * i + e);
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const int v = v0 + e;
        if (v >= 0 && v < size && !mask[v]) b |= 1u << e;
      }
    }
    return b;
  }
  __device__ __forceinline__ void store(int j, const float (&d)[N]) const {
    const int v0 = j * N - ph;
    if (vec_store && v0 >= 0 && v0 + N <= size) {
      *reinterpret_cast<uint4*>(grad + v0) = Vec<T>::pack(d);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (v0 + e >= 0 && v0 + e < size) grad[v0 + e] = to_type<T>(d[e]);
    }
  }
};

// ------------------------------------------------------------ teams
// The threads that work on one row in one block: a warp of a block of four
// (kThreads = 32), or the whole block, of which up to eight in a cluster
// share a row. Every reduction runs in a fixed order.
template <int kThreads> struct Team {
  static constexpr int kWarps = kThreads / 32;
  static constexpr int kPerBlock = kThreads == 32 ? 4 : 1;
  static constexpr int kBlock = kThreads * kPerBlock;
  static __device__ __forceinline__ int tid() { return threadIdx.x % kThreads; }
  static __device__ __forceinline__ int lane() { return threadIdx.x & 31; }
  static __device__ __forceinline__ int warp() { return tid() >> 5; }
  static __device__ __forceinline__ int slot() { return threadIdx.x / kThreads; }
  static __device__ __forceinline__ void sync() {
    if constexpr (kThreads == 32) __syncwarp(); else __syncthreads();
  }
  // sum over the team of a count, through a slot per warp
  static __device__ __forceinline__ int sum(int v, int* red) {
    v = __reduce_add_sync(0xffffffffu, v);
    if constexpr (kThreads == 32) return v;
    __syncthreads();
    if (lane() == 0) red[warp()] = v;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) s += red[w];
    return s;
  }
};

__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}
// Shared-memory address of `p` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t remote(const void* p, int rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ void remote_store(uint32_t a, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}
__device__ __forceinline__ void remote_store(uint32_t a, unsigned long long v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}

constexpr int kMaxCluster = 8;

// The vectors of one block of a row's cluster: [begin, end), in chunks of
// kThreads * kVecs that a team holds in registers. Rows that fit one chunk
// per block are read from memory once, whatever the passes over them.
struct Share {
  int begin, end;
  __device__ __forceinline__ Share(int nvec, int rank, int blocks) {
    const int per = (nvec + blocks - 1) / blocks;
    begin = min(rank * per, nvec);
    end = min(begin + per, nvec);
  }
};

// Running maximum m, s = sum 2^x and t = sum x 2^x with x = (z - m) c.
struct Sums {
  float m, s, t;
};
// Joins two; a side without entries has m = -inf and s = t = 0, and the clamp
// keeps 0 * inf out. NaN in either s stays.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b, float c) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf((a.m - m) * c, -1000.f), db = fmaxf((b.m - m) * c, -1000.f);
  const float fa = ex2(da), fb = ex2(db);
  return {m, fa * a.s + fb * b.s, fa * (a.t + da * a.s) + fb * (b.t + db * b.s)};
}
// Adds a vector set of known maximum to the running sums.
template <typename T, int kVecs, bool kEntropy>
__device__ __forceinline__ void accumulate(const uint4 (&r)[kVecs], float top, float c, Sums& a) {
  constexpr int N = Vec<T>::N;
  if (top > a.m) {                            // a.m = -inf: nothing to rescale yet
    if (a.m != neg_inf()) {
      const float d = fmaxf((a.m - top) * c, -1000.f), f = ex2(d);
      if (kEntropy) a.t = f * (a.t + d * a.s);
      a.s *= f;
    }
    a.m = top;
  }
  const float ref = a.m == neg_inf() ? 0.f : a.m;
  float s[2] = {0.f, 0.f}, t[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float f[N];
    Vec<T>::unpack(r[i], f);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = (f[e] - ref) * c, p = ex2(x);
      s[e & 1] += p;
      if (kEntropy) t[e & 1] = fmaf(p, fmaxf(x, -1000.f), t[e & 1]);
    }
  }
  a.s += s[0] + s[1];
  if (kEntropy) a.t += t[0] + t[1];
}

// Joins the team's sums (every thread gets the result).
template <int kThreads>
__device__ __forceinline__ Sums team_sums(Sums a, float c, Sums* red) {
  using Tm = Team<kThreads>;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums b{__shfl_xor_sync(0xffffffffu, a.m, o), __shfl_xor_sync(0xffffffffu, a.s, o),
                 __shfl_xor_sync(0xffffffffu, a.t, o)};
    a = join(a, b, c);
  }
  if constexpr (kThreads == 32) return a;
  if (Tm::lane() == 0) red[Tm::warp()] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int w = 1; w < Tm::kWarps; ++w) a = join(a, red[w], c);
  return a;
}

// ------------------------------------------------------------ top entries
// Order of the entries: larger logit first, then the lower index. A logit's
// key is 0 where it has no probability.
__device__ __forceinline__ uint32_t logit_key(float z) {
  if (!(z > neg_inf())) return 0u;
  const uint32_t b = __float_as_uint(z + 0.f);        // -0 orders as +0
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t b) {
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7fffffffu) : ~b);
}
__device__ __forceinline__ unsigned long long order_key(uint32_t key, int v) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ int key_index(unsigned long long key) {
  return (int)(0xffffffffu - (unsigned)key);
}

// Descending bitonic sort of one value per lane.
__device__ __forceinline__ uint32_t warp_sort(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const uint32_t o = __shfl_xor_sync(0xffffffffu, v, j);
      v = (((lane & j) == 0) == ((lane & k) == 0)) ? max(v, o) : min(v, o);
    }
  return v;
}

constexpr int kMaxCand = 512;      // entries that pass the bound of a block's top entries

template <int kThreads> struct TopShared {
  uint32_t sorted[Team<kThreads>::kWarps][32];
  unsigned long long cand[kMaxCand];
  int count;
  int red[Team<kThreads>::kWarps];
};

// Calls f(z, v) for every entry of the chunk that this thread holds.
template <typename T, int kThreads, int kVecs, typename F>
__device__ __forceinline__ void each_entry(const Row<T>& row, const uint4 (&r)[kVecs], int base,
                                           int end, F f) {
  constexpr int N = Vec<T>::N;
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int j = base + i * kThreads + Team<kThreads>::tid();
    if (j >= end) continue;
    float z[N];
    Vec<T>::unpack(r[i], z);
#pragma unroll
    for (int e = 0; e < N; ++e) f(z[e], j * N - row.ph + e);
  }
}

template <typename T, int kThreads, int kVecs>
__device__ __forceinline__ void load_chunk(const Row<T>& row, const Share& sh, int base,
                                           uint4 (&r)[kVecs]) {
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    const int j = base + i * kThreads + Team<kThreads>::tid();
    if (j < sh.end) r[i] = row.load(j);
    else r[i] = make_uint4(Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf, Vec<T>::kNegInf);
  }
}

// The share's k largest entries, in no order, into sh.cand; returns their
// number (at least k of them are there unless the share has fewer).
//
// Each thread has the maximum of its entries. With the maxima of a warp
// sorted, min over the warps of the ceil(k / warps)-th is a value that at
// least k entries reach, and so is the k-th of any one warp; every entry at
// or above the larger of the two is a candidate. On entries in no order that
// leaves about 2k of them (measured 1.1k to 2.5k). Rows that defeat the bound
// (many equal logits, sorted rows) are counted instead: bisection for the
// k-th largest logit, then for the index up to which its equals belong.
template <typename T, int kThreads, int kVecs>
__device__ int collect_top(const Row<T>& row, const Share& share, uint4 (&r)[kVecs], float top,
                           int k, TopShared<kThreads>& sh) {
  using Tm = Team<kThreads>;
  constexpr int kChunk = kThreads * kVecs;
  const bool one = share.end - share.begin <= kChunk;
  if (Tm::tid() == 0) sh.count = 0;
  const uint32_t mine = warp_sort(logit_key(top));
  sh.sorted[Tm::warp()][Tm::lane()] = mine;
  Tm::sync();
  const int each = (k + Tm::kWarps - 1) / Tm::kWarps;
  uint32_t low = 0xffffffffu, high = 0u;
#pragma unroll
  for (int w = 0; w < Tm::kWarps; ++w) {
    low = min(low, each <= 32 ? sh.sorted[w][each - 1] : 0u);
    high = max(high, k <= 32 ? sh.sorted[w][k - 1] : 0u);
  }
  const uint32_t bound = max(low, high);
  const float least = bound ? key_logit(bound) : neg_inf();
  for (int base = share.begin; base < share.end; base += kChunk) {
    if (!one) load_chunk<T, kThreads, kVecs>(row, share, base, r);
    if (one && top < least) continue;
    each_entry<T, kThreads>(row, r, base, share.end, [&](float z, int v) {
      if (z >= least && z > neg_inf()) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kMaxCand) sh.cand[at] = order_key(logit_key(z), v);
      }
    });
  }
  Tm::sync();
  if (sh.count <= kMaxCand) return sh.count;

  // how many entries have a key of at least q (of exactly q up to index v, with `equal`)
  auto count = [&](uint32_t q, bool equal, int last) {
    int n = 0;
    for (int base = share.begin; base < share.end; base += kChunk) {
      if (!one) load_chunk<T, kThreads, kVecs>(row, share, base, r);
      each_entry<T, kThreads>(row, r, base, share.end, [&](float z, int v) {
        const uint32_t key = logit_key(z);
        n += equal ? key == q && v <= last : key >= q;
      });
    }
    return Tm::sum(n, sh.red);
  };
  uint32_t lo = max(bound, 1u), hi = 0xffffffffu;      // count(lo) >= k > count(hi)
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (count(mid, false, 0) >= k) lo = mid; else hi = mid;
  }
  const int need = k - count(hi, false, 0);
  int first = -1, last = row.size - 1;                 // equals up to `last`: at least `need`
  while (last - first > 1) {
    const int mid = first + (last - first) / 2;
    if (count(lo, true, mid) >= need) last = mid; else first = mid;
  }
  Tm::sync();
  if (Tm::tid() == 0) sh.count = 0;
  Tm::sync();
  for (int base = share.begin; base < share.end; base += kChunk) {
    if (!one) load_chunk<T, kThreads, kVecs>(row, share, base, r);
    each_entry<T, kThreads>(row, r, base, share.end, [&](float z, int v) {
      const uint32_t key = logit_key(z);
      if (key > lo || (key == lo && v <= last)) sh.cand[atomicAdd(&sh.count, 1)] = order_key(key, v);
    });
  }
  Tm::sync();
  return sh.count;
}

// Place of a key among `n` different ones, the largest first.
__device__ __forceinline__ int rank_of(unsigned long long key, const unsigned long long* keys,
                                       int n) {
  int r = 0;
  for (int i = 0; i < n; ++i) r += keys[i] > key;
  return r;
}

// ------------------------------------------------------- log probabilities
template <int kThreads> struct ScoreShared {
  Sums red[Team<kThreads>::kWarps];
  TopShared<kThreads> top;
};
// What the other blocks of a row's cluster send to the first.
template <int kBlocks> struct ScoreCluster {
  float sums[kBlocks][4];
  unsigned long long keys[kBlocks][kMaxTop];
};

// One pass over the row for maximum, sum and entropy, the top entries from
// the registers, and the given entries by a gather at the end.
template <typename T, int kThreads, int kVecs, int kMinBlocks>
__global__ void __launch_bounds__(Team<kThreads>::kBlock, kMinBlocks)
log_probs_kernel(const __grid_constant__ Rows a, const ScoreArgs o, unsigned rows, int blocks) {
  using Tm = Team<kThreads>;
  constexpr int kChunk = kThreads * kVecs;
  __shared__ ScoreShared<kThreads> shared[Tm::kPerBlock];
  __shared__ ScoreCluster<kThreads >= 256 ? kMaxCluster : 1> cl;
  ScoreShared<kThreads>& sh = shared[Tm::slot()];
  const unsigned r0 = blockIdx.x / blocks * Tm::kPerBlock + Tm::slot();
  const int rank = blockIdx.x % blocks;
  if (kThreads == 32 && r0 >= rows) return;            // a whole warp, and no cluster
  if (blocks > 1) cluster_arrive();                    // the blocks of the cluster have begun
  const Row<T> row(a, r0);
  const Share share(row.nvec, rank, blocks);
  uint4 r[kVecs];
  Sums sum{neg_inf(), 0.f, 0.f};
  for (int base = share.begin; base < share.end; base += kChunk) {
    load_chunk<T, kThreads, kVecs>(row, share, base, r);
    float top = Vec<T>::max(r[0]);
#pragma unroll
    for (int i = 1; i < kVecs; ++i) top = fmaxf(top, Vec<T>::max(r[i]));
    accumulate<T, kVecs, true>(r, top, a.c, sum);
  }
  const float top = sum.m;
  sum = team_sums<kThreads>(sum, a.c, sh.red);
  int n = 0;
  if (o.top_k > 0)
    n = collect_top<T, kThreads, kVecs>(row, share, r, top, o.top_k, sh.top);
  const unsigned long long* keys = sh.top.cand;
  if (blocks > 1) {
    // the share's sums and its sorted top entries go to the first block
    cluster_wait();
    if (Tm::tid() < 3)
      remote_store(remote(&cl.sums[rank][Tm::tid()], 0),
                   Tm::tid() == 0 ? sum.m : Tm::tid() == 1 ? sum.s : sum.t);
    for (int i = Tm::tid(); i < n; i += kThreads) {
      const int at = rank_of(keys[i], keys, n);
      if (at < o.top_k) remote_store(remote(&cl.keys[rank][at], 0), keys[i]);
    }
    for (int i = n + Tm::tid(); i < o.top_k; i += kThreads)
      remote_store(remote(&cl.keys[rank][i], 0), 0ull);
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    sum = {cl.sums[0][0], cl.sums[0][1], cl.sums[0][2]};
    for (int b = 1; b < blocks; ++b)
      sum = join(sum, Sums{cl.sums[b][0], cl.sums[b][1], cl.sums[b][2]}, a.c);
  }
  const float kLn2 = 0.69314718f;
  const float m = sum.m == neg_inf() ? 0.f : sum.m, s = sum.s, log_s = logf(s);
  const bool bad = s != s;
  if (Tm::tid() == 0) {
    if (o.entropy) o.entropy[row.index] = s == 0.f ? 0.f : log_s - kLn2 * (sum.t / s);
    if (o.log_norm) o.log_norm[row.index] = m * a.inv_t + log_s;
    if (o.stats) {
      o.stats[2 * row.index] = m;
      o.stats[2 * row.index + 1] = s;
    }
  }
  for (int k = Tm::tid(); k < o.n_targets; k += kThreads) {
    const long long i = o.targets[row.index * o.n_targets + k];
    float lp = 0.f;
    if (i >= row.size || bad) {
      lp = i < 0 ? 0.f : quiet_nan();
    } else if (i >= 0) {
      const float z = row.at((int)i);
      lp = z == neg_inf() ? z : (z - m) * a.inv_t - log_s;
    }
    o.log_probs[row.index * o.n_targets + k] = lp;
  }
  if (o.top_k == 0) return;
  long long* out_i = o.top_indices + row.index * o.top_k;
  float* out_lp = o.top_log_probs + row.index * o.top_k;
  auto put = [&](int at, unsigned long long key) {
    out_i[at] = bad || !key ? -1 : key_index(key);
    out_lp[at] = bad ? quiet_nan()
                     : !key ? neg_inf() : (key_logit((uint32_t)(key >> 32)) - m) * a.inv_t - log_s;
  };
  if (blocks == 1) {
    for (int i = Tm::tid(); i < n; i += kThreads) {
      const int at = rank_of(keys[i], keys, n);
      if (at < o.top_k) put(at, keys[i]);
    }
    for (int i = n + Tm::tid(); i < o.top_k; i += kThreads) put(i, 0ull);
  } else {
    // each block's list is sorted: a key's place is its own plus the larger ones of the others
    int total = 0;
    for (int b = 0; b < blocks; ++b)
      for (int i = Tm::tid(); i < o.top_k; i += kThreads) {
        const unsigned long long key = cl.keys[b][i];
        if (!key) continue;
        int at = i;
        for (int q = 0; q < blocks; ++q) {
          if (q == b) continue;
          int lo = 0, hi = o.top_k;                    // first place with a smaller key
          while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (cl.keys[q][mid] > key) lo = mid + 1; else hi = mid;
          }
          at += lo;
        }
        if (at < o.top_k) put(at, key);
      }
    for (int b = 0; b < blocks; ++b) {
      int lo = 0, hi = o.top_k;
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (cl.keys[b][mid]) lo = mid + 1; else hi = mid;
      }
      total += lo;
    }
    for (int i = total + Tm::tid(); i < o.top_k; i += kThreads) put(i, 0ull);
  }
}

// ------------------------------------------------------- and their gradient
// dz_v = (q_v (a - g_H (log q_v + H)) + sum of the incoming gradients at v) / T
// with a = g_norm - the sum of all incoming gradients of single entries. With
// the forward's m and s that is e (A + B x) for the first term: one
// exponential and two products per entry, and no reduction over the row.
// Dynamic shared memory: per team the spots' indices and gradients.
template <typename T, int kThreads, int kVecs>
__global__ void __launch_bounds__(Team<kThreads>::kBlock)
log_probs_grad_kernel(const __grid_constant__ Rows a, const ScoreGradArgs o, unsigned rows,
                      int blocks) {
  using Tm = Team<kThreads>;
  constexpr int N = Vec<T>::N, kChunk = kThreads * kVecs;
  extern __shared__ int spots[];
  __shared__ float red[Tm::kPerBlock][Tm::kWarps];
  const unsigned r0 = blockIdx.x / blocks * Tm::kPerBlock + Tm::slot();
  if (kThreads == 32 && r0 >= rows) return;
  const Row<T> row(a, r0);
  const Share share(row.nvec, blockIdx.x % blocks, blocks);
  const int nt = o.g_log_probs ? o.n_targets : 0, n = nt + (o.g_top ? o.top_k : 0);
  int* idx = spots + Tm::slot() * 2 * n;
  float* g = reinterpret_cast<float*>(idx + n);
  uint4 r[kVecs];
  if (share.begin < share.end) load_chunk<T, kThreads, kVecs>(row, share, share.begin, r);
  const float m = o.stats[2 * row.index], s = o.stats[2 * row.index + 1];
  float sum = 0.f;
  for (int k = Tm::tid(); k < n; k += kThreads) {
    const bool given = k < nt;
    const long long i = given ? o.targets[row.index * o.n_targets + k]
                              : o.top_indices[row.index * o.top_k + k - nt];
    float gk = given ? o.g_log_probs[row.index * o.n_targets + k]
                     : o.g_top[row.index * o.top_k + k - nt];
    const bool past = i >= row.size;
    if (past) gk = quiet_nan();
    else if (i < 0 || row.at((int)i) == neg_inf()) gk = 0.f;
    idx[k] = i < 0 || past ? -1 : (int)i;
    g[k] = gk;
    sum += gk;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  if (Tm::lane() == 0) red[Tm::slot()][Tm::warp()] = sum;
  Tm::sync();
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < Tm::kWarps; ++w) sum += red[Tm::slot()][w];
  const float kLn2 = 0.69314718f;
  const float gh = o.g_entropy ? o.g_entropy[row.index] : 0.f;
  const float h = o.g_entropy ? o.entropy[row.index] : 0.f;
  const float ac = (o.g_log_norm ? o.g_log_norm[row.index] : 0.f) - sum;
  const float f = s > 0.f ? a.inv_t / s : quiet_nan();
  const float A = f * (ac - gh * (h - logf(s))), B = -f * gh * kLn2;
  // A is NaN where the row has no distribution or no entry
  auto value = [&](float z) {
    const float x = fmaxf((z - m) * a.c, -1000.f);
    return ex2(x) * fmaf(B, x, A);
  };
  for (int base = share.begin; base < share.end; base += kChunk) {
    if (base != share.begin) load_chunk<T, kThreads, kVecs>(row, share, base, r);
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int j = base + i * kThreads + Tm::tid();
      if (j >= share.end) continue;
      float z[N];
      Vec<T>::unpack(r[i], z);
      if (A == A) {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = value(z[e]);
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = z[e] == neg_inf() ? 0.f : A;
      }
      row.store(j, z);
    }
  }
  if (n == 0) return;
  Tm::sync();                                     // the spots' entries are written again
  for (int k = Tm::tid(); k < n; k += kThreads) {
    const int v = idx[k], j = v < 0 ? -1 : (v + row.ph) / N;
    if (j < share.begin || j >= share.end) continue;
    bool first = true;
    for (int q = 0; q < k; ++q) first &= idx[q] != v;
    if (!first) continue;
    float at = 0.f;
    for (int q = k; q < n; ++q) at += idx[q] == v ? g[q] : 0.f;
    const float z = row.at(v);
    row.grad[v] = to_type<T>(z == neg_inf() ? 0.f : A == A ? fmaf(at, a.inv_t, value(z)) : A);
  }
}

// ------------------------------------------------------------ distillation
// Shared memory of one team, in this order (dynamic): p, logits, indices of
// the list, and a bit per entry of the block's share (listed or not).
__host__ __device__ constexpr int distill_bytes(int listed, int vecs, int n) {
  return (16 * listed + ((vecs * n + 31) / 32) * 4 + 15) / 16 * 16;
}

// Per warp: what the list adds up to, in 64 bits.
struct ListSums {
  double mass, p_log_p, p_z, e;    // sum P, P log P, P z', 2^..: exp(z' - top)
};

// The list's entries are dropped from the vectors before the one pass over
// the row, so that pass gives maximum and sum over the rest alone, without a
// difference of nearly equal numbers; the list itself is joined in 64 bits.
// With lse_R, lse the logs of the two normalisers and q_R = exp(lse_R - lse)
//   dz_v = T w exp(z'_v - lse_R) (q_R - P_rest)     outside the list
//   dz_u = T w (exp(z'_u - lse) - P_u)              in it
// so the gradient is one more exponential per entry held in registers.
template <typename T, int kThreads, int kVecs, int kMinBlocks>
__global__ void __launch_bounds__(Team<kThreads>::kBlock, kMinBlocks)
distill_kernel(const __grid_constant__ Rows a, const DistillArgs o, unsigned rows, int blocks,
               int team_bytes) {
  using Tm = Team<kThreads>;
  constexpr int N = Vec<T>::N, kChunk = kThreads * kVecs;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Sums red[Tm::kPerBlock][Tm::kWarps];
  __shared__ ListSums lred[Tm::kPerBlock][Tm::kWarps];
  __shared__ float tops[Tm::kPerBlock][Tm::kWarps][2];
  __shared__ int flags[Tm::kPerBlock][Tm::kWarps];
  __shared__ float cl[kMaxCluster][2];            // every block's maximum and sum
  const int slot = Tm::slot(), K = o.n_listed;
  const unsigned r0 = blockIdx.x / blocks * Tm::kPerBlock + slot;
  const int rank = blockIdx.x % blocks;
  if (kThreads == 32 && r0 >= rows) return;
  if (blocks > 1) cluster_arrive();
  const Row<T> row(a, r0);
  const Share share(row.nvec, rank, blocks);
  double* p = reinterpret_cast<double*>(dyn + slot * team_bytes);
  float* zu = reinterpret_cast<float*>(p + K);
  int* idx = reinterpret_cast<int*>(zu + K);
  uint32_t* bits = reinterpret_cast<uint32_t*>(idx + K);
  float weight = o.weight ? o.weight[row.index] : 1.f;
  const bool off = weight == 0.f;
  weight *= o.scale;
  if (o.upstream) weight *= o.upstream[row.index * o.upstream_stride];
  if (off) {                                      // nothing of the row is looked at
    if (o.row_loss && rank == 0 && Tm::tid() == 0) o.row_loss[row.index] = 0.f;
    if (row.grad) {
      float zero[N];
#pragma unroll
      for (int e = 0; e < N; ++e) zero[e] = 0.f;
      for (int j = share.begin + Tm::tid(); j < share.end; j += kThreads) row.store(j, zero);
    }
    if (blocks > 1) cluster_wait();
    return;
  }
  uint4 r[kVecs];
  if (share.begin < share.end) load_chunk<T, kThreads, kVecs>(row, share, share.begin, r);
  const int words = ((share.end - share.begin) * N + 31) / 32;
  for (int w = Tm::tid(); w < words; w += kThreads) bits[w] = 0u;
  Tm::sync();
  bool bad = false, twice = false;
  float top_lp = neg_inf(), top_z = neg_inf();
  const int u0 = share.begin * N, u1 = share.end * N;
  for (int k = Tm::tid(); k < K; k += kThreads) {
    const long long i = o.indices[row.index * K + k];
    const float lp = o.log_probs[row.index * K + k];
    const float z = i >= 0 && i < row.size ? row.at((int)i) : neg_inf();
    const bool there = z != neg_inf();
    bad |= i >= row.size || (there && !(lp < -neg_inf()));
    idx[k] = there ? (int)i : -1;
    zu[k] = z;
    p[k] = (double)lp;
    if (there) {
      top_lp = fmaxf(top_lp, lp);
      top_z = fmaxf(top_z, z);
    }
  }
  // an entry in another block's share is marked there; repeats are looked for in order
  Tm::sync();
  for (int k = Tm::tid(); k < K; k += kThreads) {
    const int v = idx[k];
    if (v < 0) continue;
    const int u = v + row.ph;
    if (u >= u0 && u < u1) {
      const uint32_t old = atomicOr(&bits[(u - u0) >> 5], 1u << ((u - u0) & 31));
      twice |= (old >> ((u - u0) & 31)) & 1u;
    }
    if (blocks > 1 && !twice)
      for (int q = 0; q < k; ++q) twice |= idx[q] == v;
  }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    top_lp = fmaxf(top_lp, __shfl_xor_sync(0xffffffffu, top_lp, w));
    top_z = fmaxf(top_z, __shfl_xor_sync(0xffffffffu, top_z, w));
  }
  const int flag = __reduce_or_sync(0xffffffffu, (bad ? 1u : 0u) | (twice ? 2u : 0u));
  if (Tm::lane() == 0) {
    tops[slot][Tm::warp()][0] = top_lp;
    tops[slot][Tm::warp()][1] = top_z;
    flags[slot][Tm::warp()] = flag;
  }
  Tm::sync();
  int all = 0;
  top_lp = top_z = neg_inf();
#pragma unroll
  for (int w = 0; w < Tm::kWarps; ++w) {
    top_lp = fmaxf(top_lp, tops[slot][w][0]);
    top_z = fmaxf(top_z, tops[slot][w][1]);
    all |= flags[slot][w];
  }
  bad = all & 1;
  const double t_ = a.t, inv_t = 1.0 / t_;
  const double shift = o.renormalize && top_lp > neg_inf() ? (double)top_lp : 0.0;
  ListSums ls{0.0, 0.0, 0.0, 0.0};
  if (all & 2) {                                  // an entry listed twice counts once
    for (int k = Tm::tid(); k < K; k += kThreads) p[k] = idx[k] < 0 ? 0.0 : exp(p[k] - shift);
    Tm::sync();
    if (Tm::tid() == 0)
      for (int k = 0; k < K; ++k)
        for (int q = k + 1; q < K; ++q)
          if (idx[k] >= 0 && idx[q] == idx[k]) {
            p[k] += p[q];
            p[q] = 0.0;
            idx[q] = -1;
          }
    Tm::sync();
  }
  for (int k = Tm::tid(); k < K; k += kThreads) {
    if (idx[k] < 0) continue;
    const double lp = (all & 2) ? log(p[k]) : p[k] - shift;
    const double pk = (all & 2) ? p[k] : exp(lp);
    const double zp = ((double)zu[k] - (double)top_z) * inv_t;
    p[k] = pk;
    ls.mass += pk;
    if (pk > 0.0) {
      ls.p_log_p += pk * lp;
      ls.p_z += pk * zp;
    }
    ls.e += exp(zp);
  }
  // the rest of the row
  Sums sum{neg_inf(), 0.f, 0.f};
  for (int base = share.begin; base < share.end; base += kChunk) {
    if (base != share.begin) load_chunk<T, kThreads, kVecs>(row, share, base, r);
    float top = neg_inf();
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int j = base + i * kThreads + Tm::tid();
      if (j >= share.end) continue;
      const int u = j * N - u0;
      const uint32_t b = (bits[u >> 5] >> (u & 31)) & ((1u << N) - 1u);
      if (b) drop_bits<T>(r[i], b);
      top = fmaxf(top, Vec<T>::max(r[i]));
    }
    accumulate<T, kVecs, false>(r, top, a.c, sum);
  }
  if (Tm::warp() * 32 < K)                        // the other warps have none of the list
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    ls.mass += __shfl_xor_sync(0xffffffffu, ls.mass, w);
    ls.p_log_p += __shfl_xor_sync(0xffffffffu, ls.p_log_p, w);
    ls.p_z += __shfl_xor_sync(0xffffffffu, ls.p_z, w);
    ls.e += __shfl_xor_sync(0xffffffffu, ls.e, w);
  }
  if (Tm::lane() == 0) lred[slot][Tm::warp()] = ls;
  sum = team_sums<kThreads>(sum, a.c, red[slot]);   // orders lred, too (a barrier, or one warp)
  if constexpr (kThreads == 32) __syncwarp();
  if (blocks > 1) {
    cluster_wait();
    if (Tm::tid() < blocks) {
      remote_store(remote(&cl[rank][0], Tm::tid()), sum.m);
      remote_store(remote(&cl[rank][1], Tm::tid()), sum.s);
    }
    cluster_arrive();
    cluster_wait();
    sum = {cl[0][0], cl[0][1], 0.f};
    for (int b = 1; b < blocks; ++b) sum = join(sum, Sums{cl[b][0], cl[b][1], 0.f}, a.c);
  }
  ls = lred[slot][0];
#pragma unroll
  for (int w = 1; w < Tm::kWarps; ++w) {
    ls.mass += lred[slot][w].mass;
    ls.p_log_p += lred[slot][w].p_log_p;
    ls.p_z += lred[slot][w].p_z;
    ls.e += lred[slot][w].e;
  }
  const bool rest = sum.m != neg_inf(), listed = top_z != neg_inf();
  bad |= sum.s != sum.s || ls.e != ls.e;
  const bool whole = o.renormalize || ls.mass > 1.0 || !rest;
  const double inv = whole && ls.mass > 0.0 ? 1.0 / ls.mass : 1.0;
  const double p_r = whole ? 0.0 : 1.0 - ls.mass;
  const bool live = (rest || listed) && (ls.mass > 0.0 || !whole);
  // logs of the normalisers relative to the larger of the two maxima
  const double big = fmaxf(rest ? sum.m : neg_inf(), top_z);
  const double log_r = rest ? ((double)sum.m - big) * inv_t + log((double)sum.s) : 0.0;
  const double lift = listed ? ((double)top_z - big) * inv_t : 0.0;
  const double norm = (listed ? ls.e * exp(lift) : 0.0) + (rest ? exp(log_r) : 0.0);
  const double log_all = log(norm);
  if (rank == 0 && Tm::tid() == 0 && o.row_loss) {
    double loss = 0.0;
    if (live && ls.mass > 0.0)
      loss = inv * (ls.p_log_p - ls.p_z + (log_all - lift) * ls.mass) + log(inv) * (inv * ls.mass);
    if (p_r > 0.0) loss += p_r * (log(p_r) - (log_r - log_all));
    if (!live) loss = 0.0;
    o.row_loss[row.index] = bad ? quiet_nan() : (float)(loss * t_ * t_ * (double)weight);
  }
  if (!row.grad) return;
  const double q_r = rest ? exp(log_r - log_all) : 0.0, scale = (double)weight * t_;
  const float coef = live && rest ? (float)(scale * (q_r - p_r) / (double)sum.s) : 0.f;
  const float ref = rest ? sum.m : 0.f, nan = quiet_nan();
  bad |= coef != coef;
  for (int base = share.begin; base < share.end; base += kChunk) {
    if (share.end - share.begin > kChunk) {
      load_chunk<T, kThreads, kVecs>(row, share, base, r);
    }
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const int j = base + i * kThreads + Tm::tid();
      if (j >= share.end) continue;
      float z[N];
      Vec<T>::unpack(r[i], z);
      if (!bad) {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = ex2((z[e] - ref) * a.c) * coef;
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = z[e] == neg_inf() ? 0.f : nan;
      }
      row.store(j, z);
    }
  }
  if (K == 0) return;
  Tm::sync();                                     // the listed entries are written again
  for (int k = Tm::tid(); k < K; k += kThreads) {
    const int v = idx[k], u = v + row.ph;
    if (v < 0 || u < u0 || u >= u1) continue;
    const float q = expf((float)(((double)zu[k] - big) * inv_t - log_all));
    const double d = live ? scale * ((double)q - p[k] * inv) : 0.0;
    row.grad[v] = to_type<T>(bad ? nan : (float)d);
  }
}

// Sum of the rows' losses by one block, in 64 bits and a fixed order.
static __global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ row_loss,
                                                        long long n, float* __restrict__ loss) {
  __shared__ double red[32];
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) s += row_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = red[threadIdx.x];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (threadIdx.x == 0) *loss = (float)s;
  }
}

}  // namespace lk
}  // namespace chm
