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

#include "chm_exp64.h"
#include "chm_likelihood.h"
#include "chm_ptx.cuh"

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
  static constexpr uint32_t kFill = 0xf149f2cau;       // -1e30
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
  // running maxima of one or more vectors, kept in the type's own width
  using Max = float;
  static __device__ __forceinline__ Max lowest() { return __uint_as_float(kNegInf); }
  static __device__ __forceinline__ Max wide_max(const uint4& r) { return max(r); }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return fmaxf(a, b); }
  static __device__ __forceinline__ float to_max(Max a) { return a; }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static constexpr uint32_t kFill = 0xf14af14au;       // -1e30
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
  // running maxima of one or more vectors, kept in pairs of the type's own width
  using Max = __nv_bfloat162;
  static __device__ __forceinline__ Max lowest() {
    const uint32_t v = kNegInf;
    return reinterpret_cast<const Max&>(v);
  }
  static __device__ __forceinline__ Max wide_max(const uint4& r) {
    const Max* h = reinterpret_cast<const Max*>(&r);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2(a, b); }
  static __device__ __forceinline__ float to_max(Max a) {
    return fmaxf(__low2float(a), __high2float(a));
  }
  static __device__ __forceinline__ float max(const uint4& r) { return to_max(wide_max(r)); }
};
template <> struct Vec<__half> {
  static constexpr int N = 8;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static constexpr uint32_t kFill = 0xfbfffbffu;       // -65504, the lowest
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
  // running maxima of one or more vectors, kept in pairs of the type's own width
  using Max = __half2;
  static __device__ __forceinline__ Max lowest() {
    const uint32_t v = kNegInf;
    return reinterpret_cast<const Max&>(v);
  }
  static __device__ __forceinline__ Max wide_max(const uint4& r) {
    const Max* h = reinterpret_cast<const Max*>(&r);
    return __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
  }
  static __device__ __forceinline__ Max larger(Max a, Max b) { return __hmax2(a, b); }
  static __device__ __forceinline__ float to_max(Max a) {
    return fmaxf(__low2float(a), __high2float(a));
  }
  static __device__ __forceinline__ float max(const uint4& r) { return to_max(wide_max(r)); }
};

template <uint32_t kBits> __device__ __forceinline__ uint4 vec_of() {
  return make_uint4(kBits, kBits, kBits, kBits);
}
// a vector of a type's fill value, and that value
template <typename T> __device__ __forceinline__ float fill_value() {
  float f[Vec<T>::N];
  Vec<T>::unpack(vec_of<Vec<T>::kFill>(), f);
  return f[0];
}

// Shared memory by 32-bit address plus an offset known at compile time.
template <int kOff> __device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "r"(a), "n"(kOff)
               : "memory");
  return r;
}
template <int kOff> __device__ __forceinline__ void sts128(uint32_t a, const uint4& r) {
  asm volatile("st.shared.v4.u32 [%0 + %1], {%2, %3, %4, %5};" ::"r"(a), "n"(kOff), "r"(r.x),
               "r"(r.y), "r"(r.z), "r"(r.w)
               : "memory");
}
template <int kSOff, int kGOff>
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0 + %1], [%2 + %3], 16;" ::"r"(dst), "n"(kSOff),
               "l"(src), "n"(kGOff)
               : "memory");
}

constexpr int kBatch = 4;          // vectors that a thread takes at a time
// Batches that a thread adds to one running sum in fp32, one by one. In a row of nearly equal
// entries all roundings have one sign: 512 batches are off by up to 128 half steps, 64 by 16.
constexpr int kMaxBatches = 64;

// A thread's next kBatch vectors of a row to a place in shared memory, both
// kStride vectors apart; kBits for those behind its last.
template <int kStride, uint32_t kBits>
__device__ __forceinline__ void copy_batch(uint32_t dst, const char* src, int left) {
  constexpr int S = kStride * 16;
  if (left >= kBatch) {
    copy16<0, 0>(dst, src);
    copy16<S, S>(dst, src);
    copy16<2 * S, 2 * S>(dst, src);
    copy16<3 * S, 3 * S>(dst, src);
  } else {
    if (left > 0) copy16<0, 0>(dst, src); else sts128<0>(dst, vec_of<kBits>());
    if (left > 1) copy16<S, S>(dst, src); else sts128<S>(dst, vec_of<kBits>());
    if (left > 2) copy16<2 * S, 2 * S>(dst, src); else sts128<2 * S>(dst, vec_of<kBits>());
    sts128<3 * S>(dst, vec_of<kBits>());
  }
}
template <int kStride>
__device__ __forceinline__ void read_batch(uint32_t src, uint4 (&r)[kBatch]) {
  constexpr int S = kStride * 16;
  r[0] = lds128<0>(src);
  r[1] = lds128<S>(src);
  r[2] = lds128<2 * S>(src);
  r[3] = lds128<3 * S>(src);
}
template <int kStride>
__device__ __forceinline__ void write_batch(uint32_t dst, const uint4 (&r)[kBatch]) {
  constexpr int S = kStride * 16;
  sts128<0>(dst, r[0]);
  sts128<S>(dst, r[1]);
  sts128<2 * S>(dst, r[2]);
  sts128<3 * S>(dst, r[3]);
}

// Each byte of the result is 0xff or 0: the top bit of the byte of t that the
// selector's digit (less 8) names.
template <uint32_t kSel> __device__ __forceinline__ uint32_t spread(uint32_t t) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %1, %2;" : "=r"(r) : "r"(t), "n"(kSel));
  return r;
}

// One row of the launch. Whatever address it starts at, its entries are
// `head` single ones up to a 16-byte boundary, nin full vectors, and a few
// single ones behind; no access leaves the row.
template <typename T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* z;
  const uint8_t* mask;
  T* grad;
  int size, head, nin;
  long long index;

  __device__ __forceinline__ Row(const Rows& a, unsigned r) {
    const unsigned n = a.ng == 1 ? r : r / (unsigned)a.ng, g = r - n * (unsigned)a.ng;
    z = static_cast<const T*>(a.z) + n * a.row_stride + a.off[g];
    mask = a.mask ? a.mask + n * a.mask_stride + a.moff[g] : nullptr;
    grad = a.grad ? static_cast<T*>(a.grad) + n * a.grad_stride + a.goff[g] : nullptr;
    size = a.size[g];
    index = (long long)n * a.n_groups + a.g0 + g;
    const int ph = (int)((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    head = min(size, (N - ph) & (N - 1));
    nin = (size - head) / N;
  }
  // the gradient's row lies in its granules as the logits' row does
  __device__ __forceinline__ bool vec_store() const {
    return ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
  }
  // entry v; the mask's byte and the logit are asked for together
  __device__ __forceinline__ float at(int v) const {
    const uint8_t in = mask ? mask[v] : 1;
    const float f = to_float(z[v]);
    return in ? f : neg_inf();
  }
  __device__ __forceinline__ const T* vec(int j) const { return z + head + (long long)j * N; }
  // the mask's bytes for vector j
  struct MaskBytes {
    uint32_t w[N / 4];
  };
  __device__ __forceinline__ MaskBytes mask_bytes(int j) const {
    const uint8_t* m = mask + head + (long long)j * N;
    MaskBytes b;
    if ((reinterpret_cast<uintptr_t>(m) & (N - 1)) == 0) {
#pragma unroll
      for (int i = 0; i < N / 4; ++i) b.w[i] = reinterpret_cast<const uint32_t*>(m)[i];
    } else {
#pragma unroll
      for (int i = 0; i < N / 4; ++i)
        b.w[i] = m[4 * i] | m[4 * i + 1] << 8 | m[4 * i + 2] << 16 | (uint32_t)m[4 * i + 3] << 24;
    }
    return b;
  }
  // -inf over what the mask takes out
  static __device__ __forceinline__ void apply_mask(uint4& r, const MaskBytes& b) {
    uint32_t* v = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      // the top bit of every byte that is not zero
      const uint32_t t = ((b.w[i] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | b.w[i];
      if constexpr (sizeof(T) == 4) {
        const uint32_t on[4] = {spread<0x8888>(t), spread<0x9999>(t), spread<0xaaaa>(t),
                                spread<0xbbbb>(t)};
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (v[e] & on[e]) | (Vec<T>::kNegInf & ~on[e]);
      } else {
        const uint32_t on0 = spread<0x9988>(t), on1 = spread<0xbbaa>(t);
        v[2 * i] = (v[2 * i] & on0) | (Vec<T>::kNegInf & ~on0);
        v[2 * i + 1] = (v[2 * i + 1] & on1) | (Vec<T>::kNegInf & ~on1);
      }
    }
  }
  __device__ __forceinline__ void apply_mask(uint4& r, int j) const {
    apply_mask(r, mask_bytes(j));
  }
  __device__ __forceinline__ void store(int j, const float (&d)[N], bool vec_store) const {
    T* g = grad + head + (long long)j * N;
    if (vec_store) {
      *reinterpret_cast<uint4*>(g) = Vec<T>::pack(d);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) g[e] = to_type<T>(d[e]);
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

// A list of entries in the order of the row, each with its place in the list:
// repeats are neighbours, the first of them first. Bitonic, over n keys, a
// power of two; keys behind the list are kNoKey.
constexpr uint32_t kNoKey = 0xffffffffu;
constexpr int kPlaceBits = 11;                         // of a list of up to 2,048
static_assert(kMaxList + kMaxTop <= 1 << kPlaceBits, "entries are below 2^20");
__host__ __device__ constexpr int sort_size(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}
__device__ __forceinline__ uint32_t place_key(int v, int place) {
  return v < 0 ? kNoKey : (uint32_t)v << kPlaceBits | (uint32_t)place;
}
__device__ __forceinline__ int key_entry(uint32_t key) { return (int)(key >> kPlaceBits); }
__device__ __forceinline__ int key_place(uint32_t key) {
  return (int)(key & ((1u << kPlaceBits) - 1));
}
template <int kThreads> __device__ __noinline__ void sort_places(uint32_t* key, int n) {
  using Tm = Team<kThreads>;
#pragma unroll 1
  for (int run = 2; run <= n; run *= 2)
#pragma unroll 1
    for (int half = run / 2; half > 0; half /= 2) {
      Tm::sync();
#pragma unroll 1
      for (int t = Tm::tid(); t < n / 2; t += kThreads) {
        const int i = (t & ~(half - 1)) * 2 + (t & (half - 1));
        const uint32_t x = key[i], y = key[i + half];
        if ((x > y) == ((i & run) == 0)) {
          key[i] = y;
          key[i + half] = x;
        }
      }
    }
  Tm::sync();
}

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

// One block's part of a row: the vectors [begin, end), the entries [first,
// last), and for the first threads of the row's two ends one single entry.
template <typename T> struct Share {
  int begin, end, first, last;
  int edge;                        // this thread's single entry, or -1
  __device__ __forceinline__ Share(const Row<T>& row, int rank, int log_blocks, int tid) {
    constexpr int N = Vec<T>::N;
    const int blocks = 1 << log_blocks, per = (row.nin + blocks - 1) >> log_blocks;
    begin = min(rank * per, row.nin);
    end = min(begin + per, row.nin);
    const int tail = row.head + row.nin * N;
    first = rank == 0 ? 0 : row.head + begin * N;
    last = rank == blocks - 1 ? row.size : row.head + end * N;
    edge = -1;
    if (rank == 0 && tid < row.head) edge = tid;
    else if (rank == blocks - 1 && tid >= N && tail + tid - N < row.size) edge = tail + tid - N;
  }
};

// Vectors of [begin, end) that this thread has when they go round the team.
template <int kThreads> __device__ __forceinline__ int own_vectors(int begin, int end) {
  return max(0, end - begin - Team<kThreads>::tid() + kThreads - 1) / kThreads;
}

// The vectors of a chunk pass through shared memory by asynchronous copies:
// thread t copies, and sums up, the vectors t, t + kThreads, ... of the chunk.
// All of them are in flight at once without a register, and a row that fits
// is there for every later pass. In shared memory the chunk is as in memory.
template <typename T, int kThreads>
__device__ __forceinline__ void copy_chunk(uint32_t chunk, const Row<T>& row, int base, int n) {
  const char* src = reinterpret_cast<const char*>(row.vec(base + Team<kThreads>::tid()));
  uint32_t dst = chunk + Team<kThreads>::tid() * 16;
#pragma unroll 1
  for (; n > 0; n -= kBatch) {
    copy_batch<kThreads, Vec<T>::kNegInf>(dst, src, n);
    dst += kBatch * kThreads * 16;
    src += kBatch * kThreads * 16;
  }
  cp_async_commit();
}

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
__device__ __forceinline__ Sums single(float z, float c) {
  if (z == neg_inf()) return {z, 0.f, 0.f};
  return {z, ex2((z - z) * c), 0.f};              // NaN for NaN and +inf
}
// Adds vectors, whose maximum is `top`, to the running sums: per entry one
// exponential and half an add, a product and a sum or two. With kClamp also a
// clamp, for the entropy's 0 * -inf; without, t is NaN if there is a -inf.
// Places without an entry hold the fill value, whose exponential is 0 unless
// the maximum is as low.
template <typename T, int kVecs, bool kEntropy, bool kClamp>
__device__ __forceinline__ void accumulate(const uint4 (&r)[kVecs], float top, float c, Sums& a) {
  constexpr int N = Vec<T>::N;
  if (top > a.m) {
    if (a.m != neg_inf()) {                       // else nothing to rescale yet
      const float d = fmaxf((a.m - top) * c, -1000.f), f = ex2(d);
      if (kEntropy) a.t = f * (a.t + d * a.s);
      a.s *= f;
    }
    a.m = top;
  }
  const float ref = a.m == neg_inf() ? 0.f : -a.m;
  const float2 nref = {ref, ref}, cc = {c, c};
  float2 s = {0.f, 0.f}, t = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kVecs; ++i) {
    float f[N];
    Vec<T>::unpack(r[i], f);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      float2 x = __fmul2_rn(__fadd2_rn(float2{f[e], f[e + 1]}, nref), cc);
      const float2 p = {ex2(x.x), ex2(x.y)};
      s = __fadd2_rn(s, p);
      if (kClamp) {
        x.x = fmaxf(x.x, -1000.f);
        x.y = fmaxf(x.y, -1000.f);
      }
      if (kEntropy) t = __ffma2_rn(p, x, t);
    }
  }
  a.s += s.x + s.y;
  if (kEntropy) a.t += t.x + t.y;
}

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
// A thread's sums of a share whose entries are -inf in places, or all of them
// as low as the fill value: clamped, and read from memory without any fill. It is
// a second pass over the row with one vector in flight: 4,096 x 50,001 bf16 with
// one entry in ten at -inf take 182 us, 117 if a mask takes those out, 76 without.
template <typename T, int kThreads, bool kMask>
__device__ __noinline__ Sums careful_sums(const Row<T>& row, const Share<T>& share, float c) {
  Sums sum{neg_inf(), 0.f, 0.f}, part = sum;
  int n = 0;
#pragma unroll 1
  for (int j = share.begin + Team<kThreads>::tid(); j < share.end; j += kThreads) {
    uint4 r[1] = {*reinterpret_cast<const uint4*>(row.vec(j))};
    if (kMask) row.apply_mask(r[0], j);
    accumulate<T, 1, true, true>(r, Vec<T>::max(r[0]), c, part);
    if (++n % kMaxBatches == 0) {
      sum = join(sum, part, c);
      part = {neg_inf(), 0.f, 0.f};
    }
  }
  return join(sum, part, c);
}

// Joins the team's sums (every thread gets the result): the maximum first, so
// that each thread rescales its own sums once.
template <int kThreads>
__device__ __forceinline__ Sums team_sums(Sums a, float c, Sums* red) {
  using Tm = Team<kThreads>;
  const uint32_t top = __reduce_max_sync(0xffffffffu, logit_key(a.m));
  const float m = top ? key_logit(top) : neg_inf();
  const float d = fmaxf((a.m - m) * c, -1000.f), f = ex2(d);
  a = {m, f * a.s, f * (a.t + d * a.s)};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
  }
  if constexpr (kThreads == 32) return a;
  if (Tm::lane() == 0) red[Tm::warp()] = a;
  __syncthreads();
  float all = red[0].m;
#pragma unroll
  for (int w = 1; w < Tm::kWarps; ++w) all = fmaxf(all, red[w].m);
  Sums sum{all, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < Tm::kWarps; ++w) {
    const Sums b = red[w];
    const float db = fmaxf((b.m - all) * c, -1000.f), fb = ex2(db);
    sum.s += fb * b.s;
    sum.t += fb * (b.t + db * b.s);
  }
  return sum;
}

// A row that is read once goes through a ring of two batches per thread: one
// or two are on their way while one is added up.
constexpr int kSlots = 2 * kBatch;

template <typename T, int kThreads>
struct Ring {
  uint32_t buf;                    // this thread's first slot
  const char* src;                 // its next vector
  int left;                        // vectors not yet asked for
  int n;                           // vectors in all
  __device__ __forceinline__ Ring(const void* slots, const Row<T>& row, const Share<T>& share) {
    buf = smem_u32(slots) + Team<kThreads>::tid() * 16;
    src = reinterpret_cast<const char*>(row.vec(share.begin + Team<kThreads>::tid()));
    n = left = own_vectors<kThreads>(share.begin, share.end);
  }
  // asks for the next batch into the half `at` of the ring
  __device__ __forceinline__ void ask(uint32_t at) {
    if (left > 0) {
      copy_batch<kThreads, Vec<T>::kFill>(at, src, left);
      src += kBatch * kThreads * 16;
      left -= kBatch;
    }
    cp_async_commit();
  }
};

// ------------------------------------------------------------ top entries
__device__ __forceinline__ unsigned long long order_key(uint32_t key, int v) {
  return ((unsigned long long)key << 32) | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ int key_index(unsigned long long key) {
  return (int)(0xffffffffu - (unsigned)key);
}

template <int kThreads> struct TopShared {
  static constexpr int kMaxCand = 512;
  alignas(16) unsigned long long cand[kMaxCand];
  uint32_t bound[Team<kThreads>::kWarps];
  uint4 hold[Team<kThreads>::kWarps][32];
  int hold_at[Team<kThreads>::kWarps][32];
  uint8_t list[Team<kThreads>::kWarps][32 * kBatch];
  int count;                       // candidates found; written no more once the team has read it
  int kept;                        // what thin_out or count_top leaves of them
  int red[Team<kThreads>::kWarps];
};

// Calls f(z, v) for this thread's entries of the share, read from memory.
template <typename T, int kThreads, bool kMask, typename F>
__device__ __forceinline__ void each_entry(const Row<T>& row, const Share<T>& share, float edge,
                                           F f) {
  constexpr int N = Vec<T>::N;
  if (share.edge >= 0) f(edge, share.edge);
#pragma unroll 1
  for (int j = share.begin + Team<kThreads>::tid(); j < share.end; j += kThreads) {
    uint4 r = *reinterpret_cast<const uint4*>(row.vec(j));
    if (kMask) row.apply_mask(r, j);
    float z[N];
    Vec<T>::unpack(r, z);
#pragma unroll
    for (int e = 0; e < N; ++e) f(z[e], row.head + j * N + e);
  }
}

// Rows with more candidates than there is room for (many equal logits) are
// counted: bisection for the k-th largest logit, then for the index up to
// which its equals belong to the first k. Leaves exactly k candidates. That is up
// to about 50 passes: 4,096 x 50,001 equal bf16 logits take 5.1 ms, 1,024 x 1,000
// equal fp32 ones 0.10 ms.
template <typename T, int kThreads, bool kMask>
__device__ __noinline__ int count_top(const Row<T>& row, const Share<T>& share, float edge,
                                      uint32_t bound, int k, TopShared<kThreads>& sh) {
  using Tm = Team<kThreads>;
  // how many entries have a key of at least q (with `equal`: of exactly q, up to index v)
  auto count = [&](uint32_t q, bool equal, int last) {
    int n = 0;
    each_entry<T, kThreads, kMask>(row, share, edge, [&](float z, int v) {
      const uint32_t key = logit_key(z);
      n += equal ? key == q && v <= last : key >= q;
    });
    return Tm::sum(n, sh.red);
  };
  uint32_t lo = max(bound, 1u), hi = 0xffffffffu;      // count(lo) >= k > count(hi)
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    if (count(mid, false, 0) >= k) lo = mid; else hi = mid;
  }
  const int need = k - count(hi, false, 0);
  int before = -1, last = row.size - 1;                // equals up to `last`: at least `need`
  while (last - before > 1) {
    const int mid = before + (last - before) / 2;
    if (count(lo, true, mid) >= need) last = mid; else before = mid;
  }
  Tm::sync();
  if (Tm::tid() == 0) sh.kept = 0;
  Tm::sync();
  each_entry<T, kThreads, kMask>(row, share, edge, [&](float z, int v) {
    const uint32_t key = logit_key(z);
    if (key > lo || (key == lo && v <= last)) sh.cand[atomicAdd(&sh.kept, 1)] = order_key(key, v);
  });
  Tm::sync();
  return sh.kept;
}

// Drops candidates that are too many to be ranked one against all: the first
// warp bisects over their logits until little more than k are left.
template <int kThreads>
__device__ __noinline__ int thin_out(int n, int k, TopShared<kThreads>& sh) {
  using Tm = Team<kThreads>;
  constexpr uint32_t kAll = 0xffffffffu;
  if (Tm::warp() == 0) {
    const int lane = Tm::lane();
    uint32_t lo = 0, hi = kAll;
    for (int left = n; hi - lo > 1 && left > k + k / 4;) {
      const uint32_t mid = lo + (hi - lo) / 2;
      int r = 0;
      for (int i = lane; i < n; i += 32) r += (uint32_t)(sh.cand[i] >> 32) >= mid;
      r = __reduce_add_sync(kAll, r);
      if (r >= k) {
        lo = mid;
        left = r;
      } else {
        hi = mid;
      }
    }
    int kept = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const unsigned long long key = i0 + lane < n ? sh.cand[i0 + lane] : 0ull;
      const bool keep = key && (uint32_t)(key >> 32) >= lo;
      const uint32_t vote = __ballot_sync(kAll, keep);
      __syncwarp();
      if (keep) sh.cand[kept + __popc(vote & ((1u << lane) - 1))] = key;
      kept += __popc(vote);
      __syncwarp();
    }
    if (lane == 0) sh.kept = kept;
  }
  Tm::sync();
  return sh.kept;
}

// The k largest entries of a block's share and some more, in no order, into
// sh.cand; returns their number (all there are if the share has fewer than k).
//
// While the row passes, each thread keeps four maxima, one for every fourth of
// its vectors: 4 * kThreads groups in all. If k of the groups have a maximum
// of at least b, then k entries do, so every entry at or above b is a
// candidate and only those groups are looked at again. b is the smallest over
// the warps of the ceil(k / warps)-th largest maximum of each, and where the
// warps differ too much (a profile's summit lies in few of them) it comes from
// bisection over all.
template <typename T, int kThreads, bool kMask>
__device__ __forceinline__ int collect_top(const Row<T>& row, const Share<T>& share,
                                           const Ring<T, kThreads>& ring, float edge,
                                           const float (&top)[kBatch], int k,
                                           TopShared<kThreads>& sh) {
  using Tm = Team<kThreads>;
  constexpr int N = Vec<T>::N;
  constexpr uint32_t kAll = 0xffffffffu;
  uint32_t key[kBatch], most = 0;
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    key[u] = logit_key(top[u]);
    most = max(most, key[u]);
  }
  auto reach = [&](uint32_t q) {
    int n = 0;
#pragma unroll
    for (int u = 0; u < kBatch; ++u) n += key[u] >= q;
    return n;
  };
  const int want = (k + Tm::kWarps - 1) / Tm::kWarps;
  uint32_t lo = 0;
  if (want <= 12) {
    // the want-th largest, one by one: each lane's maxima sorted, its largest first
    uint32_t q[kBatch] = {key[0], key[1], key[2], key[3]};
    auto order = [](uint32_t& x, uint32_t& y) {
      const uint32_t t = max(x, y);
      y = min(x, y);
      x = t;
    };
    order(q[0], q[1]);
    order(q[2], q[3]);
    order(q[0], q[2]);
    order(q[1], q[3]);
    order(q[1], q[2]);
#pragma unroll 1
    for (int i = 0; i < want; ++i) {
      lo = __reduce_max_sync(kAll, q[0]);
      const uint32_t vote = __ballot_sync(kAll, q[0] == lo);
      if (Tm::lane() == __ffs(vote) - 1) {
        q[0] = q[1];
        q[1] = q[2];
        q[2] = q[3];
        q[3] = 0;
      }
    }
  } else {
    // 32 maxima reach the smallest of the lanes' largest
    if (want <= 32) lo = __reduce_min_sync(kAll, most);
    uint32_t hi = __reduce_max_sync(kAll, most) + 1;
    for (int n = 128; hi - lo > 1 && n > want + want / 16;) {
      const uint32_t mid = lo + (hi - lo) / 2;
      const int r = __reduce_add_sync(kAll, reach(mid));
      if (r >= want) {
        lo = mid;
        n = r;
      } else {
        hi = mid;
      }
    }
  }
  if (Tm::tid() == 0) sh.count = 0;
  if constexpr (Tm::kWarps > 1) {
    if (Tm::lane() == 0) sh.bound[Tm::warp()] = lo;
    __syncthreads();
    uint32_t up = 0;
#pragma unroll
    for (int w = 0; w < Tm::kWarps; ++w) {
      lo = min(lo, sh.bound[w]);
      up = max(up, sh.bound[w]);
    }
    for (int n = Tm::sum(reach(lo), sh.red); up - lo > 1 && n > 2 * k + 16;) {
      const uint32_t mid = lo + (up - lo) / 2;
      const int r = Tm::sum(reach(mid), sh.red);
      if (r >= k) {
        lo = mid;
        n = r;
      } else {
        up = mid;
      }
    }
  }
  if (lo <= logit_key(fill_value<T>())) lo = 0;   // places without an entry may be among them
  const float least = lo ? key_logit(lo) : -3.4028234664e38f;   // the lowest logit there is
  // the groups that reach it, warp by warp: their vectors, one to a lane
  uint8_t* list = sh.list[Tm::warp()];
  int groups = 0;
#pragma unroll
  for (int u = 0; u < kBatch; ++u) {
    const bool in = top[u] >= least;
    const uint32_t vote = __ballot_sync(kAll, in);
    if (in) list[groups + __popc(vote & ((1u << Tm::lane()) - 1))] = Tm::lane() * kBatch + u;
    groups += __popc(vote);
  }
  __syncwarp();                                        // and the copies of the other lanes
  const int len = share.end - share.begin;
  const int per = (len + kBatch * kThreads - 1) / (kBatch * kThreads);   // vectors of a group
  const bool here = len <= kSlots * kThreads;          // the ring still holds the row
  const uint32_t slots = ring.buf + (Tm::warp() * 32 - Tm::tid()) * 16;
  uint4* hold = sh.hold[Tm::warp()];
  int* hold_at = sh.hold_at[Tm::warp()];
  // a group's vectors side by side on a power of two of lanes, as many groups as fit
  const int lg = per > 16 ? 5 : per > 1 ? 32 - __clz(per - 1) : 0;
  const int g_lane = Tm::lane() >> lg, g_step = 32 >> lg, i_lane = Tm::lane() & ((1 << lg) - 1);
  const uint32_t before = (1u << Tm::lane()) - 1;
  int found = 0;                                       // a team of one warp needs no shared count
  const int rounds = (groups + g_step - 1) / g_step * ((per + 31) / 32);
  // the vector that this lane has in a round: its place in the share, or -1
  auto fetch = [&](int round, uint4& r) {
    const int parts = (per + 31) / 32, i_at = (parts == 1 ? 0 : round % parts * 32) + i_lane;
    const int g = (parts == 1 ? round : round / parts) * g_step + g_lane;
    if (round >= rounds || g >= groups || i_at >= per) return -1;
    const int who = list[g], i = i_at * kBatch + (who & (kBatch - 1));
    const int j = share.begin + i * kThreads + Tm::warp() * 32 + who / kBatch;
    if (j >= share.end) return -1;
    if (here) r = lds128<0>(slots + (i * kThreads + who / kBatch) * 16);
    else r = __ldg(reinterpret_cast<const uint4*>(row.vec(j)));
    return j;
  };
  uint4 r0, r1, r2;                                    // of this round and the next two
  int j0 = fetch(0, r0), j1 = fetch(1, r1);
#pragma unroll 1
  for (int round = 0; round < rounds; ++round) {
    const int j2 = fetch(round + 2, r2);
    if (kMask && !here && j0 >= 0) row.apply_mask(r0, j0);
    const bool in = j0 >= 0 && Vec<T>::max(r0) >= least;
    const uint32_t vote = __ballot_sync(kAll, in);
    // the vectors that reach the bound side by side, then one entry to a lane
    if (in) {
      hold[__popc(vote & before)] = r0;
      hold_at[__popc(vote & before)] = row.head + j0 * N;
    }
    __syncwarp();
    const int entries = __popc(vote) * N;
#pragma unroll 1
    for (int t0 = 0; t0 < entries; t0 += 32) {
      const int t = t0 + Tm::lane();
      float z = neg_inf();
      if (t < entries) z = to_float(reinterpret_cast<const T*>(hold)[t]);
      const bool top_z = z >= least;
      const uint32_t hits = __ballot_sync(kAll, top_z);
      int at = found;
      if constexpr (kThreads == 32) {
        found += __popc(hits);
      } else {
        if (Tm::lane() == 0) at = atomicAdd(&sh.count, __popc(hits));
        at = __shfl_sync(kAll, at, 0);
      }
      at += __popc(hits & before);
      if (top_z && at < TopShared<kThreads>::kMaxCand)
        sh.cand[at] = order_key(logit_key(z), hold_at[t / N] + (t & (N - 1)));
    }
    __syncwarp();
    r0 = r1;
    j0 = j1;
    r1 = r2;
    j1 = j2;
  }
  if constexpr (kThreads == 32) {
    if (Tm::lane() == 0) sh.count = found;
    __syncwarp();
  }
  if (share.edge >= 0 && edge >= least) {
    const int at = atomicAdd(&sh.count, 1);
    if (at < TopShared<kThreads>::kMaxCand) sh.cand[at] = order_key(logit_key(edge), share.edge);
  }
  Tm::sync();
  const int n = sh.count;                              // every thread takes the same way from here
  if (n <= 2 * k + 16) return n;
  if (n <= TopShared<kThreads>::kMaxCand) return thin_out<kThreads>(n, k, sh);
  return count_top<T, kThreads, kMask>(row, share, edge, lo, k, sh);
}

// Place of a key among `n` different ones, the largest first.
__device__ __forceinline__ int rank_of(unsigned long long key, const unsigned long long* keys,
                                       int n) {
  int r = 0;
#pragma unroll 2
  for (int i = 0; i + 1 < n; i += 2) {
    const ulonglong2 two = *reinterpret_cast<const ulonglong2*>(keys + i);
    r += two.x > key;
    r += two.y > key;
  }
  if (n & 1) r += keys[n - 1] > key;
  return r;
}

// ------------------------------------------------------- log probabilities
template <int kThreads> struct ScoreShared {
  Sums red[Team<kThreads>::kWarps];
  TopShared<kThreads> top;
};
// What the other blocks of a row's cluster send to the first.
struct ScoreCluster {
  float sums[kMaxCluster][4];
  unsigned long long keys[kMaxCluster][kMaxTop];
};

// One pass over the row for maximum, sum, entropy and the groups' maxima; the
// top entries from the groups that matter; the given entries by a gather at
// the end. Dynamic shared memory: per team a ring; ScoreCluster if blocks > 1.
//
// 4,096 rows of 50,001 bf16 with 8 top entries: 88 us, 4.7 TB/s. DRAM would
// take 63, the exponential unit 52 (one e^x an entry) and the issue slots 59;
// the three do not overlap fully, since every row ends with its top entries,
// of which nothing is known before. Short rows are bound by that end: 2,048
// examples of five masked groups with 64 given and 16 top entries take 50 us,
// 2.0 TB/s, 1,024 rows of 1,000 with 32 top entries 9.6.
// Rows go from the last to the first, since what wrote the logits ended there,
// and the gradient from the first to the last: L2 still holds those (2,048 x
// 65,536 bf16 forward and backward: 155 to 153 us).
template <typename T, int kThreads, bool kMask>
__global__ void __launch_bounds__(Team<kThreads>::kBlock)
log_probs_kernel(const __grid_constant__ Rows a, const ScoreArgs o, unsigned rows, int log_blocks) {
  using Tm = Team<kThreads>;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ ScoreShared<kThreads> shared[Tm::kPerBlock];
  ScoreShared<kThreads>& sh = shared[Tm::slot()];
  uint4* slots = reinterpret_cast<uint4*>(dyn) + Tm::slot() * kSlots * kThreads;
  ScoreCluster& cl = *reinterpret_cast<ScoreCluster*>(dyn + kSlots * kThreads * 16);
  const int blocks = 1 << log_blocks, rank = blockIdx.x & (blocks - 1);
  const unsigned nth = (blockIdx.x >> log_blocks) * Tm::kPerBlock + Tm::slot();
  if (kThreads == 32 && nth >= rows) return;           // a whole warp, and no cluster
  const unsigned r0 = rows - 1 - nth;
  if (blocks > 1) cluster_arrive();                    // the blocks of the cluster have begun
  const Row<T> row(a, r0);
  const Share<T> share(row, rank, log_blocks, Tm::tid());
  Ring<T, kThreads> ring(slots, row, share);
  uint32_t at = ring.buf;
  constexpr uint32_t kHalf = kBatch * kThreads * 16;
  ring.ask(at);
  ring.ask(at + kHalf);
  // single entries and the first given ones are fetched while the row is on its way
  float edge = neg_inf();
  if (share.edge >= 0) edge = row.at(share.edge);
  long long given[2];
  float given_z[2];
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const int k = Tm::tid() + q * kThreads;
    given[q] = -1;
    given_z[q] = 0.f;
    if (rank == 0 && k < o.n_targets) given[q] = o.targets[row.index * o.n_targets + k];
  }
  auto fetch_given = [&]() {
#pragma unroll
    for (int q = 0; q < 2; ++q)
      if (given[q] >= 0 && given[q] < row.size) given_z[q] = row.at((int)given[q]);
  };
  if (ring.n == 0) fetch_given();
  Sums sum{neg_inf(), 0.f, 0.f};
  typename Vec<T>::Max tops[kBatch];
#pragma unroll
  for (int u = 0; u < kBatch; ++u) tops[u] = Vec<T>::lowest();
  const bool keep = kMask && share.end - share.begin <= kSlots * kThreads;
  typename Row<T>::MaskBytes ahead[kBatch];       // of the next batch
  auto fetch_mask = [&](int i) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i + u < ring.n)
        ahead[u] = row.mask_bytes(share.begin + (i + u) * kThreads + Tm::tid());
  };
  if (kMask) fetch_mask(0);
#pragma unroll 1
  for (int i = 0; i < ring.n; i += kBatch) {
    cp_async_wait<1>();
    uint4 r[kBatch];
    read_batch<kThreads>(at, r);
    if (kMask) {
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i + u < ring.n) Row<T>::apply_mask(r[u], ahead[u]);
      fetch_mask(i + kBatch);
      if (keep) write_batch<kThreads>(at, r);
    }
    typename Vec<T>::Max most = Vec<T>::wide_max(r[0]);
    tops[0] = Vec<T>::larger(tops[0], most);
#pragma unroll
    for (int u = 1; u < kBatch; ++u) {
      const typename Vec<T>::Max t = Vec<T>::wide_max(r[u]);
      tops[u] = Vec<T>::larger(tops[u], t);
      most = Vec<T>::larger(most, t);
    }
    const float all = Vec<T>::to_max(most);
    // `all` has every vector in it: they are in registers before their slots are filled again
    asm volatile("" ::"f"(all) : "memory");
    ring.ask(at);
    at = at == ring.buf ? at + kHalf : ring.buf;
    accumulate<T, kBatch, true, kMask>(r, all, a.c, sum);
    if (i == 0) fetch_given();
  }
  // entries of -inf, or a maximum as low as the fill value
  if (sum.t != sum.t || !((sum.m - fill_value<T>()) * a.c > 64.f))
    sum = careful_sums<T, kThreads, kMask>(row, share, a.c);
  if (share.edge >= 0) sum = join(sum, single(edge, a.c), a.c);
  cp_async_wait<0>();
  sum = team_sums<kThreads>(sum, a.c, sh.red);
  int n = 0;
  if (o.top_k > 0) {
    float top[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) top[u] = Vec<T>::to_max(tops[u]);
    n = collect_top<T, kThreads, kMask>(row, share, ring, edge, top, o.top_k, sh.top);
  }
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
#pragma unroll 1
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
#pragma unroll 1
  for (int k = Tm::tid(), q = 0; k < o.n_targets; k += kThreads, ++q) {
    long long i = q == 0 ? given[0] : given[1];
    float z = q == 0 ? given_z[0] : given_z[1];
    if (q > 1) {
      i = o.targets[row.index * o.n_targets + k];
      if (i >= 0 && i < row.size) z = row.at((int)i);
    }
    float lp = z == neg_inf() ? z : (z - m) * a.inv_t - log_s;
    if (bad || i >= row.size) lp = quiet_nan();
    if (i < 0) lp = 0.f;
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
    return;
  }
  // Each block's list is sorted: a key's place is its own plus the larger ones of the
  // others. An empty place's key is 0; it ranks behind all others, by its list and place.
  for (int i = Tm::tid(); i < blocks * o.top_k; i += kThreads) {
    const int b = i / o.top_k;
    const unsigned long long key = cl.keys[b][i - b * o.top_k];
    int at = i - b * o.top_k;
    for (int q = 0; q < blocks && at < o.top_k; ++q) {
      if (q == b) continue;
      int lo = 0, hi = o.top_k;                    // places with a larger key (empty: as large)
      while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (cl.keys[q][mid] > key || (!key && (cl.keys[q][mid] || q < b))) lo = mid + 1;
        else hi = mid;
      }
      at += lo;
    }
    if (at < o.top_k) put(at, key);
  }
}

// The gradient of a row without a distribution: NaN, and 0 where an entry does
// not take part.
template <typename T, int kThreads, bool kMask>
__device__ __noinline__ void fill_bad(const Row<T>& row, const Share<T>& share) {
  constexpr int N = Vec<T>::N;
#pragma unroll 1
  for (int j = share.begin + Team<kThreads>::tid(); j < share.end; j += kThreads) {
    uint4 r = *reinterpret_cast<const uint4*>(row.vec(j));
    if (kMask) row.apply_mask(r, j);
    float z[N];
    Vec<T>::unpack(r, z);
#pragma unroll
    for (int e = 0; e < N; ++e) z[e] = z[e] == neg_inf() ? 0.f : quiet_nan();
    row.store(j, z, false);
  }
}

// ------------------------------------------------------- and their gradient
// dz_v = (q_v (a - g_H (log q_v + H)) + sum of the incoming gradients at v) / T
// with a = g_norm - the sum of all incoming gradients of single entries. With
// the forward's m and s that is e (A + B x) for the first term: one
// exponential and two products per entry, and no reduction over the row. Bound
// by memory: a read and a write, 537 MB in about 85 us at 2,048 x 65,536 bf16,
// 6.3 TB/s. The first vectors are on their way while the list is read.
// Single entries with a gradient of their own are written again at the end, each
// by one thread that adds up its gradients in the order of the list.
// Dynamic shared memory: per team the spots' sorted keys and their gradients.
template <typename T, int kThreads, bool kMask>
__global__ void __launch_bounds__(Team<kThreads>::kBlock)
log_probs_grad_kernel(const __grid_constant__ Rows a, const ScoreGradArgs o, unsigned rows,
                      int log_blocks) {
  using Tm = Team<kThreads>;
  constexpr int N = Vec<T>::N, kVecs = 4;
  extern __shared__ uint32_t spots[];
  __shared__ float red[Tm::kPerBlock][Tm::kWarps];
  const unsigned r0 = (blockIdx.x >> log_blocks) * Tm::kPerBlock + Tm::slot();
  if (kThreads == 32 && r0 >= rows) return;
  const Row<T> row(a, r0);
  const Share<T> share(row, blockIdx.x & ((1 << log_blocks) - 1), log_blocks, Tm::tid());
  uint4 r[kVecs];
  auto fetch = [&](int j0) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i)
      if (j0 + i * kThreads < share.end)
        r[i] = __ldcs(reinterpret_cast<const uint4*>(row.vec(j0 + i * kThreads)));
  };
  fetch(share.begin + Tm::tid());
  const int nt = o.g_log_probs ? o.n_targets : 0, n = nt + (o.g_top ? o.top_k : 0);
  const int keys = sort_size(n);
  uint32_t* key = spots + Tm::slot() * (keys + n);
  float* g = reinterpret_cast<float*>(key + keys);
  const float m = o.stats[2 * row.index], s = o.stats[2 * row.index + 1];
  float sum = 0.f;
#pragma unroll 1
  for (int k = Tm::tid(); k < n; k += kThreads) {
    const bool given = k < nt;
    const long long i = given ? o.targets[row.index * o.n_targets + k]
                              : o.top_indices[row.index * o.top_k + k - nt];
    float gk = given ? o.g_log_probs[row.index * o.n_targets + k]
                     : o.g_top[row.index * o.top_k + k - nt];
    const bool past = i >= row.size;
    if (past) gk = quiet_nan();
    else if (i < 0 || row.at((int)i) == neg_inf()) gk = 0.f;
    key[k] = place_key(past ? -1 : (int)i, k);
    g[k] = gk;
    sum += gk;
  }
  for (int k = n + Tm::tid(); k < keys; k += kThreads) key[k] = kNoKey;
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
  const bool fine = A == A, vec_store = row.vec_store();
  const float2 nm = {-m, -m}, cc = {a.c, a.c}, aa = {A, A}, bb = {B, B};
  auto value = [&](float2 z) {
    float2 x = __fmul2_rn(__fadd2_rn(z, nm), cc);
    x.x = fmaxf(x.x, -1000.f);
    x.y = fmaxf(x.y, -1000.f);
    return __fmul2_rn(float2{ex2(x.x), ex2(x.y)}, __ffma2_rn(bb, x, aa));
  };
  if (fine) {
#pragma unroll 1
    for (int j0 = share.begin + Tm::tid(); j0 < share.end; j0 += kVecs * kThreads) {
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int j = j0 + i * kThreads;
        if (j >= share.end) break;
        if (kMask) row.apply_mask(r[i], j);
        float z[N];
        Vec<T>::unpack(r[i], z);
#pragma unroll
        for (int e = 0; e < N; e += 2) {
          const float2 d = value(float2{z[e], z[e + 1]});
          z[e] = d.x;
          z[e + 1] = d.y;
        }
        row.store(j, z, vec_store);
      }
      fetch(j0 + kVecs * kThreads);
    }
  } else {
    fill_bad<T, kThreads, kMask>(row, share);
  }
  auto put = [&](int v, float more) {
    const float z = row.at(v);
    const float d = fmaf(more, a.inv_t, value(float2{z, z}).x);
    row.grad[v] = to_type<T>(z == neg_inf() ? 0.f : fine ? d : quiet_nan());
  };
  if (share.edge >= 0) put(share.edge, 0.f);
  if (n == 0) return;
  sort_places<kThreads>(key, keys);               // and the entries are written before they are again
#pragma unroll 1
  for (int k = Tm::tid(); k < n; k += kThreads) {
    const int v = key_entry(key[k]);
    if (v < share.first || v >= share.last || (k > 0 && key_entry(key[k - 1]) == v)) continue;
    float at = 0.f, part = g[key_place(key[k])];
    for (int q = k + 1; q < n && key_entry(key[q]) == v; ++q) {
      if ((q - k) % 32 == 0) {                    // few roundings in a row
        at += part;
        part = 0.f;
      }
      part += g[key_place(key[q])];
    }
    at += part;
    put(v, at);
  }
}

// ------------------------------------------------------------ distillation
// Shared memory of one team, in this order (dynamic): one or two chunks; p,
// logits, indices of the list; a bit per entry of the row (modulo kSeenBits),
// or the list's keys when they are sorted.
constexpr int kSeenBits = 1 << 15;
__host__ __device__ constexpr int seen_words(int size) {
  return ((size < kSeenBits ? size : kSeenBits) + 31) / 32;
}
__host__ __device__ constexpr int distill_bytes(int listed, int cap, int chunks, int largest) {
  const int words = seen_words(largest), keys = sort_size(listed);
  return chunks * cap * 16 + 16 * listed + ((words > keys ? words : keys) * 4 + 15) / 16 * 16;
}

template <typename T> __device__ __forceinline__ void sts_neg_inf(uint32_t a) {
  if constexpr (sizeof(T) == 4)
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(Vec<T>::kNegInf) : "memory");
  else
    asm volatile("st.shared.u16 [%0], %1;" ::"r"(a), "h"((uint16_t)Vec<T>::kNegInf) : "memory");
}

// Per warp: what the list adds up to.
struct ListSums {
  double mass, p_log_p, p_z;       // sum P, P log P, P z'
  float e;                         // sum exp(z')
  float top_z, top_lp;             // the warp's largest z, log P: z' and P are relative to them
};
// What a warp's part of the list (entries first, first + step, ... of its lanes)
// adds up to; p becomes P from log P.
static __device__ __noinline__ ListSums list_sums(double* p, const float* zu, const int* idx, int K,
                                           int first, int step, int renormalize, double inv_t) {
  float top_lp = neg_inf(), top_z = neg_inf();
#pragma unroll 1
  for (int k = first; k < K; k += step)
    if (idx[k] >= 0) {
      top_lp = fmaxf(top_lp, (float)p[k]);
      top_z = fmaxf(top_z, zu[k]);
    }
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) {
    top_lp = fmaxf(top_lp, __shfl_xor_sync(0xffffffffu, top_lp, w));
    top_z = fmaxf(top_z, __shfl_xor_sync(0xffffffffu, top_z, w));
  }
  if (!renormalize || top_lp == neg_inf()) top_lp = 0.f;
  ListSums ls{0.0, 0.0, 0.0, 0.f, top_z, top_lp};
#pragma unroll 1
  for (int k = first; k < K; k += step) {
    if (idx[k] < 0) continue;
    const double lp = p[k] - (double)top_lp, pk = exp64(lp);
    const double zp = ((double)zu[k] - (double)top_z) * inv_t;
    p[k] = pk;
    ls.mass += pk;
    if (pk > 0.0) {
      ls.p_log_p += pk * lp;
      ls.p_z += pk * zp;
    }
    ls.e += expf((float)zp);
  }
#pragma unroll 1
  for (int w = 16; w > 0; w >>= 1) {
    ls.mass += __shfl_xor_sync(0xffffffffu, ls.mass, w);
    ls.p_log_p += __shfl_xor_sync(0xffffffffu, ls.p_log_p, w);
    ls.p_z += __shfl_xor_sync(0xffffffffu, ls.p_z, w);
    ls.e += __shfl_xor_sync(0xffffffffu, ls.e, w);
  }
  return ls;
}

// The warps' parts of the list, relative to the largest z and log P of all;
// factor: of warp `mine`'s P to the common ones.
static __device__ __noinline__ ListSums join_list(const ListSums* part, int warps, int mine, double inv_t,
                                           float* factor) {
  float top_z = neg_inf(), top_lp = neg_inf();
  for (int w = 0; w < warps; ++w) {
    top_z = fmaxf(top_z, part[w].top_z);
    if (part[w].mass > 0.0) top_lp = fmaxf(top_lp, part[w].top_lp);
  }
  ListSums ls{0.0, 0.0, 0.0, 0.f, top_z, top_lp};
#pragma unroll 1
  for (int w = 0; w < warps; ++w) {
    const ListSums b = part[w];
    const double up = b.mass > 0.0 ? (double)b.top_lp - (double)top_lp : 0.0;
    const double f = up == 0.0 ? 1.0 : exp64(up);
    const double zp =
        b.top_z == neg_inf() ? 0.0 : ((double)b.top_z - (double)top_z) * inv_t;
    if (w == mine) *factor = (float)f;
    ls.mass += f * b.mass;
    if (b.mass > 0.0) {
      ls.p_log_p += f * (b.p_log_p + up * b.mass);
      ls.p_z += f * (b.p_z + zp * b.mass);
    }
    ls.e += b.e * expf((float)zp);
  }
  return ls;
}

// A list in which an entry may be twice: the first one takes the others' mass
// (p: log P before and after), the others leave the list. Marks can coincide
// without a repeat, so there may be none.
template <int kThreads>
__device__ __noinline__ void merge_list(double* p, int* idx, uint32_t* key, int K) {
  using Tm = Team<kThreads>;
  const int n = sort_size(K);
  for (int k = Tm::tid(); k < n; k += kThreads) key[k] = k < K ? place_key(idx[k], k) : kNoKey;
  sort_places<kThreads>(key, n);
#pragma unroll 1
  for (int k = Tm::tid(); k + 1 < K; k += kThreads) {
    const int v = key_entry(key[k]);
    if (key[k] == kNoKey || key_entry(key[k + 1]) != v || (k > 0 && key_entry(key[k - 1]) == v))
      continue;
    const int first = key_place(key[k]);
    double top = p[first], mass = 0.0;
    for (int q = k + 1; q < K && key_entry(key[q]) == v; ++q)
      top = fmax(top, p[key_place(key[q])]);
    for (int q = k; q < K && key_entry(key[q]) == v; ++q) {
      const int at = key_place(key[q]);
      mass += exp64(p[at] - top);
      if (q > k) idx[at] = -1;
    }
    if (top > (double)neg_inf()) p[first] = top + log(mass);
  }
  Tm::sync();
}

// The list's entries are overwritten by -inf in shared memory before the one
// pass over the row, so that pass gives maximum and sum over the rest alone,
// without a difference of nearly equal numbers; the teacher's masses are added
// in 64 bits, for the rest's is 1 minus their sum. With lse_R, lse the logs of
// the two normalisers and q_R = exp(lse_R - lse)
//   dz_v = T w exp(z'_v - lse_R) (q_R - P_rest)     outside the list
//   dz_u = T w (exp(z'_u - lse) - P_u)              in it
// so the gradient is one more exponential per entry in shared memory, and
// q_R - P_rest = P_list - q_list where the rest has most of the mass. Without
// a gradient the chunks are small and there are two, one on its way.
// The first warps add up the list while the others begin with the row.
//
// 8,192 x 32,768 bf16 with 64 listed: 220 us, 4.9 TB/s read and written. DRAM
// would take 165, the exponential unit 133 (two e^x an entry) and the issue
// slots 132; with three blocks to an SM one loads while another computes, but
// not all the time. A block that went from row to row and asked for the next
// early took 255. Without a gradient 1,024 x 100,003 fp32 with 100 listed take
// 85 us, 4.9 TB/s; every row has a block at once, and with it the barriers of its
// chunks. 1,024 x 1,000 fp32 with 32 listed take 9 us, the latency of one row.
// At least three blocks of 256 to an SM, which 64 KB of shared memory allow, and
// seven of 128.
// kLong joins the sums of kMaxBatches chunks to those before; as part of every kernel it costs
// registers (1,024 x 100,003 fp32 loss alone 89 us instead of 85).
template <typename T, int kThreads, bool kMask, bool kLong = false>
__global__ void
__launch_bounds__(Team<kThreads>::kBlock, kThreads == 256 ? 3 : kThreads == 128 ? 7 : 5)
distill_kernel(const __grid_constant__ Rows a, const DistillArgs o, unsigned rows, int log_blocks,
               int cap, int chunks, int team_bytes) {
  using Tm = Team<kThreads>;
  constexpr int N = Vec<T>::N;
  extern __shared__ __align__(16) unsigned char dyn[];
  __shared__ Sums red[Tm::kPerBlock][Tm::kWarps];
  __shared__ ListSums lred[Tm::kPerBlock][Tm::kWarps];
  __shared__ int flags[Tm::kPerBlock][Tm::kWarps];
  __shared__ float cl[kMaxCluster][2];            // every block's maximum and sum
  const int slot = Tm::slot(), K = o.n_listed;
  const int blocks = 1 << log_blocks, rank = blockIdx.x & (blocks - 1);
  const unsigned nth = (blockIdx.x >> log_blocks) * Tm::kPerBlock + slot;
  if (kThreads == 32 && nth >= rows) return;
  const unsigned r0 = o.upstream ? nth : rows - 1 - nth;
  if (blocks > 1) cluster_arrive();
  unsigned char* mine = dyn + slot * team_bytes;
  const uint32_t chunk = smem_u32(mine);
  // 1 / T as the exponentials have it: rounded with log2(e) in a.c, the same everywhere, so that
  // loss and gradient are those of one temperature, off by half a step of fp32
  const double inv_t = (double)a.c * 0.69314718055994531;
  double* p = reinterpret_cast<double*>(mine + chunks * cap * 16);
  float* zu = reinterpret_cast<float*>(p + K);
  int* idx = reinterpret_cast<int*>(zu + K);
  uint32_t* seen = reinterpret_cast<uint32_t*>(idx + K);
  const int load_warps = min(Tm::kWarps, (K + 31) / 32);    // they have entries to load
  // they add the list up: a power of two, about 128 entries to each
  const int list_warps = K == 0 ? 0 : min(Tm::kWarps, K <= 128 ? 1 : 1 << (32 - __clz((K - 1) / 128)));
  const Row<T> row(a, r0);
  const Share<T> share(row, rank, log_blocks, Tm::tid());
  const bool one = share.end - share.begin <= cap, vec_store = row.vec_store();
  const float weight = o.weight ? o.weight[row.index] : 1.f;
  copy_chunk<T, kThreads>(chunk, row, share.begin,
                          own_vectors<kThreads>(share.begin, min(share.begin + cap, share.end)));
  if (weight == 0.f) {                            // nothing of the row is looked at
    cp_async_wait<0>();
    if (o.row_loss && rank == 0 && Tm::tid() == 0) o.row_loss[row.index] = 0.f;
    if (row.grad) {
      float zero[N];
#pragma unroll
      for (int e = 0; e < N; ++e) zero[e] = 0.f;
      for (int j = share.begin + Tm::tid(); j < share.end; j += kThreads)
        row.store(j, zero, vec_store);
      if (share.edge >= 0) row.grad[share.edge] = to_type<T>(0.f);
    }
    if (blocks > 1) cluster_wait();
    return;
  }
  uint32_t flag = 0;              // 1: a bad entry of the list; 2: one there twice, or so it seems
  // While the row is on its way: the list, an entry to a thread.
#pragma unroll 1
  for (int k = Tm::tid(); k < K; k += kThreads) {
    const long long i = o.indices[row.index * K + k];
    const float lp = o.log_probs[row.index * K + k];
    const float z = i >= 0 && i < row.size ? row.at((int)i) : neg_inf();
    const bool there = z != neg_inf();
    if (i >= row.size || (there && !(lp < -neg_inf()))) flag = 1u;
    idx[k] = there ? (int)i : -1;
    zu[k] = z;
    p[k] = (double)lp;
  }
  const int words = seen_words(row.size);
  for (int w = Tm::tid(); w < words; w += kThreads) seen[w] = 0u;
  typename Row<T>::MaskBytes ahead[kBatch];       // the first batch's mask
  auto fetch_mask = [&](int base, int i, int n) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (i + u < n) ahead[u] = row.mask_bytes(base + (i + u) * kThreads + Tm::tid());
  };
  if (kMask)
    fetch_mask(share.begin, 0,
               own_vectors<kThreads>(share.begin, min(share.begin + cap, share.end)));
  Tm::sync();                                     // the marks are clear
  if (Tm::warp() < load_warps) {
#pragma unroll 1
    for (int k = Tm::tid(); k < K; k += kThreads) {
      const int v = idx[k] & (kSeenBits - 1);
      if (idx[k] >= 0 && ((atomicOr(&seen[v >> 5], 1u << (v & 31)) >> (v & 31)) & 1u)) flag |= 2u;
    }
    flag = __reduce_or_sync(0xffffffffu, flag);
    if (Tm::lane() == 0) flags[slot][Tm::warp()] = flag;
  }
  // the rest of the row
  Sums sum{neg_inf(), 0.f, 0.f}, before = sum;
  uint32_t now = chunk;
#pragma unroll 1
  for (int base = share.begin; base < share.end || base == share.begin; base += cap) {
    const int end = min(base + cap, share.end), n = own_vectors<kThreads>(base, end);
    const int next = base + cap;
    if (chunks > 1 && next < share.end) {
      copy_chunk<T, kThreads>(2 * chunk + cap * 16 - now, row, next,
                              own_vectors<kThreads>(next, min(next + cap, share.end)));
      cp_async_wait<1>();
    } else {
      if (chunks == 1 && base != share.begin) copy_chunk<T, kThreads>(chunk, row, base, n);
      cp_async_wait<0>();
    }
    if (kMask && base != share.begin) fetch_mask(base, 0, n);
    Tm::sync();                                   // the whole chunk is there
    const int first = row.head + base * N, last = first + (end - base) * N;
#pragma unroll 1
    for (int k = Tm::tid(); k < K; k += kThreads) {
      const int v = idx[k];
      if (v >= first && v < last) sts_neg_inf<T>(now + (v - first) * (int)sizeof(T));
    }
    Tm::sync();
    if (base == share.begin && Tm::warp() < list_warps) {
      const ListSums ls = list_sums(p, zu, idx, K, Tm::tid(), 32 * list_warps, o.renormalize, inv_t);
      if (Tm::lane() == 0) lred[slot][Tm::warp()] = ls;
    }
    uint32_t at = now + Tm::tid() * 16;
#pragma unroll 1
    for (int i = 0; i < n; i += kBatch) {
      uint4 r[kBatch];
      read_batch<kThreads>(at, r);
      if (kMask) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
          if (i + u < n) Row<T>::apply_mask(r[u], ahead[u]);
        fetch_mask(base, i + kBatch, n);
        write_batch<kThreads>(at, r);
      }
      at += kBatch * kThreads * 16;
      typename Vec<T>::Max most = Vec<T>::wide_max(r[0]);
#pragma unroll
      for (int u = 1; u < kBatch; ++u) most = Vec<T>::larger(most, Vec<T>::wide_max(r[u]));
      accumulate<T, kBatch, false, false>(r, Vec<T>::to_max(most), a.c, sum);
    }
    if (chunks > 1) now = 2 * chunk + cap * 16 - now;
    if (kLong && (next - share.begin) % (kMaxBatches * kBatch * kThreads) == 0) {
      before = join(before, sum, a.c);
      sum = {neg_inf(), 0.f, 0.f};
    }
  }
  if (kLong) sum = join(before, sum, a.c);
  float edge = neg_inf();
  if (Tm::warp() == 0 && row.size != row.nin * N) {
    // which single entries are listed: a bit per thread that may have one
    if (share.edge >= 0) edge = row.at(share.edge);
    const int tail = row.head + row.nin * N;
    uint32_t in = 0;
    for (int k = Tm::lane(); k < K; k += 32) {
      const int v = idx[k];
      if (v >= 0 && v < row.head) in |= 1u << v;
      else if (v >= tail) in |= 1u << (N + v - tail);
    }
    in = __reduce_or_sync(0xffffffffu, in);
    if (share.edge >= 0 && !((in >> Tm::tid()) & 1u)) sum = join(sum, single(edge, a.c), a.c);
  }
  int all = 0;
  for (int w = 0; w < load_warps; ++w) all |= flags[slot][w];
  if (all & 2) {                                  // an entry listed twice counts once
    Tm::sync();
    for (int k = Tm::tid(); k < K; k += kThreads) p[k] = (double)o.log_probs[row.index * K + k];
    Tm::sync();
    merge_list<kThreads>(p, idx, seen, K);
    if (Tm::warp() < list_warps) {
      const ListSums ls = list_sums(p, zu, idx, K, Tm::tid(), 32 * list_warps, o.renormalize, inv_t);
      if (Tm::lane() == 0) lred[slot][Tm::warp()] = ls;
    }
  }
  sum = team_sums<kThreads>(sum, a.c, red[slot]);   // orders lred and p, too (a barrier, or one warp)
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
#pragma unroll 1
    for (int b = 1; b < blocks; ++b) sum = join(sum, Sums{cl[b][0], cl[b][1], 0.f}, a.c);
  }
  // P of the entries that this thread writes is warp (k / 32 mod list_warps)'s
  float factor = 1.f;
  ListSums ls{0.0, 0.0, 0.0, 0.f, neg_inf(), 0.f};
  if (list_warps == 1) ls = lred[slot][0];
  else if (list_warps > 1)
    ls = join_list(lred[slot], list_warps, Tm::warp() % list_warps, inv_t, &factor);
  const bool rest = sum.m != neg_inf(), listed = ls.top_z != neg_inf();
  const bool bad = (all & 1) || sum.s != sum.s || ls.e != ls.e || ls.mass != ls.mass;
  const bool whole = o.renormalize || ls.mass > 1.0 || !rest;
  const float p_r = whole ? 0.f : (float)(1.0 - ls.mass);
  const bool live = (rest || listed) && (ls.mass > 0.0 || !whole);
  // the two normalisers relative to the larger of the two maxima
  const float big = fmaxf(rest ? sum.m : neg_inf(), ls.top_z);
  const float norm_r = rest ? sum.s * ex2((sum.m - big) * a.c) : 0.f;
  const float norm_u = listed ? ls.e * ex2((ls.top_z - big) * a.c) : 0.f;
  const float inv_norm = __fdividef(1.f, norm_r + norm_u);
  // q_R - P_rest, from the complements where those are the smaller numbers: as the difference
  // of two numbers near 1 it would keep no digits of a list with little mass
  const float over =
      p_r > 0.5f ? (float)ls.mass - norm_u * inv_norm : norm_r * inv_norm - p_r;
  const float scaled = weight * o.scale *
                       (o.upstream ? o.upstream[row.index * o.upstream_stride] : 1.f);
  // by the last warp, when the others are done; a function call to a lane
  auto write_loss = [&]() {
    if (rank != 0 || Tm::warp() != Tm::kWarps - 1 || !o.row_loss) return;
    const int lane = Tm::lane();
    const double down_r = rest ? ((double)sum.m - (double)big) * inv_t : 0.0;
    const double down_u = listed ? ((double)ls.top_z - (double)big) * inv_t : 0.0;
    const double rest_mass = whole ? 0.0 : 1.0 - ls.mass;
    double e = exp64(lane == 0 ? down_r : down_u);          // 0: the rest, 1: the list
    e *= lane == 0 ? (rest ? (double)sum.s : 0.0) : (listed ? (double)ls.e : 0.0);
    const double norm64 = __shfl_sync(0xffffffffu, e, 0) + __shfl_sync(0xffffffffu, e, 1);
    const double l = log(lane == 0 ? norm64 : lane == 1 ? ls.mass : lane == 2 ? rest_mass
                                                                              : (double)sum.s);
    const double log_all = __shfl_sync(0xffffffffu, l, 0), log_mass = __shfl_sync(0xffffffffu, l, 1);
    const double log_p_r = __shfl_sync(0xffffffffu, l, 2), log_s = __shfl_sync(0xffffffffu, l, 3);
    double loss = 0.0;
    if (live && ls.mass > 0.0) {
      loss = ls.p_log_p - ls.p_z + (log_all - down_u) * ls.mass;
      if (whole) loss = loss / ls.mass - log_mass;
    }
    if (live && rest_mass > 0.0) loss += rest_mass * (log_p_r - (down_r + log_s - log_all));
    if (lane == 0)
      o.row_loss[row.index] =
          bad ? quiet_nan() : (float)(loss * (double)a.t * (double)a.t * (double)scaled);
  };
  if (!row.grad) {
    write_loss();
    return;
  }
  const float scale = live ? scaled * a.t : 0.f, ref = rest ? sum.m : 0.f;
  const float coef = live && rest ? __fdividef(scale * over, sum.s) : 0.f;
  const float nan = bad || coef != coef ? quiet_nan() : 0.f;   // of a row without a distribution
  const float2 nref = {-ref, -ref}, cc = {a.c, a.c}, kk = {coef, coef};
  auto slope = [&](const uint4& r, int j) {
    float z[N];
    Vec<T>::unpack(r, z);
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const float2 x = __fmul2_rn(__fadd2_rn(float2{z[e], z[e + 1]}, nref), cc);
      const float2 g = __fmul2_rn(float2{ex2(x.x), ex2(x.y)}, kk);
      z[e] = g.x;
      z[e + 1] = g.y;
    }
    row.store(j, z, vec_store);
  };
  if (nan == 0.f) {
#pragma unroll 1
    for (int base = share.begin; base < share.end; base += cap) {
      const int n = own_vectors<kThreads>(base, min(base + cap, share.end));
      if (!one) {
        copy_chunk<T, kThreads>(chunk, row, base, n);
        cp_async_wait<0>();
      }
      uint32_t at = chunk + Tm::tid() * 16;
      int j = base + Tm::tid();
#pragma unroll 1
      for (int i = 0; i < n; i += kBatch) {
        uint4 r[kBatch];
        read_batch<kThreads>(at, r);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
          if (i + u >= n) break;
          if (kMask && !one) row.apply_mask(r[u], j + u * kThreads);
          slope(r[u], j + u * kThreads);
        }
        at += kBatch * kThreads * 16;
        j += kBatch * kThreads;
      }
    }
  } else {
    fill_bad<T, kThreads, kMask>(row, share);
  }
  if (share.edge >= 0)
    row.grad[share.edge] =
        to_type<T>(edge == neg_inf() ? 0.f : nan + ex2((edge - ref) * a.c) * coef);
  if (K > 0) Tm::sync();                          // the listed entries are written again
  if (Tm::warp() < load_warps) {
    const double inv = whole && ls.mass > 0.0 ? (double)factor / ls.mass : (double)factor;
#pragma unroll 1
    for (int k = Tm::tid(); k < K; k += kThreads) {
      const int v = idx[k];
      if (v < share.first || v >= share.last) continue;
      const float q = ex2((zu[k] - big) * a.c) * inv_norm;
      row.grad[v] = to_type<T>(nan + scale * (q - (float)(p[k] * inv)));
    }
  }
  write_loss();
}

// Sum of the rows' losses by one block, in 64 bits and a fixed order.
static __global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ row_loss,
                                                               long long n,
                                                               float* __restrict__ loss) {
  __shared__ double red[32];
  griddep_wait();
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
