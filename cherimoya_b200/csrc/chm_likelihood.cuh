// chm_likelihood.cuh -- softmax rows over the profile logits of a signal
// group: log probabilities of given entries with entropy and top entries,
// their gradient, and distillation from a teacher's listed entries.
//
// Notation: z the row's logits, x = (z - m) / T * log2(e) <= 0 with m the
// row's maximum, e = 2^x, s = sum e. Entries that are masked or -inf count as
// -inf throughout. z - m is formed before the scaling, so logits near the
// type's largest or lowest value neither overflow nor lose the row.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace chm {
namespace lk {

constexpr int kMaxGroups = 64;      // groups of one launch (kernel parameters)
constexpr int kMaxList = 1024;      // given / listed entries per row
constexpr int kMaxTop = 128;

struct Rows {
  const void* z;
  const uint8_t* mask;
  void* grad;
  long long row_stride, mask_stride, grad_stride;
  int n_groups, g0, ng;             // groups in all; this launch's first and count
  float c;                          // log2(e) / T
  float inv_t, t;
  long long off[kMaxGroups], moff[kMaxGroups], goff[kMaxGroups];
  int size[kMaxGroups];
};

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

// One row of the launch: pointers, length and its index in the per-row arrays.
template <typename T>
struct Row {
  const T* z;
  const uint8_t* mask;
  T* grad;
  int size;
  long long index;
  __device__ __forceinline__ Row(const Rows& a, unsigned r) {
    const unsigned n = r / (unsigned)a.ng, g = r - n * (unsigned)a.ng;
    z = static_cast<const T*>(a.z) + n * a.row_stride + a.off[g];
    mask = a.mask ? a.mask + n * a.mask_stride + a.moff[g] : nullptr;
    grad = a.grad ? static_cast<T*>(a.grad) + n * a.grad_stride + a.goff[g] : nullptr;
    size = a.size[g];
    index = (long long)n * a.n_groups + a.g0 + g;
  }
  __device__ __forceinline__ float at(int v) const {
    return (mask && !mask[v]) ? neg_inf() : to_float(z[v]);
  }
};

// Block reductions through shared memory in a fixed order (the same answer on
// every run). `red` holds one value per warp; every thread gets the result.
template <typename V, typename Op>
__device__ __forceinline__ V block_reduce(V v, V* red, Op op) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  V r = red[0];
  for (int w = 1; w < warps; ++w) r = op(r, red[w]);
  return r;
}
struct Max { template <typename V> __device__ V operator()(V a, V b) const { return a > b ? a : b; } };
struct Sum { template <typename V> __device__ V operator()(V a, V b) const { return a + b; } };

// Larger logit first, then the lower index; entries without probability are 0.
__device__ __forceinline__ unsigned long long order_key(float z, int v) {
  if (!(z > neg_inf())) return 0ull;
  z += 0.f;                                       // -0 orders as +0
  unsigned b = __float_as_uint(z);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((unsigned long long)b << 32) | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
  unsigned b = (unsigned)(key >> 32);
  b = (b & 0x80000000u) ? (b & 0x7fffffffu) : ~b;
  return __uint_as_float(b);
}
__device__ __forceinline__ int key_index(unsigned long long key) {
  return (int)(0xffffffffu - (unsigned)key);
}

// ------------------------------------------------------- log probabilities
struct ScoreArgs {
  const long long* targets;
  int n_targets, top_k;
  float *log_probs, *entropy, *log_norm, *top_log_probs;
  long long* top_indices;
  float* stats;
};

template <typename T>
__global__ void __launch_bounds__(256) log_probs_kernel(Rows a, ScoreArgs o) {
  __shared__ float red[8];
  __shared__ unsigned long long kred[8];
  const Row<T> row(a, blockIdx.x);
  float m = neg_inf();
  for (int v = threadIdx.x; v < row.size; v += blockDim.x) m = fmaxf(m, row.at(v));
  m = block_reduce(m, red, Max());
  if (m == neg_inf()) m = 0.f;
  float s = 0.f, t = 0.f;
  for (int v = threadIdx.x; v < row.size; v += blockDim.x) {
    const float x = (row.at(v) - m) * a.c;
    const float e = exp2f(x);
    s += e;
    t += e * fmaxf(x, -1000.f);                   // e = 0 there; keeps 0 * -inf out
  }
  s = block_reduce(s, red, Sum());
  t = block_reduce(t, red, Sum());
  const float kLn2 = 0.69314718f;
  const float log_s = logf(s), lse = m * a.inv_t + log_s;
  if (threadIdx.x == 0) {
    if (o.entropy) o.entropy[row.index] = s == 0.f ? 0.f : log_s - kLn2 * (t / s);
    if (o.log_norm) o.log_norm[row.index] = lse;
    if (o.stats) {
      o.stats[2 * row.index] = m;
      o.stats[2 * row.index + 1] = log_s;
    }
  }
  for (int k = threadIdx.x; k < o.n_targets; k += blockDim.x) {
    const long long i = o.targets[row.index * o.n_targets + k];
    float lp = 0.f;
    if (i >= row.size || s != s) {
      lp = i < 0 ? 0.f : quiet_nan();
    } else if (i >= 0) {
      const float z = row.at((int)i);
      lp = z == neg_inf() ? z : (z - m) * a.inv_t - log_s;
    }
    o.log_probs[row.index * o.n_targets + k] = lp;
  }
  unsigned long long last = ~0ull;
  for (int k = 0; k < o.top_k; ++k) {
    unsigned long long best = 0;
    for (int v = threadIdx.x; v < row.size; v += blockDim.x) {
      const unsigned long long key = order_key(row.at(v), v);
      if (key < last && key > best) best = key;
    }
    best = block_reduce(best, kred, Max());
    last = best;
    if (threadIdx.x == 0) {
      const bool bad = s != s;
      o.top_indices[row.index * o.top_k + k] = bad || !best ? -1 : key_index(best);
      o.top_log_probs[row.index * o.top_k + k] =
          bad ? quiet_nan() : !best ? neg_inf() : (key_logit(best) - m) * a.inv_t - log_s;
    }
  }
}

// dz_v = (q_v (a - g_H (log q_v + H)) + sum of the incoming gradients at v) / T
// with a = g_norm - the sum of all incoming gradients of single entries.
struct ScoreGradArgs {
  const long long *targets, *top_indices;
  int n_targets, top_k;
  const float *stats, *entropy, *g_log_probs, *g_entropy, *g_log_norm, *g_top;
};

template <typename T>
__global__ void __launch_bounds__(256) log_probs_grad_kernel(Rows a, ScoreGradArgs o) {
  __shared__ float red[8];
  __shared__ int idx[kMaxList + kMaxTop];
  __shared__ float g[kMaxList + kMaxTop];
  const Row<T> row(a, blockIdx.x);
  const int nt = o.g_log_probs ? o.n_targets : 0, n = nt + (o.g_top ? o.top_k : 0);
  const float m = o.stats[2 * row.index], log_s = o.stats[2 * row.index + 1];
  float sum = 0.f;
  for (int k = threadIdx.x; k < n; k += blockDim.x) {
    const bool given = k < nt;
    const long long i = given ? o.targets[row.index * o.n_targets + k]
                              : o.top_indices[row.index * o.top_k + k - nt];
    float gk = given ? o.g_log_probs[row.index * o.n_targets + k]
                     : o.g_top[row.index * o.top_k + k - nt];
    if (i >= row.size) gk = quiet_nan();
    else if (i < 0 || row.at((int)i) == neg_inf()) gk = 0.f;
    idx[k] = i < 0 || i >= row.size ? -1 : (int)i;
    g[k] = gk;
    sum += gk;
  }
  sum = block_reduce(sum, red, Sum());            // orders the writes above, too
  const float acoef = (o.g_log_norm ? o.g_log_norm[row.index] : 0.f) - sum;
  const float gh = o.g_entropy ? o.g_entropy[row.index] : 0.f;
  const float h = o.g_entropy ? o.entropy[row.index] : 0.f;
  for (int v = threadIdx.x; v < row.size; v += blockDim.x) {
    const float z = row.at(v);
    float d = 0.f;
    if (z != neg_inf()) {
      const float lq = (z - m) * a.inv_t - log_s, q = expf(lq);
      d = q * acoef - (q > 0.f ? q * gh * (lq + h) : 0.f);
      for (int k = 0; k < n; ++k)
        if (idx[k] == v) d += g[k];
    }
    row.grad[v] = to_type<T>(d * a.inv_t);
  }
}

// ------------------------------------------------------------ distillation
struct DistillArgs {
  const long long* indices;
  const float* log_probs;
  int n_listed, renormalize;
  const float *weight, *upstream;
  float scale;
  int upstream_stride;
  float* row_loss;
};

// Dynamic shared memory: one bit per entry of the row (listed or not).
template <typename T>
__global__ void __launch_bounds__(256) distill_kernel(Rows a, DistillArgs o) {
  extern __shared__ unsigned bits[];
  __shared__ double p[kMaxList];
  __shared__ float zu[kMaxList];
  __shared__ int idx[kMaxList];
  __shared__ double dred[8];
  __shared__ float red[8];
  const Row<T> row(a, blockIdx.x);
  const int K = o.n_listed;
  float weight = o.weight ? o.weight[row.index] : 1.f;
  const bool off = weight == 0.f;
  weight *= o.scale;
  if (o.upstream) weight *= o.upstream[row.index * o.upstream_stride];
  if (off) {
    if (o.row_loss && threadIdx.x == 0) o.row_loss[row.index] = 0.f;
    if (row.grad)
      for (int v = threadIdx.x; v < row.size; v += blockDim.x) row.grad[v] = to_type<T>(0.f);
    return;
  }
  for (int w = threadIdx.x; w < (row.size + 31) / 32; w += blockDim.x) bits[w] = 0u;
  __syncthreads();
  bool bad = false, twice = false;
  float top_lp = neg_inf(), top_z = neg_inf();
  for (int k = threadIdx.x; k < K; k += blockDim.x) {
    const long long i = o.indices[row.index * K + k];
    const float lp = o.log_probs[row.index * K + k];
    const float z = i >= 0 && i < row.size ? row.at((int)i) : neg_inf();
    const bool there = z != neg_inf();
    bad |= i >= row.size || (there && !(lp < -neg_inf()));
    idx[k] = there ? (int)i : -1;
    zu[k] = z;
    p[k] = there ? (double)lp : (double)neg_inf();
    if (there) {
      top_lp = fmaxf(top_lp, lp);
      top_z = fmaxf(top_z, z);
      twice |= (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1u;
    }
  }
  bad = __syncthreads_or(bad);
  twice = __syncthreads_or(twice);
  top_lp = block_reduce(top_lp, red, Max());
  top_z = block_reduce(top_z, red, Max());
  const double shift = o.renormalize && top_lp > neg_inf() ? (double)top_lp : 0.0;
  for (int k = threadIdx.x; k < K; k += blockDim.x) p[k] = idx[k] < 0 ? 0.0 : exp(p[k] - shift);
  __syncthreads();
  if (twice) {                                    // an entry listed twice counts once
    if (threadIdx.x == 0)
      for (int k = 0; k < K; ++k)
        for (int j = k + 1; j < K; ++j)
          if (idx[k] >= 0 && idx[j] == idx[k]) {
            p[k] += p[j];
            idx[j] = -1;
            p[j] = 0.0;
          }
    __syncthreads();
  }
  double mass = 0.0;
  for (int k = threadIdx.x; k < K; k += blockDim.x) mass += p[k];
  mass = block_reduce(mass, dred, Sum());
  // the entries outside the list
  float m = neg_inf();
  for (int v = threadIdx.x; v < row.size; v += blockDim.x)
    if (!((bits[v >> 5] >> (v & 31)) & 1u)) m = fmaxf(m, row.at(v));
  m = block_reduce(m, red, Max());
  const bool rest = m != neg_inf();
  float s = 0.f;
  const float ref = rest ? m : 0.f;
  for (int v = threadIdx.x; v < row.size; v += blockDim.x)
    if (!((bits[v >> 5] >> (v & 31)) & 1u)) s += exp2f((row.at(v) - ref) * a.c);
  s = block_reduce(s, red, Sum());
  if (s != s) bad = true;
  // everything relative to the larger of the two maxima, in 64 bits
  const double T_ = a.t, big = fmaxf(m, top_z);
  double sum = 0.0;
  for (int k = threadIdx.x; k < K; k += blockDim.x)
    if (idx[k] >= 0) sum += exp(((double)zu[k] - big) / T_);
  sum = block_reduce(sum, dred, Sum());
  if (sum != sum) bad = true;
  const double log_r = rest ? ((double)m - big) / T_ + log((double)s) : (double)neg_inf();
  const double log_all = log(sum + (rest ? exp(log_r) : 0.0));
  const bool whole = o.renormalize || mass > 1.0 || !rest;
  const double inv = whole && mass > 0.0 ? 1.0 / mass : 1.0;
  const double p_r = whole ? 0.0 : 1.0 - mass;
  const bool live = big > (double)neg_inf() && (mass > 0.0 || !whole);
  double loss = 0.0;
  if (live)
    for (int k = threadIdx.x; k < K; k += blockDim.x)
      if (idx[k] >= 0 && p[k] > 0.0) {
        const double pk = p[k] * inv;
        loss += pk * (log(pk) - (((double)zu[k] - big) / T_ - log_all));
      }
  loss = block_reduce(loss, dred, Sum());
  if (p_r > 0.0) loss += p_r * (log(p_r) - (log_r - log_all));
  if (!live) loss = 0.0;
  if (bad) loss = (double)quiet_nan();
  if (o.row_loss && threadIdx.x == 0)
    o.row_loss[row.index] = (float)(loss * T_ * T_ * (double)weight);
  if (!row.grad) return;
  const double q_r = rest ? exp(log_r - log_all) : 0.0;
  const double scale = (double)weight * T_;
  const float nan = quiet_nan();
  const float coef = bad ? nan : live ? (float)(scale * (q_r - p_r)) : 0.f;
  const float inv_s = rest ? 1.f / s : 0.f;
  for (int v = threadIdx.x; v < row.size; v += blockDim.x) {
    const float z = row.at(v);
    float d = 0.f;
    if ((bits[v >> 5] >> (v & 31)) & 1u) continue;
    if (z != neg_inf()) d = exp2f((z - ref) * a.c) * inv_s * coef;
    if (bad && z != neg_inf()) d = nan;
    row.grad[v] = to_type<T>(d);
  }
  for (int k = threadIdx.x; k < K; k += blockDim.x)
    if (idx[k] >= 0) {
      const double q = exp(((double)zu[k] - big) / T_ - log_all);
      row.grad[idx[k]] = to_type<T>(bad ? nan : live ? (float)(scale * (q - p[k] * inv)) : 0.f);
    }
}

// Sum of the rows' losses by one block, in 64 bits and a fixed order.
__global__ void __launch_bounds__(1024) sum_rows_kernel(const float* __restrict__ row_loss,
                                                        long long n, float* __restrict__ loss) {
  __shared__ double red[32];
  double s = 0.0;
  for (long long i = threadIdx.x; i < n; i += blockDim.x) s += row_loss[i];
  s = block_reduce(s, red, Sum());
  if (threadIdx.x == 0) *loss = (float)s;
}

}  // namespace lk
}  // namespace chm
