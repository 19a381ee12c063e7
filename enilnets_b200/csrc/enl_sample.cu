// One token per row of logits: temperature, top-k, top-p and min-p, drawn with
// a given uniform number by inverting the running sum of the kept weights.
//
//   w_i = exp((l_i - max) / T),  q_i = floor(w_i 2^40)
//
// Sums are sums of the whole numbers q_i, so they are exact whatever the order
// of addition: a row's token does not depend on how many threads shared it.
// Sorted by (l descending, i ascending), the kept tokens are a leading run,
// i.e. a threshold on the logit and, among the logits equal to it, one on the
// index; both are found by bisection over the order-preserving bits of the
// logits, one pass over the row per bit.
#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace smp {

constexpr int kThreads = 1024;
constexpr float kOne = 1099511627776.0f;  // 2^40

using u64 = unsigned long long;

// Order-preserving bits of a float: a < b as floats iff key(a) < key(b).
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

template <bool kF32>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  float f;
  if constexpr (kF32)
    f = reinterpret_cast<const float*>(row)[i];
  else
    f = __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
  if (f != f) f = -INFINITY;
  return f == 0.0f ? 0.0f : f;  // one zero: -0 and +0 are equal logits
}

// Weight of a logit; expf and the single multiply are the operator's
// definition of w (no fast approximation), so the whole numbers are reproducible.
__device__ __forceinline__ float weight_of(float x, float top, float inv_t) {
  return x == top ? 1.0f : expf((x - top) * inv_t);
}
__device__ __forceinline__ u64 whole_of(float w) { return (u64)(w * kOne); }

// floor(total * part / 2^24), part < 2^24 + 1.
__device__ __forceinline__ u64 share_of(u64 total, uint32_t part) {
  return (total >> 24) * part + (((total & 0xffffffu) * part) >> 24);
}

__device__ __forceinline__ u64 block_sum(u64 x) {
  __shared__ u64 sm[kThreads / 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm[threadIdx.x / 32] = x;
  __syncthreads();
  x = sm[threadIdx.x % 32];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
  const int b = blockIdx.x;
  const int V = p.V;
  const void* row = reinterpret_cast<const uint8_t*>(p.logits) + b * p.stride * (kF32 ? 4 : 2);
  const float T = p.temperature ? p.temperature[b] : p.temperature_all;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float min_p = fminf(p.min_p ? p.min_p[b] : p.min_p_all, 1.0f);  // the best token stays
  const float inv_t = T > 0.0f ? 1.0f / T : 1.0f;

  // The largest logit: key 0 is below every key.
  uint32_t best = 0;
  for (int i = threadIdx.x; i < V; i += kThreads) best = max(best, key_of(logit_at<kF32>(row, i)));
  __shared__ uint32_t sm_best;
  if (threadIdx.x == 0) sm_best = 0;
  __syncthreads();
  best = __reduce_max_sync(0xffffffffu, best);
  if (threadIdx.x % 32 == 0) atomicMax(&sm_best, best);
  __syncthreads();
  const float top = of_key(sm_best);
  if (top == -INFINITY) {
    if (threadIdx.x == 0) p.tokens[b] = -1;
    return;
  }

  // sum over i of f(key, i, q) for the tokens at or above a threshold.
  auto mass = [&](uint32_t key, int last, bool count) {
    // tokens with a larger key, or this key and an index <= last
    u64 s = 0;
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const float x = logit_at<kF32>(row, i);
      const uint32_t kk = key_of(x);
      if (kk > key || (kk == key && i <= last))
        s += count ? 1ull : whole_of(weight_of(x, top, inv_t));
    }
    return block_sum(s);
  };
  // The last token of the smallest leading run whose mass reaches `need`
  // (all tokens when none does): its key, then its index.
  auto run_end = [&](u64 need, bool count, uint32_t& key, int& last) {
    uint32_t lo = 0, hi = key_of(top);  // mass(lo) reaches, or nothing does
    while (lo < hi) {
      const uint32_t mid = hi - (hi - lo) / 2;
      if (mass(mid, V, count) >= need)
        lo = mid;
      else
        hi = mid - 1;
    }
    int a = 0, z = V - 1;
    while (a < z) {
      const int mid = (a + z) / 2;
      if (mass(lo, mid, count) >= need)
        z = mid;
      else
        a = mid + 1;
    }
    key = lo;
    last = a;
  };

  uint32_t key = 0;
  int last = V;
  if (!(T > 0.0f)) {
    run_end(1, true, key, last);
    if (threadIdx.x == 0) p.tokens[b] = last;
    return;
  }
  if (k > 0 && k < V) run_end((u64)k, true, key, last);
  if (top_p < 1.0f) {
    const u64 total = mass(key, last, false);
    const uint32_t part = (uint32_t)(fmaxf(top_p, 0.0f) * 16777216.0f);
    const u64 bound = share_of(total, part);
    // Kept: tokens whose sum before them is below the bound, and the first.
    run_end(bound > 0 ? bound : 1, false, key, last);
  }
  auto kept = [&](int i, u64& q) {
    const float x = logit_at<kF32>(row, i);
    const uint32_t kk = key_of(x);
    const float w = weight_of(x, top, inv_t);
    q = whole_of(w);
    return (kk > key || (kk == key && i <= last)) && w >= min_p;
  };
  auto kept_sum = [&](int end) {
    u64 s = 0, q;
    for (int i = threadIdx.x; i <= end; i += kThreads)
      if (kept(i, q)) s += q;
    return block_sum(s);
  };
  const u64 total = kept_sum(V - 1);
  const float uf = fminf(fmaxf(p.u[b], 0.0f), 0.99999994f);
  const u64 target = share_of(total, (uint32_t)(uf * 16777216.0f));
  int a = 0, z = V - 1;
  while (a < z) {
    const int mid = (a + z) / 2;
    if (kept_sum(mid) > target)
      z = mid;
    else
      a = mid + 1;
  }
  if (threadIdx.x == 0) p.tokens[b] = a;
}

}  // namespace smp

cudaError_t launch_sample(const SampleParams& p, cudaStream_t stream) {
  if (p.fp32)
    smp::sample_kernel<true><<<p.B, smp::kThreads, 0, stream>>>(p);
  else
    smp::sample_kernel<false><<<p.B, smp::kThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace enl
