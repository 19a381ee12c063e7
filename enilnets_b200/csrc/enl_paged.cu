// Attention of one new token per sequence over a paged key-value cache.
//
//   o_h = sum_j softmax_j(scale q_h . k_j - slope_h (L - 1 - j)) v_j
//
// over the positions j the query at L - 1 sees: all of them, or with a window
// the first `sinks` and those at most `window` back. Position j is slot
// j % page_size of page table[b][j / page_size].
//
// Each split of a sequence's visible positions is one block per query head;
// eight (head dim up to 64) or sixteen lanes share a key, the softmax runs
// online in fp32, and the splits are joined by log-sum-exp.
#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace paged {

constexpr int kThreads = 128;
constexpr int kSplitKeys = 512;  // visible positions per split, before the cap
constexpr int kMaxSplits = 64;

// The visible positions of a sequence of length L as one index range:
// index i < n_sink is position i, the others lie `gap` further.
struct Visible {
  int n, n_sink, gap;
};

__device__ __forceinline__ Visible visible_of(int L, int window, int sinks) {
  Visible v;
  const int first = window < 0 ? 0 : max(0, L - 1 - window);
  v.n_sink = min(sinks, first);
  v.gap = first - v.n_sink;
  v.n = L - v.gap;
  return v;
}

template <bool kF32>
__device__ __forceinline__ void load8(const void* base, long long e, float (&f)[8]) {
  if constexpr (kF32) {
    const float4* p = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + e);
    const float4 a = p[0], b = p[1];
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  } else {
    const uint4 w =
        *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + e);
    f[0] = bf16lo_to_f32(w.x), f[1] = bf16hi_to_f32(w.x);
    f[2] = bf16lo_to_f32(w.y), f[3] = bf16hi_to_f32(w.y);
    f[4] = bf16lo_to_f32(w.z), f[5] = bf16hi_to_f32(w.z);
    f[6] = bf16lo_to_f32(w.w), f[7] = bf16hi_to_f32(w.w);
  }
}

// One (split, query head, sequence): partial output (normalised) and LSE.
template <bool kF32>
__global__ void __launch_bounds__(kThreads) paged_split_kernel(const PagedDecodeParams p,
                                                               int n_splits, float* part_o,
                                                               float* part_lse) {
  constexpr int LPK = 16, kGroups = kThreads / LPK;
  const int split = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int hk = h / (p.H / p.Hkv);
  const int sub = threadIdx.x % LPK, group = threadIdx.x / LPK;
  const bool live = sub * 8 < p.D;
  int L = p.lens[b];
  if ((long long)L > (long long)p.max_pages * p.page_size) {
    if (threadIdx.x == 0) report_error(kDevBadIndex, b);
    L = p.max_pages * p.page_size;
  }
  const Visible vis = visible_of(max(L, 0), p.window, p.sinks);
  const int per = (vis.n + n_splits - 1) / n_splits;
  const int i0 = min(split * per, vis.n), i1 = min(i0 + per, vis.n);

  float q[8] = {}, acc[8] = {};
  if (live) load8<kF32>(p.q, b * p.q_sb + h * p.q_sh + sub * 8, q);
  const float slope = p.alibi ? p.alibi[h] : 0.0f;
  float m = -INFINITY, l = 0.0f;
  // Block-uniform bound: the reductions need whole warps.
  for (int i = i0; i < i1; i += kGroups) {
    const int idx = i + group;
    float s = -INFINITY, v[8] = {};
    float d = 0.0f;
    bool ok = idx < i1;
    const int j = idx < vis.n_sink ? idx : idx + vis.gap;
    if (ok) {
      const int page = p.table[b * p.t_sb + j / p.page_size];
      if (page < 0 || page >= p.n_pages) {
        if (sub == 0) report_error(kDevBadIndex, b);
        ok = false;
      } else if (live) {
        const long long e = page * p.p_sp + hk * p.p_sh + (j % p.page_size) * p.p_ss + sub * 8;
        float k[8];
        load8<kF32>(p.k, e, k);
        load8<kF32>(p.v, e, v);
#pragma unroll
        for (int x = 0; x < 8; ++x) d = fmaf(q[x], k[x], d);
      }
    }
#pragma unroll
    for (int off = LPK / 2; off > 0; off /= 2) d += __shfl_xor_sync(0xffffffffu, d, off);
    if (ok) s = d * p.scale - slope * (float)(L - 1 - j);
    const float mx = fmaxf(m, s);
    if (mx != -INFINITY) {
      const float corr = expf(m - mx), w = expf(s - mx);
      l = l * corr + w;
#pragma unroll
      for (int x = 0; x < 8; ++x) acc[x] = fmaf(w, v[x], acc[x] * corr);
      m = mx;
    }
  }
  __shared__ float sm_m[kGroups], sm_l[kGroups], sm_acc[kGroups][128];
  if (sub == 0) sm_m[group] = m, sm_l[group] = l;
#pragma unroll
  for (int x = 0; x < 8; ++x) sm_acc[group][sub * 8 + x] = acc[x];
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= p.D) return;
  float M = -INFINITY, Lsum = 0.0f, O = 0.0f;
  for (int g = 0; g < kGroups; ++g) M = fmaxf(M, sm_m[g]);
  if (M != -INFINITY)
    for (int g = 0; g < kGroups; ++g) {
      const float w = expf(sm_m[g] - M);
      Lsum = fmaf(w, sm_l[g], Lsum);
      O = fmaf(w, sm_acc[g][d], O);
    }
  const long long row = ((long long)split * p.B + b) * p.H + h;
  part_o[row * p.D + d] = Lsum > 0.0f ? O / Lsum : 0.0f;
  if (d == 0) part_lse[row] = Lsum > 0.0f ? M + logf(Lsum) : -INFINITY;
}

__global__ void __launch_bounds__(kThreads) paged_join_kernel(const PagedDecodeParams p,
                                                              int n_splits, const float* part_o,
                                                              const float* part_lse) {
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const long long row0 = (long long)b * p.H + h, step = (long long)p.B * p.H;
  float M = -INFINITY, W = 0.0f, O = 0.0f;
  for (int s = 0; s < n_splits; ++s) M = fmaxf(M, part_lse[row0 + s * step]);
  if (M != -INFINITY)
    for (int s = 0; s < n_splits; ++s) {
      const float w = expf(part_lse[row0 + s * step] - M);
      W += w;
      if (d < p.D) O = fmaf(w, part_o[(row0 + s * step) * p.D + d], O);
    }
  if (d < p.D) {
    const float val = W > 0.0f ? O / W : 0.0f;
    const long long e = b * p.o_sb + h * p.o_sh + d;
    if (p.out_fp32)
      reinterpret_cast<float*>(p.o)[e] = val;
    else
      reinterpret_cast<__nv_bfloat16*>(p.o)[e] = __float2bfloat16_rn(val);
  }
  if (d == 0 && p.lse) p.lse[row0] = W > 0.0f ? M + logf(W) : -INFINITY;
}

}  // namespace paged

size_t paged_decode_workspace(int B, int H, int Hkv, int D, int n_sms) {
  return (size_t)paged::kMaxSplits * B * H * (D + 1) * sizeof(float);
}

cudaError_t launch_paged_decode(const PagedDecodeParams& p, cudaStream_t stream) {
  const long long most = (long long)p.max_pages * p.page_size;
  const int n_splits =
      (int)std::max(1ll, std::min((long long)paged::kMaxSplits,
                                  (most + paged::kSplitKeys - 1) / paged::kSplitKeys));
  float* part_o = reinterpret_cast<float*>(p.workspace);
  float* part_lse = part_o + (size_t)n_splits * p.B * p.H * p.D;
  const dim3 grid(n_splits, p.H, p.B);
  if (p.in_fp32)
    paged::paged_split_kernel<true><<<grid, paged::kThreads, 0, stream>>>(p, n_splits, part_o,
                                                                          part_lse);
  else
    paged::paged_split_kernel<false><<<grid, paged::kThreads, 0, stream>>>(p, n_splits, part_o,
                                                                           part_lse);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  paged::paged_join_kernel<<<dim3(p.H, p.B), paged::kThreads, 0, stream>>>(p, n_splits, part_o,
                                                                           part_lse);
  return cudaGetLastError();
}

}  // namespace enl
