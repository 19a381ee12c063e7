// Per-head RMS norm of queries and keys with the rotate-half position
// rotation, in one pass; its serving form, which also writes the new keys and
// values into a paged cache; and its backward.
//
//   z = w x / sqrt(mean(x^2) + eps)
//   y1 = z1 c - z2 s,  y2 = z2 c + z1 s          (halves of the head)
// backward, dz the gradient turned by the negated angle, xh = x rstd, g = w dz:
//   dx = rstd (g - xh mean(g xh)),  dw = sum dz xh
//
// All three move each element once and compute about ten operations on it, so
// HBM bounds them. A group of D / 8 lanes (rounded up to a power of two) owns
// one head of one token: lane j holds elements 4j .. 4j+3 of the first half and
// their partners of the second half, so the rotation needs no exchange and the
// norm one reduction over the group. A group takes up to kHeads heads of a
// token at a time: their loads are all in flight together, and the token's
// angles are read once for them.
#include <algorithm>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace qkr {

constexpr int kThreads = 256;
constexpr int kHeads = 4;

struct Quad {
  float v[4];
};

template <bool kF32>
__device__ __forceinline__ Quad load4(const void* base, long long elem) {
  Quad q;
  if constexpr (kF32) {
    const float4 f = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + elem);
    q.v[0] = f.x, q.v[1] = f.y, q.v[2] = f.z, q.v[3] = f.w;
  } else {
    const uint2 w =
        *reinterpret_cast<const uint2*>(reinterpret_cast<const __nv_bfloat16*>(base) + elem);
    q.v[0] = bf16lo_to_f32(w.x), q.v[1] = bf16hi_to_f32(w.x);
    q.v[2] = bf16lo_to_f32(w.y), q.v[3] = bf16hi_to_f32(w.y);
  }
  return q;
}

template <bool kF32>
__device__ __forceinline__ void store4(void* base, long long elem, const Quad& q) {
  if constexpr (kF32) {
    *reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + elem) =
        make_float4(q.v[0], q.v[1], q.v[2], q.v[3]);
  } else {
    __nv_bfloat162 lo = __floats2bfloat162_rn(q.v[0], q.v[1]);
    __nv_bfloat162 hi = __floats2bfloat162_rn(q.v[2], q.v[3]);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(base) + elem) =
        make_uint2(*reinterpret_cast<uint32_t*>(&lo), *reinterpret_cast<uint32_t*>(&hi));
  }
}

__device__ __forceinline__ Quad quad(float x) {
  Quad q;
  q.v[0] = q.v[1] = q.v[2] = q.v[3] = x;
  return q;
}

template <int LG>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int off = LG / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// One unit: heads [h0, h0 + n) of operand `op` at one token.
struct Unit {
  int op, b, s, h0, n;
};

__device__ __forceinline__ Unit unit_of(long long u, int S, int H, int Hkv, int nq, int nk, int nch,
                                        int hc) {
  Unit t;
  const long long token = u / nch;
  int c = (int)(u - token * nch);
  t.b = (int)(token / S);
  t.s = (int)(token - (long long)t.b * S);
  t.op = c < nq ? 0 : c < nq + nk ? 1 : 2;
  c -= t.op == 0 ? 0 : t.op == 1 ? nq : nq + nk;
  const int heads = t.op == 0 ? H : Hkv;
  t.h0 = c * hc;
  t.n = min(hc, heads - t.h0);
  return t;
}

template <bool kIn32, bool kOut32, int LG>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const QkRopeParams p, int hc,
                                                                int nq, int nk, int nch,
                                                                long long n_units) {
  const long long u = ((long long)blockIdx.x * kThreads + threadIdx.x) / LG;
  const int j = threadIdx.x % LG;
  const int half = p.D / 2;
  const bool real_unit = u < n_units;
  const Unit t = unit_of(real_unit ? u : 0, p.S, p.H, p.Hkv, nq, nk, nch, hc);
  const bool live = real_unit && j * 4 < half;

  // Where the token goes, and whether it is one.
  const long long at = (p.start ? p.start[t.b] : 0) + (long long)t.s;  // cache position
  bool keep = !p.n_new || t.s < p.n_new[t.b];
  const long long row = p.pos0 + at;
  if (keep && p.cos_t && (row < 0 || row >= p.rows)) {
    if (live && j == 0) report_error(kDevBadIndex, t.s);
    keep = false;
  }
  long long slot = 0;  // element offset of the token's row in the pools, kv head 0
  if (p.pages[0] && keep) {
    const long long col = at / p.page_size;
    int page = -1;
    if (at >= 0 && col < p.max_pages) page = p.table[t.b * p.t_sb + col];
    if (page < 0 || page >= p.n_pages) {
      if (live && j == 0) report_error(kDevBadIndex, t.s);
      keep = false;
    } else {
      slot = page * p.p_sp + (at - col * p.page_size) * p.p_ss;
    }
  }

  const int op = t.op;
  const long long xb = t.b * p.x_sb[op] + t.s * p.x_ss[op];
  Quad a[kHeads], b[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    a[i] = b[i] = quad(0.0f);
    if (live && keep && i < t.n) {
      const long long e = xb + (t.h0 + i) * p.x_sh[op] + j * 4;
      a[i] = load4<kIn32>(p.x[op], e);
      b[i] = load4<kIn32>(p.x[op], e + half);
    }
  }
  float r[kHeads];
  if (p.w[0]) {
    // Every group of the warp takes part in the reduction, values (op 2) too.
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fmaf(a[i].v[e], a[i].v[e], fmaf(b[i].v[e], b[i].v[e], ss));
      r[i] = group_sum<LG>(ss);
    }
  }
  if (op < 2) {
    Quad c = quad(1.0f), s = quad(0.0f), w1 = quad(1.0f), w2 = quad(1.0f);
    if (p.cos_t && live && keep) {
      c = load4<true>(p.cos_t, row * half + j * 4);
      s = load4<true>(p.sin_t, row * half + j * 4);
    }
    const float* w = p.w[op];
    if (w && live) {
      w1 = load4<true>(w, j * 4);
      w2 = load4<true>(w, half + j * 4);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const float rstd = w ? rsqrtf(r[i] / (float)p.D + p.eps) : 1.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float z1 = a[i].v[e] * rstd * w1.v[e];
        const float z2 = b[i].v[e] * rstd * w2.v[e];
        a[i].v[e] = z1 * c.v[e] - z2 * s.v[e];
        b[i].v[e] = z2 * c.v[e] + z1 * s.v[e];
      }
    }
  }
  if (!live) return;
  if (op == 0 || !p.pages[0]) {
    if (!keep) {
#pragma unroll
      for (int i = 0; i < kHeads; ++i) a[i] = b[i] = quad(0.0f);
    }
    const long long yb = t.b * p.y_sb[op] + t.s * p.y_ss[op];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= t.n) break;
      const long long e = yb + (t.h0 + i) * p.y_sh[op] + j * 4;
      store4<kOut32>(p.y[op], e, a[i]);
      store4<kOut32>(p.y[op], e + half, b[i]);
    }
  } else if (keep) {
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      if (i >= t.n) break;
      const long long e = slot + (t.h0 + i) * p.p_sh + j * 4;
      store4<kOut32>(p.pages[op - 1], e, a[i]);
      store4<kOut32>(p.pages[op - 1], e + half, b[i]);
    }
  }
}

// ---------------------------------------------------------------- backward
template <bool kIn32, bool kGrad32, bool kOut32, int LG>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_bwd_kernel(const QkRopeBwdParams p,
                                                                    int nq, int nk,
                                                                    long long n_units) {
  constexpr int kGroups = kThreads / LG;
  const int j = threadIdx.x % LG;
  const int half = p.D / 2;
  const bool lane_live = j * 4 < half;
  const bool norm = p.w[0] != nullptr;
  float dw[2][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[0][i] = dw[1][i] = 0.0f;

  const long long first = (long long)blockIdx.x * kGroups + threadIdx.x / LG;
  // The bound is the same for every lane of a warp, which the reductions need.
  const long long warp_first = (long long)blockIdx.x * kGroups + threadIdx.x / 32 * (32 / LG);
  const long long step = (long long)gridDim.x * kGroups;
  for (long long uw = warp_first, u = first; uw < n_units; uw += step, u += step) {
    const bool live = lane_live && u < n_units;
    const Unit t = unit_of(u < n_units ? u : 0, p.S, p.H, p.Hkv, nq, nk, nq + nk, kHeads);
    const int op = t.op;
    const long long row = p.pos0 + (p.start ? p.start[t.b] : 0) + (long long)t.s;
    const bool keep = !p.cos_t || (row >= 0 && row < p.rows);
    if (!keep && live && j == 0) report_error(kDevBadIndex, t.s);
    const long long gb = t.b * p.dy_sb[op] + t.s * p.dy_ss[op];
    const long long xb = t.b * p.x_sb[op] + t.s * p.x_ss[op];
    Quad ga[kHeads], gbq[kHeads], a[kHeads], b[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      ga[i] = gbq[i] = a[i] = b[i] = quad(0.0f);
      if (live && keep && i < t.n) {
        const long long eg = gb + (t.h0 + i) * p.dy_sh[op] + j * 4;
        ga[i] = load4<kGrad32>(p.dy[op], eg);
        gbq[i] = load4<kGrad32>(p.dy[op], eg + half);
        if (norm) {
          const long long ex = xb + (t.h0 + i) * p.x_sh[op] + j * 4;
          a[i] = load4<kIn32>(p.x[op], ex);
          b[i] = load4<kIn32>(p.x[op], ex + half);
        }
      }
    }
    Quad c = quad(1.0f), s = quad(0.0f), w1 = quad(1.0f), w2 = quad(1.0f);
    if (p.cos_t && live && keep) {
      c = load4<true>(p.cos_t, row * half + j * 4);
      s = load4<true>(p.sin_t, row * half + j * 4);
    }
    if (norm && live) {
      w1 = load4<true>(p.w[op], j * 4);
      w2 = load4<true>(p.w[op], half + j * 4);
    }
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      float ss = 0.0f, gx = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d1 = ga[i].v[e] * c.v[e] + gbq[i].v[e] * s.v[e];
        const float d2 = gbq[i].v[e] * c.v[e] - ga[i].v[e] * s.v[e];
        ga[i].v[e] = d1;
        gbq[i].v[e] = d2;
        ss = fmaf(a[i].v[e], a[i].v[e], fmaf(b[i].v[e], b[i].v[e], ss));
        gx = fmaf(d1 * w1.v[e], a[i].v[e], fmaf(d2 * w2.v[e], b[i].v[e], gx));
      }
      if (!norm) continue;
      ss = group_sum<LG>(ss);
      gx = group_sum<LG>(gx);
      const float r = rsqrtf(ss / (float)p.D + p.eps);
      const float m = gx * r * r / (float)p.D;  // mean(g xh) / |x| scale: xh m' = x m
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x1 = a[i].v[e], x2 = b[i].v[e];
        const float t1 = ga[i].v[e] * x1 * r, t2 = gbq[i].v[e] * x2 * r;
        if (op == 0) {
          dw[0][e] += t1, dw[0][4 + e] += t2;
        } else {
          dw[1][e] += t1, dw[1][4 + e] += t2;
        }
        ga[i].v[e] = r * (ga[i].v[e] * w1.v[e] - x1 * m);
        gbq[i].v[e] = r * (gbq[i].v[e] * w2.v[e] - x2 * m);
      }
    }
    if (live) {
      const long long yb = t.b * p.dx_sb[op] + t.s * p.dx_ss[op];
#pragma unroll
      for (int i = 0; i < kHeads; ++i) {
        if (i >= t.n) break;
        const long long e = yb + (t.h0 + i) * p.dx_sh[op] + j * 4;
        store4<kOut32>(p.dx[op], e, ga[i]);
        store4<kOut32>(p.dx[op], e + half, gbq[i]);
      }
    }
  }
  if (!norm) return;
  // The block's sums, lane groups added in order.
  __shared__ float sm[kGroups][LG * 8];
#pragma unroll
  for (int op = 0; op < 2; ++op) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      sm[threadIdx.x / LG][j * 4 + e] = dw[op][e];
      sm[threadIdx.x / LG][LG * 4 + j * 4 + e] = dw[op][4 + e];
    }
    __syncthreads();
    for (int d = threadIdx.x; d < p.D; d += kThreads) {
      const int col = d < half ? d : LG * 4 + (d - half);
      float sum = 0.0f;
      for (int g = 0; g < kGroups; ++g) sum += sm[g][col];
      p.partial[((long long)blockIdx.x * 2 + op) * p.D + d] = sum;
    }
  }
}

// dw[op][d] = sum over blocks of partial[block][op][d]: 32 columns a block,
// eight slices of the blocks each, added in a fixed order.
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* __restrict__ partial,
                                                         int n_blocks, int D, float* dwq,
                                                         float* dwk) {
  __shared__ float sm[8][32];
  const int op = blockIdx.y, col = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int d = blockIdx.x * 32 + col;
  float sum = 0.0f;
  if (d < D)
    for (int i = slice; i < n_blocks; i += 8) sum += partial[((long long)i * 2 + op) * D + d];
  sm[slice][col] = sum;
  __syncthreads();
  if (slice == 0 && d < D) {
    for (int k = 1; k < 8; ++k) sum += sm[k][col];
    (op == 0 ? dwq : dwk)[d] = sum;
  }
}

int lanes_for(int D) { return D > 64 ? 16 : D > 32 ? 8 : 4; }

template <bool kIn32, bool kOut32>
cudaError_t launch_fwd(const QkRopeParams& p, cudaStream_t stream) {
  const int hc = kHeads;
  const int nq = (p.H + hc - 1) / hc, nk = (p.Hkv + hc - 1) / hc;
  const int nch = nq + nk + (p.pages[0] ? nk : 0);
  const long long n_units = (long long)p.B * p.S * nch;
  if (n_units == 0) return cudaSuccess;
  const int LG = lanes_for(p.D);
  const long long blocks = (n_units * LG + kThreads - 1) / kThreads;
  if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)blocks);
  if (LG == 16)
    qk_norm_rope_kernel<kIn32, kOut32, 16><<<grid, kThreads, 0, stream>>>(p, hc, nq, nk, nch, n_units);
  else if (LG == 8)
    qk_norm_rope_kernel<kIn32, kOut32, 8><<<grid, kThreads, 0, stream>>>(p, hc, nq, nk, nch, n_units);
  else
    qk_norm_rope_kernel<kIn32, kOut32, 4><<<grid, kThreads, 0, stream>>>(p, hc, nq, nk, nch, n_units);
  return cudaGetLastError();
}

template <bool kIn32, bool kGrad32, bool kOut32>
cudaError_t launch_bwd(const QkRopeBwdParams& p, cudaStream_t stream) {
  const int nq = (p.H + kHeads - 1) / kHeads, nk = (p.Hkv + kHeads - 1) / kHeads;
  const long long n_units = (long long)p.B * p.S * (nq + nk);
  const int LG = lanes_for(p.D);
  const int blocks = p.n_blocks;
  if (LG == 16)
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 16><<<blocks, kThreads, 0, stream>>>(p, nq, nk, n_units);
  else if (LG == 8)
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 8><<<blocks, kThreads, 0, stream>>>(p, nq, nk, n_units);
  else
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 4><<<blocks, kThreads, 0, stream>>>(p, nq, nk, n_units);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !p.w[0]) return e;
  qk_norm_dw_kernel<<<dim3((p.D + 31) / 32, 2), 256, 0, stream>>>(p.partial, blocks, p.D, p.dw[0],
                                                                 p.dw[1]);
  return cudaGetLastError();
}

}  // namespace qkr

cudaError_t launch_qk_norm_rope(const QkRopeParams& p, cudaStream_t stream) {
  if (p.in_fp32)
    return p.out_fp32 ? qkr::launch_fwd<true, true>(p, stream)
                      : qkr::launch_fwd<true, false>(p, stream);
  return p.out_fp32 ? qkr::launch_fwd<false, true>(p, stream)
                    : qkr::launch_fwd<false, false>(p, stream);
}

int qk_rope_bwd_blocks(int B, int S, int H, int Hkv, int D, int n_sms) {
  const long long units = (long long)B * S * ((H + qkr::kHeads - 1) / qkr::kHeads +
                                              (Hkv + qkr::kHeads - 1) / qkr::kHeads);
  const long long per_block = qkr::kThreads / qkr::lanes_for(D);
  const long long blocks = (units + per_block - 1) / per_block;
  return (int)std::max(1ll, std::min(blocks, (long long)n_sms * 4));
}

cudaError_t launch_qk_norm_rope_backward(const QkRopeBwdParams& p, cudaStream_t stream) {
  if (p.in_fp32) {
    if (p.grad_fp32)
      return p.out_fp32 ? qkr::launch_bwd<true, true, true>(p, stream)
                        : qkr::launch_bwd<true, true, false>(p, stream);
    return p.out_fp32 ? qkr::launch_bwd<true, false, true>(p, stream)
                      : qkr::launch_bwd<true, false, false>(p, stream);
  }
  if (p.grad_fp32)
    return p.out_fp32 ? qkr::launch_bwd<false, true, true>(p, stream)
                      : qkr::launch_bwd<false, true, false>(p, stream);
  return p.out_fp32 ? qkr::launch_bwd<false, false, true>(p, stream)
                    : qkr::launch_bwd<false, false, false>(p, stream);
}

}  // namespace enl
