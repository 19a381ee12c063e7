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
// HBM bounds them. A group of lanes owns one head of one token: a lane holds E
// consecutive elements of the first half and their E partners of the second,
// so the rotation needs no exchange and the norm one reduction over the group.
// A group takes several heads of a token at a time: their loads are in flight
// together, kept packed until their turn, and the token's angles are read once.
// How many, and how many blocks share an SM, is a choice between loads in
// flight and registers; measured (bf16, 8 x 4096 tokens, 16 + 16 heads of 128,
// floor 82 us): E = 8 with 8 heads and 2 blocks 86 us, 4 heads and 3 blocks
// 91 us, 2 heads and 4 blocks 102 us. The backward (4 x 4095, 16 + 4 heads,
// fp32 gradients, floor 51 us): E = 4 with 4 heads and 2 blocks 65 us, 2 heads
// and 3 blocks 66 us, E = 8 with 2 heads 68 us, 1 head and 3 blocks 99 us.
#include <algorithm>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace qkr {

constexpr int kThreads = 256;
constexpr int kBwdHeads = 4;  // heads of a token that a group takes, backward

// E elements as loaded: words of two bf16 or one fp32.
template <bool kF32, int E>
struct Raw {
  static constexpr int kWords = kF32 ? E : E / 2;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const void* base, long long elem) {
    const uint32_t* p = reinterpret_cast<const uint32_t*>(
        reinterpret_cast<const uint8_t*>(base) + elem * (kF32 ? 4 : 2));
    if constexpr (kWords == 2) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 v = *reinterpret_cast<const uint4*>(p + i);
        w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
      }
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ float at(int e) const {
    if constexpr (kF32) return __uint_as_float(w[e]);
    return e % 2 ? bf16hi_to_f32(w[e / 2]) : bf16lo_to_f32(w[e / 2]);
  }
  // Elements 2i and 2i + 1 as one operand of the packed fp32 instructions.
  __device__ __forceinline__ uint64_t pair(int i) const {
    return f2_pack(at(2 * i), at(2 * i + 1));
  }
};

__device__ __forceinline__ uint64_t both(float x) { return f2_pack(x, x); }
__device__ __forceinline__ float pair_sum(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

template <bool kF32, int E>
__device__ __forceinline__ void store(void* base, long long elem, const uint64_t (&pairs)[E / 2]) {
  float x[E];
#pragma unroll
  for (int i = 0; i < E / 2; ++i) f2_unpack(pairs[i], x[2 * i], x[2 * i + 1]);
  if constexpr (kF32) {
    float4* p = reinterpret_cast<float4*>(reinterpret_cast<float*>(base) + elem);
#pragma unroll
    for (int i = 0; i < E; i += 4) p[i / 4] = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
  } else {
    uint32_t w[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<uint32_t*>(&v);
    }
    uint8_t* p = reinterpret_cast<uint8_t*>(base) + elem * 2;
    if constexpr (E == 4)
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else
      *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

template <int LG>
__device__ __forceinline__ float group_sum(float x) {
#pragma unroll
  for (int off = LG / 2; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

// One block: kThreads / LG tokens of one head chunk. The chunks of q, then k,
// then v run fastest over the grid, so that blocks that run together read whole
// rows of a fused projection.
template <bool kIn32, bool kOut32, int E, int LG, int kHeads>
__global__ void __launch_bounds__(kThreads, kHeads > 4 ? 2 : 3) qk_norm_rope_kernel(const QkRopeParams p, int nq,
                                                                int nk, int nch) {
  const int chunk = blockIdx.x % nch;
  const int token = blockIdx.x / nch * (kThreads / LG) + threadIdx.x / LG;
  const int j = threadIdx.x % LG;
  const int half = p.D / 2;
  const int op = chunk < nq ? 0 : chunk < nq + nk ? 1 : 2;
  const int h0 = (chunk - (op == 0 ? 0 : op == 1 ? nq : nq + nk)) * kHeads;
  const int n = min(kHeads, (op == 0 ? p.H : p.Hkv) - h0);
  const bool live = token < p.B * p.S && j * E < half;
  const int b = live ? token / p.S : 0, s = live ? token % p.S : 0;

  const long long xe = b * p.x_sb[op] + s * p.x_ss[op] + h0 * p.x_sh[op] + j * E;
  Raw<kIn32, E> ra[kHeads], rb[kHeads];
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    if (live && i < n) {
      ra[i].load(p.x[op], xe + i * p.x_sh[op]);
      rb[i].load(p.x[op], xe + i * p.x_sh[op] + half);
    } else {
      ra[i].zero();
      rb[i].zero();
    }
  }

  // Where the token goes, and whether it is one.
  const long long at = (p.start ? p.start[b] : 0) + (long long)s;  // cache position
  bool keep = !p.n_new || s < p.n_new[b];
  const long long row = p.pos0 + at;
  if (keep && p.cos_t && (row < 0 || row >= p.rows)) {
    if (live && j == 0) report_error(kDevBadIndex, s);
    keep = false;
  }
  long long slot = 0;  // element offset of the token's row in the pools, kv head 0
  if (p.pages[0] && keep) {
    int page = -1, off = 0;
    if (at >= 0 && at < (long long)p.max_pages * p.page_size) {
      const int col = (int)at / p.page_size;
      off = (int)at - col * p.page_size;
      page = p.table[b * p.t_sb + col];
    }
    if (page < 0 || page >= p.n_pages) {
      if (live && j == 0) report_error(kDevBadIndex, s);
      keep = false;
    } else {
      slot = page * p.p_sp + off * p.p_ss;
    }
  }
  const bool to_pages = op > 0 && p.pages[0];
  void* y = to_pages ? p.pages[op - 1] : p.y[op];
  const long long ys = to_pages ? p.p_sh : p.y_sh[op];
  const long long ye = (to_pages ? slot : b * p.y_sb[op] + s * p.y_ss[op]) + h0 * ys + j * E;

  // The token's turn with the norm's weights in it: y1 = r (x1 c1 - x2 s2),
  // y2 = r (x2 c2 + x1 s1) with c1 = w1 c, s2 = w2 s and so on.
  constexpr int P = E / 2;
  uint64_t c1[P], c2[P], s1[P], s2[P];
#pragma unroll
  for (int i = 0; i < P; ++i) c1[i] = c2[i] = both(1.0f), s1[i] = s2[i] = both(0.0f);
  if (op < 2 && live && keep) {
    if (p.cos_t) {
      Raw<true, E> t;
      t.load(p.cos_t, row * half + j * E);
#pragma unroll
      for (int i = 0; i < P; ++i) c1[i] = c2[i] = t.pair(i);
      t.load(p.sin_t, row * half + j * E);
#pragma unroll
      for (int i = 0; i < P; ++i) s1[i] = t.pair(i), s2[i] = f2_mul(t.pair(i), both(-1.0f));
    }
    if (p.w[op]) {
      Raw<true, E> t;
      t.load(p.w[op], j * E);
#pragma unroll
      for (int i = 0; i < P; ++i) c1[i] = f2_mul(c1[i], t.pair(i)), s1[i] = f2_mul(s1[i], t.pair(i));
      t.load(p.w[op], half + j * E);
#pragma unroll
      for (int i = 0; i < P; ++i) c2[i] = f2_mul(c2[i], t.pair(i)), s2[i] = f2_mul(s2[i], t.pair(i));
    }
  }
  const float inv_d = 1.0f / (float)p.D;
#pragma unroll
  for (int i = 0; i < kHeads; ++i) {
    uint64_t x1[P], x2[P];
#pragma unroll
    for (int e = 0; e < P; ++e) x1[e] = ra[i].pair(e), x2[e] = rb[i].pair(e);
    if (op < 2) {  // the same for the whole block, which the reduction needs
      if (p.w[0]) {
        uint64_t ss = both(0.0f);
#pragma unroll
        for (int e = 0; e < P; ++e) ss = f2_fma(x1[e], x1[e], f2_fma(x2[e], x2[e], ss));
        const uint64_t r = both(rsqrtf(fmaf(group_sum<LG>(pair_sum(ss)), inv_d, p.eps)));
#pragma unroll
        for (int e = 0; e < P; ++e) x1[e] = f2_mul(x1[e], r), x2[e] = f2_mul(x2[e], r);
      }
      if (p.w[0] || p.cos_t) {
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const uint64_t y1 = f2_fma(x1[e], c1[e], f2_mul(x2[e], s2[e]));
          x2[e] = f2_fma(x2[e], c2[e], f2_mul(x1[e], s1[e]));
          x1[e] = y1;
        }
      }
    }
    if (live && i < n && (keep || !to_pages)) {
      if (!keep) {
#pragma unroll
        for (int e = 0; e < P; ++e) x1[e] = x2[e] = both(0.0f);
      }
      store<kOut32, E>(y, ye + i * ys, x1);
      store<kOut32, E>(y, ye + i * ys + half, x2);
    }
  }
}

// ---------------------------------------------------------------- backward
// Blocks [0, n_q) walk the units (token, kBwdHeads heads) of q, the others
// those of k, and keep their sums of dw in registers.
template <bool kIn32, bool kGrad32, bool kOut32, int E, int LG>
__global__ void __launch_bounds__(kThreads, 2)
    qk_norm_rope_bwd_kernel(const QkRopeBwdParams p, int n_q) {
  constexpr int kGroups = kThreads / LG;
  const int op = blockIdx.x < n_q ? 0 : 1;
  const int block = blockIdx.x - (op ? n_q : 0), blocks = op ? gridDim.x - n_q : n_q;
  const int heads = op ? p.Hkv : p.H;
  const int nch = (heads + kBwdHeads - 1) / kBwdHeads;
  const int n_units = p.B * p.S * nch;
  const int j = threadIdx.x % LG;
  const int half = p.D / 2;
  const bool lane_live = j * E < half;
  const bool norm = p.w[0] != nullptr;
  constexpr int P = E / 2;
  uint64_t dw1[P], dw2[P];
#pragma unroll
  for (int i = 0; i < P; ++i) dw1[i] = dw2[i] = both(0.0f);
  Raw<true, E> w1, w2;
  w1.zero(), w2.zero();
  if (norm && lane_live) {
    w1.load(p.w[op], j * E);
    w2.load(p.w[op], half + j * E);
  }
  const float inv_d = 1.0f / (float)p.D;

  const int step = blocks * kGroups;
  // The bound is the same for every lane of a warp, which the reductions need.
  const int warp_first = block * kGroups + threadIdx.x / 32 * (32 / LG);
  const int mine = threadIdx.x % 32 / LG;
  for (long long uw = warp_first; uw < n_units; uw += step) {
    const bool live = lane_live && uw + mine < n_units;
    const int u = live ? (int)uw + mine : 0;
    const int token = u / nch, h0 = (u - token * nch) * kBwdHeads;
    const int b = token / p.S, s = token - b * p.S;
    const int n = min(kBwdHeads, heads - h0);
    const long long row = p.pos0 + (p.start ? p.start[b] : 0) + (long long)s;
    const bool keep = !p.cos_t || (row >= 0 && row < p.rows);
    if (!keep && live && j == 0) report_error(kDevBadIndex, s);
    const long long ge = b * p.dy_sb[op] + s * p.dy_ss[op] + h0 * p.dy_sh[op] + j * E;
    const long long xe = b * p.x_sb[op] + s * p.x_ss[op] + h0 * p.x_sh[op] + j * E;
    Raw<kGrad32, E> ga[kBwdHeads], gb[kBwdHeads];
    Raw<kIn32, E> xa[kBwdHeads], xb[kBwdHeads];
#pragma unroll
    for (int i = 0; i < kBwdHeads; ++i) {
      ga[i].zero(), gb[i].zero(), xa[i].zero(), xb[i].zero();
      if (live && keep && i < n) {
        ga[i].load(p.dy[op], ge + i * p.dy_sh[op]);
        gb[i].load(p.dy[op], ge + i * p.dy_sh[op] + half);
        if (norm) {
          xa[i].load(p.x[op], xe + i * p.x_sh[op]);
          xb[i].load(p.x[op], xe + i * p.x_sh[op] + half);
        }
      }
    }
    Raw<true, E> c, sn;
    c.zero(), sn.zero();
    if (p.cos_t && live && keep) {
      c.load(p.cos_t, row * half + j * E);
      sn.load(p.sin_t, row * half + j * E);
    }
    const long long ye = b * p.dx_sb[op] + s * p.dx_ss[op] + h0 * p.dx_sh[op] + j * E;
#pragma unroll
    for (int i = 0; i < kBwdHeads; ++i) {
      uint64_t d1[P], d2[P];
#pragma unroll
      for (int e = 0; e < P; ++e) {
        d1[e] = ga[i].pair(e), d2[e] = gb[i].pair(e);
        if (p.cos_t) {
          const uint64_t t = f2_mul(d1[e], f2_mul(sn.pair(e), both(-1.0f)));
          d1[e] = f2_fma(d1[e], c.pair(e), f2_mul(d2[e], sn.pair(e)));
          d2[e] = f2_fma(d2[e], c.pair(e), t);
        }
      }
      if (norm) {
        uint64_t ss = both(0.0f), gx = both(0.0f);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const uint64_t x1 = xa[i].pair(e), x2 = xb[i].pair(e);
          ss = f2_fma(x1, x1, f2_fma(x2, x2, ss));
          gx = f2_fma(f2_mul(d1[e], w1.pair(e)), x1, f2_fma(f2_mul(d2[e], w2.pair(e)), x2, gx));
        }
        // Zeros stand in for heads that are not there: with eps = 0 the floor, the
        // smallest fp32 number, keeps their rstd finite and their share of dw zero
        // (training backward 62.8 us; with a test for them 65.9).
        const float r = rsqrtf(fmaxf(fmaf(group_sum<LG>(pair_sum(ss)), inv_d, p.eps), 1.4e-45f));
        const float m = group_sum<LG>(pair_sum(gx)) * inv_d * r * r;  // mean(g xh) rstd
        const uint64_t rr = both(r), nm = both(-m);
#pragma unroll
        for (int e = 0; e < P; ++e) {
          const uint64_t x1 = xa[i].pair(e), x2 = xb[i].pair(e);
          dw1[e] = f2_fma(d1[e], f2_mul(x1, rr), dw1[e]);
          dw2[e] = f2_fma(d2[e], f2_mul(x2, rr), dw2[e]);
          d1[e] = f2_mul(rr, f2_fma(x1, nm, f2_mul(d1[e], w1.pair(e))));
          d2[e] = f2_mul(rr, f2_fma(x2, nm, f2_mul(d2[e], w2.pair(e))));
        }
      }
      if (live && i < n) {
        store<kOut32, E>(p.dx[op], ye + i * p.dx_sh[op], d1);
        store<kOut32, E>(p.dx[op], ye + i * p.dx_sh[op] + half, d2);
      }
    }
  }
  if (!norm) return;
  // The block's sums, lane groups added in order.
  __shared__ float sm[kGroups][2 * LG * E];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float* at = &sm[threadIdx.x / LG][j * E + 2 * i];
    f2_unpack(dw1[i], at[0], at[1]);
    f2_unpack(dw2[i], at[LG * E], at[LG * E + 1]);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < p.D; d += kThreads) {
    const int col = d < half ? d : LG * E + (d - half);
    float sum = 0.0f;
    for (int g = 0; g < kGroups; ++g) sum += sm[g][col];
    p.partial[(long long)blockIdx.x * p.D + d] = sum;
  }
}

// dw[op][d] = sum of the partial sums of op's blocks: 32 columns a block, eight
// slices of the blocks each, added in a fixed order.
__global__ void __launch_bounds__(256) qk_norm_dw_kernel(const float* __restrict__ partial,
                                                         int n_q, int n_blocks, int D, float* dwq,
                                                         float* dwk) {
  __shared__ float sm[8][32];
  const int op = blockIdx.y, col = threadIdx.x % 32, slice = threadIdx.x / 32;
  const int d = blockIdx.x * 32 + col;
  const int first = op ? n_q : 0, end = op ? n_blocks : n_q;
  float sum = 0.0f;
  if (d < D) {
#pragma unroll 8
    for (int i = first + slice; i < end; i += 8) sum += partial[(long long)i * D + d];
  }
  sm[slice][col] = sum;
  __syncthreads();
  if (slice == 0 && d < D) {
    for (int k = 1; k < 8; ++k) sum += sm[k][col];
    (op == 0 ? dwq : dwk)[d] = sum;
  }
}

// Lanes of a group: the power of two that holds half a head of E elements each.
int lanes_for(int D, int E) {
  int lg = 4;
  while (lg * E * 2 < D) lg *= 2;
  return lg;
}

template <bool kIn32, bool kOut32, int E, int kHeads>
cudaError_t launch_fwd_h(const QkRopeParams& p, cudaStream_t stream) {
  const int nq = (p.H + kHeads - 1) / kHeads, nk = (p.Hkv + kHeads - 1) / kHeads;
  const int LG = lanes_for(p.D, E);
  const int groups = kThreads / LG;
  const int nch = nq + nk + (p.pages[0] ? nk : 0);
  const int grid = (p.B * p.S + groups - 1) / groups * nch;
  if constexpr (E == 4) {
    if (LG == 16)
      qk_norm_rope_kernel<kIn32, kOut32, E, 16, kHeads><<<grid, kThreads, 0, stream>>>(p, nq, nk, nch);
  }
  if (LG == 8)
    qk_norm_rope_kernel<kIn32, kOut32, E, 8, kHeads><<<grid, kThreads, 0, stream>>>(p, nq, nk, nch);
  else if (LG == 4)
    qk_norm_rope_kernel<kIn32, kOut32, E, 4, kHeads><<<grid, kThreads, 0, stream>>>(p, nq, nk, nch);
  return cudaGetLastError();
}

// 16-byte loads of bf16 need halves of a multiple of eight elements. Eight
// heads a group where they leave none over and the blocks still fill the card
// (8 x 4096 tokens, 16 + 16 heads: 86 us against 91 with four; 16 + 4 heads: 34
// against 32).
template <bool kIn32, bool kOut32>
cudaError_t launch_fwd(const QkRopeParams& p, cudaStream_t stream) {
  if constexpr (!kIn32) {
    if (p.D % 16 == 0) {
      const long long groups8 = (long long)p.B * p.S * ((p.H + p.Hkv) / 8);
      if (p.H % 8 == 0 && p.Hkv % 8 == 0 && groups8 >= 1 << 15)
        return launch_fwd_h<kIn32, kOut32, 8, 8>(p, stream);
      return launch_fwd_h<kIn32, kOut32, 8, 4>(p, stream);
    }
  }
  return launch_fwd_h<kIn32, kOut32, 4, 4>(p, stream);
}

// q's share of the backward's blocks, in proportion to the heads.
int bwd_q_blocks(int n_blocks, int H, int Hkv) {
  return std::max(1, std::min(n_blocks - 1, (int)((long long)n_blocks * H / (H + Hkv))));
}

template <bool kIn32, bool kGrad32, bool kOut32>
cudaError_t launch_bwd(const QkRopeBwdParams& p, cudaStream_t stream) {
  const int LG = lanes_for(p.D, 4), blocks = p.n_blocks;
  const int n_q = bwd_q_blocks(blocks, p.H, p.Hkv);
  if (LG == 16)
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 4, 16><<<blocks, kThreads, 0, stream>>>(p, n_q);
  else if (LG == 8)
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 4, 8><<<blocks, kThreads, 0, stream>>>(p, n_q);
  else
    qk_norm_rope_bwd_kernel<kIn32, kGrad32, kOut32, 4, 4><<<blocks, kThreads, 0, stream>>>(p, n_q);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || !p.w[0]) return e;
  qk_norm_dw_kernel<<<dim3((p.D + 31) / 32, 2), 256, 0, stream>>>(p.partial, n_q, blocks, p.D,
                                                                 p.dw[0], p.dw[1]);
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

// Two blocks a SM, or one for every group of units when there are fewer; two
// at least, since q and k have their own.
int qk_rope_bwd_blocks(int B, int S, int H, int Hkv, int D, int n_sms) {
  const long long units = (long long)B * S * ((H + qkr::kBwdHeads - 1) / qkr::kBwdHeads +
                                              (Hkv + qkr::kBwdHeads - 1) / qkr::kBwdHeads);
  const long long per_block = qkr::kThreads / qkr::lanes_for(D, 4);
  const long long blocks = (units + per_block - 1) / per_block;
  return (int)std::max(2ll, std::min(blocks, (long long)n_sms * 2));
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
