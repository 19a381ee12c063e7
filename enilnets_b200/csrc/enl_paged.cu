// Attention of one new token per sequence over a paged key-value cache.
//
//   o_h = sum_j softmax_j(scale q_h . k_j - slope_h (L - 1 - j)) v_j
//
// over the positions j the query at L - 1 sees: all of them, or with a window
// the first `sinks` and those at most `window` back. Position j is slot
// j % page_size of page table[b][j / page_size].
//
// The cache's bytes bound it: 2 D e bytes a key and kv head, against 4 D flops
// for each query head of its group. So every key is loaded once for all the
// query heads that share it, and the products run on mma.sync with the keys as
// the rows and the heads as the columns (S^T = K Q^T, O^T = V^T P^T; eight heads
// are one column tile, so a group of one wastes products but no bytes). At the
// HBM rate an SM gets 16 bf16 keys of 128 every 350 cycles and spends about 30
// issue slots of each scheduler on them; tcgen05's 128-row tiles would need the
// probabilities in shared or tensor memory for no gain.
//
// Work: a sequence's visible positions are cut into tiles of 16 keys a warp;
// tiles are numbered sequence by sequence, kv head by kv head, and every block
// takes an equal run of them (the lengths are read on the device). A block
// walks its run with the loads of the next tiles in flight (cp.async, row
// addresses from the block table one tile further ahead), whatever sequence
// they belong to. Where a (sequence, head group) ends inside its run and began
// there too, the block writes the output; a part of one goes to the workspace
// and the last block to finish joins all parts in a fixed order, so the result
// does not depend on timing.
//
// Precision: scores, softmax and sums in fp32. bf16: products of bf16 inputs
// are exact; the probabilities are split into two bf16 parts (16 bits of
// mantissa), which costs a second product and keeps their rounding out of the
// output. fp32: each factor is split into two tf32 parts (values into three) and
// the three (four) largest products are added, about 2^-21 of each.
#include <algorithm>
#include <atomic>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

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

// Kernel shapes: D is the padded head dim, NT column tiles of 8 heads per item,
// NW warps. Stages are filled while the block works on one.
template <int D_, bool kF32_, int NT_, int NW_>
struct Cfg {
  static constexpr int D = D_, NT = NT_, NW = NW_;
  static constexpr bool kF32 = kF32_;
  static constexpr int kThreads = NW * 32;
  static constexpr int kKeys = NW * 16;  // keys of a tile
  static constexpr int kEsz = kF32 ? 4 : 2;
  static constexpr int kRow = D * kEsz;  // bytes of a row in shared memory
  static constexpr int kTile = kKeys * kRow;
  static constexpr int kStage = 2 * kTile;  // K, then V
  static constexpr int kStages = kStage > 16384 ? 3 : 4;
  static constexpr int kRing = kStages + 1;  // row-address slots
  static constexpr int kMerge = (NW - 1) * 8 * D * 4;
  static constexpr int kOffMerge = kStages * kStage;
  static constexpr int kOffRows = kOffMerge + kMerge;
  static constexpr int kSmem = kOffRows + kRing * kKeys * 8;
  static constexpr int kPerSm = (227 * 1024) / (kSmem + 2048);  // blocks a SM
  static constexpr int kSlot = NT * 8 * D + NT * 16;            // floats of one part
  static constexpr int kRegs = D / 16 * 4;                      // accumulators of a column tile
};

// Partial results never take more than this per SM (the counters follow them
// at a fixed place, whatever shapes share a workspace).
constexpr size_t kPartBytesPerSm = 2 * 3 * (16 * 128 + 32) * 4;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
               : "r"(addr)
               : "memory");
  return f;
}

// x = hi + lo with hi of tf32's 11 bits; lo's own tail past them is dropped by
// the product.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  lo = __float_as_uint(x - __uint_as_float(hi));
}
// x = hi + lo + rest, exact: a probability of one returns its value unchanged.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo, uint32_t& rest) {
  float left;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  left = x - __uint_as_float(hi);
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(left));
  rest = __float_as_uint(left - __uint_as_float(lo));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Swizzled place of 16-byte chunk `chunk` of row `row`: eight rows of one chunk
// (ldmatrix), or the chunks that eight lanes read at once (fp32), fall into
// different banks.
template <class C>
__device__ __forceinline__ uint32_t place(int row, int chunk) {
  const int f = C::kF32 ? (row & 6) ^ ((row & 1) << 2) : row & 7;
  return row * C::kRow + ((chunk ^ f) << 4);
}

// One tile's place in the work: item (sequence b, kv head and head block sub),
// tile t of its nt.
struct Walker {
  int b, sub, t, nt, L;
  Visible vis;
};

template <class C>
struct Decoder {
  const PagedDecodeParams& p;
  uint8_t* smem;
  uint32_t sbase;
  int G, HB, SUB;
  int lane, warp, r, q;

  // Softmax state of the warp: heads 8 nt + 2q (+1) of the item, this lane's
  // share of the sums; O^T fragments (rows: dims, columns: heads).
  float m[C::NT][2], l[C::NT][2], o[C::NT][C::kRegs / 4][4];
  // Q^T fragments.
  uint32_t qf[C::NT][C::D / 16][C::kF32 ? 8 : 2];

  __device__ int length(int b) const {
    int L = p.lens[b];
    const long long most = (long long)p.max_pages * p.page_size;
    if (L > most) L = (int)most;
    return max(L, 0);
  }
  __device__ __forceinline__ int tiles_of(int n) const { return (n + C::kKeys - 1) / C::kKeys; }

  __device__ void enter(Walker& w, int b) const {
    w.b = b;
    w.L = length(b);
    w.vis = visible_of(w.L, p.window, p.sinks);
    w.nt = tiles_of(w.vis.n);
  }
  __device__ void advance(Walker& w) const {
    if (++w.t < w.nt) return;
    w.t = 0;
    if (++w.sub < SUB) return;
    w.sub = 0;
    int b = w.b + 1;
    while (b < p.B && length(b) == 0) ++b;
    if (b < p.B) enter(w, b);
  }

  // Element offset of key `key` of the walker's tile in the pools, or -1 for
  // none (past the end, or a page outside the pool).
  __device__ long long row_offset(const Walker& w, int key) const {
    const int i = w.t * C::kKeys + key;
    if (i >= w.vis.n) return -1;
    const int j = i < w.vis.n_sink ? i : i + w.vis.gap;
    const int col = j / p.page_size;
    const int page = p.table[w.b * p.t_sb + col];
    if (page < 0 || page >= p.n_pages) {
      report_error(kDevBadIndex, w.b);
      return -1;
    }
    return page * p.p_sp + (w.sub / HB) * p.p_sh + (j - col * p.page_size) * p.p_ss;
  }
  __device__ __forceinline__ long long* rows(int slot) const {
    return reinterpret_cast<long long*>(smem + C::kOffRows) + slot * C::kKeys;
  }

  // Starts the loads of one tile.
  __device__ __forceinline__ void load_tile(int stage, int slot) const {
    constexpr int kChunks = C::kRow / 16;
    constexpr int kRows = C::kThreads / kChunks;  // rows a pass
    const int chunk = threadIdx.x % kChunks;
    const bool real = chunk * 16 < p.D * C::kEsz;
    const uint32_t dst = sbase + stage * C::kStage;
    const uint8_t* k = reinterpret_cast<const uint8_t*>(p.k);
    const uint8_t* v = reinterpret_cast<const uint8_t*>(p.v);
#pragma unroll
    for (int i = 0; i < C::kKeys / kRows; ++i) {
      const int row = threadIdx.x / kChunks + i * kRows;
      const long long off = rows(slot)[row];
      const int bytes = real && off >= 0 ? 16 : 0;
      const long long e = bytes ? off * C::kEsz + chunk * 16 : 0;
      const uint32_t at = dst + place<C>(row, chunk);
      cp_async16(at, k + e, bytes);
      cp_async16(at + C::kTile, v + e, bytes);
    }
  }

  __device__ int heads_of(const Walker& w) const {  // real heads of the item
    return min(C::NT * 8, G - (w.sub % HB) * (C::NT * 8));
  }
  __device__ int first_head(const Walker& w) const {
    return (w.sub / HB) * G + (w.sub % HB) * (C::NT * 8);
  }

  __device__ void begin_item(const Walker& w) {
    const int n = heads_of(w);
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < C::kRegs / 4; ++i)
        o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.0f;
      const int h = nt * 8 + r;  // this lane's column
      const long long e = w.b * p.q_sb + (first_head(w) + h) * p.q_sh;
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ++ks) {
        if constexpr (C::kF32) {
          const int d = ks * 16 + q * 4;
          float4 x = make_float4(0, 0, 0, 0);
          if (h < n && d < p.D)
            x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p.q) + e + d);
          split_tf32(x.x, qf[nt][ks][0], qf[nt][ks][4]);
          split_tf32(x.y, qf[nt][ks][1], qf[nt][ks][5]);
          split_tf32(x.z, qf[nt][ks][2], qf[nt][ks][6]);
          split_tf32(x.w, qf[nt][ks][3], qf[nt][ks][7]);
        } else {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int d = ks * 16 + i * 8 + q * 2;
            qf[nt][ks][i] =
                h < n && d < p.D
                    ? *reinterpret_cast<const uint32_t*>(
                          reinterpret_cast<const __nv_bfloat16*>(p.q) + e + d)
                    : 0u;
          }
        }
      }
    }
  }

  // Scores of the warp's 16 keys: rows r and r + 8, heads 2q and 2q + 1.
  __device__ __forceinline__ void scores(uint32_t kbase, float (&s)[C::NT][4]) const {
    float s2[C::NT][4];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = s2[nt][i] = 0.0f;
    if constexpr (C::kF32) {
      const int row = warp * 16 + r;
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ++ks) {
        const float4 x = lds4(kbase + place<C>(row, ks * 4 + q));
        const float4 y = lds4(kbase + place<C>(row + 8, ks * 4 + q));
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          split_tf32(half ? x.z : x.x, hi[0], lo[0]);
          split_tf32(half ? y.z : y.x, hi[1], lo[1]);
          split_tf32(half ? x.w : x.y, hi[2], lo[2]);
          split_tf32(half ? y.w : y.y, hi[3], lo[3]);
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) {
            const uint32_t* f = qf[nt][ks] + 2 * half;
            mma_tf32(s2[nt], lo, f[0], f[1]);
            mma_tf32(s2[nt], hi, f[4], f[5]);
            mma_tf32(s[nt], hi, f[0], f[1]);
          }
        }
      }
    } else {
      const int row = warp * 16 + (lane & 15);
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ++ks) {
        uint32_t a[4];
        ldmatrix4(a, kbase + place<C>(row, ks * 2 + (lane >> 4)));
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt)
          mma_bf16(ks % 2 ? s2[nt] : s[nt], a, qf[nt][ks][0], qf[nt][ks][1]);
      }
    }
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] += s2[nt][i];
  }

  // O^T += V^T P^T for the warp's 16 keys.
  __device__ __forceinline__ void accumulate(uint32_t vbase, const float (&pr)[C::NT][4]) {
    if constexpr (C::kF32) {
      uint32_t ph[C::NT][4], pl[C::NT][4];  // keys 2q, 2q+1, 8+2q, 9+2q of head r
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const uint32_t x = __float_as_uint(pr[nt][2 * half]);
          const uint32_t y = __float_as_uint(pr[nt][2 * half + 1]);
          const uint32_t tl = transpose8(__byte_perm(x, y, 0x5410));
          const uint32_t th = transpose8(__byte_perm(x, y, 0x7632));
#pragma unroll
          for (int i = 0; i < 2; ++i)
            split_tf32(__uint_as_float(__byte_perm(tl, th, i ? 0x7632 : 0x5410)),
                       ph[nt][2 * half + i], pl[nt][2 * half + i]);
        }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int row = warp * 16 + half * 8 + 2 * q;
#pragma unroll
        for (int blk = 0; blk < C::D / 32; ++blk) {
          const float4 x = lds4(vbase + place<C>(row, blk * 8 + r));
          const float4 y = lds4(vbase + place<C>(row + 1, blk * 8 + r));
          uint32_t hi[4], lo[4], rest[4];
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            split_tf32(u ? x.z : x.x, hi[0], lo[0], rest[0]);
            split_tf32(u ? x.w : x.y, hi[1], lo[1], rest[1]);
            split_tf32(u ? y.z : y.x, hi[2], lo[2], rest[2]);
            split_tf32(u ? y.w : y.y, hi[3], lo[3], rest[3]);
#pragma unroll
            for (int nt = 0; nt < C::NT; ++nt) {
              float(&acc)[4] = o[nt][blk * 2 + u];
              mma_tf32(acc, rest, ph[nt][2 * half], ph[nt][2 * half + 1]);
              mma_tf32(acc, lo, ph[nt][2 * half], ph[nt][2 * half + 1]);
              mma_tf32(acc, hi, pl[nt][2 * half], pl[nt][2 * half + 1]);
              mma_tf32(acc, hi, ph[nt][2 * half], ph[nt][2 * half + 1]);
            }
          }
        }
      }
    } else {
      uint32_t bh[C::NT][2], bl[C::NT][2];
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float x = pr[nt][2 * half], y = pr[nt][2 * half + 1];
          const uint32_t hi = pack_bf16(x, y);
          bh[nt][half] = transpose8(hi);
          bl[nt][half] = transpose8(pack_bf16(x - bf16lo_to_f32(hi), y - bf16hi_to_f32(hi)));
        }
      const int row = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int mt = 0; mt < C::D / 16; ++mt) {
        uint32_t a[4];
        ldmatrix4_trans(a, vbase + place<C>(row, mt * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          mma_bf16(o[nt][mt], a, bl[nt][0], bl[nt][1]);
          mma_bf16(o[nt][mt], a, bh[nt][0], bh[nt][1]);
        }
      }
    }
  }

  // Takes a new maximum for the state's heads, scaling what is there.
  __device__ __forceinline__ void raise(const float (&mx)[C::NT][2]) {
    bool grew = false;
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) grew |= mx[nt][0] > m[nt][0] || mx[nt][1] > m[nt][1];
    if (!__any_sync(0xffffffffu, grew)) return;
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float top = fmaxf(m[nt][i], mx[nt][i]);
        f[i] = top > -INFINITY ? fast_exp2(m[nt][i] - top) : 1.0f;
        m[nt][i] = top;
        l[nt][i] *= f[i];
      }
#pragma unroll
      for (int i = 0; i < C::kRegs / 4; ++i) {
        o[nt][i][0] *= f[0], o[nt][i][1] *= f[1];
        o[nt][i][2] *= f[0], o[nt][i][3] *= f[1];
      }
    }
  }

  __device__ __forceinline__ void tile(const Walker& w, int stage, int slot) {
    const uint32_t kbase = sbase + stage * C::kStage;
    float s[C::NT][4];
    scores(kbase, s);
    const int key = warp * 16 + r;
    const bool ok0 = rows(slot)[key] >= 0, ok1 = rows(slot)[key + 8] >= 0;
    float mx[C::NT][2];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] *= p.scale * kLog2e;
      if (p.alibi) {
        const int n = heads_of(w), h0 = first_head(w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int h = nt * 8 + 2 * q + i % 2;
          const int idx = w.t * C::kKeys + key + i / 2 * 8;
          const int j = idx < w.vis.n_sink ? idx : idx + w.vis.gap;
          if (h < n) s[nt][i] -= p.alibi[h0 + h] * kLog2e * (float)(w.L - 1 - j);
        }
      }
      if (!ok0) s[nt][0] = s[nt][1] = -INFINITY;
      if (!ok1) s[nt][2] = s[nt][3] = -INFINITY;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(s[nt][i], s[nt][i + 2]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
        mx[nt][i] = x;
      }
    }
    raise(mx);
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float top = m[nt][i % 2] > -INFINITY ? m[nt][i % 2] : 0.0f;  // no visible key yet
        s[nt][i] = fast_exp2(s[nt][i] - top);
        l[nt][i % 2] += s[nt][i];
      }
    accumulate(kbase + C::kTile, s);
  }

  // Sums the lanes' shares of l, then joins the warps' states into warp 0's.
  __device__ void join_warps() {
    float* buf = reinterpret_cast<float*>(smem + C::kOffMerge);
    __shared__ float sm[C::NW][C::NT * 8], sl[C::NW][C::NT * 8];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1)
          l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], off);
        if (r == 0) sm[warp][nt * 8 + 2 * q + i] = m[nt][i], sl[warp][nt * 8 + 2 * q + i] = l[nt][i];
      }
    __syncthreads();
    float top[C::NT][2];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        top[nt][i] = m[nt][i];
#pragma unroll
        for (int w = 0; w < C::NW; ++w)
          top[nt][i] = fmaxf(top[nt][i], sm[w][nt * 8 + 2 * q + i]);
      }
    raise(top);
    if (warp == 0) {
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int w = 1; w < C::NW; ++w) {
            const int h = nt * 8 + 2 * q + i;
            if (sm[w][h] > -INFINITY) l[nt][i] += sl[w][h] * fast_exp2(sm[w][h] - m[nt][i]);
          }
    }
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      if (nt > 0) __syncthreads();
      if (warp > 0) {
#pragma unroll
        for (int i = 0; i < C::kRegs; ++i)
          buf[((warp - 1) * C::kRegs + i) * 32 + lane] = o[nt][i / 4][i % 4];
      }
      __syncthreads();
      if (warp == 0) {
#pragma unroll
        for (int w = 0; w < C::NW - 1; ++w)
#pragma unroll
          for (int i = 0; i < C::kRegs; ++i)
            o[nt][i / 4][i % 4] += buf[(w * C::kRegs + i) * 32 + lane];
      }
    }
  }

  // Dim of accumulator i of a column tile.
  __device__ __forceinline__ int dim_of(int i) const {
    const int tile = i / 4, second = (i % 4) / 2;  // rows r and r + 8
    return C::kF32 ? tile / 2 * 32 + r * 4 + tile % 2 * 2 + second : tile * 16 + second * 8 + r;
  }

  __device__ void write_output(const Walker& w) const {  // warp 0
    const int n = heads_of(w);
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int h = nt * 8 + 2 * q + c;
        if (h >= n) continue;
        const int head = first_head(w) + h;
        const float inv = l[nt][c] > 0.0f ? 1.0f / l[nt][c] : l[nt][c] == 0.0f ? 0.0f : l[nt][c];
        const long long e = w.b * p.o_sb + head * p.o_sh;
#pragma unroll
        for (int i = c; i < C::kRegs; i += 2) {
          const int d = dim_of(i);
          if (d >= p.D) continue;
          const float x = o[nt][i / 4][i % 4] * inv;
          if (p.out_fp32)
            reinterpret_cast<float*>(p.o)[e + d] = x;
          else
            reinterpret_cast<__nv_bfloat16*>(p.o)[e + d] = __float2bfloat16_rn(x);
        }
        if (r == 0 && p.lse)
          p.lse[(long long)w.b * p.H + head] =
              l[nt][c] == 0.0f ? -INFINITY : (m[nt][c] + log2f(l[nt][c])) * kLn2;
      }
  }

  __device__ __forceinline__ float* slot_of(long long cta, int which) const {
    return reinterpret_cast<float*>(p.workspace) + (cta * 2 + which) * C::kSlot;
  }
  __device__ void write_part(float* part) const {  // warp 0
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
#pragma unroll
      for (int i = 0; i < C::kRegs; ++i)
        part[(nt * C::kRegs + i) * 32 + lane] = o[nt][i / 4][i % 4];
      if (r == 0) {
        float* ml = part + C::NT * 8 * C::D + nt * 16;
#pragma unroll
        for (int i = 0; i < 2; ++i) ml[2 * q + i] = m[nt][i], ml[8 + 2 * q + i] = l[nt][i];
      }
    }
  }
  // Adds a part to the state (its sums count in the lanes of r == 0 only).
  __device__ void add_part(const float* part) {
    float pm[C::NT][2], pl[C::NT][2];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float* ml = part + C::NT * 8 * C::D + nt * 16;
        pm[nt][i] = __ldcg(ml + 2 * q + i);
        pl[nt][i] = __ldcg(ml + 8 + 2 * q + i);
      }
    float po[C::NT][C::kRegs];
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < C::kRegs; ++i) po[nt][i] = __ldcg(part + (nt * C::kRegs + i) * 32 + lane);
    raise(pm);
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[i] = pm[nt][i] > -INFINITY ? fast_exp2(pm[nt][i] - m[nt][i]) : 0.0f;
        if (r == 0) l[nt][i] += pl[nt][i] * f[i];
      }
#pragma unroll
      for (int i = 0; i < C::kRegs; ++i)
        o[nt][i / 4][i % 4] = fmaf(po[nt][i], f[i % 2], o[nt][i / 4][i % 4]);
    }
  }

  // The walker's item ends with this tile, or the block's run does. g: the
  // tile's number among all T; the block's run starts at `first`.
  // Block c of n takes tiles [c T / n, (c + 1) T / n).
  __device__ void end_segment(const Walker& w, long long g, long long first, long long T,
                              long long n) {
    __shared__ int last;
    join_warps();
    const long long a = g - w.t, z = a + w.nt;  // the item's tiles
    if (first <= a && g == z - 1) {
      if (warp == 0) write_output(w);
      return;
    }
    auto block_of = [&](long long t) { return ((t + 1) * n - 1) / T; };
    const long long c0 = block_of(a), c1 = block_of(z - 1);
    int* count = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(p.workspace) +
                                        p.n_sms * kPartBytesPerSm) + (w.b * SUB + w.sub);
    if (warp == 0) {
      write_part(slot_of(blockIdx.x, first >= a ? 0 : 1));
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        last = atomicAdd(count, 1) == (int)(c1 - c0);
        if (last) *count = 0;  // for the next call
        __threadfence();
      }
    }
    __syncthreads();
    if (!last) return;
    // The warps share the parts, each in ascending order.
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < C::kRegs; ++i) o[nt][i / 4][i % 4] = 0.0f;
    }
    for (long long c = c0 + warp; c <= c1; c += C::NW)
      add_part(slot_of(c, c * T / n >= a ? 0 : 1));
    join_warps();
    if (warp == 0) write_output(w);
  }

  __device__ void run() {
    constexpr int S = C::kStages;
    const int tid = threadIdx.x;
    // Every sequence's tiles: this thread's stretch of sequences, then a scan.
    __shared__ long long scan[C::NW];
    __shared__ int s_b, s_rest;
    const int per = (p.B + C::kThreads - 1) / C::kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    long long mine = 0;
    for (int b = b0; b < b1; ++b) {
      const int L = length(b);
      if (blockIdx.x == 0 && p.lens[b] > L) report_error(kDevBadIndex, b);
      mine += tiles_of(visible_of(L, p.window, p.sinks).n);
    }
    long long inc = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += y;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    long long before = 0, T = 0;
#pragma unroll
    for (int w = 0; w < C::NW; ++w) {
      if (w < warp) before += scan[w];
      T += scan[w];
    }
    before += inc - mine;
    // Sequences without a visible position: a zero output.
    for (int b = blockIdx.x; b < p.B; b += gridDim.x)
      if (length(b) == 0)
        for (int i = tid; i < p.H * p.D; i += C::kThreads) {
          const int h = i / p.D, d = i % p.D;
          const long long e = b * p.o_sb + h * p.o_sh + d;
          if (p.out_fp32)
            reinterpret_cast<float*>(p.o)[e] = 0.0f;
          else
            reinterpret_cast<__nv_bfloat16*>(p.o)[e] = __float2bfloat16_rn(0.0f);
          if (d == 0 && p.lse) p.lse[(long long)b * p.H + h] = -INFINITY;
        }
    // No more blocks than tiles take part, so none of those has an empty run.
    T *= SUB;
    const long long blocks = min((long long)gridDim.x, T);
    if (blockIdx.x >= blocks) return;
    const long long first = blockIdx.x * T / blocks, end = (blockIdx.x + 1ll) * T / blocks;
    const int n = (int)(end - first);
    // The sequence that holds the run's first tile.
    if (before * SUB <= first && first < (before + mine) * SUB) {
      long long run = before;
      int b = b0;
      for (;; ++b) {
        const int nt = tiles_of(visible_of(length(b), p.window, p.sinks).n);
        if (first < (run + nt) * SUB) break;
        run += nt;
      }
      s_b = b;
      s_rest = (int)(first - run * SUB);
    }
    __syncthreads();
    Walker ahead, here;
    enter(ahead, s_b);
    ahead.sub = s_rest / ahead.nt;
    ahead.t = s_rest % ahead.nt;
    here = ahead;

    // Row addresses of the first S tiles, loads of the first S - 1.
#pragma unroll
    for (int i = 0; i < S; ++i)
      if (i < n) {
        if (tid < C::kKeys) rows(i)[tid] = row_offset(ahead, tid);
        advance(ahead);
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S - 1; ++i) {
      if (i < n) load_tile(i, i);
      cp_commit();
    }
    begin_item(here);
    for (int i = 0; i < n; ++i) {
      cp_wait<S - 2>();
      __syncthreads();
      if (i + S - 1 < n) load_tile((i + S - 1) % S, (i + S - 1) % C::kRing);
      cp_commit();
      long long next = -1;
      const bool more = i + S < n;
      if (more && tid < C::kKeys) next = row_offset(ahead, tid);
      tile(here, i % S, i % C::kRing);
      if (more) {
        if (tid < C::kKeys) rows((i + S) % C::kRing)[tid] = next;
        advance(ahead);
      }
      if (here.t == here.nt - 1 || i == n - 1) end_segment(here, first + i, first, T, blocks);
      advance(here);
      if (here.t == 0 && i + 1 < n) begin_item(here);
    }
  }
};

template <class C>
__global__ void __launch_bounds__(C::kThreads) paged_kernel(const PagedDecodeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  Decoder<C> d{p};
  d.smem = smem;
  d.sbase = smem_u32(smem);
  d.G = p.H / p.Hkv;
  d.HB = (d.G + C::NT * 8 - 1) / (C::NT * 8);
  d.SUB = p.Hkv * d.HB;
  d.lane = threadIdx.x % 32;
  d.warp = threadIdx.x / 32;
  d.r = d.lane / 4;
  d.q = d.lane % 4;
  d.run();
}

template <class C>
cudaError_t launch(const PagedDecodeParams& p, cudaStream_t stream) {
  static_assert(C::kPerSm * 2 * C::kSlot * 4 <= kPartBytesPerSm, "parts fit the workspace");
  static_assert(C::kPerSm >= 1, "a block fits an SM");
  const int G = p.H / p.Hkv;
  const long long most = std::min<long long>((long long)p.max_pages * p.page_size, 0x7fffffff);
  const long long tiles = (long long)p.B * p.Hkv * ((G + C::NT * 8 - 1) / (C::NT * 8)) *
                          ((most + C::kKeys - 1) / C::kKeys);
  const int grid = (int)std::min<long long>(tiles, (long long)p.n_sms * C::kPerSm);
  static std::atomic<unsigned long long> ready{0};  // devices whose limit is raised
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= 64 || !(ready.load() >> dev & 1)) {
    e = cudaFuncSetAttribute(paged_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < 64) ready.fetch_or(1ull << dev);
  }
  paged_kernel<C><<<grid, C::kThreads, C::kSmem, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace paged

size_t paged_decode_workspace(int B, int H, int Hkv, int D, int n_sms) {
  // One counter per item at most: a head block is never smaller than a group's
  // eight heads.
  const size_t blocks = (H / Hkv + 7) / 8;
  return n_sms * paged::kPartBytesPerSm + ((size_t)B * Hkv * blocks * 4 + 255) / 256 * 256;
}

cudaError_t launch_paged_decode(const PagedDecodeParams& p, cudaStream_t stream) {
  using namespace paged;
  const bool wide = p.H / p.Hkv > 8;  // more than one column tile
  if (p.in_fp32)
    return p.D > 64 ? launch<Cfg<128, true, 1, 2>>(p, stream)
                    : launch<Cfg<64, true, 1, 4>>(p, stream);
  if (p.D > 64)
    return wide ? launch<Cfg<128, false, 2, 4>>(p, stream)
                : launch<Cfg<128, false, 1, 4>>(p, stream);
  return wide ? launch<Cfg<64, false, 2, 4>>(p, stream) : launch<Cfg<64, false, 1, 4>>(p, stream);
}

}  // namespace enl
