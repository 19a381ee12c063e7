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
// are one column tile, so a group of one wastes products but no bytes). fp32
// products on that pipe take three or four tf32 ones and the splits of every
// element, so up to four fp32 heads a group are computed on the FMA pipe instead,
// two products an instruction, each element used as it is loaded (16 x 6144 keys
// of 128: 130 us against 186). At the HBM rate an SM gets 16 bf16 keys of 128
// every 350 cycles and spends about 30 issue slots of each scheduler on them;
// tcgen05's 128-row tiles would need the probabilities in shared or tensor memory
// for no gain.
//
// Work: a sequence's visible positions are cut into tiles of 16 keys a warp;
// tiles are numbered sequence by sequence, head group by head group, and every
// block takes an equal run of them (the lengths are read on the device). One
// or two warps of a block only load: they walk the run through a ring of stages
// with cp.async, which takes pages of any size, alignment and order, and leave
// with each tile a note of whose it is and which keys exist. The other warps
// wait for a stage, compute and hand it back, each at its own pace. (With the
// loads issued by the computing warps and a block barrier a tile, every
// instruction of the address work added to the time: 287 us against 244 for 64
// sequences of 6144.) Where a (sequence, head group) ends inside its run
// and began there too, the block writes the output; a part of one goes to the
// workspace and the last block to finish joins all parts in a fixed order, so
// the result does not depend on timing. Short sequences (up to kWholeTiles
// tiles) are not divided: joining two parts costs about four tiles' time.
//
// Precision: scores, softmax and sums in fp32. bf16: products of bf16 inputs are
// exact, and a probability is cut into three bf16 parts that hold it exactly. (With
// two parts the relative error of an fp32 output over 4000 random keys is 1.7e-6
// instead of 1.8e-7, in the same time up to eight heads a group, where the bytes
// bound it.) The parts have one sign and none is zero, so that an infinite value
// comes out infinite. fp32 on the FMA pipe: a tile's sum by itself, then added to
// the running one, so that equal values do not add up equal roundings. fp32 on the
// tensor pipe: each factor is split into two tf32 parts (values into three) and the
// three (four) largest products are added, about 2^-21 of each; infinities are kept
// whole, and no part of a probability is zero. The tensor pipe cuts its sums instead
// of rounding them, always towards zero, so nothing is summed in it for long: a few
// products at a time start from zero and are added to the running sums by rounded
// additions, two an instruction (without that, 16000 equal fp32 values came out
// 3e-5 small). With two column tiles these additions show: 64
// sequences of 12288, four key heads of 128 with 16 query heads each, take 308 us,
// against 304 with sums that stay in the pipe (16000 equal values then come out
// 1e-5 small instead of 4e-7) and 293 with two parts of a probability as well.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace paged {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kSite = 70;  // of this file's waits in the device error word

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

constexpr int kLens = 256;  // sequence lengths kept in shared memory
constexpr int kWholeTiles = 6;

// Kernel shapes: D is the padded head dim, NT column tiles of 8 heads per item,
// NW computing warps, S stages. kFma: not on the tensor pipe, with that many
// heads per item (fp32).
template <int D_, bool kF32_, int NT_, int NW_, int S_, int kFma_ = 0>
struct Cfg {
  static constexpr int D = D_, NT = NT_, NW = NW_, S = S_;
  static constexpr bool kF32 = kF32_;
  static constexpr int kFma = kFma_;
  static constexpr int kItem = kFma ? kFma : NT * 8;  // heads of an item
  static constexpr int kKeys = NW * 16;  // keys of a tile
  static constexpr int NP = kKeys / 32;  // loading warps, a key a lane
  static constexpr int kThreads = (NW + NP) * 32;
  static constexpr int kEsz = kF32 ? 4 : 2;
  static constexpr int kRow = D * kEsz;  // bytes of a row in shared memory
  static constexpr int kTile = kKeys * kRow;
  static constexpr int kStage = 2 * kTile;  // K, then V
  static constexpr int kMerge = (kFma ? (2 * NW - 1) * kFma : (NW - 1) * 8) * D * 4;
  static constexpr int kSmem = S * kStage + kMerge;
  static constexpr int kStatic = kLens * 4 + S * 64 + 768;           // at most
  static constexpr int kFit = 228 * 1024 / (kSmem + kStatic + 1024);
  static constexpr int kPerSm = NT > 1 && kFit > 2 ? 2 : kFit;  // blocks a SM (registers)
  static constexpr int kSlot = kFma ? kFma * (D + 4) : NT * 8 * D + NT * 16;  // floats of a part
  static constexpr int kRegs = D / 16 * 4;  // accumulators of a column tile
};

// What the loading warps say about a stage's tile.
struct Note {
  uint32_t ok[2];  // bit k: key k exists
  int b, sub, t, nt, L, n_sink, gap, n_keys;
};

// Partial results never take more than this per SM (the counters follow them
// at a fixed place, whatever shapes share a workspace).
constexpr size_t kPartBytesPerSm = 2 * 3 * (16 * 128 + 32) * 4;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(bytes)
               : "memory");
}
// Arrives on the barrier when this thread's copies so far have landed.
__device__ __forceinline__ void cp_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
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
// c = a b, for sums that start here.
__device__ __forceinline__ void mma_bf16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                               uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%10, %10, %10, %10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void add4(float (&c)[4], const float (&t)[4]) {
  f2_unpack(f2_add(f2_pack(c[0], c[1]), f2_pack(t[0], t[1])), c[0], c[1]);
  f2_unpack(f2_add(f2_pack(c[2], c[3]), f2_pack(t[2], t[3])), c[2], c[3]);
}
__device__ __forceinline__ float4 lds4(uint32_t addr) {
  float4 f;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
               : "r"(addr)
               : "memory");
  return f;
}

__device__ __forceinline__ void lds2x2(uint32_t addr, uint64_t& a, uint64_t& b) {
  asm volatile("ld.shared.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "r"(addr) : "memory");
}

// x = hi + lo with hi the upper 11 bits (tf32); lo's own tail past 11 bits is
// dropped by the product. Cutting takes one logic instruction where rounding
// takes a conversion at a quarter of the rate. kInf: of an infinity too, whose
// difference would be NaN.
template <bool kInf = false>
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = __float_as_uint(x) & 0xffffe000u;
  const float h = __uint_as_float(hi);
  lo = __float_as_uint(kInf && x == h ? 0.0f : x - h);
}
// x = hi + lo + rest, exact (of an infinity, hi): a probability of one returns its
// value unchanged.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo, uint32_t& rest) {
  split_tf32<true>(x, hi, lo);
  const float left = __uint_as_float(lo);
  lo &= 0xffffe000u;
  rest = __float_as_uint(left - __uint_as_float(lo));
}
// For a lower part of zero the smallest normal number of the upper part's sign:
// zero times infinity would be NaN.
__device__ __forceinline__ uint32_t not_zero(uint32_t lo, uint32_t hi) {
  return lo << 1 ? lo : (hi & 0x80000000u) | 0x00800000u;
}
// The upper 8 bits of the mantissas of x and y as two bf16; x and y are left with
// the rest. After three cuts nothing is left.
__device__ __forceinline__ uint32_t cut_bf16(float& x, float& y) {
  const uint32_t u = __float_as_uint(x), v = __float_as_uint(y);
  x -= __uint_as_float(u & 0xffff0000u);
  y -= __uint_as_float(v & 0xffff0000u);
  return __byte_perm(u, v, 0x7632);
}
// The smallest normal number in place of zeros: a probability's lower parts times
// an infinite value are infinite like the upper part times it, where zero (or a
// part of the other sign) would make NaN.
__device__ __forceinline__ uint32_t above_zero(uint32_t pair) {
  const uint32_t tiny = 0x00800080u;
  const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&pair),
                                   *reinterpret_cast<const __nv_bfloat162*>(&tiny));
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Swizzled place of 16-byte chunk `chunk` of row `row`: eight rows of one chunk
// (ldmatrix), or the chunks that eight lanes read at once (fp32), fall into
// different banks.
template <class C>
__device__ __forceinline__ uint32_t place(int row, int chunk) {
  const int f = C::kF32 ? (row & 6) ^ ((row & 1) << 2) : row & 7;
  return row * C::kRow + ((chunk ^ f) << 4);
}

// Adds 16 dims' products of 16 keys with eight heads, in fp32 on the tensor pipe. x, y:
// this lane's dims of keys r and r + 8, f: of its head, split.
template <bool kInf>
__device__ __forceinline__ void add_scores(float (&s)[4], const float4& x, const float4& y,
                                           const uint32_t* f) {
  uint32_t hi[2][4], lo[2][4];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    split_tf32<kInf>(half ? x.z : x.x, hi[half][0], lo[half][0]);
    split_tf32<kInf>(half ? y.z : y.x, hi[half][1], lo[half][1]);
    split_tf32<kInf>(half ? x.w : x.y, hi[half][2], lo[half][2]);
    split_tf32<kInf>(half ? y.w : y.y, hi[half][3], lo[half][3]);
  }
  float t[4];  // the small products first
  mma_tf32_first(t, lo[0], f[0], f[1]);
  mma_tf32(t, hi[0], f[4], f[5]);
  mma_tf32(t, lo[1], f[2], f[3]);
  mma_tf32(t, hi[1], f[6], f[7]);
  mma_tf32(t, hi[0], f[0], f[1]);
  mma_tf32(t, hi[1], f[2], f[3]);
  add4(s, t);
}

// A warp's scores once more, for infinite keys: the common path's splits make their
// products NaN, for every head (an infinite query's weights are NaN in any case). row: of key r in the tile; query: this
// lane's dims of its head, or null. A function of its own, which the common path's
// registers do not pay for: splits for infinities everywhere would make 16
// sequences of 6144 keys, 8 key heads of 128 with 8 query heads each, 193 us
// instead of 186, checks of the values' products like this one 204.
template <class C>
__device__ __noinline__ float4 scores_again(uint32_t kbase, int row, int q, const float* query,
                                            int D) {
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
  for (int ks = 0; ks < C::D / 16; ++ks) {
    float4 x = make_float4(0, 0, 0, 0);
    if (query && ks * 16 + q * 4 < D) x = *reinterpret_cast<const float4*>(query + ks * 16);
    uint32_t f[8];
    split_tf32<true>(x.x, f[0], f[4]);
    split_tf32<true>(x.y, f[1], f[5]);
    split_tf32<true>(x.z, f[2], f[6]);
    split_tf32<true>(x.w, f[3], f[7]);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[4 + i] = not_zero(f[4 + i], f[i]);
    add_scores<true>(s, lds4(kbase + place<C>(row, ks * 4 + q)),
                     lds4(kbase + place<C>(row + 8, ks * 4 + q)), f);
  }
  return make_float4(s[0], s[1], s[2], s[3]);
}

// One tile's place in the work: item (sequence b, kv head and head block sub),
// tile t of its nt.
struct Walker {
  int b, sub, t, nt, L;
  Visible vis;
};

struct Block {  // shared by a block's warps
  int lens[kLens];  // lengths of sequences [lens_b, lens_b + kLens)
  uint64_t full[4], empty[4];
  Note note[4];
  long long scan[8];
  int longest[8];
  int b;  // where the run starts: the sequence, and the units of it before
  long long rest;
  int last;
  int abort;  // a wait ran out: the others stop waiting
  float m[4][16], l[4][16];
};

// What a block's warps know.
template <class C>
struct Base {
  const PagedDecodeParams& p;
  Block& sh;
  uint8_t* smem;
  uint32_t sbase;
  int G, HB, SUB;  // heads a group, head blocks a group, head blocks in all
  int lane, warp;

  __device__ Base(const PagedDecodeParams& p_, Block& sh_, uint8_t* smem_)
      : p(p_), sh(sh_), smem(smem_), sbase(smem_u32(smem_)) {
    G = p.H / p.Hkv;
    HB = (G + C::kItem - 1) / C::kItem;
    SUB = p.Hkv * HB;
    lane = threadIdx.x % 32;
    warp = threadIdx.x / 32;
  }

  __device__ __forceinline__ void sync_warps() const { named_bar_sync(1, C::NW * 32); }

  __device__ int heads_of(const Note& w) const {  // real heads of the item
    return min(C::kItem, G - (w.sub % HB) * (C::kItem));
  }
  __device__ int first_head(const Note& w) const {
    return (w.sub / HB) * G + (w.sub % HB) * (C::kItem);
  }
};

// The computing warps on the tensor pipe.
template <class C>
struct MmaMath : Base<C> {
  using Base<C>::p;
  using Base<C>::sh;
  using Base<C>::smem;
  using Base<C>::sbase;
  using Base<C>::lane;
  using Base<C>::warp;
  using Base<C>::sync_warps;
  using Base<C>::heads_of;
  using Base<C>::first_head;
  const int r = lane / 4, q = lane % 4;

  // Softmax state of the warp: heads 8 nt + 2q (+1) of the item, this lane's
  // share of the sums; O^T fragments (rows: dims, columns: heads).
  float m[C::NT][2], l[C::NT][2], o[C::NT][C::kRegs / 4][4];
  // Q^T fragments.
  uint32_t qf[C::NT][C::D / 16][C::kF32 ? 8 : 2];

  using Base<C>::Base;

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.0f;
#pragma unroll
      for (int i = 0; i < C::kRegs; ++i) o[nt][i / 4][i % 4] = 0.0f;
    }
  }
  __device__ __forceinline__ void fold() {}

  __device__ void begin_item(const Note& w) {
    const int n = heads_of(w);
    const long long q0 = w.b * p.q_sb + first_head(w) * p.q_sh;
    clear();
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      const int h = nt * 8 + r;  // this lane's column
      const long long e = q0 + h * p.q_sh;
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
  __device__ __forceinline__ void scores(const Note& w, uint32_t kbase,
                                         float (&s)[C::NT][4]) const {
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[nt][i] = 0.0f;
    if constexpr (C::kF32) {
      static_assert(C::NT == 1, "one column tile in fp32");
      const int row = warp * 16 + r;
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ++ks)
        add_scores<false>(s[0], lds4(kbase + place<C>(row, ks * 4 + q)),
                          lds4(kbase + place<C>(row + 8, ks * 4 + q)), qf[0][ks]);
      if (__any_sync(0xffffffffu, isnan(s[0][0] + s[0][2]))) {  // key r, key r + 8
        const float* query = reinterpret_cast<const float*>(p.q) + w.b * p.q_sb +
                             (first_head(w) + r) * p.q_sh + q * 4;
        const float4 x =
            scores_again<C>(kbase, row, q, r < heads_of(w) ? query : nullptr, p.D);
        s[0][0] = x.x, s[0][1] = x.y, s[0][2] = x.z, s[0][3] = x.w;
      }
    } else {
      const int row = warp * 16 + (lane & 15);
#pragma unroll
      for (int ks = 0; ks < C::D / 16; ks += 2) {
        uint32_t a[4], b[4];
        ldmatrix4(a, kbase + place<C>(row, ks * 2 + (lane >> 4)));
        ldmatrix4(b, kbase + place<C>(row, ks * 2 + 2 + (lane >> 4)));
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          float t[4];
          mma_bf16_first(t, a, qf[nt][ks][0], qf[nt][ks][1]);
          mma_bf16(t, b, qf[nt][ks + 1][0], qf[nt][ks + 1][1]);
          add4(s[nt], t);
        }
      }
    }
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
          for (int i = 0; i < 2; ++i) {
            uint32_t &hi = ph[nt][2 * half + i], &lo = pl[nt][2 * half + i];
            split_tf32(__uint_as_float(__byte_perm(tl, th, i ? 0x7632 : 0x5410)), hi, lo);
            lo = not_zero(lo, hi);
          }
        }
      const int row = warp * 16 + 2 * q;  // and row + 1; row + 8, row + 9
#pragma unroll
      for (int blk = 0; blk < C::D / 32; ++blk) {
        float4 x[2], y[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          x[half] = lds4(vbase + place<C>(row + 8 * half, blk * 8 + r));
          y[half] = lds4(vbase + place<C>(row + 8 * half + 1, blk * 8 + r));
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t hi[2][4], lo[2][4], rest[2][4];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            split_tf32(u ? x[half].z : x[half].x, hi[half][0], lo[half][0], rest[half][0]);
            split_tf32(u ? x[half].w : x[half].y, hi[half][1], lo[half][1], rest[half][1]);
            split_tf32(u ? y[half].z : y[half].x, hi[half][2], lo[half][2], rest[half][2]);
            split_tf32(u ? y[half].w : y[half].y, hi[half][3], lo[half][3], rest[half][3]);
          }
#pragma unroll
          for (int nt = 0; nt < C::NT; ++nt) {
            float t[4];
            mma_tf32_first(t, rest[0], ph[nt][0], ph[nt][1]);
            mma_tf32(t, rest[1], ph[nt][2], ph[nt][3]);
            mma_tf32(t, lo[0], ph[nt][0], ph[nt][1]);
            mma_tf32(t, lo[1], ph[nt][2], ph[nt][3]);
            mma_tf32(t, hi[0], pl[nt][0], pl[nt][1]);
            mma_tf32(t, hi[1], pl[nt][2], pl[nt][3]);
            mma_tf32(t, hi[0], ph[nt][0], ph[nt][1]);
            mma_tf32(t, hi[1], ph[nt][2], ph[nt][3]);
            add4(o[nt][blk * 2 + u], t);
          }
        }
      }
    } else {
      uint32_t hi[C::NT][2], mid[C::NT][2], lo[C::NT][2];
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x = pr[nt][2 * half], y = pr[nt][2 * half + 1];
          hi[nt][half] = transpose8(cut_bf16(x, y));
          mid[nt][half] = transpose8(above_zero(cut_bf16(x, y)));
          lo[nt][half] = transpose8(above_zero(cut_bf16(x, y)));
        }
      const int row = warp * 16 + (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
      for (int mt = 0; mt < C::D / 16; ++mt) {
        uint32_t a[4];
        ldmatrix4_trans(a, vbase + place<C>(row, mt * 2 + ((lane >> 3) & 1)));
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
          float t[4];
          mma_bf16_first(t, a, lo[nt][0], lo[nt][1]);
          mma_bf16(t, a, mid[nt][0], mid[nt][1]);
          mma_bf16(t, a, hi[nt][0], hi[nt][1]);
          add4(o[nt][mt], t);
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

  __device__ __forceinline__ void tile(const Note& w, int stage) {
    const uint32_t kbase = sbase + stage * C::kStage;
    float s[C::NT][4];
    scores(w, kbase, s);
    const int key = warp * 16 + r;  // this lane's keys: key and key + 8
    const uint32_t ok = w.ok[C::NP > 1 ? warp / 2 : 0] >> (key & 31);
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
          const int j = idx < w.n_sink ? idx : idx + w.gap;
          if (h < n) s[nt][i] -= p.alibi[h0 + h] * kLog2e * (float)(w.L - 1 - j);
        }
      }
      if (!(ok & 1)) s[nt][0] = s[nt][1] = -INFINITY;
      if (!(ok & 256)) s[nt][2] = s[nt][3] = -INFINITY;
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

  // Sums the lanes' shares of l, then joins the states of the first n warps,
  // the others having none, into warp 0's.
  __device__ void join_warps(int n) {
    float* buf = reinterpret_cast<float*>(smem + C::S * C::kStage);
    if (warp < n) {
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int off = 4; off < 32; off <<= 1)
            l[nt][i] += __shfl_xor_sync(0xffffffffu, l[nt][i], off);
          if (r == 0) {
            sh.m[warp][nt * 8 + 2 * q + i] = m[nt][i];
            sh.l[warp][nt * 8 + 2 * q + i] = l[nt][i];
          }
        }
    }
    if (n == 1) return;
    sync_warps();
    if (warp < n) {
      float top[C::NT][2];
#pragma unroll
      for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          top[nt][i] = m[nt][i];
          for (int w = 0; w < n; ++w) top[nt][i] = fmaxf(top[nt][i], sh.m[w][nt * 8 + 2 * q + i]);
        }
      raise(top);
      if (warp == 0) {
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            for (int w = 1; w < n; ++w) {
              const int h = nt * 8 + 2 * q + i;
              if (sh.m[w][h] > -INFINITY) l[nt][i] += sh.l[w][h] * fast_exp2(sh.m[w][h] - m[nt][i]);
            }
      }
    }
#pragma unroll
    for (int nt = 0; nt < C::NT; ++nt) {
      if (nt > 0) sync_warps();
      if (warp > 0 && warp < n) {
#pragma unroll
        for (int i = 0; i < C::kRegs; ++i)
          buf[((warp - 1) * C::kRegs + i) * 32 + lane] = o[nt][i / 4][i % 4];
      }
      sync_warps();
      if (warp == 0) {
        for (int w = 0; w < n - 1; ++w)
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

  __device__ void write_output(const Note& w) const {  // warp 0
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
};

// The computing warps on the FMA pipe: two lanes share a key's dims for its
// score, then each lane adds up four dims over its keys (with 64 dims, half a
// warp each for the even and the odd keys).
template <class C>
struct FmaMath : Base<C> {
  using Base<C>::p;
  using Base<C>::sh;
  using Base<C>::smem;
  using Base<C>::sbase;
  using Base<C>::lane;
  using Base<C>::warp;
  using Base<C>::sync_warps;
  using Base<C>::heads_of;
  using Base<C>::first_head;
  static constexpr int N = C::kFma;
  static constexpr int kAlike = 128 / C::D;  // keys at a time
  const int chunk = lane % (C::D / 4), odd = lane / (C::D / 4);

  float m[N], l[N];     // l: this lane's share
  uint64_t o[N][2];     // dims 4 chunk + {0, 1}, {2, 3}
  using Base<C>::Base;

  __device__ __forceinline__ float* merge_buffer() const {
    return reinterpret_cast<float*>(smem + C::S * C::kStage);
  }
  // This warp's queries.
  __device__ __forceinline__ float* queries() const {
    return merge_buffer() + (C::NW - 1 + warp) * N * C::D;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int g = 0; g < N; ++g) m[g] = -INFINITY, l[g] = 0.0f, o[g][0] = o[g][1] = 0;
  }
  __device__ void begin_item(const Note& w) {
    clear();
    const int n = heads_of(w);
    const float* src = reinterpret_cast<const float*>(p.q) + w.b * p.q_sb + first_head(w) * p.q_sh;
    for (int i = lane; i < N * (C::D / 4); i += 32) {
      const int g = i / (C::D / 4), d = i % (C::D / 4) * 4;
      float4 x = make_float4(0, 0, 0, 0);
      if (g < n && d < p.D) x = *reinterpret_cast<const float4*>(src + g * p.q_sh + d);
      *reinterpret_cast<float4*>(queries() + g * C::D + d) = x;
    }
    __syncwarp();
  }

  __device__ __forceinline__ void raise(const float (&mx)[N]) {
#pragma unroll
    for (int g = 0; g < N; ++g)
      if (mx[g] > m[g]) {  // alike in all lanes
        const float f = fast_exp2(m[g] - mx[g]);
        const uint64_t ff = f2_pack(f, f);
        m[g] = mx[g];
        l[g] *= f;
        o[g][0] = f2_mul(o[g][0], ff), o[g][1] = f2_mul(o[g][1], ff);
      }
  }

  __device__ __forceinline__ void tile(const Note& w, int stage) {
    const uint32_t kbase = sbase + stage * C::kStage, vbase = kbase + C::kTile;
    const int key = warp * 16 + lane / 2;
    const uint32_t qbase = smem_u32(queries());
    uint64_t acc[N][2];
#pragma unroll
    for (int g = 0; g < N; ++g) acc[g][0] = acc[g][1] = 0;
#pragma unroll
    for (int i = 0; i < C::D / 8; ++i) {
      const int c = 2 * i + lane % 2;  // (other halves would share banks)
      uint64_t k0, k1;
      lds2x2(kbase + place<C>(key, c), k0, k1);
#pragma unroll
      for (int g = 0; g < N; ++g) {
        uint64_t q0, q1;
        lds2x2(qbase + (g * C::D + c * 4) * 4, q0, q1);
        acc[g][0] = f2_fma(k0, q0, acc[g][0]);
        acc[g][1] = f2_fma(k1, q1, acc[g][1]);
      }
    }
    const bool ok = w.ok[C::NP > 1 ? warp / 2 : 0] >> (key & 31) & 1;
    const int n = heads_of(w), h0 = first_head(w);
    float s[N], mx[N];
#pragma unroll
    for (int g = 0; g < N; ++g) {
      float a, b;
      f2_unpack(f2_add(acc[g][0], acc[g][1]), a, b);
      s[g] = a + b;
      s[g] += __shfl_xor_sync(0xffffffffu, s[g], 1);
      s[g] *= p.scale * kLog2e;
      if (p.alibi && g < n) {
        const int idx = w.t * C::kKeys + key;
        const int j = idx < w.n_sink ? idx : idx + w.gap;
        s[g] -= p.alibi[h0 + g] * kLog2e * (float)(w.L - 1 - j);
      }
      if (!ok) s[g] = -INFINITY;
      mx[g] = s[g];
#pragma unroll
      for (int off = 2; off < 32; off <<= 1)
        mx[g] = fmaxf(mx[g], __shfl_xor_sync(0xffffffffu, mx[g], off));
    }
    raise(mx);
#pragma unroll
    for (int g = 0; g < N; ++g) {
      s[g] = fast_exp2(s[g] - (m[g] > -INFINITY ? m[g] : 0.0f));  // no visible key yet
      if (lane % 2 == 0) l[g] += s[g];
      acc[g][0] = acc[g][1] = 0;
    }
    // A tile's sum by itself, then one addition to the running one.
#pragma unroll
    for (int i = 0; i < 16 / kAlike; ++i) {
      const int at = i * kAlike + odd;
      uint64_t v0, v1;
      lds2x2(vbase + place<C>(warp * 16 + at, chunk), v0, v1);
#pragma unroll
      for (int g = 0; g < N; ++g) {
        const float x = __shfl_sync(0xffffffffu, s[g], at * 2);
        const uint64_t xx = f2_pack(x, x);
        acc[g][0] = f2_fma(v0, xx, acc[g][0]);
        acc[g][1] = f2_fma(v1, xx, acc[g][1]);
      }
    }
#pragma unroll
    for (int g = 0; g < N; ++g)
#pragma unroll
      for (int i = 0; i < 2; ++i) o[g][i] = f2_add(o[g][i], acc[g][i]);
  }

  // Even and odd keys together, in both.
  __device__ __forceinline__ void fold() {
    if constexpr (kAlike > 1) {
#pragma unroll
      for (int g = 0; g < N; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          o[g][i] = f2_add(o[g][i], __shfl_xor_sync(0xffffffffu, o[g][i], 16));
    }
  }

  // As MmaMath's.
  __device__ void join_warps(int n) {
    float* buf = merge_buffer();
    if (warp < n) {
#pragma unroll
      for (int g = 0; g < N; ++g) {
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], off);
        if (lane == 0) sh.m[warp][g] = m[g], sh.l[warp][g] = l[g];
      }
    }
    if (n == 1) return;
    sync_warps();
    if (warp < n) {
      float top[N];
#pragma unroll
      for (int g = 0; g < N; ++g) {
        top[g] = m[g];
        for (int w = 0; w < n; ++w) top[g] = fmaxf(top[g], sh.m[w][g]);
      }
      raise(top);
      if (warp == 0) {
#pragma unroll
        for (int g = 0; g < N; ++g)
          for (int w = 1; w < n; ++w)
            if (sh.m[w][g] > -INFINITY) l[g] += sh.l[w][g] * fast_exp2(sh.m[w][g] - m[g]);
      } else if (odd == 0) {
#pragma unroll
        for (int g = 0; g < N; ++g)
          *reinterpret_cast<ulonglong2*>(buf + ((warp - 1) * N + g) * C::D + chunk * 4) =
              make_ulonglong2(o[g][0], o[g][1]);
      }
    }
    sync_warps();
    if (warp == 0) {
      for (int w = 0; w < n - 1; ++w)
#pragma unroll
        for (int g = 0; g < N; ++g) {
          const ulonglong2 x =
              *reinterpret_cast<const ulonglong2*>(buf + (w * N + g) * C::D + chunk * 4);
          o[g][0] = f2_add(o[g][0], x.x), o[g][1] = f2_add(o[g][1], x.y);
        }
    }
  }

  __device__ void write_output(const Note& w) const {  // warp 0
    const int n = heads_of(w);
#pragma unroll
    for (int g = 0; g < N; ++g) {
      if (g >= n) break;
      const int head = first_head(w) + g;
      const float inv = l[g] > 0.0f ? 1.0f / l[g] : l[g] == 0.0f ? 0.0f : l[g];
      const long long e = w.b * p.o_sb + head * p.o_sh + chunk * 4;
      if (odd == 0 && chunk * 4 < p.D) {
        float x[4];
        f2_unpack(o[g][0], x[0], x[1]);
        f2_unpack(o[g][1], x[2], x[3]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p.out_fp32)
            reinterpret_cast<float*>(p.o)[e + i] = x[i] * inv;
          else
            reinterpret_cast<__nv_bfloat16*>(p.o)[e + i] = __float2bfloat16_rn(x[i] * inv);
        }
      }
      if (lane == 0 && p.lse)
        p.lse[(long long)w.b * p.H + head] =
            l[g] == 0.0f ? -INFINITY : (m[g] + log2f(l[g])) * kLn2;
    }
  }

  __device__ void write_part(float* part) const {  // warp 0
#pragma unroll
    for (int g = 0; g < N; ++g) {
      if (odd == 0)
        *reinterpret_cast<ulonglong2*>(part + g * C::D + chunk * 4) =
            make_ulonglong2(o[g][0], o[g][1]);
      if (lane == 0) part[N * C::D + 2 * g] = m[g], part[N * C::D + 2 * g + 1] = l[g];
    }
  }
  // Adds a part to the state (its sums count in lane 0 only).
  __device__ void add_part(const float* part) {
    float pm[N], pl[N];
    ulonglong2 po[N];
#pragma unroll
    for (int g = 0; g < N; ++g) {
      pm[g] = __ldcg(part + N * C::D + 2 * g);
      pl[g] = __ldcg(part + N * C::D + 2 * g + 1);
      po[g] = __ldcg(reinterpret_cast<const ulonglong2*>(part + g * C::D + chunk * 4));
    }
    raise(pm);
#pragma unroll
    for (int g = 0; g < N; ++g) {
      const float f = pm[g] > -INFINITY ? fast_exp2(pm[g] - m[g]) : 0.0f;
      const uint64_t ff = f2_pack(f, f);
      if (lane == 0) l[g] += pl[g] * f;
      o[g][0] = f2_fma(po[g].x, ff, o[g][0]);
      o[g][1] = f2_fma(po[g].y, ff, o[g][1]);
    }
  }
};

template <class C>
struct Decoder : std::conditional_t<(C::kFma > 0), FmaMath<C>, MmaMath<C>> {
  using Math = std::conditional_t<(C::kFma > 0), FmaMath<C>, MmaMath<C>>;
  using Base<C>::p;
  using Base<C>::sh;
  using Base<C>::smem;
  using Base<C>::sbase;
  using Base<C>::lane;
  using Base<C>::warp;
  using Base<C>::sync_warps;
  using Base<C>::heads_of;
  using Base<C>::first_head;
  using Base<C>::HB;
  using Base<C>::SUB;
  using Math::begin_item;
  using Math::tile;
  using Math::clear;
  using Math::fold;
  using Math::join_warps;
  using Math::write_output;
  using Math::write_part;
  using Math::add_part;
  using Math::Math;
  int lens_b = 0;

  __device__ int read_length(int b) const {
    int L = p.lens[b];
    const long long most = (long long)p.max_pages * p.page_size;
    if (L > most) L = (int)most;
    return max(L, 0);
  }
  __device__ int length(int b) const {
    const int at = b - lens_b;
    return at >= 0 && at < kLens ? sh.lens[at] : read_length(b);
  }
  __device__ __forceinline__ int tiles_of(int n) const {  // (n is up to 2^31 - 1)
    return n / C::kKeys + (n % C::kKeys > 0);
  }

  // ------------------------------------------------------- loading warps
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

  // A key's row in the pools: the page number as read (whose latency passes
  // while the tile before is loaded), then the address.
  struct Key {
    int page, slot;  // slot < 0: past the end
  };
  __device__ __forceinline__ Key find_key(const Walker& w, int key) const {
    Key k{0, -1};
    const uint32_t i = (uint32_t)w.t * C::kKeys + key;  // past 2^31 in the last tile
    if (i < (uint32_t)w.vis.n) {
      const int j = (int)i < w.vis.n_sink ? (int)i : (int)i + w.vis.gap;
      const int col = j / p.page_size;
      k.slot = j - col * p.page_size;
      k.page = p.table[w.b * p.t_sb + col];
    }
    return k;
  }

  __device__ void load_run(const Walker& start, int n) {
    constexpr int kChunks = C::kRow / 16, kRows = 32 / kChunks;  // rows a pass
    const int pw = warp - C::NW;
    const int chunk = lane % kChunks, sub_row = lane / kChunks;
    const bool real = chunk * 16 < p.D * C::kEsz;
    const uint8_t* kb = reinterpret_cast<const uint8_t*>(p.k) + chunk * 16;
    const uint8_t* vb = reinterpret_cast<const uint8_t*>(p.v) + chunk * 16;
    Walker w = start;
    Key next = find_key(w, pw * 32 + lane);
    for (int i = 0; i < n; ++i) {
      const Walker now = w;
      const Key key = next;
      if (i + 1 < n) {
        advance(w);
        next = find_key(w, pw * 32 + lane);
      }
      const int stage = i % C::S;
      if (i >= C::S) mbar_wait(&sh.empty[stage], (i / C::S - 1) & 1, &sh.abort, kSite);
      // Byte offset of this lane's key, or -1 for none or a page outside the
      // pool (which counts as masked).
      long long off = -1;
      if (key.slot >= 0) {
        if (key.page < 0 || key.page >= p.n_pages)
          report_error(kDevBadIndex, now.b);
        else
          off = (key.page * p.p_sp + (now.sub / HB) * p.p_sh + key.slot * p.p_ss) * C::kEsz;
      }
      const uint32_t ok = __ballot_sync(0xffffffffu, off >= 0);
      const int n_keys = min(C::kKeys, now.vis.n - now.t * C::kKeys);
      const uint32_t dst = sbase + stage * C::kStage;
      // Rows of warps without keys stay as they are: those skip the tile.
      const int passes = min(32, (n_keys + 15) / 16 * 16 - pw * 32) / kRows;
#pragma unroll 4
      for (int s = 0; s < passes; ++s) {
        const int row = s * kRows + sub_row;
        const long long o = __shfl_sync(0xffffffffu, off, row);
        const int bytes = real && o >= 0 ? 16 : 0;
        const long long e = bytes ? o : -chunk * 16;
        const uint32_t at = dst + place<C>(pw * 32 + row, chunk);
        cp_async16(at, kb + e, bytes);
        cp_async16(at + C::kTile, vb + e, bytes);
      }
      cp_arrive(&sh.full[stage]);
      if (lane == 0) {
        Note& note = sh.note[stage];
        note.ok[pw] = ok;
        if (pw == 0) {
          note.b = now.b, note.sub = now.sub, note.t = now.t, note.nt = now.nt;
          note.L = now.L, note.n_sink = now.vis.n_sink, note.gap = now.vis.gap;
          note.n_keys = n_keys;
        }
        mbar_arrive(&sh.full[stage]);
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  }

  __device__ __forceinline__ float* slot_of(long long cta, int which) const {
    return reinterpret_cast<float*>(p.workspace) + (cta * 2 + which) * C::kSlot;
  }
  // How the tiles are shared out: block c of n takes tiles [c T / n, (c + 1) T / n);
  // this one's run starts at `first`. Whole: runs of whole items instead.
  struct Share {
    long long first, T, n;
    bool whole;

    // x / y of values whose product fits: 32-bit where possible, since parts are
    // joined by few threads at the end of a call.
    static __device__ __forceinline__ long long quot(long long x, long long y) {
      return x >> 32 ? x / y : (long long)((uint32_t)x / (uint32_t)y);
    }
    __device__ __forceinline__ long long begin(long long c) const { return quot(c * T, n); }
    __device__ __forceinline__ long long block_of(long long t) const {
      return quot((t + 1) * n - 1, T);
    }
  };

  // The note's item ends with this tile, or the block's run does. g: the tile's
  // number among all.
  __device__ void end_segment(const Note& w, long long g, const Share& share) {
    fold();
    // A segment of one tile may leave warps without keys.
    join_warps(w.t > 0 && g > share.first ? C::NW : min(C::NW, (w.n_keys + 15) / 16));
    const long long a = g - w.t, z = a + w.nt;  // the item's tiles
    if (share.whole || (share.first <= a && g == z - 1)) {
      if (warp == 0) write_output(w);
      return;
    }
    const long long c0 = share.block_of(a), c1 = share.block_of(z - 1);
    int* count = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(p.workspace) +
                                        p.n_sms * kPartBytesPerSm) + (w.b * SUB + w.sub);
    if (warp == 0) {
      write_part(slot_of(blockIdx.x, share.first >= a ? 0 : 1));
      __threadfence();
      __syncwarp();
      if (lane == 0) {
        const bool last = atomicAdd(count, 1) == (int)(c1 - c0);
        if (last) *count = 0;  // for the next call
        __threadfence();
        sh.last = last;
      }
    }
    sync_warps();
    if (!sh.last) {
      sync_warps();  // read by all before the next one is written
      return;
    }
    // The warps share the parts, each in ascending order.
    clear();
    for (long long c = c0 + warp; c <= c1; c += C::NW)
      add_part(slot_of(c, share.begin(c) >= a ? 0 : 1));
    join_warps((int)min((long long)C::NW, c1 - c0 + 1));
    if (warp == 0) write_output(w);
  }

  __device__ void compute_run(const Share& share, int n) {
    for (int i = 0; i < n; ++i) {
      const int stage = i % C::S;
      mbar_wait(&sh.full[stage], (i / C::S) & 1, &sh.abort, kSite + 1);
      const Note w = sh.note[stage];
      if (i == 0 || w.t == 0) begin_item(w);
      if (warp * 16 < w.n_keys) tile(w, stage);
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[stage]);
      if (w.t == w.nt - 1 || i == n - 1) end_segment(w, share.first + i, share);
    }
  }

  __device__ void run() {
    const int tid = threadIdx.x;
    constexpr int kWarps = C::NW + C::NP;
    if (tid == 0) {
      for (int s = 0; s < C::S; ++s) {
        mbar_init(&sh.full[s], C::NP * 33);  // each loading lane's copies, and its warp's note
        mbar_init(&sh.empty[s], C::NW);
      }
      sh.abort = 0;
      fence_barrier_init();
    }
    // Every sequence's tiles: this thread's stretch of sequences, then a scan.
    const int per = (p.B + C::kThreads - 1) / C::kThreads;
    const int b0 = min(p.B, tid * per), b1 = min(p.B, b0 + per);
    // (tiles, and in the upper half sequences that have some)
    constexpr long long kSeq = 1ll << 40;
    long long mine = 0;
    int longest = 0;
    for (int b = b0; b < b1; ++b) {
      const int L = read_length(b);
      if (b < kLens) sh.lens[b] = L;
      if (blockIdx.x == 0 && p.lens[b] > L) report_error(kDevBadIndex, b);
      const int nt = tiles_of(visible_of(L, p.window, p.sinks).n);
      mine += nt > 0 ? nt + kSeq : 0;
      longest = max(longest, nt);
    }
    long long inc = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, inc, off);
      if (lane >= off) inc += y;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 31) sh.scan[warp] = inc, sh.longest[warp] = longest;
    __syncthreads();
    lens_b = 0;
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += sh.scan[w];
      all += sh.scan[w];
      longest = max(longest, sh.longest[w]);
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
    // Units shared out: whole items, or tiles. No more blocks than units take
    // part, so none of those has an empty run.
    Share share;
    const long long items = (all >> 40) * SUB;
    share.whole = longest <= kWholeTiles && items <= 16ll * gridDim.x;
    auto units = [&](long long x) { return (share.whole ? x >> 40 : x & (kSeq - 1)) * SUB; };
    share.T = units(all);
    share.n = min((long long)gridDim.x, share.T);
    if (blockIdx.x >= share.n) return;
    const long long first = share.begin(blockIdx.x), end = share.begin(blockIdx.x + 1ll);
    share.first = share.whole ? 0 : first;
    // The sequence that holds the run's first unit.
    if (units(before) <= first && first < units(before + mine)) {
      long long run = units(before);
      int b = b0;
      for (;; ++b) {
        const int nt = tiles_of(visible_of(length(b), p.window, p.sinks).n);
        const long long u = (long long)(share.whole ? min(nt, 1) : nt) * SUB;
        if (first < run + u) break;
        run += u;
      }
      sh.b = b;
      sh.rest = first - run;
    }
    __syncthreads();
    if (p.B > kLens) {  // keep the lengths that this run meets first
      const int b = sh.b;
      for (int i = tid; i < kLens && b + i < p.B; i += C::kThreads)
        sh.lens[i] = read_length(b + i);
      lens_b = b;
      __syncthreads();
    }
    Walker w;
    enter(w, sh.b);
    w.sub = (int)(share.whole ? sh.rest : sh.rest / w.nt);
    w.t = share.whole ? 0 : (int)(sh.rest % w.nt);
    int n = (int)(end - first);  // tiles of the run
    if (share.whole) {
      Walker x = w;
      int tiles = 0;
      for (int i = 0; i < n; ++i) {
        tiles += x.nt;
        x.t = x.nt - 1;
        advance(x);
      }
      n = tiles;
    }
    if (warp >= C::NW)
      load_run(w, n);
    else
      compute_run(share, n);
  }
};

template <class C>
__global__ void __launch_bounds__(C::kThreads, C::kPerSm) paged_kernel(const PagedDecodeParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Block sh;
  Decoder<C> d(p, sh, smem);
  d.run();
}

template <class C>
cudaError_t launch(const PagedDecodeParams& p, cudaStream_t stream) {
  static_assert(C::kPerSm * 2 * C::kSlot * 4 <= kPartBytesPerSm, "parts fit the workspace");
  static_assert(C::kPerSm >= 1 && sizeof(Block) <= C::kStatic && C::S <= 4, "a block fits an SM");
  const int G = p.H / p.Hkv;
  const long long most = std::min<long long>((long long)p.max_pages * p.page_size, 0x7fffffff);
  const long long tiles = (long long)p.B * p.Hkv * ((G + C::kItem - 1) / C::kItem) *
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
  // Warps and stages, measured (us). fp32 on the FMA pipe (16 x 6144 keys,
  // floor 123), 8 kv heads of 128: 2 warps with 2 stages, 3 blocks a SM, 130 for
  // one or two heads a group, 138 for four; 3 stages, 2 blocks 128, 142, 156;
  // 4 warps with 2 stages 147, 148, 169. 16 kv heads of 64: 4 warps with 3 stages,
  // 2 blocks, 129, 127, 136; 2 stages, 3 blocks 132, 131, 139; 2 warps with 4
  // stages 128, 138, and 24 against 15 for one sequence of 5000. On the tensor pipe
  // any group of fp32 heads takes 186 (128 dims) or 155 (64).
  // bf16, heads of 128 (64 x 6144 keys, floor 246): 4 warps with 3 stages, 2 blocks,
  // 244; with 2 stages, 3 blocks 259.
  const int group = p.H / p.Hkv;
  const bool wide = group > 8;  // more than one column tile
  if (p.in_fp32) {
    if (p.D > 64)
      return group == 1   ? launch<Cfg<128, true, 1, 2, 2, 1>>(p, stream)
             : group == 2 ? launch<Cfg<128, true, 1, 2, 2, 2>>(p, stream)
             : group <= 4 ? launch<Cfg<128, true, 1, 2, 2, 4>>(p, stream)
                          : launch<Cfg<128, true, 1, 2, 2>>(p, stream);
    return group == 1   ? launch<Cfg<64, true, 1, 4, 3, 1>>(p, stream)
           : group == 2 ? launch<Cfg<64, true, 1, 4, 3, 2>>(p, stream)
           : group <= 4 ? launch<Cfg<64, true, 1, 4, 3, 4>>(p, stream)
                        : launch<Cfg<64, true, 1, 2, 3>>(p, stream);
  }
  if (p.D > 64)
    return wide ? launch<Cfg<128, false, 2, 4, 3>>(p, stream)
                : launch<Cfg<128, false, 1, 4, 3>>(p, stream);
  return wide ? launch<Cfg<64, false, 2, 4, 4>>(p, stream)
              : launch<Cfg<64, false, 1, 4, 4>>(p, stream);
}

}  // namespace enl
