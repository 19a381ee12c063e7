// One token per row of logits: temperature, top-k, top-p and min-p, drawn with
// a given uniform number by inverting the running sum of the kept weights.
//
//   w_i = exp((l_i - max) / T),  q_i = floor(w_i 2^40)
//
// Sums are sums of the whole numbers q_i, so they are exact whatever the order
// of addition: a row's token does not depend on how its work was shared out.
// Sorted by (l descending, i ascending), the kept tokens are a leading run,
// i.e. they are the tokens at or above one 64-bit composite of the logit's
// order-preserving bits and the complement of the index.
//
// A row belongs to one block, or to a cluster of 2 to 8 when there are fewer rows
// than SMs (choose_cluster). The first pass streams the row from HBM and keeps
// only extremes: the row's and, per thread, the maxima of four parts of what it
// read (2048 groups a block). What follows reads the row again from L2, and only
// where it has to:
//  * top-k up to kSmallK: the k-th largest group maximum bounds the k-th largest
//    logit from below, so only groups at or above it (about k of them) are read
//    again. Their few candidates go to one list in shared memory, where they
//    are ranked, and the rest of the row is never touched.
//  * min-p alone: the same with the groups whose maximum weighs min_p or more.
//  * top-p alone: the groups whose maxima carry the wanted share of a total
//    estimated from the maxima and one vector a thread, one more pass for the
//    exact total, and the same list, provided that it carries the exact share.
//  * larger top-k, flatter nuclei: a histogram of a quarter of the logits guesses
//    the bins around the cut (16 us a row of 131072; one of all the logits would
//    cost more than the wrong guesses do); one pass (34 us) sums what lies above
//    them, and the total where it is not known, and lists their
//    tokens. The exact sums confirm the guess or correct it for another pass.
//    The cut and the draw follow from the list and the warps' sums.
//  * rows that defeat the bins (thousands of equal logits at the cut): bisection
//    over the composite, one pass per bit.
// With temperature alone one pass sums the row in ranges and the range that
// holds the draw is walked again.
#include <cstdint>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace smp {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = 4;       // group maxima per thread
constexpr int kCap = 2048;       // candidates that fit the list
constexpr int kSmallK = 1024;    // largest top-k of the group path
constexpr int kNucleus = 1200;   // most groups that a top-p list is made of
constexpr int kRank = 256;       // entries that are ranked by counting
constexpr int kMaxCluster = 8;
constexpr int kGroupBins = 256;  // bins over the group maxima
constexpr int kBins = 2048;      // bins over the row
constexpr int kTries = 16;       // passes with guessed bins (the last halve what is left)
// One vector in kSample goes into the histogram, kWindow tokens are listed to
// each side of a guessed cut. Measured (256 flat rows of 131072, top-p 0.9 and
// 0.99, us): 4 and 650: 159, 179; 4 and 500: 168, 153; 4 and 780: 212, 214 (lists
// that overflow); 2 and 650: 172, 179.
constexpr int kSample = 4;
constexpr int kWindow = 650;
// Tokens above e^-kHeavy are weighed one by one in the histogram, lighter ones by
// their bin's centre: the second atomic costs more than it tells (one flat row's
// histogram: 4: 16 us, 7: 22 us, 7 with float atomics: 30 us). In
// whole units of 2^-13; rows so long that they overflow only guess worse.
constexpr float kHeavy = 4.0f;
constexpr float kOne = 1099511627776.0f;  // 2^40
constexpr uint32_t kNoCut = ~0u;  // in place of a top-p share
constexpr float kLive = 28.0f;   // weights below exp(-28) < 2^-40 are zero

// Order-preserving bits of a float: a < b as floats iff key(a) < key(b).
__device__ __forceinline__ uint32_t key_of(float f) {
  const uint32_t u = __float_as_uint(f == 0.0f ? 0.0f : f);  // one zero
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ u64 composite(float x, int i) {
  return ((u64)key_of(x) << 32) | (uint32_t)~i;
}

// Weight of a logit; expf and the single multiply are the operator's
// definition of w (no fast approximation), so the whole numbers are reproducible.
__device__ __forceinline__ float weight_of(float x, float top, float inv_t) {
  return x == top ? 1.0f : expf((x - top) * inv_t);
}
__device__ __forceinline__ u64 whole_of(float w) { return (u64)(w * kOne); }

// floor(total * part / 2^24), part <= 2^24.
__device__ __forceinline__ u64 share_of(u64 total, uint32_t part) {
  return (total >> 24) * part + (((total & 0xffffffu) * part) >> 24);
}

// Sum of whole weights over a stretch of at most 2048 tokens without 64-bit or
// conversion instructions per token: floor(w 2^20) and the floor of 2^20 times
// the exact remainder, each read off the low bits of a float in [2^23, 2^24).
struct WholeSum {
  uint32_t hi = 0, lo = 0;
  int n = 0;
  __device__ __forceinline__ void add(float w) {
    const float a = __fmaf_rd(w, 1048576.0f, 8388608.0f);
    const float r = __fmaf_rn(w, 1048576.0f, 8388608.0f - a);
    const float b = __fmaf_rd(r, 1048576.0f, 8388608.0f);
    hi += __float_as_uint(a);
    lo += __float_as_uint(b);
    ++n;
  }
  __device__ __forceinline__ static WholeSum of(float w) {
    WholeSum s;
    s.add(w);
    return s;
  }
  __device__ __forceinline__ void operator+=(const WholeSum& s) {
    hi += s.hi, lo += s.lo, n += s.n;
  }
  __device__ __forceinline__ u64 total() const {
    const uint32_t off = (uint32_t)n * 0x4B000000u;
    return ((u64)(hi - off) << 20) + (lo - off);
  }
};

// One 16-byte load of logits, kept packed until they are used.
template <bool kF32>
struct Vec {
  static constexpr int E = kF32 ? 4 : 8;
  uint32_t w[4];

  __device__ __forceinline__ float at(int e) const {  // e is a constant after unrolling
    if constexpr (kF32) return __uint_as_float(w[e]);
    return e % 2 ? bf16hi_to_f32(w[e / 2]) : bf16lo_to_f32(w[e / 2]);
  }
  __device__ __forceinline__ float pick(int e) const {  // any e, by selection
    const int i = kF32 ? e : e >> 1;
    const uint32_t lo = i & 1 ? w[1] : w[0], hi = i & 1 ? w[3] : w[2];
    const uint32_t v = i & 2 ? hi : lo;
    if constexpr (kF32) return __uint_as_float(v);
    return e & 1 ? bf16hi_to_f32(v) : bf16lo_to_f32(v);
  }
};

// Running maximum of a group's vectors, and (in `row`) the smallest logit of
// all of them; NaN is dropped. bf16 stays packed.
template <bool kF32>
struct Extremes {
  float f = -INFINITY, g = INFINITY;
  __nv_bfloat162 h = __float2bfloat162_rn(-INFINITY), l = __float2bfloat162_rn(INFINITY);

  __device__ __forceinline__ void add(const Vec<kF32>& x, Extremes& row) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kF32) {
        f = fmaxf(f, __uint_as_float(x.w[i]));
        row.g = fminf(row.g, __uint_as_float(x.w[i]));
      } else {
        const __nv_bfloat162 v = *reinterpret_cast<const __nv_bfloat162*>(&x.w[i]);
        h = __hmax2(h, v);
        row.l = __hmin2(row.l, v);
      }
    }
  }
  __device__ __forceinline__ float max() const {
    return kF32 ? f : fmaxf(__low2float(h), __high2float(h));
  }
  __device__ __forceinline__ float min() const {
    return kF32 ? g : fminf(__low2float(l), __high2float(l));
  }
};

// The row as 16-byte vectors counted from the aligned address at or below its
// start: vector j holds indices j E - mis .. j E - mis + E - 1.
template <bool kF32>
struct Row {
  static constexpr int E = Vec<kF32>::E;
  const uint8_t* base;  // aligned address of vector 0
  int V, mis, n_vec;

  __device__ __forceinline__ Row(const void* p, int V_) : V(V_) {
    const uintptr_t u = reinterpret_cast<uintptr_t>(p);
    base = reinterpret_cast<const uint8_t*>(u & ~uintptr_t(15));
    mis = (int)(u & 15) / (kF32 ? 4 : 2);
    n_vec = (mis + V + E - 1) / E;
  }
  __device__ __forceinline__ bool inside(int j) const {
    return j * E >= mis && (j + 1) * E - mis <= V;
  }
  __device__ __forceinline__ float one(int i) const {  // logit i of the row
    if constexpr (kF32)
      return reinterpret_cast<const float*>(base)[mis + i];
    else
      return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[mis + i]);
  }
  __device__ __forceinline__ float logit_or_nan(int i) const {
    return i >= 0 && i < V ? one(i) : __uint_as_float(0x7fff0000u);
  }
  // Vector j; indices outside the row read as NaN, which counts nowhere (and
  // touch no memory).
  __device__ __forceinline__ Vec<kF32> get(int j) const {
    Vec<kF32> r;
    if (inside(j)) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + (size_t)j * 16);
      r.w[0] = w.x, r.w[1] = w.y, r.w[2] = w.z, r.w[3] = w.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kF32) {
          r.w[e] = __float_as_uint(logit_or_nan(j * E - mis + e));
        } else {
          r.w[e] = __float_as_uint(logit_or_nan(j * E - mis + 2 * e)) >> 16 |
                   __float_as_uint(logit_or_nan(j * E - mis + 2 * e + 1));
        }
      }
    }
    return r;
  }
};

// A composite list entry's token, and its logit's bits.
__device__ __forceinline__ uint32_t index_of(u64 comp) { return ~(uint32_t)comp; }

struct Pair {
  u64 a, b;
};
struct Sums {
  u64 above, all;
  uint32_t count;
};

// What a block knows about its row, for the paths that are functions of their
// own: inlined they would take the common path's registers.
struct Case {
  const void* row;
  int V, n_blocks, turn;
  uint32_t rank;
  float top, inv_t, min_p, least, u;
  long long* token;
};

struct Shared {
  union {
    u64 list[kCap];  // candidates (composites)
    struct {
      uint32_t bins[kBins];   // histogram: tokens, and the
      uint32_t heavy[kBins];  // weight of those that are weighed one by one, in 2^-13
    };
  };
  float cum_n[kBins], cum_m[kBins];  // guessed tokens and weight before each bin
  u64 q[kRank];           // whole weights of entries that are ranked
  u64 mass[kGroupBins];   // of the entries in select()'s bins
  u64 part[kWarps];
  u64 wsum[kWarps * kMaxCluster];  // rank 0: kept weight of every warp's range
  float fpart[kWarps];
  // Warps' shares of the estimated total: not in `part`, whose extremes slower
  // warps of a lone block may still be reading.
  u64 est[kWarps];
  Pair swap[2][kMaxCluster];  // what the cluster's blocks tell each other
  uint32_t gbins[kGroupBins], gmass[kGroupBins];  // groups, and their maxima's weight
  union {
    int groups[kThreads * kGroups];  // first vectors of the groups to read again
    u64 few[kRank];                  // entries that select() ranks
  };
  u64 cut, rest;  // composite and draw found by rank 0
  Case row;
  int count, found, n_groups, pick;
};

// ------------------------------------------------------- block and cluster
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Shared-memory address of `p` in block `rank` of the cluster.
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void remote_store(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void remote_store32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ u64 remote_load64(uint32_t addr) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t remote_load(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ u64 warp_sum(u64 x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

__device__ u64 block_sum(u64 x, Shared& sm) {
  x = warp_sum(x);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sm.part[threadIdx.x / 32] = x;
  __syncthreads();
  x = threadIdx.x % 32 < kWarps ? sm.part[threadIdx.x % 32] : 0;
  return warp_sum(x);
}

// Sum over the threads before this one; `total` gets the block's.
__device__ u64 block_scan(u64 x, u64& total, Shared& sm) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  u64 inc = x;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, inc, off);
    if (lane >= off) inc += y;
  }
  __syncthreads();
  if (lane == 31) sm.part[warp] = inc;
  __syncthreads();
  u64 before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const u64 y = sm.part[w];
    if (w < warp) before += y;
    all += y;
  }
  total = all;
  return before + inc - x;
}

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

__device__ __forceinline__ uint32_t draw_part(float u) {
  return (uint32_t)(fminf(fmaxf(u, 0.0f), 0.99999994f) * 16777216.0f);
}

struct Groups {  // maxima of a thread's groups
  float m[kGroups];
};
template <bool kF32>
__device__ __noinline__ void draw_by_bins(Shared& sm, Groups gm, int k, uint32_t part, u64 total);
template <bool kF32>
__device__ __noinline__ Sums split_row(Shared& sm, float hi, float lo, float least, bool weigh,
                                       bool all);
template <bool kF32>
__device__ __noinline__ void draw_by_weight(Shared& sm, Groups gm, u64 C);
template <bool kF32>
__device__ __noinline__ void draw_from_row(Shared& sm, u64 C);
template <bool kF32>
__device__ __noinline__ void draw_long_list(Shared& sm, int n, u64 C, int n_k, bool use_p, u64 bound,
                                            uint32_t part);

// ------------------------------------------------------------------- sampler
template <bool kF32>
struct Sampler {
  static constexpr int E = Vec<kF32>::E;
  Row<kF32> row;
  Shared& sm;
  const int n_blocks;   // of the cluster
  const uint32_t rank;  // of this block
  int turn = 0;         // exchanges so far
  float top = 0.0f, inv_t = 1.0f, min_p = 0.0f;
  int per_warp;   // vectors of a warp's contiguous range, a multiple of 32
  int per_group;  // steps of 32 vectors of a group (the last may have fewer)
  Groups gm;      // maxima of this thread's groups

  __device__ Sampler(const void* p, int V, Shared& s, int blocks, uint32_t r)
      : row(p, V), sm(s), n_blocks(blocks), rank(r) {
    const int ranges = blocks * kWarps * 32;
    per_warp = (row.n_vec + ranges - 1) / ranges * 32;
    per_group = (per_warp / 32 + kGroups - 1) / kGroups;
  }
  // The block's row again, in another function.
  __device__ explicit Sampler(Shared& s) : Sampler(s.row.row, s.row.V, s, s.row.n_blocks, s.row.rank) {
    turn = s.row.turn;
    top = s.row.top, inv_t = s.row.inv_t, min_p = s.row.min_p;
  }
  // ... for which this leaves it (every thread calls it, after its last
  // exchange here).
  __device__ void leave(const void* p, float least, float u, long long* token) const {
    if (threadIdx.x == 0)
      sm.row = Case{p, row.V, n_blocks, turn, rank, top, inv_t, min_p, least, u, token};
    __syncthreads();
  }
  __device__ __forceinline__ int warp_begin() const {
    return ((int)rank * kWarps + threadIdx.x / 32) * per_warp;
  }
  __device__ __forceinline__ int first_vec() const { return warp_begin() + threadIdx.x % 32; }
  __device__ __forceinline__ int end_vec() const { return min(row.n_vec, warp_begin() + per_warp); }
  __device__ __forceinline__ int group_first(int g) const { return first_vec() + 32 * per_group * g; }
  __device__ __forceinline__ float weight(float x) const { return weight_of(x, top, inv_t); }
  __device__ __forceinline__ float logit_of(u64 comp) const { return of_key((uint32_t)(comp >> 32)); }
  __device__ __forceinline__ u64 whole(u64 comp) const { return whole_of(weight(logit_of(comp))); }
  // Logits below this have no weight.
  __device__ __forceinline__ float cutoff() const {
    return top == INFINITY ? top : top - kLive / inv_t;
  }

  // A block's shared memory may be reached only once the block runs: each says so
  // at its start and waits for the others before its first access to theirs.
  __device__ __forceinline__ void started() const {
    if (n_blocks > 1) asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory");
  }
  __device__ __forceinline__ void wait_started() const {
    if (n_blocks > 1) asm volatile("barrier.cluster.wait;" ::: "memory");
  }
  // Waits for the cluster's blocks; shared memory written before is visible
  // after, to all of them.
  __device__ __forceinline__ void sync() const {
    if (n_blocks == 1) {
      __syncthreads();
    } else {
      asm volatile("barrier.cluster.arrive.release;\n"
                   "barrier.cluster.wait.acquire;" ::: "memory");
    }
  }
  // Every block's x and y (the same in all its threads), by rank. Two buffers
  // in turn: one is written again only after every block has passed the wait
  // that follows its reading.
  __device__ __forceinline__ const Pair* exchange(u64 x, u64 y) {
    Pair* buf = sm.swap[turn & 1];
    ++turn;
    if (n_blocks == 1) {
      __syncthreads();  // the buffer's last readers are done
      if (threadIdx.x == 0) buf[0] = Pair{x, y};
    } else if (threadIdx.x < n_blocks) {
      const uint32_t a = remote(&buf[rank], threadIdx.x);
      remote_store(a, x);
      remote_store(a + 8, y);
    }
    sync();
    return buf;
  }
  __device__ Pair cluster_sum(u64 x, u64 y) {
    x = block_sum(x, sm);
    y = block_sum(y, sm);
    if (n_blocks == 1) return Pair{x, y};
    const Pair* p = exchange(x, y);
    Pair s{0, 0};
    for (int r = 0; r < n_blocks; ++r) s.a += p[r].a, s.b += p[r].b;
    return s;
  }
  __device__ u64 cluster_sum(u64 x) {
    x = block_sum(x, sm);
    if (n_blocks == 1) return x;
    const Pair* p = exchange(x, 0);
    u64 s = 0;
    for (int r = 0; r < n_blocks; ++r) s += p[r].a;
    return s;
  }

  // f(value, index) for the logits of vectors j, j + 32, ... below end, four
  // loads in flight.
  template <class F>
  __device__ __forceinline__ void each_in(int j, int end, F f) const {
    for (; j < end; j += 128) {
      Vec<kF32> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + 32 * u < end) x[u] = row.get(j + 32 * u);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + 32 * u < end) {
#pragma unroll
          for (int e = 0; e < E; ++e) f(x[u].at(e), (j + 32 * u) * E - row.mis + e);
        }
    }
  }
  // f(vector, its number) likewise, for the vectors from j0 to below end,
  // `apart` apart.
  template <class F>
  __device__ __forceinline__ void each_vec(int j0, int end, int apart, F f) const {
    for (int j = j0; j < end; j += 4 * apart) {
      Vec<kF32> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + apart * u < end) x[u] = row.get(j + apart * u);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (j + apart * u < end) f(x[u], j + apart * u);
    }
  }
  // ... for every logit that this thread reads.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    each_in(first_vec(), end_vec(), f);
  }

  // This thread's sum of the whole weights of its logits.
  __device__ u64 mass() const {
    u64 s = 0;
    const int end = end_vec();
    if (top == INFINITY) {  // only the infinite logits weigh anything, 2^40 each
      each([&](float x, int) { s += x == top ? whole_of(1.0f) : 0; });
      return s;
    }
    for (int j0 = first_vec(); j0 < end; j0 += 32 * 128) {  // at most 1024 logits a stretch
      WholeSum w;
      each_vec(j0, min(end, j0 + 32 * 128), 32, [&](const Vec<kF32>& x, int) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          // NaN and -inf take the bound, whose weight is zero; at the top the
          // argument is zero.
          const float a = fmaxf((x.at(e) - top) * inv_t, -100.0f);
          w.add(expf(a));
        }
      });
      s += w.total();
    }
    return s;
  }

  // Adds the tokens of vector j whose bits are set to the block's list, which
  // may overflow (its count says so).
  __device__ __forceinline__ void push(const Vec<kF32>& x, int j, uint32_t bits) const {
    if (!bits) return;
    int at = atomicAdd(&sm.count, __popc(bits));
    for (; bits && at < kCap; bits &= bits - 1, ++at) {
      const int e = __ffs(bits) - 1;
      sm.list[at] = composite(x.pick(e), j * E - row.mis + e);
    }
  }
  // Empties the lists, before a pass that fills them.
  __device__ __forceinline__ void clear_list() const {
    sync();  // rank 0's has been read
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
  }
  // Brings the blocks' lists together in rank 0's; returns its size (above kCap:
  // too long, nothing was moved).
  __device__ int collect_list() {
    if (n_blocks == 1) {
      __syncthreads();
      return sm.count;
    }
    __syncthreads();
    const int mine = sm.count;
    const Pair* p = exchange((u64)mine, 0);
    u64 total = 0, before = 0;
    for (int r = 0; r < n_blocks; ++r) {
      if (r < (int)rank) before += p[r].a;
      total += p[r].a;
    }
    if (total <= kCap && rank > 0)
      for (int t = threadIdx.x; t < mine; t += kThreads)
        remote_store(remote(&sm.list[before + t], 0), sm.list[t]);
    sync();
    return (int)min(total, (u64)kCap + 1);
  }

  // ------------------------------------------------------ rank 0: the list
  // Draws from the list's n entries at or above C: the first n_k by rank, of those the
  // leading run that reaches `bound` (part of the n_k's total when bound is 0
  // and use_p is set), of those the ones with w >= min_p.
  __device__ void draw_ranked(int n, u64 C, int n_k, bool use_p, u64 bound, uint32_t part, float u,
                              long long* token) const {
    // Threads share each entry's count over the others.
    const int shared = kThreads / max(16, pow2_at_least(n));
    const int i = threadIdx.x / shared, sub = threadIdx.x % shared;
    const bool live = i < n;
    if (threadIdx.x < n) sm.q[threadIdx.x] = whole(sm.list[threadIdx.x]);
    __syncthreads();
    const u64 mine = live ? sm.list[i] : 0;
    const u64 q = live ? sm.q[i] : 0;
    int before_n = 0;
    u64 before = 0;
    for (int j = sub; j < n; j += shared)
      if (sm.list[j] > mine) ++before_n, before += sm.q[j];
    for (int off = shared / 2; off > 0; off >>= 1) {
      before_n += __shfl_xor_sync(0xffffffffu, before_n, off);
      before += __shfl_xor_sync(0xffffffffu, before, off);
    }
    const bool in_k = live && mine >= C && before_n < n_k;
    if (use_p && bound == 0)
      bound = max(share_of(block_sum(in_k && sub == 0 ? q : 0, sm), part), (u64)1);
    const bool keep = in_k && (!use_p || before < bound) && weight(logit_of(mine)) >= min_p;
    __syncthreads();  // the weights have been read
    if (live && sub == 0) sm.q[i] = keep ? q : 0;
    const u64 target = share_of(block_sum(keep && sub == 0 ? q : 0, sm), draw_part(u));
    u64 run = 0;
    for (int j = sub; j < n; j += shared)
      if (index_of(sm.list[j]) < index_of(mine)) run += sm.q[j];
    for (int off = shared / 2; off > 0; off >>= 1) run += __shfl_xor_sync(0xffffffffu, run, off);
    if (keep && sub == 0 && run <= target && target < run + q) *token = index_of(mine);
  }

  enum Order { kCount, kMass, kIndex };

  // The entry of the list (n of them) at which the running sum reaches `need`:
  // of ones or whole weights from the largest composite down, or (kIndex) of
  // those with w >= min_p in index order; only entries at or above C count.
  // Entries are narrowed to one of 256 bins of the order's value at a time, and
  // the last few ranked by counting.
  template <Order kOrder>
  __device__ u64 select(int n, u64 need, u64 C) const {
    const int tid = threadIdx.x;
    auto weight_in = [&](u64 c) -> u64 {
      if (c < C) return 0;
      if constexpr (kOrder == kCount) return 1;
      if (kOrder == kIndex && weight(logit_of(c)) < min_p) return 0;
      return whole(c);
    };
    u64 c[4], q[4];
    int alive = 0;  // bits
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = tid + e * kThreads;
      c[e] = r < n ? sm.list[r] : 0;
      q[e] = r < n ? weight_in(c[e]) : 0;
      if (q[e]) alive |= 1 << e;
    }
    u64 base = 0;  // weight before the entries that are left
    // Bins are even in the distance from the top. Unequal logits can share that
    // distance (1e-9 and 2e-9 are both 1 away from 1), so where all that are left
    // do, bins go by the logits' bits, and where those are equal, by index.
    enum { kValue, kBits, kPlace } by = kOrder == kIndex ? kPlace : kValue;
    auto distance = [&](u64 x) { return top - logit_of(x); };
    auto number = [&](u64 x) { return by == kBits ? ~(uint32_t)(x >> 32) : index_of(x); };
    int left = (int)block_sum(__popc(alive), sm);
    while (left > kRank) {
      float lo = INFINITY, hi = -INFINITY;
      uint32_t first = ~0u, last = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (alive >> e & 1) {
          if (by == kValue)
            lo = fminf(lo, distance(c[e])), hi = fmaxf(hi, distance(c[e]));
          else
            first = min(first, number(c[e])), last = max(last, number(c[e]));
        }
      if (by == kValue) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
          lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        }
      } else {
        first = __reduce_min_sync(0xffffffffu, first);
        last = __reduce_max_sync(0xffffffffu, last);
      }
      __syncthreads();
      if (tid % 32 == 0)
        sm.part[tid / 32] = by == kValue
                                ? ((u64)__float_as_uint(lo) << 32) | __float_as_uint(hi)
                                : ((u64)first << 32) | last;
      if (tid < kGroupBins) sm.mass[tid] = 0;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const uint32_t a = (uint32_t)(sm.part[w] >> 32), b = (uint32_t)sm.part[w];
        if (by == kValue)
          lo = fminf(lo, __uint_as_float(a)), hi = fmaxf(hi, __uint_as_float(b));
        else
          first = min(first, a), last = max(last, b);
      }
      if (by == kValue ? !(hi > lo) : first == last) {  // never by index: those differ
        by = by == kValue ? kBits : kPlace;
        continue;
      }
      const float scale = (float)kGroupBins / fminf(hi - lo, 3.0e38f);
      const u64 span = (u64)(last - first) + 1;
      auto bin_of = [&](u64 x) {
        return by == kValue ? min(kGroupBins - 1, (int)((distance(x) - lo) * scale))
                            : (int)((u64)(number(x) - first) * kGroupBins / span);
      };
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (alive >> e & 1) atomicAdd(&sm.mass[bin_of(c[e])], q[e]);
      __syncthreads();
      u64 all;
      const u64 mine = tid < kGroupBins ? sm.mass[tid] : 0;
      const u64 before = base + block_scan(mine, all, sm);
      if (before < need && need <= before + mine) sm.found = tid, sm.rest = before;
      __syncthreads();
      base = sm.rest;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if ((alive >> e & 1) && bin_of(c[e]) != sm.found) alive &= ~(1 << e);
      left = (int)block_sum(__popc(alive), sm);
    }
    __syncthreads();
    if (tid == 0) sm.found = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (alive >> e & 1) {
        const int at = atomicAdd(&sm.found, 1);
        sm.few[at] = c[e];
        sm.q[at] = q[e];
      }
    __syncthreads();
    const int each_of = kThreads / max(16, pow2_at_least(left));
    const int i = tid / each_of, sub = tid % each_of;
    const bool live = i < left;
    const u64 mine = live ? sm.few[i] : 0;
    u64 before = 0;
    for (int j = sub; j < left; j += each_of) {
      const u64 other = sm.few[j];
      const bool ahead = kOrder == kIndex ? index_of(other) < index_of(mine) : other > mine;
      before += ahead ? sm.q[j] : 0;
    }
    for (int off = each_of / 2; off > 0; off >>= 1)
      before += __shfl_xor_sync(0xffffffffu, before, off);
    before += base;
    if (live && sub == 0 && before < need && need <= before + sm.q[i]) sm.cut = mine;
    __syncthreads();
    return sm.cut;
  }

  // Whole weight of the list's entries at or above C (with w >= min_p where
  // `kept` asks for it).
  __device__ u64 list_mass(int n, u64 C, bool kept) const {
    u64 s = 0;
    for (int r = threadIdx.x; r < n; r += kThreads) {
      const u64 c = sm.list[r];
      if (c >= C && (!kept || weight(logit_of(c)) >= min_p)) s += whole(c);
    }
    return block_sum(s, sm);
  }

  __device__ void long_list(int n, u64 C, int n_k, bool use_p, u64 bound, uint32_t part, float u,
                            long long* token) const {
    if (n_k < n) C = select<kCount>(n, (u64)n_k, C);
    if (use_p) {
      if (bound == 0) bound = max(share_of(list_mass(n, C, false), part), (u64)1);
      C = select<kMass>(n, bound, C);
    }
    const u64 target = share_of(list_mass(n, C, true), draw_part(u));
    const u64 c = select<kIndex>(n, target + 1, C);
    if (threadIdx.x == 0) *token = index_of(c);
  }
  __device__ void draw_from_list(int n, u64 C, int n_k, bool use_p, u64 bound, uint32_t part,
                                 float u, long long* token) const {
    if (n <= kRank)
      draw_ranked(n, C, n_k, use_p, bound, part, u, token);
    else
      draw_long_list<kF32>(sm, n, C, n_k, use_p, bound, part);
  }

  // -------------------------------------------------------- whole-row draws
  // Whole weight of a token if it is kept: at or above C, w >= min_p.
  __device__ __forceinline__ u64 kept_mass(float x, int i, u64 C) const {
    if (!(x > -INFINITY)) return 0;  // NaN too
    const float w = weight(x);
    return w >= min_p && (C == 0 || composite(x, i) >= C) ? whole_of(w) : 0;
  }

  // The draw falls into warp range w of the row, `target` into its kept weight:
  // the range in contiguous pieces, one per thread.
  __device__ void draw_from_range(int w, u64 target, u64 C, long long* token) const {
    const int begin = w * per_warp, end = min(row.n_vec, begin + per_warp);
    const int piece = (per_warp + kThreads - 1) / kThreads;
    const int j0 = begin + threadIdx.x * piece, j1 = min(end, j0 + piece);
    u64 mine = 0, all;
    for (int j = j0; j < j1; ++j) {
      const Vec<kF32> x = row.get(j);
#pragma unroll
      for (int e = 0; e < E; ++e) mine += kept_mass(x.at(e), j * E - row.mis + e, C);
    }
    u64 run = block_scan(mine, all, sm);
    if (run <= target && target < run + mine) {
      for (int j = j0; j < j1; ++j) {
        const Vec<kF32> x = row.get(j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = j * E - row.mis + e;
          const u64 q = kept_mass(x.at(e), i, C);
          if (q && run <= target && target < run + q) *token = i;
          run += q;
        }
      }
    }
  }

  // Draw among the kept tokens by sums of the blocks' and warps' ranges.
  __device__ void by_row(u64 C, float u, long long* token) {
    u64 mine = 0;
    if (C == 0 && min_p <= 0.0f) {
      mine = mass();
    } else {
      const float least = C == 0 ? -INFINITY : logit_of(C);
      each([&](float x, int i) {
        if (x >= least) mine += kept_mass(x, i, C);
      });
    }
    mine = warp_sum(mine);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sm.part[threadIdx.x / 32] = mine;
    __syncthreads();
    u64 ours = 0;
    for (int w = 0; w < kWarps; ++w) ours += sm.part[w];
    const Pair* p = exchange(ours, 0);
    u64 total = 0, before = 0;
    for (int r = 0; r < n_blocks; ++r) {
      if (r < (int)rank) before += p[r].a;
      total += p[r].a;
    }
    const u64 target = share_of(total, draw_part(u));
    if (target < before || target >= before + ours) return;  // another block's
    int w = 0;
    while (w < kWarps - 1 && before + sm.part[w] <= target) before += sm.part[w++];
    draw_from_range((int)rank * kWarps + w, target - before, C, token);
  }

  // Composite of the last token of the smallest leading run of the tokens at
  // or above C that holds `need` tokens, or whole weight `need`.
  __device__ u64 bisect(u64 need, bool count, u64 C) {
    u64 lo = C, hi = composite(top, 0) | 0xffffffffull;
    while (lo < hi) {
      const u64 mid = hi - (hi - lo) / 2;
      u64 s = 0;
      each([&](float x, int i) {
        if (x > -INFINITY && composite(x, i) >= mid) s += count ? 1ull : whole_of(weight(x));
      });
      if (cluster_sum(s) >= need)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  }

  // Rank 0's `cut`, for every block.
  __device__ __forceinline__ u64 shared_cut() const {
    sync();
    return n_blocks == 1 ? sm.cut : remote_load64(remote(&sm.cut, 0));
  }

  // ------------------------------------------------------------ histograms
  // Bins are linear in the logit over the live range [low, top].
  struct Bins {
    float top, low, scale, width;
    int light;  // bins from here on weigh by their centre

    __device__ __forceinline__ int of(float x) const {
      const float t = fminf((top - x) * scale, (float)(kBins - 1));  // NaN: the last
      return __float_as_uint(__fadd_rd(t, 8388608.0f)) & (kBins - 1);
    }
    __device__ __forceinline__ float upper(int b) const {  // value where bin b begins
      return b <= 0 ? INFINITY : top - (float)b * width;
    }
    __device__ __forceinline__ float lower(int b) const {
      return b >= kBins - 1 ? low : top - (float)(b + 1) * width;
    }
  };
  __device__ Bins bins_over(float least) const {
    Bins b;
    b.top = top;
    b.low = fmaxf(least, cutoff());
    const float range = fminf(top - b.low, 3.0e38f);
    b.scale = range > 0.0f ? (float)kBins / range : 0.0f;
    b.width = range / kBins;
    b.light = 0;
    b.light = b.of(top - kHeavy / inv_t);
    return b;
  }
  __device__ __forceinline__ void count_in(const Bins& bins, float x, bool weigh, int n) const {
    if (!(x >= bins.low)) return;
    const int b = bins.of(x);
    atomicAdd(&sm.bins[b], (uint32_t)n);
    if (b < bins.light && weigh)
      atomicAdd(&sm.heavy[b],
                (uint32_t)((float)(n << 13) * (x == top ? 1.0f : __expf((x - top) * inv_t)) + 0.5f));
  }
  __device__ void clear_bins() const {
    for (int t = threadIdx.x; t < kBins; t += kThreads) sm.bins[t] = sm.heavy[t] = 0;
    __syncthreads();
  }
  // One pass that divides the row by value: this thread's sum of the whole
  // weights above `hi` (where weigh is set), their number, and where asked for
  // the sum of all; the tokens of [lo, hi] that are not below `least` go to the
  // list (its users leave out those with C's logit and a higher index).
  __device__ Sums split(float hi, float lo, float least, bool weigh, bool all) const {
    Sums s{0, 0, 0};
    lo = fmaxf(lo, least);
    const int end = end_vec();
    for (int j0 = first_vec(); j0 < end; j0 += 32 * 128) {
      WholeSum w, a;
      each_vec(j0, min(end, j0 + 32 * 128), 32, [&](const Vec<kF32>& x, int j) {
        uint32_t above = 0, inside = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          above |= x.at(e) > hi ? 1u << e : 0u;
          inside |= x.at(e) >= lo ? 1u << e : 0u;
        }
        push(x, j, inside & ~above);
        if (all || (above && weigh)) {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const float v = x.at(e);  // NaN and -inf take the bound, whose weight is zero
            const float t = v == top ? 0.0f : fmaxf((v - top) * inv_t, -100.0f);
            const WholeSum one = WholeSum::of(expf(t));
            a += one;
            if (above >> e & 1) w += one;
          }
        }
        s.count += __popc(above);
      });
      s.above += w.total();
      s.all += a.total();
    }
    return s;
  }

  // The draw among the tokens at or above C: `mine` is this thread's weight
  // above the list's range; rank 0's list (n entries) has the other kept ones.
  __device__ void draw_from_split(u64 mine, int n, u64 C, float u, long long* token) {
    mine = warp_sum(mine);
    if (threadIdx.x % 32 == 0) {
      const int at = (int)rank * kWarps + threadIdx.x / 32;
      if (n_blocks == 1)
        sm.wsum[at] = mine;
      else
        remote_store(remote(&sm.wsum[at], 0), mine);
    }
    sync();
    if (rank == 0) {
      for (int t = threadIdx.x; t < n; t += kThreads) {
        const u64 c = sm.list[t];
        if (c >= C) atomicAdd(&sm.wsum[((int)index_of(c) + row.mis) / E / per_warp], whole(c));
      }
      __syncthreads();
      u64 all;
      const int ranges = n_blocks * kWarps;
      const u64 ours = threadIdx.x < ranges ? sm.wsum[threadIdx.x] : 0;
      const u64 before = block_scan(ours, all, sm);
      const u64 target = share_of(all, draw_part(u));
      if (before <= target && target < before + ours)
        sm.pick = threadIdx.x, sm.rest = target - before;
    }
    sync();
    const int w = n_blocks == 1 ? sm.pick : (int)remote_load(remote(&sm.pick, 0));
    const u64 target = n_blocks == 1 ? sm.rest : remote_load64(remote(&sm.rest, 0));
    if (w / kWarps == (int)rank) draw_from_range(w, target, C, token);
  }

  // Fills cum_n and cum_m of every block from the groups' maxima and a sample of
  // the rest of the row: a few heavy tokens, mostly maxima, may carry much of it.
  __device__ void guess_bins(const Bins& bins, bool weigh) {
    const int tid = threadIdx.x;
    clear_bins();
    const int every = per_warp / 32 > 8 ? kSample : 1;
    const int end = end_vec();
#pragma unroll
    for (int g = 0; g < kGroups; ++g) count_in(bins, gm.m[g], weigh, 1);
    each_vec(first_vec(), end, 32 * every, [&](const Vec<kF32>& x, int j) {
      const int g = (j - first_vec()) / 32 / per_group;
      const float most = g & 2 ? (g & 1 ? gm.m[3] : gm.m[2]) : (g & 1 ? gm.m[1] : gm.m[0]);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (x.at(e) < most) count_in(bins, x.at(e), weigh, every);
    });
    sync();
    // Each block takes a run of the bins over the whole row, a thread up to four
    // of them: tokens, and roughly their weight.
    const int per = kBins / n_blocks, each_of = (per + kThreads - 1) / kThreads;
    const int first_bin = (int)rank * per + tid * each_of;
    const int n_bins = tid * each_of < per ? each_of : 0;
    float c[4], m[4], c_mine = 0.0f, m_mine = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = first_bin + e;
      uint32_t n = 0, heavy = 0;
      if (e < n_bins) {
        if (n_blocks == 1) {
          n = sm.bins[b], heavy = sm.heavy[b];
        } else {
          for (int r = 0; r < n_blocks; ++r) {
            n += remote_load(remote(&sm.bins[b], r));
            heavy += remote_load(remote(&sm.heavy[b], r));
          }
        }
      }
      c[e] = (float)n;
      m[e] = b < bins.light ? (float)heavy * (1.0f / 8192.0f)
                            : c[e] * __expf(-((float)b + 0.5f) * bins.width * inv_t);
      c_mine += c[e];
      m_mine += m[e];
    }
    float c_inc = c_mine, m_inc = m_mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float x = __shfl_up_sync(0xffffffffu, c_inc, off);
      const float y = __shfl_up_sync(0xffffffffu, m_inc, off);
      if (tid % 32 >= off) c_inc += x, m_inc += y;
    }
    __syncthreads();
    if (tid % 32 == 31)
      sm.part[tid / 32] = ((u64)__float_as_uint(c_inc) << 32) | __float_as_uint(m_inc);
    __syncthreads();
    float c_run = c_inc - c_mine, m_run = m_inc - m_mine, c_ours = 0.0f, m_ours = 0.0f;
    for (int w = 0; w < kWarps; ++w) {
      const float x = __uint_as_float((uint32_t)(sm.part[w] >> 32));
      const float y = __uint_as_float((uint32_t)sm.part[w]);
      if (w < tid / 32) c_run += x, m_run += y;
      c_ours += x, m_ours += y;
    }
    const Pair* p = exchange(__float_as_uint(c_ours), __float_as_uint(m_ours));
    for (int r = 0; r < (int)rank; ++r) {
      c_run += __uint_as_float((uint32_t)p[r].a);
      m_run += __uint_as_float((uint32_t)p[r].b);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= n_bins) break;
      const int b = first_bin + e;
      if (n_blocks == 1) {
        sm.cum_n[b] = c_run, sm.cum_m[b] = m_run;
      } else {
        for (int r = 0; r < n_blocks; ++r) {
          remote_store32(remote(&sm.cum_n[b], r), __float_as_uint(c_run));
          remote_store32(remote(&sm.cum_m[b], r), __float_as_uint(m_run));
        }
      }
      c_run += c[e], m_run += m[e];
    }
    sync();
  }
  // The last bin before which `cum` is below `want`.
  __device__ __forceinline__ int bin_at(const float* cum, float want) const {
    int lo = 0, hi = kBins - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (cum[mid] < want)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  }
  // The bin to look at next: where `want` is guessed, within the bins that are
  // left; after three misses the one that halves them.
  __device__ __forceinline__ int guess(const float* cum, float want, int tries, int from,
                                       int upto) const {
    return tries < 3 ? max(from, min(upto, bin_at(cum, want))) : (from + upto) / 2;
  }
  // The bins around bin `at`, `half` tokens to each side.
  __device__ __forceinline__ void window(int at, float half, int& b0, int& b1) const {
    b0 = min(max(0, at - 1), bin_at(sm.cum_n, sm.cum_n[at] - half));
    b1 = max(min(kBins - 1, at + 1), bin_at(sm.cum_n, sm.cum_n[min(kBins - 1, at + 1)] + half));
  }

  // The draw where the cuts go by histogram (see the head of the file). k <= 0:
  // no top-k, then `total` is the row's weight where it is known (else 0).
  __device__ void by_bins(int k, bool use_p, uint32_t part, u64 total, float least, float u,
                          long long* token) {
    const Bins bins = bins_over(least);
    guess_bins(bins, use_p);
    u64 C = 0;
    if (k > 0) {
      bool known = false;
      float want = (float)k, half = kWindow;
      int from = 0, upto = kBins - 1;  // bins that can hold the cut
      for (int tries = 0; tries < kTries && !known; ++tries) {
        int b0, b1;
        window(guess(sm.cum_n, want, tries, from, upto), half, b0, b1);
        clear_list();
        const Sums sums = split_row<kF32>(sm, bins.upper(b0), bins.lower(b1), -INFINITY,
                                          use_p || min_p <= 0.0f, false);
        const u64 mine = sums.above;
        const Pair above = cluster_sum(mine, sums.count);
        const int n = collect_list();
        if (n > kCap) {
          half *= 0.25f;
        } else if (above.b < (u64)k && (u64)k <= above.b + n) {
          u64 within = 0;
          if (rank == 0) {
            const u64 c = select<kCount>(n, (u64)k - above.b, 0);
            within = list_mass(n, c, false);
          }
          C = shared_cut();
          if (!use_p) {
            if (min_p > 0.0f)
              by_weight(C, u, token);
            else
              draw_from_split(mine, n, C, u, token);
            return;
          }
          total = above.a + exchange(within, 0)[0].a;
          known = true;
        } else if (b1 == kBins - 1 && above.b < (u64)k) {  // fewer live tokens: all are kept
          if (!use_p) {
            if (min_p > 0.0f)
              by_weight(0, u, token);
            else
              draw_from_split(mine, n, 0, u, token);
            return;
          }
          u64 within = 0;
          if (rank == 0) within = list_mass(n, 0, false);
          total = above.a + exchange(within, 0)[0].a;
          known = true;
        } else {
          want = sm.cum_n[b0] + ((float)k - (float)above.b);
          if (above.b >= (u64)k)
            upto = max(from, b0);
          else
            from = min(upto, b1);
        }
      }
      if (!known) {
        C = bisect((u64)k, true, 0);
        if (!use_p) {
          by_row(C, u, token);
          return;
        }
        u64 s = 0;
        each([&](float x, int i) {
          if (x > -INFINITY && composite(x, i) >= C) s += whole_of(weight(x));
        });
        total = cluster_sum(s);
      }
    }
    // Where the weight reaches its share.
    const float most = C ? logit_of(C) : -INFINITY;
    const float share = (float)part * (1.0f / 16777216.0f);
    // (an unknown total is guessed too: the last bin's start is nearly all)
    float want = total ? (float)total / kOne * share : sm.cum_m[kBins - 1] * share;
    float half = kWindow;
    int from = 0, upto = kBins - 1;
    for (int tries = 0; tries < kTries; ++tries) {
      int b0, b1;
      window(guess(sm.cum_m, want, tries, from, upto), half, b0, b1);
      clear_list();
      const float hi = fmaxf(bins.upper(b0), most), lo = bins.lower(b1);
      const Sums sums = split_row<kF32>(sm, hi, lo, most, true, total == 0);
      const u64 mine = sums.above;
      const Pair both = cluster_sum(mine, sums.all);
      const u64 above = both.a;
      if (total == 0) total = both.b;
      const int n = collect_list();
      const u64 bound = max(share_of(total, part), (u64)1);
      if (n > kCap) {
        half *= 0.25f;
        continue;
      }
      u64 listed = 0;
      if (rank == 0) listed = list_mass(n, C, false);
      listed = exchange(listed, 0)[0].a;
      if (above < bound && bound <= above + listed) {
        if (rank == 0) select<kMass>(n, bound - above, C);
        C = shared_cut();
        if (min_p > 0.0f)
          by_weight(C, u, token);
        else
          draw_from_split(mine, n, C, u, token);
        return;
      }
      // The guess before bin b0 is off by what the exact sum says.
      want = sm.cum_m[b0] + ((float)bound - (float)above) / kOne;
      if (above >= bound)
        upto = max(from, b0);
      else
        from = min(upto, b1);
    }
    by_row(bisect(max(share_of(total, part), (u64)1), false, C), u, token);
  }

  // ------------------------------------------------------- group candidates
  // Lists the tokens of the groups whose maximum is a candidate, those that are
  // candidates themselves.
  template <class F>
  __device__ void list_candidates(F candidate) {
    const int tid = threadIdx.x;
    if (tid == 0) sm.n_groups = 0;
    clear_list();
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (candidate(gm.m[g])) sm.groups[atomicAdd(&sm.n_groups, 1)] = group_first(g);
    __syncthreads();
    // Their vectors, shared among all threads.
    const int items = sm.n_groups * per_group;
    for (int it0 = tid; it0 < items; it0 += 4 * kThreads) {
      Vec<kF32> x[4];
      int at[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // Step s of a group, unless past the end of the group's warp range.
        const int it = it0 + e * kThreads;
        at[e] = -1;
        if (it < items) {
          const int f = sm.groups[it / per_group], j = f + it % per_group * 32;
          if (j < min(row.n_vec, (f / per_warp + 1) * per_warp)) at[e] = j;
        }
        if (at[e] >= 0) x[e] = row.get(at[e]);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (at[e] >= 0) {
          uint32_t bits = 0;
#pragma unroll
          for (int i = 0; i < E; ++i) bits |= candidate(x[e].at(i)) ? 1u << i : 0u;
          push(x[e], at[e], bits);
        }
    }
  }

  // Draw among the tokens at or above C with w >= min_p, min_p > 0.
  __device__ void by_weight(u64 C, float u, long long* token) {
    const float least = C ? logit_of(C) : -INFINITY;
    list_candidates([&](float x) { return x > -INFINITY && x >= least && weight(x) >= min_p; });
    const int n = collect_list();
    if (n > kCap)
      by_row(C, u, token);
    else if (rank == 0)
      draw_from_list(n, C, n, false, 0, 0, u, token);
  }

  // --------------------------------------------------------------- one row
  __device__ void run(const void* p, float T, int k, float top_p, float u, long long* token) {
    const int tid = threadIdx.x, lane = tid % 32;
    // Maxima of the thread's groups, and the row's extremes.
    const int end = end_vec();
    Extremes<kF32> all;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
      Extremes<kF32> m;
      int j = group_first(g);
      const int stop = min(end, j + 32 * per_group);
      for (; j + 224 < stop; j += 256) {
        Vec<kF32> x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = row.get(j + 32 * i);
#pragma unroll
        for (int i = 0; i < 8; ++i) m.add(x[i], all);
      }
      for (; j < stop; j += 32) m.add(row.get(j), all);
      gm.m[g] = m.max();
    }
    if (tid < kGroupBins) sm.gbins[tid] = sm.gmass[tid] = 0;
    if (tid == 0) sm.count = 0, sm.n_groups = 0, sm.found = 0x7fffffff;
    float low, least;  // smallest group maximum, smallest logit
    {
      float hi = fmaxf(fmaxf(gm.m[0], gm.m[1]), fmaxf(gm.m[2], gm.m[3])), lo = INFINITY;
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (gm.m[g] > -INFINITY) lo = fminf(lo, gm.m[g]);
      float mn = all.min();
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
      }
      if (lane == 0) {
        sm.fpart[tid / 32] = hi;
        sm.part[tid / 32] = ((u64)__float_as_uint(lo) << 32) | __float_as_uint(mn);
      }
      __syncthreads();
      top = -INFINITY, low = INFINITY, least = INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        top = fmaxf(top, sm.fpart[w]);
        low = fminf(low, __uint_as_float((uint32_t)(sm.part[w] >> 32)));
        least = fminf(least, __uint_as_float((uint32_t)sm.part[w]));
      }
    }
    if (n_blocks > 1) {
      wait_started();
      const Pair* p = exchange(__float_as_uint(top),
                               ((u64)__float_as_uint(low) << 32) | __float_as_uint(least));
      for (int r = 0; r < n_blocks; ++r) {
        top = fmaxf(top, __uint_as_float((uint32_t)p[r].a));
        low = fminf(low, __uint_as_float((uint32_t)(p[r].b >> 32)));
        least = fminf(least, __uint_as_float((uint32_t)p[r].b));
      }
    }
    if (top == -INFINITY) {
      if (rank == 0 && tid == 0) *token = -1;
      return;
    }
    if (!(T > 0.0f)) {
      // Greedy: the lowest index that holds the maximum.
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (gm.m[g] == top)
          each_in(group_first(g), min(end, group_first(g) + 32 * per_group), [&](float x, int i) {
            if (x == top) atomicMin(&sm.found, i);
          });
      __syncthreads();
      int best = sm.found;
      if (n_blocks > 1) {
        const Pair* p = exchange((u64)best, 0);
        for (int r = 0; r < n_blocks; ++r) best = min(best, (int)p[r].a);
      }
      if (rank == 0 && tid == 0) *token = best;
      return;
    }
    const bool use_k = k > 0 && k < row.V, use_p = top_p < 1.0f;
    const uint32_t part = (uint32_t)(fmaxf(top_p, 0.0f) * 16777216.0f);
    if (!use_k && !use_p) {
      leave(p, least, u, token);
      if (min_p > 0.0f)
        draw_by_weight<kF32>(sm, gm, 0);
      else
        draw_from_row<kF32>(sm, 0);
      return;
    }
    u64 total = 0;
    if (!use_k || k <= kSmallK) {
      // Bins over the group maxima; a bin also decides which logits are
      // candidates, so that those are a leading run up to ties.
      const float live = cutoff();
      const float range = fminf(top - low, fminf(kLive / inv_t, 3.0e38f));
      const float scale = range > 0.0f ? (float)kGroupBins / range : 0.0f;
      auto bin_of = [&](float x) { return min(kGroupBins - 1, (int)((top - x) * scale)); };
      float sure = 0.0f, sample = 0.0f;  // weight of the maxima, and of a vector's rest
#pragma unroll
      for (int g = 0; g < kGroups; ++g)
        if (gm.m[g] > -INFINITY && gm.m[g] >= live) {
          const int b = bin_of(gm.m[g]);
          atomicAdd(&sm.gbins[b], 1u);
          if (!use_k) {
            const float w = __expf((gm.m[g] - top) * inv_t);
            sure += gm.m[g] == top ? 1.0f : w;
            atomicAdd(&sm.gmass[b], (uint32_t)((gm.m[g] == top ? 1.0f : w) * 131072.0f));
          }
        }
      if (!use_k) {
        const int j = first_vec();
        if (j < end) {
          const Vec<kF32> x = row.get(j);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (x.at(e) < gm.m[0]) sample += __expf((x.at(e) - top) * inv_t);
        }
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) {
          sure += __shfl_xor_sync(0xffffffffu, sure, off);
          sample += __shfl_xor_sync(0xffffffffu, sample, off);
        }
        if (lane == 0)
          sm.est[tid / 32] = ((u64)__float_as_uint(sure) << 32) | __float_as_uint(sample);
        __syncthreads();
        sure = sample = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          sure += __uint_as_float((uint32_t)(sm.est[w] >> 32));
          sample += __uint_as_float((uint32_t)sm.est[w]);
        }
        if (n_blocks > 1) {
          const Pair* p = exchange(__float_as_uint(sure), __float_as_uint(sample));
          sure = sample = 0.0f;
          for (int r = 0; r < n_blocks; ++r) {
            sure += __uint_as_float((uint32_t)p[r].a);
            sample += __uint_as_float((uint32_t)p[r].b);
          }
        }
      }
      sync();
      if (n_blocks > 1) {
        uint32_t n = 0, w = 0;
        if (tid < kGroupBins)
          for (int r = 0; r < n_blocks; ++r) {
            n += remote_load(remote(&sm.gbins[tid], r));
            w += remote_load(remote(&sm.gmass[tid], r));
          }
        sync();  // read by all before it is overwritten
        if (tid < kGroupBins) sm.gbins[tid] = n, sm.gmass[tid] = w;
        __syncthreads();
      }
      // The first bin up to which the groups suffice (the last if none does), by
      // number for top-k, by weight for top-p; every warp finds it for itself.
      float want = (float)k;
      if (!use_k) {
        const int sampled = min(row.n_vec, n_blocks * kThreads);
        const float est = sure + sample * ((float)row.n_vec / (float)sampled);
        want = fminf(1.05f * est * (float)part * (131072.0f / 16777216.0f), 4.0e9f);
      }
      constexpr int kEach = kGroupBins / 32;
      const uint32_t* goal = use_k ? sm.gbins : sm.gmass;
      uint32_t mine = 0, mine_n = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        mine += goal[lane * kEach + e], mine_n += sm.gbins[lane * kEach + e];
      uint32_t inc = mine, inc_n = mine_n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, inc, off);
        const uint32_t z = __shfl_up_sync(0xffffffffu, inc_n, off);
        if (lane >= off) inc += y, inc_n += z;
      }
      uint32_t run = inc - mine, run_n = inc_n - mine_n;
      int at = kGroupBins;
      uint32_t at_n = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) {
        run += goal[lane * kEach + e], run_n += sm.gbins[lane * kEach + e];
        if (at == kGroupBins && (float)run >= want) at = lane * kEach + e, at_n = run_n;
      }
      const int cut = __reduce_min_sync(0xffffffffu, at);
      const uint32_t n_cut = __reduce_max_sync(0xffffffffu, at == cut ? at_n : 0u);
      // A flat nucleus: its tokens are found by the row's histogram.
      if (!use_k && (cut == kGroupBins || n_cut > kNucleus)) {
        leave(p, least, u, token);
        draw_by_bins<kF32>(sm, gm, 0, part, 0);
        return;
      }
      list_candidates(
          [&](float x) { return x > -INFINITY && x >= live && bin_of(x) <= cut; });
      const int n = collect_list();
      u64 bound = 0;
      bool enough = n <= kCap;
      if (!use_k) {
        // Rank 0 adds the list's weight, which the others need not know of.
        const u64 listed = rank == 0 && n <= kCap ? list_mass(n, 0, false) : 0;
        const Pair s = cluster_sum(mass(), threadIdx.x == 0 ? listed : 0);
        total = s.a;
        bound = max(share_of(total, part), (u64)1);
        enough = enough && s.b >= bound;
      }
      if (enough) {
        if (n > kRank) leave(p, least, u, token);
        if (rank == 0) draw_from_list(n, 0, use_k ? min(n, k) : n, use_p, bound, part, u, token);
        return;
      }
    }
    leave(p, least, u, token);
    draw_by_bins<kF32>(sm, gm, use_k ? k : 0, use_p ? part : kNoCut, total);
  }
};

template <bool kF32>
__device__ __noinline__ void draw_by_bins(Shared& sm, Groups gm, int k, uint32_t part, u64 total) {
  Sampler<kF32> s(sm);
  s.gm = gm;
  s.by_bins(k, part != kNoCut, part, total, sm.row.least, sm.row.u, sm.row.token);
}
template <bool kF32>
__device__ __noinline__ Sums split_row(Shared& sm, float hi, float lo, float least, bool weigh,
                                       bool all) {
  return Sampler<kF32>(sm).split(hi, lo, least, weigh, all);
}
template <bool kF32>
__device__ __noinline__ void draw_by_weight(Shared& sm, Groups gm, u64 C) {
  Sampler<kF32> s(sm);
  s.gm = gm;
  s.by_weight(C, sm.row.u, sm.row.token);
}
template <bool kF32>
__device__ __noinline__ void draw_from_row(Shared& sm, u64 C) {
  Sampler<kF32> s(sm);
  s.by_row(C, sm.row.u, sm.row.token);
}
template <bool kF32>
__device__ __noinline__ void draw_long_list(Shared& sm, int n, u64 C, int n_k, bool use_p, u64 bound,
                                            uint32_t part) {
  Sampler<kF32> s(sm);
  s.long_list(n, C, n_k, use_p, bound, part, sm.row.u, sm.row.token);
}

template <bool kF32>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p, int n_blocks) {
  __shared__ Shared sm;
  const int b = blockIdx.x / n_blocks;
  const uint8_t* row = reinterpret_cast<const uint8_t*>(p.logits) + b * p.stride * (kF32 ? 4 : 2);
  Sampler<kF32> s(row, p.V, sm, n_blocks, n_blocks > 1 ? cluster_rank() : 0);
  s.started();
  const float T = p.temperature ? p.temperature[b] : p.temperature_all;
  // (finite and not zero: a difference of zero weighs one at any temperature)
  s.inv_t = T > 0.0f ? 1.0f / fminf(fmaxf(T, 1.2e-38f), 1.0e38f) : 1.0f;
  s.min_p = fminf(p.min_p ? p.min_p[b] : p.min_p_all, 1.0f);  // the best token stays
  s.run(row, T, p.top_k ? p.top_k[b] : p.top_k_all, p.top_p ? p.top_p[b] : p.top_p_all, p.u[b],
        p.tokens + b);
  if (n_blocks > 1) s.sync();  // no block's shared memory goes while another reads it
}

// Blocks per row: a power of two up to 8, doubled while the blocks before it leave
// room for two a SM, with at least one vector for each thread. Flat rows gain by it
// and sharp ones under a small top-k, which read little more than once, lose the
// exchanges' time. Measured, us with 1, 2, 4 and 8 blocks a row (the rule's choice in
// brackets): 16 rows of 131072 bf16, top-p alone 70, 60, 55, [48], top-k and top-p
// 11, 14, 13, [15]; 64 rows of 100003 fp32 with mixed settings 121, 94, [81], 90, top-k
// and top-p 24, 26, [21], 36; 128 rows of 131072 bf16, top-p alone 92, [89], 103, 147,
// top-k and top-p 15, [22], 35, 63. 256 rows of 131072 with two: top-k and top-p 42
// against [21].
int choose_cluster(int B, int V, bool fp32, int n_sms) {
  const int per_block = kThreads * (fp32 ? 4 : 8);
  int c = 1;
  while (c < kMaxCluster && (long long)B * c * 2 <= 2 * n_sms && (long long)c * per_block < V)
    c *= 2;
  return c;
}

template <bool kF32>
cudaError_t launch(const SampleParams& p, cudaStream_t stream) {
  const int c = choose_cluster(p.B, p.V, kF32, p.n_sms);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.B * c);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)c, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = c > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, sample_kernel<kF32>, p, c);
}

}  // namespace smp

cudaError_t launch_sample(const SampleParams& p, cudaStream_t stream) {
  return p.fp32 ? smp::launch<true>(p, stream) : smp::launch<false>(p, stream);
}

}  // namespace enl
