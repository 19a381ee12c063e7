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
// One block per row. The first pass streams the row from HBM and keeps only
// maxima: the row's and, per thread, those of four parts of what it read
// (2048 groups). What follows reads the row again from L2, and only where it
// has to:
//  * top-k up to kSmallK: the k-th largest group maximum bounds the k-th largest
//    logit from below, so only groups at or above it (about k of them) are read
//    again. Their few candidates are sorted in shared memory, and the rest of
//    the row is never touched.
//  * top-p alone: one more pass for the exact total, then the same with about
//    kNucleus candidates, provided that they carry the wanted mass.
//  * larger top-k, flatter nuclei: a histogram of the logits finds the bin that
//    the cut falls into, one pass sums what lies above it and collects the bin's
//    tokens, which are sorted.
//  * rows that defeat the bins (thousands of equal logits at the cut): bisection
//    over the composite, one pass per bit.
// Without a cut (temperature alone, min-p) one pass sums the row in ranges and
// the range that holds the draw is walked again.
#include <cstdint>

#include "enl_common.cuh"
#include "enl_kernels.h"

namespace enl {

namespace smp {

using u64 = unsigned long long;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = 4;       // group maxima per thread
constexpr int kCap = 2048;       // candidates that fit the shared-memory sort
constexpr int kSmallK = 1024;    // largest top-k of the group path
constexpr int kNucleus = 640;    // groups asked for when only top-p cuts
constexpr int kGroupBins = 256;  // bins over the group maxima
constexpr int kBins = 2048;      // bins over the row
constexpr float kOne = 1099511627776.0f;  // 2^40
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
};

// Running maximum of vectors; NaN is dropped. bf16 stays packed.
template <bool kF32>
struct Maximum {
  float f = -INFINITY;
  __nv_bfloat162 h = __float2bfloat162_rn(-INFINITY);

  __device__ __forceinline__ void add(const Vec<kF32>& x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (kF32)
        f = fmaxf(f, __uint_as_float(x.w[i]));
      else
        h = __hmax2(h, *reinterpret_cast<const __nv_bfloat162*>(&x.w[i]));
    }
  }
  __device__ __forceinline__ float get() const {
    return kF32 ? f : fmaxf(__low2float(h), __high2float(h));
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
  __device__ __forceinline__ float logit_or_low(int i) const {
    return i >= 0 && i < V ? one(i) : -INFINITY;
  }
  // Vector j; indices outside the row read as -inf (and touch no memory).
  __device__ __forceinline__ Vec<kF32> get(int j) const {
    Vec<kF32> r;
    if (inside(j)) {
      const uint4 w = *reinterpret_cast<const uint4*>(base + (size_t)j * 16);
      r.w[0] = w.x, r.w[1] = w.y, r.w[2] = w.z, r.w[3] = w.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kF32) {
          r.w[e] = __float_as_uint(logit_or_low(j * E - mis + e));
        } else {
          r.w[e] = __float_as_uint(logit_or_low(j * E - mis + 2 * e)) >> 16 |
                   __float_as_uint(logit_or_low(j * E - mis + 2 * e + 1));
        }
      }
    }
    return r;
  }
};

struct Shared {
  union {
    u64 list[kCap];         // candidates (composites), sorted in place
    uint32_t bins[kBins];   // histogram
  };
  u64 order[kCap];          // kept candidates by index
  u64 part[kWarps + 1];
  float fpart[kWarps];
  uint32_t gbins[kGroupBins];
  int count, found;
};

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

// Bitonic sort of a[0 .. n), n a power of two.
template <bool kDescending>
__device__ void block_sort(u64* a, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < n / 2; t += kThreads) {
        const int i = 2 * t - (t & (stride - 1)), j = i + stride;
        const u64 x = a[i], y = a[j];
        const bool up = ((i & size) == 0) != kDescending;
        if ((x > y) == up) a[i] = y, a[j] = x;
      }
    }
  __syncthreads();
}

__device__ __forceinline__ int pow2_at_least(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

template <bool kF32>
struct Sampler {
  static constexpr int E = Vec<kF32>::E;
  Row<kF32> row;
  Shared& sm;
  float top, inv_t, min_p;
  int per_warp;  // vectors of a warp's contiguous range, a multiple of 32

  __device__ Sampler(const void* p, int V, Shared& s) : row(p, V), sm(s) {
    per_warp = (row.n_vec + kWarps * 32 - 1) / (kWarps * 32) * 32;
  }
  __device__ __forceinline__ int first_vec() const {
    return (threadIdx.x / 32) * per_warp + threadIdx.x % 32;
  }
  __device__ __forceinline__ int end_vec() const {
    return min(row.n_vec, (int)(threadIdx.x / 32 + 1) * per_warp);
  }
  __device__ __forceinline__ float weight(float x) const { return weight_of(x, top, inv_t); }
  __device__ __forceinline__ u64 whole(u64 comp) const {
    return whole_of(weight(of_key((uint32_t)(comp >> 32))));
  }

  // Logits below this have no weight.
  __device__ __forceinline__ float cutoff() const {
    return top == INFINITY ? top : top - kLive / inv_t;
  }

  // f(value, index) for every logit that this thread reads.
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    const int end = end_vec();
    int j = first_vec();
    for (; j + 96 < end; j += 128) {
      Vec<kF32> x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = row.get(j + 32 * u);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int e = 0; e < E; ++e) f(x[u].at(e), (j + 32 * u) * E - row.mis + e);
    }
    for (; j < end; j += 32) {
      const Vec<kF32> x = row.get(j);
#pragma unroll
      for (int e = 0; e < E; ++e) f(x.at(e), j * E - row.mis + e);
    }
  }

  // Exact sum of the whole weights of the row.
  __device__ u64 row_mass() const {
    u64 s = 0;
    const int end = end_vec();
    for (int j0 = first_vec(); j0 < end; j0 += 32 * 64) {  // at most 512 tokens a stretch
      WholeSum w;
#pragma unroll 4
      for (int j = j0; j < min(end, j0 + 32 * 64); j += 32) {
        const Vec<kF32> x = row.get(j);
#pragma unroll
        for (int e = 0; e < E; ++e) w.add(x.at(e) > -INFINITY ? weight(x.at(e)) : 0.0f);
      }
      s += w.total();
    }
    return block_sum(s, sm);
  }

  // Appends a composite to the list; the list may overflow (count says so).
  __device__ __forceinline__ void push(float x, int i) const {
    const int at = atomicAdd(&sm.count, 1);
    if (at < kCap) sm.list[at] = composite(x, i);
  }

  // Sorts the list (n entries) with the largest composite first.
  __device__ void sort_list(int n) const {
    const int N = pow2_at_least(n);
    for (int t = n + threadIdx.x; t < N; t += kThreads) sm.list[t] = 0;
    block_sort<true>(sm.list, N);
  }

  // In the sorted list: sums of whole weights of this thread's four entries,
  // before (exclusive) and in all.
  __device__ u64 list_scan(const u64* list, int n, u64 (&q)[4], u64& total) const {
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = threadIdx.x * 4 + e;
      q[e] = r < n ? whole(list[r]) : 0;
      mine += q[e];
    }
    return block_scan(mine, total, sm);
  }

  // Index-order draw among the first n entries of the sorted list.
  __device__ void draw_from_list(int n, float u, long long* token) const {
    const int N = pow2_at_least(n);
    for (int t = threadIdx.x; t < N; t += kThreads) {
      const u64 c = sm.list[t];
      sm.order[t] = t < n ? ((u64)(uint32_t)~(uint32_t)c << 32) | (c >> 32) : ~0ull;
    }
    block_sort<false>(sm.order, N);
    u64 q[4], total, mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = threadIdx.x * 4 + e;
      q[e] = r < n ? whole_of(weight(of_key((uint32_t)sm.order[r]))) : 0;
      mine += q[e];
    }
    u64 run = block_scan(mine, total, sm);
    const u64 target = share_of(total, draw_part(u));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (q[e] && run <= target && target < run + q[e])
        *token = (long long)(sm.order[threadIdx.x * 4 + e] >> 32);
      run += q[e];
    }
  }

  static __device__ __forceinline__ uint32_t draw_part(float u) {
    return (uint32_t)(fminf(fmaxf(u, 0.0f), 0.99999994f) * 16777216.0f);
  }

  // Draw among the tokens at or above the composite C with w >= min_p: sums of
  // the warps' ranges, then of the range that holds the draw.
  __device__ void draw_from_row(u64 C, float u, long long* token) const {
    auto mass_of = [&](float x, int i) -> u64 {
      if (!(x > -INFINITY)) return 0;  // NaN too
      const float w = weight(x);
      return w >= min_p && (C == 0 || composite(x, i) >= C) ? whole_of(w) : 0;
    };
    u64 mine = 0;
    each([&](float x, int i) { mine += mass_of(x, i); });
    mine = warp_sum(mine);
    __syncthreads();
    if (threadIdx.x % 32 == 0) sm.part[threadIdx.x / 32] = mine;
    __syncthreads();
    u64 total = 0, before = 0;
    for (int w = 0; w < kWarps; ++w) total += sm.part[w];
    const u64 target = share_of(total, draw_part(u));
    int w = 0;
    while (w < kWarps - 1 && before + sm.part[w] <= target) before += sm.part[w++];
    // The range in contiguous pieces, one per thread.
    const int begin = w * per_warp, end = min(row.n_vec, begin + per_warp);
    const int piece = (per_warp + kThreads - 1) / kThreads;
    const int j0 = begin + threadIdx.x * piece, j1 = min(end, j0 + piece);
    mine = 0;
    for (int j = j0; j < j1; ++j) {
      const Vec<kF32> x = row.get(j);
#pragma unroll
      for (int e = 0; e < E; ++e) mine += mass_of(x.at(e), j * E - row.mis + e);
    }
    u64 all;
    u64 run = before + block_scan(mine, all, sm);
    if (run <= target && target < run + mine) {
      for (int j = j0; j < j1; ++j) {
        const Vec<kF32> x = row.get(j);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const int i = j * E - row.mis + e;
          const u64 q = mass_of(x.at(e), i);
          if (q && run <= target && target < run + q) *token = i;
          run += q;
        }
      }
    }
  }

  // Composite of the last token of the smallest leading run of the tokens at
  // or above C that holds `need` tokens, or whole weight `need`; 0 if none does.
  __device__ u64 bisect(u64 need, bool count, u64 C) const {
    u64 lo = C, hi = composite(top, 0) | 0xffffffffull;  // run at lo: the answer or all
    while (lo < hi) {
      const u64 mid = hi - (hi - lo) / 2;
      u64 s = 0;
      each([&](float x, int i) {
        if (x > -INFINITY && composite(x, i) >= mid) s += count ? 1ull : whole_of(weight(x));
      });
      if (block_sum(s, sm) >= need)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  }

  // The cuts by histogram (see the head of the file): the composite at or
  // above which a token is kept. k <= 0: no top-k; bound by top_p part of 2^24.
  __device__ u64 cut_by_bins(int k, bool use_p, uint32_t part) const {
    const int tid = threadIdx.x;
    // Bins are linear in the logit over the live range [low, top].
    float low = INFINITY;
    const float live = cutoff();
    each([&](float x, int) {
      if (x > -INFINITY && x >= live) low = fminf(low, x);
    });
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, off));
    __syncthreads();
    if (tid % 32 == 0) sm.fpart[tid / 32] = low;
    for (int t = tid; t < kBins; t += kThreads) sm.bins[t] = 0;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) low = fminf(low, sm.fpart[w]);
    const float range = fminf(top - low, 3.0e38f);
    const float scale = range > 0.0f ? (float)kBins / range : 0.0f;
    auto bin_of = [&](float x) { return min(kBins - 1, (int)((top - x) * scale)); };
    each([&](float x, int) {
      if (x >= low) atomicAdd(&sm.bins[bin_of(x)], 1u);
    });
    __syncthreads();
    // This thread's four bins, and the tokens and (roughly) the weight before.
    uint32_t c[4];
    float m[4];
    u64 n_mine = 0;
    float m_mine = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int b = tid * 4 + e;
      c[e] = sm.bins[b];
      m[e] = c[e] * expf(-((float)b + 0.5f) * (range / kBins) * inv_t);
      n_mine += c[e];
      m_mine += m[e];
    }
    u64 n_all;
    u64 n_before = block_scan(n_mine, n_all, sm);

    u64 C = 0;
    u64 mass_k = 0;  // exact weight of the top-k, once known
    int last_bin = kBins - 1;
    if (k > 0 && (u64)k < n_all) {
      if (tid == 0) sm.count = 0;
      __syncthreads();  // the bins have been read; `found` may be written
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (n_before < (u64)k && (u64)k <= n_before + c[e]) {
          sm.found = tid * 4 + e;
          sm.part[kWarps] = n_before;
        }
        n_before += c[e];
      }
      __syncthreads();
      const int cut = sm.found;
      const int need = (int)((u64)k - sm.part[kWarps]);
      u64 above = 0;
      each([&](float x, int i) {
        if (!(x >= low)) return;
        const int b = bin_of(x);
        if (b < cut && use_p) above += whole_of(weight(x));
        if (b == cut) push(x, i);
      });
      above = block_sum(above, sm);
      const int n = sm.count;
      last_bin = cut;
      if (n > kCap) {
        C = bisect((u64)k, true, 0);
        if (use_p) {
          u64 s = 0;
          each([&](float x, int i) {
            if (x > -INFINITY && composite(x, i) >= C) s += whole_of(weight(x));
          });
          mass_k = block_sum(s, sm);
        }
      } else {
        sort_list(n);
        C = sm.list[need - 1];
        u64 q[4], all;
        list_scan(sm.list, need, q, all);
        mass_k = above + all;
      }
    } else if (use_p) {
      mass_k = row_mass();
    }
    if (!use_p) return C;

    // The bin that the mass bound falls into, by the rough weights; it and its
    // neighbours are collected and the exact sums decide.
    const u64 bound = max(share_of(mass_k, part), (u64)1);
    float m_inc = m_mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, m_inc, off);
      if (tid % 32 >= off) m_inc += y;
    }
    __syncthreads();
    if (tid % 32 == 31) sm.fpart[tid / 32] = m_inc;
    if (tid == 0) sm.found = last_bin, sm.count = 0;
    __syncthreads();
    float run = m_inc - m_mine;
    for (int w = 0; w < (int)(tid / 32); ++w) run += sm.fpart[w];
    const float want = (float)bound / kOne;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      run += m[e];
      if (run >= want) {
        atomicMin(&sm.found, tid * 4 + e);
        break;
      }
    }
    __syncthreads();
    const int b0 = max(0, sm.found - 1), b1 = min(last_bin, sm.found + 1);
    u64 above = 0;
    each([&](float x, int i) {
      if (!(x >= low)) return;
      const int b = bin_of(x);
      if (b > b1 || (b == last_bin && C != 0 && composite(x, i) < C)) return;
      if (b < b0)
        above += whole_of(weight(x));
      else
        push(x, i);
    });
    above = block_sum(above, sm);
    const int n = sm.count;
    if (n > kCap || n == 0 || above >= bound) return bisect(bound, false, C);
    sort_list(n);
    u64 q[4], all;
    u64 before = above + list_scan(sm.list, n, q, all);
    if (above + all < bound) return bisect(bound, false, C);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (q[e] && before < bound && bound <= before + q[e])
        sm.part[kWarps] = sm.list[tid * 4 + e];
      before += q[e];
    }
    __syncthreads();
    return sm.part[kWarps];
  }
};

template <bool kF32>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleParams p) {
  __shared__ Shared sm;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid % 32;
  const float T = p.temperature ? p.temperature[b] : p.temperature_all;
  const int k = p.top_k ? p.top_k[b] : p.top_k_all;
  const float top_p = p.top_p ? p.top_p[b] : p.top_p_all;
  const float u = p.u[b];
  Sampler<kF32> s(reinterpret_cast<const uint8_t*>(p.logits) + b * p.stride * (kF32 ? 4 : 2), p.V,
                  sm);
  s.min_p = fminf(p.min_p ? p.min_p[b] : p.min_p_all, 1.0f);  // the best token stays
  s.inv_t = T > 0.0f ? 1.0f / fminf(T, 1.0e38f) : 1.0f;
  constexpr int E = Vec<kF32>::E;

  // Maxima of the row and of each thread's groups. fmaxf drops NaN.
  const int v0 = s.first_vec(), v1 = s.end_vec();
  const int steps = s.per_warp / 32;
  auto group_first = [&](int g) { return v0 + 32 * (steps * g / kGroups); };
  auto group_end = [&](int g) { return min(v1, v0 + 32 * (steps * (g + 1) / kGroups)); };
  float gm[kGroups];
#pragma unroll
  for (int g = 0; g < kGroups; ++g) {
    Maximum<kF32> m;
    const int end = group_end(g);
    int j = group_first(g);
    for (; j + 224 < end; j += 256) {
      Vec<kF32> x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = s.row.get(j + 32 * i);
#pragma unroll
      for (int i = 0; i < 8; ++i) m.add(x[i]);
    }
    for (; j < end; j += 32) m.add(s.row.get(j));
    gm[g] = m.get();
  }
  if (tid < kGroupBins) sm.gbins[tid] = 0;
  if (tid == 0) sm.count = 0, sm.found = 0x7fffffff;
  {
    float hi = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3])), lo = INFINITY;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (gm[g] > -INFINITY) lo = fminf(lo, gm[g]);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, off));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, off));
    }
    if (lane == 0) sm.fpart[tid / 32] = hi, sm.part[tid / 32] = __float_as_uint(lo);
  }
  __syncthreads();
  float top = -INFINITY, low = INFINITY;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    top = fmaxf(top, sm.fpart[w]);
    low = fminf(low, __uint_as_float((uint32_t)sm.part[w]));
  }
  s.top = top;
  long long* token = p.tokens + b;
  if (top == -INFINITY) {
    if (tid == 0) *token = -1;
    return;
  }
  if (!(T > 0.0f)) {
    // Greedy: the lowest index that holds the maximum.
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (gm[g] == top)
        for (int j = group_first(g); j < group_end(g); j += 32) {
          const Vec<kF32> x = s.row.get(j);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (x.at(e) == top) atomicMin(&sm.found, j * E - s.row.mis + e);
        }
    __syncthreads();
    if (tid == 0) *token = sm.found;
    return;
  }
  const bool use_k = k > 0 && k < p.V, use_p = top_p < 1.0f;
  const uint32_t part = (uint32_t)(fmaxf(top_p, 0.0f) * 16777216.0f);
  if (!use_k && !use_p) {
    s.draw_from_row(0, u, token);
    return;
  }
  if (!use_k || k <= kSmallK) {
    // Bins over the group maxima; a group's bin also decides which of its
    // logits are candidates, so the candidates are a leading run up to ties.
    const float range = fminf(top - low, fminf(kLive / s.inv_t, 3.0e38f));
    const float scale = range > 0.0f ? (float)kGroupBins / range : 0.0f;
    const float cutoff = s.cutoff();
    auto bin_of = [&](float x) { return min(kGroupBins - 1, (int)((top - x) * scale)); };
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (gm[g] > -INFINITY && gm[g] >= cutoff) atomicAdd(&sm.gbins[bin_of(gm[g])], 1u);
    __syncthreads();
    // The first bin up to which the groups suffice (all of them if none does).
    const u64 want = use_k ? (u64)k : (u64)kNucleus;
    u64 all, mine = tid < kGroupBins ? sm.gbins[tid] : 0;
    const u64 before = block_scan(mine, all, sm);
    if (tid == 0) sm.found = kGroupBins - 1;
    __syncthreads();
    if (tid < kGroupBins && before < want && want <= before + mine) sm.found = tid;
    __syncthreads();
    const int cut = sm.found;
#pragma unroll
    for (int g = 0; g < kGroups; ++g)
      if (gm[g] > -INFINITY && gm[g] >= cutoff && bin_of(gm[g]) <= cut)
        for (int j = group_first(g); j < group_end(g); j += 32) {
          const Vec<kF32> x = s.row.get(j);
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (x.at(e) > -INFINITY && x.at(e) >= cutoff && bin_of(x.at(e)) <= cut)
              s.push(x.at(e), j * E - s.row.mis + e);
        }
    __syncthreads();
    const int n = sm.count;
    if (n <= kCap) {
      u64 bound = ~0ull, q[4], total;
      bool enough = true;
      if (!use_k) {
        bound = max(share_of(s.row_mass(), part), (u64)1);
        s.list_scan(sm.list, n, q, total);
        enough = total >= bound;
      }
      if (enough) {
        s.sort_list(n);
        const int n_k = use_k ? min(n, k) : n;
        u64 run = s.list_scan(sm.list, n_k, q, total);
        if (use_k && use_p) bound = max(share_of(total, part), (u64)1);
        u64 keep = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = tid * 4 + e;
          keep += r < n_k && run < bound && q[e] &&
                  s.weight(of_key((uint32_t)(sm.list[r] >> 32))) >= s.min_p;
          run += q[e];
        }
        s.draw_from_list((int)block_sum(keep, sm), u, token);
        return;
      }
    }
    __syncthreads();
  }
  s.draw_from_row(s.cut_by_bins(use_k ? k : 0, use_p, part), u, token);
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
