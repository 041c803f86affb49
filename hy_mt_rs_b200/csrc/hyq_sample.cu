// Sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (include/hyq.h states the rule).  Weights and their sums are whole numbers,
// so neither the order of summation nor the split over threads changes a
// token.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstdlib>

#include "../../include/hyq.h"
#include "hyq_common.cuh"
#include "hyq_kernels.h"

namespace hyq {
namespace sample {

using u64 = unsigned long long;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kGrid = 24;              // u and top_p in steps of 2^-24
constexpr float kOne = 1099511627776.0f;  // 2^40: the weight of the largest logit

struct Args {
  const float* logits;
  int64_t stride;
  int n;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* token;
  float* prob;
};

// Ascending order of the logits as an unsigned key: NaN as -inf, -0 as +0.
__device__ __forceinline__ unsigned key_of(float x) {
  if (isnan(x)) x = -INFINITY;
  const unsigned b = __float_as_uint(x == 0.0f ? 0.0f : x);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key);
}

// exp((x - max) / temperature) of a key, at most 1 (exactly 1 at the maximum,
// an infinite one included)
__device__ __forceinline__ float exp_of(unsigned key, unsigned max_key, float max, float inverse) {
  return key == max_key ? 1.0f : expf(__fmul_rn(__fsub_rn(value_of(key), max), inverse));
}
__device__ __forceinline__ u64 weight_of(float e) { return (u64)__fmul_rn(e, kOne); }

// floor(a * m / 2^24) for m <= 2^24 (a below 2^64 / 2^24 in the low part only)
__device__ __forceinline__ u64 scaled(u64 a, u64 m, u64 round) {
  return (a >> kGrid) * m + (((a & ((1u << kGrid) - 1)) * m + round) >> kGrid);
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// ---------------------------------------------------------------------------
// Rows held in shared memory by a cluster of CTAs
// ---------------------------------------------------------------------------
//
// The row is read from memory once, a slice per CTA.  What the CTAs of a row
// tell one another goes through distributed shared memory, one cluster
// barrier per exchange:
//   1. the largest and the smallest logit;
//   2. with top-k or top-p, a histogram of z = (max - logit) / temperature
//      over at most 28 (past it a weight is 0: e^-28 < 2^-40) in 512 equal
//      bins; every CTA adds up all of them and finds the bin in which the
//      k-th logit, or the top_p of the mass, falls;
//   3. the tokens up to that bin, usually a few hundred at most, go to the
//      first CTA of the cluster, which sorts them and finishes the row alone.
// Where they are more than kList (a wide nucleus, ties), the exact cut is
// found over the whole cluster instead: the bin's own tokens, listed in every
// CTA, are ranked by value and index; a bin with too many is divided again by
// the bits of the key, then by index.  Then each CTA adds up its kept mass,
// and the one that holds the draw walks its part.
namespace cluster {

constexpr int kT = 512;                // threads of a CTA
constexpr int kW = kT / 32;
constexpr int kUnit = kT * 4;          // a slice is whole groups of 128 per warp
constexpr int kBins = 512;
static_assert(kBins == kT, "one bin per thread");
constexpr int kList = 2048;            // tokens the first CTA sorts
constexpr int kRanked = 1024;          // tokens ranked pair by pair
constexpr int kMaxCluster = 16;
constexpr int kMaxSlice = 24 * kUnit;  // floats: 192 KB
constexpr float kSpan = 28.0f;

__device__ __forceinline__ unsigned ctarank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned nctas() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The same shared address in CTA `rank`.
__device__ __forceinline__ uint32_t remote(const void* p, unsigned rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(p)), "r"(rank));
  return a;
}
__device__ __forceinline__ void put64(uint32_t a, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(a), "l"(v) : "memory");
}
__device__ __forceinline__ void put32(uint32_t a, unsigned v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(a), "r"(v) : "memory");
}
__device__ __forceinline__ unsigned get32(uint32_t a) {
  unsigned v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

struct Shared {
  // counts, and the masses in parts of 14, 14 and 13 bits (a slice's sums stay
  // below 2^32; shared 32-bit atomics are native, 64-bit ones are not)
  unsigned hist[4][kBins];
  u64 list[kList];              // the order of a part's tokens
  float max_of[kMaxCluster], min_of[kMaxCluster];
  unsigned first_of[kMaxCluster];
  u64 mass_of[kMaxCluster];
  u64 warp_a[kW], warp_b[kW];
  unsigned fill;                // entries of the list so far
  unsigned bin;
  u64 above_n, above_w, in_n;
};
static_assert(2 * kUnit * sizeof(float) >= kList * sizeof(u64), "the masses of a sorted list");
static_assert((u64)kMaxSlice << 14 < 1ull << 32, "sums of 14-bit parts");

// This thread's logits: four at a time, index() + 0 .. 3, in the order of the
// row within a warp.
struct Slice {
  const float* x;  // shared, the warp's part
  int first;       // index in the row of this thread's first four
  int n, groups;
  __device__ __forceinline__ float4 at(int j) const { return reinterpret_cast<const float4*>(x)[32 * j + (threadIdx.x & 31)]; }
  __device__ __forceinline__ int index(int j) const { return first + 128 * j; }
  // f(logit, index) for each
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
    for (int j = 0; j < groups; ++j) {
      const int i = index(j);
      const float4 v = at(j);
      if (i < n) f(v.x, i);
      if (i + 1 < n) f(v.y, i + 1);
      if (i + 2 < n) f(v.z, i + 2);
      if (i + 3 < n) f(v.w, i + 3);
    }
  }
};

struct Scale {
  float max, inverse, bins;
  __device__ __forceinline__ float e(float x) const {
    return x == max ? 1.0f : expf(__fmul_rn(__fsub_rn(x, max), inverse));
  }
  // (max - x) / temperature in bins, to the nearest whole number (the sum with
  // 2^23 rounds it into the low bits): monotone in the logit; kBins and more:
  // no weight.  `bins` carries the 1 / temperature.
  __device__ __forceinline__ unsigned bin(float x) const {
    return __float_as_uint(fminf(__fmul_rn(__fsub_rn(max, x), bins), 4.0f * kBins) + 8388608.0f) & 0x7fffffu;
  }
};

// Order of the tokens: larger logits first, ties by index.
__device__ __forceinline__ u64 order_of(float x, int index) { return ((u64)~key_of(x) << 32) | (unsigned)index; }

// Which part of the row is divided next: all of it by z, or a z bin and leading
// bits of the order, 9 at a time.
struct Part {
  unsigned zbin;
  u64 prefix, mask;
  int shift;  // of the next 9 bits; 64: by z
};

__device__ __forceinline__ unsigned sub_bin(const Scale& sc, const Part& p, float x, int index) {
  const unsigned z = sc.bin(x);
  if (p.shift == 64) return z;
  const u64 order = order_of(x, index);
  if (z != p.zbin || (order & p.mask) != p.prefix) return kBins;
  return (unsigned)(order >> p.shift) & (kBins - 1);
}

// Exclusive sums over the CTA's bins of two values, one bin per thread.
__device__ __forceinline__ void scan2(Shared& sh, u64 a, u64 b, u64& before_a, u64& before_b) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = a, y = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
    if (lane >= o) {
      x += p;
      y += q;
    }
  }
  __syncthreads();
  if (lane == 31) {
    sh.warp_a[warp] = x;
    sh.warp_b[warp] = y;
  }
  __syncthreads();
  before_a = x - a;
  before_b = y - b;
  for (int w = 0; w < warp; ++w) {
    before_a += sh.warp_a[w];
    before_b += sh.warp_b[w];
  }
}

// The cut: the last token kept when the tokens up to `limit` (an earlier cut)
// are cut either to the first `want` (BY_MASS false) or to those whose
// predecessors weigh less than `want`.  Returns its order; `limit` when they
// count or weigh less.
template <bool BY_MASS>
__device__ u64 find_cut(Shared& sh, const Slice& row, const Scale& sc, u64 limit, u64 want) {
  const unsigned rank = ctarank(), ctas = nctas();
  u64 above_n = 0, above_w = 0;  // tokens before the part, their mass
  Part part{0, 0, 0, 64};
  // (8 levels divide a 64-bit order to single tokens; the bound is for safety)
  for (int level = 0; level < 10; ++level) {
    for (int i = threadIdx.x; i < (BY_MASS ? 4 : 1) * kBins; i += kT) (&sh.hist[0][0])[i] = 0;
    if (threadIdx.x == 0) sh.bin = kBins;
    __syncthreads();
    row.each([&](float x, int i) {
      const unsigned b = sub_bin(sc, part, x, i);
      if (b >= kBins || order_of(x, i) > limit) return;
      if constexpr (BY_MASS) {
        const u64 w = weight_of(sc.e(x));
        if (w == 0) return;
        atomicAdd(&sh.hist[1][b], (unsigned)(w & 0x3fff));
        atomicAdd(&sh.hist[2][b], (unsigned)(w >> 14 & 0x3fff));
        atomicAdd(&sh.hist[3][b], (unsigned)(w >> 28));
      }
      atomicAdd(&sh.hist[0][b], 1u);
    });
    barrier();
    u64 count = 0, weight = 0, lower = 0;  // of this thread's bin; its tokens in the CTAs before this one
#pragma unroll 4
    for (unsigned c = 0; c < ctas; ++c) {
      const uint32_t h = remote(&sh.hist[0][threadIdx.x], c);
      const unsigned k = get32(h);
      if (c < rank) lower += k;
      count += k;
      if constexpr (BY_MASS)
        weight += (u64)get32(h + 4 * kBins) + ((u64)get32(h + 8 * kBins) << 14) + ((u64)get32(h + 12 * kBins) << 28);
    }
    u64 before_n, before_w;
    scan2(sh, count, weight, before_n, before_w);
    before_n += above_n;
    before_w += above_w;
    if (BY_MASS ? before_w < want && before_w + weight >= want : before_n < want && before_n + count >= want) {
      sh.bin = threadIdx.x;
      sh.above_n = before_n;
      sh.above_w = before_w;
      sh.in_n = count;
      sh.fill = (unsigned)min(lower, (u64)kRanked);
    }
    __syncthreads();
    const unsigned b = sh.bin;
    if (b == kBins) return limit;  // (at the first level only)
    above_n = sh.above_n;
    above_w = sh.above_w;
    const int m = (int)min(sh.in_n, (u64)kRanked + 1);
    if (m <= kRanked) {
      row.each([&](float x, int i) {
        if (sub_bin(sc, part, x, i) != b) return;
        const u64 order = order_of(x, i);
        if (order > limit || (BY_MASS && weight_of(sc.e(x)) == 0)) return;
        const unsigned slot = atomicAdd(&sh.fill, 1u);
        if (slot < kRanked)
          for (unsigned c = 0; c < ctas; ++c) put64(remote(&sh.list[slot], c), order);
      });
      barrier();
      // place of each of the part's tokens, or the mass before it
      u64 last = 0;
      for (int t = threadIdx.x; t < m; t += kT) {
        const u64 mine = sh.list[t];
        u64 before = BY_MASS ? above_w : above_n;
        for (int j = 0; j < m; ++j) {
          const u64 other = sh.list[j];
          if (other < mine) before += BY_MASS ? weight_of(sc.e(value_of(~(unsigned)(other >> 32)))) : 1;
        }
        if (before < want) last = max(last, mine);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = last;
      __syncthreads();
      for (int w = 0; w < kW; ++w) last = max(last, sh.warp_a[w]);
      __syncthreads();
      return last;
    }
    barrier();  // the histograms are read; divide the part
    if (part.shift == 64) {
      part.zbin = b;
      part.shift = 55;
    } else {
      part.prefix |= (u64)b << part.shift;
      part.mask |= (u64)(kBins - 1) << part.shift;
      part.shift = part.shift >= 9 ? part.shift - 9 : 0;
    }
  }
  return limit;
}

// Mass of the tokens up to `cut` with e >= floor: of this thread's warp and of
// the warps and CTAs before it; returns the row's.
__device__ __forceinline__ u64 mass_upto(Shared& sh, const Slice& row, const Scale& sc, u64 cut, float floor_e,
                                         u64& before, u64& mine) {
  const unsigned rank = ctarank(), ctas = nctas();
  const int warp = threadIdx.x >> 5;
  u64 m = 0;
  row.each([&](float x, int i) {
    if (order_of(x, i) > cut) return;
    const float e = sc.e(x);
    if (e >= floor_e) m += weight_of(e);
  });
  mine = warp_sum_u64(m);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_a[warp] = mine;
  __syncthreads();
  if (threadIdx.x < ctas) {
    m = 0;
    for (int w = 0; w < kW; ++w) m += sh.warp_a[w];
    put64(remote(&sh.mass_of[rank], threadIdx.x), m);
  }
  barrier();
  u64 total = 0;
  before = 0;
  for (unsigned c = 0; c < ctas; ++c) {
    if (c == rank) before = total;
    total += sh.mass_of[c];
  }
  for (int w = 0; w < warp; ++w) before += sh.warp_a[w];
  return total;
}

// Exclusive sum over the CTA of one value per thread; `total` of all.
__device__ __forceinline__ u64 scan1(Shared& sh, u64 a, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 x = a;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 p = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += p;
  }
  __syncthreads();
  if (lane == 31) sh.warp_a[warp] = x;
  __syncthreads();
  u64 before = x - a;
  total = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    if (w == warp) before += total;
    total += sh.warp_a[w];
  }
  return before;
}

// Bitonic sort of list[0 .. n), n a power of two from 64 to kList, ascending,
// by the CTA.  A warp's pairs at distances up to 32 stay inside its own 64
// entries (per 512 threads' turn), so only the longer ones meet at a barrier.
__device__ __forceinline__ void sort_list(u64* list, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int dist = size >> 1; dist > 0; dist >>= 1) {
      if (dist >= 32) __syncthreads();
      else __syncwarp();
      for (int t = threadIdx.x; t < n / 2; t += kT) {
        const int i = 2 * t - (t & (dist - 1)), j = i + dist;
        const u64 a = list[i], b = list[j];
        if ((a > b) == ((i & size) == 0)) {
          list[i] = b;
          list[j] = a;
        }
      }
      if (dist >= 32) __syncthreads();
    }
  __syncthreads();
}

// The rest of a row by one CTA: list[0 .. m) holds the order of every token
// that can be kept.  `k`: keep at most that many; `want`: then those whose
// predecessors weigh less (0: not yet known, top_p of what k keeps).
__device__ void finish(Shared& sh, u64* mass_s, const Scale& sc, const Args& a, int r, int m, int k, u64 want,
                       bool by_mass, u64 share_p, float floor_e) {
  int n = 64;
  while (n < m) n <<= 1;
  for (int t = m + threadIdx.x; t < n; t += kT) sh.list[t] = ~0ull;
  __syncthreads();
  sort_list(sh.list, n);
  // consecutive tokens per thread
  const int per = (n + kT - 1) / kT, t0 = threadIdx.x * per;
  constexpr int kPer = kList / kT;
  u64 w[kPer], mine = 0;
  float e[kPer];
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int t = t0 + q;
    const bool in = q < per && t < m && t < k;
    e[q] = in ? sc.e(value_of(~(unsigned)(sh.list[t] >> 32))) : -1.0f;
    w[q] = in ? weight_of(e[q]) : 0;
    mine += w[q];
  }
  u64 total;
  u64 before = scan1(sh, mine, total);
  if (by_mass && want == 0) want = max(scaled(total, share_p, (1u << kGrid) - 1), 1ull);
  mine = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const u64 v = w[q];
    if (e[q] < floor_e || (by_mass && before >= want)) w[q] = 0;
    before += v;
    mine += w[q];
  }
  __syncthreads();
  // the kept ones in the order of their indexes
#pragma unroll
  for (int q = 0; q < kPer; ++q)
    if (q < per && t0 + q < n) {
      mass_s[t0 + q] = w[q];
      sh.list[t0 + q] = w[q] ? (sh.list[t0 + q] << 32) | (unsigned)(t0 + q) : ~0ull;
    }
  scan1(sh, mine, total);
  sort_list(sh.list, n);
  const float uf = fminf(fmaxf(a.u[r], 0.0f), 1.0f);
  const u64 ui = min((u64)__fmul_rn(uf, 16777216.0f), (u64)(1u << kGrid) - 1);
  const u64 aim = scaled(total, ui, 0);
  mine = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const u64 entry = q < per && t0 + q < n ? sh.list[t0 + q] : ~0ull;
    w[q] = entry == ~0ull ? 0 : mass_s[(unsigned)entry];
    mine += w[q];
  }
  u64 ignored;
  before = scan1(sh, mine, ignored);
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    if (aim >= before && aim < before + w[q]) {
      a.token[r] = (int)(sh.list[t0 + q] >> 32);
      if (a.prob) a.prob[r] = __fdiv_rn((float)w[q], (float)total);
    }
    before += w[q];
  }
}

// The bin up to which the first k logits of the row lie, at least: the k-th
// largest of the threads' own maxima (this CTA alone holds k logits there).
__device__ __forceinline__ unsigned local_bound(Shared& sh, const Scale& sc, float thread_max, int k) {
  sh.hist[0][threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.bin = kBins - 1;
  __syncthreads();
  const unsigned b = sc.bin(thread_max);
  if (b < kBins) atomicAdd(&sh.hist[0][b], 1u);
  __syncthreads();
  const u64 count = sh.hist[0][threadIdx.x];
  u64 total;
  const u64 before = scan1(sh, count, total);
  if (before < (u64)k && before + count >= (u64)k) sh.bin = threadIdx.x;
  __syncthreads();
  const unsigned bound = sh.bin;
  __syncthreads();
  return bound;
}

__global__ void __launch_bounds__(kT) sample_cluster_kernel(const __grid_constant__ Args a, int slice) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ Shared sh;
  extern __shared__ __align__(16) float x_s[];
  const unsigned rank = ctarank(), ctas = nctas();
  const int r = blockIdx.x / ctas, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* x = a.logits + r * a.stride;
  const int share = slice / kW;  // of a warp
  float* mine_s = x_s + warp * share;
  const Slice row{mine_s, (int)rank * slice + warp * share + 4 * lane, a.n, share / 128};
  float top = -INFINITY, low = INFINITY;
  const bool vec = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
#pragma unroll 4
  for (int j = 0; j < row.groups; ++j) {
    const int i = row.index(j);
    float v[4];
    if (vec && i + 4 <= a.n) {
      const float4 f = __ldcs(reinterpret_cast<const float4*>(x + i));
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = i + k < a.n ? __ldcs(x + i + k) : -INFINITY;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (isnan(v[k])) v[k] = -INFINITY;
      top = fmaxf(top, v[k]);
      if (i + k < a.n) low = fminf(low, v[k]);
    }
    reinterpret_cast<float4*>(mine_s)[32 * j + lane] = make_float4(v[0], v[1], v[2], v[3]);
  }
  const float thread_max = top;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  }
  float* warp_max = reinterpret_cast<float*>(sh.warp_a);
  float* warp_min = reinterpret_cast<float*>(sh.warp_b);
  if (lane == 0) {
    warp_max[warp] = top;
    warp_min[warp] = low;
  }
  barrier();  // every CTA of the cluster runs before its shared memory is written to
  if (threadIdx.x < ctas) {
    for (int w = 0; w < kW; ++w) {
      top = fmaxf(top, warp_max[w]);
      low = fminf(low, warp_min[w]);
    }
    put32(remote(&sh.max_of[rank], threadIdx.x), __float_as_uint(top));
    put32(remote(&sh.min_of[rank], threadIdx.x), __float_as_uint(low));
  }
  barrier();
  top = -INFINITY;
  low = INFINITY;
  for (unsigned c = 0; c < ctas; ++c) {
    top = fmaxf(top, sh.max_of[c]);
    low = fminf(low, sh.min_of[c]);
  }
  const float temperature = a.temperature ? a.temperature[r] : 1.0f;
  if (top == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      a.token[r] = 0;
      if (a.prob) a.prob[r] = 0.0f;
    }
    return;
  }
  if (!(temperature > 0.0f)) {  // greedy: the first index of the largest
    unsigned first = 0xffffffffu;
    if (thread_max == top)
      row.each([&](float v, int i) {
        if (v == top) first = min(first, (unsigned)i);
      });
    first = __reduce_min_sync(0xffffffffu, first);
    if (threadIdx.x == 0) sh.fill = 0xffffffffu;
    __syncthreads();
    if (lane == 0) atomicMin(&sh.fill, first);
    __syncthreads();
    if (threadIdx.x == 0) put32(remote(&sh.first_of[rank], 0), sh.fill);
    barrier();
    if (rank == 0 && threadIdx.x == 0) {
      for (unsigned c = 0; c < ctas; ++c) first = min(first, sh.first_of[c]);
      a.token[r] = (int)first;
      if (a.prob) a.prob[r] = 1.0f;
    }
    return;
  }
  float own_max = thread_max;
  if (top == INFINITY) {  // +inf logits share the weight: the others weigh nothing
    for (int j = 0; j < row.groups; ++j) {
      float4& v = reinterpret_cast<float4*>(mine_s)[32 * j + lane];
      v.x = v.x == INFINITY ? 0.0f : -INFINITY;
      v.y = v.y == INFINITY ? 0.0f : -INFINITY;
      v.z = v.z == INFINITY ? 0.0f : -INFINITY;
      v.w = v.w == INFINITY ? 0.0f : -INFINITY;
    }
    own_max = thread_max == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
    low = -INFINITY;
    __syncthreads();
  }
  Scale sc;
  sc.max = top;
  sc.inverse = __fdiv_rn(1.0f, temperature);
  const float span = (top - low) * sc.inverse;
  sc.bins = fminf((kBins - 1) / fminf(fmaxf(span, 1e-20f), kSpan) * sc.inverse, 1e38f);
  const int k = a.top_k ? a.top_k[r] : 0;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  const float floor_e = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;
  const bool by_count = k > 0 && k < a.n, by_mass = p < 1.0f;
  const u64 share_p = by_mass ? (u64)ceilf(__fmul_rn(fmaxf(p, 0.0f), 16777216.0f)) : 0;
  if (by_count || by_mass) {
    const bool weigh = !by_count;  // the bin is chosen by mass
    const unsigned bound = by_count && k <= kT / 2 ? local_bound(sh, sc, own_max, k) : kBins - 1;
    for (int i = threadIdx.x; i < (weigh ? 4 : 1) * kBins; i += kT) (&sh.hist[0][0])[i] = 0;
    if (threadIdx.x == 0) {
      sh.bin = kBins;
      sh.fill = 0;
    }
    __syncthreads();
    if (weigh) {
      row.each([&](float v, int) {
        const unsigned b = sc.bin(v);
        if (b >= kBins) return;
        const u64 w = weight_of(sc.e(v));
        if (w == 0) return;
        atomicAdd(&sh.hist[0][b], 1u);
        atomicAdd(&sh.hist[1][b], (unsigned)(w & 0x3fff));
        atomicAdd(&sh.hist[2][b], (unsigned)(w >> 14 & 0x3fff));
        atomicAdd(&sh.hist[3][b], (unsigned)(w >> 28));
      });
    } else {
      row.each([&](float v, int) {
        const unsigned b = sc.bin(v);
        if (b <= bound) atomicAdd(&sh.hist[0][b], 1u);
      });
    }
    barrier();
    u64 count = 0, weight = 0;
    unsigned lower = 0;
#pragma unroll 4
    for (unsigned c = 0; c < ctas; ++c) {
      const uint32_t h = remote(&sh.hist[0][threadIdx.x], c);
      const unsigned in = get32(h);
      if (c < rank) lower += in;
      count += in;
      if (weigh)
        weight += (u64)get32(h + 4 * kBins) + ((u64)get32(h + 8 * kBins) << 14) + ((u64)get32(h + 12 * kBins) << 28);
    }
    u64 before_n, before_w;
    scan2(sh, count, weight, before_n, before_w);
    u64 want = 0, all = 0;
    if (weigh) {
      for (int w = 0; w < kW; ++w) all += sh.warp_b[w];
      want = max(scaled(all, share_p, (1u << kGrid) - 1), 1ull);
    }
    if (weigh ? before_w < want && before_w + weight >= want : before_n < (u64)k && before_n + count >= (u64)k) {
      sh.bin = threadIdx.x;
      sh.in_n = before_n + count;
    }
    __syncthreads();
    // a row with fewer than k weighty tokens: all of them
    unsigned b = sh.bin;
    u64 listed = b < kBins ? sh.in_n : 0;
    if (b == kBins) {
      b = kBins - 1;
      for (int w = 0; w < kW; ++w) listed += sh.warp_a[w];
    }
    if (listed <= kList) {
      // this CTA's place in the list: the tokens of the CTAs before it
      unsigned mine = threadIdx.x <= b ? lower : 0;
      mine = __reduce_add_sync(0xffffffffu, mine);
      if (lane == 0 && mine) atomicAdd(&sh.fill, mine);
      __syncthreads();
      row.each([&](float v, int i) {
        if (sc.bin(v) > b || (weigh && weight_of(sc.e(v)) == 0)) return;
        const unsigned slot = atomicAdd(&sh.fill, 1u);
        if (slot < kList) put64(remote(&sh.list[slot], 0), order_of(v, i));
      });
      barrier();
      if (rank == 0)
        finish(sh, reinterpret_cast<u64*>(x_s), sc, a, r, (int)listed, by_count ? k : a.n, want, by_mass, share_p, floor_e);
      return;
    }
    barrier();  // the histograms are read
  }
  u64 cut = ~0ull, before, mine;
  if (by_count) cut = find_cut<false>(sh, row, sc, cut, (u64)k);
  if (by_mass) {
    const u64 mass = mass_upto(sh, row, sc, cut, 0.0f, before, mine);
    cut = find_cut<true>(sh, row, sc, cut, max(scaled(mass, share_p, (1u << kGrid) - 1), 1ull));
  }
  const u64 total = mass_upto(sh, row, sc, cut, floor_e, before, mine);
  const float uf = fminf(fmaxf(a.u[r], 0.0f), 1.0f);
  const u64 ui = min((u64)__fmul_rn(uf, 16777216.0f), (u64)(1u << kGrid) - 1);
  const u64 aim = scaled(total, ui, 0);
  if (aim < before || aim >= before + mine) return;
  // this warp holds the token: index order is group by group of 128
  u64 run = before;
  for (int j = 0; j < row.groups; ++j) {
    const float4 f = row.at(j);
    const float v[4] = {f.x, f.y, f.z, f.w};
    u64 w[4], s = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = row.index(j) + q;
      w[q] = 0;
      if (i < a.n && order_of(v[q], i) <= cut) {
        const float e = sc.e(v[q]);
        if (e >= floor_e) w[q] = weight_of(e);
      }
      s += w[q];
    }
    u64 upto = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    u64 at = run + upto - s;
    if (aim >= at && aim < at + s) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (aim >= at && aim < at + w[q]) {
          a.token[r] = row.index(j) + q;
          if (a.prob) a.prob[r] = __fdiv_rn((float)w[q], (float)total);
        }
        at += w[q];
      }
    }
    run += __shfl_sync(0xffffffffu, upto, 31);
    if (aim < run) return;
  }
}

cudaError_t launch(const Args& a, int64_t rows, int ctas, cudaStream_t st) {
  auto k = sample_cluster_kernel;
  // (at least two units: the first CTA keeps kList masses there)
  const int slice = std::max(((a.n + ctas - 1) / ctas + kUnit - 1) / kUnit * kUnit, 2 * kUnit);
  cudaError_t e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxSlice * (int)sizeof(float));
  if (e != cudaSuccess) return e;
  if (ctas > 8 && (e = cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess) return e;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(rows * ctas));
  cfg.blockDim = dim3(kT);
  cfg.dynamicSmemBytes = slice * sizeof(float);
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = launch_overlap() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, a, slice);
}

}  // namespace cluster

// ---------------------------------------------------------------------------
// Rows past what a cluster holds: one CTA per row, every pass reads it again
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ Args a) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ u64 hist[256];
  __shared__ u64 warp_mass[kWarps];
  __shared__ int warp_ties[kWarps];
  __shared__ unsigned max_s;
  __shared__ int first_s;
  __shared__ unsigned sel_key;
  __shared__ u64 sel_rest;
  __shared__ u64 total_s;
  const int row = blockIdx.x, n = a.n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* x = a.logits + row * a.stride;
  if (threadIdx.x == 0) {
    max_s = 0;
    first_s = n;
    total_s = 0;
  }
  __syncthreads();
  unsigned mk = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) mk = max(mk, key_of(x[i]));
  atomicMax(&max_s, __reduce_max_sync(0xffffffffu, mk));
  __syncthreads();
  const unsigned max_key = max_s;
  const float max_x = value_of(max_key);
  const float temperature = a.temperature ? a.temperature[row] : 1.0f;
  if (max_x == -INFINITY || !(temperature > 0.0f)) {
    for (int i = threadIdx.x; i < n; i += kThreads)
      if (key_of(x[i]) == max_key) {
        atomicMin(&first_s, i);
        break;
      }
    __syncthreads();
    if (threadIdx.x == 0) {
      a.token[row] = max_x == -INFINITY ? 0 : first_s;
      if (a.prob) a.prob[row] = max_x == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }
  const float inverse = __fdiv_rn(1.0f, temperature);
  const int k = a.top_k ? a.top_k[row] : 0;
  const float p = a.top_p ? a.top_p[row] : 1.0f;
  const float floor_e = a.min_p ? fminf(a.min_p[row], 1.0f) : 0.0f;
  // kept: keys above `cut`, and the first `ties` (by index) equal to it
  unsigned cut = 0;
  int ties = n;
  if (k > 0 && k < n) {
    // the k-th largest key, eight bits at a time
    unsigned prefix = 0, mask = 0;
    u64 want = k;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256) hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned key = key_of(x[i]);
        if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255], 1ull);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int b = 255;
        u64 above = 0;
        while (b > 0 && above + hist[b] < want) above += hist[b--];
        sel_key = prefix | ((unsigned)b << shift);
        sel_rest = want - above;
      }
      __syncthreads();
      prefix = sel_key;
      want = sel_rest;
      mask |= 255u << shift;
    }
    cut = prefix;
    ties = (int)want;
  }
  if (p < 1.0f) {
    // the total of what top-k keeps, then the key at which the running mass
    // from the top reaches top_p of it
    u64 mass = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const unsigned key = key_of(x[i]);
      if (key > cut) mass += weight_of(exp_of(key, max_key, max_x, inverse));
    }
    mass = warp_sum_u64(mass);
    if (lane == 0) atomicAdd(&total_s, mass);
    __syncthreads();
    const u64 tie_mass = cut ? ties * weight_of(exp_of(cut, max_key, max_x, inverse)) : 0;
    const u64 total = total_s + tie_mass;
    const u64 share = (u64)ceilf(__fmul_rn(fmaxf(p, 0.0f), 16777216.0f));
    u64 want = scaled(total, share, (1u << kGrid) - 1);
    if (want == 0) want = 1;
    unsigned prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (threadIdx.x < 256) hist[threadIdx.x] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned key = key_of(x[i]);
        if (key > cut && (key & mask) == prefix)
          atomicAdd(&hist[(key >> shift) & 255], weight_of(exp_of(key, max_key, max_x, inverse)));
      }
      if (threadIdx.x == 0 && (cut & mask) == prefix && tie_mass) atomicAdd(&hist[(cut >> shift) & 255], tie_mass);
      __syncthreads();
      if (threadIdx.x == 0) {
        int b = 255;
        u64 above = 0;
        while (b > 0 && above + hist[b] < want) above += hist[b--];
        sel_key = prefix | ((unsigned)b << shift);
        sel_rest = want - above;
      }
      __syncthreads();
      prefix = sel_key;
      want = sel_rest;
      mask |= 255u << shift;
    }
    // ties at the key: as many as still start below the limit
    const u64 each = weight_of(exp_of(prefix, max_key, max_x, inverse));
    const u64 take = (want + each - 1) / each;
    ties = prefix == cut ? (int)min((u64)ties, take) : (int)min((u64)n, take);
    cut = prefix;
  }
  // kept weights, a contiguous share of the row per warp
  const float cut_e = exp_of(cut, max_key, max_x, inverse);
  const u64 cut_w = cut_e >= floor_e ? weight_of(cut_e) : 0;
  const int share = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
  const int i0 = min(n, warp * share), i1 = min(n, i0 + share);
  u64 mass = 0;
  int tied = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const unsigned key = key_of(x[i]);
    if (key > cut) {
      const float e = exp_of(key, max_key, max_x, inverse);
      if (e >= floor_e) mass += weight_of(e);
    } else if (key == cut) {
      ++tied;
    }
  }
  mass = warp_sum_u64(mass);
  tied = __reduce_add_sync(0xffffffffu, tied);
  if (lane == 0) {
    warp_mass[warp] = mass;
    warp_ties[warp] = tied;
  }
  __syncthreads();
  // every warp: kept mass and ties before its share, and the total
  int my_ties = warp_ties[lane], before_ties = my_ties;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, before_ties, o);
    if (lane >= o) before_ties += y;
  }
  before_ties -= my_ties;
  const int kept_ties = max(0, min(my_ties, ties - before_ties));
  u64 w = warp_mass[lane] + kept_ties * cut_w, upto = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 y = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += y;
  }
  const u64 total = __shfl_sync(0xffffffffu, upto, 31);
  const float uf = fminf(fmaxf(a.u[row], 0.0f), 1.0f);
  const u64 ui = min((u64)__fmul_rn(uf, 16777216.0f), (u64)(1u << kGrid) - 1);
  const u64 aim = scaled(total, ui, 0);
  const u64 start = __shfl_sync(0xffffffffu, upto - w, warp), mine = __shfl_sync(0xffffffffu, w, warp);
  if (aim < start || aim >= start + mine) return;
  // this warp holds the token: walk its share
  u64 run = start;
  int seen = __shfl_sync(0xffffffffu, before_ties, warp);
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const unsigned key = i < i1 ? key_of(x[i]) : 0;
    const unsigned tied_lanes = __ballot_sync(0xffffffffu, i < i1 && key == cut);
    u64 v = 0;
    if (i < i1 && key > cut) {
      const float e = exp_of(key, max_key, max_x, inverse);
      if (e >= floor_e) v = weight_of(e);
    } else if (i < i1 && key == cut && seen + __popc(tied_lanes & ((1u << lane) - 1)) < ties) {
      v = cut_w;
    }
    u64 s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, run + s > aim);
    if (hit) {
      if (lane == __ffs(hit) - 1) {
        a.token[row] = i;
        if (a.prob) a.prob[row] = __fdiv_rn((float)v, (float)total);
      }
      return;
    }
    run += __shfl_sync(0xffffffffu, s, 31);
    seen += __popc(tied_lanes);
  }
}

}  // namespace sample
}  // namespace hyq

extern "C" {

int hyq_sample(const float* logits, int64_t n, int64_t stride, int64_t rows, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
               float* prob, void* stream) {
  const char* name = "sample";
  if (n <= 0 || n >= 1 << 23 || rows < 0 || rows > INT32_MAX || stride < n)
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape (1 to 8388607 logits a row)", name);
  if (rows == 0) return HYQ_OK;
  if (!logits || !u || !token) return hyq::api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  for (const void* p : {(const void*)logits, (const void*)temperature, (const void*)top_k, (const void*)top_p,
                        (const void*)min_p, (const void*)u, (const void*)token, (const void*)prob})
    if (reinterpret_cast<uintptr_t>(p) % 4)
      return hyq::api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  const hyq::sample::Args a{logits, stride, (int)n, temperature, top_k, top_p, min_p, u, token, prob};
  const cudaStream_t st = (cudaStream_t)stream;
  namespace sc = hyq::sample::cluster;
  cudaError_t e;
  static const char* tune = getenv("HYQ_TUNE_C");
  const int want = tune ? atoi(tune) : 8;
  const int ctas = (int)std::max<int64_t>(std::min<int64_t>(want, (n + sc::kUnit - 1) / sc::kUnit), (n + sc::kMaxSlice - 1) / sc::kMaxSlice);
  if (ctas <= sc::kMaxCluster && rows <= INT32_MAX / sc::kMaxCluster)
    e = sc::launch(a, rows, ctas, st);
  else
    e = hyq::launch_ex(hyq::sample::sample_kernel, dim3((unsigned)rows), dim3(hyq::sample::kThreads), 0, st, a);
  return e == cudaSuccess ? HYQ_OK : hyq::api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

}  // extern "C"
