// Sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (include/hyq.h states the rule).  Weights and their sums are whole numbers,
// so neither the order of summation nor the split over threads changes a
// token.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/hyq.h"
#include "hyq_common.cuh"
#include "hyq_kernels.h"

namespace hyq {
namespace sample {

using u64 = unsigned long long;

constexpr int kGrid = 24;              // u and top_p in steps of 2^-24

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

// floor(2^40 e) of 0 <= e <= 1 without 64-bit arithmetic or conversions: e 2^20
// is split at the nearest whole number, both parts read from the low bits of a
// sum with 2^23 or 1.5 2^23; the second is rounded down, so that the pair is
// exact.
constexpr unsigned kHighBase = 0x4b000000u, kLowBase = 0x4b400000u;
__device__ __forceinline__ void weight_parts(float e, unsigned& high, unsigned& low) {
  const float t = __fmul_rn(e, 1048576.0f), h = __fadd_rn(t, 8388608.0f);
  high = __float_as_uint(h);
  low = __float_as_uint(__fmaf_rd(__fsub_rn(t, __fsub_rn(h, 8388608.0f)), 1048576.0f, 12582912.0f));
}
__device__ __forceinline__ u64 weight_of(float e) {
  unsigned high, low;
  weight_parts(e, high, low);
  return (u64)((int64_t)(int)(high - kHighBase) * (1 << 20) + (int)(low - kLowBase));
}
// A sum of weights: the parts' own bits are added up, and their bases taken out
// every 2,048 terms at most (4,095 would still fit).
struct WeightSum {
  unsigned high = 0, low = 0, terms = 0;
  u64 whole = 0;
  __device__ __forceinline__ void add(float e) {
    unsigned h, l;
    weight_parts(e, h, l);
    high += h;
    low += l;
  }
  __device__ __forceinline__ void added(unsigned n) {
    terms += n;
    if (terms >= 2048) flush();
  }
  __device__ __forceinline__ void flush() {
    whole += (u64)((int64_t)(high - terms * kHighBase) * (1 << 20) + (int)(low - terms * kLowBase));
    high = low = terms = 0;
  }
};

// floor(a * m / 2^24) for m <= 2^24 (a below 2^64 / 2^24 in the low part only)
__device__ __forceinline__ u64 scaled(u64 a, u64 m, u64 round) {
  return (a >> kGrid) * m + (((a & ((1u << kGrid) - 1)) * m + round) >> kGrid);
}

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row is worked on by a cluster of CTAs, a slice each.  With few rows the
// slices are staged in shared memory (the row is read from memory once and
// the passes below read it from there); with many, or a row too long for
// that, each pass reads them from memory again, and a greedy row or one with a
// top-k of up to kDirect has one CTA, in a launch of its own.  What the CTAs of
// a row tell one another goes through distributed shared memory, one cluster
// barrier per exchange:
//   1. the largest and the smallest logit;
//   2. with top-k, a bound from the threads' own maxima; one CTA alone then
//      takes the tokens up to it (step 4).  Several, or a top-k past kDirect: a
//      histogram of z = (max - logit) / temperature over at most 28 (past it a
//      weight is 0: e^-28 < 2^-40) in 512 equal bins; every CTA adds up all of
//      them and finds the bin in which the k-th logit falls;
//   3. with top-p alone, the masses of sixteen ranges of z, then the histogram,
//      with masses, of the one in which the top_p of the mass falls;
//   4. the tokens up to that bin, usually a few hundred at most, go to the
//      first CTA of the cluster, which finds the cuts among them and finishes
//      the row alone.
// Where they are more than kList (a wide nucleus, ties), the exact cut is
// found over the whole cluster instead: the bin's own tokens, listed in every
// CTA, are sorted by value and index; a bin with too many is divided again by
// the bits of the key, then by index.  Then each CTA adds up its kept mass,
// and the one that holds the draw walks its part.
//
// What bounds it: one row is latency (14 us for 0.5 MB: a handful of exchanges
// and scans); many rows, the passes over them: 256 rows of 120,832 logits (124
// MB) take 24 us greedy (one pass, 5.2 TB/s), 47 us with top-k 40 (two), 92 us
// without filters (two, 31 M exponentials), 187 us with top-p 0.9 at 0.7 (four)
// and 300 us at 1.0 (six: the nucleus is 14,000 tokens wide).

constexpr int kT = 512;                // threads of a CTA
constexpr int kW = kT / 32;
constexpr int kUnit = kT * 4;          // a slice is whole groups of 128 per warp
constexpr int kBins = 512;
static_assert(kBins == kT, "one bin per thread");
constexpr int kList = 2048;            // tokens the first CTA sorts
constexpr int kMaxCluster = 16;
constexpr int kMaxSlice = 16 * kUnit;  // floats: 128 KB
constexpr float kSpan = 28.0f;
constexpr int kCoarse = 16;            // ranges of bins (with one or the other shift)
constexpr int kFine = kCoarse * kBins;
static_assert(kCoarse == kW, "a warp adds up a range");

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
// All threads of the row's `ctas`.
__device__ __forceinline__ void barrier(unsigned ctas) {
  if (ctas == 1) {
    __syncthreads();
    return;
  }
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
__device__ __forceinline__ u64 get64(uint32_t a) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(a) : "memory");
  return v;
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
  u64 range_of[kMaxCluster][kCoarse], range[kCoarse];
  unsigned fill;                // entries of the list so far
  int bin;
  unsigned lower_in, above;     // above: this CTA's tokens before the bins
  u64 above_n, above_w, in_n;
};
// Logits of a slice up to which the sums of 14-bit parts stay below 2^32;
// past it (one CTA, a longer row) the masses are 64-bit atomics.
constexpr int kPartMax = 1 << 18;

// This thread's logits: four at a time, index() + 0 .. 3, in the order of the
// row within a warp; -inf past the row's end (no weight, past every bin).  NaN
// stays: it fails every comparison, falls past the bins and weighs nothing.
// With `infinite` (the row has a +inf), +inf reads as 0 and the rest as -inf,
// so that the infinite ones share the weight.
template <bool STAGED>
struct Slice {
  const float* x;  // STAGED: shared, the warp's part; else the row
  int first;       // index in the row of this thread's first four
  int n, groups;
  bool vec, infinite;
  unsigned ctas;   // that share the row
  __device__ __forceinline__ int index(int j) const { return first + 128 * j; }
  __device__ __forceinline__ float4 from_memory(const float* row, int j) const {
    const int i = index(j);
    if (vec && i + 4 <= n) return __ldg(reinterpret_cast<const float4*>(row + i));
    float4 v;
    v.x = i < n ? __ldg(row + i) : -INFINITY;
    v.y = i + 1 < n ? __ldg(row + i + 1) : -INFINITY;
    v.z = i + 2 < n ? __ldg(row + i + 2) : -INFINITY;
    v.w = i + 3 < n ? __ldg(row + i + 3) : -INFINITY;
    return v;
  }
  __device__ __forceinline__ float4 only_infinite(float4 v) const {
    return make_float4(v.x == INFINITY ? 0.0f : -INFINITY, v.y == INFINITY ? 0.0f : -INFINITY,
                       v.z == INFINITY ? 0.0f : -INFINITY, v.w == INFINITY ? 0.0f : -INFINITY);
  }
  __device__ __forceinline__ float4 load(int j) const {
    if constexpr (STAGED) return reinterpret_cast<const float4*>(x)[32 * j + (threadIdx.x & 31)];
    else return from_memory(x, j);
  }
  __device__ __forceinline__ float4 at(int j) const {
    const float4 v = load(j);
    return infinite ? only_infinite(v) : v;
  }
  // groups j0 .. j0 + N - 1, all loads issued before any value is used
  template <int N>
  __device__ __forceinline__ void batch(int j0, float4 (&v)[N]) const {
    if (!STAGED && vec && j0 + N <= groups && index(j0 + N - 1) + 4 <= n) {
#pragma unroll
      for (int q = 0; q < N; ++q)
        asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(v[q].x), "=f"(v[q].y), "=f"(v[q].z), "=f"(v[q].w)
                     : "l"(x + index(j0 + q)));
    } else {
#pragma unroll
      for (int q = 0; q < N; ++q)
        v[q] = j0 + q < groups ? load(j0 + q) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
    }
  }
  // f(four logits, index of the first), with several loads in flight
  template <typename F>
  __device__ __forceinline__ void groups_of_4(F f) const {
    constexpr int AHEAD = STAGED ? 2 : 4;
    for (int j0 = 0; j0 < groups; j0 += AHEAD) {
      float4 v[AHEAD];
      batch(j0, v);
      if (infinite) {
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) v[q] = only_infinite(v[q]);
      }
#pragma unroll
      for (int q = 0; q < AHEAD; ++q) f(v[q], index(j0 + q));
    }
  }
  // f(logit, index) for those of the groups that reach `least`
  template <typename F>
  __device__ __forceinline__ void each_from(float least, F f) const {
    groups_of_4([&](float4 v, int i) {
      if (fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least) {
        f(v.x, i);
        f(v.y, i + 1);
        f(v.z, i + 2);
        f(v.w, i + 3);
      }
    });
  }
  // put(slot, logit, index) for those of the groups that reach `least` and
  // satisfy f(logit, index); slots count up from `fill`, one addition to it per
  // warp and group.
  template <typename F, typename P>
  __device__ __forceinline__ void collect(float least, unsigned* fill, F f, P put) const {
    const int lane = threadIdx.x & 31;
    groups_of_4([&](float4 v, int i) {
      if (!__any_sync(0xffffffffu, fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least)) return;
      const bool in[4] = {f(v.x, i), f(v.y, i + 1), f(v.z, i + 2), f(v.w, i + 3)};
      const unsigned own = in[0] + in[1] + in[2] + in[3];
      unsigned upto = own;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      unsigned slot = 0;
      if (lane == 31 && upto) slot = atomicAdd(fill, upto);
      slot = __shfl_sync(0xffffffffu, slot, 31) + upto - own;
      if (in[0]) put(slot++, v.x, i);
      if (in[1]) put(slot++, v.y, i + 1);
      if (in[2]) put(slot++, v.z, i + 2);
      if (in[3]) put(slot++, v.w, i + 3);
    });
  }
};

// The tokens kept so far: those up to logit x, and of that logit up to index i.
struct Cut {
  float x;
  int i;
  __device__ __forceinline__ bool keeps(float v, int at) const { return v > x || (v == x && at <= i); }
  __device__ __forceinline__ bool all() const { return x == -INFINITY && i == INT32_MAX; }
};

struct Scale {
  float max, inverse, bins;
  int base, shift;  // bins of 2^shift steps from `base` on
  __device__ __forceinline__ float e(float x) const {
    return fmaxf(expf(__fmul_rn(__fsub_rn(x, max), inverse)), 0.0f);  // (0 for NaN)
  }
  // a logit below which every bin is past `b` (two bins of slack for rounding)
  __device__ __forceinline__ float least(int b) const {
    return max - (float)((base + b + 2) << shift) / bins * 1.0001f;
  }
  // (max - x) / temperature in 2^13 steps over the span, to the nearest whole
  // number (the sum with 2^23 rounds it into the low bits): monotone in the
  // logit; kFine and more: no weight.  `bins` carries the 1 / temperature.
  __device__ __forceinline__ unsigned fine(float x) const {
    return __float_as_uint(fminf(__fmul_rn(__fsub_rn(max, x), bins), 4.0f * kFine) + 8388608.0f) & 0x7fffffu;
  }
  // the bin of the range that is looked at: below 0 before it, kBins and more
  // past it
  __device__ __forceinline__ int bin(float x) const { return (int)(fine(x) >> shift) - base; }
};

// Order of the tokens: larger logits first, ties by index.
__device__ __forceinline__ u64 order_of(float x, int index) { return ((u64)~key_of(x) << 32) | (unsigned)index; }

// Which part of the row is divided next: all of it by z, or a z bin and leading
// bits of the order, 9 at a time.
struct Part {
  int zbin;
  u64 prefix, mask;
  int shift;  // of the next 9 bits; 64: by z
};

__device__ __forceinline__ int sub_bin(const Scale& sc, const Part& p, float x, int index) {
  const int z = sc.bin(x);
  if (p.shift == 64) return z;
  const u64 order = order_of(x, index);
  if (z != p.zbin || (order & p.mask) != p.prefix) return kBins;
  return (int)(order >> p.shift) & (kBins - 1);
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

// Bitonic sort of kT P values, P consecutive ones per thread (P 2 or 4),
// ascending: distances inside a thread in registers, inside a warp by
// shuffles, past it through `buffer` (kT P values of shared memory).
template <int P>
__device__ __forceinline__ void sort_values(u64 (&v)[P], u64* buffer) {
  const int p0 = threadIdx.x * P;
#pragma unroll 1
  for (int size = 2; size <= kT * P; size <<= 1)
#pragma unroll 1
    for (int dist = size >> 1; dist > 0; dist >>= 1) {
      const bool up = (p0 & size) == 0;
      if (dist >= 32 * P) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < P; ++q) buffer[p0 + q] = v[q];
        __syncthreads();
        const bool low = (p0 & dist) == 0;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const u64 other = buffer[(p0 + q) ^ dist];
          v[q] = (low == up) == (other < v[q]) ? other : v[q];
        }
      } else if (dist >= P) {
        const bool low = (p0 & dist) == 0;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const u64 other = __shfl_xor_sync(0xffffffffu, v[q], dist / P);
          v[q] = (low == up) == (other < v[q]) ? other : v[q];
        }
      } else {
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const int o = dist == 1 ? (q ^ 1) : (q ^ 2) % P;
          if (o > q) {
            const bool rising = size < P ? ((p0 + q) & size) == 0 : up;
            const u64 a = v[q], b = v[o];
            if ((b < a) == rising) {
              v[q] = b;
              v[o] = a;
            }
          }
        }
      }
    }
  __syncthreads();
}
// Sorts the m entries of the list, into the list, ~0 past them.
template <int P>
__device__ __forceinline__ void sort_list(Shared& sh, int m) {
  u64 v[P];
  const int p0 = threadIdx.x * P;
#pragma unroll
  for (int q = 0; q < P; ++q) v[q] = p0 + q < m ? sh.list[p0 + q] : ~0ull;
  sort_values<P>(v, sh.list);
#pragma unroll
  for (int q = 0; q < P; ++q) sh.list[p0 + q] = v[q];
  __syncthreads();
}
// Up to this many tokens are compared pair by pair, which costs less than a
// sort's 45 rounds (m^2 / 512 comparisons a thread).
constexpr int kPairs = 256;
__device__ __forceinline__ void sort_tokens(Shared& sh, int m) {
  if (m <= kPairs) {
    const u64 mine = (int)threadIdx.x < m ? sh.list[threadIdx.x] : ~0ull;
    int place = 0;
    if ((int)threadIdx.x < m)
      for (int j = 0; j < m; ++j) place += sh.list[j] < mine;
    __syncthreads();
    if ((int)threadIdx.x < m) sh.list[place] = mine;
    else if (threadIdx.x < 2 * kT) sh.list[threadIdx.x] = ~0ull;
    __syncthreads();
  } else if (m <= 2 * kT) {
    sort_list<2>(sh, m);
  } else {
    sort_list<4>(sh, m);
  }
}

constexpr int kPer = kList / kT;  // tokens of a sorted list per thread

// Where a cut falls: bin `b` of a part, the tokens and the mass before it, its
// own tokens, and this CTA's place among them (of the bin, of all up to it).
struct Found {
  int b;
  u64 above_n, above_w, in_n, want;
  unsigned lower_in, lower_upto;
};

// For a cut by mass of a whole row: the sixteenth of the span in which it
// falls becomes the scale's bins, so that only the tokens there go into
// locate()'s histogram (its shared-memory atomics cost more than the
// exponentials).  The sums are each thread's own, in shared memory at `own`
// (kCoarse x kT), and need no atomics.  Returns the mass before the range; want:
// `share` of the row's.
template <bool STAGED>
__device__ u64 coarse_range(Shared& sh, const Slice<STAGED>& row, Scale& sc, u64* own, u64 share, u64& want) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned rank = ctarank(), ctas = row.ctas;
#pragma unroll
  for (int j = 0; j < kCoarse; ++j) own[j * kT + threadIdx.x] = 0;
  row.groups_of_4([&](float4 v, int) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w;
      const unsigned j = sc.fine(x) / kBins;
      if (j < kCoarse) own[j * kT + threadIdx.x] += weight_of(sc.e(x));
    }
  });
  __syncthreads();
  u64 m = 0;
#pragma unroll
  for (int q = 0; q < kT / 32; ++q) m += own[warp * kT + 32 * q + lane];
  m = warp_sum_u64(m);
  if (lane < ctas) put64(remote(&sh.range_of[rank][warp], lane), m);
  barrier(row.ctas);
  if (threadIdx.x < kCoarse) {
    m = 0;
    for (unsigned c = 0; c < ctas; ++c) m += sh.range_of[c][threadIdx.x];
    sh.range[threadIdx.x] = m;
  }
  __syncthreads();
  u64 total = 0, before = 0;
#pragma unroll
  for (int j = 0; j < kCoarse; ++j) total += sh.range[j];
  want = max(scaled(total, share, (1u << kGrid) - 1), 1ull);
  int j = 0;
  while (j < kCoarse - 1 && before + sh.range[j] < want) before += sh.range[j++];
  sc.base = j * kBins;
  sc.shift = 0;
  return before;
}

// Finds the bin of `part` in which token number `want`, or (BY_MASS) the
// `want`-th unit of mass, falls, among the tokens up to `limit`.  b = kBins:
// there are fewer.  Bins past `bound` are known not to matter.
template <bool BY_MASS, bool STAGED>
__device__ Found locate(Shared& sh, const Slice<STAGED>& row, const Scale& sc, const Part& part, Cut limit, u64 want,
                        u64 above_n, u64 above_w, int bound) {
  const unsigned rank = ctarank(), ctas = row.ctas;
  for (int i = threadIdx.x; i < (BY_MASS ? 4 : 1) * kBins; i += kT) (&sh.hist[0][0])[i] = 0;
  if (threadIdx.x == 0) {
    sh.bin = kBins;
    sh.fill = 0;
    sh.above = 0;
  }
  __syncthreads();
  const bool all = part.shift == 64 && limit.all();
  unsigned over = 0;  // tokens before the bins
  row.each_from(sc.least(bound), [&](float x, int i) {
    const int b = all ? sc.bin(x) : sub_bin(sc, part, x, i);
    if (b > bound || (!all && !limit.keeps(x, i))) return;
    if (BY_MASS && b < 0) {
      ++over;
      return;
    }
    if constexpr (BY_MASS) {
      const u64 w = weight_of(sc.e(x));
      if (w == 0) return;
      if (row.groups * (128 * kW) <= kPartMax) {
        atomicAdd(&sh.hist[1][b], (unsigned)(w & 0x3fff));
        atomicAdd(&sh.hist[2][b], (unsigned)(w >> 14 & 0x3fff));
        atomicAdd(&sh.hist[3][b], (unsigned)(w >> 28));
      } else {
        atomicAdd(reinterpret_cast<u64*>(&sh.hist[2][0]) + b, w);
      }
    }
    atomicAdd(&sh.hist[0][b], 1u);
  });
  if constexpr (BY_MASS) {
    over = __reduce_add_sync(0xffffffffu, over);
    if ((threadIdx.x & 31) == 0 && over) atomicAdd(&sh.above, over);
  }
  barrier(row.ctas);
  u64 count = 0, weight = 0;
  unsigned lower_over = 0;
  unsigned lower = 0;  // tokens of this thread's bin in the CTAs before this one
#pragma unroll 4
  for (unsigned c = 0; c < ctas; ++c) {
    const uint32_t h = remote(&sh.hist[0][threadIdx.x], c);
    const unsigned in = get32(h);
    if (c < rank) lower += in;
    count += in;
    if constexpr (BY_MASS) {
      over = get32(remote(&sh.above, c));
      if (c < rank) lower_over += over;
      above_n += over;
    }
    if constexpr (BY_MASS) {
      if (row.groups * (128 * kW) <= kPartMax)
        weight += (u64)get32(h + 4 * kBins) + ((u64)get32(h + 8 * kBins) << 14) + ((u64)get32(h + 12 * kBins) << 28);
      else
        weight += get64(remote(reinterpret_cast<u64*>(&sh.hist[2][0]) + threadIdx.x, c));
    }
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
    sh.lower_in = lower;
  }
  __syncthreads();
  Found f;
  f.b = sh.bin;
  f.want = want;
  if (f.b == kBins) {
    f.above_n = above_n;
    for (int w = 0; w < kW; ++w) f.above_n += sh.warp_a[w];
    f.above_w = f.in_n = 0;
    f.lower_in = 0;
  } else {
    f.above_n = sh.above_n;
    f.above_w = sh.above_w;
    f.in_n = sh.in_n;
    f.lower_in = sh.lower_in;
  }
  unsigned mine = (int)threadIdx.x < f.b ? lower : 0;
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && mine) atomicAdd(&sh.fill, mine);
  __syncthreads();
  f.lower_upto = sh.fill + f.lower_in + lower_over;
  __syncthreads();
  return f;
}

// The exact cut inside a bin that locate() found.
template <bool BY_MASS, bool STAGED>
__device__ Cut resolve(Shared& sh, const Slice<STAGED>& row, const Scale& sc, Found f, Cut limit) {
  const unsigned ctas = row.ctas;
  Part part{0, 0, 0, 64};
  // (8 levels divide a 64-bit order to single tokens; the bound is for safety)
  for (int level = 0; level < 10 && f.b < kBins; ++level) {
    if (f.in_n <= kList) {
      const int m = (int)f.in_n;
      if (threadIdx.x == 0) sh.fill = f.lower_in;
      __syncthreads();
      row.collect(
          sc.least(part.shift == 64 ? f.b : part.zbin), &sh.fill,
          [&](float x, int i) {
            return sub_bin(sc, part, x, i) == f.b && limit.keeps(x, i) && (!BY_MASS || weight_of(sc.e(x)) != 0);
          },
          [&](unsigned slot, float x, int i) {
            if (slot < kList)
              for (unsigned c = 0; c < ctas; ++c) put64(remote(&sh.list[slot], c), order_of(x, i));
          });
      barrier(row.ctas);
      sort_tokens(sh, m);
      const int per = (m + kT - 1) / kT, t0 = threadIdx.x * per;
      u64 w[kPer], mine = 0, total, last = 0;
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        const bool in = q < per && t0 + q < m;
        w[q] = !in ? 0 : BY_MASS ? weight_of(sc.e(value_of(~(unsigned)(sh.list[t0 + q] >> 32)))) : 1;
        mine += w[q];
      }
      u64 before = scan1(sh, mine, total) + (BY_MASS ? f.above_w : f.above_n);
#pragma unroll
      for (int q = 0; q < kPer; ++q) {
        if (w[q] && before < f.want) last = sh.list[t0 + q];  // ascending
        before += w[q];
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
      __syncthreads();
      if ((threadIdx.x & 31) == 0) sh.warp_a[threadIdx.x >> 5] = last;
      __syncthreads();
      for (int v = 0; v < kW; ++v) last = max(last, sh.warp_a[v]);
      __syncthreads();
      return Cut{value_of(~(unsigned)(last >> 32)), (int)(unsigned)last};
    }
    barrier(row.ctas);  // the histograms are read; divide the bin
    if (part.shift == 64) {
      part.zbin = f.b;
      part.shift = 55;
    } else {
      part.prefix |= (u64)f.b << part.shift;
      part.mask |= (u64)(kBins - 1) << part.shift;
      part.shift = part.shift >= 9 ? part.shift - 9 : 0;
    }
    f = locate<BY_MASS>(sh, row, sc, part, limit, f.want, f.above_n, f.above_w, kBins - 1);
  }
  return limit;  // fewer, or lighter, than what is wanted: all
}

// Mass of the tokens up to `cut` with e >= floor: of this thread's warp and of
// the warps and CTAs before it; returns the row's.
template <bool STAGED>
__device__ __forceinline__ u64 mass_upto(Shared& sh, const Slice<STAGED>& row, const Scale& sc, Cut cut, float floor_e,
                                         u64& before, u64& mine) {
  const unsigned rank = ctarank(), ctas = row.ctas;
  const int warp = threadIdx.x >> 5;
  u64 m;
  WeightSum sum;
  const bool all = cut.all();
  row.groups_of_4([&](float4 v, int i) {
    if (!all && !(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= cut.x)) return;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x = k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w, e = sc.e(x);
      sum.add(e >= floor_e && (all || cut.keeps(x, i + k)) ? e : 0.0f);
    }
    sum.added(4);
  });
  sum.flush();
  mine = warp_sum_u64(sum.whole);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.warp_a[warp] = mine;
  __syncthreads();
  if (threadIdx.x < ctas) {
    m = 0;
    for (int w = 0; w < kW; ++w) m += sh.warp_a[w];
    put64(remote(&sh.mass_of[rank], threadIdx.x), m);
  }
  barrier(row.ctas);
  u64 total = 0;
  before = 0;
  for (unsigned c = 0; c < ctas; ++c) {
    if (c == rank) before = total;
    total += sh.mass_of[c];
  }
  for (int w = 0; w < warp; ++w) before += sh.warp_a[w];
  return total;
}

// The unit of a row's mass that is drawn.
__device__ __forceinline__ u64 aim_of(const Args& a, int r, u64 total) {
  const float uf = fminf(fmaxf(a.u[r], 0.0f), 1.0f);
  return scaled(total, min((u64)__fmul_rn(uf, 16777216.0f), (u64)(1u << kGrid) - 1), 0);
}
__device__ __forceinline__ u64 weight_in(const Shared& sh, int b) {
  return (u64)sh.hist[1][b] + ((u64)sh.hist[2][b] << 14) + ((u64)sh.hist[3][b] << 28);
}
__device__ __forceinline__ void add_weight(Shared& sh, int b, u64 w) {
  atomicAdd(&sh.hist[1][b], (unsigned)(w & 0x3fff));
  atomicAdd(&sh.hist[2][b], (unsigned)(w >> 14 & 0x3fff));
  atomicAdd(&sh.hist[3][b], (unsigned)(w >> 28));
}

// finish() without sorting, for more than kPairs tokens: the cuts' bins from a
// histogram of the list, the cuts themselves by comparing the tokens of one bin;
// then the masses of 512 ranges of indexes, and the tokens of the one that
// holds the draw.  False, with nothing done, if a bin has more than kPairs.
__device__ bool finish_by_bins(Shared& sh, u64* few, const Scale& sc, const Args& a, int r, int m, int k, u64 want,
                               bool by_mass, u64 share_p, float floor_e) {
  u64* few_w = few + kList;
  u64 order[kPer], w[kPer];
  int bin[kPer];
  for (int i = threadIdx.x; i < 4 * kBins; i += kT) (&sh.hist[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const int t = threadIdx.x + q * kT;
    order[q] = t < m ? sh.list[t] : ~0ull;
    w[q] = 0;
    bin[q] = kBins;
    if (t < m) {
      const float x = value_of(~(unsigned)(order[q] >> 32));
      w[q] = weight_of(sc.e(x));
      bin[q] = min((int)(sc.fine(x) / kCoarse), kBins - 1);
      atomicAdd(&sh.hist[0][bin[q]], 1u);
      add_weight(sh, bin[q], w[q]);
    }
  }
  __syncthreads();
  const u64 count = sh.hist[0][threadIdx.x], weight = weight_in(sh, threadIdx.x);
  u64 before_n, before_w;
  scan2(sh, count, weight, before_n, before_w);
  u64 total = 0;
  for (int i = 0; i < kW; ++i) total += sh.warp_b[i];
  // tokens of the bin that thread `at` found, and their number
  auto gather = [&](bool at, u64 cut) {
    if (threadIdx.x == 0) sh.fill = 0;
    if (at) {
      sh.bin = threadIdx.x;
      sh.above_n = before_n;
      sh.above_w = before_w;
    }
    __syncthreads();
    const int b = sh.bin;
#pragma unroll
    for (int q = 0; q < kPer; ++q)
      if (bin[q] == b && order[q] <= cut) {
        const unsigned slot = atomicAdd(&sh.fill, 1u);
        few[slot] = order[q];
        few_w[slot] = w[q];
      }
    __syncthreads();
    return (int)sh.fill;
  };
  u64 cut = ~0ull;  // the last token that is kept
  if (k < m) {
    const int n = gather(before_n < (u64)k && before_n + count >= (u64)k, cut);
    if (n > kPairs) return false;
    if ((int)threadIdx.x < n) {
      u64 lighter = 0;
      int place = (int)sh.above_n;
      for (int j = 0; j < n; ++j)
        if (few[j] < few[threadIdx.x]) {
          ++place;
          lighter += few_w[j];
        }
      if (place == k - 1) {
        sh.warp_a[0] = few[threadIdx.x];
        sh.warp_a[1] = sh.above_w + lighter + few_w[threadIdx.x];
      }
    }
    __syncthreads();
    cut = sh.warp_a[0];
    total = sh.warp_a[1];
    __syncthreads();
  }
  if (by_mass) {
    if (want == 0) want = max(scaled(total, share_p, (1u << kGrid) - 1), 1ull);
    const int n = gather(before_w < want && before_w + weight >= want, cut);
    if (n > kPairs) return false;
    if ((int)threadIdx.x < n) {
      u64 at = sh.above_w;
      for (int j = 0; j < n; ++j)
        if (few[j] < few[threadIdx.x]) at += few_w[j];
      if (at < want && at + few_w[threadIdx.x] >= want) sh.warp_a[0] = few[threadIdx.x];
    }
    __syncthreads();
    cut = sh.warp_a[0];
    __syncthreads();
  }
  // the draw, in the order of the indexes
  const int width = (a.n + kBins - 1) / kBins;
  for (int i = threadIdx.x; i < 4 * kBins; i += kT) (&sh.hist[0][0])[i] = 0;
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    bin[q] = kBins;
    if (w[q] && order[q] <= cut && sc.e(value_of(~(unsigned)(order[q] >> 32))) >= floor_e) {
      bin[q] = (int)((unsigned)order[q] / (unsigned)width);
      add_weight(sh, bin[q], w[q]);
    }
  }
  __syncthreads();
  const u64 mine = weight_in(sh, threadIdx.x);
  before_w = scan1(sh, mine, total);
  const u64 aim = aim_of(a, r, total);
  const int n = gather(aim >= before_w && aim < before_w + mine, ~0ull);
  for (int i = threadIdx.x; i < n; i += kT) {
    u64 at = sh.above_w;
    for (int j = 0; j < n; ++j)
      if ((unsigned)few[j] < (unsigned)few[i]) at += few_w[j];
    if (aim >= at && aim < at + few_w[i]) {
      a.token[r] = (int)(unsigned)few[i];
      if (a.prob) a.prob[r] = __fdiv_rn((float)few_w[i], (float)total);
    }
  }
  return true;
}

// The rest of a row by one CTA: list[0 .. m) holds the order of every token
// that can be kept.  `k`: keep at most that many; `want`: then those whose
// predecessors weigh less (0: not yet known, top_p of what k keeps).
__device__ void finish(Shared& sh, u64* mass_s, const Scale& sc, const Args& a, int r, int m, int k, u64 want,
                       bool by_mass, u64 share_p, float floor_e) {
  if (m > kPairs && finish_by_bins(sh, mass_s, sc, a, r, m, k, want, by_mass, share_p, floor_e)) return;
  // consecutive tokens per thread
  sort_tokens(sh, m);
  const int per = (m + kT - 1) / kT, t0 = threadIdx.x * per;
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
    if (q < per && t0 + q < m) {
      mass_s[t0 + q] = w[q];
      sh.list[t0 + q] = w[q] ? (sh.list[t0 + q] << 32) | (unsigned)(t0 + q) : ~0ull - (unsigned)(t0 + q);
    }
  scan1(sh, mine, total);
  sort_tokens(sh, m);
  const u64 aim = aim_of(a, r, total);
  mine = 0;
#pragma unroll
  for (int q = 0; q < kPer; ++q) {
    const u64 entry = q < per && t0 + q < m ? sh.list[t0 + q] : ~0ull;
    w[q] = entry >> 32 == 0xffffffffu ? 0 : mass_s[(unsigned)entry];
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

// The bin of the k-th largest of the threads' own maxima: this CTA alone holds k
// logits up to there.
__device__ __forceinline__ int local_bound(Shared& sh, const Scale& sc, float thread_max, int k) {
  sh.hist[0][threadIdx.x] = 0;
  if (threadIdx.x == 0) sh.bin = kBins - 1;
  __syncthreads();
  const int b = sc.bin(thread_max);
  if (b < kBins) atomicAdd(&sh.hist[0][b], 1u);
  __syncthreads();
  const u64 count = sh.hist[0][threadIdx.x];
  u64 total;
  const u64 before = scan1(sh, count, total);
  if (before < (u64)k && before + count >= (u64)k) sh.bin = threadIdx.x;
  __syncthreads();
  const int bound = sh.bin;
  __syncthreads();
  return bound;
}

// Of a row's kT threads' maxima, which one has about 1.3 k + 16 logits up to it,
// if they lie at random: k of them nearly always, and kList hardly ever (for
// k <= kDirect).
constexpr int kDirect = 1400;
__device__ __forceinline__ int likely(int k) { return (int)(kT * (1.0f - __expf(-(1.3f * k + 16.0f) / kT))); }

// Rows that take one pass more than the maximum's at most: greedy ones, and
// those with a top-k whose candidates one CTA collects at once.
__device__ __forceinline__ bool light(const Args& a, int r) {
  const int k = a.top_k ? a.top_k[r] : 0;
  return (a.temperature && !(a.temperature[r] > 0.0f)) || (k > 0 && k < a.n && k <= kDirect);
}

// A row by `ctas` CTAs, `slice` logits each; STAGED: kept in shared memory at
// x_s.  The sums and lists come after them.
template <bool STAGED>
__device__ __forceinline__ void sample_row(Shared& sh, float* x_s, const Args& a, int r, unsigned ctas, int slice) {
  const unsigned rank = ctarank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float* x = a.logits + r * a.stride;
  const float temperature = a.temperature ? a.temperature[r] : 1.0f;
  const int k = a.top_k ? a.top_k[r] : 0;
  const bool by_count = k > 0 && k < a.n;
  const int share = slice / kW;  // of a warp
  float* mine_s = x_s + warp * share;
  Slice<STAGED> row{STAGED ? mine_s : x, (int)rank * slice + warp * share + 4 * lane, a.n, share / 128,
                    (reinterpret_cast<uintptr_t>(x) & 15) == 0, false, ctas};
  float top = -INFINITY, low = INFINITY;
  int top_group = 0;  // where this thread first saw its largest
  for (int j0 = 0; j0 < row.groups; j0 += 4) {
    float4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (j0 + q < row.groups) v[q] = row.from_memory(x, j0 + q);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int j = j0 + q, i = row.index(j);
      if (j >= row.groups) break;
      const float4 f = v[q];
      const float most = fmaxf(fmaxf(f.x, f.y), fmaxf(f.z, f.w));
      if (most > top) {
        top = most;
        top_group = j;
      }
      if (i + 4 <= a.n) {
        low = fminf(fminf(fminf(low, f.x), fminf(f.y, f.z)), f.w);
      } else {
        if (i < a.n) low = fminf(low, f.x);
        if (i + 1 < a.n) low = fminf(low, f.y);
        if (i + 2 < a.n) low = fminf(low, f.z);
      }
      if constexpr (STAGED) reinterpret_cast<float4*>(mine_s)[32 * j + lane] = f;
    }
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
  barrier(row.ctas);  // every CTA of the cluster runs before its shared memory is written to
  if (threadIdx.x < ctas) {
    for (int w = 0; w < kW; ++w) {
      top = fmaxf(top, warp_max[w]);
      low = fminf(low, warp_min[w]);
    }
    put32(remote(&sh.max_of[rank], threadIdx.x), __float_as_uint(top));
    put32(remote(&sh.min_of[rank], threadIdx.x), __float_as_uint(low));
  }
  barrier(row.ctas);
  top = -INFINITY;
  low = INFINITY;
  for (unsigned c = 0; c < ctas; ++c) {
    top = fmaxf(top, sh.max_of[c]);
    low = fminf(low, sh.min_of[c]);
  }
  if (top == -INFINITY) {
    if (rank == 0 && threadIdx.x == 0) {
      a.token[r] = 0;
      if (a.prob) a.prob[r] = 0.0f;
    }
    return;
  }
  if (!(temperature > 0.0f)) {  // greedy: the first index of the largest
    unsigned first = 0xffffffffu;
    if (thread_max == top) {
      const float4 v = row.at(top_group);
      const int at = v.x == top ? 0 : v.y == top ? 1 : v.z == top ? 2 : 3;
      first = (unsigned)(row.index(top_group) + at);
    }
    first = __reduce_min_sync(0xffffffffu, first);
    if (threadIdx.x == 0) sh.fill = 0xffffffffu;
    __syncthreads();
    if (lane == 0) atomicMin(&sh.fill, first);
    __syncthreads();
    if (threadIdx.x == 0) put32(remote(&sh.first_of[rank], 0), sh.fill);
    barrier(row.ctas);
    if (rank == 0 && threadIdx.x == 0) {
      for (unsigned c = 0; c < ctas; ++c) first = min(first, sh.first_of[c]);
      a.token[r] = (int)first;
      if (a.prob) a.prob[r] = 1.0f;
    }
    return;
  }
  float own_max = thread_max;
  if (top == INFINITY) {  // +inf logits share the weight: the others weigh nothing
    row.infinite = true;
    own_max = thread_max == INFINITY ? 0.0f : -INFINITY;
    top = 0.0f;
    low = -INFINITY;
  }
  Scale sc;
  sc.max = top;
  sc.inverse = fminf(__fdiv_rn(1.0f, temperature), 3e38f);
  const float span = (top - low) * sc.inverse;
  sc.bins = fminf((kFine - 1) / fminf(fmaxf(span, 1e-20f), kSpan) * sc.inverse, 1e38f);
  sc.base = 0;
  sc.shift = 4;
  const float p = a.top_p ? a.top_p[r] : 1.0f;
  const float floor_e = a.min_p ? fminf(a.min_p[r], 1.0f) : 0.0f;
  const bool by_mass = p < 1.0f;
  const u64 share_p = by_mass ? (u64)ceilf(__fmul_rn(fmaxf(p, 0.0f), 16777216.0f)) : 0;
  Cut cut{-INFINITY, INT32_MAX};
  u64 before, mine;
  if (by_count || by_mass) {
    const Part whole{0, 0, 0, 64};
    int bound = kBins - 1;
    if (by_count && k <= kDirect) {
      bound = local_bound(sh, sc, own_max, k <= kT / 2 ? k : likely(k));
      if (ctas == 1) {
        if (threadIdx.x == 0) sh.fill = 0;
        __syncthreads();
        row.collect(sc.least(bound), &sh.fill, [&](float v, int) { return sc.bin(v) <= bound; },
                    [&](unsigned slot, float v, int i) {
                      if (slot < kList) sh.list[slot] = order_of(v, i);
                    });
        __syncthreads();
        const unsigned n = sh.fill;
        __syncthreads();
        if (n <= kList && (n >= (unsigned)k || bound == kBins - 1)) {
          finish(sh, reinterpret_cast<u64*>(x_s), sc, a, r, (int)n, k, 0, by_mass, share_p, floor_e);
          return;
        }
      }
      if (k > kT / 2) bound = kBins - 1;  // a guess that did not hold
    }
    u64 want = (u64)k;
    Found f;
    if (by_count) {
      f = locate<false>(sh, row, sc, whole, cut, want, 0, 0, bound);
    } else {
      u64* own = reinterpret_cast<u64*>(x_s + (STAGED ? slice : 0));
      const u64 above_w = coarse_range(sh, row, sc, own, share_p, want);
      f = locate<true>(sh, row, sc, whole, cut, want, 0, above_w, bound);
    }
    // (a row with fewer than k weighty tokens: all of them)
    if (f.above_n + f.in_n <= kList) {
      const int upto = min(f.b, kBins - 1);
      if (threadIdx.x == 0) sh.fill = f.lower_upto;
      __syncthreads();
      row.collect(
          sc.least(upto), &sh.fill,
          [&](float v, int) { return sc.bin(v) <= upto && (by_count || weight_of(sc.e(v)) != 0); },
          [&](unsigned slot, float v, int i) {
            if (slot < kList) put64(remote(&sh.list[slot], 0), order_of(v, i));
          });
      barrier(row.ctas);
      if (rank == 0)
        finish(sh, reinterpret_cast<u64*>(x_s), sc, a, r, (int)(f.above_n + f.in_n), by_count ? k : a.n,
               by_count ? 0 : want, by_mass, share_p, floor_e);
      return;
    }
    if (by_count) {
      cut = resolve<false>(sh, row, sc, f, cut);
      if (by_mass) {
        const u64 mass = mass_upto(sh, row, sc, cut, 0.0f, before, mine);
        f = locate<true>(sh, row, sc, whole, cut, max(scaled(mass, share_p, (1u << kGrid) - 1), 1ull), 0, 0, kBins - 1);
        cut = resolve<true>(sh, row, sc, f, cut);
      }
    } else {
      cut = resolve<true>(sh, row, sc, f, cut);
    }
  }
  const u64 total = mass_upto(sh, row, sc, cut, floor_e, before, mine);
  const u64 aim = aim_of(a, r, total);
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
      if (i < a.n && cut.keeps(v[q], i)) {
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

constexpr int kOwnBytes = kCoarse * kT * sizeof(u64);  // coarse_range's sums
static_assert(kOwnBytes >= 2 * kList * (int)sizeof(u64), "finish()'s lists");
__host__ __device__ inline int slice_of(int n, int ctas) { return ((n + ctas - 1) / ctas + kUnit - 1) / kUnit * kUnit; }

// A cluster per row, its slices in shared memory.
__global__ void __launch_bounds__(kT, 2) staged_kernel(const __grid_constant__ Args a) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ Shared sh;
  extern __shared__ __align__(16) float x_s[];
  sample_row<true>(sh, x_s, a, blockIdx.x / nctas(), nctas(), slice_of(a.n, nctas()));
}

// A CTA per light row.
__global__ void __launch_bounds__(kT, 2) light_kernel(const __grid_constant__ Args a) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ Shared sh;
  extern __shared__ __align__(16) float x_s[];
  if (light(a, blockIdx.x)) sample_row<false>(sh, x_s, a, blockIdx.x, 1, slice_of(a.n, 1));
}

// A cluster per other row, next to light_kernel: this one does not wait for that
// to start (when it may, every CTA of that has seen what came before them
// both), and ends after it, so that what waits for this kernel has waited for
// both.
__global__ void __launch_bounds__(kT, 2) wide_kernel(const __grid_constant__ Args a) {
  allow_dependents_launch();
  __shared__ Shared sh;
  extern __shared__ __align__(16) float x_s[];
  const int r = blockIdx.x / nctas();
  if (!light(a, r)) sample_row<false>(sh, x_s, a, r, nctas(), slice_of(a.n, nctas()));
  if (blockIdx.x == 0) grid_dependency_wait();
}

template <typename K, typename... X>
cudaError_t launch_clusters(K k, int grid, int ctas, int smem, bool overlap, cudaStream_t st, X... x) {
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = overlap ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, k, x...);
}

cudaError_t launch_staged(const Args& a, int64_t rows, int ctas, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(staged_kernel, kMaxSlice * (int)sizeof(float) + kOwnBytes, done);
  if (e != cudaSuccess) return e;
  return launch_clusters(staged_kernel, (int)rows * ctas, ctas, slice_of(a.n, ctas) * (int)sizeof(float) + kOwnBytes,
                         launch_overlap(), st, a);
}

cudaError_t launch_rows(const Args& a, int64_t rows, int ctas, cudaStream_t st) {
  static std::atomic<uint64_t> done[2];
  cudaError_t e = allow_smem(light_kernel, kOwnBytes, done[0]);
  if (e == cudaSuccess) e = allow_smem(wide_kernel, kOwnBytes, done[1]);
  if (e == cudaSuccess) e = launch_ex(light_kernel, dim3((unsigned)rows), dim3(kT), kOwnBytes, st, a);
  if (e == cudaSuccess) e = launch_clusters(wide_kernel, (int)rows * ctas, ctas, kOwnBytes, true, st, a);
  return e;
}

}  // namespace sample
}  // namespace hyq

extern "C" {

int hyq_sample(const float* logits, int64_t n, int64_t stride, int64_t rows, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
               float* prob, void* stream) {
  const char* name = "sample";
  if (n <= 0 || n >= 1 << 23 || rows < 0 || rows > INT32_MAX / 8 || stride < n)  // (up to 8 CTAs a row)
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape (1 to 8388607 logits a row)", name);
  if (rows == 0) return HYQ_OK;
  if (!logits || !u || !token) return hyq::api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  for (const void* p : {(const void*)logits, (const void*)temperature, (const void*)top_k, (const void*)top_p,
                        (const void*)min_p, (const void*)u, (const void*)token, (const void*)prob})
    if (reinterpret_cast<uintptr_t>(p) % 4)
      return hyq::api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  const hyq::sample::Args a{logits, stride, (int)n, temperature, top_k, top_p, min_p, u, token, prob};
  const cudaStream_t st = (cudaStream_t)stream;
  // Few rows: as many CTAs per row as there are SMs for, the slices in their
  // shared memory.  Many: one per light row, four per other row, from memory.
  // Measured at 120,832 logits (temperature 0.7, top-k 40, top-p 0.9 / mixed
  // parameters / top-p 0.9 alone, us): 1 row 14 / 15 / 21 with eight, 16 / 16 / 24
  // with four; 16 rows 16 / 27 / 34 with six, 24 / 25 / 46 with eight; 32 rows 17
  // / 58 / 48 with four, 23 / 66 / 60 (48 rows) from memory; 64 rows 32 / 59 / 81
  // staged, 23 / 72 / 61 from memory; 256 rows 123 / 162 / 259 staged, 45 / 104 /
  // 187 from memory, 84 / 115 / 182 in one launch with idle CTAs on light rows.
  const int64_t units = (n + hyq::sample::kUnit - 1) / hyq::sample::kUnit;
  const int ctas = (int)std::min<int64_t>(rows <= 12 ? 8 : rows <= 16 ? 6 : 4, units);
  const bool staged = rows <= 32 && ctas > 1 && n <= (int64_t)ctas * hyq::sample::kMaxSlice;
  const cudaError_t e = staged ? hyq::sample::launch_staged(a, rows, ctas, st) : hyq::sample::launch_rows(a, rows, ctas, st);
  return e == cudaSuccess ? HYQ_OK : hyq::api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

}  // extern "C"
