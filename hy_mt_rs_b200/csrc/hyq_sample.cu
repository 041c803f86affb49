// Sampling with temperature, top-k, top-p and min-p from given uniform numbers
// (include/hyq.h states the rule).  Weights and their sums are whole numbers,
// so neither the order of summation nor the split over threads changes a
// token.
#include <cuda_runtime.h>

#include <cstdint>

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

// One CTA per row; every pass reads the row again.
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
  const cudaError_t e = hyq::launch_ex(hyq::sample::sample_kernel, dim3((unsigned)rows), dim3(hyq::sample::kThreads), 0,
                                       (cudaStream_t)stream, a);
  return e == cudaSuccess ? HYQ_OK : hyq::api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

}  // extern "C"
