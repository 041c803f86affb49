// Penalties for repeated tokens, biases and masks on rows of logits, in one pass
// (include/hyq.h states the rule).
//
// A CTA takes a slice of a row: it asks for its logits first, and while they
// come counts the slice's tokens among the row's history in shared memory (whole
// numbers: the order of the atomics does not matter).  Biases, which are few, come
// after the slice is out: the last entry of each token is found in the counts' place.
// Bound by memory, 8 bytes a logit; the history is read by every slice of its row,
// mostly from L2, so slices are as long as registers hold, unless a call has too few
// to fill the SMs with.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>

#include "../../include/hyq.h"
#include "hyq_common.cuh"
#include "hyq_kernels.h"

namespace hyq {
namespace logits {

constexpr int kThreads = 256;
constexpr unsigned kSeen = 0x80000000u;       // of a count: the token stands in the prompt

struct Args {
  const float* x;
  float* out;
  int64_t x_stride, out_stride;
  int n, slices;
  hyq_adjust a;
  unsigned* status;
};

// The tokens of a list from thread to thread, four loads in flight: f(token, index).
template <typename F>
__device__ __forceinline__ void each(const int32_t* list, int count, F f) {
  int i = threadIdx.x;
  for (; i + 3 * kThreads < count; i += 4 * kThreads) {
    int32_t t[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) t[k] = list[i + k * kThreads];
#pragma unroll
    for (int k = 0; k < 4; ++k) f(t[k], i + k * kThreads);
  }
  for (; i < count; i += kThreads) f(list[i], i);
}

// PER: logits of a thread.
template <int PER>
__global__ void __launch_bounds__(kThreads, PER == 32 ? 4 : 8) adjust_kernel(const __grid_constant__ Args a) {
  constexpr int kPer = PER, kSlice = kThreads * PER;
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ __align__(16) unsigned count_s[kSlice];
  const int r = blockIdx.x / a.slices, lo = (blockIdx.x - r * a.slices) * kSlice, size = min(kSlice, a.n - lo);
  const float* x = a.x + r * a.x_stride + lo;
  float* out = a.out + r * a.out_stride + lo;
  const bool vec = ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  // element k of this thread: four neighbours at a time, or one
  auto at = [&](int k) { return vec ? 4 * (int)threadIdx.x + (k >> 2) * 4 * kThreads + (k & 3) : (int)threadIdx.x + k * kThreads; };
  float v[kPer];
  if (vec) {
#pragma unroll
    for (int k = 0; k < kPer; k += 4) {
      if (at(k) + 3 < size) {
        const float4 f = *reinterpret_cast<const float4*>(x + at(k));
        v[k] = f.x, v[k + 1] = f.y, v[k + 2] = f.z, v[k + 3] = f.w;
      } else {
#pragma unroll
        for (int i = k; i < k + 4; ++i) v[i] = at(i) < size ? x[at(i)] : 0.f;
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) v[k] = at(k) < size ? x[at(k)] : 0.f;
  }
  const hyq_adjust& p = a.a;
  auto bad = [&] {
    if (threadIdx.x == 0) atomicOr(a.status, DEV_BAD_ARGS);
  };
  // the row's history
  float rep = p.repetition ? p.repetition[r] : 1.f;
  if (!(rep > 0.f)) rep = 1.f;
  const float presence = p.presence ? p.presence[r] : 0.f, frequency = p.frequency ? p.frequency[r] : 0.f;
  const int32_t* past = nullptr;
  int length = 0, prompt = 0;
  if (p.history && (rep != 1.f || presence != 0.f || frequency != 0.f)) {
    const int slot = p.slot ? p.slot[r] : r;
    if (slot >= p.slots) {
      bad();
    } else if (slot >= 0) {
      length = p.length[slot];
      prompt = p.prompt ? p.prompt[slot] : 0;
      if (length < 0 || length > p.history_width) {
        bad();
        length = 0;
      }
      past = p.history + slot * p.history_stride;
    }
  }
  int biases = 0, bias0 = 0;
  if (p.bias_start) {
    bias0 = p.bias_start[r];
    biases = p.bias_start[r + 1] - bias0;
    if (bias0 < 0 || biases < 0 || (int64_t)bias0 + biases > p.bias_count) {
      bad();
      biases = 0;
    }
  }
  const int32_t* words = nullptr;
  if (p.mask) {
    const int m = p.mask_row ? p.mask_row[r] : r;
    if (m >= p.masks) bad();
    else if (m >= 0) words = p.mask + m * p.mask_stride;
  }
  // (uniform over the CTA from here on)
  if (length > 0) {
#pragma unroll
    for (int i = 0; i < kPer / 4; ++i) reinterpret_cast<uint4*>(count_s)[threadIdx.x + i * kThreads] = make_uint4(0, 0, 0, 0);
    __syncthreads();
    each(past, length, [&](int t, int i) {
      const unsigned j = (unsigned)t - (unsigned)lo;
      if (j >= (unsigned)size) return;
      if (i < prompt) atomicOr(&count_s[j], kSeen);
      else atomicAdd(&count_s[j], 1u);
    });
    __syncthreads();
  }
  auto adjust = [&](float y, unsigned count, bool allowed) {
    if (count) {
      y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      const unsigned made = count & ~kSeen;
      if (made) y = __fsub_rn(y, __fadd_rn(__fmul_rn(frequency, (float)made), presence));
    }
    return allowed ? y : -INFINITY;
  };
  if (vec) {
#pragma unroll
    for (int k = 0; k < kPer; k += 4) {
      const int j = at(k);
      if (j >= size) break;
      uint4 c = make_uint4(0, 0, 0, 0);
      if (length > 0) c = *reinterpret_cast<const uint4*>(count_s + j);
      const unsigned w = words ? (unsigned)words[(lo + j) >> 5] >> ((lo + j) & 31) : 0xfu;
      if ((c.x | c.y | c.z | c.w) != 0 || (w & 0xfu) != 0xfu) {
        v[k] = adjust(v[k], c.x, w & 1u);
        v[k + 1] = adjust(v[k + 1], c.y, w & 2u);
        v[k + 2] = adjust(v[k + 2], c.z, w & 4u);
        v[k + 3] = adjust(v[k + 3], c.w, w & 8u);
      }
      if (j + 3 < size) {
        *reinterpret_cast<float4*>(out + j) = make_float4(v[k], v[k + 1], v[k + 2], v[k + 3]);
      } else {
#pragma unroll
        for (int i = k; i < k + 4; ++i)
          if (at(i) < size) out[at(i)] = v[i];
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int j = at(k);
      if (j >= size) break;
      const unsigned c = length > 0 ? count_s[j] : 0u;
      const unsigned w = words ? (unsigned)words[(lo + j) >> 5] >> ((lo + j) & 31) : 1u;
      out[j] = c || !(w & 1u) ? adjust(v[k], c, w & 1u) : v[k];
    }
  }
  if (biases == 0) return;
  // f(index of the token in the slice, entry) for the row's entries in this slice
  auto entries = [&](auto f) {
    each(p.bias_token + bias0, biases, [&](int t, int i) {
      const unsigned j = (unsigned)t - (unsigned)lo;
      if (j < (unsigned)size) f(j, (unsigned)i);
    });
  };
  __syncthreads();
  entries([&](unsigned j, unsigned) { count_s[j] = 0; });
  __syncthreads();
  entries([&](unsigned j, unsigned i) { atomicMax(&count_s[j], i + 1); });
  __syncthreads();
  entries([&](unsigned j, unsigned i) {
    const bool allowed = !words || ((unsigned)words[(lo + j) >> 5] >> ((lo + j) & 31) & 1u);
    if (count_s[j] == i + 1 && allowed) out[j] = __fadd_rn(out[j], p.bias_value[bias0 + i]);
  });
}

template <int PER>
cudaError_t launch(Args a, int64_t rows, int64_t slices, cudaStream_t st) {
  a.slices = (int)slices;
  return launch_ex(adjust_kernel<PER>, dim3((unsigned)(rows * slices)), dim3(kThreads), 0, st, a);
}

}  // namespace logits
}  // namespace hyq

extern "C" int hyq_logits_adjust(const float* logits, int64_t n, int64_t stride, int64_t rows, const hyq_adjust* adjust, float* out,
                                 int64_t out_stride, void* stream) {
  using namespace hyq::logits;
  const char* name = "logits_adjust";
  auto aligned = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; };
  if (!adjust) return hyq::api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  constexpr int kLong = 32, kShort = 8;  // logits of a thread
  const int64_t slices = (n + kThreads * kLong - 1) / (kThreads * kLong), shorter = (n + kThreads * kShort - 1) / (kThreads * kShort);
  if (n <= 0 || n > INT32_MAX - kThreads * kLong || stride < n || out_stride < n || rows < 0 || rows > INT32_MAX / shorter)
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape of the logits", name);
  const hyq_adjust& p = *adjust;
  if (rows == 0) return HYQ_OK;
  if (!logits || !out || (p.history && !p.length) || (!p.history && (p.repetition || p.presence || p.frequency)) ||
      (p.bias_start && (!p.bias_token || !p.bias_value)))
    return hyq::api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (p.history && (p.slots <= 0 || p.slots > INT32_MAX || p.history_width < 0 || p.history_width > INT32_MAX ||
                    p.history_stride < p.history_width || (!p.slot && rows > p.slots)))
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape of the history", name);
  if (p.bias_start && (p.bias_count < 0 || p.bias_count > INT32_MAX)) return hyq::api_fail(HYQ_E_SHAPE, "%s: number of biases", name);
  if (p.mask && (p.masks <= 0 || p.masks > INT32_MAX || p.mask_stride < (n + 31) / 32 || (!p.mask_row && rows > p.masks)))
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape of the mask", name);
  if (logits == out && stride != out_stride) return hyq::api_fail(HYQ_E_SHAPE, "%s: in place with two strides", name);
  for (const void* q : {(const void*)logits, (const void*)out, (const void*)p.history, (const void*)p.slot, (const void*)p.length,
                        (const void*)p.prompt, (const void*)p.repetition, (const void*)p.presence, (const void*)p.frequency,
                        (const void*)p.bias_start, (const void*)p.bias_token, (const void*)p.bias_value, (const void*)p.mask,
                        (const void*)p.mask_row})
    if (!aligned(q)) return hyq::api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  Args a{logits, out, stride, out_stride, (int)n, 0, p, nullptr};
  const int rc = hyq::api_status_word(&a.status);
  if (rc) return rc;
  // TUNE
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = rows * slices >= 2 * 148 ? launch<kLong>(a, rows, slices, st) : launch<kShort>(a, rows, shorter, st);
  return e == cudaSuccess ? HYQ_OK : hyq::api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}
