// Penalties for repeated tokens, biases and masks on rows of logits, in one pass
// (include/hyq.h states the rule).
//
// A CTA takes a slice of a row: it copies it, masked, while the row's history comes,
// and then changes the logits of the slice's tokens in that (noted down in shared
// memory as they come), each once, by whoever of their occurrences takes the count
// (whole numbers: the order of the atomics does not matter); the last bias entry of
// each token likewise.  Bound by memory, 8 bytes a logit: 256 rows of 120,832 in 39 us
// without histories (6.4 TB/s, the rate of a copy), 65 us with histories of 2,000
// tokens, 40 biases and masks: every slice of a row goes through its history (from L2),
// 14 us, and changes its tokens' logits, 8 us.
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
// Entries of a row's history and of the bias lists: the loops over them look up to this
// many past the last, in 32 bits.
constexpr int kPastEnd = 65536;
constexpr int64_t kMostEntries = INT32_MAX - kPastEnd;
static_assert(kPastEnd >= 16 * kThreads, "eight entries of each thread at a time, four turns unrolled");

struct Args {
  const float* x;
  float* out;
  int64_t x_stride, out_stride;
  int n, slices;
  hyq_adjust a;
  unsigned* status;
};

// PER: logits of a thread.
template <int PER>
__global__ void __launch_bounds__(kThreads, PER == 32 ? 4 : 8) adjust_kernel(const __grid_constant__ Args a) {
  constexpr int kPer = PER, kSlice = kThreads * PER;
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ unsigned count_s[kSlice];
  constexpr int kNotes = 4096;
  __shared__ uint16_t note_s[kNotes];  // the slice's tokens in the history: place, from 0x8000 up in the prompt
  __shared__ int notes_s;
  static_assert(kSlice <= 0x8000, "a place in 15 bits");
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
  if (threadIdx.x == 0) notes_s = 0;
  __syncthreads();
  const hyq_adjust& p = a.a;
  auto bad = [&] {
    if (threadIdx.x == 0) atomicOr(a.status, DEV_BAD_ARGS);
  };
  // what the row has, each list's loads as early as what they need is there
  float rep = p.repetition ? p.repetition[r] : 1.f;
  const float presence = p.presence ? p.presence[r] : 0.f, frequency = p.frequency ? p.frequency[r] : 0.f;
  const int slot = !p.history ? -1 : p.slot ? p.slot[r] : r, mask = !p.mask ? -1 : p.mask_row ? p.mask_row[r] : r;
  int bias0 = p.bias_start ? p.bias_start[r] : 0, biases = p.bias_start ? p.bias_start[r + 1] - bias0 : 0;
  if (!(rep > 0.f)) rep = 1.f;
  const int32_t* past = nullptr;
  int length = 0, prompt = 0;
  if (slot >= p.slots && slot >= 0) bad();
  if (slot >= 0 && slot < p.slots && (rep != 1.f || presence != 0.f || frequency != 0.f)) {
    length = p.length[slot];
    prompt = p.prompt ? p.prompt[slot] : 0;
    if (length < 0 || length > p.history_width) {
      bad();
      length = 0;
    }
    past = p.history + slot * p.history_stride;
  }
  if (bias0 < 0 || biases < 0 || (int64_t)bias0 + biases > p.bias_count) {
    bad();
    biases = 0;
  }
  if (mask >= p.masks && mask >= 0) bad();
  // the words of this thread's logits (one of each four neighbours, or of each one)
  constexpr int kWords = kPer / 4;
  const int32_t* words = mask >= 0 && mask < p.masks ? p.mask + mask * p.mask_stride : nullptr;
  unsigned bits[kWords];
#pragma unroll
  for (int k = 0; k < kWords; ++k) bits[k] = words && vec && at(4 * k) < size ? (unsigned)words[(lo + at(4 * k)) >> 5] : ~0u;
  // the lists' first tokens, for all of their passes
  constexpr int kTokens = 8, kEntries = 2;
  int token[kTokens], entry[kEntries];
#pragma unroll
  for (int k = 0; k < kTokens; ++k) token[k] = (int)threadIdx.x + k * kThreads < length ? past[threadIdx.x + k * kThreads] : -1;
#pragma unroll
  for (int k = 0; k < kEntries; ++k)
    entry[k] = (int)threadIdx.x + k * kThreads < biases ? p.bias_token[bias0 + threadIdx.x + k * kThreads] : -1;
  // the slice, masked
  if (vec) {
#pragma unroll
    for (int k = 0; k < kPer; k += 4) {
      const int j = at(k);
      if (j >= size) break;
      const unsigned w = bits[k / 4] >> ((lo + j) & 31);
      if ((w & 0xfu) != 0xfu) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!(w >> i & 1u)) v[k + i] = -INFINITY;
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
      out[j] = words && !((unsigned)words[(lo + j) >> 5] >> ((lo + j) & 31) & 1u) ? -INFINITY : v[k];
    }
  }
  // (length and biases are the same for the whole CTA)
  if (length == 0 && biases == 0) return;
  // f(place in the slice, index in the list) for the slice's tokens of a list, whose
  // first ones are held
  auto each = [&](const int32_t* list, int count, const auto& held, auto f) {
    constexpr int N = sizeof(held) / sizeof(int) == 1 ? 0 : sizeof(held) / sizeof(int);  // (one: none)
    auto one = [&](int t, int i) {
      const unsigned j = (unsigned)t - (unsigned)lo;
      if (j < (unsigned)size) f(j, i);
    };
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((int)threadIdx.x + k * kThreads < count) one(held[k], threadIdx.x + k * kThreads);
#pragma unroll 4
    for (int i = threadIdx.x + N * kThreads; i < count; i += kThreads) one(list[i], i);
  };
  auto allowed = [&](unsigned j) { return !words || ((unsigned)words[(lo + j) >> 5] >> ((lo + j) & 31) & 1u); };
  if (length > 0) {
    auto count = [&](unsigned j, bool in_prompt) {
      if (in_prompt) atomicOr(&count_s[j], kSeen);
      else atomicAdd(&count_s[j], 1u);
    };
    auto change = [&](unsigned j) {
      const unsigned n = atomicExch(&count_s[j], 0u), made = n & ~kSeen;
      if (n == 0 || !allowed(j)) return;
      float y = out[j];
      y = y > 0.f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
      if (made) y = __fsub_rn(y, __fadd_rn(__fmul_rn(frequency, (float)made), presence));
      out[j] = y;
    };
    const int lane = threadIdx.x & 31;
    auto note = [&](int t, int i) {
      const unsigned j = (unsigned)t - (unsigned)lo;
      const bool in = i < length && j < (unsigned)size;
      const unsigned hits = __ballot_sync(0xffffffffu, in);
      if (hits == 0) return;
      int first = 0;
      if (lane == 0) first = atomicAdd(&notes_s, __popc(hits));
      first = __shfl_sync(0xffffffffu, first, 0) + __popc(hits & ((1u << lane) - 1));
      if (in) {
        count_s[j] = 0;
        if (first < kNotes) note_s[first] = (uint16_t)(j | (i < prompt ? 0x8000u : 0u));
      }
    };
#pragma unroll
    for (int k = 0; k < kTokens; ++k) note(token[k], threadIdx.x + k * kThreads);
#pragma unroll 1
    for (int i0 = kTokens * kThreads; i0 < length; i0 += kTokens * kThreads) {
#pragma unroll
      for (int k = 0; k < kTokens; ++k) {
        const int i = i0 + k * kThreads + (int)threadIdx.x;
        token[k] = i < length ? past[i] : -1;
      }
#pragma unroll
      for (int k = 0; k < kTokens; ++k) note(token[k], i0 + k * kThreads + (int)threadIdx.x);
    }
    __syncthreads();  // (the copies are out, too)
    const int notes = notes_s;
    if (notes <= kNotes) {
      for (int n = threadIdx.x; n < notes; n += kThreads) count(note_s[n] & 0x7fffu, note_s[n] & 0x8000u);
      __syncthreads();
      for (int n = threadIdx.x; n < notes; n += kThreads) change(note_s[n] & 0x7fffu);
    } else {  // through the history again
      constexpr int none[1] = {-1};
      each(past, length, none, [&](unsigned j, int i) { count(j, i < prompt); });
      __syncthreads();
      each(past, length, none, [&](unsigned j, int) { change(j); });
    }
  }
  if (biases > 0) {
    const int32_t* list = p.bias_token + bias0;
    __syncthreads();
    each(list, biases, entry, [&](unsigned j, int) { count_s[j] = 0; });
    __syncthreads();
    each(list, biases, entry, [&](unsigned j, int i) { atomicMax(&count_s[j], (unsigned)i + 1); });
    __syncthreads();
    each(list, biases, entry, [&](unsigned j, int i) {
      if (count_s[j] == (unsigned)i + 1 && allowed(j)) out[j] = __fadd_rn(out[j], p.bias_value[bias0 + i]);
    });
  }
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
  if (p.history && (p.slots <= 0 || p.slots > INT32_MAX || p.history_width < 0 || p.history_width > kMostEntries ||
                    p.history_stride < p.history_width || (!p.slot && rows > p.slots)))
    return hyq::api_fail(HYQ_E_SHAPE, "%s: shape of the history", name);
  if (p.bias_start && (p.bias_count < 0 || p.bias_count > kMostEntries)) return hyq::api_fail(HYQ_E_SHAPE, "%s: number of biases", name);
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
  // Long slices read the history less often, short ones fill the SMs.  Measured at
  // 120,832 logits, histories of 10 to 4,000 tokens, long / short, us: 1 row 10.5 / 9.4,
  // 8 rows 10.7 / 10.5, 16 (240 long slices) 12.1 / 12.3, 32 14.2 / 17.4, 128 39 / 54.
  const cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = rows * slices >= 148 ? launch<kLong>(a, rows, slices, st) : launch<kShort>(a, rows, shorter, st);
  return e == cudaSuccess ? HYQ_OK : hyq::api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}
