// Attention of sequences that share a prefix: a group's prefix is taken once, by
// all its tokens together, with the tcgen05 kernels of chunks (every token sees
// all of it); each sequence's own positions by the few-token kernel beside it.
// Both leave normalised outputs with their references and sums of weights, which
// merge_kernel puts together.
#include <algorithm>
#include <cmath>

#include "../../include/hyq.h"
#include "hyq_kernels.h"
#include "hyq_paged.cuh"
#include "hyq_paged_shared.h"

namespace hyq {
namespace paged {
namespace {

struct MergeArgs {
  const int32_t* token_prefix;
  const float* prefix;         // [tokens, heads, dim]
  const float2* prefix_ml;     // [tokens, heads]
  const float2* own_ml;
  float* out;                  // holds the sequences' own positions' outputs
  int64_t out_stride;
  int heads, dim;
};

// One CTA per token, a warp per head: y = (w0 y0 + w1 y1) / (w0 + w1), w = l 2^(m -
// max).  An output that is not finite stays so whatever its weight, which is above
// zero.
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ MergeArgs a) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (a.token_prefix[t] == 0) return;
  for (int h = warp; h < a.heads; h += 8) {
    const int64_t row = (int64_t)t * a.heads + h;
    const float2 ml[2] = {a.prefix_ml[row], a.own_ml[row]};
    const float top = fmaxf(ml[0].x, ml[1].x);
    float w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)  // (a part without a score above -inf has no weight, or NaN to pass on)
      w[i] = ml[i].x == -INFINITY ? (ml[i].y == 0.f ? 0.f : ml[i].y) : ml[i].y * ex2(ml[i].x - top);
    const bool none[2] = {ml[0].x == -INFINITY && ml[0].y == 0.f, ml[1].x == -INFINITY && ml[1].y == 0.f};
    const float inv = 1.0f / (w[0] + w[1]);
    const float* y0 = a.prefix + row * a.dim;
    float* y1 = a.out + t * a.out_stride + (int64_t)h * a.dim;
    for (int d = lane; d < a.dim; d += 32) {
      const float p = y0[d], o = y1[d];
      const float f0 = none[0] ? 0.f : isfinite(p) ? p * (w[0] * inv) : p, f1 = none[1] ? 0.f : isfinite(o) ? o * (w[1] * inv) : o;
      y1[d] = none[0] && none[1] ? inv * 0.f : f0 + f1;
    }
  }
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace

// The few-token kernel's counters, which stay zero between calls, come first in a
// workspace; what follows them is one way's or the other's.
size_t shared_workspace_bytes(int heads, int dim, int64_t tokens) {
  const size_t rows = (size_t)tokens * heads;
  const size_t chunks = rounded(rows * dim * sizeof(float)) + 2 * rounded(rows * sizeof(float2)) + rounded(kMaxSeqs * sizeof(int32_t)) +
                        rounded(tokens * sizeof(int32_t));
  return rounded(mma_workspace_bytes(dim) + tc_workspace_bytes(dim)) + std::max(chunks, line_workspace_bytes(heads, dim, tokens));
}

bool shared_supported(const AttendArgs& a, Kv kv) { return line_supported(a, kv) || (mma_supported(a, kv) && chunks_tc_supported(a, kv)); }

cudaError_t launch_shared(const AttendArgs& given, Kv kv, int64_t max_shared, cudaStream_t st) {
  if (line_supported(given, kv) && (!chunks_tc_supported(given, kv) || true))
    return launch_line(given, kv, static_cast<char*>(given.ws) + rounded(mma_workspace_bytes(given.c.dim) + tc_workspace_bytes(given.c.dim)), st);
  AttendArgs a = given;  // the prefixes' pass
  const size_t rows = (size_t)a.c.tokens * a.heads;
  char* p = static_cast<char*>(a.ws) + rounded(mma_workspace_bytes(a.c.dim) + tc_workspace_bytes(a.c.dim));
  auto take = [&](size_t bytes) {
    void* x = p;
    p += rounded(bytes);
    return x;
  };
  a.groups.out = given.out;
  a.groups.out_stride = given.out_stride;
  a.out = static_cast<float*>(take(rows * a.c.dim * sizeof(float)));
  a.out_stride = (int64_t)a.heads * a.c.dim;
  a.ml = static_cast<float2*>(take(rows * sizeof(float2)));
  a.groups.ml = static_cast<float2*>(take(rows * sizeof(float2)));
  a.groups.first = static_cast<int32_t*>(take(kMaxSeqs * sizeof(int32_t)));
  a.groups.token_prefix = static_cast<int32_t*>(take(a.c.tokens * sizeof(int32_t)));
  const cudaError_t e = launch_chunks_tc(a, kv, st);
  if (e != cudaSuccess) return e;
  const MergeArgs m{a.groups.token_prefix, a.out, a.ml, a.groups.ml, given.out, given.out_stride, a.heads, a.c.dim};
  return launch_next(merge_kernel, dim3((unsigned)a.c.tokens), dim3(256), 0, st, m);
}

}  // namespace paged
}  // namespace hyq
