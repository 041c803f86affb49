// Attention of sequences that share a prefix: a group's prefix is taken once, by all
// its tokens together, with the tcgen05 kernels of chunks (every token sees all of
// it); each sequence's own positions by the few-token kernel beside it; merge_kernel
// (hyq_paged_tc.cuh) puts the two together.  Here: the workspace of that.
#include "hyq_paged_shared.h"

#include "hyq_kernels.h"

namespace hyq {
namespace paged {
namespace {
size_t rounded(size_t n) { return (n + 255) / 256 * 256; }
}  // namespace

size_t shared_workspace_bytes(int heads, int dim, int64_t tokens) {
  const size_t rows = (size_t)tokens * heads;
  return rounded(mma_workspace_bytes(dim) + tc_workspace_bytes(dim)) + rounded(rows * dim * sizeof(float)) + 2 * rounded(rows * sizeof(float2)) +
         rounded(kMaxSeqs * sizeof(int32_t)) + rounded(tokens * sizeof(int2));
}

// Whether a call's prefixes are worth their own kernels: reading them for every
// sequence costs 5 to 6 TB/s of L2, which reaches the three launches' own time at about
// 130 (f32) to 230 MB (f16).  Measured with 16 query and 4 kv heads, one group, shared /
// each on its own, us in a graph: f16, 16 sequences of 2,000 (61 MB) 43 / 23, 32 (127 MB)
// 45 / 31, 48 (193 MB) 46 / 40, 64 (258 MB) 46 / 50, 16 of 8,000 (246 MB) 47 / 46; int8 and
// e4m3, 32 of 2,000 (65 MB) 50 / 32, 64 (133 MB) 56 / 51, 16 of 8,000 (127 MB) 50 / 45, 32
// (262 MB) 51 / 77; f32, 16 of 2,000 (123 MB) 44 / 40, 8 of 8,000 (229 MB) 43 / 63, 32 of
// 2,000 (254 MB) 46 / 67.
bool worth_sharing(const AttendArgs& a, Kv kv, int64_t groups, int64_t max_shared) {
  const int64_t row = 2 * ((int64_t)a.c.dim * value_bytes(kv) + (is_8bit(kv) ? 4 : 0)) * a.c.kv_heads;
  return groups > 0 && (double)((a.c.seqs - groups) * max_shared) * row >= 150e6;
}

bool shared_supported(const AttendArgs& a, Kv kv) { return mma_supported(a, kv) && chunks_tc_supported(a, kv); }

cudaError_t launch_shared(const AttendArgs& given, Kv kv, cudaStream_t st) {
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
  a.groups.token = static_cast<int2*>(take(a.c.tokens * sizeof(int2)));
  return launch_chunks_tc(a, kv, st);
}

}  // namespace paged
}  // namespace hyq
