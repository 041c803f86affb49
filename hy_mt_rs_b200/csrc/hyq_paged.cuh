// Device view of a paged KV cache and of a batch of new tokens, shared by the
// append and attention kernels over it.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hyq_common.cuh"

namespace hyq {
namespace paged {

constexpr int kMaxDim = 256;
constexpr int kMaxGroup = 16;  // query heads per kv head

// hyq_paged_kv + hyq_paged_batch (include/hyq.h), as the kernels take them.
struct Cache {
  void* k;
  void* v;
  int kv_heads, dim, page_size;
  int pages;
  int64_t page_stride, head_stride, row_stride;  // elements
  const int32_t* table;                          // [slots, width]
  int slots, width;
  const int32_t* slot;       // [seqs] or null
  const int32_t* row_start;  // [seqs + 1]
  const int32_t* pos;        // [seqs]
  int seqs, tokens;
  unsigned* status;
};

// One sequence's new tokens.
struct Seq {
  int row0;             // first row of the activations
  int n;                // new tokens (0: none, or a bad sequence)
  int pos;              // position of the first one
  const int32_t* pages; // its table row
};

// Sequence s, checked: rows inside the activations, positions inside the
// table row.  A bad one comes back empty and raises DEV_BAD_ARGS.
__device__ __forceinline__ Seq load_seq(const Cache& c, int s) {
  Seq q;
  q.row0 = c.row_start[s];
  const int end = c.row_start[s + 1];
  q.pos = c.pos[s];
  const int slot = c.slot ? c.slot[s] : s;
  q.n = end - q.row0;
  const bool ok = q.row0 >= 0 && q.n >= 0 && end <= c.tokens && q.pos >= 0 && slot >= 0 && slot < c.slots &&
                  (int64_t)q.pos + q.n <= (int64_t)c.width * c.page_size;
  if (!ok) {
    atomicOr(c.status, DEV_BAD_ARGS);
    q.n = 0;
  }
  q.pages = c.table + (ok ? (int64_t)slot * c.width : 0);
  return q;
}

// The sequence that row t belongs to (row_start ascending), or -1; by a whole
// warp, 32 entries per round of loads.
__device__ __forceinline__ int seq_of_row(const Cache& c, int t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = c.seqs + 1;  // the last entry <= t is among lo .. lo + n - 1, if any
  while (n > 0) {
    const int step = (n + 31) / 32, i = lo + lane * step;
    const bool in = i < lo + n && c.row_start[i] <= t;
    const int hits = __popc(__ballot_sync(0xffffffffu, in));  // a prefix of the lanes
    if (hits == 0) return -1;
    const int next = lo + (hits - 1) * step;
    if (step == 1) return next < c.seqs ? next : -1;
    n = min(step, lo + n - next);
    lo = next;
  }
  return -1;
}

// Page of a table entry, or -1 with DEV_BAD_ARGS when it is no page of the pool.
__device__ __forceinline__ int checked_page(const Cache& c, int page) {
  if (page >= 0 && page < c.pages) return page;
  atomicOr(c.status, DEV_BAD_ARGS);
  return -1;
}

// A tile of `rows` of a sequence's (token, query head) rows of one kv head.
// Tiles are numbered over the sequences with more than kFewRows such rows.
constexpr int kFewRows = 16;

// The sequence and the tile within it of tile `want`; false past the last.
// By a whole warp.
__device__ __forceinline__ bool find_tile(const Cache& c, int group, int rows, int want, int& seq, int& tile) {
  const int lane = threadIdx.x & 31;
  int carry = 0;
  for (int s0 = 0; s0 < c.seqs; s0 += 32) {
    int tiles = 0;
    if (s0 + lane < c.seqs) {
      const Seq s = load_seq(c, s0 + lane);
      if (s.n * group > kFewRows) tiles = (s.n * group + rows - 1) / rows;
    }
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const int before = carry + x - tiles;
    const unsigned hit = __ballot_sync(0xffffffffu, before <= want && want < before + tiles);
    if (hit) {
      const int l = __ffs(hit) - 1;
      seq = s0 + l;
      tile = want - __shfl_sync(0xffffffffu, before, l);
      return true;
    }
    carry += __shfl_sync(0xffffffffu, x, 31);
  }
  return false;
}

// hyq_paged_attention's activations and output.
struct AttendArgs {
  Cache c;
  const float* q;
  int64_t q_stride;
  int heads;
  float* out;
  int64_t out_stride;
  void* ws;
};

// The kernels round a sequence's length up to tiles and look some tiles ahead, in
// 32 bits: a table row ends this far below 2^31.
constexpr int kPastEnd = 4096;

// Largest number of sequences of a call (the kernels keep a prefix sum over
// them in shared memory).
constexpr int kMaxSeqs = 4096;

// hyq_paged_mma.cu: head sizes 64 and 128 over 16-byte aligned rows.
bool mma_supported(const AttendArgs& a, bool kv16);
size_t mma_workspace_bytes(int dim);
// Whether launch_few's 32-bit sum of tiles holds that many sequences of any
// length up to `reach` (4,096 of 16 million positions).
bool sums_fit(int64_t seqs, int64_t reach);
// Sequences of up to kFewRows rows; `beside`: next to the kernel that the same
// call launched before.
cudaError_t launch_few(const AttendArgs& a, bool kv16, bool beside, cudaStream_t st);
cudaError_t launch_chunks(const AttendArgs& a, bool kv16, cudaStream_t st);  // the others
// Whether that is faster than the kernels on tcgen05: one launch instead of
// three, but every CTA goes through its rows' positions alone, at 0.04 us (f16
// caches) or 0.16 us (f32) for each.  Measured with 16 query and 4 kv heads, us
// here / there: f16, 40 tokens at 100, 8 sequences 20 / 35; 200 tokens at 0 21 /
// 28; 5 tokens at 300, 64 sequences 31 / 51; 64 tokens at 500 36 / 34; 40 tokens
// at 300, 32 sequences 60 / 48; f32, 16 tokens at 0 13 / 21; 64 tokens at 0 21 /
// 21; 8 tokens at 100, 8 sequences 29 / 22.
bool chunks_short(const AttendArgs& a, bool kv16, int64_t max_len);
// hyq_paged_tc.cu: the others on tcgen05 (f16 caches; the workspace past
// mma_workspace_bytes), and launch_few beside them.
bool tc_supported(const AttendArgs& a);
size_t tc_workspace_bytes(int dim);
cudaError_t launch_chunks_tc(const AttendArgs& a, cudaStream_t st);
// hyq_paged_tc32.cu: the same over f32 caches, in the same workspace.
bool tc32_supported(const AttendArgs& a);
cudaError_t launch_chunks_tc32(const AttendArgs& a, cudaStream_t st);

// Weights are 2^(s - m) of the scores s, which carry log2(e) through the queries,
// with a reference m of 10 below the row's maximum: kept 2^10 times their size,
// their lo halves stay normal f16 numbers down to 2^-24 of the largest.  The
// reference is rounded up, so that no weight passes 2^10 (and f16's range)
// however coarse the scores are, and kept with the bias taken off, so that a
// weight is 2^(s - m) to the last bit of s and m.
constexpr float kBias = 10.0f;
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float reference(float top) { return __fsub_ru(top, kBias); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The non-finite values of V at positions first + 1 .. last of a sequence, in N
// neighbouring columns: their sums (0 where there are none).  An infinity that
// a row sees is its output whatever the weight, which is above zero: products
// do not give that (the halves of a split weight or value, and weights that
// round to zero, make NaN of it), so rows whose output is not finite though the
// sum of their weights is get it from here.  Likewise the kernels that multiply
// V by weights of zero take such values out first and add them back, with this,
// for the rows that see them.
template <int N>
struct Sums {
  float v[N];
};
template <bool KV16, int N>
__device__ __noinline__ Sums<N> non_finite(const Cache& c, const Seq& s, int kvh, int first, int last, int d) {
  constexpr int AHEAD = 8;  // positions whose loads are in flight together
  Sums<N> x{};
  for (int p0 = first + 1; p0 <= last; p0 += AHEAD) {
    float v[AHEAD][N];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int p = min(p0 + i, last), page = s.pages[p / c.page_size];
      const bool in = p0 + i <= last && page >= 0 && page < c.pages;
      const int64_t at = in ? (int64_t)page * c.page_stride + (int64_t)kvh * c.head_stride +
                                  (int64_t)(p % c.page_size) * c.row_stride + d
                            : 0;
#pragma unroll
      for (int k = 0; k < N; ++k)
        v[i][k] = !in ? 0.f : KV16 ? __half2float(static_cast<const __half*>(c.v)[at + k]) : static_cast<const float*>(c.v)[at + k];
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (!isfinite(v[i][k])) x.v[k] += v[i][k];
  }
  return x;
}

}  // namespace paged
}  // namespace hyq
