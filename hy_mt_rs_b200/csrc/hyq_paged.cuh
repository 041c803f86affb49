// Device view of a paged KV cache and of a batch of new tokens, shared by the
// append and attention kernels over it.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "hyq_common.cuh"

namespace hyq {
namespace paged {

constexpr int kMaxDim = 256;
constexpr int kMaxGroup = 16;  // query heads per kv head

// Type of a cache (HYQ_KV_*).  A row of an 8-bit one is dim codes and one f32
// scale: a value is code * scale.
enum Kv { kF32 = 0, kF16 = 1, kI8 = 2, kF8 = 3 };
__host__ __device__ constexpr bool is_8bit(Kv kv) { return kv == kI8 || kv == kF8; }
__host__ __device__ constexpr int value_bytes(Kv kv) { return kv == kF32 ? 4 : kv == kF16 ? 2 : 1; }

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
  float* k_scale;  // 8-bit caches: a scale per row
  float* v_scale;
  int64_t scale_page_stride, scale_head_stride, scale_row_stride;  // elements
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

// Four codes of an 8-bit cache as two f16 pairs: bytes 0 and 2 in `even`, 1 and 3
// in `odd`, exactly.  int8: 1024 + 128 + code is built in the bits of an f16 and
// 1152 taken off.  e4m3: its exponent and mantissa bits are an f16's three places
// further up, which makes 2^-8 of the value (code_unit(); subnormals too); there is no
// code for NaN, 0x7f and 0xff are +-480.
template <Kv KV>
__device__ __forceinline__ void decode4(uint32_t w, uint32_t& even, uint32_t& odd) {
  if constexpr (KV == kI8) {
    const __half2 off = __floats2half2_rn(1152.f, 1152.f);
    const uint32_t e = (w & 0x00ff00ffu) ^ 0x64806480u, o = ((w >> 8) & 0x00ff00ffu) ^ 0x64806480u;
    const __half2 he = __hsub2(*reinterpret_cast<const __half2*>(&e), off), ho = __hsub2(*reinterpret_cast<const __half2*>(&o), off);
    even = *reinterpret_cast<const uint32_t*>(&he);
    odd = *reinterpret_cast<const uint32_t*>(&ho);
  } else {
    even = ((w << 8) & 0x80008000u) | ((w << 7) & 0x3f803f80u);
    odd = (w & 0x80008000u) | ((w >> 1) & 0x3f803f80u);
  }
}
template <Kv KV>
__device__ __forceinline__ constexpr float code_unit() { return KV == kF8 ? 256.f : 1.f; }
template <Kv KV>
__device__ __forceinline__ float code_value(uint8_t c) {
  if constexpr (KV == kI8) return (float)(int8_t)c;
  const __half_raw h{(unsigned short)(((c & 0x80u) << 8) | ((c & 0x7fu) << 7))};
  return 256.f * __half2float(h);
}
// Scales of a row (element offset for page, kv head and row in the page).
__device__ __forceinline__ int64_t scale_at(const Cache& c, int page, int kvh, int row) {
  return (int64_t)page * c.scale_page_stride + (int64_t)kvh * c.scale_head_stride + (int64_t)row * c.scale_row_stride;
}
// A row's scale, and what takes its values to codes, from the bits of its largest
// magnitude: NaN and 0 for a row with an infinity or NaN, which then reads back as
// NaN throughout; 0 and 0 for one of zeros, or below 2^-90.
struct RowCode {
  float scale, inverse;
};
template <Kv KV>
constexpr double kLargest = KV == kI8 ? 127.0 : 448.0;  // code
template <Kv KV>
__device__ __forceinline__ RowCode row_code(uint32_t top) {
  constexpr float largest = (float)kLargest<KV>;
  if (top >= 0x7f800000u) return {__uint_as_float(0x7fc00000u), 0.f};
  if (top < (127u - 90u) << 23) return {0.f, 0.f};
  const float x = __uint_as_float(top);
  return {__fdiv_rn(x, largest), __fdiv_rn(largest, x)};
}
// Code of y, a value of magnitude kLargest (1 + 2^-22) at most in a row's unit: the
// nearest, ties to even; and how near the border between two codes is: how far y is
// from its code's value (int8), from the border (e4m3, whose numbers below 2^-6 are as
// far apart as those above).
template <Kv KV>
__device__ __forceinline__ uint8_t encode(float y, float& edge) {
  if constexpr (KV == kI8) {
    const float t = __fadd_rn(y, 12582912.f);  // 1.5 * 2^23: the whole number in the low bits
    edge = fmaxf(edge, fabsf(y - __fsub_rn(t, 12582912.f)));
    return (uint8_t)__float_as_uint(t);
  } else {
    const float z = fmaf(fabsf(y) < 0.015625f ? 1.f : 0.f, 0.015625f, fabsf(y));
    edge = fminf(edge, fabsf(z - __uint_as_float((__float_as_uint(z) & 0xfff00000u) | 0x80000u)));
    return (uint8_t)__nv_cvt_float_to_fp8(y, __NV_SATFINITE, __NV_E4M3);
  }
}
// Whether a border is as near as f32 arithmetic may have moved y over it.  From a row as
// it came, in units of 2^-24 of its largest magnitude: rotation (two roundings of a
// pair's length, which is at most sqrt(2) times that magnitude: 2.9), norm (two of the
// value itself), the magnitude as much again, its quotient and the product 2: 11.7 *
// 2^-24 * 127 (448) < 2^-13 (2^-11); without norm and rotation 2 * 2^-24 * 127 < 2^-16
// (2^-14).  Where weights follow the rotation, a value's share of its pair's error goes
// by its own weight, and the largest magnitude may be the other one's: with `uneven`,
// the largest ratio of a pair's weights, 2.9 becomes 2.9 * uneven, and 11.7
// 6 + 5.7 * uneven, which is less than (1 + uneven) / 2 of those limits.
template <Kv KV>
__device__ __forceinline__ constexpr float border_limit(float uneven) {
  return (0.5f + 0.5f * uneven) / (KV == kI8 ? 8192 : 2048);
}
constexpr float kUnrotated = -0.75f;  // (1 + this) / 2 is 1 / 8
template <Kv KV>
__device__ __forceinline__ bool near_border(float edge, float limit) {
  return KV == kI8 ? edge > 0.5f - limit : edge < limit;
}
// The ratio of two weights, 1 at least (1 of zeros, whose products are exact).
__device__ __forceinline__ float ratio_of(float a, float b) {
  const float hi = fmaxf(fabsf(a), fabsf(b)), lo = fminf(fabsf(a), fabsf(b));
  return hi == 0.f ? 1.f : 1.000001f * __fdividef(hi, lo);
}
// The code in 64 bits, y off by less than 2^-43 * uneven (e4m3: 2^-41): int8's is rounded
// to 2^-40 first and e4m3's to f32, so that what lies on a border goes to the even side.
// (No quotient x * 127 / top of f32 numbers is nearer to a border than 2^-32 and not on
// it; a rotated key may be.)
template <Kv KV>
__device__ __forceinline__ uint8_t encode(double y) {
  if constexpr (KV == kI8) return (uint8_t)(int8_t)max(-127, min(127, __double2int_rn(__dsub_rn(__dadd_rn(y, 6144.0), 6144.0))));
  else return (uint8_t)__nv_cvt_float_to_fp8((float)y, __NV_SATFINITE, __NV_E4M3);
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

// Groups of sequences with a prefix in common (n 0: none), for the kernels that
// take the prefixes; `out` and `ml` are those of the sequences' own positions then.
struct Groups {
  const int32_t* start;   // [n + 1] first sequence of each
  const int32_t* shared;  // [n] positions in common
  int n;
  int32_t* first;         // [seqs] prefix that a sequence takes from its group (0: none)
  int2* token;            // [tokens] first segment of a token's group (-1: none), its place among the group's
  float* out;
  int64_t out_stride;
  float2* ml;
  int64_t max_new;        // of any sequence
};

// The last group that starts at or before sequence i (start ascending).
__device__ __forceinline__ int group_of(const Groups& g, int i) {
  int lo = 0, hi = g.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (g.start[mid] <= i) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
// Whether group i's entries are none that a batch can have.
__device__ __forceinline__ bool bad_group(const Cache& c, const Groups& g, int i) {
  const int first = g.start[i], last = g.start[i + 1];
  return first < 0 || first > last || last > c.seqs || g.shared[i] < 0;
}
// The groups of a call whose sequences are taken each on their own all the same, looked
// over by all threads of the grid's first dimension: a bad one is reported.  INDEX: holds
// the number of threads.
template <typename INDEX>
__device__ __forceinline__ void check_groups(const Cache& c, const Groups& g) {
  const INDEX threads = (INDEX)gridDim.x * blockDim.x, mine = (INDEX)blockIdx.x * blockDim.x + threadIdx.x;
  bool bad = false;
  for (INDEX i = mine; i < g.n; i += threads) bad = bad || bad_group(c, g, (int)i);
  for (INDEX i = mine; i < c.seqs; i += threads) {
    const int k = group_of(g, (int)i), first = g.start[k], last = g.start[k + 1], p = g.shared[k];
    const bool in = first <= i && i < last && last - first > 1 && p > 0;
    bad = bad || (in && (c.pos[i] < p || (int64_t)c.row_start[i + 1] - c.row_start[i] > g.max_new));
  }
  if (bad) atomicOr(c.status, DEV_BAD_ARGS);
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
  // attention over a part of the positions only (null otherwise):
  const int32_t* first;  // [seqs] a sequence's positions from here on
  float2* ml;            // [tokens, heads] each output's reference and sum of weights, written with it
  Groups groups;
};

// The kernels round a sequence's length up to tiles and look some tiles ahead, in
// 32 bits: a table row ends this far below 2^31.
constexpr int kPastEnd = 4096;

// Largest number of sequences of a call (the kernels keep a prefix sum over
// them in shared memory).
constexpr int kMaxSeqs = 4096;

// hyq_paged_mma.cu: head sizes 64 and 128 over 16-byte aligned rows.
bool mma_supported(const AttendArgs& a, Kv kv);
size_t mma_workspace_bytes(int dim);
// Whether launch_few's 32-bit sum of tiles holds that many sequences of any
// length up to `reach` (4,096 of 16 million positions).
bool sums_fit(int64_t seqs, int64_t reach);
// Sequences of up to kFewRows rows (and, when that is less, as many as max_new tokens
// have); `beside`: next to the kernel that the same call launched before.
cudaError_t launch_few(const AttendArgs& a, Kv kv, int64_t max_new, bool beside, cudaStream_t st);
cudaError_t launch_chunks(const AttendArgs& a, Kv kv, cudaStream_t st);  // the others
// Whether that is faster than the kernels on tcgen05: one launch instead of
// three, but every CTA goes through its rows' positions alone, at 0.04 us (f16
// caches), 0.05 us (8-bit) or 0.16 us (f32) for each.  Measured with 16 query and 4 kv
// heads, us here / there: f16, 40 tokens at 100, 8 sequences 20 / 35; 200 tokens at 0
// 21 / 28; 5 tokens at 300, 64 sequences 31 / 51; 64 tokens at 500 36 / 34; 40 tokens
// at 300, 32 sequences 60 / 48; int8 (e4m3 within 1), the same five 23 / 35, 24 / 30,
// 38 / 60, 45 / 35 and, at 100, 53 / 47; 64 tokens at 200 30 / 33, at 350 37 / 35, 40
// at 300, 8 sequences 33 / 37; f32, 16 tokens at 0 13 / 21; 64 tokens at 0 21 / 21;
// 8 tokens at 100, 8 sequences 29 / 22.
bool chunks_short(const AttendArgs& a, Kv kv, int64_t max_len);
// hyq_paged_tc.cu: the others on tcgen05 (f16 caches; the workspace past
// mma_workspace_bytes), and launch_few beside them.
bool tc_supported(const AttendArgs& a);
size_t tc_workspace_bytes(int dim);
cudaError_t launch_chunks_tc(const AttendArgs& a, cudaStream_t st);
// hyq_paged_tc32.cu: the same over f32 caches, in the same workspace.
bool tc32_supported(const AttendArgs& a);
cudaError_t launch_chunks_tc32(const AttendArgs& a, cudaStream_t st);

// hyq_paged_tc8.cu: the same over 8-bit caches.
bool tc8_supported(const AttendArgs& a);
cudaError_t launch_chunks_tc8(const AttendArgs& a, Kv kv, cudaStream_t st);

// The kernels on tcgen05 for a cache type.
inline bool chunks_tc_supported(const AttendArgs& a, Kv kv) {
  return kv == kF16 ? tc_supported(a) : kv == kF32 ? tc32_supported(a) : tc8_supported(a);
}
inline cudaError_t launch_chunks_tc(const AttendArgs& a, Kv kv, cudaStream_t st) {
  return kv == kF16 ? launch_chunks_tc(a, st) : kv == kF32 ? launch_chunks_tc32(a, st) : launch_chunks_tc8(a, kv, st);
}

// Weights are 2^(s - m) of the scores s, which carry log2(e) through the queries,
// with a reference m of 10 below the row's maximum: kept 2^10 times their size,
// their lo halves stay normal f16 numbers down to 2^-24 of the largest.  The
// reference is rounded up, so that no weight passes 2^10 (and f16's range)
// however coarse the scores are, and kept with the bias taken off, so that a
// weight is 2^(s - m) to the last bit of s and m.
constexpr float kBias = 10.0f;
constexpr float kSlack = 5.0f;  // where the reference lags behind: a weight is at most 2^(kBias + kSlack), below f16's 65504
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
