// What the tcgen05 attention kernels share (f16 caches: hyq_paged_tc.cu, f32
// caches: hyq_paged_tc32.cu): the plan of a call's work, the join of partial
// results, operand descriptors, tensor memory access.
#pragma once

#include <algorithm>

#include "hyq_kernels.h"
#include "hyq_paged.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kTile = 128;               // rows of a row tile, positions of a position tile
constexpr int kMaxCtas = 148;
constexpr int kMaxParts = 2 * kMaxCtas;  // partial results in the workspace: a CTA's first and last piece
constexpr int kMaxSegs = 65536;          // segments of a call
constexpr int kMinTiles = 2;             // cost of a CTA's range, at least
constexpr int kSegTiles = 1;             // cost of a segment, in tiles
// Floats of a partial result of a segment of ROWS rows: outputs, then
// (maximum, sum) of each row, then whether a value may have been taken out.
template <int ROWS>
__host__ __device__ constexpr size_t part_floats(int dim) {
  return (size_t)ROWS * (dim + 2) + 4;
}
constexpr float kSlack = 5.0f;           // a weight is at most 2^(kBias + kSlack): below f16's 65504

// A segment: its sequence (n rows of tokens from row0 at pos, pages in `slot`),
// which of the sequence's it is, and the position tiles that come before and
// up to its end among one kv head's.
struct alignas(16) Segment {
  int row0, n, pos, slot;
  int tile, first, end, unused;
};
// Where a CTA's range begins: position tile `begin` of all kv heads', in
// segment t of kv head kvh.
struct alignas(16) Start {
  int64_t begin;
  int t, kvh;
};
struct Plan {
  int* count;      // segments, then the total of their tiles
  Start* start;    // [kMaxCtas + 1]
  Segment* seg;    // [kMaxSegs]
  int most;        // segments that the rows of the call can make
};
constexpr size_t kPlanBytes = 16 + (kMaxCtas + 1) * sizeof(Start) + (size_t)kMaxSegs * sizeof(Segment);
template <int ROWS>
inline int64_t most_segments(const AttendArgs& a) {
  return ((int64_t)a.c.tokens * (a.heads / a.c.kv_heads) + ROWS - 1) / ROWS + a.c.seqs;
}
template <int ROWS>
inline Plan plan_of(const AttendArgs& a, void* ws) {
  char* p = static_cast<char*>(ws);
  return {reinterpret_cast<int*>(p), reinterpret_cast<Start*>(p + 16),
          reinterpret_cast<Segment*>(p + 16 + (kMaxCtas + 1) * sizeof(Start)), (int)most_segments<ROWS>(a)};
}

struct Params {
  AttendArgs a;
  Plan plan;
  int box;        // rows of a TMA box: min(page_size, 128) (f16 caches)
  float* parts;   // [CTA][first piece, last piece] (part_floats)
};

// Whether the plan holds a call's segments of ROWS rows: their number, and the
// 32-bit sum of their tiles at any length.
template <int ROWS>
inline bool plan_fits(const AttendArgs& a) {
  const int64_t segs = most_segments<ROWS>(a);
  return segs <= kMaxSegs && segs * ((int64_t)a.c.width * a.c.page_size / kTile + 1 + kSegTiles) <= INT32_MAX;
}

// Position tiles that the rows of a segment see.
template <int ROWS>
__device__ __forceinline__ int seen_tiles(const Seq& s, int group, int tile) {
  const int last = min((tile + 1) * ROWS, s.n * group) - 1;
  return (s.pos + last / group + kTile) / kTile;
}

// One CTA: the sequences' segments, each one's place in line, and the CTAs'
// ranges of it.  The line is cut by equal cost, kSegTiles more than its tiles
// for each segment (its queries in, its results out, a start of the pipeline).
template <int ROWS>
__global__ void __launch_bounds__(1024) plan_kernel(const __grid_constant__ AttendArgs a, const __grid_constant__ Plan plan) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ int off_s[kMaxSeqs + 1];
  __shared__ int warp_s[32];
  const int group = a.heads / a.c.kv_heads, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](int v, int& total) {
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    int w = warp_s[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = __shfl_sync(0xffffffffu, w, max(warp - 1, 0));
    return (warp ? before : 0) + x - v;
  };
  int segs = 0, total;
  for (int s0 = 0; s0 < a.c.seqs; s0 += 1024) {
    const int i = s0 + (int)threadIdx.x;
    int n = 0;
    if (i < a.c.seqs) {
      const Seq s = load_seq(a.c, i);
      if (s.n * group > kFewRows) n = (s.n * group + ROWS - 1) / ROWS;
    }
    const int at = segs + scan(n, total);
    if (i < a.c.seqs) off_s[i] = at;
    segs += total;
  }
  __syncthreads();
  segs = min(segs, plan.most);  // (more: rows of several sequences, row_start not ascending)
  int tiles = 0;
  for (int t0 = 0; t0 < segs; t0 += 1024) {
    const int t = t0 + (int)threadIdx.x;
    int cost = 0, seq = 0, tile = 0;
    Seq s{};
    if (t < segs) {
      int lo = 0, hi = a.c.seqs - 1;  // the last sequence with off <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (off_s[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      seq = lo;
      tile = t - off_s[lo];
      s = load_seq(a.c, seq);
      cost = seen_tiles<ROWS>(s, group, tile);
    }
    const int at = tiles + scan(cost, total);
    if (t < segs) plan.seg[t] = {s.row0, s.n, s.pos, a.c.slot ? a.c.slot[seq] : seq, tile, at, at + cost, 0};
    tiles += total;
  }
  __syncthreads();
  if (threadIdx.x <= kMaxCtas) {
    const int64_t per = tiles + (int64_t)kSegTiles * segs, work = per * a.c.kv_heads;
    const int64_t ctas = min((int64_t)kMaxCtas, max(work / kMinTiles, (int64_t)1));
    const int64_t unit = work * min((int64_t)threadIdx.x, ctas) / ctas;
    const int kvh = per ? (int)(unit / per) : 0;
    const int64_t rest = unit - kvh * per;
    int lo = 0, hi = segs - 1;  // the last segment that begins at `rest` or before
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (plan.seg[mid].first + (int64_t)kSegTiles * mid <= rest) lo = mid;
      else hi = mid - 1;
    }
    const int first = segs ? plan.seg[lo].first : 0;
    plan.start[threadIdx.x] = {(int64_t)kvh * tiles + first + max(rest - first - (int64_t)kSegTiles * (lo + 1), (int64_t)0), lo, kvh};
  }
  if (threadIdx.x == 0) {
    plan.count[0] = segs;
    plan.count[1] = tiles;
  }
}

// What a CTA does of a segment.
struct Piece {
  Seq s;
  int kvh, r0, rows, first_tok, len, j0, nt, jm;
  int64_t seg0;
  bool two, whole;
};
template <int ROWS>
__device__ __forceinline__ Piece piece_of(const Params& p, int group, int t, int kvh, int64_t at, int64_t end) {
  Piece x;
  const Plan& plan = p.plan;
  const int4* seg = reinterpret_cast<const int4*>(plan.seg + t);
  const int4 s = seg[0], place = seg[1];
  const int tile = place.x, first = place.y, tiles = place.z - place.y;
  x.s = {s.x, s.y, s.z, p.a.c.table + (int64_t)s.w * p.a.c.width};
  x.kvh = kvh;
  x.seg0 = (int64_t)kvh * plan.count[1] + first;
  x.r0 = tile * ROWS;
  x.rows = min(ROWS, x.s.n * group - x.r0);
  x.two = x.rows > kTile;          // the second row tile has rows
  x.first_tok = x.r0 / group;
  x.len = x.s.pos + (x.r0 + x.rows - 1) / group + 1;  // positions the last row sees
  x.j0 = (int)(at - x.seg0);
  x.nt = (int)(min(end, x.seg0 + tiles) - at);
  x.whole = x.j0 == 0 && x.nt == tiles;
  // tiles from here on hold positions that some row does not see
  x.jm = max(0, (x.s.pos + x.first_tok + 1) / kTile - x.j0);
  return x;
}

// Shared-memory operand descriptors, 128-byte swizzle, version 1.  Rows of 64
// f16 along the inner (K) dimension: 8-row groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t a) {
  return (uint64_t)((a >> 4) & 0x3fffu) | ((uint64_t)1 << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}
// V as the right operand: rows are the inner (K) dimension, 64 columns of N
// contiguous; the next 64 columns `half` bytes further, 8-row groups 1024.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t a, uint32_t half) {
  return (uint64_t)((a >> 4) & 0x3fffu) | ((uint64_t)(half >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// 16 columns of this thread's tensor memory lane.
__device__ __forceinline__ void tmem_ld(float (&v)[16], uint32_t a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(a));
}
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld(float (&v)[32], uint32_t a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(a));
}
__device__ __forceinline__ void tmem_st(uint32_t a, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
// f(columns, index of the first) over N columns from `a`, 16 at a time, the next
// load in flight while one is worked on.
template <int N, typename F>
__device__ __forceinline__ void tmem_each(uint32_t a, F f) {
  float v[2][16];
  tmem_ld(v[0], a);
#pragma unroll
  for (int c = 0; c < N / 16; ++c) {
    tmem_wait_ld();
    if (c + 1 < N / 16) tmem_ld(v[(c + 1) & 1], a + 16 * (c + 1));
    f(v[c & 1], 16 * c);
  }
}

// Ten mantissa bits of a weight (exact in f16 from 2^-14 up).
__device__ __forceinline__ float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// The same value in every lane, known to be so: descriptors and addresses made
// of such values stay in uniform registers, and a tcgen05.mma then takes 3
// cycles to issue instead of 46 (64 to run), so that the queue of a handful
// stays full across the waits between products.
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
  return p != 0;
}

// A wait of a whole warp: true only if every lane saw the phase complete.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}

// A row tile's queries, 32 rows by each of four warps: rows r0 .. of the
// segment's (token, head) rows, scaled to [1, 2) by a power of two that goes
// back into the scores (the result, for the thread's own row), hi and lo to
// q_s.  The rows come as they are, all in flight together, to the places that
// their own halves then take.
template <int DIM>
__device__ __forceinline__ float stage_rows(const AttendArgs& a, const Piece& x, int group, int r0, uint8_t* q_s) {
  constexpr float scale = (DIM == 128 ? 0.08838834764831845f : 0.125f) * kLog2e;  // log2(e) / sqrt(DIM)
  constexpr int N = DIM / 32, kLanes = DIM / 4;  // values per lane; lanes per row of 16-byte pieces
  constexpr int half = kTile * 128, tile = half * (DIM / 64);
  const int lane = threadIdx.x & 31, row0 = threadIdx.x & 96;
  const int rr = r0 + row0 + lane, tk = rr / group;
  const int64_t mine =
      tk < x.s.n ? (int64_t)(x.s.row0 + tk) * a.q_stride + (int64_t)(x.kvh * group + rr - tk * group) * DIM : -1;
  const bool vec = ((reinterpret_cast<uintptr_t>(a.q) | (uintptr_t)a.q_stride * 4) & 15) == 0;
  q_s += row0 * 128;
  const int c = lane % kLanes;
#pragma unroll 4
  for (int i = lane / kLanes; i < 32; i += 32 / kLanes) {
    const int64_t off = __shfl_sync(0xffffffffu, mine, i);
    const float* from = a.q + max(off, (int64_t)0) + 4 * c;
    const uint32_t to = smem_addr(q_s) + i * 128 + (c >> 3) * half + (((c ^ i) & 7) << 4), n = off >= 0 ? 4 : 0;
    if (vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(4 * n) : "memory");
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * k), "l"(from + k), "r"(n) : "memory");
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
  float factor = 1.0f;
  const int d = N * lane;
#pragma unroll 1
  for (int i0 = 0; i0 < 32; i0 += 4) {
    float v[4][N];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint8_t* from = q_s + (i0 + i) * 128 + (d >> 5) * half + ((((d >> 2) ^ (i0 + i)) & 7) << 4) + (d & 3) * 4;
#pragma unroll
      for (int k = 0; k < N; ++k) v[i][k] = reinterpret_cast<const float*>(from)[k] * scale;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t bits = 0;
#pragma unroll
      for (int k = 0; k < N; ++k) bits = max(bits, __float_as_uint(v[i][k]) & 0x7fffffffu);
      const int e = min(max((int)(__reduce_max_sync(0xffffffffu, bits) >> 23), 1), 253);
      if (lane == i0 + i) factor = __uint_as_float((uint32_t)e << 23);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        hi[k] = pack_f16(v[i][2 * k] * down, v[i][2 * k + 1] * down);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
        lo[k] = pack_f16(v[i][2 * k] * down - f.x, v[i][2 * k + 1] * down - f.y);
      }
      uint8_t* to = q_s + (i0 + i) * 128 + (d >> 6) * half + ((((d >> 3) ^ (i0 + i)) & 7) << 4) + (d & 7) * 2;
      if constexpr (N == 4) {
        *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
        *reinterpret_cast<uint2*>(to + tile) = make_uint2(lo[0], lo[1]);
      } else {
        *reinterpret_cast<uint32_t*>(to) = hi[0];
        *reinterpret_cast<uint32_t*>(to + tile) = lo[0];
      }
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
  return factor;
}

// One row's scores of a tile, in tensor memory at `st`, to weights, hi and lo
// (8 columns each for 16 positions), over them.  Weights are 2^(s - m) with a
// reference m kBias below the row's maximum (reference()) that follows it only
// when that is more than kSlack further up: the maximum pass over a tile's
// scores is then needed for a row's first tile alone.  l is the sum of the
// weights so far, `down` what the outputs so far are to be multiplied by.
// scale(v, c) is applied to the scores of columns c .. c + 31 before `factor`.
template <typename Scale>
__device__ __forceinline__ void scores_to_weights(uint32_t st, bool first, bool masked, int unseen_from, float factor, float& m,
                                                  float& l, float& down, Scale scale) {
  auto mask = [&](float (&v)[32], int c) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (c + i >= unseen_from) v[i] = -INFINITY;
  };
  auto largest = [&](const float (&v)[32]) {
    float a0 = fmaxf(v[0], v[1]), a1 = fmaxf(v[2], v[3]);
#pragma unroll
    for (int i = 4; i < 32; i += 4) {
      a0 = fmaxf(fmaxf(a0, v[i]), v[i + 1]);
      a1 = fmaxf(fmaxf(a1, v[i + 2]), v[i + 3]);
    }
    return fmaxf(a0, a1);
  };
  if (first) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kTile; c += 32) {
      float v[32];
      tmem_ld(v, st + c);
      tmem_wait_ld();
      scale(v, c);
      if (masked) mask(v, c);
      top = fmaxf(top, largest(v));
    }
    m = reference(top * factor);
  }
  float back = m == -INFINITY ? 0.f : -m, sum = 0.f, sum2 = 0.f;
  down = 1.f;
  // 32 columns: scores to weights, hi and lo over them.  (Loops of 32
  // columns, not unrolled, and two copies of them: the comparisons of a
  // masked tile take as long as the rest, and the unrolled code ran out
  // of the instruction cache.)
  auto weigh = [&](float (&v)[32], int c) {
    const float top = largest(v) * factor, over = top - m - kBias;
    if (__any_sync(0xffffffffu, over > kSlack)) {
      // raise the reference, by whole powers of two where what there is so far
      // still counts (2^-64 of it does not: nor does a sum from before the first
      // score above -inf); what this tile has so far follows
      float f = 1.f;
      if (over > 64.f) {
        f = 0.f;
        m = reference(top);
      } else if (over > kSlack) {
        const float before = m;
        m = fmaxf(m + ceilf(over), reference(top));
        f = ex2(before - m);
      }
      back = m == -INFINITY ? 0.f : -m;
      down *= f;
      sum *= f;
      sum2 *= f;
      tmem_wait_st();
#pragma unroll 1
      for (int b = 0; b < c; b += 16) {
        float w[16];
        uint32_t u[16];
        tmem_ld(w, st + b);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t hi = __float_as_uint(w[i]), lo = __float_as_uint(w[8 + i]);
          const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float y0 = (a0.x + a1.x) * f, y1 = (a0.y + a1.y) * f, h0 = high_part(y0), h1 = high_part(y1);
          u[i] = pack_f16(h0, h1);
          u[8 + i] = pack_f16(y0 - h0, y1 - h1);
        }
        tmem_st(st + b, u);
      }
    }
    uint32_t w[32];
#pragma unroll
    for (int g = 0; g < 32; g += 16)
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        const float y0 = ex2(fmaf(v[g + i], factor, back)), y1 = ex2(fmaf(v[g + i + 1], factor, back));
        sum += y0;
        sum2 += y1;
        const float h0 = high_part(y0), h1 = high_part(y1);
        w[g + (i >> 1)] = pack_f16(h0, h1);
        w[g + 8 + (i >> 1)] = pack_f16(y0 - h0, y1 - h1);
      }
    tmem_st(st + c, w);
  };
  if (masked) {
#pragma unroll 1
    for (int c = 0; c < kTile; c += 32) {
      float v[32];
      tmem_ld(v, st + c);
      tmem_wait_ld();
      scale(v, c);
      mask(v, c);
      weigh(v, c);
    }
  } else {
#pragma unroll 1
    for (int c = 0; c < kTile; c += 32) {
      float v[32];
      tmem_ld(v, st + c);
      tmem_wait_ld();
      scale(v, c);
      weigh(v, c);
    }
  }
  l = fmaf(l, down, sum + sum2);
}

// The results of a warp's 32 rows of a piece, row r this thread's: outputs, or
// a partial result.  They go through the rows' own places in q_s, whose
// queries no product reads any more, so that rows are written whole.
template <int DIM, int ROWS, bool KV16>
__device__ __forceinline__ void store_rows(const Params& p, const Piece& x, int group, int cta, bool second, int r,
                                           uint8_t* q_s, const float (&o)[DIM], float m, float l, bool dirty) {
  constexpr int half = kTile * 128, kLanes = DIM / 4;  // lanes of a row
  const AttendArgs& a = p.a;
  const int lane = threadIdx.x & 31, row0 = threadIdx.x & 96, tok = r / group;
  const bool in = r < x.s.n * group;
  float* part = p.parts + (size_t)(2 * cta + second) * part_floats<ROWS>(DIM);
  int64_t mine = -1;
  if (in && x.whole) {
    mine = (int64_t)(x.s.row0 + tok) * a.out_stride + (int64_t)(x.kvh * group + r - tok * group) * DIM;
  } else if (in) {
    mine = (int64_t)(r - x.r0) * DIM;
    *reinterpret_cast<float2*>(part + (size_t)ROWS * DIM + 2 * (r - x.r0)) = make_float2(m, l);
    if (KV16 && r == x.r0) part[(size_t)ROWS * (DIM + 2)] = dirty ? 1.0f : 0.0f;
  }
  const float inv = x.whole ? 1.0f / l : 1.0f;
  uint8_t* row = q_s + (row0 + lane) * 128;
#pragma unroll
  for (int c = 0; c < DIM / 4; ++c)
    *reinterpret_cast<float4*>(row + (c >> 3) * half + (((c ^ lane) & 7) << 4)) =
        make_float4(o[4 * c] * inv, o[4 * c + 1] * inv, o[4 * c + 2] * inv, o[4 * c + 3] * inv);
  __syncwarp();
  float* to = x.whole ? a.out : part;
  const bool vec = !x.whole || ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)a.out_stride * 4) & 15) == 0;
  const int c = lane % kLanes;
  bool odd = false;
#pragma unroll 4
  for (int i = lane / kLanes; i < 32; i += 32 / kLanes) {
    const int64_t off = __shfl_sync(0xffffffffu, mine, i);
    const float4 f = *reinterpret_cast<const float4*>(q_s + (row0 + i) * 128 + (c >> 3) * half + (((c ^ i) & 7) << 4));
    if (off < 0) continue;
    odd = odd || !isfinite((f.x + f.y) + (f.z + f.w));
    float* y = to + off + 4 * c;
    if (vec) {
      *reinterpret_cast<float4*>(y) = f;
    } else {
      y[0] = f.x, y[1] = f.y, y[2] = f.z, y[3] = f.w;
    }
  }
  __syncwarp();
  odd = __any_sync(0xffffffffu, odd);
  if (!x.whole || !(odd || dirty)) return;
  // infinities and NaN of V that the rows see (non_finite()); one that all see
  // shows in their outputs
  const int first = x.s.pos + x.first_tok;
  Sums<4> before{};
  if (odd) before = non_finite<KV16, 4>(a.c, x.s, x.kvh, -1, first, 4 * c);
#pragma unroll 1
  for (int i = lane / kLanes; i < 32; i += 32 / kLanes) {
    const int64_t off = __shfl_sync(0xffffffffu, mine, i);
    const int last = x.s.pos + __shfl_sync(0xffffffffu, tok, i);
    const float sum = __shfl_sync(0xffffffffu, l, i);
    if (off >= 0 && isfinite(sum)) {
      const Sums<4> own = non_finite<KV16, 4>(a.c, x.s, x.kvh, first, last, 4 * c);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (before.v[k] + own.v[k] != 0.f) to[off + 4 * c + k] = before.v[k] + own.v[k];
    }
    __syncwarp();
  }
}

// The pieces of the segment that starts in CTA blockIdx.x's range and goes on
// past it (there is at most one) added up, in the order of the CTAs; blockIdx.y
// picks 32 of its rows.  The pieces' factors of all rows first, then four rows
// of outputs per warp with the loads of four pieces in flight together.
constexpr int kJoinRows = 32;
template <int DIM, int ROWS, bool KV16>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p) {
  const AttendArgs& a = p.a;
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ float2 ml_s[kMaxCtas][kJoinRows];  // maximum (then factor) and sum
  __shared__ float l_s[kJoinRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.heads / a.c.kv_heads, cta = blockIdx.x;
  const int64_t begin = p.plan.start[cta].begin, end = p.plan.start[cta + 1].begin;
  if (begin == end) return;
  // the segment of tile end - 1: the one before the next range's, if that
  // range begins with one
  const int total = p.plan.count[1];
  int t = p.plan.start[cta + 1].t, kvh = p.plan.start[cta + 1].kvh;
  if ((int64_t)kvh * total + p.plan.seg[t].first == end) return;  // it ends with this range
  const int64_t seg0 = (int64_t)kvh * total + p.plan.seg[t].first, seg1 = (int64_t)kvh * total + p.plan.seg[t].end;
  if (seg0 < begin) return;
  int n = 1;  // and the ranges that begin inside it
  for (int c = cta + 1; c < kMaxCtas; c += 32) {
    const int hits = __popc(__ballot_sync(0xffffffffu, c + lane < kMaxCtas && p.plan.start[c + lane].begin < seg1));
    n += hits;
    if (hits < 32) break;
  }
  const int4 seq = *reinterpret_cast<const int4*>(p.plan.seg + t);
  const Seq s{seq.x, seq.y, seq.z, a.c.table + (int64_t)seq.w * a.c.width};
  const int r0 = p.plan.seg[t].tile * ROWS, row0 = blockIdx.y * kJoinRows;
  const int rows = min(kJoinRows, s.n * group - r0 - row0);
  if (rows <= 0) return;
  const float* part0 = p.parts + (size_t)(2 * cta + (seg0 != begin)) * part_floats<ROWS>(DIM);
  const float* part1 = p.parts + (size_t)(2 * cta) * part_floats<ROWS>(DIM);
  auto part = [&](int i) { return i ? part1 + (size_t)(2 * i) * part_floats<ROWS>(DIM) : part0; };
  bool dirty = false;
  for (int i = lane; KV16 && i < n; i += 32) dirty = dirty || part(i)[(size_t)ROWS * (DIM + 2)] != 0.f;
  for (int x = threadIdx.x; x < n * kJoinRows; x += 256) {
    const int row = x % kJoinRows, i = x / kJoinRows;
    ml_s[i][row] = row < rows ? reinterpret_cast<const float2*>(part(i) + (size_t)ROWS * DIM)[row0 + row] : make_float2(0.f, 1.f);
  }
  dirty = __any_sync(0xffffffffu, dirty);
  __syncthreads();
  // a thread per row: the pieces' factors
  if (threadIdx.x < kJoinRows) {
    const int row = threadIdx.x;
    float top = -INFINITY, l = 0.f;
    for (int i = 0; i < n; ++i) top = fmaxf(top, ml_s[i][row].x);
    for (int i = 0; i < n; ++i) {
      const float2 v = ml_s[i][row];
      const float f = v.x == -INFINITY ? 0.f : ex2(v.x - top);
      l = fmaf(f, v.y, l);
      ml_s[i][row].x = f;
    }
    l_s[row] = l;
  }
  __syncthreads();
  constexpr int N = DIM / 32;  // neighbouring values per lane, rows warp, warp + 8 ..
  float o[4][N] = {};
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* x = part(i) + (size_t)row0 * DIM + N * lane;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int row = min(warp + 8 * q, rows - 1);
      const float f = ml_s[i][row].x;
      float v[N];
      if constexpr (N == 4) {
        const float4 y = *reinterpret_cast<const float4*>(x + (size_t)row * DIM);
        v[0] = y.x, v[1] = y.y, v[2] = y.z, v[3] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(x + (size_t)row * DIM);
        v[0] = y.x, v[1] = y.y;
      }
#pragma unroll
      for (int k = 0; k < N; ++k) o[q][k] = fmaf(f, v[k], o[q][k]);
    }
  }
  auto place = [&](int r) {
    return a.out + (int64_t)(s.row0 + r / group) * a.out_stride + (int64_t)(kvh * group + r % group) * DIM + N * lane;
  };
  bool odd = false;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int row = warp + 8 * q;
    if (row >= rows) break;
    float* to = place(r0 + row0 + row);
    const float l = l_s[row];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float y = o[q][k] / l;
      odd = odd || !isfinite(y);
      to[k] = y;
    }
  }
  if (!odd && !dirty) return;
  const int first = s.pos + r0 / group;
  Sums<N> before{};
  if (odd) before = non_finite<KV16, N>(a.c, s, kvh, -1, first, N * lane);
#pragma unroll 1
  for (int row = warp; row < rows; row += 8) {
    if (!isfinite(l_s[row])) continue;
    float* to = place(r0 + row0 + row);
    const Sums<N> own = non_finite<KV16, N>(a.c, s, kvh, first, s.pos + (r0 + row0 + row) / group, N * lane);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (before.v[k] + own.v[k] != 0.f) to[k] = before.v[k] + own.v[k];
  }
}

}  // namespace
}  // namespace paged
}  // namespace hyq
