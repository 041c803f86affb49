// Attention over pages on the warp-level tensor instructions, head sizes 64
// and 128 (the rows' arithmetic is hyq_paged_rows.cuh's): the kernel for few new tokens (the cache is read once, bound by
// memory) and the one for chunks (16 rows of a chunk per warp).
//
// Both keep f32 accuracy with split operands.  Over an f16 cache K and V are
// exact, and the scaled queries and the weights are hi + lo, both f16 (22
// bits): two products each.  Over an f32 cache every operand is hi + lo in
// tf32 (hi rounded, lo cut: 22 bits, the full f32 range) and
// lo.lo is left out: three products each.  The tensor cores cut their sums
// instead of rounding them, which over a long context adds up (8e-6 at 1,100
// positions), so each block's output is added to the running one in f32
// arithmetic, and within a block small products go first.  Weights are 2^(x - m): the scores carry log2(e) through the
// queries.
//
// Few tokens, bound by memory: 64 requests of 90 to 4,000 positions (16 query
// and 4 kv heads of 128, f16, 269 MB) 54 us, 5.0 TB/s; 4 of 60,000 to 100,000
// (32 and 8 heads, 1.3 GB) 205 to 215 us, 6.1 to 6.4 TB/s; one of 512 positions (f32) 10.4 to 11.1 us,
// all latency: the plan of the line, the copies, the partial results' join.
// Over 8-bit caches (half the bytes) the same kernel is bound by its instructions'
// latencies: the 64 requests 54 us (139 MB, 2.6 TB/s), the four long ones 166 us (e4m3,
// 677 MB, 4.1 TB/s) at 53 % of the issue slots and 10.7 warps an SM, the integer pipe
// 58 % busy (1,240 instructions for 32 positions; it takes e4m3 codes to f16).  Sixteen
// positions at a time and four CTAs an SM instead of 32 and three: 186 us (registers
// spill at 128 a thread).
// Chunks, bound by the products and by each CTA's own walk over the positions:
// 200 tokens at 0 21 us, 8 sequences of 40 at 100 20 us (f16); longer ones go to
// the kernels on tcgen05.
#include "hyq_paged_rows.cuh"

namespace hyq {
namespace paged {
namespace {

// ---------------------------------------------------------------------------
// Few new tokens: at most 16 (token, head) rows per kv head
// ---------------------------------------------------------------------------

// Workspace: one counter per CTA, then two partial results per CTA: 16 rows of
// DIM outputs, then the rows' (maximum, sum), then whether clean() took a value
// out.
constexpr size_t kCounterBytes = HYQ_PAGED_ATTENTION_ZEROED;
constexpr int kSms = 148;
template <int ROWS = kRows>
__host__ __device__ constexpr int partial_floats(int dim) {
  return ROWS * (dim + 2) + 4;
}
// (kernels with more CTAs have smaller partial results)
constexpr int kMaxCtas = kSms * Geo<128, kF16>::ctas;
static_assert(kCounterBytes >= kSms * Geo<128, kI8, 1>::ctas * sizeof(unsigned), "a counter per CTA");
static_assert(kMaxCtas * partial_floats(64) >= kSms * Geo<64, kI8, 1>::ctas * partial_floats<8>(64) &&
                  kMaxCtas * partial_floats(128) >= kSms * Geo<128, kI8, 1>::ctas * partial_floats<8>(128),
              "one workspace for all");

// What a segment costs beside its tiles (queries, first copies, joining the
// warps), in tiles: the time of about four at full bandwidth.
constexpr int kSegmentCost = 4;

// The (sequence, kv head) segments' tiles, with kSegmentCost empty ones after
// each, form one line, cut into equal ranges, one per CTA: any mix of lengths
// loads every SM alike and the whole cache is read once.  A segment inside one
// CTA's range is finished there; one that spans CTAs leaves partial results,
// and the last CTA to get there adds them in the order of the CTAs (the result does not depend on which one
// that is).  Within a tile each warp takes its own POS positions for all 16
// rows, through its own ring of asynchronous copies; the warps meet at the
// end of a segment.
// `beside`: the kernel before is the same call's and has nothing that this one
// reads: it starts without waiting for that (when it may, every CTA of that has
// seen what came before them both), and ends after it.
// PART: only a sequence's positions from a.first on, and a.ml is written too.
// NB 1: a sequence with more than eight rows counts as several, of as many tokens as
// eight rows hold each (at most `shares`).
template <int DIM, Kv KV, bool PART, int NB>
__global__ void __launch_bounds__(kThreads, Geo<DIM, KV, NB>::ctas)
    few_kernel(const __grid_constant__ AttendArgs a, int shift, bool beside, int shares) {
  using G = Geo<DIM, KV, NB>;
  using R = RowsOf<DIM, KV, NB>;
  constexpr int kRows = G::rows;
  if (!beside) grid_dependency_wait();
  allow_dependents_launch();
  extern __shared__ __align__(1024) char smem[];
  int* first_s = reinterpret_cast<int*>(smem + G::smem);  // [seqs + 1] tiles (of one kv head) before each sequence (or share)
  __shared__ float ml_s[kWarps][kRows][2];
  __shared__ float factor_s[kRows];
  __shared__ int warp_s[kWarps];
  __shared__ int last_s;
  __shared__ int dirty_s;  // the last piece (of this CTA's) that clean() took a value out of
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads, seqs = NB == 1 ? a.c.seqs * shares : a.c.seqs, kvh_n = a.c.kv_heads;
  auto load = [&](int i) {
    if (NB > 1 || shares == 1) return load_seq(a.c, i);
    Seq s = load_seq(a.c, i / shares);
    if (s.n * group > kFewRows) return s;
    const int before = min(i % shares * (kRows / group), s.n);
    s.row0 += before;
    s.pos += before;
    s.n = min(s.n - before, kRows / group);
    return s;
  };
  if (!PART && a.groups.n) check_groups<int>(a.c, a.groups);
  // prefix sum of the sequences' tiles; sequences with more rows are the
  // chunk kernel's
  int carry = 0;
  for (int s0 = 0; s0 < seqs; s0 += kThreads) {
    const int i = s0 + (int)threadIdx.x;
    int tiles = 0;
    if (i < seqs) {
      const Seq s = load(i);
      if (s.n > 0 && s.n * group <= kRows) tiles = (s.pos + s.n - (PART ? a.first[NB == 1 ? i / shares : i] : 0) + G::tile - 1) / G::tile + kSegmentCost;
      else if (s.n > 0 && !beside) atomicOr(a.c.status, DEV_BAD_ARGS);  // max_new was too small: nobody takes it
    }
    int x = tiles;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    int before = carry;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += warp_s[w];
      carry += warp_s[w];
    }
    if (i < seqs) first_s[i] = before + x - tiles;
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    first_s[seqs] = carry;
    dirty_s = 0;
  }
  __syncthreads();
  const int64_t work = (int64_t)carry * kvh_n;
  const int ctas = (int)min((int64_t)gridDim.x, work), cta = blockIdx.x;
  if (cta >= ctas) {
    if (beside && cta == 0) grid_dependency_wait();
    return;
  }
  int64_t at = work * cta / ctas;
  const int64_t end = work * (cta + 1) / ctas;
  const int64_t begin = at;
  int si = 0;
  {
    int lo = 0, hi = seqs - 1;  // the last sequence whose segments start at or before `at`
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((int64_t)first_s[mid] * kvh_n <= at) lo = mid;
      else hi = mid - 1;
    }
    si = lo;
  }
  float* parts = reinterpret_cast<float*>(static_cast<char*>(a.ws) + kCounterBytes);
  unsigned* counters = static_cast<unsigned*>(a.ws);
  R rows;
  const uint32_t ring = smem_addr(smem) + warp * G::stages * G::block;
  float* o_s = reinterpret_cast<float*>(smem + G::ring);  // [rows][pitch]; the queries before
  const int off = warp * G::pos;
  // the piece of a segment that this CTA takes: tiles j0 .. j1 - 1 of `tiles`
  struct {
    Seq s;
    int kvh, j0, j1, tiles, first;  // (first: position of tile 0)
    int64_t seg0;
  } cur, done;
  int page = -1;  // of this lane's row in the next block to copy
  // the piece at `at`, and its first copies
  // (at the end of the range when only empty tiles are left)
  auto open = [&](bool same_seq) {
    for (;;) {
      while ((int64_t)first_s[si + 1] * kvh_n <= at) {  // past empty sequences
        ++si;
        same_seq = false;
      }
      const int units = first_s[si + 1] - first_s[si];
      const int64_t s_at = (int64_t)first_s[si] * kvh_n;
      cur.tiles = units - kSegmentCost;
      cur.kvh = (int)((at - s_at) / units);
      cur.seg0 = s_at + (int64_t)cur.kvh * units;
      if (at - cur.seg0 < cur.tiles) break;
      at = cur.seg0 + units;
      if (at >= end) return;
    }
    cur.j0 = (int)(at - cur.seg0);
    cur.j1 = (int)(min(end, cur.seg0 + cur.tiles) - cur.seg0);
    if (!same_seq) {
      cur.s = load(si);
      cur.first = PART ? a.first[NB == 1 ? si / shares : si] + off : off;
    }
    const Feed<DIM, KV, NB> feed{a, cur.s, cur.kvh, cur.s.pos + cur.s.n, shift};
    page = feed.page(cur.j0 * G::tile + cur.first);
    // (the ring's last stage is not copied to before the first turn)
    fetch_queries<DIM>(ring + (G::stages - 1) * G::block, a, cur.s, cur.kvh, group, 0, cur.s.n * group, warp, kWarps);
    cp_async_commit();
#pragma unroll
    for (int i = 0; i < G::stages - 1; ++i) {
      const int now = page;
      page = feed.page((cur.j0 + i + 1) * G::tile + cur.first);
      if (cur.j0 + i < cur.j1) feed.copy(ring + i * G::block, (cur.j0 + i) * G::tile + cur.first, now);
      cp_async_commit();
    }
  };
  open(false);
  for (int piece = 1; at < end; ++piece) {
    {
      const Seq& s = cur.s;
      const uint32_t q_s = smem_addr(o_s);
      cp_async_wait<G::stages - 1>();
      __syncwarp();
      stage_queries<DIM, KV, kRows>(q_s, factor_s, ring + (G::stages - 1) * G::block, s.n * group, warp, kWarps);
      __syncthreads();
      rows.load(q_s, factor_s, s, group, 0, s.n * group);
      const Feed<DIM, KV, NB> feed{a, s, cur.kvh, s.pos + s.n, shift};
      int stage = 0;
      for (int j = cur.j0; j < cur.j1; ++j) {
        const int ahead = j + G::stages - 1, now = page;
        page = feed.page((ahead + 1) * G::tile + cur.first);
        int put = stage + G::stages - 1;
        if (put >= G::stages) put -= G::stages;
        __syncwarp();
        if (ahead < cur.j1) feed.copy(ring + put * G::block, ahead * G::tile + cur.first, now);
        cp_async_commit();
        cp_async_wait<G::stages - 1>();
        __syncwarp();
        const int p0 = j * G::tile + cur.first;
        const bool masked = p0 + G::pos - 1 > s.pos;
        if (masked && feed.clean(ring + stage * G::block, p0, s.pos)) dirty_s = piece;
        rows.step(ring + stage * G::block, p0, masked);
        if (++stage == G::stages) stage = 0;
      }
    }
    const bool second = at != begin;  // not at this CTA's range's start
    done = cur;
    at = cur.j1 < cur.tiles ? end : cur.seg0 + cur.tiles;
    __syncwarp();
    if (at < end) open(true);  // the next piece's copies run while this one is joined
    // the warps' results: maximum and sum of each row, then the outputs scaled
    // to the common maximum, added up warp after warp
    const Seq& s = done.s;
    const int kvh = done.kvh, live = s.n * group;
#pragma unroll
    for (int i = 0; i < R::kPer; ++i) {
      const float l = rows.total(i);
      if (R::writes()) {
        ml_s[warp][R::row(i)][0] = rows.m[i];
        ml_s[warp][R::row(i)][1] = l;
      }
    }
    __syncthreads();
    float down[R::kPer];
#pragma unroll
    for (int i = 0; i < R::kPer; ++i) {
      const int r = R::row(i);
      float top = ml_s[0][r][0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ml_s[w][r][0]);
      down[i] = rows.m[i] == -INFINITY ? 0.f : ex2(rows.m[i] - top);
    }
#pragma unroll 1
    for (int w = 0; w < kWarps; ++w) {
      if (warp == w) {
#pragma unroll
        for (int i = 0; i < R::kPer; ++i)
          if (R::row(i) < live) rows.add(o_s + R::row(i) * G::pitch, i, down[i], w == 0);
      }
      __syncthreads();
    }
    const bool whole = done.j0 == 0 && done.j1 == done.tiles, dirty = dirty_s == piece;
    float* part = parts + (size_t)(2 * cta + second) * partial_floats<kRows>(DIM);
    constexpr int N = DIM / 32;  // values per lane, a warp per row
    for (int r = warp; r < live; r += kWarps) {
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml_s[w][r][0]);
#pragma unroll
      for (int w = 0; w < kWarps; ++w)  // (a warp without a score above -inf has 0, or NaN to pass on)
        l = fmaf(ml_s[w][r][1], ml_s[w][r][0] == -INFINITY ? 0.f : ex2(ml_s[w][r][0] - top), l);
      const float* from = o_s + r * G::pitch;
      if (whole) {
        const int tok = r / group;
        float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r - tok * group) * DIM;
        const float inv = 1.0f / l;
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int d = lane + 32 * k;
          to[d] = settled<KV>(from[d] * inv, l, dirty, a.c, s, kvh, s.pos, s.pos + tok, d);
        }
        if (PART && lane == 0) a.ml[(int64_t)(s.row0 + tok) * a.heads + kvh * group + r - tok * group] = make_float2(top, l);
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) part[r * DIM + lane + 32 * k] = from[lane + 32 * k];
        if (lane == 0) {
          part[kRows * DIM + 2 * r] = top;
          part[kRows * DIM + 2 * r + 1] = l;
        }
      }
    }
    if (!whole) {
      if (s.n > 1 && threadIdx.x == 0) part[kRows * (DIM + 2)] = dirty ? 1.0f : 0.0f;
      // the CTAs that share the segment: cf holds its first tile, cl its last
      const int64_t seg0 = done.seg0, seg1 = seg0 + done.tiles;
      int cf = (int)(seg0 * ctas / work);
      while (work * (cf + 1) / ctas <= seg0) ++cf;
      while (cf > 0 && work * cf / ctas > seg0) --cf;
      int cl = (int)((seg1 - 1) * ctas / work);
      while (work * (cl + 1) / ctas <= seg1 - 1) ++cl;
      while (cl > 0 && work * cl / ctas > seg1 - 1) --cl;
      // the CTA's stores come before the count by the barrier and this fence
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();
        last_s = atomicAdd(&counters[cf], 1u) == (unsigned)(cl - cf);
      }
      __syncthreads();
      if (last_s) {
        __threadfence();
        // partials cf .. cl, in order; only cf's may be its CTA's second
        const int n = cl - cf + 1;
        const float* part0 = parts + (size_t)(2 * cf + (work * cf / ctas < seg0)) * partial_floats<kRows>(DIM);
        const float* part1 = parts + (size_t)(2 * cf) * partial_floats<kRows>(DIM);
        auto part_at = [&](int i) { return i ? part1 + (size_t)(2 * i) * partial_floats<kRows>(DIM) : part0; };
        bool any = false;  // a piece was dirty
        for (int i = lane; s.n > 1 && i < n; i += 32) any = any || __ldcg(part_at(i) + kRows * (DIM + 2)) != 0.f;
        any = __any_sync(0xffffffffu, any);
        for (int r = warp; r < live; r += kWarps) {
          float top = -INFINITY, l = 0.f, sum[N] = {};
          for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(part_at(i) + kRows * DIM + 2 * r));
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          for (int i0 = 0; i0 < n; i0 += 32) {
            float f = 0.f;  // the weight of partial i0 + lane
            if (i0 + lane < n) {
              const float2 ml = __ldcg(reinterpret_cast<const float2*>(part_at(i0 + lane) + kRows * DIM + 2 * r));
              f = ml.x == -INFINITY ? 0.f : ex2(ml.x - top);
              l = fmaf(f, ml.y, l);
            }
            const int m = min(32, n - i0);
#pragma unroll 8
            for (int i = 0; i < m; ++i) {
              const float w = __shfl_sync(0xffffffffu, f, i);
              const float* from = part_at(i0 + i) + r * DIM + lane;
#pragma unroll
              for (int k = 0; k < N; ++k) sum[k] = fmaf(w, __ldcg(from + 32 * k), sum[k]);
            }
          }
          l = warp_sum(l);
          const float inv = 1.0f / l;
          const int tok = r / group;
          float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r - tok * group) * DIM;
#pragma unroll
          for (int k = 0; k < N; ++k) {
            const int d = lane + 32 * k;
            to[d] = settled<KV>(sum[k] * inv, l, any, a.c, s, kvh, s.pos, s.pos + tok, d);
          }
          if (PART && lane == 0) a.ml[(int64_t)(s.row0 + tok) * a.heads + kvh * group + r - tok * group] = make_float2(top, l);
        }
        if (threadIdx.x == 0) counters[cf] = 0;
      }
    }
    __syncthreads();  // o_s and ml_s are free again
  }
  if (beside && cta == 0) grid_dependency_wait();
}

// ---------------------------------------------------------------------------
// Chunks: 16 rows of a sequence's (token, head) rows per warp
// ---------------------------------------------------------------------------

constexpr int kChunkRows = kWarps * kRows;

// Grid (row tiles, kv heads): tile x belongs to the sequence whose tiles
// (64 rows each) contain it.  The four warps share every tile of positions, each
// copying a quarter of it.
template <int DIM, Kv KV>
__global__ void __launch_bounds__(kThreads, Geo<DIM, KV>::ctas) chunk_kernel(const __grid_constant__ AttendArgs a, int shift) {
  using G = Geo<DIM, KV>;
  using R = RowsOf<DIM, KV, 2>;
  grid_dependency_wait();
  allow_dependents_launch();
  extern __shared__ __align__(1024) char smem[];
  __shared__ int found_s[2];
  __shared__ float factor_s[kWarps][kRows];
  __shared__ int dirty_s;  // clean() took something out
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads, kvh = blockIdx.y;
  if (threadIdx.x == 0) {
    found_s[0] = -1;
    dirty_s = 0;
  }
  __syncthreads();
  if (warp == 0) {
    int seq, tile;  // the last (longest) tiles first
    if (find_tile(a.c, group, kChunkRows, gridDim.x - 1 - blockIdx.x, seq, tile) && lane == 0) {
      found_s[0] = seq;
      found_s[1] = tile;
    }
  }
  __syncthreads();
  if (found_s[0] < 0) return;
  const Seq s = load_seq(a.c, found_s[0]);
  const int r0 = found_s[1] * kChunkRows + warp * kRows;
  // positions the tile's last row sees
  const int last_tok = min(s.n - 1, (found_s[1] * kChunkRows + kChunkRows - 1) / group);
  const int len = s.pos + last_tok + 1, tiles = (len + G::tile - 1) / G::tile;
  const int first_tok = min(s.n - 1, found_s[1] * kChunkRows / group);
  const Feed<DIM, KV> feed{a, s, kvh, len, shift};
  const uint32_t ring = smem_addr(smem);
  // the queries: each warp's own 16 rows, through its part of the ring
  static_assert(G::stages * G::block >= 2 * kRows * DIM * 4, "a warp's queries, as they come and as they are read");
  R rows;
  const bool any = r0 < s.n * group;
  if (any) {
    const uint32_t q_s = ring + warp * G::stages * G::block, raw_s = q_s + kRows * DIM * 4;
    const int n = min(kRows, s.n * group - r0);
    fetch_queries<DIM>(raw_s, a, s, kvh, group, r0, n, 0, 1);
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    stage_queries<DIM, KV>(q_s, factor_s[warp], raw_s, n, 0, 1);
    __syncwarp();
    rows.load(q_s, factor_s[warp], s, group, r0, n);
  }
  __syncthreads();
  constexpr int stage_bytes = kWarps * G::block;
  const int off = warp * G::pos;
  int page = feed.page(off);
#pragma unroll
  for (int i = 0; i < G::stages - 1; ++i) {
    const int now = page;
    page = feed.page((i + 1) * G::tile + off);
    if (i < tiles) feed.copy(ring + i * stage_bytes + warp * G::block, i * G::tile + off, now);
    cp_async_commit();
  }
  int stage = 0;
  for (int j = 0; j < tiles; ++j) {
    cp_async_wait<G::stages - 2>();
    __syncwarp();
    if ((j + 1) * G::tile - 1 > s.pos + first_tok &&
        feed.clean(ring + stage * stage_bytes + warp * G::block, j * G::tile + off, s.pos + first_tok))
      dirty_s = 1;
    __syncthreads();  // tile j has landed; tile j - 1 has been read
    const int ahead = j + G::stages - 1, now = page;
    page = feed.page((ahead + 1) * G::tile + off);
    int put = stage + G::stages - 1;
    if (put >= G::stages) put -= G::stages;
    if (ahead < tiles) feed.copy(ring + put * stage_bytes + warp * G::block, ahead * G::tile + off, now);
    cp_async_commit();
    if (any) {
#pragma unroll 1
      for (int b = 0; b < kWarps; ++b) {
        const int p0 = j * G::tile + b * G::pos;
        if (p0 >= len) break;
        rows.step(ring + stage * stage_bytes + b * G::block, p0, p0 + G::pos - 1 > s.pos + first_tok);
      }
    }
    if (++stage == G::stages) stage = 0;
  }
  cp_async_wait<0>();
  __syncthreads();
  if (!any) return;
#pragma unroll
  for (int i = 0; i < R::kPer; ++i) {
    const float l = rows.total(i);
    const int r = r0 + R::row(i), tok = r / group;
    if (tok >= s.n) continue;
    float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r - tok * group) * DIM;
    bool odd = dirty_s;
    rows.each(i, [&](int d, float x) {
      const float y = x / l;
      odd = odd || !isfinite(y);
      to[d] = y;
    });
    if constexpr (!is_8bit(KV)) {
      if (odd) {
#pragma unroll 1
        for (int d = 0; d < DIM / 8; ++d)
#pragma unroll 1
          for (int j = 0; j < 2; ++j) {
            const int at = 8 * d + 2 * (lane & 3) + j;
            to[at] = settled<KV>(to[at], l, dirty_s, a.c, s, kvh, s.pos + first_tok, s.pos + tok, at);
          }
      }
    }
  }
}

int64_t chunk_tiles(const AttendArgs& a) {
  return ((int64_t)a.c.tokens * (a.heads / a.c.kv_heads) + kChunkRows - 1) / kChunkRows + a.c.seqs;
}

int page_shift(const AttendArgs& a) {
  return (a.c.page_size & (a.c.page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.c.page_size) : -1;
}

template <int DIM, Kv KV>
cudaError_t chunks(const AttendArgs& a, cudaStream_t st) {
  using G = Geo<DIM, KV>;
  const int64_t tiles = chunk_tiles(a);
  auto k = chunk_kernel<DIM, KV>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, G::smem, done);
  if (e != cudaSuccess) return e;
  return launch_ex(k, dim3((unsigned)tiles, (unsigned)a.c.kv_heads), dim3(kThreads), G::smem, st, a, page_shift(a));
}

template <int DIM, Kv KV, bool PART, int NB>
cudaError_t few(const AttendArgs& a, int shares, bool beside, cudaStream_t st) {
  using G = Geo<DIM, KV, NB>;
  auto k = few_kernel<DIM, KV, PART, NB>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, G::smem + ((NB == 1 ? 3 : 1) * kMaxSeqs + 1) * 4, done);
  if (e != cudaSuccess) return e;
  return launch_dependent(beside || launch_overlap(), k, dim3(kSms * G::ctas), dim3(kThreads),
                          (size_t)G::smem + (shares * a.c.seqs + 1) * 4, st, a, page_shift(a), beside, shares);
}

template <int DIM, Kv KV, int NB>
cudaError_t few(const AttendArgs& a, int shares, bool beside, cudaStream_t st) {
  return a.first ? few<DIM, KV, true, NB>(a, shares, beside, st) : few<DIM, KV, false, NB>(a, shares, beside, st);
}

template <Kv KV>
cudaError_t few(const AttendArgs& a, int64_t rows, bool beside, cudaStream_t st) {
  if constexpr (is_8bit(KV)) {
    const int group = a.heads / a.c.kv_heads;
    // Shares of a sequence with more than eight rows, 3 at most: as many as 16 rows need,
    // whatever max_new says (one with more tokens than that would lose its last ones).
    // None where max_new fits eight rows: such a sequence is reported then.
    const int shares = rows <= 8 || group > 8 ? 1 : (kRows / group + 8 / group - 1) / (8 / group);
    if (group <= 8)
      return a.c.dim == 128 ? few<128, KV, 1>(a, shares, beside, st) : few<64, KV, 1>(a, shares, beside, st);
  }
  return a.c.dim == 128 ? few<128, KV, 2>(a, 1, beside, st) : few<64, KV, 2>(a, 1, beside, st);
}

template <Kv KV>
cudaError_t chunks(const AttendArgs& a, cudaStream_t st) {
  return a.c.dim == 128 ? chunks<128, KV>(a, st) : chunks<64, KV>(a, st);
}

}  // namespace

bool mma_supported(const AttendArgs& a, Kv kv) {
  const int64_t strides = (a.c.page_stride | a.c.head_stride | a.c.row_stride) * value_bytes(kv);
  return (a.c.dim == 64 || a.c.dim == 128) && strides % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(a.c.k) | reinterpret_cast<uintptr_t>(a.c.v)) % 16 == 0;
}

bool sums_fit(int64_t seqs, int64_t reach) {
  constexpr int tile = Geo<128, kF32>::tile;  // the smallest one
  return seqs * (reach / tile + 1 + kSegmentCost) <= INT32_MAX;
}

bool chunks_short(const AttendArgs& a, Kv kv, int64_t max_len) {
  const int64_t tiles = (chunk_tiles(a) - a.c.seqs / 2) * a.c.kv_heads;  // sequences' last tiles are half full
  const int64_t rounds = (tiles + kMaxCtas - 1) / kMaxCtas;
  return rounds * max_len <= (kv == kF32 ? 64 : 350);
}

size_t mma_workspace_bytes(int dim) { return kCounterBytes + 2 * (size_t)kMaxCtas * partial_floats(dim) * sizeof(float); }

cudaError_t launch_few(const AttendArgs& a, Kv kv, int64_t max_new, bool beside, cudaStream_t st) {
  const int64_t rows = std::min<int64_t>(max_new * (a.heads / a.c.kv_heads), kRows);
  return kv == kF32   ? few<kF32>(a, rows, beside, st)
         : kv == kF16 ? few<kF16>(a, rows, beside, st)
         : kv == kI8  ? few<kI8>(a, rows, beside, st)
                      : few<kF8>(a, rows, beside, st);
}

cudaError_t launch_chunks(const AttendArgs& a, Kv kv, cudaStream_t st) {
  return kv == kF32 ? chunks<kF32>(a, st) : kv == kF16 ? chunks<kF16>(a, st) : kv == kI8 ? chunks<kI8>(a, st) : chunks<kF8>(a, st);
}

}  // namespace paged
}  // namespace hyq
