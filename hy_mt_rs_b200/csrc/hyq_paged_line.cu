// Attention of groups of sequences with shared prefixes on the warp-level products,
// in two launches: one line of work for prefixes and sequences alike, and the join
// of its results.
//
// Items of the line are (64 of a group's rows, kv head) over the group's prefix and
// (sequence, kv head) over the sequence's own positions behind it, cut into tiles of
// positions and the line into equal ranges, one per CTA, as the few-token kernel
// does.  Of a wide item each warp takes 16 rows and all four blocks of a tile, so
// that a group's keys and values are read once for 64 rows; of an item of up to 16
// (32) rows all warps share (pairs of warps share) the rows and take a block (two)
// each.  An item inside one CTA's range leaves its rows' sums in the rows' own
// places, pieces of others go to the CTA's two partial results; merge_kernel adds up
// what a row has, in the order of the line.
#include "hyq_paged_rows.cuh"
#include "hyq_paged_shared.h"

namespace hyq {
namespace paged {
namespace {

constexpr int kWide = 64;                  // rows of a wide item
constexpr int kLineCtas = 148 * 2;
constexpr int kMaxUnits = 1024;            // sequences and groups of a call (the plan is in shared memory)
// What an item costs beside its tiles, in tiles of 16 rows: its queries, first copies
// and results.
constexpr int kItemCost = 4;

__host__ __device__ constexpr size_t part_floats(int dim) { return (size_t)kWide * (dim + 2); }

struct LineArgs {
  AttendArgs a;             // with groups' start, shared and n
  float* parts;             // [kLineCtas][2] (part_floats): outputs, then (reference, sum) of each row
  float* prefix;            // [tokens, heads, dim] of prefixes inside one CTA's range
  float2* prefix_ml;        // [tokens, heads]
  float2* own_ml;           // [tokens, heads], beside a.out
  int32_t* group_first;     // [groups + 1] units before each group, of one kv head
  int32_t* seq_first;       // [seqs + 1] units before each sequence, of one kv head, groups' included
  int32_t* seq_group;       // [seqs] group whose prefix a sequence takes, or -1
  int32_t* seq_prefix;      // [seqs] positions of that
};

// An item in the line: its first unit, tiles, and units per tile.
struct Item {
  int64_t u0;
  int tiles, per;
  __device__ __forceinline__ int units() const { return tiles * per + kItemCost; }
  // first tile at unit `at` or behind it
  __device__ __forceinline__ int tile_from(int64_t at) const {
    if (at <= u0) return 0;
    const int64_t j = (at - u0 + per - 1) / per;
    return j < tiles ? (int)j : tiles;
  }
};
// Warps of a row block stand `ways` apart: 1, 2 or 4 row blocks of a group's items.
__device__ __forceinline__ int ways_of(int rows) { return rows > 32 ? 4 : rows > 16 ? 2 : 1; }

template <int DIM, Kv KV>
__global__ void __launch_bounds__(kThreads, 2) line_kernel(const __grid_constant__ LineArgs p, int shift) {
  using G = Geo<DIM, KV>;
  using R = RowsOf<DIM, KV, 2>;
  static_assert(G::stages * G::block >= 2 * kRows * DIM * 4, "a warp's queries, as they come and as they are read");
  static_assert(G::ring >= kWide * G::pitch * 4, "the rows' joined outputs");
  grid_dependency_wait();
  allow_dependents_launch();
  extern __shared__ __align__(1024) char smem[];
  const AttendArgs& a = p.a;
  const int groups = a.groups.n, seqs = a.c.seqs, group = a.heads / a.c.kv_heads, kvh_n = a.c.kv_heads;
  int* start_s = reinterpret_cast<int*>(smem + G::ring);   // [groups + 1]
  int* prefix_s = start_s + groups + 1;                    // [groups]
  int* first_s = prefix_s + groups;                        // [groups + seqs + 1] units before each
  __shared__ float ml_s[kWarps][kRows][2];
  __shared__ float factor_s[kWarps][kRows];
  __shared__ int warp_s[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, cta = blockIdx.x;
  // the groups, checked: one whose prefix some sequence does not hold has none, nor has
  // a single sequence; starts that do not ascend from 0 to seqs: no groups
  bool bad = false;
  for (int i = threadIdx.x; i <= groups; i += kThreads) {
    const int first = a.groups.start[i];
    start_s[i] = first;
    bad = bad || first < 0 || first > seqs;
    if (i < groups) {
      const int last = a.groups.start[i + 1], shared = a.groups.shared[i];
      bad = bad || first > last || shared < 0;
      prefix_s[i] = last - first > 1 ? shared : 0;
    }
  }
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0) atomicOr(a.c.status, DEV_BAD_ARGS);
    for (int i = threadIdx.x; i < groups; i += kThreads) prefix_s[i] = 0;
    __syncthreads();
  }
  // the last group that starts at or before sequence i, if it is among them
  auto group_of = [&](int i) {
    int lo = 0, hi = groups - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (start_s[mid] <= i) lo = mid;
      else hi = mid - 1;
    }
    return start_s[lo] <= i && i < start_s[lo + 1] ? lo : -1;
  };
  for (int i = threadIdx.x; i < seqs; i += kThreads) {
    const int g = group_of(i);
    if (g < 0) continue;
    const Seq s = load_seq(a.c, i);
    const int slot = a.c.slot ? a.c.slot[i] : i, shared = prefix_s[g];
    if (shared > 0 && (a.c.row_start[i + 1] - a.c.row_start[i] != s.n || slot < 0 || slot >= a.c.slots || s.pos < shared ||
                       (int64_t)s.pos + s.n > (int64_t)a.c.width * a.c.page_size || s.n * group > kFewRows)) {
      atomicOr(a.c.status, DEV_BAD_ARGS);
      atomicExch(&prefix_s[g], 0);
    }
  }
  __syncthreads();
  auto group_rows = [&](int g) { return (a.c.row_start[start_s[g + 1]] - a.c.row_start[start_s[g]]) * group; };
  // units before each group, then before each sequence
  int carry = 0;
  for (int i0 = 0; i0 < groups + seqs; i0 += kThreads) {
    const int i = i0 + (int)threadIdx.x;
    int units = 0;
    if (i < groups) {
      if (prefix_s[i] > 0) {
        const int rows = group_rows(i);
        units = (rows + kWide - 1) / kWide * ((prefix_s[i] + G::tile - 1) / G::tile * ways_of(rows) + kItemCost);
      }
    } else if (i < groups + seqs) {
      const int q = i - groups, g = group_of(q), prefix = g >= 0 ? prefix_s[g] : 0;
      const Seq s = load_seq(a.c, q);
      if (s.n > 0 && s.n * group <= kRows) units = (s.pos + s.n - prefix + G::tile - 1) / G::tile + kItemCost;
      else if (s.n > 0) atomicOr(a.c.status, DEV_BAD_ARGS);  // max_new was too small: nobody takes it
      if (cta == 0) {
        p.seq_group[q] = prefix > 0 ? g : -1;
        p.seq_prefix[q] = prefix;
      }
    }
    int x = units;
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
    if (i < groups + seqs) first_s[i] = before + x - units;
    __syncthreads();
  }
  if (threadIdx.x == 0) first_s[groups + seqs] = carry;
  __syncthreads();
  if (cta == 0) {
    for (int i = threadIdx.x; i <= groups; i += kThreads) p.group_first[i] = first_s[i];
    for (int i = threadIdx.x; i <= seqs; i += kThreads) p.seq_first[i] = first_s[groups + i];
  }
  const int64_t work = (int64_t)carry * kvh_n;
  int64_t at = work * cta / kLineCtas;
  const int64_t end = work * (cta + 1) / kLineCtas;
  const uint32_t ring = smem_addr(smem);
  constexpr int part = G::stages * G::block;  // of a warp
  float* o_s = reinterpret_cast<float*>(smem);
  R rows;
  while (at < end) {
    // the item at `at`
    int u;
    {
      int lo = 0, hi = groups + seqs - 1;  // the last unit whose items start at or before `at`
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if ((int64_t)first_s[mid] * kvh_n <= at) lo = mid;
        else hi = mid - 1;
      }
      u = lo;
    }
    const int all = first_s[u + 1] - first_s[u];
    const int64_t base = (int64_t)first_s[u] * kvh_n;
    const int kvh = (int)((at - base) / all);
    Seq s;
    Item item;
    int r0 = 0, live, len, first = 0, ways = 1, limit;
    const bool wide = u < groups;
    if (wide) {
      const int q = start_s[u], total = group_rows(u), tiles_of_rows = (total + kWide - 1) / kWide, each = all / tiles_of_rows;
      const int64_t in = at - base - (int64_t)kvh * all;
      const int rt = (int)(in / each);
      ways = ways_of(total);
      len = prefix_s[u];
      item = {base + (int64_t)kvh * all + (int64_t)rt * each, (len + G::tile - 1) / G::tile, ways};
      r0 = rt * kWide;
      live = min(kWide, total - r0);
      s = load_seq(a.c, q);
      s.row0 = a.c.row_start[q];
      s.n = total / group;
      s.pos = limit = len - 1;
    } else {
      const int q = u - groups, g = group_of(q);
      first = g >= 0 ? prefix_s[g] : 0;
      s = load_seq(a.c, q);
      len = s.pos + s.n;
      item = {base + (int64_t)kvh * all, (len - first + G::tile - 1) / G::tile, 1};
      live = s.n * group;
      limit = s.pos;
    }
    const int j0 = item.tile_from(at), j1 = item.tile_from(end);
    at = item.u0 + item.units();
    if (j0 >= j1) continue;
    const int rb = warp & (ways - 1), ph = warp / ways, mine = min(kRows, live - kRows * rb);  // rows of this warp
    const bool any = mine > 0;
    if (any) {
      const uint32_t q_s = ring + warp * part, raw_s = q_s + kRows * DIM * 4;
      fetch_queries<DIM>(raw_s, a, s, kvh, group, r0 + kRows * rb, mine, 0, 1);
      cp_async_commit();
      cp_async_wait<0>();
      __syncwarp();
      stage_queries<DIM, KV>(q_s, factor_s[warp], raw_s, mine, 0, 1);
      __syncwarp();
      rows.load(q_s, factor_s[warp], s, group, r0 + kRows * rb, mine, wide ? 0 : 1);
      __syncwarp();
    }
    const Feed<DIM, KV> feed{a, s, kvh, len, shift};
    const int off = first + warp * G::pos;
    int page = feed.page(off + j0 * G::tile);
#pragma unroll
    for (int i = 0; i < G::stages - 1; ++i) {
      const int now = page;
      page = feed.page(off + (j0 + i + 1) * G::tile);
      if (j0 + i < j1) feed.copy(ring + warp * part + i * G::block, off + (j0 + i) * G::tile, now);
      cp_async_commit();
    }
    int stage = 0;
    for (int j = j0; j < j1; ++j) {
      cp_async_wait<G::stages - 2>();
      if (ways > 1) __syncthreads();  // tile j has landed; tile j - 1 has been read
      else __syncwarp();
      const int ahead = j + G::stages - 1, now = page;
      page = feed.page(off + (ahead + 1) * G::tile);
      int put = stage + G::stages - 1;
      if (put >= G::stages) put -= G::stages;
      if (ahead < j1) feed.copy(ring + warp * part + put * G::block, off + ahead * G::tile, now);
      cp_async_commit();
      if (any) {
#pragma unroll 1
        for (int b = ph; b < kWarps; b += kWarps / ways) {
          const int p0 = first + j * G::tile + b * G::pos;
          if (p0 >= len) break;
          const uint32_t at_b = ring + b * part + stage * G::block;
          const bool masked = p0 + G::pos - 1 > limit;
          // (values that are not finite at positions that some row does not see: the
          // merge puts them back)
          if (masked && !wide) feed.clean(at_b, p0, limit);
          rows.step(at_b, p0, masked);
        }
      }
      if (++stage == G::stages) stage = 0;
    }
    cp_async_wait<0>();
    if (any) {
#pragma unroll
      for (int i = 0; i < R::kPer; ++i) {
        const float l = rows.total(i);
        if (R::writes()) {
          ml_s[warp][R::row(i)][0] = rows.m[i];
          ml_s[warp][R::row(i)][1] = l;
        }
      }
    }
    __syncthreads();
    if (any) {
      float down[R::kPer];
#pragma unroll
      for (int i = 0; i < R::kPer; ++i) {
        float top = -INFINITY;
        for (int w = rb; w < kWarps; w += ways) top = fmaxf(top, ml_s[w][R::row(i)][0]);
        down[i] = rows.m[i] == -INFINITY ? 0.f : ex2(rows.m[i] - top);
      }
#pragma unroll 1
      for (int k = 0; k < kWarps / ways; ++k) {
        if (ph == k) {
#pragma unroll
          for (int i = 0; i < R::kPer; ++i)
            if (R::row(i) < mine) rows.add(o_s + (kRows * rb + R::row(i)) * G::pitch, i, down[i], k == 0);
        }
        if (ways < kWarps) __syncthreads();
      }
    } else if (ways < kWarps) {
      for (int k = 0; k < kWarps / ways; ++k) __syncthreads();
    }
    __syncthreads();
    const bool whole = j0 == 0 && j1 == item.tiles;
    float* to_part = p.parts + (size_t)(2 * cta + (j0 == 0)) * part_floats(DIM);
    for (int r = warp; r < live; r += kWarps) {
      const int row = r % kRows;
      float top = -INFINITY, l = 0.f;
      for (int w = r / kRows; w < kWarps; w += ways) top = fmaxf(top, ml_s[w][row][0]);
      for (int w = r / kRows; w < kWarps; w += ways)  // (a warp without a score above -inf has 0, or NaN to pass on)
        l = fmaf(ml_s[w][row][1], ml_s[w][row][0] == -INFINITY ? 0.f : ex2(ml_s[w][row][0] - top), l);
      const int tok = (r0 + r) / group, h = kvh * group + r0 + r - tok * group;
      const int64_t place_of = (int64_t)(s.row0 + tok) * a.heads + h;
      float* to = !whole ? to_part + r * DIM
                  : wide ? p.prefix + place_of * DIM
                         : a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)h * DIM;
#pragma unroll
      for (int k = 0; k < DIM / 32; ++k) to[lane + 32 * k] = o_s[r * G::pitch + lane + 32 * k];
      if (lane == 0)
        *(!whole ? reinterpret_cast<float2*>(to_part + (size_t)kWide * DIM) + r : (wide ? p.prefix_ml : p.own_ml) + place_of) =
            make_float2(top, l);
    }
    __syncthreads();  // o_s and ml_s are free again
  }
}

// One CTA per token, a warp per head in turn: the row's sums over the prefix and over
// its own positions, added up in the order of the line, over the sum of their weights.
template <int DIM, Kv KV>
__global__ void __launch_bounds__(256) merge_kernel(const __grid_constant__ LineArgs p) {
  using G = Geo<DIM, KV>;
  constexpr int N = DIM / 32;
  grid_dependency_wait();
  allow_dependents_launch();
  const AttendArgs& a = p.a;
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads, kvh_n = a.c.kv_heads;
  const int q = seq_of_row(a.c, t);
  if (q < 0) return;
  const Seq s = load_seq(a.c, q);
  if (t - s.row0 >= s.n || s.n * group > kFewRows) return;
  const int g = p.seq_group[q], prefix = p.seq_prefix[q], tok = t - s.row0;
  const int64_t work = (int64_t)p.seq_first[a.c.seqs] * kvh_n;
  const int seq_first = p.seq_first[q], seq_units = p.seq_first[q + 1] - seq_first;
  int group_first = 0, group_units = 0, group_row = 0, rows = 0;
  if (g >= 0) {
    const int q0 = a.groups.start[g], row0 = a.c.row_start[q0];
    group_first = p.group_first[g];
    group_units = p.group_first[g + 1] - group_first;
    group_row = t - row0;
    rows = (a.c.row_start[a.groups.start[g + 1]] - row0) * group;
  }
  for (int h = warp; h < a.heads; h += 8) {
    const int kvh = h / group;
    float* out = a.out + t * a.out_stride + (int64_t)h * DIM;
    float top = -INFINITY, l = 0.f, o[N] = {};
    // the results of the row (r of its item) over an item
    auto take = [&](const Item& item, int r, const float* whole_o, const float2* whole_ml) {
      int c = (int)(item.u0 * kLineCtas / work);  // the CTA that holds the item's first unit
      while (c > 0 && work * c / kLineCtas > item.u0) --c;
      while (work * (c + 1) / kLineCtas <= item.u0) ++c;
      const int64_t last = item.u0 + (int64_t)item.tiles * item.per;
      for (; c < kLineCtas && work * c / kLineCtas < last; c += 32) {
        // 32 CTAs' pieces: references and sums by the lanes ...
        const bool in = c + lane < kLineCtas;
        const int j0 = in ? item.tile_from(work * (c + lane) / kLineCtas) : 0;
        const int j1 = in ? item.tile_from(work * (c + lane + 1) / kLineCtas) : 0;
        const float* from = nullptr;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (j0 < j1) {
          if (j0 == 0 && j1 == item.tiles) {
            from = whole_o;
            ml = *whole_ml;
          } else {
            const float* part = p.parts + (size_t)(2 * (c + lane) + (j0 == 0)) * part_floats(DIM);
            from = part + r * DIM;
            ml = reinterpret_cast<const float2*>(part + (size_t)kWide * DIM)[r];
          }
        }
        float now = fmaxf(top, ml.x);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) now = fmaxf(now, __shfl_xor_sync(0xffffffffu, now, x));
        const float f0 = top == -INFINITY ? 0.f : ex2(top - now);
        const float f = from == nullptr || ml.x == -INFINITY ? 0.f : ex2(ml.x - now);
        // (a piece without a score above -inf has a sum of 0, or NaN to pass on)
        const float own = from == nullptr ? 0.f : ml.x == -INFINITY ? ml.y : f * ml.y;
        l = fmaf(l, f0, warp_sum(own));
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] *= f0;
        top = now;
        // ... then the outputs, piece after piece
        unsigned left = __ballot_sync(0xffffffffu, from != nullptr);
        const uint64_t address = reinterpret_cast<uint64_t>(from);
#pragma unroll 4
        while (left) {
          const int i = __ffs(left) - 1;
          left &= left - 1;
          const float* x = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, address, i));
          const float w = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
          for (int k = 0; k < N; ++k) o[k] = fmaf(w, x[lane + 32 * k], o[k]);
        }
      }
    };
    const int64_t row = (int64_t)t * a.heads + h;
    if (g >= 0) {
      const int r = group_row * group + h - kvh * group, ways = ways_of(rows), tiles = (prefix + G::tile - 1) / G::tile;
      const Item item{(int64_t)group_first * kvh_n + (int64_t)kvh * group_units + (int64_t)(r / kWide) * (tiles * ways + kItemCost),
                      tiles, ways};
      take(item, r % kWide, p.prefix + row * DIM, p.prefix_ml + row);
    }
    const Item item{(int64_t)seq_first * kvh_n + (int64_t)kvh * seq_units, seq_units - kItemCost, 1};
    take(item, tok * group + h - kvh * group, out, p.own_ml + row);
    const float inv = 1.0f / l;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int d = lane + 32 * k;
      out[d] = settled<KV>(o[k] * inv, l, tok > 0, a.c, s, kvh, s.pos, s.pos + tok, d);
    }
  }
}

size_t rounded(size_t n) { return (n + 255) / 256 * 256; }

template <int DIM, Kv KV>
cudaError_t launch(const LineArgs& p, cudaStream_t st) {
  using G = Geo<DIM, KV>;
  auto k = line_kernel<DIM, KV>;
  const int plan = (3 * p.a.groups.n + p.a.c.seqs + 2) * 4;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(k, G::ring + (3 * kMaxUnits + 2) * 4, done);
  const int page = p.a.c.page_size, shift = (page & (page - 1)) == 0 ? __builtin_ctz((unsigned)page) : -1;
  if (e == cudaSuccess) e = launch_ex(k, dim3(kLineCtas), dim3(kThreads), G::ring + plan, st, p, shift);
  if (e == cudaSuccess) e = launch_next(merge_kernel<DIM, KV>, dim3((unsigned)p.a.c.tokens), dim3(256), 0, st, p);
  return e;
}

template <Kv KV>
cudaError_t launch(const LineArgs& p, cudaStream_t st) {
  return p.a.c.dim == 128 ? launch<128, KV>(p, st) : launch<64, KV>(p, st);
}

}  // namespace

size_t line_workspace_bytes(int heads, int dim, int64_t tokens) {
  const size_t rows = (size_t)tokens * heads;
  return 2 * kLineCtas * part_floats(dim) * sizeof(float) + rounded(rows * dim * sizeof(float)) + 2 * rounded(rows * sizeof(float2)) +
         4 * rounded((kMaxUnits + 1) * sizeof(int32_t));
}

bool line_supported(const AttendArgs& a, Kv kv) {
  // (32-bit sums of units: a prefix's tiles count up to four times for each 64 rows)
  const int64_t reach = (int64_t)a.c.width * a.c.page_size / Geo<64, kF32>::tile + 1 + kItemCost;
  const int64_t tiles_of_rows = (int64_t)a.c.tokens * (a.heads / a.c.kv_heads) / kWide + a.groups.n;
  return mma_supported(a, kv) && a.groups.n + a.c.seqs <= kMaxUnits && (4 * tiles_of_rows + a.c.seqs) * reach <= INT32_MAX;
}

cudaError_t launch_line(const AttendArgs& a, Kv kv, void* workspace, cudaStream_t st) {
  const size_t rows = (size_t)a.c.tokens * a.heads;
  char* at = static_cast<char*>(workspace);
  auto take = [&](size_t bytes) {
    void* x = at;
    at += rounded(bytes);
    return x;
  };
  LineArgs p{};
  p.a = a;
  p.parts = static_cast<float*>(take(2 * kLineCtas * part_floats(a.c.dim) * sizeof(float)));
  p.prefix = static_cast<float*>(take(rows * a.c.dim * sizeof(float)));
  p.prefix_ml = static_cast<float2*>(take(rows * sizeof(float2)));
  p.own_ml = static_cast<float2*>(take(rows * sizeof(float2)));
  p.group_first = static_cast<int32_t*>(take((kMaxUnits + 1) * sizeof(int32_t)));
  p.seq_first = static_cast<int32_t*>(take((kMaxUnits + 1) * sizeof(int32_t)));
  p.seq_group = static_cast<int32_t*>(take((kMaxUnits + 1) * sizeof(int32_t)));
  p.seq_prefix = static_cast<int32_t*>(take((kMaxUnits + 1) * sizeof(int32_t)));
  return kv == kF32   ? launch<kF32>(p, st)
         : kv == kF16 ? launch<kF16>(p, st)
         : kv == kI8  ? launch<kI8>(p, st)
                      : launch<kF8>(p, st);
}

}  // namespace paged
}  // namespace hyq
