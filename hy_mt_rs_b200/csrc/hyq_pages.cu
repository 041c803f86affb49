// Bookkeeping of a paged cache on the device: reserve, free, fork and compact
// sequences' pages (include/hyq.h).  The integer work of a call is one CTA;
// the page copies of fork and compact follow in a second launch that reads
// the list of copies from the workspace.  The first is latency, about 5 us for
// eight forks of 16 pages (dependent reads of the tables, two scans); the
// second is bound by memory.
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/hyq.h"
#include "hyq_common.cuh"
#include "hyq_kernels.h"

namespace hyq {
namespace pages {

constexpr int kThreads = 1024;
constexpr int kMaxSeqs = 1024;  // sequences per call: one thread each

struct Table {
  int32_t* table;   // [slots, width]
  int32_t* length;  // [slots]
  int32_t* refs;    // [pages]
  int32_t* shortage;
  int slots, width, pages, page_size;
  unsigned* status;
};

// Workspace: the number of page copies, then the lists they come from and go
// to, then the new name of every page.
struct Plan {
  int32_t* count;
  int32_t* from;  // [pages]
  int32_t* to;    // [pages]
  int32_t* name;  // [pages]
};

__host__ __device__ inline Plan plan_of(void* ws, int64_t pages) {
  int32_t* p = static_cast<int32_t*>(ws);
  return {p, p + 4, p + 4 + pages, p + 4 + 2 * pages};
}

// Sum of two counts, CAPPED at kMost: 1,024 sequences may ask for more than 2^31
// pages together, and must not seem to ask for few.
constexpr unsigned kMost = HYQ_PAGES_REFUSED - 1;
template <bool CAPPED>
__device__ __forceinline__ int sum_of(int a, int b) {
  return CAPPED ? (int)min((unsigned)a + (unsigned)b, kMost) : a + b;
}

// Exclusive prefix sum of one value per thread over the CTA (1024 threads),
// right while the total is below kMost; every thread gets the total.
template <bool CAPPED = false>
__device__ __forceinline__ int block_scan(int v, int& total) {
  __shared__ int warp_s[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x = sum_of<CAPPED>(x, y);
  }
  if (lane == 31) warp_s[warp] = x;
  __syncthreads();
  int w = warp_s[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w = sum_of<CAPPED>(w, y);
  }
  total = __shfl_sync(0xffffffffu, w, 31);
  const int base = warp == 0 ? 0 : __shfl_sync(0xffffffffu, w, warp - 1);
  __syncthreads();  // warp_s may be written again
  return sum_of<CAPPED>(base, x) - v;
}

// The `need` lowest-numbered free pages, in ascending order, into list (as
// many as there are); returns how many there are, at most need.
__device__ int find_free(const int32_t* refs, int pages, int need, int32_t* list) {
  int found = 0;
  for (int p0 = 0; p0 < pages && found < need; p0 += 4 * kThreads) {
    int free[4], n = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + 4 * (int)threadIdx.x + j;
      free[j] = p < pages && refs[p] == 0;
      n += free[j];
    }
    int total;
    int at = found + block_scan(n, total);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (free[j] && at < need) list[at] = p0 + 4 * (int)threadIdx.x + j;
      at += free[j];
    }
    found += total;
  }
  __syncthreads();
  return min(found, need);
}

// Give a sequence's pages back (one warp).
__device__ void release(const Table& t, int slot) {
  const int lane = threadIdx.x & 31;
  const int used = min((t.length[slot] + t.page_size - 1) / t.page_size, t.width);
  int32_t* row = t.table + (int64_t)slot * t.width;
  for (int j = lane; j < used; j += 32) {
    const int p = row[j];
    row[j] = -1;
    if (p < 0 || p >= t.pages || atomicSub(&t.refs[p], 1) <= 0) atomicOr(t.status, DEV_BAD_ARGS);
  }
  __syncwarp();
  if (lane == 0) t.length[slot] = 0;
}

// slot[] in range and distinct (and, with `not_in`, none of those): the same
// answer for every thread.
__device__ bool slots_ok(const Table& t, const int32_t* slot, int n, const int32_t* not_in) {
  bool ok = true;
  if (threadIdx.x < n) {
    const int s = slot[threadIdx.x];
    ok = s >= 0 && s < t.slots;
    for (int i = 0; i < (int)threadIdx.x; ++i) ok = ok && slot[i] != s;
    if (not_in) {
      ok = ok && not_in[threadIdx.x] >= 0 && not_in[threadIdx.x] < t.slots;
      for (int i = 0; i < n; ++i) ok = ok && not_in[i] != s;
    }
  }
  return __syncthreads_and(ok);
}

// A reserve or fork with a bad sequence (one thread).
__device__ __forceinline__ void refuse(const Table& t) {
  *t.shortage = HYQ_PAGES_REFUSED;
  atomicOr(t.status, DEV_BAD_ARGS);
}

__global__ void __launch_bounds__(kThreads)
    reserve_kernel(Table t, const int32_t* slot, const int32_t* extra, int n, int32_t* pos, Plan w) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ int at_s[kMaxSeqs];
  const int i = threadIdx.x;
  bool ok = slots_ok(t, slot, n, nullptr);
  int before = 0, held = 0, need = 0, add = 0;
  if (ok && i < n) {
    before = t.length[slot[i]];
    add = extra[i];
    held = (before + t.page_size - 1) / t.page_size;
    const int64_t after = (int64_t)before + add;
    ok = before >= 0 && add >= 0 && after <= (int64_t)t.width * t.page_size;
    if (ok) need = (int)((after + t.page_size - 1) / t.page_size) - held;
  }
  if (!__syncthreads_and(ok)) {  // what goes on with these positions skips the sequences
    if (pos && i < n) pos[i] = -1;
    if (i == 0) refuse(t);
    return;
  }
  int total;  // (kMost is more than there can be pages)
  const int at = block_scan<true>(need, total);
  at_s[i] = at;
  const int found = total ? find_free(t.refs, t.pages, total, w.to) : 0;
  if (pos && i < n) pos[i] = before;
  if (i == 0) *t.shortage = total - found;
  if (found < total) return;
  __syncthreads();
  for (int s = i >> 5; s < n; s += kThreads / 32) {  // a warp per sequence
    const int a0 = at_s[s], a1 = s + 1 < n ? at_s[s + 1] : total;
    const int have = (t.length[slot[s]] + t.page_size - 1) / t.page_size;
    int32_t* row = t.table + (int64_t)slot[s] * t.width + have;
    for (int j = i & 31; j < a1 - a0; j += 32) {
      const int p = w.to[a0 + j];
      row[j] = p;
      t.refs[p] = 1;
    }
  }
  __syncthreads();
  if (i < n) t.length[slot[i]] = before + add;
}

__global__ void __launch_bounds__(kThreads) free_kernel(Table t, const int32_t* slot, int n) {
  grid_dependency_wait();
  allow_dependents_launch();
  if (!slots_ok(t, slot, n, nullptr)) {
    if (threadIdx.x == 0) atomicOr(t.status, DEV_BAD_ARGS);
    return;
  }
  for (int s = threadIdx.x >> 5; s < n; s += kThreads / 32) release(t, slot[s]);
}

__global__ void __launch_bounds__(kThreads)
    fork_kernel(Table t, const int32_t* src, const int32_t* dst, int n, Plan w) {
  grid_dependency_wait();
  allow_dependents_launch();
  __shared__ int at_s[kMaxSeqs];
  const int i = threadIdx.x;
  if (i == 0) *w.count = 0;
  bool ok = slots_ok(t, dst, n, src);
  int part = 0;
  if (ok && i < n) {
    const int len = t.length[src[i]];
    ok = len >= 0 && len <= (int64_t)t.width * t.page_size;
    part = ok && len % t.page_size != 0;
  }
  if (!__syncthreads_and(ok)) {
    if (i == 0) refuse(t);
    return;
  }
  for (int s = i >> 5; s < n; s += kThreads / 32) release(t, dst[s]);
  __syncthreads();
  int total;
  at_s[i] = block_scan(part, total);
  const int found = total ? find_free(t.refs, t.pages, total, w.to) : 0;
  if (i == 0) *t.shortage = total - found;
  if (found < total) return;
  __syncthreads();
  for (int s = i >> 5; s < n; s += kThreads / 32) {
    const int len = t.length[src[s]], full = len / t.page_size;
    const int32_t* from = t.table + (int64_t)src[s] * t.width;
    int32_t* to = t.table + (int64_t)dst[s] * t.width;
    for (int j = i & 31; j < full; j += 32) {
      const int p = from[j];
      to[j] = p;
      if (p < 0 || p >= t.pages) atomicOr(t.status, DEV_BAD_ARGS);
      else atomicAdd(&t.refs[p], 1);
    }
    if ((i & 31) == 0) {
      t.length[dst[s]] = len;
      if (len % t.page_size) {
        const int p = w.to[at_s[s]];
        to[full] = p;
        t.refs[p] = 1;
        w.from[at_s[s]] = from[full];
      }
    }
  }
  if (i == 0) *w.count = total;
}

__global__ void __launch_bounds__(kThreads) compact_kernel(Table t, Plan w) {
  grid_dependency_wait();
  allow_dependents_launch();
  int live = 0;
  for (int p0 = 0; p0 < t.pages; p0 += kThreads) {
    const int p = p0 + (int)threadIdx.x;
    live += __syncthreads_count(p < t.pages && t.refs[p] > 0);
  }
  // the j-th free page below `live` takes the j-th live page past it
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < t.pages; p0 += kThreads) {
    const int p = p0 + (int)threadIdx.x;
    const bool used = p < t.pages && t.refs[p] > 0;
    const int hole = p < live && !used, mover = p >= live && used;
    int n_hole, n_mover;
    const int at_hole = holes + block_scan(hole, n_hole), at_mover = movers + block_scan(mover, n_mover);
    if (hole) w.to[at_hole] = p;
    if (mover) w.from[at_mover] = p;
    if (p < t.pages) w.name[p] = p;
    holes += n_hole;
    movers += n_mover;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < movers; j += kThreads) {
    const int a = w.from[j], b = w.to[j];
    w.name[a] = b;
    t.refs[b] = t.refs[a];
    t.refs[a] = 0;
  }
  if (threadIdx.x == 0) *w.count = movers;
}

struct Pool {
  char* base;
  int64_t planes, plane_stride, page_stride, page_bytes;
};

// The copies of the plan in every plane, and (rename) the table's entries.
// Bound by memory: a CTA copies 16 KB of a page at a time, four vectors of a
// thread in flight.  The piece (plane, copy, part) is followed up by additions,
// since the divisions that name it by its number took as long as the copy.
// Two waves of CTAs, so that the SMs that are done first get more (500 MB of
// moves 90 us, 5.8 TB/s; 98 with one wave; 67 MB of copies of one page for each
// of 8 forks 15 to 16 us with fork_kernel, 2 more with four waves or 4 KB at a
// time).
constexpr int kCopyThreads = 256, kCopyEach = 4, kCopyCtas = 148 * 16;
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(Table t, Pool pool, Plan w, bool rename) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int count = *w.count;
  if (count <= 0) return;
  if (rename) {
    const int64_t all = (int64_t)gridDim.x * blockDim.x;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (int64_t)t.slots * t.width; i += all) {
      const int p = t.table[i];
      if (p >= 0 && p < t.pages) t.table[i] = w.name[p];
    }
  }
  struct Piece {
    int64_t plane, copy, part;
  };
  constexpr int kPiece = kCopyThreads * kCopyEach;  // vectors
  const int64_t vecs = pool.page_bytes / 16, parts = (vecs + kPiece - 1) / kPiece;
  auto piece_of = [&](int64_t i) {
    const int64_t c = i / parts, plane = c / count;
    return Piece{plane, c - plane * count, i - c * parts};
  };
  Piece at = piece_of(blockIdx.x);
  const Piece step = piece_of(gridDim.x);
  while (at.plane < pool.planes) {
    const int from = w.from[at.copy];
    if (from >= 0 && from < t.pages) {
      const int64_t vec = at.part * kPiece + threadIdx.x;
      char* base = pool.base + at.plane * pool.plane_stride + 16 * vec;
      const uint4* src = reinterpret_cast<const uint4*>(base + from * pool.page_stride);
      uint4* dst = reinterpret_cast<uint4*>(base + w.to[at.copy] * pool.page_stride);
      uint4 v[kCopyEach];
#pragma unroll
      for (int e = 0; e < kCopyEach; ++e)
        if (vec + e * kCopyThreads < vecs) v[e] = src[e * kCopyThreads];
#pragma unroll
      for (int e = 0; e < kCopyEach; ++e)
        if (vec + e * kCopyThreads < vecs) dst[e * kCopyThreads] = v[e];
    } else {
      atomicOr(t.status, DEV_BAD_ARGS);
    }
    at.part += step.part;
    at.copy += step.copy;
    at.plane += step.plane;
    if (at.part >= parts) {
      at.part -= parts;
      ++at.copy;
    }
    if (at.copy >= count) {
      at.copy -= count;
      ++at.plane;
    }
  }
}

}  // namespace pages
}  // namespace hyq

namespace {

using hyq::api_fail;

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int make_table(const hyq_pages* p, const char* name, hyq::pages::Table& t) {
  if (!p || !p->table || !p->length || !p->refs || !p->shortage) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (p->slots <= 0 || p->slots > INT32_MAX || p->table_width <= 0 || p->page_size <= 0 ||
      p->table_width > INT32_MAX / p->page_size || p->pages <= 0 || p->pages > INT32_MAX - 8192)
    return api_fail(HYQ_E_SHAPE, "%s: shape of the table", name);
  if (!aligned(p->table, 4) || !aligned(p->length, 4) || !aligned(p->refs, 4) || !aligned(p->shortage, 4))
    return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  t = {p->table, p->length, p->refs, p->shortage, (int)p->slots, (int)p->table_width, (int)p->pages, p->page_size, nullptr};
  return hyq::api_status_word(&t.status);
}

int make_pool(const hyq_page_pool* p, const char* name, hyq::pages::Pool& pool) {
  if (!p || !p->base) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (p->planes <= 0 || p->page_bytes <= 0 || p->page_stride < p->page_bytes || p->plane_stride < 0 ||
      (p->planes > 1 && p->plane_stride < p->page_bytes))
    return api_fail(HYQ_E_SHAPE, "%s: shape of the pool", name);
  if (!aligned(p->base, 16) || (p->plane_stride | p->page_stride | p->page_bytes) % 16)
    return api_fail(HYQ_E_ALIGN, "%s: the pool's base, strides and pages are multiples of 16 bytes", name);
  pool = {static_cast<char*>(p->base), p->planes, p->plane_stride, p->page_stride, p->page_bytes};
  return HYQ_OK;
}

int check_workspace(const void* workspace, const char* name) {
  if (!workspace) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (!aligned(workspace, 16)) return api_fail(HYQ_E_ALIGN, "%s: workspace alignment", name);
  return HYQ_OK;
}

// The sequences of a call: how many, and their device arrays.
int check_seqs(int64_t n, const void* a, const void* b, const char* name) {
  if (n < 0 || n > hyq::pages::kMaxSeqs)
    return api_fail(HYQ_E_SHAPE, "%s: at most %d sequences", name, hyq::pages::kMaxSeqs);
  if (n > 0 && (!a || !b)) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (!aligned(a, 4) || !aligned(b, 4)) return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  return HYQ_OK;
}

int done(cudaError_t e, const char* name) {
  return e == cudaSuccess ? HYQ_OK : api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

cudaError_t launch_copy(const hyq::pages::Table& t, const hyq::pages::Pool& pool, const hyq::pages::Plan& w, bool rename,
                        cudaStream_t st) {
  return hyq::launch_next(hyq::pages::copy_kernel, dim3(hyq::pages::kCopyCtas), dim3(hyq::pages::kCopyThreads), 0, st, t,
                          pool, w, rename);
}

}  // namespace

extern "C" {

int hyq_pages_workspace_bytes(int64_t pages, size_t* bytes) {
  if (!bytes) return api_fail(HYQ_E_INVALID, "pages_workspace_bytes: null pointer");
  if (pages <= 0 || pages > INT32_MAX - 8192) return api_fail(HYQ_E_SHAPE, "pages_workspace_bytes: shape");
  *bytes = 16 + 3 * (size_t)pages * sizeof(int32_t);
  return HYQ_OK;
}

int hyq_pages_reserve(const hyq_pages* p, const int32_t* slot, const int32_t* extra, int64_t n, int32_t* pos,
                      void* workspace, void* stream) {
  const char* name = "pages_reserve";
  hyq::pages::Table t;
  int rc = make_table(p, name, t);
  if (rc || (rc = check_workspace(workspace, name)) || (rc = check_seqs(n, slot, extra, name))) return rc;
  return done(hyq::launch_ex(hyq::pages::reserve_kernel, dim3(1), dim3(hyq::pages::kThreads), 0, (cudaStream_t)stream,
                             t, slot, extra, (int)n, pos, hyq::pages::plan_of(workspace, p->pages)),
              name);
}

int hyq_pages_free(const hyq_pages* p, const int32_t* slot, int64_t n, void* stream) {
  const char* name = "pages_free";
  hyq::pages::Table t;
  int rc = make_table(p, name, t);
  if (rc || (rc = check_seqs(n, slot, slot, name))) return rc;
  if (n == 0) return HYQ_OK;
  return done(hyq::launch_ex(hyq::pages::free_kernel, dim3(1), dim3(hyq::pages::kThreads), 0, (cudaStream_t)stream, t,
                             slot, (int)n),
              name);
}

int hyq_pages_fork(const hyq_pages* p, const hyq_page_pool* pool, const int32_t* src, const int32_t* dst, int64_t n,
                   void* workspace, void* stream) {
  const char* name = "pages_fork";
  hyq::pages::Table t;
  hyq::pages::Pool pl;
  int rc = make_table(p, name, t);
  if (rc || (rc = make_pool(pool, name, pl)) || (rc = check_workspace(workspace, name)) ||
      (rc = check_seqs(n, src, dst, name)))
    return rc;
  const hyq::pages::Plan w = hyq::pages::plan_of(workspace, p->pages);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = hyq::launch_ex(hyq::pages::fork_kernel, dim3(1), dim3(hyq::pages::kThreads), 0, st, t, src, dst,
                                 (int)n, w);
  if (e == cudaSuccess && n > 0) e = launch_copy(t, pl, w, false, st);
  return done(e, name);
}

int hyq_pages_compact(const hyq_pages* p, const hyq_page_pool* pool, void* workspace, void* stream) {
  const char* name = "pages_compact";
  hyq::pages::Table t;
  hyq::pages::Pool pl;
  int rc = make_table(p, name, t);
  if (rc || (rc = make_pool(pool, name, pl)) || (rc = check_workspace(workspace, name))) return rc;
  const hyq::pages::Plan w = hyq::pages::plan_of(workspace, p->pages);
  const cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = hyq::launch_ex(hyq::pages::compact_kernel, dim3(1), dim3(hyq::pages::kThreads), 0, st, t, w);
  if (e == cudaSuccess) e = launch_copy(t, pl, w, true, st);
  return done(e, name);
}

}  // extern "C"
