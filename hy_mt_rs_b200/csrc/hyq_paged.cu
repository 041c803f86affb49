// Operators over a paged KV cache: RoPE + q/k RMSNorm + append of new tokens,
// and attention of the new tokens over the pages (include/hyq.h).
#include <cmath>

#include "../../include/hyq.h"
#include "hyq_kernels.h"
#include "hyq_paged.cuh"

namespace hyq {
namespace paged {

// ---------------------------------------------------------------------------
// RoPE + RMSNorm + append
// ---------------------------------------------------------------------------

struct AppendArgs {
  Cache c;
  const float* q;
  const float* k;
  const float* v;
  int64_t q_stride, k_stride, v_stride;
  int heads;
  const float* cos_tab;  // [positions, dim / 2]
  const float* sin_tab;
  int64_t positions;
  const float* q_norm;   // [dim] or null
  const float* k_norm;
  float eps;
  int norm_first;
  float* q_out;
  int64_t out_stride;
};

template <bool KV16>
__device__ __forceinline__ void store_kv(void* base, int64_t i, float x) {
  if constexpr (KV16) static_cast<__half*>(base)[i] = __float2half_rn(x);
  else static_cast<float*>(base)[i] = x;
}

// One CTA per row of the activations, 16 lanes per head: lane l holds values
// l, l + 16, ... of its head, so that the sum of squares runs in dot_x86's
// order (one accumulator a lane, then the lane sum) and the two values of a
// rotated pair meet in one thread: no value leaves its registers between the
// load and the store.  Each group takes BATCH heads at a time, their loads in
// flight together, and with those of the tables.  Bound by memory: 8,208 tokens
// of 32 query and 8 kv heads of 128 into an f32 cache (403 MB) 84 us, 4.8 TB/s, in
// accesses of 4 bytes a lane, 64 contiguous bytes of a head, with 35 % of the warps
// (108 us with registers for six CTAs an SM instead of three); 64 tokens 3.6 us.
template <int DIM, bool KV16>
__global__ void __launch_bounds__(256) append_rows_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int EL = DIM / 16, BATCH = 3;
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x, l = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int units = a.heads + 2 * a.c.kv_heads;
  auto source = [&](int u) {
    return u < a.heads                    ? a.q + t * a.q_stride + u * DIM
           : u < a.heads + a.c.kv_heads ? a.k + t * a.k_stride + (u - a.heads) * DIM
                                          : a.v + t * a.v_stride + (u - a.heads - a.c.kv_heads) * DIM;
  };
  float x[BATCH][EL];
  auto load = [&](int u0) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int u = u0 + 16 * b;
      const float* src = source(u < units ? u : 0);
#pragma unroll
      for (int i = 0; i < EL; ++i) x[b][i] = u < units ? src[l + 16 * i] : 0.f;
    }
  };
  load(part);  // these do not wait for the tables
  float wq[EL], wk[EL];
#pragma unroll
  for (int i = 0; i < EL; ++i) {
    wq[i] = a.q_norm ? a.q_norm[l + 16 * i] : 1.f;
    wk[i] = a.k_norm ? a.k_norm[l + 16 * i] : 1.f;
  }
  const int s = seq_of_row(a.c, t);
  if (s < 0) return;
  const Seq sq = load_seq(a.c, s);
  if (t - sq.row0 >= sq.n) return;
  const int pos = sq.pos + (t - sq.row0);
  const int page = checked_page(a.c, sq.pages[pos / a.c.page_size]);
  if (page < 0 || pos >= a.positions) {
    if (threadIdx.x == 0) atomicOr(a.c.status, DEV_BAD_ARGS);
    return;
  }
  float cs[EL / 2], sn[EL / 2];
#pragma unroll
  for (int i = 0; i < EL / 2; ++i) {
    cs[i] = a.cos_tab[(int64_t)pos * (DIM / 2) + l + 16 * i];
    sn[i] = a.sin_tab[(int64_t)pos * (DIM / 2) + l + 16 * i];
  }
  const int64_t row = (int64_t)page * a.c.page_stride + (int64_t)(pos % a.c.page_size) * a.c.row_stride;
  for (int u0 = part; u0 - part < units; u0 += 16 * BATCH) {
    if (u0 != part) load(u0);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int u = u0 + 16 * b;
      if (u - part >= units) break;  // the same for the whole CTA
      const bool rotated = u < a.heads + a.c.kv_heads, is_q = u < a.heads;
      const float* w = is_q ? a.q_norm : a.k_norm;
      auto norm = [&]() {
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < EL; ++i) acc = fmaf(x[b][i], x[b][i], acc);
        const float d = x86_lane_sum(acc, 0xffffffffu);
        const float scale = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(d, (float)DIM), a.eps)));
        if (w && rotated) {
#pragma unroll
          for (int i = 0; i < EL; ++i) x[b][i] = __fmul_rn(__fmul_rn(x[b][i], scale), is_q ? wq[i] : wk[i]);
        }
      };
      if (a.norm_first) norm();
      if (rotated) {
#pragma unroll
        for (int i = 0; i < EL / 2; ++i) {
          const float x0 = x[b][i], x1 = x[b][i + EL / 2];
          x[b][i] = __fsub_rn(__fmul_rn(x0, cs[i]), __fmul_rn(x1, sn[i]));
          x[b][i + EL / 2] = __fadd_rn(__fmul_rn(x0, sn[i]), __fmul_rn(x1, cs[i]));
        }
      }
      if (!a.norm_first) norm();
      if (u >= units) continue;
      if (is_q) {
        float* to = a.q_out + t * a.out_stride + u * DIM + l;
#pragma unroll
        for (int i = 0; i < EL; ++i) to[16 * i] = x[b][i];
      } else {
        const int kh = (u - a.heads) % a.c.kv_heads;
        const int64_t to = row + kh * a.c.head_stride + l;
#pragma unroll
        for (int i = 0; i < EL; ++i) store_kv<KV16>(rotated ? a.c.k : a.c.v, to + 16 * i, x[b][i]);
      }
    }
  }
}

// Any other even head size: a warp per head at a time, the head in
// shared memory; sums in the order of dot_x86.
template <bool KV16>
__global__ void __launch_bounds__(256) append_kernel(const __grid_constant__ AppendArgs a) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int s = seq_of_row(a.c, t);
  if (s < 0) return;
  const Seq q = load_seq(a.c, s);
  if (t - q.row0 >= q.n) return;
  const int pos = q.pos + (t - q.row0), dim = a.c.dim, half = dim / 2;
  const int page = checked_page(a.c, q.pages[pos / a.c.page_size]);
  if (page < 0 || pos >= a.positions) {
    if (threadIdx.x == 0) atomicOr(a.c.status, DEV_BAD_ARGS);
    return;
  }
  __shared__ float hs[8][kMaxDim];
  float* h = hs[warp];
  const float* cs = a.cos_tab + (int64_t)pos * half;
  const float* sn = a.sin_tab + (int64_t)pos * half;
  const int64_t row = (int64_t)page * a.c.page_stride + (int64_t)(pos % a.c.page_size) * a.c.row_stride;
  for (int u = warp; u < a.heads + 2 * a.c.kv_heads; u += 8) {
    if (u >= a.heads + a.c.kv_heads) {  // a value head: copied as it is
      const int kh = u - a.heads - a.c.kv_heads;
      const float* x = a.v + t * a.v_stride + kh * dim;
      for (int i = lane; i < dim; i += 32) store_kv<KV16>(a.c.v, row + kh * a.c.head_stride + i, x[i]);
      continue;
    }
    const bool is_q = u < a.heads;
    const int kh = u - a.heads;
    const float* x = is_q ? a.q + t * a.q_stride + u * dim : a.k + t * a.k_stride + kh * dim;
    const float* w = is_q ? a.q_norm : a.k_norm;
    __syncwarp();
    for (int i = lane; i < dim; i += 32) h[i] = x[i];
    __syncwarp();
    for (int step = 0; step < 2; ++step) {
      if ((step == 0) == (a.norm_first != 0)) {
        if (!w) continue;
        const float d = dot_x86(h, h, dim, 0xffffffffu);
        const float scale = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(d, (float)dim), a.eps)));
        __syncwarp();
        for (int i = lane; i < dim; i += 32) h[i] = __fmul_rn(__fmul_rn(h[i], scale), w[i]);
      } else {
        for (int j = lane; j < half; j += 32) {
          const float x0 = h[j], x1 = h[j + half], c = cs[j], n = sn[j];
          h[j] = __fsub_rn(__fmul_rn(x0, c), __fmul_rn(x1, n));
          h[j + half] = __fadd_rn(__fmul_rn(x0, n), __fmul_rn(x1, c));
        }
      }
      __syncwarp();
    }
    for (int i = lane; i < dim; i += 32) {
      if (is_q) a.q_out[t * a.out_stride + u * dim + i] = h[i];
      else store_kv<KV16>(a.c.k, row + kh * a.c.head_stride + i, h[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

template <bool KV16>
__device__ __forceinline__ float load_kv(const void* base, int64_t i) {
  if constexpr (KV16) return __half2float(static_cast<const __half*>(base)[i]);
  else return static_cast<const float*>(base)[i];
}

// Any head size, strides and page size.  One CTA per (row, kv head): chunks
// of 32 positions staged in shared memory as f32, one thread per (query head,
// position) score, a running maximum and sum per query head (online softmax),
// OUTS outputs of the group's heads x dim per thread in registers.  Reads
// only positions the row sees.  For what the others do not take: head sizes
// other than 64 and 128, rows that are not 16-byte aligned.
constexpr int kChunk = 32;
constexpr int kThreads = 128;

template <bool KV16, int OUTS>
__global__ void __launch_bounds__(kThreads) attend_kernel(const __grid_constant__ AttendArgs a) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x, kvh = blockIdx.y, dim = a.c.dim, G = a.heads / a.c.kv_heads;
  const int s = seq_of_row(a.c, t);
  if (s < 0) return;
  const Seq sq = load_seq(a.c, s);
  if (t - sq.row0 >= sq.n) return;
  const int seen = sq.pos + (t - sq.row0) + 1;
  extern __shared__ float smem[];
  const int ks = dim + 1;
  float* k_s = smem;                   // [kChunk][ks]
  float* v_s = k_s + kChunk * ks;      // [kChunk][ks]
  float* q_s = v_s + kChunk * ks;      // [G][ks]
  float* e_s = q_s + G * ks;           // [G][kChunk]
  float* m_s = e_s + G * kChunk;       // [G] running maximum
  float* l_s = m_s + G;                // [G] running sum
  float* c_s = l_s + G;                // [G] factor of the chunk before
  const float* q = a.q + t * a.q_stride + (int64_t)kvh * G * dim;
  const float scale = 1.0f / sqrtf((float)dim);
  for (int i = threadIdx.x; i < G * dim; i += kThreads) q_s[(i / dim) * ks + i % dim] = q[i] * scale;
  if (threadIdx.x < G) {
    m_s[threadIdx.x] = -INFINITY;
    l_s[threadIdx.x] = 0.f;
  }
  float o[OUTS];
#pragma unroll
  for (int j = 0; j < OUTS; ++j) o[j] = 0.f;
  for (int p0 = 0; p0 < seen; p0 += kChunk) {
    const int n = min(kChunk, seen - p0);
    __syncthreads();
    for (int i = threadIdx.x >> 5; i < n; i += kThreads / 32) {
      const int p = p0 + i, page = checked_page(a.c, sq.pages[p / a.c.page_size]);
      const int64_t at = (int64_t)max(page, 0) * a.c.page_stride + (int64_t)kvh * a.c.head_stride +
                         (int64_t)(p % a.c.page_size) * a.c.row_stride;
      for (int d = threadIdx.x & 31; d < dim; d += 32) {
        k_s[i * ks + d] = page < 0 ? 0.f : load_kv<KV16>(a.c.k, at + d);
        v_s[i * ks + d] = page < 0 ? 0.f : load_kv<KV16>(a.c.v, at + d);
      }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * kChunk; i += kThreads) {
      const int g = i / kChunk, p = i % kChunk;
      float x = -INFINITY;
      if (p < n) {
        x = 0.f;
        for (int d = 0; d < dim; ++d) x = fmaf(q_s[g * ks + d], k_s[p * ks + d], x);
      }
      e_s[i] = x;
    }
    __syncthreads();
    for (int g = threadIdx.x >> 5; g < G; g += kThreads / 32) {
      const float x = e_s[g * kChunk + (threadIdx.x & 31)];
      float m = x;
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
      const float before = m_s[g], now = fmaxf(before, m);
      const float e = x == -INFINITY ? 0.f : expf(x - now);  // (NaN scores stay NaN)
      const float sum = warp_sum(e);
      __syncwarp();
      e_s[g * kChunk + (threadIdx.x & 31)] = e;
      if ((threadIdx.x & 31) == 0) {
        const float f = before == -INFINITY ? 0.f : expf(before - now);
        c_s[g] = f;
        m_s[g] = now;
        l_s[g] = l_s[g] * f + sum;
      }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < OUTS; ++j) {
      const int i = threadIdx.x + j * kThreads;
      if (i >= G * dim) break;
      const int g = i / dim, d = i - g * dim;
      float x = o[j] * c_s[g];
      for (int p = 0; p < n; ++p) x = fmaf(e_s[g * kChunk + p], v_s[p * ks + d], x);
      o[j] = x;
    }
  }
#pragma unroll
  for (int j = 0; j < OUTS; ++j) {
    const int i = threadIdx.x + j * kThreads;
    if (i >= G * dim) break;
    const float l = l_s[i / dim];
    float y = o[j] / l;
    if (!isfinite(y) && isfinite(l)) {
      const float x = non_finite<KV16, 1>(a.c, sq, kvh, -1, seen - 1, i % dim).v[0];
      if (x != 0.f) y = x;
    }
    a.out[t * a.out_stride + (int64_t)kvh * G * dim + i] = y;
  }
}

size_t attend_smem(int dim, int group) {
  return sizeof(float) * ((2 * kChunk + group) * (size_t)(dim + 1) + (size_t)group * (kChunk + 3));
}

template <bool KV16>
cudaError_t launch_attend(const AttendArgs& a, cudaStream_t st) {
  const int group = a.heads / a.c.kv_heads, outs = (group * a.c.dim + kThreads - 1) / kThreads;
  const int variant = outs <= 4 ? 0 : outs <= 8 ? 1 : 2;
  auto k = variant == 0 ? attend_kernel<KV16, 4> : variant == 1 ? attend_kernel<KV16, 8> : attend_kernel<KV16, 32>;
  static std::atomic<uint64_t> done[3] = {};
  const cudaError_t e = allow_smem(k, (int)attend_smem(kMaxDim, kMaxGroup), done[variant]);
  if (e != cudaSuccess) return e;
  return launch_ex(k, dim3((unsigned)a.c.tokens, (unsigned)a.c.kv_heads), dim3(kThreads),
                   attend_smem(a.c.dim, group), st, a);
}

}  // namespace paged
}  // namespace hyq

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
namespace {

using hyq::api_fail;

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

int make_cache(const hyq_paged_kv* kv, const hyq_paged_batch* b, int heads, const char* name, bool attends,
               hyq::paged::Cache& c) {
  if (!kv || !b || !kv->k || !kv->v || !kv->table || (b->seqs > 0 && (!b->row_start || !b->pos)))
    return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (kv->dtype != HYQ_KV_F32 && kv->dtype != HYQ_KV_F16)
    return api_fail(HYQ_E_INVALID, "%s: unknown cache type %d", name, kv->dtype);
  if (kv->kv_heads <= 0 || kv->head_dim <= 0 || kv->page_size <= 0 || kv->pages <= 0 || kv->pages > INT32_MAX ||
      kv->slots <= 0 || kv->slots > INT32_MAX || kv->table_width <= 0 ||
      kv->table_width > (INT32_MAX - hyq::paged::kPastEnd) / kv->page_size)
    return api_fail(HYQ_E_SHAPE, "%s: shape of the cache", name);
  if (heads <= 0 || heads % kv->kv_heads)
    return api_fail(HYQ_E_SHAPE, "%s: %d query heads over %d kv heads", name, heads, kv->kv_heads);
  if (kv->head_dim > hyq::paged::kMaxDim || heads / kv->kv_heads > hyq::paged::kMaxGroup)
    return api_fail(HYQ_E_SHAPE, "%s: head_dim at most %d, at most %d query heads per kv head", name,
                    hyq::paged::kMaxDim, hyq::paged::kMaxGroup);
  if (kv->row_stride < kv->head_dim || kv->head_stride < kv->head_dim || kv->page_stride < kv->head_dim)
    return api_fail(HYQ_E_SHAPE, "%s: strides of the cache overlap", name);
  if (b->seqs < 0 || b->seqs > hyq::paged::kMaxSeqs || b->tokens < 0 || b->tokens > INT32_MAX || b->max_new < 0 ||
      b->max_len < b->max_new || b->max_len > kv->table_width * kv->page_size)
    return api_fail(HYQ_E_SHAPE, "%s: shape of the batch", name);
  if (attends && !hyq::paged::sums_fit(b->seqs, kv->table_width * kv->page_size))
    return api_fail(HYQ_E_SHAPE, "%s: %lld sequences of up to %lld positions: more than the kernels' sums hold", name,
                    (long long)b->seqs, (long long)(kv->table_width * kv->page_size));
  if (!b->slot && b->seqs > kv->slots)
    return api_fail(HYQ_E_SHAPE, "%s: %lld sequences, %lld table rows", name, (long long)b->seqs, (long long)kv->slots);
  const size_t esize = kv->dtype == HYQ_KV_F16 ? 2 : 4;
  if (!aligned(kv->k, esize) || !aligned(kv->v, esize) || !aligned(kv->table, 4) || !aligned(b->row_start, 4) ||
      !aligned(b->pos, 4) || !aligned(b->slot, 4))
    return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  c.k = kv->k;
  c.v = kv->v;
  c.kv_heads = kv->kv_heads;
  c.dim = kv->head_dim;
  c.page_size = kv->page_size;
  c.pages = (int)kv->pages;
  c.page_stride = kv->page_stride;
  c.head_stride = kv->head_stride;
  c.row_stride = kv->row_stride;
  c.table = kv->table;
  c.slots = (int)kv->slots;
  c.width = (int)kv->table_width;
  c.slot = b->slot;
  c.row_start = b->row_start;
  c.pos = b->pos;
  c.seqs = (int)b->seqs;
  c.tokens = (int)b->tokens;
  return hyq::api_status_word(&c.status);
}

int done(cudaError_t e, const char* name) {
  return e == cudaSuccess ? HYQ_OK : api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int hyq_paged_rope_append(const hyq_paged_kv* kv, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                          int heads, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                          const float* cos_tab, const float* sin_tab, int64_t positions, const float* q_norm,
                          const float* k_norm, float eps, int norm_first, float* q_out, int64_t out_stride,
                          void* stream) {
  const char* name = "paged_rope_append";
  hyq::paged::AppendArgs a{};
  const int rc = make_cache(kv, batch, heads, name, false, a.c);
  if (rc) return rc;
  if (batch->seqs == 0 || batch->tokens == 0) return HYQ_OK;
  if (!q || !k || !v || !cos_tab || !sin_tab || !q_out) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (kv->head_dim & 1) return api_fail(HYQ_E_SHAPE, "%s: odd head_dim", name);
  const int64_t qw = (int64_t)heads * kv->head_dim, kw = (int64_t)kv->kv_heads * kv->head_dim;
  if (q_stride < qw || out_stride < qw || k_stride < kw || v_stride < kw || positions <= 0)
    return api_fail(HYQ_E_SHAPE, "%s: shape of the activations", name);
  if (q == q_out && q_stride != out_stride) return api_fail(HYQ_E_SHAPE, "%s: in place with two strides", name);
  for (const void* p : {(const void*)q, (const void*)k, (const void*)v, (const void*)cos_tab, (const void*)sin_tab,
                        (const void*)q_norm, (const void*)k_norm, (const void*)q_out})
    if (!aligned(p, 4)) return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  if (batch->seqs == 0 || batch->tokens == 0) return HYQ_OK;
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.heads = heads;
  a.cos_tab = cos_tab;
  a.sin_tab = sin_tab;
  a.positions = positions;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.eps = eps;
  a.norm_first = norm_first;
  a.q_out = q_out;
  a.out_stride = out_stride;
  using namespace hyq::paged;
  const bool kv16 = kv->dtype == HYQ_KV_F16;
  auto kern = kv->head_dim == 128  ? (kv16 ? append_rows_kernel<128, true> : append_rows_kernel<128, false>)
              : kv->head_dim == 64 ? (kv16 ? append_rows_kernel<64, true> : append_rows_kernel<64, false>)
                                   : (kv16 ? append_kernel<true> : append_kernel<false>);
  return done(hyq::launch_ex(kern, dim3((unsigned)batch->tokens), dim3(256), 0, (cudaStream_t)stream, a), name);
}

int hyq_paged_attention_workspace_bytes(int heads, int head_dim, size_t* bytes) {
  if (!bytes) return api_fail(HYQ_E_INVALID, "paged_attention_workspace_bytes: null pointer");
  if (heads <= 0 || head_dim <= 0 || head_dim > hyq::paged::kMaxDim)
    return api_fail(HYQ_E_SHAPE, "paged_attention_workspace_bytes: shape");
  *bytes = hyq::paged::mma_workspace_bytes(head_dim) + hyq::paged::tc_workspace_bytes(head_dim);
  return HYQ_OK;
}

int hyq_paged_attention(const hyq_paged_kv* kv, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                        int heads, float* out, int64_t out_stride, void* workspace, void* stream) {
  const char* name = "paged_attention";
  hyq::paged::AttendArgs a{};
  const int rc = make_cache(kv, batch, heads, name, true, a.c);
  if (rc) return rc;
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return HYQ_OK;
  if (!q || !out || !workspace) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  const int64_t qw = (int64_t)heads * kv->head_dim;
  if (q_stride < qw || out_stride < qw) return api_fail(HYQ_E_SHAPE, "%s: shape of the activations", name);
  if (!aligned(q, 4) || !aligned(out, 4) || !aligned(workspace, 16))
    return api_fail(HYQ_E_ALIGN, "%s: alignment of q, out or the workspace", name);
  a.q = q;
  a.q_stride = q_stride;
  a.heads = heads;
  a.out = out;
  a.out_stride = out_stride;
  a.ws = workspace;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool kv16 = kv->dtype == HYQ_KV_F16;
  if (hyq::paged::mma_supported(a, kv16)) {
    cudaError_t e;
    if (batch->max_new * (heads / kv->kv_heads) <= hyq::paged::kFewRows) {
      e = hyq::paged::launch_few(a, kv16, false, st);
    } else if (hyq::paged::chunks_short(a, kv16, batch->max_len) ||
               !(kv16 ? hyq::paged::tc_supported(a) : hyq::paged::tc32_supported(a))) {
      e = hyq::paged::launch_chunks(a, kv16, st);
      if (e == cudaSuccess) e = hyq::paged::launch_few(a, kv16, true, st);
    } else {
      e = kv16 ? hyq::paged::launch_chunks_tc(a, st) : hyq::paged::launch_chunks_tc32(a, st);
    }
    return done(e, name);
  }
  return done(kv16 ? hyq::paged::launch_attend<true>(a, st) : hyq::paged::launch_attend<false>(a, st), name);
}

}  // extern "C"
