// Operators over a paged KV cache: RoPE + q/k RMSNorm + append of new tokens,
// and attention of the new tokens over the pages (include/hyq.h).
#include <cmath>

#include "../../include/hyq.h"
#include "hyq_kernels.h"
#include "hyq_paged.cuh"
#include "hyq_paged_shared.h"

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
  bool vec;  // 8-bit: the codes of a row are 8-byte aligned
  bool staged;  // the rows of q, k and v are 16-byte aligned
};
// Calls of more rows than append_rows_kernel holds at once (three CTAs an SM) stage
// their rows in shared memory, of up to 64 KB.  Measured, 32 query and 8 kv heads of 128,
// staged / not, f16 cache, us: 1 row 5.1 / 4.1, 256 rows 6.2 / 5.1, 512 rows 7.5 / 8.1,
// 8,208 rows 65 / 77 (int8, with some more to do: 512 rows 10.3 / 11.0, 8,208 rows 77 / 98);
// 8,208 rows of 14 and 2 heads of 64 24 / 41, of 64 and 8 of 128 (int8) 138 / 152.
constexpr int kStageMax = 64 * 1024;
constexpr int kStagedRows = 3 * 148 + 1;

template <Kv KV>
__device__ __forceinline__ void store_kv(void* base, int64_t i, float x) {
  if constexpr (KV == kF16) static_cast<__half*>(base)[i] = __float2half_rn(x);
  else static_cast<float*>(base)[i] = x;
}

// One CTA per row of the activations, 16 lanes per head: lane l holds values
// l, l + 16, ... of its head, so that the sum of squares runs in dot_x86's
// order (one accumulator a lane, then the lane sum) and the two values of a
// rotated pair meet in one thread.  Few rows are bound by latency (64 tokens 3.6 us):
// each group takes BATCH heads at a time, their loads in flight together, and with
// those of the tables.  Many rows (STAGED) come whole, by three bulk copies, while the
// CTA finds their page and tables: the loads above are 4 bytes a lane, and three CTAs an
// SM keep too few of them in flight, where eight CTAs of four warps have a row of 25 KB
// each under way.  Bound by memory and by that search (row, page, tables, one after the
// other): 8,208 tokens of 32 query and 8 kv heads of 128 into an f32 cache (403 MB)
// 69 us, 5.8 TB/s, f16 65 us, e4m3 75 us (353 MB; with the norm after the rotation 77,
// and 88 where weights of a pair are 10 to 50 times each other's: more heads are next to
// borders then and done again).
// Into an 8-bit cache a head's largest magnitude comes from its 16 lanes, and the
// codes go through shared memory, so that a lane writes neighbouring ones.
template <int DIM, Kv KV, bool STAGED>
__global__ void __launch_bounds__(STAGED ? 128 : 256, STAGED ? 8 : 3) append_rows_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int EL = DIM / 16, BATCH = STAGED ? 1 : 3, THREADS = STAGED ? 128 : 256, GROUPS = THREADS / 16;
  __shared__ __align__(8) uint8_t codes_s[is_8bit(KV) ? THREADS : 8][is_8bit(KV) ? EL : 8];  // DIM of each group of 16 lanes
  __shared__ float limit_s[is_8bit(KV) ? THREADS / 32 : 1];  // each warp's border_limit() of keys
  extern __shared__ __align__(16) float stage[];  // STAGED: the row's heads, queries, keys, values
  __shared__ __align__(8) uint64_t bar_s;
  const int t = blockIdx.x, l = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int units = a.heads + 2 * a.c.kv_heads;
  if (STAGED && threadIdx.x == 0) {
    mbar_init(smem_addr(&bar_s), 1);
    mbar_fence_init();
  }
  grid_dependency_wait();
  allow_dependents_launch();
  if constexpr (STAGED) {
    if (threadIdx.x == 0) {
      const uint32_t bar = smem_addr(&bar_s), to = smem_addr(stage), qb = a.heads * DIM * 4, kb = a.c.kv_heads * DIM * 4;
      mbar_arrive_expect_tx(bar, qb + 2 * kb);
      bulk_g2s(to, a.q + t * a.q_stride, qb, bar);
      bulk_g2s(to + qb, a.k + t * a.k_stride, kb, bar);
      bulk_g2s(to + qb + kb, a.v + t * a.v_stride, kb, bar);
    }
    __syncthreads();
  }
  auto source = [&](int u) {
    return u < a.heads                    ? a.q + t * a.q_stride + u * DIM
           : u < a.heads + a.c.kv_heads ? a.k + t * a.k_stride + (u - a.heads) * DIM
                                          : a.v + t * a.v_stride + (u - a.heads - a.c.kv_heads) * DIM;
  };
  float x[BATCH][EL];
  auto load = [&](int u0) {
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int u = u0 + GROUPS * b;
      const float* src = STAGED ? stage + (u < units ? u : 0) * DIM : source(u < units ? u : 0);
#pragma unroll
      for (int i = 0; i < EL; ++i) x[b][i] = u < units ? src[l + 16 * i] : 0.f;
    }
  };
  if (!STAGED) load(part);  // these do not wait for the tables
  float wq[EL], wk[EL];
#pragma unroll
  for (int i = 0; i < EL; ++i) {
    wq[i] = a.q_norm ? a.q_norm[l + 16 * i] : 1.f;
    wk[i] = a.k_norm ? a.k_norm[l + 16 * i] : 1.f;
  }
  if constexpr (is_8bit(KV)) {
    float uneven = 1.f;  // the key weights' largest ratio in a rotated pair, where they come after
    if (a.k_norm && !a.norm_first) {
#pragma unroll
      for (int i = 0; i < EL / 2; ++i) uneven = fmaxf(uneven, ratio_of(wk[i], wk[i + EL / 2]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) uneven = fmaxf(uneven, __shfl_xor_sync(0xffffffffu, uneven, o));
    }
    if ((threadIdx.x & 31) == 0) limit_s[threadIdx.x >> 5] = border_limit<KV>(uneven);
    __syncwarp();
  }
  const int s = seq_of_row(a.c, t);
  const Seq sq = s < 0 ? Seq{} : load_seq(a.c, s);
  const int pos = sq.pos + (t - sq.row0);
  int page = -1;
  if (s >= 0 && t - sq.row0 < sq.n) {
    page = checked_page(a.c, sq.pages[pos / a.c.page_size]);
    if (pos >= a.positions) page = -1;
    if (page < 0 && threadIdx.x == 0) atomicOr(a.c.status, DEV_BAD_ARGS);
  }
  if (page < 0) {
    if (STAGED && threadIdx.x == 0 && !mbar_wait(smem_addr(&bar_s), 0, nullptr)) atomicOr(a.c.status, DEV_TIMEOUT_DRAIN);
    return;
  }
  float cs[EL / 2], sn[EL / 2];
#pragma unroll
  for (int i = 0; i < EL / 2; ++i) {
    cs[i] = a.cos_tab[(int64_t)pos * (DIM / 2) + l + 16 * i];
    sn[i] = a.sin_tab[(int64_t)pos * (DIM / 2) + l + 16 * i];
  }
  const int64_t row = (int64_t)page * a.c.page_stride + (int64_t)(pos % a.c.page_size) * a.c.row_stride;
  const int64_t scales = is_8bit(KV) ? scale_at(a.c, page, 0, pos % a.c.page_size) : 0;
  if (STAGED && !mbar_wait(smem_addr(&bar_s), 0, nullptr)) {
    if (threadIdx.x == 0) {  // (not before the copies are in, if that can be)
      atomicOr(a.c.status, DEV_TIMEOUT_FULL);
      if (!mbar_wait(smem_addr(&bar_s), 0, nullptr)) atomicOr(a.c.status, DEV_TIMEOUT_DRAIN);
    }
    return;
  }
  uint32_t again = 0;  // turns of this warp with codes that f32 leaves open (31: and later ones)
  for (int u0 = part; u0 - part < units; u0 += GROUPS * BATCH) {
    if (STAGED || u0 != part) load(u0);
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int u = u0 + GROUPS * b;
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
      uint32_t top = 0;
      const bool coded = is_8bit(KV) && u - (part & 1) + 1 >= a.heads;  // one of the warp's two heads
      if (coded) {
#pragma unroll
        for (int i = 0; i < EL; ++i) top = max(top, __float_as_uint(x[b][i]) & 0x7fffffffu);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
      }
      if (coded) __syncwarp();  // the codes of the heads before are out
      RowCode code{};
      if constexpr (is_8bit(KV)) if (coded) {
        code = row_code<KV>(top);
        uint8_t* mine = codes_s[threadIdx.x & ~15];
        bool close = false;
        if (!is_q && u < units) {
          float edge = KV == kI8 ? 0.f : INFINITY;
          uint8_t codes[EL];
#pragma unroll
          for (int i = 0; i < EL; ++i) codes[i] = encode<KV>(__fmul_rn(x[b][i], code.inverse), edge);
#pragma unroll
          for (int i = 0; i < EL; ++i) mine[l + 16 * i] = code.inverse == 0.f ? 0 : codes[i];
          close = code.inverse != 0.f && near_border<KV>(edge, rotated ? limit_s[threadIdx.x >> 5] : border_limit<KV>(kUnrotated));
        }
        const int turn = min((u - part) / GROUPS, 31);
        if (__any_sync(0xffffffffu, close)) again |= 1u << turn;
        __syncwarp();
      }
      if (u >= units) continue;
      if (is_q) {
        float* to = a.q_out + t * a.out_stride + u * DIM + l;
#pragma unroll
        for (int i = 0; i < EL; ++i) to[16 * i] = x[b][i];
      } else {
        const int kh = (u - a.heads) % a.c.kv_heads;
        const int64_t to = row + kh * a.c.head_stride + l;
        void* base = rotated ? a.c.k : a.c.v;
        if constexpr (is_8bit(KV)) {
          uint8_t* y = static_cast<uint8_t*>(base) + to + (EL - 1) * l;
          const uint8_t* from = codes_s[threadIdx.x];
          if (a.vec) {
            if constexpr (EL == 8) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(from);
            else *reinterpret_cast<uint32_t*>(y) = *reinterpret_cast<const uint32_t*>(from);
          } else {
#pragma unroll
            for (int i = 0; i < EL; ++i) y[i] = from[i];
          }
          if (l == 0) (rotated ? a.c.k_scale : a.c.v_scale)[scales + kh * a.c.scale_head_stride] = code.scale;
        } else {
#pragma unroll
          for (int i = 0; i < EL; ++i) store_kv<KV>(base, to + 16 * i, x[b][i]);
        }
      }
    }
  }
  // Those codes in 64 bits, without the row's norm, which they do not depend on.  (After
  // the others, when the registers are free: amid them 87 us where this took 80.)
  if constexpr (is_8bit(KV)) {
    if (!again) return;
    __syncwarp();  // the codes and scales from above are written
    for (int turn = 0; turn * GROUPS < units; ++turn) {
      if (!(again >> min(turn, 31) & 1)) continue;
      const int u = part + GROUPS * turn, kh = (u - a.heads) % a.c.kv_heads;
      const bool coded = u >= a.heads && u < units, key = u < a.heads + a.c.kv_heads;
      const float* src = (STAGED ? stage + (coded ? u : 0) * DIM : source(coded ? u : 0)) + l;
      double y[EL], largest = 0;
#pragma unroll
      for (int i = 0; i < EL; ++i) y[i] = src[16 * i];
      if (key) {
#pragma unroll
        for (int i = 0; i < EL / 2; ++i) {
          const double w0 = wk[i], w1 = wk[i + EL / 2], c = cs[i], n = sn[i];
          const double x0 = a.norm_first ? y[i] * w0 : y[i], x1 = a.norm_first ? y[i + EL / 2] * w1 : y[i + EL / 2];
          y[i] = x0 * c - x1 * n;
          y[i + EL / 2] = x0 * n + x1 * c;
          if (!a.norm_first) y[i] *= w0, y[i + EL / 2] *= w1;
        }
      }
#pragma unroll
      for (int i = 0; i < EL; ++i) largest = fmax(largest, fabs(y[i]));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) largest = fmax(largest, __shfl_xor_sync(0xffffffffu, largest, o));
      if (!coded || !((key ? a.c.k_scale : a.c.v_scale)[scales + kh * a.c.scale_head_stride] > 0.f)) continue;  // 0, NaN: codes are 0
      uint8_t* to = static_cast<uint8_t*>(key ? a.c.k : a.c.v) + row + kh * a.c.head_stride + l;
      const double inverse = kLargest<KV> / largest;
#pragma unroll
      for (int i = 0; i < EL; ++i) to[16 * i] = encode<KV>(y[i] * inverse);
    }
  }
}

// Any other even head size: a warp per head at a time, the head in
// shared memory; sums in the order of dot_x86.
template <Kv KV>
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
  // a head's values into an 8-bit cache: x in f32, value(i) in 64 bits up to a factor
  auto quantise = [&](const float* x, auto value, void* base, float* scale_base, int kh) {
    uint32_t top = 0;
    double largest = 0;
    for (int i = lane; i < dim; i += 32) {
      top = max(top, __float_as_uint(x[i]) & 0x7fffffffu);
      largest = fmax(largest, fabs(value(i)));
    }
    const RowCode code = row_code<KV>(__reduce_max_sync(0xffffffffu, top));
    for (int o = 16; o > 0; o >>= 1) largest = fmax(largest, __shfl_xor_sync(0xffffffffu, largest, o));
    const double inverse = kLargest<KV> / largest;
    for (int i = lane; i < dim; i += 32)
      static_cast<uint8_t*>(base)[row + kh * a.c.head_stride + i] = code.inverse == 0.f ? 0 : encode<KV>(value(i) * inverse);
    if (lane == 0) scale_base[scale_at(a.c, page, kh, pos % a.c.page_size)] = code.scale;
  };
  for (int u = warp; u < a.heads + 2 * a.c.kv_heads; u += 8) {
    if (u >= a.heads + a.c.kv_heads) {  // a value head: copied as it is
      const int kh = u - a.heads - a.c.kv_heads;
      const float* x = a.v + t * a.v_stride + kh * dim;
      if constexpr (is_8bit(KV)) {
        quantise(x, [&](int i) { return (double)x[i]; }, a.c.v, a.c.v_scale, kh);
      } else {
        for (int i = lane; i < dim; i += 32) store_kv<KV>(a.c.v, row + kh * a.c.head_stride + i, x[i]);
      }
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
    if (is_8bit(KV) && !is_q) {
      if constexpr (is_8bit(KV)) {
        auto value = [&](int i) {
          const int j = i < half ? i : i - half;
          const double w0 = w && a.norm_first ? w[j] : 1.f, w1 = w && a.norm_first ? w[j + half] : 1.f;
          const double x0 = x[j] * w0, x1 = x[j + half] * w1;
          const double y = i < half ? x0 * cs[j] - x1 * sn[j] : x0 * sn[j] + x1 * cs[j];
          return w && !a.norm_first ? y * w[i] : y;
        };
        quantise(h, value, a.c.k, a.c.k_scale, kh);
      }
      continue;
    }
    for (int i = lane; i < dim; i += 32) {
      if (is_q) a.q_out[t * a.out_stride + u * dim + i] = h[i];
      else store_kv<KV>(a.c.k, row + kh * a.c.head_stride + i, h[i]);
    }
  }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

template <Kv KV>
__device__ __forceinline__ float load_kv(const void* base, int64_t i) {
  if constexpr (KV == kF16) return __half2float(static_cast<const __half*>(base)[i]);
  else if constexpr (KV == kF32) return static_cast<const float*>(base)[i];
  else return code_value<KV>(static_cast<const uint8_t*>(base)[i]);
}

// Any head size, strides and page size.  One CTA per (row, kv head): chunks
// of 32 positions staged in shared memory as f32, one thread per (query head,
// position) score, a running maximum and sum per query head (online softmax),
// OUTS outputs of the group's heads x dim per thread in registers.  Reads
// only positions the row sees.  For what the others do not take: head sizes
// other than 64 and 128, rows that are not 16-byte aligned.  (Of an 8-bit cache it
// stages code * scale.)
constexpr int kChunk = 32;
constexpr int kThreads = 128;

template <Kv KV, int OUTS>
__global__ void __launch_bounds__(kThreads) attend_kernel(const __grid_constant__ AttendArgs a) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x, kvh = blockIdx.y, dim = a.c.dim, G = a.heads / a.c.kv_heads;
  if (a.groups.n && kvh == 0) check_groups<int64_t>(a.c, a.groups);
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
      float k_unit = 1.f, v_unit = 1.f;
      if constexpr (is_8bit(KV)) {
        const int64_t s = scale_at(a.c, max(page, 0), kvh, p % a.c.page_size);
        k_unit = page < 0 ? 0.f : a.c.k_scale[s];
        v_unit = page < 0 ? 0.f : a.c.v_scale[s];
      }
      for (int d = threadIdx.x & 31; d < dim; d += 32) {
        k_s[i * ks + d] = page < 0 ? 0.f : load_kv<KV>(a.c.k, at + d);
        v_s[i * ks + d] = page < 0 ? 0.f : load_kv<KV>(a.c.v, at + d);
        if constexpr (is_8bit(KV)) {
          k_s[i * ks + d] *= k_unit;
          v_s[i * ks + d] *= v_unit;
        }
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
    if (!is_8bit(KV) && !isfinite(y) && isfinite(l)) {
      const float x = non_finite<KV == kF16, 1>(a.c, sq, kvh, -1, seen - 1, i % dim).v[0];
      if (x != 0.f) y = x;
    }
    a.out[t * a.out_stride + (int64_t)kvh * G * dim + i] = y;
  }
}

size_t attend_smem(int dim, int group) {
  return sizeof(float) * ((2 * kChunk + group) * (size_t)(dim + 1) + (size_t)group * (kChunk + 3));
}

template <Kv KV>
cudaError_t launch_attend(const AttendArgs& a, cudaStream_t st) {
  const int group = a.heads / a.c.kv_heads, outs = (group * a.c.dim + kThreads - 1) / kThreads;
  const int variant = outs <= 4 ? 0 : outs <= 8 ? 1 : 2;
  auto k = variant == 0 ? attend_kernel<KV, 4> : variant == 1 ? attend_kernel<KV, 8> : attend_kernel<KV, 32>;
  static std::atomic<uint64_t> done[3] = {};
  const cudaError_t e = allow_smem(k, (int)attend_smem(kMaxDim, kMaxGroup), done[variant]);
  if (e != cudaSuccess) return e;
  return launch_ex(k, dim3((unsigned)a.c.tokens, (unsigned)a.c.kv_heads), dim3(kThreads),
                   attend_smem(a.c.dim, group), st, a);
}

// ---------------------------------------------------------------------------
// Reading rows back
// ---------------------------------------------------------------------------

struct GatherArgs {
  Cache c;
  void* k;
  void* v;
  int64_t k_stride, v_stride;  // elements
  bool vec;                    // 16 bytes of a row at a time are aligned, in and out
};

// A warp per row of the output, 16 bytes of the cache a lane (or one value, where
// they are not aligned), four loads in flight.  Bound by memory.
constexpr int kGatherThreads = 64;

template <Kv KV, typename T>
__global__ void __launch_bounds__(kGatherThreads) gather_kernel(const __grid_constant__ GatherArgs a) {
  grid_dependency_wait();
  allow_dependents_launch();
  const int t = blockIdx.x * (kGatherThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31, dim = a.c.dim;
  if (t >= a.c.tokens) return;
  const int s = seq_of_row(a.c, t);
  if (s < 0) return;
  const Seq sq = load_seq(a.c, s);
  if (t - sq.row0 >= sq.n) return;
  const int pos = sq.pos + (t - sq.row0), in_page = pos % a.c.page_size;
  const int page = checked_page(a.c, sq.pages[pos / a.c.page_size]);
  const int64_t row = (int64_t)max(page, 0) * a.c.page_stride + (int64_t)in_page * a.c.row_stride;
  // unit u of `per` values: head u / units of K, then of V
  auto each = [&](int per, auto f) {
    const int units = dim / per, all = 2 * a.c.kv_heads * units;
#pragma unroll 4
    for (int u = lane; u < all; u += 32) {
      const int head = u / units, d = (u - head * units) * per;
      const bool is_k = head < a.c.kv_heads;
      const int kh = is_k ? head : head - a.c.kv_heads;
      float unit = 1.f;
      if constexpr (is_8bit(KV)) unit = page < 0 ? 0.f : (is_k ? a.c.k_scale : a.c.v_scale)[scale_at(a.c, page, kh, in_page)];
      T* to = static_cast<T*>(is_k ? a.k : a.v) + t * (is_k ? a.k_stride : a.v_stride) + (int64_t)kh * dim + d;
      f(is_k ? a.c.k : a.c.v, row + (int64_t)kh * a.c.head_stride + d, unit, to);
    }
  };
  if (a.vec) {
    constexpr int PER = 16 / value_bytes(KV);
    each(PER, [&](const void* base, int64_t at, float unit, T* to) {
      const uint4 w = *reinterpret_cast<const uint4*>(static_cast<const char*>(base) + at * value_bytes(KV));
      const uint32_t in[4] = {w.x, w.y, w.z, w.w};
      float x[PER];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (KV == kF32) {
          x[i] = __uint_as_float(in[i]);
        } else if constexpr (KV == kF16) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&in[i]));
          x[2 * i] = f.x, x[2 * i + 1] = f.y;
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) x[4 * i + k] = code_value<KV>((uint8_t)(in[i] >> (8 * k))) * unit;
        }
      }
      if (page < 0) {
#pragma unroll
        for (int i = 0; i < PER; ++i) x[i] = 0.f;
      }
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < PER; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
      } else if constexpr (PER == 4) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_f16(x[0], x[1]), pack_f16(x[2], x[3]));
      } else {
#pragma unroll
        for (int i = 0; i < PER; i += 8)
          *reinterpret_cast<uint4*>(to + i) = make_uint4(pack_f16(x[i], x[i + 1]), pack_f16(x[i + 2], x[i + 3]),
                                                         pack_f16(x[i + 4], x[i + 5]), pack_f16(x[i + 6], x[i + 7]));
      }
    });
  } else {
    each(1, [&](const void* base, int64_t at, float unit, T* to) {
      *to = (T)(page < 0 ? 0.f : load_kv<KV>(base, at) * unit);
    });
  }
}

template <Kv KV>
cudaError_t launch_gather(const GatherArgs& a, bool f16, cudaStream_t st) {
  constexpr int per = kGatherThreads / 32;
  return launch_ex(f16 ? gather_kernel<KV, __half> : gather_kernel<KV, float>, dim3((unsigned)((a.c.tokens + per - 1) / per)),
                   dim3(kGatherThreads), 0, st, a);
}

template <Kv KV>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t st) {
  const int64_t bytes = (int64_t)(a.heads + 2 * a.c.kv_heads) * a.c.dim * 4;
  if (a.staged && (a.c.dim == 128 || a.c.dim == 64) && bytes <= kStageMax && a.c.tokens >= kStagedRows) {
    static std::atomic<uint64_t> set[2];
    auto kern = a.c.dim == 128 ? append_rows_kernel<128, KV, true> : append_rows_kernel<64, KV, true>;
    const cudaError_t e = allow_smem(kern, kStageMax, set[a.c.dim == 128]);
    return e != cudaSuccess ? e : launch_ex(kern, dim3((unsigned)a.c.tokens), dim3(128), (size_t)bytes, st, a);
  }
  auto kern = a.c.dim == 128 ? append_rows_kernel<128, KV, false> : a.c.dim == 64 ? append_rows_kernel<64, KV, false> : append_kernel<KV>;
  return launch_ex(kern, dim3((unsigned)a.c.tokens), dim3(256), 0, st, a);
}

}  // namespace paged
}  // namespace hyq

// ---------------------------------------------------------------------------
// C ABI
// ---------------------------------------------------------------------------
namespace {

using hyq::api_fail;

bool aligned(const void* p, size_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }

// kv8: the same cache's scales, where the call takes 8-bit ones.
int make_cache(const hyq_paged_kv* kv, const hyq_paged_kv8* kv8, const hyq_paged_batch* b, int heads, const char* name,
               bool attends, hyq::paged::Cache& c) {
  if (!kv || !b || !kv->k || !kv->v || !kv->table || (b->seqs > 0 && (!b->row_start || !b->pos)))
    return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  const bool coded = kv8 && (kv->dtype == HYQ_KV_I8 || kv->dtype == HYQ_KV_F8);
  if (kv->dtype != HYQ_KV_F32 && kv->dtype != HYQ_KV_F16 && !coded)
    return api_fail(HYQ_E_INVALID, "%s: unknown cache type %d", name, kv->dtype);
  if (coded && (!kv8->k_scale || !kv8->v_scale)) return api_fail(HYQ_E_INVALID, "%s: an 8-bit cache without scales", name);
  if (coded && (kv8->scale_page_stride <= 0 || kv8->scale_head_stride <= 0 || kv8->scale_row_stride <= 0))
    return api_fail(HYQ_E_SHAPE, "%s: strides of the scales", name);
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
  const size_t esize = hyq::paged::value_bytes((hyq::paged::Kv)kv->dtype);
  if (coded && (!aligned(kv8->k_scale, 4) || !aligned(kv8->v_scale, 4)))
    return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
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
  if (coded) {
    c.k_scale = kv8->k_scale;
    c.v_scale = kv8->v_scale;
    c.scale_page_stride = kv8->scale_page_stride;
    c.scale_head_stride = kv8->scale_head_stride;
    c.scale_row_stride = kv8->scale_row_stride;
  }
  return hyq::api_status_word(&c.status);
}

int done(cudaError_t e, const char* name) {
  return e == cudaSuccess ? HYQ_OK : api_fail(HYQ_E_CUDA, "%s: %s", name, cudaGetErrorString(e));
}

int rope_append(const hyq_paged_kv* kv, const hyq_paged_kv8* kv8, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                int heads, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                          const float* cos_tab, const float* sin_tab, int64_t positions, const float* q_norm,
                          const float* k_norm, float eps, int norm_first, float* q_out, int64_t out_stride,
                          void* stream) {
  const char* name = "paged_rope_append";
  hyq::paged::AppendArgs a{};
  const int rc = make_cache(kv, kv8, batch, heads, name, false, a.c);
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
  a.vec = a.c.dim % 8 == 0 && ((a.c.page_stride | a.c.head_stride | a.c.row_stride) & 7) == 0 && aligned(a.c.k, 8) && aligned(a.c.v, 8);
  a.staged = aligned(q, 16) && aligned(k, 16) && aligned(v, 16) && ((q_stride | k_stride | v_stride) & 3) == 0;
  const cudaStream_t st = (cudaStream_t)stream;
  switch (kv->dtype) {
    case kF32: return done(launch_append<kF32>(a, st), name);
    case kF16: return done(launch_append<kF16>(a, st), name);
    case kI8: return done(launch_append<kI8>(a, st), name);
    default: return done(launch_append<kF8>(a, st), name);
  }
}

// The checks of an attention call; `nothing`: it has nothing to do.
int attend_args(const hyq_paged_kv* kv, const hyq_paged_kv8* kv8, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                int heads, float* out, int64_t out_stride, void* workspace, const char* name, hyq::paged::AttendArgs& a,
                bool& nothing) {
  nothing = true;
  const int rc = make_cache(kv, kv8, batch, heads, name, true, a.c);
  if (rc) return rc;
  if (batch->seqs == 0 || batch->tokens == 0 || batch->max_new == 0) return HYQ_OK;
  if (!q || !out || !workspace) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  const int64_t qw = (int64_t)heads * kv->head_dim;
  if (q_stride < qw || out_stride < qw) return api_fail(HYQ_E_SHAPE, "%s: shape of the activations", name);
  if (q == out && q_stride != out_stride && batch->tokens > 1) return api_fail(HYQ_E_SHAPE, "%s: in place with two strides", name);
  if (!aligned(q, 4) || !aligned(out, 4) || !aligned(workspace, 16))
    return api_fail(HYQ_E_ALIGN, "%s: alignment of q, out or the workspace", name);
  a.q = q;
  a.q_stride = q_stride;
  a.heads = heads;
  a.out = out;
  a.out_stride = out_stride;
  a.ws = workspace;
  nothing = false;
  return HYQ_OK;
}

int attend(const hyq::paged::AttendArgs& a, hyq::paged::Kv type, int64_t max_new, int64_t max_len, const char* name,
           cudaStream_t st) {
  using namespace hyq::paged;
  if (mma_supported(a, type)) {
    cudaError_t e;
    if (max_new * (a.heads / a.c.kv_heads) <= kFewRows) {
      e = launch_few(a, type, max_new, false, st);
    } else if (chunks_short(a, type, max_len) || !chunks_tc_supported(a, type)) {
      e = launch_chunks(a, type, st);
      if (e == cudaSuccess) e = launch_few(a, type, max_new, true, st);
    } else {
      e = launch_chunks_tc(a, type, st);
    }
    return done(e, name);
  }
  switch (type) {
    case kF32: return done(launch_attend<kF32>(a, st), name);
    case kF16: return done(launch_attend<kF16>(a, st), name);
    case kI8: return done(launch_attend<kI8>(a, st), name);
    default: return done(launch_attend<kF8>(a, st), name);
  }
}

int attention(const hyq_paged_kv* kv, const hyq_paged_kv8* kv8, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
              int heads, float* out, int64_t out_stride, void* workspace, void* stream) {
  const char* name = "paged_attention";
  hyq::paged::AttendArgs a{};
  bool nothing;
  const int rc = attend_args(kv, kv8, batch, q, q_stride, heads, out, out_stride, workspace, name, a, nothing);
  if (rc || nothing) return rc;
  return attend(a, (hyq::paged::Kv)kv->dtype, batch->max_new, batch->max_len, name, (cudaStream_t)stream);
}

}  // namespace

extern "C" {

int hyq_paged_rope_append(const hyq_paged_kv* kv, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                          int heads, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                          const float* cos_tab, const float* sin_tab, int64_t positions, const float* q_norm,
                          const float* k_norm, float eps, int norm_first, float* q_out, int64_t out_stride,
                          void* stream) {
  return rope_append(kv, nullptr, batch, q, q_stride, heads, k, k_stride, v, v_stride, cos_tab, sin_tab, positions, q_norm, k_norm,
                     eps, norm_first, q_out, out_stride, stream);
}

int hyq_paged_rope_append_kv8(const hyq_paged_kv8* kv, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                              int heads, const float* k, int64_t k_stride, const float* v, int64_t v_stride,
                              const float* cos_tab, const float* sin_tab, int64_t positions, const float* q_norm,
                              const float* k_norm, float eps, int norm_first, float* q_out, int64_t out_stride,
                              void* stream) {
  return rope_append(kv ? &kv->kv : nullptr, kv, batch, q, q_stride, heads, k, k_stride, v, v_stride, cos_tab, sin_tab, positions,
                     q_norm, k_norm, eps, norm_first, q_out, out_stride, stream);
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
  return attention(kv, nullptr, batch, q, q_stride, heads, out, out_stride, workspace, stream);
}

int hyq_paged_attention_kv8(const hyq_paged_kv8* kv, const hyq_paged_batch* batch, const float* q, int64_t q_stride,
                            int heads, float* out, int64_t out_stride, void* workspace, void* stream) {
  return attention(kv ? &kv->kv : nullptr, kv, batch, q, q_stride, heads, out, out_stride, workspace, stream);
}

int hyq_paged_attention_shared_workspace_bytes(int heads, int head_dim, int64_t tokens, size_t* bytes) {
  const char* name = "paged_attention_shared_workspace_bytes";
  if (!bytes) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (heads <= 0 || heads > 1 << 16 || head_dim <= 0 || head_dim > hyq::paged::kMaxDim || tokens < 0 || tokens > INT32_MAX)
    return api_fail(HYQ_E_SHAPE, "%s: shape", name);
  *bytes = hyq::paged::shared_workspace_bytes(heads, head_dim, tokens);
  return HYQ_OK;
}

int hyq_paged_attention_shared(const hyq_paged_kv8* kv, const hyq_paged_batch* batch, const int32_t* group_start,
                               const int32_t* shared, int64_t groups, int64_t max_shared, const float* q, int64_t q_stride,
                               int heads, float* out, int64_t out_stride, void* workspace, void* stream) {
  const char* name = "paged_attention_shared";
  using namespace hyq::paged;
  AttendArgs a{};
  bool nothing;
  const int rc = attend_args(kv ? &kv->kv : nullptr, kv, batch, q, q_stride, heads, out, out_stride, workspace, name, a, nothing);
  if (rc || nothing) return rc;
  if (groups < 0 || groups > kMaxSeqs || max_shared < 0 || max_shared > batch->max_len)
    return api_fail(HYQ_E_SHAPE, "%s: shape of the groups", name);
  if (batch->max_new * (heads / kv->kv.kv_heads) > kFewRows)
    return api_fail(HYQ_E_SHAPE, "%s: at most %d rows (new tokens x query heads per kv head) of a sequence", name, kFewRows);
  if (groups > 0 && (!group_start || !shared)) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  if (!aligned(group_start, 4) || !aligned(shared, 4))
    return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  const Kv type = (Kv)kv->kv.dtype;
  const cudaStream_t st = (cudaStream_t)stream;
  a.groups.start = group_start;
  a.groups.shared = shared;
  a.groups.n = (int)groups;
  a.groups.max_new = batch->max_new;
  // (its kernels of few rows look the groups over)
  if (!shared_supported(a, type) || !worth_sharing(a, type, groups, max_shared))
    return attend(a, type, batch->max_new, batch->max_len, name, st);
  return done(launch_shared(a, type, st), name);
}

int hyq_paged_gather(const hyq_paged_kv8* kv, const hyq_paged_batch* batch, int f16, void* k, int64_t k_stride, void* v,
                     int64_t v_stride, void* stream) {
  const char* name = "paged_gather";
  using namespace hyq::paged;
  GatherArgs a{};
  const int rc = make_cache(kv ? &kv->kv : nullptr, kv, batch, kv ? kv->kv.kv_heads : 1, name, false, a.c);
  if (rc) return rc;
  if (batch->seqs == 0 || batch->tokens == 0) return HYQ_OK;
  if (!k || !v) return api_fail(HYQ_E_INVALID, "%s: null pointer", name);
  const int64_t width = (int64_t)a.c.kv_heads * a.c.dim;
  if (k_stride < width || v_stride < width) return api_fail(HYQ_E_SHAPE, "%s: shape of the outputs", name);
  const size_t esize = f16 ? 2 : 4;
  if (!aligned(k, esize) || !aligned(v, esize)) return api_fail(HYQ_E_ALIGN, "%s: a pointer is not aligned to its element size", name);
  const Kv type = (Kv)kv->kv.dtype;
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  const int per = 16 / value_bytes(type), align = f16 && per == 4 ? 8 : 16;  // values of 16 bytes; alignment of what they make
  a.vec = (a.c.dim | a.c.page_stride | a.c.head_stride | a.c.row_stride) % per == 0 && aligned(a.c.k, 16) && aligned(a.c.v, 16) &&
          a.c.dim * esize % align == 0 && k_stride * esize % align == 0 && v_stride * esize % align == 0 && aligned(k, align) &&
          aligned(v, align);
  const cudaStream_t st = (cudaStream_t)stream;
  switch (type) {
    case kF32: return done(launch_gather<kF32>(a, f16, st), name);
    case kF16: return done(launch_gather<kF16>(a, f16, st), name);
    case kI8: return done(launch_gather<kI8>(a, f16, st), name);
    default: return done(launch_gather<kF8>(a, f16, st), name);
  }
}

}  // extern "C"
