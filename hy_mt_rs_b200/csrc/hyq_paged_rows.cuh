// What the attention kernels on the warp-level tensor instructions share, head sizes
// 64 and 128: a warp's block of positions and the copies that bring it, its query
// rows over f32 and f16 caches (Rows) and over 8-bit ones (CodeRows).
#pragma once

#include <type_traits>

#include "../../include/hyq.h"
#include "hyq_kernels.h"
#include "hyq_paged.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = kFewRows;      // query rows of a warp at most: (token, head) pairs

// A warp's block of positions: POS rows of K, then of V, in 16-byte chunks
// whose low three index bits are xored with the row (reads by ldmatrix and by
// words then fall into distinct banks; 8-bit caches: place()).  8 KB for head
// size 128.
// NB: query rows of a warp in eights (1: 8-bit caches only).
template <int DIM, Kv KV, int NB = 2>
struct Geo {
  static constexpr int rows = 8 * NB;
  static constexpr int ctas = NB == 1 ? 3 : 2;         // of an SM
  static constexpr int pos = is_8bit(KV) ? 32 : KV == kF16 ? 16 : 8;
  static constexpr int row_bytes = DIM * value_bytes(KV);
  static constexpr int chunks = row_bytes / 16;
  static constexpr int scales = 2 * pos * row_bytes;   // 8-bit: K's, then V's, behind the codes
  static constexpr int block = scales + (is_8bit(KV) ? 2 * pos * 4 : 0);
  static constexpr int stages = (NB == 1 ? 16896 : is_8bit(KV) ? 25344 : 24576) / block;  // 3 (2), head size 64: 6, 5 (3)
  static constexpr int tile = kWarps * pos;           // positions of a CTA's step
  static constexpr int copies = pos * chunks / 32;    // 16-byte copies per lane, K or V
  static constexpr int ring = kWarps * stages * block;
  // 16 rows of queries (hi and lo f16, or f32), later of the warps' joined
  // outputs, eight floats apart more than they need (banks)
  static constexpr int pitch = DIM + 8;
  static constexpr int smem = ring + rows * pitch * 4;
};

// Place of chunk c of row `row` of an 8-bit cache's K or V.  The products' operands
// come by 16-byte (V of head size 64: 8-byte) loads of a whole warp: of K, chunks
// 0 .. 3 of eight neighbouring rows, of V, neighbouring chunks of every other row.
template <int DIM>
__device__ __forceinline__ int place(int row, int c, bool v) {
  if constexpr (DIM == 128) return row * 128 + ((c ^ (v ? row & 7 : (row & 1) << 2)) << 4);
  else return (row >> 1) * 128 + (((((row & 1) << 2) | c) ^ (((row >> 1) & 3) << 1)) << 4);
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(a)
               : "memory");
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 16-byte asynchronous copy, zeros instead when `bytes` is 0.
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ void split_f16(float a, float b, uint32_t& hi, uint32_t& lo) {
  hi = pack_f16(a, b);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  lo = pack_f16(a - f.x, b - f.y);
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;  // rounded to 10 mantissa bits; lo's 11 bits or so remain
  lo = __float_as_uint(x - __uint_as_float(hi)) & 0xffffe000u;
}

// The queries of a block of 16 (token, head) rows (block row 0 is row r0 of the
// sequence): rows first, first + step, .. below `rows` by a warp.  First their
// f32 values into shared memory, DIM of them per row one after another ...
template <int DIM>
__device__ __forceinline__ void fetch_queries(uint32_t raw_s, const AttendArgs& a, const Seq& s, int kvh, int group,
                                              int r0, int rows, int first, int step) {
  const int lane = threadIdx.x & 31;
  int i = 0;
  for (int row = first; row < rows; row += step, ++i) {
    const int r = r0 + row, tok = r / group;
    const float* q = a.q + (int64_t)(s.row0 + tok) * a.q_stride + (int64_t)(kvh * group + r - tok * group) * DIM + lane;
#pragma unroll
    for (int k = 0; k < DIM / 32; ++k)  // 4 bytes each: queries need no alignment
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(raw_s + 4 * (i * DIM + 32 * k + lane)), "l"(q + 32 * k)
                   : "memory");
  }
}
// ... then, scaled by log2(e) / sqrt(DIM), as f32, or as hi and lo f16 after an
// exact power of two that brings the row's largest value to [1, 2) and goes back
// into its scores, so that no query overflows f16.  Rows are DIM values in
// 16-byte chunks xored like the cache's.
template <int DIM, Kv KV, int ROWS = kRows>
__device__ __forceinline__ void stage_queries(uint32_t q_s, float* factor_s, uint32_t raw_s, int rows, int first, int step) {
  constexpr float scale = (DIM == 128 ? 0.08838834764831845f : 0.125f) * kLog2e;
  constexpr int N = DIM / 32;  // values per lane
  const int lane = threadIdx.x & 31;
  int i = 0;
  for (int row = first; row < rows; row += step, ++i) {
    float x[N], top = 0.f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x[k]) : "r"(raw_s + 4 * (i * DIM + N * lane + k)) : "memory");
      x[k] *= scale;
      top = fmaxf(top, fabsf(x[k]));
    }
    const int d = N * lane;
    if constexpr (KV != kF32) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // exponent bits of the largest value, kept where both powers are normal
      const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      if (lane == 0) factor_s[row] = __uint_as_float((uint32_t)e << 23);
      if constexpr (is_8bit(KV)) {
        // in the order in which K's codes meet them: of 16 codes that a lane t of
        // four loads, bytes 0 and 2 of word i are inner indexes 2 t and 2 t + 1
        // of step i, bytes 1 and 3 the ones 8 further
#pragma unroll
        for (int k = 0; k < N; ++k) {
          const int y = d + k, e16 = 16 * (4 * (y >> 6) + ((y >> 2) & 3)) + 2 * ((y >> 4) & 3) + ((y >> 1) & 1) + 8 * (y & 1);
          const int c = e16 >> 3;
          const uint32_t at = q_s + row * (2 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4) + (e16 & 7) * 2;
          const __half hi = __float2half_rn(x[k] * down), lo = __float2half_rn(x[k] * down - __half2float(hi));
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(__half_as_ushort(hi)) : "memory");
          asm volatile("st.shared.u16 [%0], %1;" ::"r"(at + ROWS * 2 * DIM), "h"(__half_as_ushort(lo)) : "memory");
        }
        continue;
      }
      const int c = d >> 3;
      const uint32_t at = q_s + row * (2 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4) + (d & 7) * 2;
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        uint32_t hi, lo;
        split_f16(x[k] * down, x[k + 1] * down, hi, lo);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 2 * k), "r"(hi) : "memory");
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 2 * k + ROWS * 2 * DIM), "r"(lo) : "memory");
      }
    } else {
      const int c = d >> 2;
      const uint32_t at = q_s + row * (4 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4) + (d & 3) * 4;
#pragma unroll
      for (int k = 0; k < N; ++k) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at + 4 * k), "f"(x[k]) : "memory");
    }
  }
}

// What a warp holds of its 16 rows: the queries as the left operand of the
// score products, the running maximum and sum, and the output.  Lane l holds
// rows l / 4 and l / 4 + 8.
template <int DIM, Kv KV>
struct Rows {
  static constexpr int kPer = 2;        // rows of a lane, row(i) of the block
  static __device__ __forceinline__ int row(int i) { return ((threadIdx.x & 31) >> 2) + 8 * i; }
  static __device__ __forceinline__ bool writes() { return (threadIdx.x & 3) == 0; }  // for its rows
  static constexpr bool F32 = KV == kF32;
  uint32_t qh[F32 ? 1 : DIM / 16][4];   // hi and lo fragments
  uint32_t ql[F32 ? 1 : DIM / 16][4];
  float qf[F32 ? DIM / 8 : 1][4];       // f32: split where they are used
  float factor[2];                      // 2^e taken out of a row's queries (not f32)
  int sees[2];                          // last position each row sees
  float o[DIM / 8][4];
  float m[2], l[2];                     // reference and sum of the weights

  // Fragments of the `live` rows that stage_queries() left at q_s.
  __device__ __forceinline__ void load(uint32_t q_s, const float* factor_s, const Seq& s, int group, int r0, int live) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, row = 8 * (mat & 1) + (lane & 7);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (lane >> 2) + 8 * i;
      sees[i] = s.pos + min((r0 + r) / group, s.n - 1);
      factor[i] = F32 ? 1.0f : factor_s[r];
    }
    if constexpr (!F32) {
#pragma unroll
      for (int k = 0; k < DIM / 16; ++k) {
        const int c = 2 * k + (mat >> 1);
        const uint32_t at = q_s + row * (2 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4);
        ldsm4(qh[k], at);
        ldsm4(ql[k], at + kRows * 2 * DIM);
      }
    } else {
#pragma unroll
      for (int k = 0; k < DIM / 8; ++k) {
        const int c = 2 * k + (mat >> 1);
        uint32_t x[4];
        ldsm4(x, q_s + row * (4 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) qf[k][j] = __uint_as_float(x[j]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int d = 0; d < DIM / 8; ++d)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[d][j] = 0.f;
  }

  // One block of positions p0 .. p0 + POS - 1 (K at k_s, V behind it); with
  // `masked`, positions a row does not see are left out.
  __device__ __forceinline__ void step(uint32_t k_s, int p0, bool masked) {
    using G = Geo<DIM, KV>;
    const int lane = threadIdx.x & 31, t = lane & 3;
    const uint32_t v_s = k_s + G::pos * G::row_bytes;
    constexpr int NT = G::pos / 8;  // score tiles of 8 positions
    float s[NT][4];
    if constexpr (KV == kF16) {
      float lo[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = lo[n][j] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < DIM / 32; ++k)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int row = 8 * n + (lane & 7), c = 4 * k + (lane >> 3);
          uint32_t b[4];
          ldsm4(b, k_s + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4));
          mma_f16(s[n], qh[2 * k], b[0], b[1]);
          mma_f16(lo[n], ql[2 * k], b[0], b[1]);
          mma_f16(s[n], qh[2 * k + 1], b[2], b[3]);
          mma_f16(lo[n], ql[2 * k + 1], b[2], b[3]);
        }
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[n][j] = (s[n][j] + lo[n][j]) * factor[j >> 1];
    } else {
      // (the large products in two sums: half as many cut additions in each)
      float lo[4] = {}, lo2[4] = {}, odd[4] = {};
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0][j] = 0.f;
#pragma unroll
      for (int k = 0; k < DIM / 16; ++k) {
        const int row = lane & 7, c = 4 * k + (lane >> 3);
        uint32_t b[4];
        ldsm4(b, k_s + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t qh_[4], ql_[4], bh[2], bl[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) split_tf32(qf[2 * k + h][j], qh_[j], ql_[j]);
#pragma unroll
          for (int j = 0; j < 2; ++j) split_tf32(__uint_as_float(b[2 * h + j]), bh[j], bl[j]);
          mma_tf32(h ? odd : s[0], qh_, bh[0], bh[1]);
          mma_tf32(lo, qh_, bl[0], bl[1]);
          mma_tf32(lo2, ql_, bh[0], bh[1]);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) s[0][j] += odd[j] + (lo[j] + lo2[j]);
    }
    if (masked) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (p0 + 8 * n + 2 * t + (j & 1) > sees[j >> 1]) s[n][j] = -INFINITY;
    }
    float top[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      top[i] = fmaxf(s[0][2 * i], s[0][2 * i + 1]);
#pragma unroll
      for (int n = 1; n < NT; ++n) top[i] = fmaxf(top[i], fmaxf(s[n][2 * i], s[n][2 * i + 1]));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
    }
    float down[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float now = fmaxf(m[i], reference(top[i]));
      down[i] = now == -INFINITY ? 1.0f : ex2(m[i] - now);
      m[i] = now;
      l[i] *= down[i];
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float base = m[i] == -INFINITY ? 0.f : m[i];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          s[n][2 * i + j] = ex2(s[n][2 * i + j] - base);
          l[i] += s[n][2 * i + j];
        }
    }
    if constexpr (KV == kF16) {
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) split_f16(s[j >> 1][2 * (j & 1)], s[j >> 1][2 * (j & 1) + 1], ph[j], pl[j]);
#pragma unroll
      for (int d = 0; d < DIM / 16; ++d) {
        const int mat = lane >> 3, row = 8 * (mat & 1) + (lane & 7), c = 2 * d + (mat >> 1);
        uint32_t b[4];
        ldsm4_t(b, v_s + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4));
        float x[2][4] = {};
        mma_f16(x[0], pl, b[0], b[1]);
        mma_f16(x[1], pl, b[2], b[3]);
        mma_f16(x[0], ph, b[0], b[1]);
        mma_f16(x[1], ph, b[2], b[3]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[2 * d][j] = fmaf(o[2 * d][j], down[j >> 1], x[0][j]);
          o[2 * d + 1][j] = fmaf(o[2 * d + 1][j], down[j >> 1], x[1][j]);
        }
      }
    } else {
      // the product's inner index t stands for position 2 t, t + 4 for 2 t + 1:
      // the scores' own layout
      uint32_t ph[4], pl[4];
      split_tf32(s[0][0], ph[0], pl[0]);
      split_tf32(s[0][2], ph[1], pl[1]);
      split_tf32(s[0][1], ph[2], pl[2]);
      split_tf32(s[0][3], ph[3], pl[3]);
#pragma unroll
      for (int d = 0; d < DIM / 8; ++d) {
        uint32_t bh[2], bl[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int row = 2 * t + j, c = 2 * d + (lane >> 4);
          float y;
          asm volatile("ld.shared.f32 %0, [%1];"
                       : "=f"(y)
                       : "r"(v_s + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4) + ((lane >> 2) & 3) * 4)
                       : "memory");
          split_tf32(y, bh[j], bl[j]);
        }
        float x[4] = {};
        mma_tf32(x, ph, bl[0], bl[1]);
        mma_tf32(x, pl, bh[0], bh[1]);
        mma_tf32(x, ph, bh[0], bh[1]);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][j] = fmaf(o[d][j], down[j >> 1], x[j]);
      }
    }
  }

  // Sum of the weights of row(i), from all lanes that share it.
  __device__ __forceinline__ float total(int i) const {
    float x = l[i];
    x += __shfl_xor_sync(0xffffffffu, x, 1);
    x += __shfl_xor_sync(0xffffffffu, x, 2);
    return x;
  }
  // This lane's outputs of row(i) times f, added to (`first`: put into) the row at `to`.
  __device__ __forceinline__ void add(float* to, int i, float f, bool first) const {
    float2* at = reinterpret_cast<float2*>(to + 2 * (threadIdx.x & 3));
#pragma unroll
    for (int d = 0; d < DIM / 8; ++d) {
      const float2 before = first ? make_float2(0.f, 0.f) : at[4 * d];
      at[4 * d] = make_float2(fmaf(o[d][2 * i], f, before.x), fmaf(o[d][2 * i + 1], f, before.y));
    }
  }
  // f(d, output) for this lane's outputs of row(i).
  template <typename F>
  __device__ __forceinline__ void each(int i, F f) const {
#pragma unroll
    for (int d = 0; d < DIM / 8; ++d)
#pragma unroll
      for (int j = 0; j < 2; ++j) f(8 * d + 2 * ((int)threadIdx.x & 3) + j, o[d][2 * i + j]);
  }
};

__device__ __forceinline__ void lds128(uint32_t (&w)[4], uint32_t a) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t a) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(a) : "memory");
  return x;
}
// An 8 x 8 matrix of f16 over a warp (lane l: row l / 4, columns 2 (l % 4) and the
// next), transposed.
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// Rows over an 8-bit cache: the products turned round, positions (then values of
// the head) on the left, 8 NB query rows on the right, so that a token's few rows
// fill what is multiplied and the codes, decoded in registers, are left operands of
// either product: of K, a lane's words are codes of its own positions, of V, bytes of
// two positions' words go together.  Weights carry their position's scale of V,
// 2^(s + log2 v - m), with a reference m that follows the largest of a row's only when
// that is more than kSlack further up; the sum of weights takes 1 / v back out.  Lane
// l holds rows 2 (l % 4) and the next, of every eight.
template <int DIM, Kv KV, int NB>
struct CodeRows {
  static constexpr int kPer = 2 * NB;
  static __device__ __forceinline__ int row(int i) { return 8 * (i >> 1) + 2 * ((int)threadIdx.x & 3) + (i & 1); }
  static __device__ __forceinline__ bool writes() { return (threadIdx.x & 31) < 4; }
  static constexpr int KS = DIM / 16, VT = DIM / 16;  // steps along the head; V's tiles of 16 values
  uint32_t qh[NB][KS][2], ql[NB][KS][2];
  float factor[kPer];
  int sees[kPer];
  float o[VT][NB][4];
  float m[kPer], l[kPer];

  __device__ __forceinline__ void load(uint32_t q_s, const float* factor_s, const Seq& s, int group, int r0, int live) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      factor[i] = factor_s[row(i)] * code_unit<KV>();
      sees[i] = s.pos + min((r0 + row(i)) / group, s.n - 1);
      // (rows without a query never raise the references, whatever was in their place)
      m[i] = row(i) < live ? -INFINITY : INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int k = 0; k < KS; k += 2) {
        const int r = 8 * nb + (lane & 7), c = 2 * k + (lane >> 3);
        const uint32_t at = q_s + r * (2 * DIM) + (((c & ~7) | ((c ^ r) & 7)) << 4);
        uint32_t x[4];
        ldsm4(x, at);
        qh[nb][k][0] = x[0], qh[nb][k][1] = x[1], qh[nb][k + 1][0] = x[2], qh[nb][k + 1][1] = x[3];
        ldsm4(x, at + 8 * NB * 2 * DIM);
        ql[nb][k][0] = x[0], ql[nb][k][1] = x[1], ql[nb][k + 1][0] = x[2], ql[nb][k + 1][1] = x[3];
      }
#pragma unroll
    for (int d = 0; d < VT; ++d)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[d][nb][j] = 0.f;
  }

  // One block of 32 positions from p0 (K at k_s, V and the scales behind it); with
  // `masked`, positions a row does not see are left out.
  __device__ __forceinline__ void step(uint32_t k_s, int p0, bool masked) {
    using G = Geo<DIM, KV, NB>;
    static_assert(G::pos == 32, "two steps of 16 positions");
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t v_s = k_s + G::pos * G::row_bytes, ks_s = k_s + G::scales, vs_s = ks_s + 4 * G::pos;
    // scores: value j of s[b][nb] is position 16 b + g + 8 (j / 2), row 2 t + j % 2
    float s[2][NB][4];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      float lo[NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[b][nb][j] = lo[nb][j] = 0.f;
#pragma unroll
      for (int h = 0; h < DIM / 64; ++h) {
        uint32_t w0[4], w1[4];
        lds128(w0, k_s + place<DIM>(16 * b + g, 4 * h + t, false));
        lds128(w1, k_s + place<DIM>(16 * b + g + 8, 4 * h + t, false));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t a[4];
          decode4<KV>(w0[i], a[0], a[2]);
          decode4<KV>(w1[i], a[1], a[3]);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            mma_f16(s[b][nb], a, qh[nb][4 * h + i][0], qh[nb][4 * h + i][1]);
            mma_f16(lo[nb], a, ql[nb][4 * h + i][0], ql[nb][4 * h + i][1]);
          }
        }
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[b][nb][j] = (s[b][nb][j] + lo[nb][j]) * factor[2 * nb + (j & 1)];
    }
    float inverse[4], keep[4];  // of position g + 8 e: 1 / |scale of V|, and its sign, or 0 where it is below 2^-100
    bool up = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float ks = lds_f32(ks_s + 4 * (g + 8 * e)), vs = lds_f32(vs_s + 4 * (g + 8 * e));
      const bool finite = fabsf(vs) < INFINITY;
      keep[e] = fabsf(vs) < 7.8886091e-31f ? 0.f : copysignf(1.f, vs);  // 2^-100
      const float v = keep[e] == 0.f ? 8.6736174e-19f : fabsf(vs);      // 2^-60: the weight of a row of zeros
      inverse[e] = finite ? __frcp_rn(v) : 1.f;
      const float lift = finite ? __log2f(v) : __uint_as_float(0x7fc00000u);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float& u = s[e >> 1][nb][2 * (e & 1) + j];
          u = fmaf(u, ks, lift);
          if (masked && p0 + g + 8 * e > sees[2 * nb + j]) u = -INFINITY;
          up = up || u > m[2 * nb + j] + (kBias + kSlack);
        }
    }
    if (__any_sync(0xffffffffu, up)) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[e >> 1][i >> 1][2 * (e & 1) + (i & 1)]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float now = fmaxf(m[i], reference(top)), f = now == -INFINITY ? 1.0f : ex2(m[i] - now);
        m[i] = now;
        l[i] *= f;
#pragma unroll
        for (int d = 0; d < VT; ++d) {
          o[d][i >> 1][i & 1] *= f;
          o[d][i >> 1][2 + (i & 1)] *= f;
        }
      }
    }
    uint32_t ph[2][NB][2], pl[2][NB][2];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        float y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float base = m[2 * nb + j] == -INFINITY ? 0.f : m[2 * nb + j];
          y[j] = ex2(s[e >> 1][nb][2 * (e & 1) + j] - base);
          l[2 * nb + j] = fmaf(y[j], inverse[e], l[2 * nb + j]);
          y[j] *= keep[e];
        }
        uint32_t hi, lo;
        split_f16(y[0], y[1], hi, lo);
        ph[e >> 1][nb][e & 1] = transposed(hi);
        pl[e >> 1][nb][e & 1] = transposed(lo);
      }
    // outputs: row g (g + 8) of tile d is value (DIM / 8) g + 2 d (and the next)
    constexpr int W = DIM / 32;  // words of a lane's values
    uint32_t w[2][4][W];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * b + 2 * t + (r & 1) + 8 * (r >> 1);
        if constexpr (W == 4) lds128(w[b][r], v_s + place<DIM>(row, g, true));
        else
          asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];"
                       : "=r"(w[b][r][0]), "=r"(w[b][r][1])
                       : "r"(v_s + place<DIM>(row, g >> 1, true) + 8 * (g & 1))
                       : "memory");
      }
#pragma unroll
    for (int c = 0; c < W; ++c)
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // values 4 c + 2 h and the next
        uint32_t a[2][4];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          decode4<KV>(__byte_perm(w[b][0][c], w[b][1][c], h ? 0x7632 : 0x5410), a[b][0], a[b][1]);
          decode4<KV>(__byte_perm(w[b][2][c], w[b][3][c], h ? 0x7632 : 0x5410), a[b][2], a[b][3]);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float x[4] = {};
          mma_f16(x, a[0], pl[0][nb][0], pl[0][nb][1]);
          mma_f16(x, a[1], pl[1][nb][0], pl[1][nb][1]);
          mma_f16(x, a[0], ph[0][nb][0], ph[0][nb][1]);
          mma_f16(x, a[1], ph[1][nb][0], ph[1][nb][1]);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[2 * c + h][nb][j] += x[j];
        }
      }
  }

  __device__ __forceinline__ float total(int i) const {
    float x = l[i];
#pragma unroll
    for (int k = 4; k < 32; k <<= 1) x += __shfl_xor_sync(0xffffffffu, x, k);
    return x;
  }
  __device__ __forceinline__ void add(float* to, int i, float f, bool first) const {
    float4* at = reinterpret_cast<float4*>(to + DIM / 8 * ((threadIdx.x & 31) >> 2));
    f *= code_unit<KV>();
#pragma unroll
    for (int d = 0; d < VT; d += 2) {
      const float4 before = first ? make_float4(0.f, 0.f, 0.f, 0.f) : at[d / 2];
      const int nb = i >> 1, j = i & 1;
      at[d / 2] = make_float4(fmaf(o[d][nb][j], f, before.x), fmaf(o[d][nb][2 + j], f, before.y), fmaf(o[d + 1][nb][j], f, before.z),
                              fmaf(o[d + 1][nb][2 + j], f, before.w));
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(int i, F f) const {
#pragma unroll
    for (int d = 0; d < VT; ++d)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        f(DIM / 8 * (((int)threadIdx.x & 31) >> 2) + 2 * d + j, o[d][i >> 1][2 * j + (i & 1)] * code_unit<KV>());
  }
};

template <int DIM, Kv KV, int NB>
using RowsOf = std::conditional_t<is_8bit(KV), CodeRows<DIM, KV, NB>, Rows<DIM, KV>>;

// The copies of a warp's block of positions into its stage.
template <int DIM, Kv KV, int NB = 2>
struct Feed {
  using G = Geo<DIM, KV, NB>;
  const AttendArgs& a;
  const Seq& s;
  int kvh, len, shift;

  // page of this lane's row (lane % POS) of the block at p0; -1: no row
  __device__ __forceinline__ int page(int p0) const {
    const int p = p0 + (threadIdx.x & 31) % G::pos;
    return p < len ? s.pages[shift >= 0 ? p >> shift : p / a.c.page_size] : -1;
  }
  __device__ __forceinline__ void copy(uint32_t dst, int p0, int page) const {
    const int lane = threadIdx.x & 31, p = p0 + lane % G::pos;
    int64_t at = 0;
    int ok = 0;
    if (p < len) {
      if (page >= 0 && page < a.c.pages) {
        const int row = shift >= 0 ? p & ((1 << shift) - 1) : p % a.c.page_size;
        at = (int64_t)page * a.c.page_stride + (int64_t)kvh * a.c.head_stride + (int64_t)row * a.c.row_stride;
        ok = 16;
      } else {
        atomicOr(a.c.status, DEV_BAD_ARGS);
      }
    }
    constexpr int esize = value_bytes(KV);
    const char* k = static_cast<const char*>(a.c.k);
    const char* v = static_cast<const char*>(a.c.v);
#pragma unroll
    for (int i = 0; i < G::copies; ++i) {
      const int x = i * 32 + lane, row = x / G::chunks, c = x % G::chunks;
      const int64_t off = __shfl_sync(0xffffffffu, at, row) * esize + 16 * c;
      const int n = __shfl_sync(0xffffffffu, ok, row);
      if constexpr (is_8bit(KV)) {
        copy16(dst + place<DIM>(row, c, false), k + (n ? off : 0), n);
        copy16(dst + G::pos * G::row_bytes + place<DIM>(row, c, true), v + (n ? off : 0), n);
      } else {
        const uint32_t to = dst + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4);
        copy16(to, k + (n ? off : 0), n);
        copy16(to + G::pos * G::row_bytes, v + (n ? off : 0), n);
      }
    }
    if constexpr (is_8bit(KV)) {
      const int row = shift >= 0 ? p & ((1 << shift) - 1) : p % a.c.page_size;
      const int64_t from = ok ? scale_at(a.c, page, kvh, row) : 0;
      const uint32_t to = dst + G::scales + 4 * lane;
      const int n = ok ? 4 : 0;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(a.c.k_scale + from), "r"(n) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 4 * G::pos), "l"(a.c.v_scale + from), "r"(n) : "memory");
    }
  }
  // Non-finite values of V at positions past `first` (the first new token's
  // own) become zero in shared memory: a row that does not see them would
  // multiply them by a weight of zero.  The rows that see them add them back
  // at the end (non_finite()).  Returns whether this lane found any.
  // (An 8-bit cache has none: what is not finite there is a row's scale.)
  __device__ __forceinline__ bool clean(uint32_t dst, int p0, int first) const {
    if constexpr (is_8bit(KV)) return false;
    if (p0 + G::pos - 1 <= first) return false;
    const int lane = threadIdx.x & 31;
    bool found = false;
#pragma unroll 1
    for (int i = 0; i < G::copies; ++i) {
      const int x = i * 32 + lane, row = x / G::chunks, c = x % G::chunks;
      if (p0 + row <= first) continue;
      const uint32_t at = dst + (G::pos + row) * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4);
      uint32_t w[4];
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (KV == kF16) {
          if ((w[j] & 0x7c00u) == 0x7c00u) w[j] &= 0xffff0000u, bad = true;
          if ((w[j] & 0x7c000000u) == 0x7c000000u) w[j] &= 0xffffu, bad = true;
        } else {
          if ((w[j] & 0x7f800000u) == 0x7f800000u) w[j] = 0, bad = true;
        }
      }
      found = found || bad;
      if (bad)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    }
    __syncwarp();
    return found;
  }
};

// An output y of a row that sees positions up to `last`, l the sum of its
// weights; `dirty`: values at positions past `first` were taken out.
template <Kv KV>
__device__ __forceinline__ float settled(float y, float l, bool dirty, const Cache& c, const Seq& s, int kvh, int first, int last,
                                         int d) {
  if constexpr (is_8bit(KV)) return y;
  constexpr bool KV16 = KV == kF16;
  if (!isfinite(y) && isfinite(l)) {
    const float x = non_finite<KV16, 1>(c, s, kvh, -1, first, d).v[0];
    if (x != 0.f) y = x;
  }
  if (dirty) y += non_finite<KV16, 1>(c, s, kvh, first, last, d).v[0];
  return y;
}

}  // namespace
}  // namespace paged
}  // namespace hyq
