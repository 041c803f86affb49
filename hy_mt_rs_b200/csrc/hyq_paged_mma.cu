// Attention over pages on the warp-level tensor instructions, head sizes 64
// and 128: the kernel for few new tokens (the cache is read once, bound by
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
// Chunks, bound by the products and by each CTA's own walk over the positions:
// 200 tokens at 0 21 us, 8 sequences of 40 at 100 20 us (f16); longer ones go to
// the kernels on tcgen05.
#include "../../include/hyq.h"
#include "hyq_kernels.h"
#include "hyq_paged.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = kFewRows;      // query rows of a warp: (token, head) pairs
constexpr int kCtasPerSm = 2;
constexpr int kMaxCtas = 148 * kCtasPerSm;

// A warp's block of positions: POS rows of K, then of V, in 16-byte chunks
// whose low three index bits are xored with the row (reads by ldmatrix and by
// words then fall into distinct banks).  8 KB for head size 128.
template <int DIM, bool KV16>
struct Geo {
  static constexpr int pos = KV16 ? 16 : 8;
  static constexpr int row_bytes = DIM * (KV16 ? 2 : 4);
  static constexpr int chunks = row_bytes / 16;
  static constexpr int block = 2 * pos * row_bytes;
  static constexpr int stages = 24576 / block;        // 3 (head size 128), 6 (64)
  static constexpr int tile = kWarps * pos;           // positions of a CTA's step
  static constexpr int copies = pos * chunks / 32;    // 16-byte copies per lane, K or V
  static constexpr int ring = kWarps * stages * block;
  // 16 rows of queries (hi and lo f16, or f32), later of the warps' joined
  // outputs, eight floats apart more than they need (banks)
  static constexpr int pitch = DIM + 8;
  static constexpr int smem = ring + kRows * pitch * 4;
};

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
template <int DIM, bool KV16>
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
    if constexpr (KV16) {
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      // exponent bits of the largest value, kept where both powers are normal
      const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      if (lane == 0) factor_s[row] = __uint_as_float((uint32_t)e << 23);
      const int c = d >> 3;
      const uint32_t at = q_s + row * (2 * DIM) + (((c & ~7) | ((c ^ row) & 7)) << 4) + (d & 7) * 2;
#pragma unroll
      for (int k = 0; k < N; k += 2) {
        uint32_t hi, lo;
        split_f16(x[k] * down, x[k + 1] * down, hi, lo);
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 2 * k), "r"(hi) : "memory");
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + 2 * k + kRows * 2 * DIM), "r"(lo) : "memory");
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
template <int DIM, bool KV16>
struct Rows {
  uint32_t qh[KV16 ? DIM / 16 : 1][4];  // f16: hi and lo fragments
  uint32_t ql[KV16 ? DIM / 16 : 1][4];
  float qf[KV16 ? 1 : DIM / 8][4];      // f32: split where they are used
  float factor[2];                      // 2^e taken out of a row's queries (f16)
  int sees[2];                          // last position each row sees
  float o[DIM / 8][4];
  float m[2], l[2];                     // reference and sum of the weights

  // Fragments of the rows that stage_queries() left at q_s.
  __device__ __forceinline__ void load(uint32_t q_s, const float* factor_s, const Seq& s, int group, int r0) {
    const int lane = threadIdx.x & 31, mat = lane >> 3, row = 8 * (mat & 1) + (lane & 7);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (lane >> 2) + 8 * i;
      sees[i] = s.pos + min((r0 + r) / group, s.n - 1);
      factor[i] = KV16 ? factor_s[r] : 1.0f;
    }
    if constexpr (KV16) {
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
    using G = Geo<DIM, KV16>;
    const int lane = threadIdx.x & 31, t = lane & 3;
    const uint32_t v_s = k_s + G::pos * G::row_bytes;
    constexpr int NT = G::pos / 8;  // score tiles of 8 positions
    float s[NT][4];
    if constexpr (KV16) {
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
    if constexpr (KV16) {
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
};

// The copies of a warp's block of positions into its stage.
template <int DIM, bool KV16>
struct Feed {
  using G = Geo<DIM, KV16>;
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
    constexpr int esize = KV16 ? 2 : 4;
    const char* k = static_cast<const char*>(a.c.k);
    const char* v = static_cast<const char*>(a.c.v);
#pragma unroll
    for (int i = 0; i < G::copies; ++i) {
      const int x = i * 32 + lane, row = x / G::chunks, c = x % G::chunks;
      const int64_t off = __shfl_sync(0xffffffffu, at, row) * esize + 16 * c;
      const int n = __shfl_sync(0xffffffffu, ok, row);
      const uint32_t to = dst + row * G::row_bytes + (((c & ~7) | ((c ^ row) & 7)) << 4);
      copy16(to, k + (n ? off : 0), n);
      copy16(to + G::pos * G::row_bytes, v + (n ? off : 0), n);
    }
  }
  // Non-finite values of V at positions past `first` (the first new token's
  // own) become zero in shared memory: a row that does not see them would
  // multiply them by a weight of zero.  The rows that see them add them back
  // at the end (non_finite()).  Returns whether this lane found any.
  __device__ __forceinline__ bool clean(uint32_t dst, int p0, int first) const {
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
        if constexpr (KV16) {
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
template <bool KV16>
__device__ __forceinline__ float settled(float y, float l, bool dirty, const Cache& c, const Seq& s, int kvh, int first, int last,
                                         int d) {
  if (!isfinite(y) && isfinite(l)) {
    const float x = non_finite<KV16, 1>(c, s, kvh, -1, first, d).v[0];
    if (x != 0.f) y = x;
  }
  if (dirty) y += non_finite<KV16, 1>(c, s, kvh, first, last, d).v[0];
  return y;
}

// ---------------------------------------------------------------------------
// Few new tokens: at most 16 (token, head) rows per kv head
// ---------------------------------------------------------------------------

// Workspace: one counter per CTA, then two partial results per CTA: 16 rows of
// DIM outputs, then the rows' (maximum, sum), then whether clean() took a value
// out.
constexpr size_t kCounterBytes = HYQ_PAGED_ATTENTION_ZEROED;
static_assert(kCounterBytes >= kMaxCtas * sizeof(unsigned), "a counter per CTA");
__host__ __device__ constexpr int partial_floats(int dim) { return kRows * (dim + 2) + 4; }

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
template <int DIM, bool KV16>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) few_kernel(const __grid_constant__ AttendArgs a, int shift, bool beside) {
  using G = Geo<DIM, KV16>;
  if (!beside) grid_dependency_wait();
  allow_dependents_launch();
  extern __shared__ __align__(1024) char smem[];
  int* first_s = reinterpret_cast<int*>(smem + G::smem);  // [seqs + 1] tiles (of one kv head) before each sequence
  __shared__ float ml_s[kWarps][kRows][2];
  __shared__ float factor_s[kRows];
  __shared__ int warp_s[kWarps];
  __shared__ int last_s;
  __shared__ int dirty_s;  // the last piece (of this CTA's) that clean() took a value out of
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads, seqs = a.c.seqs, kvh_n = a.c.kv_heads;
  // prefix sum of the sequences' tiles; sequences with more rows are the
  // chunk kernel's
  int carry = 0;
  for (int s0 = 0; s0 < seqs; s0 += kThreads) {
    const int i = s0 + (int)threadIdx.x;
    int tiles = 0;
    if (i < seqs) {
      const Seq s = load_seq(a.c, i);
      if (s.n > 0 && s.n * group <= kRows) tiles = (s.pos + s.n + G::tile - 1) / G::tile + kSegmentCost;
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
  Rows<DIM, KV16> rows;
  const uint32_t ring = smem_addr(smem) + warp * G::stages * G::block;
  float* o_s = reinterpret_cast<float*>(smem + G::ring);  // [16][pitch]; the queries before
  const int off = warp * G::pos;
  // the piece of a segment that this CTA takes: tiles j0 .. j1 - 1 of `tiles`
  struct {
    Seq s;
    int kvh, j0, j1, tiles;
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
    if (!same_seq) cur.s = load_seq(a.c, si);
    const Feed<DIM, KV16> feed{a, cur.s, cur.kvh, cur.s.pos + cur.s.n, shift};
    page = feed.page(cur.j0 * G::tile + off);
    // (the ring's last stage is not copied to before the first turn)
    fetch_queries<DIM>(ring + (G::stages - 1) * G::block, a, cur.s, cur.kvh, group, 0, cur.s.n * group, warp, kWarps);
    cp_async_commit();
#pragma unroll
    for (int i = 0; i < G::stages - 1; ++i) {
      const int now = page;
      page = feed.page((cur.j0 + i + 1) * G::tile + off);
      if (cur.j0 + i < cur.j1) feed.copy(ring + i * G::block, (cur.j0 + i) * G::tile + off, now);
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
      stage_queries<DIM, KV16>(q_s, factor_s, ring + (G::stages - 1) * G::block, s.n * group, warp, kWarps);
      __syncthreads();
      rows.load(q_s, factor_s, s, group, 0);
      const Feed<DIM, KV16> feed{a, s, cur.kvh, s.pos + s.n, shift};
      int stage = 0;
      for (int j = cur.j0; j < cur.j1; ++j) {
        const int ahead = j + G::stages - 1, now = page;
        page = feed.page((ahead + 1) * G::tile + off);
        int put = stage + G::stages - 1;
        if (put >= G::stages) put -= G::stages;
        __syncwarp();
        if (ahead < cur.j1) feed.copy(ring + put * G::block, ahead * G::tile + off, now);
        cp_async_commit();
        cp_async_wait<G::stages - 1>();
        __syncwarp();
        const int p0 = j * G::tile + off;
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
    for (int i = 0; i < 2; ++i) {
      float l = rows.l[i];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      if ((lane & 3) == 0) {
        ml_s[warp][(lane >> 2) + 8 * i][0] = rows.m[i];
        ml_s[warp][(lane >> 2) + 8 * i][1] = l;
      }
    }
    __syncthreads();
    float down[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = (lane >> 2) + 8 * i;
      float top = ml_s[0][r][0];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) top = fmaxf(top, ml_s[w][r][0]);
      down[i] = rows.m[i] == -INFINITY ? 0.f : ex2(rows.m[i] - top);
    }
#pragma unroll 1
    for (int w = 0; w < kWarps; ++w) {
      if (warp == w) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = (lane >> 2) + 8 * i;
          if (r >= live) continue;
          float2* to = reinterpret_cast<float2*>(o_s + r * G::pitch + 2 * (lane & 3));
#pragma unroll
          for (int d = 0; d < DIM / 8; ++d) {
            const float2 before = w ? to[4 * d] : make_float2(0.f, 0.f);
            to[4 * d] = make_float2(fmaf(rows.o[d][2 * i], down[i], before.x), fmaf(rows.o[d][2 * i + 1], down[i], before.y));
          }
        }
      }
      __syncthreads();
    }
    const bool whole = done.j0 == 0 && done.j1 == done.tiles, dirty = dirty_s == piece;
    float* part = parts + (size_t)(2 * cta + second) * partial_floats(DIM);
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
          to[d] = settled<KV16>(from[d] * inv, l, dirty, a.c, s, kvh, s.pos, s.pos + tok, d);
        }
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
        const float* part0 = parts + (size_t)(2 * cf + (work * cf / ctas < seg0)) * partial_floats(DIM);
        const float* part1 = parts + (size_t)(2 * cf) * partial_floats(DIM);
        auto part_at = [&](int i) { return i ? part1 + (size_t)(2 * i) * partial_floats(DIM) : part0; };
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
            to[d] = settled<KV16>(sum[k] * inv, l, any, a.c, s, kvh, s.pos, s.pos + tok, d);
          }
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
template <int DIM, bool KV16>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) chunk_kernel(const __grid_constant__ AttendArgs a, int shift) {
  using G = Geo<DIM, KV16>;
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
  const Feed<DIM, KV16> feed{a, s, kvh, len, shift};
  const uint32_t ring = smem_addr(smem);
  // the queries: each warp's own 16 rows, through its part of the ring
  static_assert(G::stages * G::block >= 2 * kRows * DIM * 4, "a warp's queries, as they come and as they are read");
  Rows<DIM, KV16> rows;
  const bool any = r0 < s.n * group;
  if (any) {
    const uint32_t q_s = ring + warp * G::stages * G::block, raw_s = q_s + kRows * DIM * 4;
    const int n = min(kRows, s.n * group - r0);
    fetch_queries<DIM>(raw_s, a, s, kvh, group, r0, n, 0, 1);
    cp_async_commit();
    cp_async_wait<0>();
    __syncwarp();
    stage_queries<DIM, KV16>(q_s, factor_s[warp], raw_s, n, 0, 1);
    __syncwarp();
    rows.load(q_s, factor_s[warp], s, group, r0);
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
  for (int i = 0; i < 2; ++i) {
    float l = rows.l[i];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int r = r0 + (lane >> 2) + 8 * i, tok = r / group;
    if (tok >= s.n) continue;
    float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r - tok * group) * DIM + 2 * (lane & 3);
    bool odd = dirty_s;
#pragma unroll
    for (int d = 0; d < DIM / 8; ++d) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float y = rows.o[d][2 * i + j] / l;
        odd = odd || !isfinite(y);
        to[8 * d + j] = y;
      }
    }
    if (odd) {
#pragma unroll 1
      for (int d = 0; d < DIM / 8; ++d)
#pragma unroll 1
        for (int j = 0; j < 2; ++j)
          to[8 * d + j] = settled<KV16>(to[8 * d + j], l, dirty_s, a.c, s, kvh, s.pos + first_tok, s.pos + tok,
                                        8 * d + 2 * (lane & 3) + j);
    }
  }
}

int64_t chunk_tiles(const AttendArgs& a) {
  return ((int64_t)a.c.tokens * (a.heads / a.c.kv_heads) + kChunkRows - 1) / kChunkRows + a.c.seqs;
}

int page_shift(const AttendArgs& a) {
  return (a.c.page_size & (a.c.page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.c.page_size) : -1;
}

template <int DIM, bool KV16>
cudaError_t chunks(const AttendArgs& a, cudaStream_t st) {
  using G = Geo<DIM, KV16>;
  const int64_t tiles = chunk_tiles(a);
  auto k = chunk_kernel<DIM, KV16>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, G::smem, done);
  if (e != cudaSuccess) return e;
  return launch_ex(k, dim3((unsigned)tiles, (unsigned)a.c.kv_heads), dim3(kThreads), G::smem, st, a, page_shift(a));
}

template <int DIM, bool KV16>
cudaError_t few(const AttendArgs& a, bool beside, cudaStream_t st) {
  using G = Geo<DIM, KV16>;
  auto k = few_kernel<DIM, KV16>;
  static std::atomic<uint64_t> done{0};
  const cudaError_t e = allow_smem(k, G::smem + (kMaxSeqs + 1) * 4, done);
  if (e != cudaSuccess) return e;
  return launch_dependent(beside || launch_overlap(), k, dim3(kMaxCtas), dim3(kThreads), (size_t)G::smem + (a.c.seqs + 1) * 4, st,
                          a, page_shift(a), beside);
}

}  // namespace

bool mma_supported(const AttendArgs& a, bool kv16) {
  const int64_t strides = (a.c.page_stride | a.c.head_stride | a.c.row_stride) * (kv16 ? 2 : 4);
  return (a.c.dim == 64 || a.c.dim == 128) && strides % 16 == 0 &&
         (reinterpret_cast<uintptr_t>(a.c.k) | reinterpret_cast<uintptr_t>(a.c.v)) % 16 == 0;
}

bool sums_fit(int64_t seqs, int64_t reach) {
  constexpr int tile = Geo<128, false>::tile;  // the smaller one
  return seqs * (reach / tile + 1 + kSegmentCost) <= INT32_MAX;
}

bool chunks_short(const AttendArgs& a, bool kv16, int64_t max_len) {
  const int64_t tiles = (chunk_tiles(a) - a.c.seqs / 2) * a.c.kv_heads;  // sequences' last tiles are half full
  const int64_t rounds = (tiles + kMaxCtas - 1) / kMaxCtas;
  return rounds * max_len <= (kv16 ? 350 : 64);
}

size_t mma_workspace_bytes(int dim) { return kCounterBytes + 2 * (size_t)kMaxCtas * partial_floats(dim) * sizeof(float); }

cudaError_t launch_few(const AttendArgs& a, bool kv16, bool beside, cudaStream_t st) {
  if (a.c.dim == 128) return kv16 ? few<128, true>(a, beside, st) : few<128, false>(a, beside, st);
  return kv16 ? few<64, true>(a, beside, st) : few<64, false>(a, beside, st);
}

cudaError_t launch_chunks(const AttendArgs& a, bool kv16, cudaStream_t st) {
  if (a.c.dim == 128) return kv16 ? chunks<128, true>(a, st) : chunks<128, false>(a, st);
  return kv16 ? chunks<64, true>(a, st) : chunks<64, false>(a, st);
}

}  // namespace paged
}  // namespace hyq
