// Attention of chunks of new tokens over an f16 paged cache on tcgen05, head
// sizes 64 and 128, at f32 accuracy.
//
// A CTA takes two tiles of 128 (token, query head) rows of one sequence and kv
// head, and walks the positions they see in tiles of 128.  Queries and weights
// are hi + lo, both f16 (22 bits), K and V exact, so a tile pair costs
//   S = Qh K' + Ql K'   and   X = Ph V + Pl V,
// four 128 x 128 x 128 products: twice those of plain f16 attention, which is
// what bounds the kernel (half the tensor cores' f16 rate).
//
//   warp 0      TMA: pages of K and V into a ring of three tiles (128-byte
//               swizzle; pages past the sequence come as zeros);
//   warp 1      tcgen05.mma: S of one row tile while the other's softmax runs;
//   warps 2-3   take non-finite values out of V at positions that some row of
//               the CTA does not see (0 times them would be NaN);
//   warps 4-7, 8-11   softmax of row tile 0 and 1, a thread per row: S from
//               tensor memory twice (maximum, then weights), the weights back
//               over S as the left operand of the second product, and the
//               tile's output X added to the row's own in registers.
//
// Tensor memory: S / P and X of both row tiles, 128 columns each: all 512.
// X is not accumulated there over the tiles: the tensor cores cut their sums,
// which over 1,000 steps would cost 1e-5.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "hyq_kernels.h"
#include "hyq_paged.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kTile = 128;               // rows of a row tile, positions of a position tile
constexpr int kCtaRows = 2 * kTile;
constexpr int kThreads = 384;
constexpr int kSlots = 3;                // tiles of K or V in shared memory
constexpr int kMaxParts = 296;           // partial results of 256 rows in the workspace
// Floats of one: outputs, then (maximum, sum) of each row, then whether a value
// was taken out.
__host__ __device__ constexpr size_t part_floats(int dim) { return (size_t)kCtaRows * (dim + 2) + 4; }
constexpr float kBias = 10.0f;           // weights are kept 2^10 times their size (hyq_paged_mma.cu)
constexpr float kLog2e = 1.4426950408889634f;

template <int DIM>
struct Smem {
  static constexpr int half = kTile * 128;               // 128 rows of 64 f16
  static constexpr int tile = half * (DIM / 64);         // K, V, or one half (hi or lo) of a Q tile
  static constexpr int q = 0;                            // [row tile][hi, lo]
  static constexpr int ring = 4 * tile;
  static constexpr int bars = ring + kSlots * tile;
  // full[3], empty[3], s_full[2], p_full[2], o_full[2], clean[2]
  static constexpr int n_bars = 2 * kSlots + 8;
  static constexpr int misc = bars + 8 * n_bars;         // tensor memory address, abort, dirty, sequence, tile
  static constexpr int total = misc + 32 + 1024;         // the base is moved to 1024 bytes
};

struct Params {
  AttendArgs a;
  int box;        // rows of a TMA box: min(page_size, 128)
  int splits;     // parts of the positions; > 1: partial results
  float* parts;   // [row tile pair][kv head][split] (part_floats)
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(bar)
      : "memory");
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

// 32 columns of this thread's tensor memory lane.
__device__ __forceinline__ void tmem_ld32(float (&v)[32], uint32_t a) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(a));
}
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(a),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]),
      "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]),
      "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// Ten mantissa bits of a weight (exact in f16 from 2^-14 up).
__device__ __forceinline__ float high_part(float x) { return __uint_as_float(__float_as_uint(x) & 0xffffe000u); }

// A wait of a whole warp: true only if every lane saw the phase complete.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const volatile int* abort) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort));
}

template <int DIM>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ Params p) {
  using L = Smem<DIM>;
  constexpr int KS = DIM / 16;            // steps of 16 along the head
  constexpr int HALVES = DIM / 64;
  constexpr uint32_t kTmemCols = 512;
  const AttendArgs& a = p.a;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* base_g = smem_raw + (base - raw);
  auto full = [&](int s) { return base + L::bars + 8 * s; };
  auto empty = [&](int s) { return base + L::bars + 8 * (kSlots + s); };
  auto s_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + w); };
  auto p_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 2 + w); };
  auto o_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 4 + w); };
  auto clean = [&](int i) { return base + L::bars + 8 * (2 * kSlots + 6 + (i & 1)); };  // of masked tile i
  volatile int* misc = reinterpret_cast<volatile int*>(base_g + L::misc);
  volatile int* abort_flag = misc + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads, kvh = blockIdx.y;

  grid_dependency_wait();
  if (warp == 0) {
    int seq = -1, tile = 0;  // the last (longest) tiles first
    if (!find_tile(a.c, group, kCtaRows, gridDim.x - 1 - blockIdx.x, seq, tile)) seq = -1;
    if (lane == 0) {
      misc[1] = 0;
      misc[2] = 0;
      misc[3] = seq;
      misc[4] = tile;
      for (int s = 0; s < kSlots; ++s) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), 3);  // the products that read it, and warps 2 and 3
      }
      for (int w = 0; w < 2; ++w) {
        mbar_init(s_full(w), 1);
        mbar_init(p_full(w), 4);
        mbar_init(o_full(w), 1);
        mbar_init(clean(w), 2);
      }
      mbar_fence_init();
    }
  }
  __syncthreads();
  allow_dependents_launch();
  if (misc[3] < 0) return;  // nothing allocated yet
  const Seq s = load_seq(a.c, misc[3]);
  const int r0 = misc[4] * kCtaRows, rows = min(kCtaRows, s.n * group - r0);
  const bool two = rows > kTile;          // the second row tile has rows
  const int first_tok = r0 / group, last_tok = (r0 + rows - 1) / group;
  const int len = s.pos + last_tok + 1;   // positions the last row sees
  const int all_tiles = (len + kTile - 1) / kTile;
  const int j0 = (int)((int64_t)all_tiles * blockIdx.z / p.splits);
  const int nt = (int)((int64_t)all_tiles * (blockIdx.z + 1) / p.splits) - j0;
  // tiles from here on hold positions that some row does not see
  const int jm = max(0, (s.pos + first_tok + 1) / kTile - j0);
  float* part = p.splits > 1 ? p.parts + ((size_t)((gridDim.x - 1 - blockIdx.x) * gridDim.y + kvh) * p.splits + blockIdx.z) *
                                             part_floats(DIM)
                             : nullptr;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::misc), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // The queries, a row at a time per warp: scaled to [1, 2) by a power of two
  // that goes back into the scores, hi and lo into shared memory.
  const int wg = warp >= 8 ? 1 : 0;                          // row tile (softmax warps)
  const int r = r0 + wg * kTile + 32 * (warp & 3) + lane;    // row of the sequence, of this thread
  const int tok = min(r / group, s.n - 1);
  float factor = 1.0f;
  if (warp >= 4 && (wg == 0 || two)) {
    constexpr float scale = (DIM == 128 ? 0.08838834764831845f : 0.125f) * kLog2e;  // log2(e) / sqrt(DIM)
    constexpr int N = DIM / 32;  // values per lane
    uint8_t* q_s = base_g + L::q + wg * 2 * L::tile;
#pragma unroll 4
    for (int i = 0; i < 32; ++i) {
      const int row = 32 * (warp & 3) + i, rr = r0 + wg * kTile + row, t = rr / group;
      float x[N], top = 0.f;
      const float* q = a.q + (int64_t)(s.row0 + min(t, s.n - 1)) * a.q_stride + (int64_t)(kvh * group + rr % group) * DIM + N * lane;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        x[k] = t < s.n ? q[k] * scale : 0.f;
        top = fmaxf(top, fabsf(x[k]));
      }
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const int e = min(max((int)(__float_as_uint(top) >> 23), 1), 253);
      if (lane == i) factor = __uint_as_float((uint32_t)e << 23);
      const float down = __uint_as_float((uint32_t)(254 - e) << 23);
      uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        hi[k] = pack_f16(x[2 * k] * down, x[2 * k + 1] * down);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
        lo[k] = pack_f16(x[2 * k] * down - f.x, x[2 * k + 1] * down - f.y);
      }
      const int d = N * lane, c = d >> 3;  // 16-byte chunk of the row
      uint8_t* at = q_s + (c >> 3) * L::half + row * 128 + (((c ^ row) & 7) << 4) + (d & 7) * 2;
#pragma unroll
      for (int k = 0; k < N / 2; ++k) {
        *reinterpret_cast<uint32_t*>(at + 4 * k) = hi[k];
        *reinterpret_cast<uint32_t*>(at + L::tile + 4 * k) = lo[k];
      }
    }
    fence_proxy_async_smem();
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = (uint32_t)misc[0];

  if (warp < 4) {
    // launch: 168 registers x 384 threads; 72 x 128 + 216 x 256 is the same
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == 0) {
      // ------------------------------ pages in -------------------------------
      const int per = kTile / p.box;  // boxes of a tile: one lane each
      int issued = 0;
      bool ok = true;
      for (int i = 0; i < 2 * nt && ok; ++i) {  // K and V of each tile
        const int slot = i % kSlots, j = j0 + (i >> 1);
        const int pos = j * kTile + lane * p.box;
        int page = a.c.pages;  // past the pool: zeros
        if (lane < per && pos < len) {
          page = s.pages[pos / a.c.page_size];
          if (page < 0 || page >= a.c.pages) {
            atomicOr(a.c.status, DEV_BAD_ARGS);
            page = a.c.pages;
          }
        }
        if (i >= kSlots && !warp_wait(empty(slot), ((i / kSlots) - 1) & 1, abort_flag)) {
          ok = false;
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(full(slot), L::tile);
        __syncwarp();
        if (lane < per) {
          const CUtensorMap* map = (i & 1) ? &map_v : &map_k;
          const uint32_t dst = base + L::ring + slot * L::tile + lane * p.box * 128;
#pragma unroll
          for (int h = 0; h < HALVES; ++h)
            tma_load_4d(dst + h * L::half, map, 64 * h, pos % a.c.page_size, kvh, page, full(slot));
        }
        ++issued;
      }
      if (!ok) {
        if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_EMPTY);
        *abort_flag = 1;
      }
      // no copy may land after this CTA is gone
      for (int i = max(0, issued - kSlots); i < issued; ++i)
        if (!warp_wait(full(i % kSlots), (i / kSlots) & 1, nullptr) && lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_DRAIN);
    } else if (warp == 1) {
      // ------------------------------ products -------------------------------
      // f32 sums, f16 operands, M 128; N 128 positions, or DIM columns with V
      // along its rows (bit 16)
      constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
      constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DIM >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
      auto wait = [&](uint32_t bar, uint32_t parity) {
        if (warp_wait(bar, parity, abort_flag)) return true;
        if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_FULL);
        *abort_flag = 1;
        return false;
      };
      // lo first: the large sums then take half the (cut) additions
      auto scores = [&](int w, int slot) {
        const uint32_t q = base + L::q + w * 2 * L::tile, k = base + L::ring + slot * L::tile;
#pragma unroll
        for (int t = 0; t < KS; ++t) {
          const uint32_t off = (t >> 2) * L::half + (t & 3) * 32;
          mma_ss(tmem + 256 * w, desc_k_major(q + L::tile + off), desc_k_major(k + off), idesc_s, t > 0);
        }
#pragma unroll
        for (int t = 0; t < KS; ++t) {
          const uint32_t off = (t >> 2) * L::half + (t & 3) * 32;
          mma_ss(tmem + 256 * w, desc_k_major(q + off), desc_k_major(k + off), idesc_s, 1);
        }
      };
      auto outputs = [&](int w, int slot) {
        const uint32_t v = base + L::ring + slot * L::tile, pw = tmem + 256 * w;
#pragma unroll
        for (int h = 1; h >= 0; --h)
#pragma unroll
          for (int t = 0; t < kTile / 16; ++t)  // 16 positions: hi at 32 (t / 2) + 8 (t % 2), lo 16 columns on
            mma_ts(pw + 128, pw + 32 * (t >> 1) + 8 * (t & 1) + 16 * h, desc_mn_major(v + t * 16 * 128, L::half), idesc_o,
                   h == 0 || t > 0);
      };
      bool ok = nt > 0 && wait(full(0), 0);
      if (ok) {
        fence_after();
        if (lane == 0) {
          scores(0, 0);
          commit(s_full(0));
          if (two) {
            scores(1, 0);
            commit(s_full(1));
          }
          commit(empty(0));
        }
        __syncwarp();
      }
      for (int j = 0; j < nt && ok; ++j) {
        const int iv = 2 * j + 1, ik = 2 * j + 2;
        ok = wait(full(iv % kSlots), (iv / kSlots) & 1) && (j < jm || wait(clean(j - jm), ((j - jm) >> 1) & 1)) &&
             (j + 1 >= nt || wait(full(ik % kSlots), (ik / kSlots) & 1));
        for (int w = 0; w < (two ? 2 : 1) && ok; ++w) {
          ok = wait(p_full(w), j & 1);
          if (!ok) break;
          fence_after();
          if (lane == 0) {
            outputs(w, iv % kSlots);
            const bool last = w == (two ? 1 : 0);
            if (last) commit(empty(iv % kSlots));
            if (j + 1 < nt) {
              scores(w, ik % kSlots);
              commit(s_full(w));
              if (last) commit(empty(ik % kSlots));
            } else {
              commit(o_full(w));
            }
          }
          __syncwarp();
        }
      }
    } else {
      // --------------------------- what rows do not see -----------------------
      // (these warps follow every tile, and hold its slot: a wait that skipped
      // phases would take an earlier one for its own)
      bool ok = true;
      for (int i = 0; i < 2 * nt; ++i) {
        const int slot = i % kSlots, j = i >> 1;
        ok = warp_wait(full(slot), (i / kSlots) & 1, abort_flag);
        if (!ok) break;
        if (!(i & 1) || j < jm) {
          if (lane == 0) mbar_arrive(empty(slot));
          continue;
        }
        bool found = false;
        for (int x = threadIdx.x - 64; x < kTile * 8 * HALVES; x += 64) {  // 16-byte chunks
          const int row = (x >> 3) & (kTile - 1), pos = (j0 + j) * kTile + row;
          if (pos <= s.pos + first_tok) continue;
          uint4* at = reinterpret_cast<uint4*>(base_g + L::ring + slot * L::tile + x * 16);
          uint4 v = *at;
          uint32_t w[4] = {v.x, v.y, v.z, v.w};
          bool bad = false;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((w[k] & 0x7c00u) == 0x7c00u) w[k] &= 0xffff0000u, bad = true;
            if ((w[k] & 0x7c000000u) == 0x7c000000u) w[k] &= 0xffffu, bad = true;
          }
          if (bad) {
            *at = make_uint4(w[0], w[1], w[2], w[3]);
            found = found || pos < len;
          }
        }
        if (found) misc[2] = 1;
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(clean(j - jm));
          mbar_arrive(empty(slot));
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    if (wg == 0 || two) {
      // -------------------------------- softmax -------------------------------
      const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16), st = lanes + 256 * wg;
      const int sees = s.pos + tok;
      float o[DIM];
#pragma unroll
      for (int d = 0; d < DIM; ++d) o[d] = 0.f;
      float m = -INFINITY, l = 0.f, down = 1.f;
      bool ok = true;
      for (int j = 0; j < nt; ++j) {
        ok = warp_wait(s_full(wg), j & 1, abort_flag);
        if (!ok) break;
        fence_after();
        const int p0 = (j0 + j) * kTile;
        const bool masked = j >= jm;
        float top = -INFINITY;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          tmem_ld32(v, st + 32 * c);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (p0 + 32 * c + i > sees) v[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, v[i]);
        }
        const float now = fmaxf(m, top * factor);
        const float next_down = now == -INFINITY ? 1.f : ex2(m - now);
        const float back = kBias - (now == -INFINITY ? 0.f : now);
        float sum = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v[32];
          uint32_t w[32];
          tmem_ld32(v, st + 32 * c);
          tmem_wait_ld();
          if (masked) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (p0 + 32 * c + i > sees) v[i] = -INFINITY;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float x = ex2(fmaf(v[i], factor, back)), y = ex2(fmaf(v[i + 1], factor, back));
            sum += x + y;
            const float xh = high_part(x), yh = high_part(y);
            w[i >> 1] = pack_f16(xh, yh);
            w[16 + (i >> 1)] = pack_f16(x - xh, y - yh);
          }
          tmem_st32(st + 32 * c, w);
        }
        l = fmaf(l, next_down, sum);
        m = now;
        if (j > 0) {  // the tile before: its product is done (the scores came after it)
#pragma unroll
          for (int c = 0; c < DIM / 32; ++c) {
            float v[32];
            tmem_ld32(v, st + 128 + 32 * c);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[32 * c + i] = fmaf(o[32 * c + i], down, v[i]);
          }
        }
        down = next_down;
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(wg));
      }
      ok = ok && nt > 0 && warp_wait(o_full(wg), 0, abort_flag);
      if (ok) {
        fence_after();
#pragma unroll
        for (int c = 0; c < DIM / 32; ++c) {
          float v[32];
          tmem_ld32(v, st + 128 + 32 * c);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[32 * c + i] = fmaf(o[32 * c + i], down, v[i]);
        }
      } else if (nt > 0) {
        if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_FULL);
        *abort_flag = 1;
      }
      if (r < s.n * group && (ok || nt == 0)) {
        if (part) {
          float* to = part + (size_t)(r - r0) * DIM;
#pragma unroll
          for (int d = 0; d < DIM; d += 4) *reinterpret_cast<float4*>(to + d) = make_float4(o[d], o[d + 1], o[d + 2], o[d + 3]);
          float* ml = part + (size_t)kCtaRows * DIM + 2 * (r - r0);
          ml[0] = m;
          ml[1] = l;
          if (r == r0) part[(size_t)kCtaRows * (DIM + 2)] = misc[2] != 0 ? 1.0f : 0.0f;
        } else {
          float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r % group) * DIM;
          const float inv = 1.0f / l;
          const bool dirty = misc[2] != 0;
          if ((reinterpret_cast<uintptr_t>(to) & 15) == 0 && !dirty) {
#pragma unroll
            for (int d = 0; d < DIM; d += 4)
              *reinterpret_cast<float4*>(to + d) = make_float4(o[d] * inv, o[d + 1] * inv, o[d + 2] * inv, o[d + 3] * inv);
          } else {
#pragma unroll
            for (int d = 0; d < DIM; ++d)
              to[d] = o[d] * inv + (dirty ? non_finite<true>(a.c, s, kvh, s.pos + first_tok, sees, d) : 0.f);
          }
        }
      }
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

// The splits of a row joined: one warp per row, in the order of the splits.
template <int DIM>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Params p) {
  const AttendArgs& a = p.a;
  grid_dependency_wait();
  allow_dependents_launch();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = a.heads / a.c.kv_heads, kvh = blockIdx.y;
  const int want = blockIdx.x / (kCtaRows / 8), row = blockIdx.x % (kCtaRows / 8) * 8 + warp;
  int seq, tile;
  if (!find_tile(a.c, group, kCtaRows, want, seq, tile)) return;
  const Seq s = load_seq(a.c, seq);
  const int r0 = tile * kCtaRows, r = r0 + row;
  if (r >= s.n * group) return;
  const float* part = p.parts + (size_t)(want * gridDim.y + kvh) * p.splits * part_floats(DIM);
  constexpr size_t stride = part_floats(DIM);
  const float* ml = part + (size_t)kCtaRows * DIM + 2 * row;
  float m = lane < p.splits ? ml[lane * stride] : -INFINITY, top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float f = m == -INFINITY ? 0.f : ex2(m - top);
  const float l = warp_sum(lane < p.splits ? f * ml[lane * stride + 1] : 0.f);
  constexpr int N = DIM / 32;
  float o[N] = {};
  for (int i = 0; i < p.splits; ++i) {
    const float w = __shfl_sync(0xffffffffu, f, i);
#pragma unroll
    for (int k = 0; k < N; ++k) o[k] = fmaf(w, part[i * stride + (size_t)row * DIM + lane + 32 * k], o[k]);
  }
  const bool dirty = __any_sync(0xffffffffu, lane < p.splits && part[lane * stride + (size_t)kCtaRows * (DIM + 2)] != 0.f);
  const int tok = r / group, first = s.pos + r0 / group;
  float* to = a.out + (int64_t)(s.row0 + tok) * a.out_stride + (int64_t)(kvh * group + r % group) * DIM;
#pragma unroll
  for (int k = 0; k < N; ++k)
    to[lane + 32 * k] = o[k] / l + (dirty ? non_finite<true>(a.c, s, kvh, first, s.pos + tok, lane + 32 * k) : 0.f);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  });
  return fn;
}

// Pages as (head value, row, kv head, page); boxes of 64 values x `box` rows.
bool page_map(CUtensorMap* map, const void* base, const Cache& c, int box) {
  const cuuint64_t dims[4] = {(cuuint64_t)c.dim, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)c.row_stride * 2, (cuuint64_t)c.head_stride * 2, (cuuint64_t)c.page_stride * 2};
  const cuuint32_t size[4] = {64, (cuuint32_t)box, 1, 1}, step[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), dims, strides, size, step,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DIM>
cudaError_t launch(const AttendArgs& a, int64_t max_len, cudaStream_t st) {
  CUtensorMap mk, mv;
  Params p;
  p.a = a;
  p.box = std::min(a.c.page_size, kTile);
  if (!page_map(&mk, a.c.k, a.c, p.box) || !page_map(&mv, a.c.v, a.c, p.box)) return cudaErrorInvalidValue;
  const int64_t tiles = ((int64_t)a.c.tokens * (a.heads / a.c.kv_heads) + kCtaRows - 1) / kCtaRows + a.c.seqs;
  // Few CTAs (a chunk of one request): the positions are cut so that every SM
  // has one, at least four tiles each.
  const int64_t ctas = tiles * a.c.kv_heads;
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({148 / ctas, kMaxParts / ctas, max_len / (4 * kTile), 32}));
  p.parts = reinterpret_cast<float*>(static_cast<char*>(a.ws) + mma_workspace_bytes(DIM));
  auto k = chunk_tc_kernel<DIM>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(k, Smem<DIM>::total, done);
  if (e != cudaSuccess) return e;
  e = launch_ex(k, dim3((unsigned)tiles, (unsigned)a.c.kv_heads, (unsigned)p.splits), dim3(kThreads), Smem<DIM>::total, st,
                mk, mv, p);
  if (e != cudaSuccess || p.splits == 1) return e;
  return launch_ex(join_kernel<DIM>, dim3((unsigned)(tiles * (kCtaRows / 8)), (unsigned)a.c.kv_heads), dim3(256), 0, st, p);
}

}  // namespace

bool tc_supported(const AttendArgs& a, bool kv16) {
  const int ps = a.c.page_size;
  return kv16 && (ps == 16 || ps == 32 || ps == 64 || ps % kTile == 0) && encode_fn() != nullptr;
}

size_t tc_workspace_bytes(int dim) { return kMaxParts * part_floats(dim) * sizeof(float); }

cudaError_t launch_chunks_tc(const AttendArgs& a, int64_t max_len, cudaStream_t st) {
  return a.c.dim == 128 ? launch<128>(a, max_len, st) : launch<64>(a, max_len, st);
}

}  // namespace paged
}  // namespace hyq
