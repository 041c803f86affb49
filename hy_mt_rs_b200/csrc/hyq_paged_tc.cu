// Attention of chunks of new tokens over an f16 paged cache on tcgen05, head
// sizes 64 and 128, at f32 accuracy.
//
// Work is cut into segments: two tiles of 128 (token, query head) rows of one
// sequence and kv head, over the positions they see in tiles of 128.  All
// segments' position tiles form one line, cut into equal ranges, one per SM
// (plan_kernel lists the segments); a segment that spans CTAs leaves partial
// results, which join_kernel adds up.  Queries and weights
// are hi + lo, both f16 (22 bits), K and V exact, so a tile pair costs
//   S = Qh K' + Ql K'   and   X = Ph V + Pl V,
// four 128 x 128 x 128 products: twice those of plain f16 attention, which is
// what bounds the kernel (half the tensor cores' f16 rate), together with the
// power limit.  4,096 tokens over 12,288 positions, 32 query and 8 kv heads of
// 128: 1.43 ms at 1,965 MHz (ten calls after a pause), 1.64 ms back to back, where
// the card draws 989 W of its 1,000 and holds 1,507 to 1,575 MHz: 585 to 670
// TFLOP/s of 2 x 2 x heads x head size x pairs, 71 to 81 % of half the measured
// 1,657 (tensor pipe 69 % busy).  Two row tiles, so
// that one's products run under the other's softmax; a tile's 32 steps of 16 take
// 64 cycles each, its softmax about as long.
//
//   warp 0      TMA: pages of K and V into a ring of three tiles (128-byte
//               swizzle; pages past the sequence come as zeros);
//   warp 1      tcgen05.mma: S of one row tile while the other's softmax runs;
//   warps 2-3   take non-finite values out of V at positions that some row of
//               the CTA does not see (0 times them would be NaN);
//   warps 4-7, 8-11   softmax of row tile 0 and 1, a thread per row: S from
//               tensor memory, the weights back over it as the left operand of
//               the second product, and the tile's output X added to the row's
//               own in registers.
//
// Tensor memory: S / P and X of both row tiles, 128 columns each: all 512.
// X is not accumulated there over the tiles: the tensor cores cut their sums,
// which over 1,000 steps would cost 1e-5.
//
// PREFIX: the segments are groups' tokens over their shared prefix, few rows over many
// positions: one row tile a segment, whose position tiles the two softmax groups take
// in turn (their halves meet through tensor memory at the end), and five slots in the
// ring, in the place of the other row tile's queries.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>

#include "hyq_kernels.h"
#include "hyq_paged_tc.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kCtaRows = 2 * kTile;      // rows of a segment
constexpr int kThreads = 384;

template <int DIM, bool PREFIX>
struct Smem {
  static constexpr int slots = PREFIX ? kPrefixSlots : 3;
  static constexpr int half = kTile * 128;               // 128 rows of 64 f16
  static constexpr int tile = half * (DIM / 64);         // K, V, or one half (hi or lo) of a Q tile
  static constexpr int q = 0;                            // [row tile][hi, lo]
  static constexpr int ring = (PREFIX ? 2 : 4) * tile;
  static constexpr int bars = ring + slots * tile;
  // A tile's turn among these comes when the products have waited for the one that had
  // it before: V of masked tile i + cleans is in a slot of the ring that is only free
  // when a product behind that wait is done (five slots: of K of the next piece).
  static constexpr int cleans = PREFIX ? 3 : 2;
  // full[slots], empty[slots], s_full[2], p_full[2], x_full[2], q_full[2], half[2], clean[cleans]
  static constexpr int n_bars = 2 * slots + 10 + cleans;
  static constexpr int factors = bars + 8 * n_bars;      // (prefixes) powers of two of the rows' queries
  static constexpr int misc = factors + (PREFIX ? kTile * 4 : 0);         // tensor memory address, abort, unused, dirty
  static constexpr int total = misc + 32 + 1024;         // the base is moved to 1024 bytes
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int row, int head, int page, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(row), "r"(head), "r"(page), "r"(bar)
      : "memory");
}

template <int DIM, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1)
    chunk_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ Params p) {
  using L = Smem<DIM, PREFIX>;
  constexpr int kSlots = L::slots, ROWS = PREFIX ? kPrefixRows : kCtaRows;
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
  auto x_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 4 + w); };
  auto q_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 6 + w); };
  auto half = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 8 + w); };  // given, taken (split pieces)
  auto clean = [&](int i) { return base + L::bars + 8 * (2 * kSlots + 10 + i % L::cleans); };  // of masked tile i: phase i / cleans
  volatile int* misc = reinterpret_cast<volatile int*>(base_g + L::misc);
  volatile int* abort_flag = misc + 1;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads;

  grid_dependency_wait();
  allow_dependents_launch();
  const int cta = blockIdx.x;
  const Start start = p.plan.start[cta];
  const int64_t begin = start.begin, end = p.plan.start[cta + 1].begin;
  if (begin == end) return;  // nothing allocated yet
  if (warp == 0) {
    if (lane == 0) {
      misc[1] = 0;
      misc[3] = 0;
      for (int s = 0; s < kSlots; ++s) {
        mbar_init(full(s), 1);
        mbar_init(empty(s), 3);  // the products that read it, and warps 2 and 3
      }
      for (int w = 0; w < 2; ++w) {
        mbar_init(s_full(w), 1);
        mbar_init(p_full(w), 4);
        mbar_init(x_full(w), 1);
        mbar_init(q_full(w), 4);
        mbar_init(half(w), 4);
      }
      for (int i = 0; i < L::cleans; ++i) mbar_init(clean(i), 2);
      mbar_fence_init();
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::misc), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = (uint32_t)uniform(misc[0]);
  // every warp walks the same pieces: (segment, kv head), at its tile `at`
  int t = start.t, kvh = start.kvh;
  int64_t at = begin;
  auto next = [&](const Piece& x) {
    at += x.nt;
    if (++t == p.plan.count[0]) {
      t = 0;
      ++kvh;
    }
  };

  if (warp < 4) {
    // launch: 168 registers x 384 threads; 104 x 128 + 200 x 256 is the same
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    if (warp == 0) {
      // ------------------------------ pages in -------------------------------
      const int per = kTile / p.box;  // boxes of a tile: one lane each
      int issued = 0;
      bool ok = true;
      while (at < end && ok) {
        const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
        for (int i = 0; i < 2 * x.nt; ++i) {  // K and V of each tile
          const int slot = issued % kSlots, pos = (x.j0 + (i >> 1)) * kTile + lane * p.box;
          int page = a.c.pages;  // past the pool: zeros
          if (lane < per && pos < x.len) {
            page = x.s.pages[pos / a.c.page_size];
            if (page < 0 || page >= a.c.pages) {
              atomicOr(a.c.status, DEV_BAD_ARGS);
              page = a.c.pages;
            }
          }
          if (issued >= kSlots && !warp_wait(empty(slot), ((issued / kSlots) - 1) & 1, abort_flag)) {
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
              tma_load_4d(dst + h * L::half, map, 64 * h, pos % a.c.page_size, x.kvh, page, full(slot));
          }
          ++issued;
        }
        next(x);
      }
      if (!ok) {
        if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_EMPTY);
        *abort_flag = 1;
      }
      // no copy may land after this CTA is gone, and no product's arrival
      for (int i = max(0, issued - kSlots); i < issued; ++i) {
        const bool in = warp_wait(full(i % kSlots), (i / kSlots) & 1, nullptr);
        const bool out = warp_wait(empty(i % kSlots), (i / kSlots) & 1, abort_flag);
        if (!(in && out) && lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_DRAIN);
      }
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
      // (addresses are in the low bits of a descriptor, 16 bytes a unit)
      const uint64_t q_desc = desc_k_major(base + L::q), k_desc = desc_k_major(base + L::ring);
      const uint64_t v_desc = desc_mn_major(base + L::ring, L::half);
      const bool one = elect();
      // lo first: the large sums then take half the (cut) additions
      auto scores = [&](int w, int slot) {
        const uint64_t q = q_desc + (PREFIX ? 0 : w) * (2 * L::tile >> 4), k = k_desc + slot * (L::tile >> 4);
#pragma unroll
        for (int h = 1; h >= 0; --h)
#pragma unroll
          for (int t = 0; t < KS; ++t) {
            const int off = ((t >> 2) * L::half + (t & 3) * 32) >> 4;
            mma_ss(tmem + 256 * w, q + h * (L::tile >> 4) + off, k + off, idesc_s, h == 0 || t > 0);
          }
      };
      auto outputs = [&](int w, int slot) {
        const uint64_t v = v_desc + slot * (L::tile >> 4);
        const uint32_t pw = tmem + 256 * w;
#pragma unroll
        for (int h = 1; h >= 0; --h)
#pragma unroll
          for (int t = 0; t < kTile / 16; ++t)  // 16 positions: hi in 8 columns from 16 t, lo in the next 8
            mma_ts(pw + 128, pw + 16 * t + 8 * h, v + t * (16 * 128 >> 4), idesc_o, h == 0 || t > 0);
      };
      // slot and phase of the ring's next tile
      int slot = 0, phase = 0, masked = 0, operand = 0;
      auto advance = [&]() {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      int steps[2] = {0, 0}, pieces[2] = {0, 0};
      bool ok = true;
      while (at < end && ok) {
        const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
        const int active = uniform(x.two ? 2 : 1), nt = uniform(x.nt), jm = uniform(x.jm);
        if constexpr (PREFIX) {
          // tile j is group j % 2's; operands 2 j (K) and 2 j + 1 (V) behind `operand`
          const int first = operand;
          operand += 2 * nt;
          auto scores_of = [&](int j) {
            const int n = first + 2 * j, w = j & 1;
            ok = wait(full(n % kSlots), (n / kSlots) & 1);
            if (!ok) return;
            fence_after();
            if (one) {
              scores(w, n % kSlots);
              commit(s_full(w));
              commit(empty(n % kSlots));
            }
            __syncwarp();
          };
          ok = wait(q_full(0), pieces[0] & 1);
          ++pieces[0];
          if (ok) scores_of(0);
          if (ok && nt > 1) scores_of(1);
          for (int j = 0; j < nt && ok; ++j) {
            const int n = first + 2 * j + 1, w = j & 1;
            ok = wait(full(n % kSlots), (n / kSlots) & 1);
            if (ok && j >= jm) {
              ok = wait(clean(masked), (masked / L::cleans) & 1);
              ++masked;
            }
            ok = ok && wait(p_full(w), steps[w] & 1);
            if (!ok) break;
            ++steps[w];
            fence_after();
            if (one) {
              outputs(w, n % kSlots);
              commit(x_full(w));
              commit(empty(n % kSlots));
            }
            __syncwarp();
            if (j + 2 < nt) scores_of(j + 2);
          }
          next(x);
          continue;
        }
        ok = wait(full(slot), phase);
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          if (w >= active || !ok) break;
          ok = wait(q_full(w), pieces[w] & 1);
          if (!ok) break;
          fence_after();
          if (one) {
            scores(w, slot);
            commit(s_full(w));
            if (w == active - 1) commit(empty(slot));
          }
          __syncwarp();
        }
        advance();
        for (int j = 0; j < nt && ok; ++j) {
          const int v_slot = slot;
          ok = wait(full(slot), phase);
          advance();
          if (ok && j >= jm) {
            ok = wait(clean(masked), (masked / L::cleans) & 1);
            ++masked;
          }
          const int k_slot = slot;
          if (ok && j + 1 < nt) {
            ok = wait(full(slot), phase);
            advance();
          }
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            if (w >= active || !ok) break;
            ok = wait(p_full(w), steps[w] & 1);
            if (!ok) break;
            ++steps[w];
            fence_after();
            if (one) {
              outputs(w, v_slot);
              commit(x_full(w));
              if (w == active - 1) commit(empty(v_slot));
              if (j + 1 < nt) {
                scores(w, k_slot);
                commit(s_full(w));
                if (w == active - 1) commit(empty(k_slot));
              }
            }
            __syncwarp();
          }
        }
        ++pieces[0];
        if (active == 2) ++pieces[1];
        next(x);
      }
    } else {
      // --------------------------- what rows do not see -----------------------
      // (these warps follow every tile, and hold its slot: a wait that skipped
      // phases would take an earlier one for its own)
      bool ok = true;
      int i0 = 0, masked = 0;
      while (at < end && ok) {
        const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
        for (int i = 0; i < 2 * x.nt; ++i, ++i0) {
          const int slot = i0 % kSlots, j = i >> 1;
          ok = warp_wait(full(slot), (i0 / kSlots) & 1, abort_flag);
          if (!ok) break;
          if (!(i & 1) || j < x.jm) {
            if (lane == 0) mbar_arrive(empty(slot));
            continue;
          }
          bool found = false;
          for (int c = threadIdx.x - 64; c < kTile * 8 * HALVES; c += 64) {  // 16-byte chunks
            const int pos = (x.j0 + j) * kTile + ((c >> 3) & (kTile - 1));
            if (pos <= x.s.pos + x.first_tok) continue;
            uint4* ptr = reinterpret_cast<uint4*>(base_g + L::ring + slot * L::tile + c * 16);
            const uint4 v = *ptr;
            uint32_t w[4] = {v.x, v.y, v.z, v.w};
            bool bad = false;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if ((w[k] & 0x7c00u) == 0x7c00u) w[k] &= 0xffff0000u, bad = true;
              if ((w[k] & 0x7c000000u) == 0x7c000000u) w[k] &= 0xffffu, bad = true;
            }
            if (bad) {
              *ptr = make_uint4(w[0], w[1], w[2], w[3]);
              found = found || pos < x.len;
            }
          }
          if (found) misc[3] = 1;  // (from here on: these warps may be pieces ahead of the rows that ask)
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(clean(masked));
            mbar_arrive(empty(slot));
          }
          ++masked;
        }
        next(x);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // -------------------------------- softmax -------------------------------
    const int wg = warp >= 8 ? 1 : 0;  // row tile
    const uint32_t st = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 256 * wg;
    int steps = 0, splits = 0;
    bool ok = true;
    while (at < end && ok) {
      const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
      const int r0 = x.r0 + (PREFIX ? 0 : wg * kTile), r = r0 + 32 * (warp & 3) + lane;  // row of the sequence
      const int tok = min(r / group, x.s.n - 1), sees = x.s.pos + x.step * tok;
      const int64_t piece_at = at;
      next(x);
      if (!PREFIX && wg == 1 && !x.two) continue;
      float factor;
      float* factor_s = reinterpret_cast<float*>(base_g + L::factors) + 32 * (warp & 3) + lane;
      uint8_t* q_s = base_g + L::q + (PREFIX ? 0 : wg) * 2 * L::tile;
      if (!PREFIX || wg == 0) {
        factor = stage_rows<DIM>(a, x, group, r0, q_s);
        if (PREFIX) *factor_s = factor;
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full(wg));
      } else {
        ok = warp_wait(q_full(0), splits & 1, abort_flag);
        factor = *factor_s;
      }
      float o[DIM];
#pragma unroll
      for (int d = 0; d < DIM; ++d) o[d] = 0.f;
      float m = -INFINITY, l = 0.f, down = 1.f;
      // the product of the tile before, added to the row's outputs
      auto collect = [&](int step) {
        if (!warp_wait(x_full(wg), step & 1, abort_flag)) return false;
        fence_after();
        tmem_each<DIM>(st + 128, [&](float (&v)[16], int c) {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[c + i] = fmaf(o[c + i], down, v[i]);
        });
        return true;
      };
      const int j0 = PREFIX ? wg : 0, by = PREFIX ? 2 : 1;
      for (int j = j0; j < x.nt && ok; j += by, ++steps) {
        // (while the tensor cores are at this tile's scores)
        ok = (j == j0 || collect(steps - 1)) && warp_wait(s_full(wg), steps & 1, abort_flag);
        if (!ok) break;
        fence_after();
        scores_to_weights(st, j == j0, j >= x.jm, sees - (x.j0 + j) * kTile + 1, factor, m, l, down, [](float (&)[32], int) {});
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(wg));
      }
      ok = ok && (j0 >= x.nt || collect(steps - 1));
      if (PREFIX && ok) {
        if (wg == 1) {
          give_half<DIM>(st, o, m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(half(0));
          ok = warp_wait(half(1), splits & 1, abort_flag);
        } else {
          ok = warp_wait(half(0), splits & 1, abort_flag);
          if (ok) take_half<DIM>(st + 256, o, m, l);
          __syncwarp();
          if (lane == 0) mbar_arrive(half(1));
        }
        ++splits;
      }
      if (!ok) {
        if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_FULL);
        *abort_flag = 1;
        break;
      }
      if (PREFIX && wg == 1) continue;
      const bool dirty = misc[3] != 0;
      store_rows<DIM, ROWS, kF16>(p, x, group, cta, piece_at != begin, r, q_s, o, m, l, dirty);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
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

template <int DIM, bool PREFIX>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
  CUtensorMap mk, mv;
  constexpr int ROWS = PREFIX ? kPrefixRows : kCtaRows;
  Params p;
  p.a = a;
  p.box = std::min(a.c.page_size, kTile);
  if (!page_map(&mk, a.c.k, a.c, p.box) || !page_map(&mv, a.c.v, a.c, p.box)) return cudaErrorInvalidValue;
  char* ws = static_cast<char*>(a.ws) + mma_workspace_bytes(DIM);
  p.plan = plan_of<ROWS>(a, ws);
  p.plan.least = 6;
  p.parts = reinterpret_cast<float*>(ws + kPlanBytes);
  auto k = chunk_tc_kernel<DIM, PREFIX>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(k, Smem<DIM, PREFIX>::total, done);
  if (e == cudaSuccess) e = launch_plan<ROWS, PREFIX>(a, p.plan, st);
  if (e == cudaSuccess) e = launch_next(k, dim3(kMaxCtas), dim3(kThreads), Smem<DIM, PREFIX>::total, st, mk, mv, p);
  if (e == cudaSuccess) e = launch_beside(a, kF16, st);
  if (e == cudaSuccess) e = launch_last<DIM, ROWS, PREFIX, kF16>(p, st);
  return e;
}

}  // namespace

bool tc_supported(const AttendArgs& a) {
  const int ps = a.c.page_size;
  return (ps == 16 || ps == 32 || ps == 64 || ps % kTile == 0) &&
         (a.groups.n ? plan_fits<kPrefixRows>(a) : plan_fits<kCtaRows>(a)) && encode_fn() != nullptr;
}

size_t tc_workspace_bytes(int dim) { return kPlanBytes + kMaxParts * part_floats<kCtaRows>(dim) * sizeof(float); }

cudaError_t launch_chunks_tc(const AttendArgs& a, cudaStream_t st) {
  if (a.groups.n) return a.c.dim == 128 ? launch<128, true>(a, st) : launch<64, true>(a, st);
  return a.c.dim == 128 ? launch<128, false>(a, st) : launch<64, false>(a, st);
}

}  // namespace paged
}  // namespace hyq
