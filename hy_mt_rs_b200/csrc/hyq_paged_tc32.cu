// Attention of chunks of new tokens over an f32 paged cache on tcgen05, head
// sizes 64 and 128, at f32 accuracy.
//
// The f16 kernel's line of segments and its softmax (hyq_paged_tc.cuh), with
// segments of one tile of 128 rows and with both operands split: a position of
// K and a tile of V are scaled by a power of two that puts their largest value
// in [2^14, 2^15) and written as hi + lo, both f16 (22 bits of every value down
// to 2^-18 of the largest, 2^-40 of that below), and
//   S = Qh Kh' + Qh Kl' + Ql Kh'   and   X = Ph Vh + Ph Vl + Pl Vh,
// six 128 x 128 x 128 products a tile (Ql Kl' is below f32's last bit).  tf32
// operands would need no scales, but run at half the rate and fill twice the
// shared memory.
//
//   warps 0-3    softmax, a thread per row;
//   warps 4-11   K and V from global memory, 16 positions a warp, a row per
//                load: to registers while the tensor cores read the tile
//                before, then split into shared memory.  K has a scale for
//                each position, undone in its column of scores; V one for the
//                tile, known when all warps have seen their part, undone in X;
//   warp 12      the products S, into two buffers in turn;
//   warp 13      the products X, likewise: a tile's is added to the outputs while
//                the next tile's weights are multiplied.
//
// Three chunks of 201 to 256 tokens over up to 2,300 positions, 16 query and 4
// kv heads of 128: 63 us with plan and join (the warp-level kernel on tf32 took
// 470).  A CTA's start takes 10 us and a tile of positions 5 us, the chain of its
// split, scores, weights and outputs; the six products alone take 1.6.
//
// A tile with an infinity or NaN, or whose positions' largest values of V are
// more than 2^14 apart, is left out of the products (V and the weights are
// zeros there); each softmax thread then goes through the positions that its
// row sees, in f32 (a value that a row does not see can then not reach it).
#include "hyq_paged_tc.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kRows = kTile;          // rows of a segment
constexpr int kThreads = 512;
constexpr int kSplitWarps = 8;
constexpr int kPart = kTile / kSplitWarps;   // positions of a warp
constexpr int kSpread = 14;           // of the positions' largest exponents of V

template <int DIM>
struct Smem {
  static constexpr int half = kTile * 128;               // 128 rows of 64 f16
  static constexpr int tile = half * (DIM / 64);
  static constexpr int q = 0, k = 2 * tile, v = 4 * tile;  // [hi, lo] each
  static constexpr int scale = 6 * tile;                 // [2][128]: 2^-n of K's positions
  static constexpr int top = scale + 2 * kTile * 4;      // [2][8 warps] largest, smallest bits of V
  static constexpr int bars = top + 2 * kSplitWarps * 8;
  // k_full, v_full, v_top, p_full[2], s_full[2], x_full[2]
  static constexpr int n_bars = 9;
  // tensor memory address, abort, unused, then [2] of: tile that is left
  // out (its number + 1), scale of X
  static constexpr int misc = bars + 8 * n_bars;
  static constexpr int total = misc + 32 + 1024;         // the base is moved to 1024 bytes
};

// A row's values of one lane, hi and lo, to their places in a tile at `to`
// (128-byte swizzle, lo one tile behind).
template <int DIM>
__device__ __forceinline__ void put_row(uint8_t* to, int row, const float (&x)[DIM / 32], float scale) {
  constexpr int N = DIM / 32, half = kTile * 128, tile = half * (DIM / 64);
  const int d = N * (threadIdx.x & 31), c = d >> 3;
  to += (c >> 3) * half + row * 128 + (((c ^ row) & 7) << 4) + (d & 7) * 2;
  uint32_t hi[N / 2], lo[N / 2];
#pragma unroll
  for (int k = 0; k < N / 2; ++k) {
    const float x0 = x[2 * k] * scale, x1 = x[2 * k + 1] * scale;
    hi[k] = pack_f16(x0, x1);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hi[k]));
    lo[k] = pack_f16(x0 - f.x, x1 - f.y);
  }
  if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(to) = make_uint2(hi[0], hi[1]);
    *reinterpret_cast<uint2*>(to + tile) = make_uint2(lo[0], lo[1]);
  } else {
    *reinterpret_cast<uint32_t*>(to) = hi[0];
    *reinterpret_cast<uint32_t*>(to + tile) = lo[0];
  }
}

// Bits of the largest magnitude of a row, the same in all lanes (from
// 0x7f800000 up: the row has an infinity or NaN).
template <int N>
__device__ __forceinline__ uint32_t row_top(const float (&x)[N]) {
  uint32_t t = 0;
#pragma unroll
  for (int k = 0; k < N; ++k) t = max(t, __float_as_uint(x[k]) & 0x7fffffffu);
  return __reduce_max_sync(0xffffffffu, t);
}
// 2^n that takes values whose largest has these bits below 2^15 (to 2^14 and
// more, unless they are below 2^-86), and 2^-n.
__device__ __forceinline__ uint32_t exponent(uint32_t top) { return max(min(top >> 23, 254u), 41u); }
__device__ __forceinline__ float scale_of(uint32_t top) { return __uint_as_float((268u - exponent(top)) << 23); }
__device__ __forceinline__ float unscale_of(uint32_t top) { return __uint_as_float((exponent(top) - 14u) << 23); }

template <int DIM, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1) chunk_tc32_kernel(const __grid_constant__ Params p) {
  using L = Smem<DIM>;
  constexpr int KS = DIM / 16;            // steps of 16 along the head
  constexpr int N = DIM / 32;             // values of a lane
  constexpr uint32_t kTmemCols = 512;     // S and P twice 128, X twice 128
  const AttendArgs& a = p.a;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* base_g = smem_raw + (base - raw);
  const uint32_t k_full = base + L::bars, v_full = k_full + 8, v_top = k_full + 16;
  // Of tile i: phase i / 2.  (Two of p_full as well: a softmax warp may be done
  // with tile i + 1 before another is with i, and its arrival must not count for
  // i; with i + 2 it is done only after X(i), which takes all of i's.)
  auto p_full = [&](int i) { return k_full + 24 + 8 * (i & 1); };
  auto s_full = [&](int i) { return k_full + 40 + 8 * (i & 1); };
  auto x_full = [&](int i) { return k_full + 56 + 8 * (i & 1); };
  float* scale_s = reinterpret_cast<float*>(base_g + L::scale);
  volatile int* misc = reinterpret_cast<volatile int*>(base_g + L::misc);
  volatile int* abort_flag = misc + 1;
  volatile int* out_s = misc + 3;
  volatile float* back_s = reinterpret_cast<volatile float*>(misc + 5);
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads;

  grid_dependency_wait();
  allow_dependents_launch();
  const int cta = blockIdx.x;
  const Start start = p.plan.start[cta];
  const int64_t begin = start.begin, end = p.plan.start[cta + 1].begin;
  if (begin == end) return;  // nothing allocated yet
  const int tiles = uniform((int)(end - begin));
  if (warp == 0) {
    if (lane == 0) {
      misc[1] = 0;
      misc[3] = misc[4] = 0;
      mbar_init(k_full, kSplitWarps + 4);  // K is there, and the queries: the softmax warps
      mbar_init(v_full, kSplitWarps);
      mbar_init(v_top, kSplitWarps);
      for (int i = 0; i < 2; ++i) {
        mbar_init(p_full(i), 4);
        mbar_init(s_full(i), 1);
        mbar_init(x_full(i), 1);
      }
      mbar_fence_init();
    }
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + L::misc), "r"(kTmemCols));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = (uint32_t)uniform(misc[0]);
  int t = start.t, kvh = start.kvh;
  int64_t at = begin;
  auto next = [&](const Piece& x) {
    at += x.nt;
    if (++t == p.plan.count[0]) {
      t = 0;
      ++kvh;
    }
  };
  bool ok = true;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    ok = ok && warp_wait(bar, parity & 1, abort_flag);
    return ok;
  };

  // launch: 128 registers x 512 threads = (200 + 2 x 136 + 40) x 128
  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // f32 sums, f16 operands, M 128; N 128 positions, or DIM columns with V
    // along its rows (bit 16).  Small products first: the large sums then take
    // fewer (cut) additions.
    constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kTile >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
    constexpr uint32_t idesc_o = (1u << 4) | (1u << 16) | ((uint32_t)(DIM >> 3) << 17) | ((uint32_t)(kTile >> 4) << 24);
    const bool one = elect();
    if (warp == 12) {
      const uint64_t q = desc_k_major(base + L::q), k = desc_k_major(base + L::k);
      for (int i = 0; i < tiles && wait(k_full, i); ++i) {
        fence_after();
        if (one) {
#pragma unroll
          for (int h = 0; h < 3; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s) {
              const int off = ((s >> 2) * L::half + (s & 3) * 32) >> 4;
              mma_ss(tmem + 128 * (i & 1), q + (h == 0 ? L::tile >> 4 : 0) + off, k + (h == 1 ? L::tile >> 4 : 0) + off, idesc_s,
                     h > 0 || s > 0);
            }
          commit(s_full(i));
        }
        __syncwarp();
      }
    } else if (warp == 13) {
      const uint64_t v = desc_mn_major(base + L::v, L::half);
      for (int i = 0; i < tiles && wait(v_full, i) && wait(p_full(i), i >> 1); ++i) {
        fence_after();
        if (one) {
          const uint32_t pw = tmem + 128 * (i & 1);
#pragma unroll
          for (int h = 0; h < 3; ++h)
#pragma unroll
            for (int s = 0; s < kTile / 16; ++s)  // 16 positions: hi in 8 columns from 16 s, lo in the next 8
              mma_ts(tmem + 256 + 128 * (i & 1), pw + 16 * s + (h == 0 ? 8 : 0), v + (h == 1 ? L::tile >> 4 : 0) + s * (16 * 128 >> 4), idesc_o,
                     h > 0 || s > 0);
          commit(x_full(i));
        }
        __syncwarp();
      }
    }
  } else if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
    // ------------------------------ K and V ---------------------------------
    const int sw = warp - 4, row0 = kPart * sw;
    uint8_t* k_s = base_g + L::k;
    uint8_t* v_s = base_g + L::v;
    uint2* top_s = reinterpret_cast<uint2*>(base_g + L::top);
    Piece x = piece_of<kRows, PREFIX>(p, group, t, kvh, at, end);
    int j = 0;
    // where position row0 + lane % 16 of the tile begins, or -1
    auto place = [&]() {
      const int pos = (x.j0 + j) * kTile + row0 + (lane & (kPart - 1));
      if (pos >= x.len) return (int64_t)-1;
      const int page = checked_page(a.c, x.s.pages[pos / a.c.page_size]);
      if (page < 0) return (int64_t)-1;
      return (int64_t)page * a.c.page_stride + (int64_t)x.kvh * a.c.head_stride + (int64_t)(pos % a.c.page_size) * a.c.row_stride;
    };
    auto load = [&](float (&v)[N], const void* from, int64_t places, int i) {
      const int64_t o = __shfl_sync(0xffffffffu, places, i);
      const float* row = static_cast<const float*>(from) + o + N * lane;
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = 0.f;
      // (predicated, not branched around: branches would keep the rows apart)
      if constexpr (N == 4)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %4, 0;\n\t@p ld.global.v4.f32 {%0, %1, %2, %3}, [%5];\n\t}"
                     : "+f"(v[0]), "+f"(v[1]), "+f"(v[N - 2]), "+f"(v[N - 1])
                     : "l"(o), "l"(row));
      else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %2, 0;\n\t@p ld.global.v2.f32 {%0, %1}, [%3];\n\t}"
                     : "+f"(v[0]), "+f"(v[1])
                     : "l"(o), "l"(row));
    };
    float kr[kPart / 2][N], vr[kPart][N];
    int64_t here = place(), there = -1;
#pragma unroll
    for (int r = 0; r < kPart / 2; ++r) load(kr[r], a.c.k, here, r);
#pragma unroll
    for (int r = 0; r < kPart; ++r) load(vr[r], a.c.v, here, r);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      if (i + 1 < tiles) {
        if (++j == x.nt) {
          next(x);
          x = piece_of<kRows, PREFIX>(p, group, t, kvh, at, end);
          j = 0;
        }
        there = place();
      } else {
        there = -1;
      }
      if (i > 0 && !wait(s_full(i - 1), (i - 1) >> 1)) break;
      auto put_keys = [&](int r0) {
        uint32_t top[kPart / 2], own = 0;  // own: of row r0 + lane
#pragma unroll
        for (int r = 0; r < kPart / 2; ++r) {
          top[r] = row_top(kr[r]);
          own = lane == r ? top[r] : own;
        }
#pragma unroll
        for (int r = 0; r < kPart / 2; ++r) put_row<DIM>(k_s, row0 + r0 + r, kr[r], scale_of(top[r]));
        if (lane < kPart / 2) {
          scale_s[(i & 1) * kTile + row0 + r0 + lane] = unscale_of(own);
          if (own >= 0x7f800000u) out_s[i & 1] = i + 1;
        }
      };
      put_keys(0);
#pragma unroll
      for (int r = 0; r < kPart / 2; ++r) load(kr[r], a.c.k, here, kPart / 2 + r);
      // V's largest value, and the smallest of its positions' largest
      uint32_t most = 0, least = 0xffffffffu;
#pragma unroll
      for (int r = 0; r < kPart; ++r) {
        const uint32_t top = row_top(vr[r]);
        most = max(most, top);
        least = min(least, top ? top : 0xffffffffu);
      }
      if (lane == 0) {
        top_s[(i & 1) * kSplitWarps + sw] = make_uint2(most, least);
        mbar_arrive(v_top);
      }
      if (!wait(v_top, i)) break;
#pragma unroll
      for (int w = 0; w < kSplitWarps; ++w) {
        const uint2 o = top_s[(i & 1) * kSplitWarps + w];
        most = max(most, o.x);
        least = min(least, o.y);
      }
      const bool out = most >= 0x7f800000u || (most >> 23) > min(least, most) / (1u << 23) + kSpread;
      if (sw == 0 && lane == 0) {
        back_s[i & 1] = unscale_of(most);
        if (out) out_s[i & 1] = i + 1;
      }
      put_keys(kPart / 2);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(k_full);
#pragma unroll
      for (int r = 0; r < kPart / 2; ++r) load(kr[r], a.c.k, there, r);
      if (i > 0 && !wait(x_full(i - 1), (i - 1) >> 1)) break;
      if (out) {
#pragma unroll
        for (int r = 0; r < kPart; ++r)
#pragma unroll
          for (int k = 0; k < N; ++k) vr[r][k] = 0.f;
      }
      const float scale = scale_of(most);
#pragma unroll
      for (int r = 0; r < kPart; ++r) put_row<DIM>(v_s, row0 + r, vr[r], scale);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(v_full);
#pragma unroll
      for (int r = 0; r < kPart; ++r) load(vr[r], a.c.v, there, r);
      here = there;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // -------------------------------- softmax -------------------------------
    const uint32_t lanes = (uint32_t)(32 * warp) << 16;
    int i = 0;
    while (at < end && ok) {
      const Piece x = piece_of<kRows, PREFIX>(p, group, t, kvh, at, end);
      const int r = x.r0 + 32 * warp + lane;  // row of the sequence
      const int tok = min(r / group, x.s.n - 1), sees = x.s.pos + x.step * tok;
      const bool second = at != begin;
      next(x);
      const float factor = stage_rows<DIM>(a, x, group, x.r0, base_g + L::q);
      if (lane == 0) mbar_arrive(k_full);
      float o[DIM];
#pragma unroll
      for (int d = 0; d < DIM; ++d) o[d] = 0.f;
      float m = -INFINITY, l = 0.f, down = 1.f, back = 1.f;
      // the product of tile i - 1, which was weighed with `down` and `back`,
      // added to the row's outputs
      auto collect = [&](float down, float back) {
        if (!wait(x_full(i - 1), (i - 1) >> 1)) return;
        fence_after();
        tmem_each<DIM>(tmem + lanes + 256 + 128 * ((i - 1) & 1), [&](float (&v)[16], int c) {
#pragma unroll
          for (int k = 0; k < 16; ++k) o[c + k] = fmaf(v[k], back, o[c + k] * down);
        });
      };
      for (int j = 0; j < x.nt; ++j, ++i) {
        // (the second: this warp has part in that phase, and reads what came with it)
        if (!wait(s_full(i), i >> 1) || !wait(k_full, i)) break;
        fence_after();
        if (j + 1 < x.nt && lane == 0) mbar_arrive(k_full);  // the next tile's queries are there
        const uint32_t st = tmem + lanes + 128 * (i & 1);
        const int p0 = (x.j0 + j) * kTile;
        const float before_down = down, before_back = back;
        const bool out = uniform(out_s[i & 1]) == i + 1;
        back = back_s[i & 1];
        if (out) {
          if (j > 0) collect(before_down, before_back);
          constexpr float scale = (DIM == 128 ? 0.08838834764831845f : 0.125f) * kLog2e;
          const float* q = a.q + (int64_t)(x.s.row0 + tok) * a.q_stride + (int64_t)(x.kvh * group + r % group) * DIM;
#pragma unroll 1
          for (int pos = p0; pos < min(p0 + kTile, sees + 1); ++pos) {
            const int page = x.s.pages[pos / a.c.page_size];
            const bool in = page >= 0 && page < a.c.pages;  // (no page: zeros, as for the products)
            const int64_t row = (int64_t)(in ? page : 0) * a.c.page_stride + (int64_t)x.kvh * a.c.head_stride +
                                (int64_t)(pos % a.c.page_size) * a.c.row_stride;
            const float4* kf = reinterpret_cast<const float4*>(static_cast<const float*>(a.c.k) + row);
            const float4* vf = reinterpret_cast<const float4*>(static_cast<const float*>(a.c.v) + row);
            float s = 0.f;
#pragma unroll 4
            for (int d = 0; d < DIM / 4; ++d) {
              const float4 f = in ? kf[d] : make_float4(0.f, 0.f, 0.f, 0.f);
              s = fmaf(q[4 * d], f.x, fmaf(q[4 * d + 1], f.y, fmaf(q[4 * d + 2], f.z, fmaf(q[4 * d + 3], f.w, s))));
            }
            s *= scale;
            if (m == -INFINITY) {
              m = reference(s);
            } else if (s - m > kBias + kSlack) {
              const float f = ex2(m - reference(s));
              m = reference(s);
              l *= f;
#pragma unroll
              for (int d = 0; d < DIM; ++d) o[d] *= f;
            }
            const float w = s == -INFINITY ? 0.f : ex2(s - m);
            l += w;
#pragma unroll
            for (int d = 0; d < DIM / 4; ++d) {
              const float4 f = in ? vf[d] : make_float4(0.f, 0.f, 0.f, 0.f);
              o[4 * d] = fmaf(w, f.x, o[4 * d]);
              o[4 * d + 1] = fmaf(w, f.y, o[4 * d + 1]);
              o[4 * d + 2] = fmaf(w, f.z, o[4 * d + 2]);
              o[4 * d + 3] = fmaf(w, f.w, o[4 * d + 3]);
            }
          }
          __syncwarp();
          down = 1.f;
          const uint32_t zero[16] = {};
#pragma unroll 1
          for (int c = 0; c < kTile; c += 16) tmem_st(st + c, zero);
        } else {
          const float4* scale = reinterpret_cast<const float4*>(scale_s + (i & 1) * kTile);
          scores_to_weights(st, j == 0, j >= x.jm, sees - p0 + 1, factor, m, l, down, [&](float (&v)[32], int c) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 f = scale[c / 4 + k];
              v[4 * k] *= f.x, v[4 * k + 1] *= f.y, v[4 * k + 2] *= f.z, v[4 * k + 3] *= f.w;
            }
          });
        }
        tmem_wait_st();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(i));
        if (j > 0 && !out) collect(before_down, before_back);
      }
      if (ok) collect(down, back);
      if (!ok) break;
      store_rows<DIM, kRows, kF32>(p, x, group, cta, second, r, base_g + L::q, o, m, l, false);
    }
  }
  if (!ok) {
    if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_FULL);
    *abort_flag = 1;
  }
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <int DIM, bool PREFIX>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
  Params p;
  p.a = a;
  p.box = 0;
  char* ws = static_cast<char*>(a.ws) + mma_workspace_bytes(DIM);
  p.plan = plan_of<kRows>(a, ws);
  p.plan.least = 4;
  p.parts = reinterpret_cast<float*>(ws + kPlanBytes);
  auto k = chunk_tc32_kernel<DIM, PREFIX>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(k, Smem<DIM>::total, done);
  if (e == cudaSuccess) e = launch_plan<kRows, PREFIX>(a, p.plan, st);
  if (e == cudaSuccess) e = launch_next(k, dim3(kMaxCtas), dim3(kThreads), Smem<DIM>::total, st, p);
  if (e == cudaSuccess) e = launch_beside(a, kF32, st);
  if (e == cudaSuccess) e = launch_last<DIM, kRows, PREFIX, kF32>(p, st);
  return e;
}

}  // namespace

bool tc32_supported(const AttendArgs& a) { return plan_fits<kRows>(a); }

cudaError_t launch_chunks_tc32(const AttendArgs& a, cudaStream_t st) {
  if (a.groups.n) return a.c.dim == 128 ? launch<128, true>(a, st) : launch<64, true>(a, st);
  return a.c.dim == 128 ? launch<128, false>(a, st) : launch<64, false>(a, st);
}

}  // namespace paged
}  // namespace hyq
