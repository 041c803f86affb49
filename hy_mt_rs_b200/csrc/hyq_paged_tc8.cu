// Attention of chunks of new tokens over an 8-bit paged cache on tcgen05, head
// sizes 64 and 128, at f32 accuracy over the values that the codes stand for.
//
// The f16 kernel's line of segments, products and softmax (hyq_paged_tc.cu,
// hyq_paged_tc.cuh): a code is a whole f16 number (or 2^-8 of an e4m3 value), so the
// products are the same four, S = Qh K' + Ql K' and X = Ph V + Pl V.  K's scales
// multiply the columns of S.  V's go into the weights, as f16 pairs in the unit of
// the tile's largest scale; the running reference of a row counts that unit in
// (code_scores_to_weights()), so that tiles of any units may follow each other.
//
//   warp 1       tcgen05.mma, as in the f16 kernel;
//   warps 4-7    codes and scales from global memory (a tile's while the tensor
//                cores are at the one before), to f16 in a ring of three tiles of K
//                and V, in the layout that TMA gives the f16 kernel;
//   warps 8-11, 12-15   softmax of row tile 0 and 1, a thread per row.
//
// A tile whose scales of V are more than 2^10 apart, or not finite at a position of
// the sequence, is left out of the products (its weights are zeros there); each
// softmax thread then goes through the positions that its row sees, in f32, with its
// queries from global memory: 2.3 ms a tile, whatever the call (200 tokens at 500, int8,
// with one row of V 2^12 smaller than the others 38 us -> 2.3 ms; 2,048 at 8,192 0.79 ->
// 5.5 ms, with one in every fourth tile 77 ms).  Rows of zeros do not count.
//
// Bound by the turn of a ring's slot (codes to registers, decoded, four products,
// softmax): 2,048 tokens at 8,192, 32 query and 8 kv heads of 128, int8, 772 us, where
// the tensor cores take 368 for the split operands' four products at the rate of a
// library product (the f16 cache's kernel, whose tiles TMA brings as they are: 518).  Measured on the way: codes
// decoded from registers at the slot's turn 807 us, V's by asynchronous copies into
// their own tile 793, K's held in registers until their slot is free 768 (772 since the
// loaders carry their waits' results to their barrier); the products alone about 430.
#include "hyq_paged_tc.cuh"

namespace hyq {
namespace paged {
namespace {

constexpr int kCtaRows = 2 * kTile;      // rows of a segment
constexpr int kThreads = 512;
constexpr int kSpread = 10;              // of the exponents of a tile's scales of V

template <int DIM, bool PREFIX>
struct Smem {
  static constexpr int slots = PREFIX ? kPrefixSlots : 3;
  static constexpr int half = kTile * 128;               // 128 rows of 64 f16
  static constexpr int tile = half * (DIM / 64);         // K, V, or one half (hi or lo) of a Q tile
  static constexpr int q = 0;                            // [row tile][hi, lo]
  static constexpr int ring = (PREFIX ? 2 : 4) * tile;
  static constexpr int k_scale = ring + slots * tile;   // [2][128]: of tile i in i & 1
  static constexpr int v_scale = k_scale + 2 * kTile * 4;
  static constexpr int top = v_scale + 2 * kTile * 4;    // [2][4 warps] largest and smallest scale's bits
  static constexpr int bars = top + 2 * 4 * 8;
  // full[slots], empty[slots], s_full[2], p_full[2], x_full[2], q_full[2], scales[2], half[2]
  static constexpr int n_bars = 2 * slots + 12;
  // tensor memory address, abort, then [2] of: tile that is left out (its number +
  // 1), exponent of the tile's unit
  static constexpr int factors = bars + 8 * n_bars;      // (prefixes) powers of two of the rows' queries
  static constexpr int misc = factors + (PREFIX ? kTile * 4 : 0);
  static constexpr int total = misc + 32;
};

// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) { return (uint64_t)__float_as_uint(a) | (uint64_t)__float_as_uint(b) << 32; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t sub2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("sub.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ float low(uint64_t a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float high(uint64_t a) { return __uint_as_float((uint32_t)(a >> 32)); }

// scores_to_weights() over codes: the columns' scores are times ks[c], and the
// weights times vs[c], up to 1, V's scales in the tile's unit 2^lift.  A weight is
// 2^(s + lift - m) before that, and l the sum of 2^(s - m): the reference follows what
// the stored products can be at most, over all tiles, whatever their units.  So it may
// rise by the units alone, and what there is so far counts all the same: outputs and
// sum go down by 2^(before - m) however far that is.  (In f32 they reach zero 2^126
// further down: see the header on scales that far apart.)
__device__ __forceinline__ void code_scores_to_weights(uint32_t st, bool first, bool masked, int unseen_from, float factor, float& m,
                                                       float& l, float& down, const float* ks, const float* vs, float lift) {
  // the scores of columns c .. c + 31, and the largest
  auto scores = [&](uint64_t (&u)[16], int c) {
    float v[32];
    tmem_ld(v, st + c);
    const float4* k4 = reinterpret_cast<const float4*>(ks + c);
    float4 k[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = k4[i];
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[2 * i] = mul2(pair(v[4 * i], v[4 * i + 1]), pair(k[i & 3].x, k[i & 3].y));
      u[2 * i + 1] = mul2(pair(v[4 * i + 2], v[4 * i + 3]), pair(k[i & 3].z, k[i & 3].w));
      if (i < 4) k[i] = k4[i + 4];
    }
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        u[i] = pair(c + 2 * i >= unseen_from ? -INFINITY : low(u[i]), c + 2 * i + 1 >= unseen_from ? -INFINITY : high(u[i]));
    }
    float a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = fmaxf(low(u[i]), high(u[i]));
#pragma unroll
    for (int i = 4; i < 16; ++i) a[i & 3] = fmaxf(fmaxf(a[i & 3], low(u[i])), high(u[i]));
    return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
  };
  if (first) {
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < kTile; c += 32) {
      uint64_t u[16];
      top = fmaxf(top, scores(u, c));
    }
    m = reference(fmaf(top, factor, lift));
  }
  const uint64_t factors = pair(factor, factor);
  float back = (m == -INFINITY ? 0.f : -m) + lift;
  uint64_t sum = 0, sum2 = 0;
  down = 1.f;
#pragma unroll 1
  for (int c = 0; c < kTile; c += 32) {
    uint64_t u[16];
    const float top = fmaf(scores(u, c), factor, lift), over = top - m - kBias;
    if (__any_sync(0xffffffffu, over > kSlack)) {
      // raise the reference, by whole powers of two unless it is far (or the first
      // above -inf); what this tile has so far follows
      float f = 1.f;
      if (over > kSlack) {
        const float before = m;
        m = over > 64.f ? reference(top) : fmaxf(m + ceilf(over), reference(top));
        f = ex2(before - m);
      }
      back = (m == -INFINITY ? 0.f : -m) + lift;
      down *= f;
      sum = mul2(sum, pair(f, f));
      sum2 = mul2(sum2, pair(f, f));
      tmem_wait_st();
#pragma unroll 1
      for (int b = 0; b < c; b += 16) {
        float w[16];
        uint32_t x[16];
        tmem_ld(w, st + b);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t hi = __float_as_uint(w[i]), lo = __float_as_uint(w[8 + i]);
          const float2 a0 = __half22float2(*reinterpret_cast<const __half2*>(&hi));
          const float2 a1 = __half22float2(*reinterpret_cast<const __half2*>(&lo));
          const float y0 = (a0.x + a1.x) * f, y1 = (a0.y + a1.y) * f, h0 = high_part(y0), h1 = high_part(y1);
          x[i] = pack_f16(h0, h1);
          x[8 + i] = pack_f16(y0 - h0, y1 - h1);
        }
        tmem_st(st + b, x);
      }
    }
    const uint64_t backs = pair(back, back);
    const float4* v4 = reinterpret_cast<const float4*>(vs + c);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      float4 f4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f4[i] = v4[4 * g + i];
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint64_t e = fma2(u[8 * g + i], factors, backs);
        const uint64_t y = pair(ex2(low(e)), ex2(high(e)));
        if (i & 1) sum2 = add2(sum2, y);
        else sum = add2(sum, y);
        const float4 f = f4[i >> 1];
        const uint64_t z = mul2(y, i & 1 ? pair(f.z, f.w) : pair(f.x, f.y));
        const float h0 = high_part(low(z)), h1 = high_part(high(z));
        const uint64_t rest = sub2(z, pair(h0, h1));
        w[i] = pack_f16(h0, h1);
        w[8 + i] = pack_f16(low(rest), high(rest));
      }
      tmem_st(st + c + 16 * g, w);
    }
  }
  sum = add2(sum, sum2);
  l = fmaf(l, down, (low(sum) + high(sum)) * __uint_as_float((uint32_t)(127 - (int)lift) << 23));
}

// (the base is aligned to 1024 bytes by its declaration, and checked)
template <int DIM, Kv KV, bool PREFIX>
__global__ void __launch_bounds__(kThreads, 1) chunk_tc8_kernel(const __grid_constant__ Params p) {
  using L = Smem<DIM, PREFIX>;
  constexpr int kSlots = L::slots, ROWS = PREFIX ? kPrefixRows : kCtaRows;
  constexpr int KS = DIM / 16;            // steps of 16 along the head
  constexpr uint32_t kTmemCols = 512;
  const AttendArgs& a = p.a;
  extern __shared__ __align__(1024) uint8_t smem[];
  const uint32_t base = smem_addr(smem);
  auto full = [&](int s) { return base + L::bars + 8 * s; };
  auto empty = [&](int s) { return base + L::bars + 8 * (kSlots + s); };
  auto s_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + w); };
  auto p_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 2 + w); };
  auto x_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 4 + w); };
  auto q_full = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 6 + w); };
  auto half = [&](int w) { return base + L::bars + 8 * (2 * kSlots + 10 + w); };  // given, taken (split pieces)
  auto scales = [&](int i) { return base + L::bars + 8 * (2 * kSlots + 8 + (i & 1)); };  // of tile i: phase i / 2
  float* k_scale_s = reinterpret_cast<float*>(smem + L::k_scale);
  float* v_scale_s = reinterpret_cast<float*>(smem + L::v_scale);
  volatile int* misc = reinterpret_cast<volatile int*>(smem + L::misc);
  volatile int* abort_flag = misc + 1;
  volatile int* out_s = misc + 2;
  volatile int* lift_s = misc + 4;
  const int warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int group = a.heads / a.c.kv_heads;

  grid_dependency_wait();
  allow_dependents_launch();
  const int cta = blockIdx.x;
  const Start start = p.plan.start[cta];
  const int64_t begin = start.begin, end = p.plan.start[cta + 1].begin;
  if (begin == end) return;  // nothing allocated yet
  if (base & 1023u) {        // (the swizzled layouts need it)
    if (threadIdx.x == 0) atomicOr(a.c.status, DEV_BAD_ARGS);
    return;
  }
  if (warp == 0) {
    if (lane == 0) {
      misc[1] = 0;
      misc[2] = misc[3] = 0;
      for (int s = 0; s < kSlots; ++s) {
        mbar_init(full(s), 4);
        mbar_init(empty(s), 1);
      }
      for (int w = 0; w < 2; ++w) {
        mbar_init(s_full(w), 1);
        mbar_init(p_full(w), 4);
        mbar_init(x_full(w), 1);
        mbar_init(q_full(w), 4);
        mbar_init(scales(w), 4);
        mbar_init(half(w), 4);
      }
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

  // launch: 128 registers x 512 threads = (40 + 72 + 2 x 200) x 128
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == 1) {
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
      int slot = 0, phase = 0, operand = 0;
      auto advance = [&]() {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      int steps[2] = {0, 0}, pieces[2] = {0, 0}, issued = 0;
      bool ok = true;
      while (at < end && ok) {
        const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
        const int active = uniform(x.two ? 2 : 1), nt = uniform(x.nt);
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
            ++issued;
          };
          ok = wait(q_full(0), pieces[0] & 1);
          ++pieces[0];
          if (ok) scores_of(0);
          if (ok && nt > 1) scores_of(1);
          for (int j = 0; j < nt && ok; ++j) {
            const int n = first + 2 * j + 1, w = j & 1;
            ok = wait(full(n % kSlots), (n / kSlots) & 1);
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
            ++issued;
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
        if (ok) ++issued;
        advance();
        for (int j = 0; j < nt && ok; ++j) {
          const int v_slot = slot;
          ok = wait(full(slot), phase);
          advance();
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
          if (ok) issued += j + 1 < nt ? 2 : 1;
        }
        ++pieces[0];
        if (active == 2) ++pieces[1];
        next(x);
      }
      // no product's arrival may come after this CTA is gone
      for (int i = max(0, issued - kSlots); i < issued; ++i)
        if (!warp_wait(empty(i % kSlots), (i / kSlots) & 1, nullptr) && lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_DRAIN);
    }
  } else if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    // ------------------------------- K and V --------------------------------
    constexpr int LPR = DIM / 16;         // lanes of a row, 16 codes each
    constexpr int RPI = 32 / LPR, IT = LPR;
    const int lw = warp - 4, pos_in = threadIdx.x - 128;
    uint2* top_s = reinterpret_cast<uint2*>(smem + L::top);
    Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
    const int tiles = uniform((int)(end - begin));
    int j = 0, issued = 0, lift = 0;
    bool ok = true;
    // A lane's position is pos_in of the tile; its warp puts the 32 rows of its lanes.
    const int shift = p.box;
    auto entry = [&](int j) {  // of that position in its sequence's table row, -1: none
      const int pos = (x.j0 + j) * kTile + pos_in;
      return pos < x.len ? x.s.pages[shift >= 0 ? pos >> shift : pos / a.c.page_size] : -1;
    };
    int64_t here = -1;     // where the position's row begins, or -1
    float ks = 0.f, vs = 0.f;
    bool held = false;     // it is one of the sequence's
    int ahead = entry(0);  // the next tile's
    auto open = [&]() {
      const int pos = (x.j0 + j) * kTile + pos_in, in_page = shift >= 0 ? pos & ((1 << shift) - 1) : pos % a.c.page_size;
      const int page = pos < x.len ? checked_page(a.c, ahead) : -1;
      held = page >= 0;
      here = held ? (int64_t)page * a.c.page_stride + (int64_t)x.kvh * a.c.head_stride + (int64_t)in_page * a.c.row_stride : -1;
      const int64_t at_scale = held ? scale_at(a.c, page, x.kvh, in_page) : 0;
      ks = held ? a.c.k_scale[at_scale] : 0.f;
      vs = held ? a.c.v_scale[at_scale] : 0.f;
    };
    // A lane's 16 codes of each of the warp's rows become two 16-byte chunks of f16.  K's
    // wait in registers for their slot, which comes free half a tile before the tensor
    // cores want them; V's, which have a tile and a half, come to the place of one of
    // the chunks (`mine`), where the same lane takes them from.  (The other chunk's place
    // for half the lanes: they meet distinct banks.)
    const int c0 = 2 * (lane % LPR);
    const bool second = DIM == 128 && (c0 & 8);
    auto line = [&](int slot, int row) { return base + L::ring + slot * L::tile + (c0 >> 3) * L::half + row * 128; };
    auto mine = [&](int row) { return (((c0 & 7) | (second ? 1 : 0)) ^ (row & 7)) << 4; };
    auto row_of = [&](int i) { return 32 * lw + i * RPI + lane / LPR; };
    uint4 kr[IT];
    auto load_keys = [&]() {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int64_t o = __shfl_sync(0xffffffffu, here, i * RPI + lane / LPR);
        const uint8_t* row = static_cast<const uint8_t*>(a.c.k) + o + 16 * (lane % LPR);
        kr[i] = make_uint4(0, 0, 0, 0);
        // (predicated, not branched around: branches would keep the rows apart)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ge.s64 p, %4, 0;\n\t@p ld.global.v4.u32 {%0, %1, %2, %3}, [%5];\n\t}"
                     : "+r"(kr[i].x), "+r"(kr[i].y), "+r"(kr[i].z), "+r"(kr[i].w)
                     : "l"(o), "l"(row));
      }
    };
    // A warp whose wait ran out does nothing more, raises the abort flag, which ends the
    // others' waits, and goes on to the next tile's barrier, where all four leave: none
    // may be left waiting there for it.
    auto waited = [&](uint32_t bar, uint32_t parity) {
      if (ok && !warp_wait(bar, parity, abort_flag)) {
        ok = false;
        *abort_flag = 1;
      }
    };
    auto take = [&]() {  // the ring's next slot
      const int slot = issued % kSlots;
      if (issued >= kSlots) waited(empty(slot), ((issued / kSlots) - 1) & 1);
      ++issued;
      return slot;
    };
    auto ask_values = [&](int slot) {
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int64_t o = __shfl_sync(0xffffffffu, here, i * RPI + lane / LPR);
        const uint8_t* row = static_cast<const uint8_t*>(a.c.v) + max(o, (int64_t)0) + 16 * (lane % LPR);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(line(slot, row_of(i)) + mine(row_of(i))), "l"(row),
                     "r"(o >= 0 ? 16 : 0)
                     : "memory");
      }
    };
    // 16 codes of row_of(i) to f16
    auto put = [&](int slot, int i, uint32_t x, uint32_t y, uint32_t z, uint32_t u) {
      const uint32_t to = line(slot, row_of(i)), at = mine(row_of(i));
      const uint32_t in[4] = {x, y, z, u};
      uint32_t w[8];
#pragma unroll
      for (int k = 0; k < 4; ++k) decode4<KV>(__byte_perm(in[k], 0, 0x3120), w[2 * k], w[2 * k + 1]);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const bool hi = (k == 0) == second;
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + (k == 0 ? at : at ^ 16)), "r"(hi ? w[4] : w[0]),
                     "r"(hi ? w[5] : w[1]), "r"(hi ? w[6] : w[2]), "r"(hi ? w[7] : w[3])
                     : "memory");
      }
    };
    open();
    load_keys();
    ahead = entry(1);
#pragma unroll 1
    for (int i = 0; i < tiles; ++i) {
      const uint32_t bits = __float_as_uint(vs) & 0x7fffffffu;
      const bool usable = bits - 1u < 0x7f7fffffu;  // finite and not zero
      const uint32_t most = __reduce_max_sync(0xffffffffu, usable ? bits : 0u),
                     least = __reduce_min_sync(0xffffffffu, usable ? bits : 0x7f800000u);
      const bool bad = __any_sync(0xffffffffu, held && !isfinite(vs));
      if (lane == 0) top_s[(i & 1) * 4 + lw] = make_uint2(most, bad ? 0u : least);
      const int k_slot = take();
      // (V of tile i - 2 was there, whose products followed that tile's softmax)
      if (ok) {
#pragma unroll
        for (int r = 0; r < IT; ++r) put(k_slot, r, kr[r].x, kr[r].y, kr[r].z, kr[r].w);
        fence_proxy_async_smem();
      }
      ok = bar_red_and(1, 128, ok);
      if (!ok) break;
      uint32_t top = 0, low = 0x7f800000u;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint2 o = top_s[(i & 1) * 4 + w];
        top = max(top, o.x);
        low = min(low, o.y);
      }
      int v_slot = 0;
      auto ask = [&]() {
        v_slot = take();
        if (!ok) return;
        ask_values(v_slot);
        asm volatile("cp.async.commit_group;" ::: "memory");
      };
      if constexpr (PREFIX) {
        // (here the ring alone does not say that the softmax of tile i - 2, whose scales
        // these replace, is done: its V's products do)
        ask();
        if (i >= 2) waited(empty((2 * i - 3) % kSlots), ((2 * i - 3) / kSlots) & 1);
        if (!ok) continue;
      }
      // the unit: above the largest scale (a tile of zeros keeps the one before, and the
      // first of a piece takes 2^-60, as the few-token kernel's rows of zeros do: small
      // values behind it keep their bits, whatever the piece before this one held)
      if (top) lift = min(max((int)(top >> 23) - 126, -100), 100);
      else if (j == 0) lift = -60;
      const float unit = code_unit<KV>(), down = __uint_as_float((uint32_t)(127 - lift) << 23);
      k_scale_s[(i & 1) * kTile + pos_in] = ks * unit;
      v_scale_s[(i & 1) * kTile + pos_in] = isfinite(vs) ? vs * down : 0.f;
      if (pos_in == 0) {
        lift_s[i & 1] = lift;
        out_s[i & 1] = low == 0u || (top && (top >> 23) > (low >> 23) + kSpread) ? i + 1 : 0;
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(scales(i));
        mbar_arrive(full(k_slot));
      }
      if constexpr (!PREFIX) {
        ask();
        if (!ok) continue;
      }
      if (i + 1 < tiles) {
        if (++j == x.nt) {
          next(x);
          x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
          j = 0;
          ahead = entry(0);
        }
        open();
        load_keys();
        ahead = entry(j + 1);
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
      for (int r = 0; r < IT; ++r) {
        uint32_t in[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(in[0]), "=r"(in[1]), "=r"(in[2]), "=r"(in[3])
                     : "r"(line(v_slot, row_of(r)) + mine(row_of(r)))
                     : "memory");
        put(v_slot, r, in[0], in[1], in[2], in[3]);
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(full(v_slot));
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!ok) {
      if (lane == 0) atomicOr(a.c.status, DEV_TIMEOUT_EMPTY);
      *abort_flag = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    // -------------------------------- softmax -------------------------------
    const int wg = warp >= 12 ? 1 : 0;  // row tile
    const uint32_t st = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 256 * wg;
    int steps = 0, tiles = 0, splits = 0;  // this row tile's steps, all tiles of the pieces before
    bool ok = true;
    while (at < end && ok) {
      const Piece x = piece_of<ROWS, PREFIX>(p, group, t, kvh, at, end);
      const int r0 = x.r0 + (PREFIX ? 0 : wg * kTile), r = r0 + 32 * (warp & 3) + lane;  // row of the sequence
      const int tok = min(r / group, x.s.n - 1), sees = x.s.pos + x.step * tok;
      const int64_t piece_at = at;
      next(x);
      const int tile0 = tiles;
      tiles += x.nt;
      if (!PREFIX && wg == 1 && !x.two) continue;
      float factor;
      float* factor_s = reinterpret_cast<float*>(smem + L::factors) + 32 * (warp & 3) + lane;
      uint8_t* q_s = smem + L::q + (PREFIX ? 0 : wg) * 2 * L::tile;
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
        const int tile = tile0 + j;
        // (while the tensor cores are at this tile's scores, which follow its scales:
        // the wait for those skips no phase)
        ok = (j == j0 || collect(steps - 1)) && warp_wait(s_full(wg), steps & 1, abort_flag) &&
             warp_wait(scales(tile), (tile >> 1) & 1, abort_flag);
        if (!ok) break;
        fence_after();
        const int p0 = (x.j0 + j) * kTile;
        const float* ks = k_scale_s + (tile & 1) * kTile;
        if (uniform(out_s[tile & 1]) == tile + 1) {
          // in f32, each position in the unit of its own scale
          constexpr float scale = (DIM == 128 ? 0.08838834764831845f : 0.125f) * kLog2e;
          const float* q = a.q + (int64_t)(x.s.row0 + tok) * a.q_stride + (int64_t)(x.kvh * group + r % group) * DIM;
          const float lift = (float)lift_s[tile & 1];
#pragma unroll 1
          for (int pos = p0; pos < min(p0 + kTile, sees + 1); ++pos) {
            const int page = x.s.pages[pos / a.c.page_size], in_page = pos % a.c.page_size;
            const bool in = page >= 0 && page < a.c.pages;  // (no page: zeros, as for the products)
            const int64_t row = (int64_t)(in ? page : 0) * a.c.page_stride + (int64_t)x.kvh * a.c.head_stride +
                                (int64_t)in_page * a.c.row_stride;
            const uint32_t* kc = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.k) + row);
            const uint32_t* vc = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.c.v) + row);
            const float v_unit = in ? a.c.v_scale[scale_at(a.c, page, x.kvh, in_page)] : 0.f;
            float s = 0.f;
#pragma unroll 4
            for (int d = 0; d < DIM / 4; ++d) {
              const uint32_t w = in ? kc[d] : 0u;
#pragma unroll
              for (int i = 0; i < 4; ++i) s = fmaf(q[4 * d + i], code_value<KV>((uint8_t)(w >> (8 * i))), s);
            }
            s *= scale * (ks[pos - p0] / code_unit<KV>());
            const bool usable = v_unit != 0.f && isfinite(v_unit);
            const float own = usable ? fminf(fmaxf((float)((int)(__float_as_uint(v_unit) >> 23 & 0xffu) - 126), -100.f), 100.f) : lift;
            const float u = s + own, back = __uint_as_float((uint32_t)(127 - (int)own) << 23);
            if (m == -INFINITY) {
              m = reference(u);
            } else if (u - m > kBias + kSlack) {
              const float f = ex2(m - reference(u));
              m = reference(u);
              l *= f;
#pragma unroll
              for (int d = 0; d < DIM; ++d) o[d] *= f;
            }
            const float w = u == -INFINITY ? 0.f : ex2(u - m);
            l = fmaf(w, back, l);
            const float wv = w * (v_unit * back);
#pragma unroll
            for (int d = 0; d < DIM / 4; ++d) {
              const uint32_t c = in ? vc[d] : 0u;
#pragma unroll
              for (int i = 0; i < 4; ++i) o[4 * d + i] = fmaf(wv, code_value<KV>((uint8_t)(c >> (8 * i))) / code_unit<KV>(), o[4 * d + i]);
            }
          }
          __syncwarp();
          down = 1.f;
          const uint32_t zero[16] = {};
#pragma unroll 1
          for (int c = 0; c < kTile; c += 16) tmem_st(st + c, zero);
        } else {
          code_scores_to_weights(st, j == j0, j >= x.jm, sees - p0 + 1, factor, m, l, down, ks, v_scale_s + (tile & 1) * kTile,
                                 (float)lift_s[tile & 1]);
        }
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
      if constexpr (KV == kF8) {
#pragma unroll
        for (int d = 0; d < DIM; ++d) o[d] *= code_unit<KV>();
      }
      store_rows<DIM, ROWS, KV>(p, x, group, cta, piece_at != begin, r, q_s, o, m, l, false);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
  }
}

template <int DIM, Kv KV, bool PREFIX>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
  constexpr int ROWS = PREFIX ? kPrefixRows : kCtaRows;
  Params p;
  p.a = a;
  p.box = (a.c.page_size & (a.c.page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.c.page_size) : -1;
  char* ws = static_cast<char*>(a.ws) + mma_workspace_bytes(DIM);
  p.plan = plan_of<ROWS>(a, ws);
  p.plan.least = 8;
  p.parts = reinterpret_cast<float*>(ws + kPlanBytes);
  auto k = chunk_tc8_kernel<DIM, KV, PREFIX>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(k, Smem<DIM, PREFIX>::total, done);
  if (e == cudaSuccess) e = launch_plan<ROWS, PREFIX>(a, p.plan, st);
  if (e == cudaSuccess) e = launch_next(k, dim3(kMaxCtas), dim3(kThreads), Smem<DIM, PREFIX>::total, st, p);
  if (e == cudaSuccess) e = launch_beside(a, KV, st);
  if (e == cudaSuccess) e = launch_last<DIM, ROWS, PREFIX, KV>(p, st);
  return e;
}

template <Kv KV>
cudaError_t launch(const AttendArgs& a, cudaStream_t st) {
  if (a.groups.n) return a.c.dim == 128 ? launch<128, KV, true>(a, st) : launch<64, KV, true>(a, st);
  return a.c.dim == 128 ? launch<128, KV, false>(a, st) : launch<64, KV, false>(a, st);
}

}  // namespace

bool tc8_supported(const AttendArgs& a) { return a.groups.n ? plan_fits<kPrefixRows>(a) : plan_fits<kCtaRows>(a); }

cudaError_t launch_chunks_tc8(const AttendArgs& a, Kv kv, cudaStream_t st) { return kv == kI8 ? launch<kI8>(a, st) : launch<kF8>(a, st); }

}  // namespace paged
}  // namespace hyq
