// Attention on the 5th-generation tensor cores: causal packed prompts, and
// drafted trees over a paged cache.
//
// A tile of 128 query rows (prompt: 128 tokens of one head; tree: the (node,
// head) rows of one kv head) walks its slots in tiles of 128:
//   S = Q K^T (128 x 128, fp32 in tensor memory), p = exp2(c S - m), O += P V
// with c = scale log2 e and P back in tensor memory as the A operand, over the
// first half of its S.  The reference m of a row moves only when its maximum
// passes it by 2^8 (sums and O are rescaled then); p stays below 2^8, in f16
// multiplied by 2^7 so that small weights keep their bits, and both factors
// cancel in O / sum p.
//
// Roles: warps 0-3 and 4-7 take the softmax of alternate tiles, one row per
// thread; warp 8 issues the MMAs (two S tiles in flight, so the tensor cores
// work on one while the other's softmax runs); warp 9 (prompt: TMA tensor maps)
// or warps 9-12 (tree, and prompts whose rows TMA cannot address) fill a ring of
// 16 KB pieces in the order in which the MMAs use them: K as 128 slots x 64
// dims, V as 8192/HD slots x HD dims, both with 128-byte swizzle.
//
// f32 rows are split in two f16 parts, x 2^e = hi + lo to 2^-22 of x, and every
// product is hi hi + lo hi + hi lo (lo lo is below 2^-22 of it): three f16 MMAs
// for one.  e is exact per row of Q; for K and V it comes from the largest
// value of a window's first piece, with 2^7 to spare above it: what passes that
// becomes infinite and goes the way of the last paragraph, what is small keeps
// 2^-33 of that largest value.  The tensor cores add with truncation, which drifts
// by up to 2^-24 of O per step of 16 slots, so O is taken out every WIN tiles and
// added up in fp32 in the output (or part) rows.
//
// Rows that come out non-finite, and tiles that met a bad page id, are done
// again by exact_row: a masked place must not reach a row even as 0 x NaN.
#include <cuda.h>
#include <string.h>

#include <type_traits>

#include "attn_tc.cuh"

namespace cw {

namespace {

constexpr int PIECE = 16384;
constexpr int TMA_WARPS = 3;
constexpr float P_SHIFT_F16 = 7.f;  // p <= 2^(8+7) < 65504
constexpr float RESCALE_AT = 8.f;

enum { TY_F32, TY_F16, TY_BF16 };
template <int TY> struct TypeOf;
template <> struct TypeOf<TY_F32> { using T = float; };
template <> struct TypeOf<TY_F16> { using T = __half; };
template <> struct TypeOf<TY_BF16> { using T = __nv_bfloat16; };

template <int TY, int HD>
struct Geo {
  static constexpr bool F32 = TY == TY_F32;
  static constexpr int CB = HD / 64;         // 64-dim blocks of a row
  static constexpr int Q_BYTES = CB * 16384; // [block][128 rows][128 B]; f32: hi, then lo
  static constexpr int NP = CB;              // pieces of a K or a V tile (f32: pairs of pieces)
  static constexpr int VK = 8192 / HD;       // slots of a V piece
  static constexpr int NS = F32 ? (HD == 256 ? 5 : HD == 128 ? 9 : 11) : (HD == 256 ? 9 : HD == 128 ? 11 : 12);
  static constexpr int SMEM = Q_BYTES * (F32 ? 2 : 1) + NS * PIECE + 1024;
  static constexpr int LOADERS = F32 ? 256 : 128;
  static constexpr int threads(bool tma) { return 288 + (tma ? 32 * TMA_WARPS : LOADERS); }
};
constexpr int WIN = 4;  // f32: tiles of a window

struct Ctl {
  uint64_t full[12], empty[12], s_full[2], p_ready[2], pv_done, q_full, o_free, o_done, drained;
  int64_t u0, u1;
  uint32_t tmem;
  volatile int abort, bad;
  int s0, tile0, begin, end;
  int64_t rem;
  unsigned badrows[4];
  float mref[TC_ROWS];
  float2 ml[2][TC_ROWS];
  uint32_t rowoff[2][TC_KEYS];
  // f32: exponents that Q rows, and a window's K and V, were multiplied by (the loaders run up to three windows ahead)
  int qe[TC_ROWS], ke[8], ve[8];
  float amax[8];
};

// Where one segment of work lies: the tiles [w0, w1) of a row tile's nt, and
// the window [t0, t1) of them at hand.
struct Seg {
  int s, hk, mt, t0, t1, nt, w0, w1;
  TreeSeq ts;
};

CW_HOST_DEV int tree_tiles(int n) { return (n + TC_KEYS - 1) / TC_KEYS; }
CW_DEV int64_t seq_units(const AttnOp &a, int s) {
  const TreeSeq q = tree_seq(a, s);
  const int G = a.nh / a.nkv;
  return q.live ? (int64_t)a.nkv * ((q.live * G + TC_ROWS - 1) / TC_ROWS) * tree_tiles(q.n) : 0;
}
CW_DEV int64_t warp_scan(int64_t v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Walks a CTA's share of the units, segment by segment; every role does it for
// itself, from the same start.
struct TreeWalk {
  int s, hk, mt, t0;
  int64_t left;
  CW_DEV void start(const AttnOp &a, const Ctl &c) {
    s = c.s0;
    left = c.u1 - c.u0;
    const TreeSeq q = tree_seq(a, s);
    const int G = a.nh / a.nkv, nt = tree_tiles(q.n), mts = (q.live * G + TC_ROWS - 1) / TC_ROWS;
    const int64_t i = c.rem / nt;
    t0 = (int)(c.rem - i * nt);
    mt = (int)(i % mts);
    hk = (int)(i / mts);
  }
  CW_DEV bool next(const AttnOp &a, Seg &g) {
    if (left <= 0) return false;
    const int G = a.nh / a.nkv;
    g.ts = tree_seq(a, s);
    while (g.ts.live == 0) g.ts = tree_seq(a, ++s);
    g.nt = tree_tiles(g.ts.n);
    g.s = s;
    g.hk = hk;
    g.mt = mt;
    g.t0 = t0;
    g.t1 = (int)min((int64_t)g.nt, t0 + left);
    left -= g.t1 - g.t0;
    t0 = 0;
    if (g.t1 == g.nt && ++mt * TC_ROWS >= g.ts.live * G) {
      mt = 0;
      if (++hk == a.nkv) {
        hk = 0;
        s++;
      }
    }
    return true;
  }
};

// 2^e, e cut to the normal floats.
CW_DEV float exp2_int(int e) { return __int_as_float((min(max(e, -126), 127) + 127) << 23); }
// The exponent that brings a largest value into [2^8, 2^9); 0 for zeros and non-finite ones.
CW_DEV int scale_exp(float amax) {
  if (!(amax > 1e-30f) || !(amax < INFINITY)) return 0;
  return 8 - ((__float_as_int(amax) >> 23) - 127);
}
// Two floats as f16 hi and lo parts.
CW_DEV void split2(float x, float y, uint32_t &hi, uint32_t &lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
  hi = *(const uint32_t *)&h;
  lo = *(const uint32_t *)&l;
}

CW_DEV uint32_t pack2(bool bf, float lo, float hi) {
  uint32_t r;
  if (bf) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Maximum of 32 scores over the slots of w.
CW_DEV float max32(const uint32_t (&x)[32], uint32_t w, float mx) {
  float m0 = mx, m1 = -INFINITY, m2 = -INFINITY, m3 = -INFINITY;
  if (w == ~0u) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      m0 = fmaxf(m0, fmaxf(__uint_as_float(x[i]), __uint_as_float(x[i + 1])));
      m1 = fmaxf(m1, fmaxf(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])));
      m2 = fmaxf(m2, fmaxf(__uint_as_float(x[i + 4]), __uint_as_float(x[i + 5])));
      m3 = fmaxf(m3, fmaxf(__uint_as_float(x[i + 6]), __uint_as_float(x[i + 7])));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 32; i++) m0 = (w >> i) & 1 ? fmaxf(m0, __uint_as_float(x[i])) : m0;
  }
  return fmaxf(fmaxf(m0, m1), fmaxf(m2, m3));
}
// p = exp2(c s - m) of 32 scores, 0 outside w: as pairs of 16 bits (f32: hi and lo parts), and added to sum.
template <bool F32, bool BF>
CW_DEV void exp32(const uint32_t (&x)[32], uint32_t w, float sc, float mm, uint64_t &sum, uint32_t (&p)[16],
                  uint32_t (&q)[F32 ? 16 : 1]) {
  const uint64_t c2 = pack_f2(sc, sc), m2 = pack_f2(-mm, -mm);
#pragma unroll
  for (int i = 0; i < 32; i += 2) {
    float a, b;
    unpack_f2(fma_f2(pack_f2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), c2, m2), a, b);
    a = ex2(a);
    b = ex2(b);
    if (w != ~0u) {
      a = (w >> i) & 1 ? a : 0.f;
      b = (w >> (i + 1)) & 1 ? b : 0.f;
    }
    sum = add_f2(sum, pack_f2(a, b));
    if constexpr (F32) split2(a, b, p[i >> 1], q[i >> 1]);
    else p[i >> 1] = pack2(BF, a, b);
  }
}

// 32 slots from `base` that a tree row sees.
CW_DEV uint32_t tree_word(const TreeSeq &q, uint64_t bits, int base) {
  const int d = q.len - base;  // committed slots of the word
  if (d >= 32) return ~0u;
  uint32_t w = d > 0 ? (1u << d) - 1 : 0u;
  if (d >= 0) w |= (uint32_t)(bits << d);
  else if (d > -64) w |= (uint32_t)(bits >> -d);
  return w;
}

}  // namespace

template <int TY, int HD, bool TREE, bool TMA>
__global__ void __launch_bounds__(Geo<TY, HD>::threads(TMA), 1)
    attn_tc_kernel(const __grid_constant__ AttnOp a, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv) {
  using G_ = Geo<TY, HD>;
  using T = typename TypeOf<TY>::T;
  constexpr bool F32 = TY == TY_F32, BF = TY == TY_BF16;
  constexpr int LD = G_::LOADERS;
  constexpr int CB = G_::CB, NP = G_::NP, VK = G_::VK, NS = G_::NS;
  constexpr int O_COL = 0, S_COL = 256;
  __shared__ Ctl c;
  extern __shared__ uint8_t dyn[];
  uint8_t *qs = (uint8_t *)(((uintptr_t)dyn + 1023) & ~(uintptr_t)1023);
  uint8_t *ring = qs + G_::Q_BYTES * (F32 ? 2 : 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.nh / a.nkv;

  pdl_trigger();
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&c.full[i], TMA ? 1 : LD);
      mbar_init(&c.empty[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&c.s_full[i], 1);
      mbar_init(&c.p_ready[i], 128);
    }
    mbar_init(&c.pv_done, 1);
    mbar_init(&c.q_full, 256);
    mbar_init(&c.o_free, 256);
    mbar_init(&c.o_done, 1);
    mbar_init(&c.drained, 1);
    mbar_fence_init();
    c.abort = 0;
    c.bad = 0;
  }
  if (tid < 4) c.badrows[tid] = 0;
  pdl_wait();
  if (warp == 0) {  // this CTA's work
    const int ch = (a.n_seq + 31) / 32, i0 = min(a.n_seq, lane * ch), i1 = min(a.n_seq, i0 + ch);
    int64_t mine = 0;
    for (int i = i0; i < i1; i++) {
      if constexpr (TREE) {
        mine += seq_units(a, i);
      } else {
        int b, e;
        prompt_seq(a, i, b, e);
        mine += (e - b + TC_ROWS - 1) / TC_ROWS;
      }
    }
    const int64_t incl = warp_scan(mine), total = __shfl_sync(0xffffffffu, incl, 31);
    int64_t u0, u1;
    if constexpr (TREE) {
      u0 = total * blockIdx.x / gridDim.x;
      u1 = total * (blockIdx.x + 1) / gridDim.x;
    } else {  // the tiles with most slots first
      u0 = total - 1 - blockIdx.x / a.nh;
      u1 = u0 < 0 ? u0 : u0 + 1;
    }
    if (lane == 0) {
      c.u0 = u0;
      c.u1 = u1;
    }
    int64_t at = incl - mine;
    if (u0 >= at && u0 < incl) {
      for (int i = i0; i < i1; i++) {
        int64_t n;
        int b = 0, e = 0;
        if constexpr (TREE) {
          n = seq_units(a, i);
        } else {
          prompt_seq(a, i, b, e);
          n = (e - b + TC_ROWS - 1) / TC_ROWS;
        }
        if (u0 < at + n) {
          c.s0 = i;
          c.rem = u0 - at;
          c.begin = b;
          c.end = e;
          c.tile0 = (int)(u0 - at);
          break;
        }
        at += n;
      }
    }
  }
  __syncthreads();
  if (c.u0 >= c.u1) return;
  if (warp == 0) tmem_alloc(&c.tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = c.tmem;

  auto wait = [&](uint64_t *bar, uint32_t parity) {
    if (!mbar_wait(bar, parity, &c.abort)) {
      if (!c.abort) atomicOr(a.err, OPE_WAIT);
      c.abort = 1;
    }
  };
  // prompt: one segment
  const int ph = TREE ? 0 : (int)(blockIdx.x % a.nh), pbegin = c.begin, pend = c.end, ptile = c.tile0;
  TreeWalk walk;
  if constexpr (TREE) walk.start(a, c);
  bool once = true;
  int w_at = 0, w_end = 0;  // f32: what is left of the segment
  auto next = [&](Seg &g) -> bool {
    if (F32 && w_at < w_end) {
      g.t0 = w_at;
    } else {
      if constexpr (TREE) {
        if (!walk.next(a, g)) return false;
      } else {
        if (!once) return false;
        once = false;
        g.s = 0;
        g.hk = ph / G;
        g.mt = ptile;
        g.t0 = 0;
        g.t1 = g.nt = ptile + 1;
      }
      g.w0 = g.t0;
      g.w1 = w_end = g.t1;
    }
    if (F32) {
      g.t1 = min(g.w1, g.t0 + WIN);
      w_at = g.t1;
    }
    return true;
  };

  if (warp < 8) {
    // ------------------------------------------------------------ softmax
    const int wg = warp >> 2, r = tid & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    float sc = fabsf(a.scale) * 1.4426950408889634f;
    constexpr float SHIFT = BF ? 0.f : P_SHIFT_F16;
    constexpr int AL = 16 / sizeof(T);
    const bool qvec = (F32 || a.scale >= 0.f) && ((uintptr_t)a.q % 16) == 0 && a.qrow % AL == 0 && a.qhead % AL == 0;
    const bool ovec = ((uintptr_t)a.o % 16) == 0 && a.orow % AL == 0 && a.ohead % AL == 0;
    float m_acc = -INFINITY, l_acc = 0.f;  // f32: of the windows so far
    int gt = 0;  // tiles of the CTA so far
    Seg g;
    for (int si = 0; next(g); si++) {
      // rows of the tile: where they lie, and whether they are there
      auto place = [&](int i, int64_t &row, int &h, int &t) -> bool {
        if constexpr (TREE) {
          const int item = g.mt * TC_ROWS + i;
          t = item / G;
          h = g.hk * G + item - t * G;
          row = (int64_t)g.s * a.T + t;
          return item < g.ts.live * G;
        } else {
          t = 0;
          h = ph;
          row = (int64_t)pbegin + g.mt * TC_ROWS + i;
          return row < pend;
        }
      };
      const bool first = g.t0 == g.w0, last = g.t1 == g.w1;  // window of the segment
      if (first) {
      for (int i = tid; i < 128 * CB * 8; i += 256) {
        const int rr = i / (CB * 8), u = i % (CB * 8);
        int64_t row;
        int h, t;
        const bool have = place(rr, row, h, t);
        uint8_t *dst = qs + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4);
        const T *src = (const T *)a.q + (have ? row * a.qrow + h * a.qhead + u * 8 : 0);
        if constexpr (F32) {
          float x[8];
          if (qvec && have) {
            *(float4 *)x = *(const float4 *)src;
            *(float4 *)(x + 4) = *(const float4 *)(src + 4);
          } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = have ? src[k] : 0.f;
          }
          float mx = 0.f;
#pragma unroll
          for (int k = 0; k < 8; k++) mx = fmaxf(mx, fabsf(x[k]));
#pragma unroll
          for (int k = 1; k < CB * 8; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
          const int e = scale_exp(mx);
          const float f = a.scale < 0.f ? -exp2_int(e) : exp2_int(e);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; k++) split2(x[2 * k] * f, x[2 * k + 1] * f, hi[k], lo[k]);
          *(uint4 *)dst = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *(uint4 *)(dst + G_::Q_BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          if (u == 0) c.qe[rr] = e;
        } else if (qvec) {
          cp_async16(smem_u32(dst), src, have);
        } else {
          T e[8];
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const float x = have ? to_f<T>(src[k]) : 0.f;
            e[k] = from_f<T>(a.scale < 0.f ? -x : x);  // exact: |scale| is used below
          }
          *(uint4 *)dst = *(uint4 *)e;
        }
      }
      }
      int64_t row;
      int h, t;
      const bool have = place(r, row, h, t);
      uint64_t bits = 0;
      if constexpr (TREE)
        if (have) bits = tree_bits(a, g.ts, g.s, t);
      const bool warp_live = __any_sync(0xffffffffu, have);
      if (first) {
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        if (F32) named_bar(3, 256);  // qe
        mbar_arrive(&c.q_full);
      }

      const int nt = g.t1 - g.t0;
      float m_own = -INFINITY, l_own = 0.f;
      for (int j = 0; j < nt; j++) {
        const int gi = gt + j;
        if ((gi & 1) != wg) continue;
        const uint32_t S = tm + lane_base + S_COL + 128 * wg;
        wait(&c.s_full[wg], (gi >> 1) & 1);
        tc_fence_after();
        if (F32) sc = fabsf(a.scale) * 1.4426950408889634f * exp2_int(-c.qe[r]) * exp2_int(-c.ke[si & 7]);
        const int tile = g.t0 + j;
        const bool masked = TREE ? (tile + 1) * TC_KEYS > g.ts.len : tile == g.mt;
        auto word = [&](int k) -> uint32_t {
          if (!masked) return ~0u;
          if constexpr (TREE) return tree_word(g.ts, bits, tile * TC_KEYS + 32 * k);
          const int d = r - 32 * k;  // columns 0..r
          return d >= 31 ? ~0u : (d < 0 ? 0u : (2u << d) - 1);
        };
        float mx = -INFINITY;
        if (warp_live) {
          // the next 32 columns are on their way while these are looked at (f32 has no registers for that)
          uint32_t x[F32 ? 1 : 2][32];
          if (!F32) tmem_ld32(S, x[0]);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            uint32_t(&y)[32] = x[F32 ? 0 : k & 1];
            if (F32) tmem_ld32(S + 32 * k, y);
            tmem_wait_ld();
            if (!F32 && k < 3) tmem_ld32(S + 32 * (k + 1), x[F32 ? 0 : (k + 1) & 1]);
            mx = max32(y, word(k), mx);
          }
          if (mx != -INFINITY) mx *= sc;
        }
        // the reference from the tile before, ours to the tile after
        if (j > 0) named_bar(1 + wg, 256);
        const float m_old = j > 0 ? c.mref[r] : -INFINITY;
        const bool move = mx > m_old + RESCALE_AT || (m_old == -INFINITY && mx > m_old);
        const float m = move ? mx : m_old;
        c.mref[r] = m;
        if (j + 1 < nt) named_bar_arrive(1 + (wg ^ 1), 256);
        if (j > 0 && __any_sync(0xffffffffu, move)) {
          // O holds the tiles before (S of this tile came after the PV two tiles ago: one phase open at most)
          wait(&c.pv_done, (gi - 1) & 1);
          tc_fence_after();
          const float f = move ? (m_old == -INFINITY ? 0.f : ex2(m_old - m)) : 1.f;
#pragma unroll 1
          for (int k = 0; k < HD / 32; k++) {
            uint32_t x[32];
            tmem_ld32(tm + lane_base + O_COL + 32 * k, x);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; i++) x[i] = __float_as_uint(__uint_as_float(x[i]) * f);
            tmem_st32(tm + lane_base + O_COL + 32 * k, x);
          }
        }
        if (warp_live) {
          l_own = m_own == -INFINITY ? 0.f : l_own * ex2(m_own - m);
          m_own = m;
          const float mm = (m == -INFINITY ? 0.f : m) - SHIFT;
          uint64_t sum = 0;
          uint32_t x[F32 ? 1 : 2][32];
          if (!F32) tmem_ld32(S, x[0]);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            uint32_t(&y)[32] = x[F32 ? 0 : k & 1];
            uint32_t p[16], q[F32 ? 16 : 1];
            if (F32) tmem_ld32(S + 32 * k, y);
            tmem_wait_ld();
            if (!F32 && k < 3) tmem_ld32(S + 32 * (k + 1), x[F32 ? 0 : (k + 1) & 1]);
            const uint32_t w = word(k);
            if (w == ~0u) exp32<F32, BF>(y, ~0u, sc, mm, sum, p, q);
            else exp32<F32, BF>(y, w, sc, mm, sum, p, q);
            // P over S columns already read: 16 slots in 8 columns, f32 with 32 slots' lo parts behind their hi parts
            tmem_st16(S + (F32 ? 32 : 16) * k, p);
            if constexpr (F32) tmem_st16(S + 32 * k + 16, q);
          }
          float s0, s1;
          unpack_f2(sum, s0, s1);
          l_own += s0 + s1;
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&c.p_ready[wg]);
      }
      // ---------------------------------------------------------- epilogue
      c.ml[wg][r] = make_float2(m_own, l_own);
      named_bar(3, 256);
      const float m = c.mref[r];
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < 2; w++) {
        const float2 x = c.ml[w][r];
        if (x.x != -INFINITY) l = fmaf(x.y, ex2(x.x - m), l);
        if (x.y != x.y) l = x.y;
      }
      wait(&c.o_done, si & 1);
      tc_fence_after();
      const bool whole = g.w0 == 0 && g.w1 == g.nt;
      float f_old = 0.f, f_new = 1.f;  // f32: of the rows so far, of this window
      if constexpr (F32) {
        const float M = first ? m : fmaxf(m_acc, m);
        f_old = first || m_acc == -INFINITY ? 0.f : ex2(m_acc - M);
        f_new = m == -INFINITY ? 0.f : ex2(m - M);
        l_acc = first ? l : l_acc * f_old + l * f_new;
        m_acc = M;
        l = l_acc;
        f_new *= exp2_int(-c.ve[si & 7]);
      }
      bool bad = c.bad || !(l < INFINITY);
      const float inv = whole && last ? (l == 0.f ? 0.f : 1.f / l) : 1.f;
      float *part = nullptr;
      if constexpr (TREE) {
        if (!whole) {
          const int64_t pr = ((int64_t)blockIdx.x * 2 + (g.w0 == 0)) * a.part_rows + r;
          part = a.part + pr * HD;
          if (have && wg == 0 && last) {
            a.ml[2 * pr] = F32 ? m_acc : m;
            a.ml[2 * pr + 1] = c.bad ? __int_as_float(0x7fffffff) : l;
          }
        }
      }
      if (warp_live) {
#pragma unroll 1
        for (int k = 0; k < HD / 64; k++) {
          const int col = wg * (HD / 2) + 32 * k;
          uint32_t x[32];
          tmem_ld32(tm + lane_base + O_COL + col, x);
          tmem_wait_ld();
          if (!have) continue;
          T *o = (T *)a.o + row * a.orow + h * a.ohead + col;
          if constexpr (F32) {
            float *dst = part ? part + col : (float *)o;
            const bool v4 = part || ovec;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
              float old[4] = {0.f, 0.f, 0.f, 0.f}, f[4];
              if (!first) {
                if (v4) *(float4 *)old = *(const float4 *)(dst + i);
                else
                  for (int d = 0; d < 4; d++) old[d] = dst[i + d];
              }
#pragma unroll
              for (int d = 0; d < 4; d++) {
                f[d] = __uint_as_float(x[i + d]) * f_new;
                if (!first) f[d] = fmaf(old[d], f_old, f[d]);
                f[d] = l == 0.f ? 0.f : f[d] * inv;
                bad |= !(fabsf(f[d]) < INFINITY);
              }
              if (v4) *(float4 *)(dst + i) = *(const float4 *)f;
              else
                for (int d = 0; d < 4; d++) dst[i + d] = f[d];
            }
          } else {
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
              f[i] = l == 0.f ? 0.f : __uint_as_float(x[i]) * inv;
              bad |= !(fabsf(f[i]) < INFINITY);
            }
            if (TREE && part) {
#pragma unroll
              for (int i = 0; i < 32; i += 4)
                *(float4 *)(part + col + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
            } else if (ovec) {
#pragma unroll
              for (int i = 0; i < 32; i += 8)
                *(uint4 *)(o + i) = make_uint4(pack2(BF, f[i], f[i + 1]), pack2(BF, f[i + 2], f[i + 3]),
                                               pack2(BF, f[i + 4], f[i + 5]), pack2(BF, f[i + 6], f[i + 7]));
            } else {
#pragma unroll
              for (int i = 0; i < 32; i++) o[i] = from_f<T>(f[i]);
            }
          }
        }
      }
      if (have && bad && whole && last) atomicOr(&c.badrows[r >> 5], 1u << (r & 31));
      tc_fence_before();
      mbar_arrive(&c.o_free);
      named_bar(3, 256);
      if (wg == 0) {
        unsigned w = c.badrows[warp];
        __syncwarp();
        if (w) {
          if (lane == 0) c.badrows[warp] = 0;
          for (; w; w &= w - 1) {
            int64_t row2;
            int h2, t2;
            place(warp * 32 + __ffs(w) - 1, row2, h2, t2);
            exact_row<T, HD, TREE>(a, g.s, t2, pbegin, (int)row2, h2);
          }
        }
      }
      gt += nt;
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------ MMA issue
    if (lane == 0) {
      constexpr uint32_t I_S = tc_idesc_16(BF, false, 128, 128), I_O = tc_idesc_16(BF, true, 128, HD);
      const uint32_t q_lo = sw128_lo(smem_u32(qs), 16), k_lo = sw128_lo(smem_u32(ring), 16), v_lo = sw128_lo(smem_u32(ring), VK * 128);
      int slot = 0, par = 0, gt = 0;
      auto take = [&]() {
        wait(&c.full[slot], par);
        tc_fence_after();
      };
      auto give = [&]() {
        tc_commit(&c.empty[slot]);
        if (++slot == NS) {
          slot = 0;
          par ^= 1;
        }
      };
      auto qk = [&](int gi) {
        const uint32_t d = tm + S_COL + 128 * (gi & 1);
        auto block = [&](uint32_t q, bool add) {
          const uint32_t kk = k_lo + slot * (PIECE >> 4);
#pragma unroll
          for (int k = 0; k < 4; k++) tc_mma_ss_sw128(d, q + k * 2, kk + k * 2, I_S, add || k);
        };
        for (int b = 0; b < NP; b++) {
          const uint32_t q = q_lo + b * 1024;
          take();
          block(q, b != 0);
          if (F32) block(q + (G_::Q_BYTES >> 4), true);
          give();
          if (F32) {
            take();
            block(q, true);
            give();
          }
        }
        tc_commit(&c.s_full[gi & 1]);
      };
      Seg g;
      int qi = 0;
      for (int si = 0; next(g); si++) {
        const int nt = g.t1 - g.t0;
        if (g.t0 == g.w0) {
          wait(&c.q_full, qi++ & 1);
          tc_fence_after();
        }
        qk(gt);
        if (nt > 1) qk(gt + 1);
        if (si > 0) {
          wait(&c.o_free, (si - 1) & 1);
          tc_fence_after();
        }
        for (int j = 0; j < nt; j++) {
          const int gi = gt + j;
          wait(&c.p_ready[gi & 1], (gi >> 1) & 1);
          tc_fence_after();
          const uint32_t p = tm + S_COL + 128 * (gi & 1);
          auto block = [&](int b, int lo, bool add) {
            const uint32_t vv = v_lo + slot * (PIECE >> 4);
#pragma unroll
            for (int k = 0; k < VK / 16; k++) {
              const int ks = b * (VK / 16) + k;
              tc_mma_ts_sw128(tm + O_COL, p + (F32 ? 32 * (ks >> 1) + 8 * (ks & 1) + 16 * lo : 8 * ks), vv + k * 128, I_O,
                              add || k);
            }
          };
          for (int b = 0; b < NP; b++) {
            take();
            block(b, 0, (j | b) != 0);
            if (F32) block(b, 1, true);
            give();
            if (F32) {
              take();
              block(b, 0, true);
              give();
            }
          }
          tc_commit(&c.pv_done);
          if (j + 2 < nt) qk(gi + 2);
        }
        tc_commit(&c.o_done);  // pv_done may be two phases behind here, which its parity cannot tell
        gt += nt;
      }
      // nothing may be in flight when the CTA frees its memory, even after a wait gave up
      tc_commit(&c.drained);
      const int no = 0;
      mbar_wait(&c.drained, 0, &no);
    }
    __syncwarp();
  } else if constexpr (TMA) {
    // ------------------------------------------------------------ loads, TMA
    if (lane == 0) {
      // one tensor copy occupies its thread for a fraction of a microsecond: the pieces go round the warps
      const int mine = warp - 9;
      int slot = 0, par = 1, turn = 0;  // the first pass over the ring waits for nothing
      auto put = [&](bool is_v, int z, int b, int hk) {
        if (turn == mine) {
          wait(&c.empty[slot], par);
          mbar_expect_tx(&c.full[slot], PIECE);
          uint8_t *dst = ring + slot * PIECE;
          if (!is_v) tma_4d(dst, &mk, 0, z, b, hk, &c.full[slot]);
          else tma_4d(dst, &mv, 0, z + b * VK, 0, hk, &c.full[slot]);
        }
        if (++turn == TMA_WARPS) turn = 0;
        if (++slot == NS) {
          slot = 0;
          par ^= 1;
        }
      };
      Seg g;
      while (next(g)) {
        for (int j = 0; j <= g.nt; j++) {
          if (j < g.nt)
            for (int b = 0; b < NP; b++) put(false, pbegin + j * TC_KEYS, b, g.hk);
          if (j > 0)
            for (int b = 0; b < NP; b++) put(true, pbegin + (j - 1) * TC_KEYS, b, g.hk);
        }
      }
      if (c.abort) {  // copies may still be landing: a millisecond is far beyond any of them
        const long long t0 = cycles_now();
        while (cycles_now() - t0 < 2000000ll) {
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ loads, one 16-byte unit per thread
    const int lt = tid - 288;
    // A thread copies 16-byte units (8 dims) of the rows lt/8, lt/8 + LD/8, ...  of a tile, K and V alike, so its row
    // pointers are made once per tile: K piece b takes the block b of all of its rows, V piece b every block of the
    // rows that lie in it.
    constexpr int RSTEP = LD / 8, NR = TC_KEYS / RSTEP, RV = VK / RSTEP;
    const int r0 = lt >> 3, u0 = lt & 7, swz = r0 * 128 + ((u0 ^ (r0 & 7)) << 4);
    // unit i (of NR) of a piece: its row and its block, and its place in the piece
    auto unit_row = [&](bool is_v, int b, int i) { return is_v ? b * RV + i % RV : i; };
    auto unit_block = [&](bool is_v, int b, int i) { return is_v ? i / RV : b; };
    auto unit_at = [&](bool is_v, int i) { return swz + (is_v ? (i / RV) * (VK * 128) + (i % RV) * (RSTEP * 128) : i * (RSTEP * 128)); };
    const T *row_p[NR];  // nullptr: no such slot
    constexpr uint32_t NONE = 0xffffffffu;
    // pool rows (or prompt rows) of a tile's slots
    auto offsets = [&](const Seg &g, int tile) {
      named_bar(4, LD);  // the readers of two tiles ago are through
      const int sl = tile * TC_KEYS + lt;
      if (lt < TC_KEYS) {
        uint32_t o = NONE;
        if constexpr (TREE) {
          if (sl < g.ts.n) {
            const int64_t x = cwp_row(a.kv.table + (int64_t)g.s * a.kv.stride, a.kv.stride, a.kv.n_pages, a.kv.page_size, sl);
            if (x >= 0) {
              o = (uint32_t)x;
            } else {
              c.bad = 1;
              atomicOr(a.err, OPE_PAGE);
            }
          }
          if (g.ts.cut && lt == 0) atomicOr(a.err, OPE_PAGE);
        } else if (pbegin + sl < pend) {
          o = (uint32_t)(pbegin + sl);
        }
        c.rowoff[tile & 1][lt] = o;
      }
      named_bar(4, LD);
    };
    auto rows_of = [&](bool is_v, int tile, int hk) {
#pragma unroll
      for (int i = 0; i < NR; i++) {
        const uint32_t o = c.rowoff[tile & 1][r0 + i * RSTEP];
        const T *p;
        if constexpr (TREE) p = (const T *)(is_v ? a.kv.v : a.kv.k) + ((int64_t)o * a.nkv + hk) * HD;
        else p = (const T *)(is_v ? a.v : a.k) + (int64_t)o * (is_v ? a.vrow : a.krow) + hk * (is_v ? a.vhead : a.khead);
        row_p[i] = o == NONE ? nullptr : p + u0 * 8;
      }
    };
    // the pieces in the order of their use: K(t0), then K(j), V(j - 1), then V(t1 - 1)
    Seg g;
    int si = -1, pj = 0, pb = 0;
    bool is_v = false, more = false;
    auto advance = [&]() -> bool {
      if (more && ++pb == NP) {
        pb = 0;
        if (!is_v && pj > g.t0) {
          is_v = true;
        } else {
          is_v = ++pj == g.t1;
          more = pj <= g.t1;
        }
      }
      if (!more) {
        if (!next(g)) return false;
        si++;
        pj = g.t0;
        pb = 0;
        is_v = false;
        more = true;
      }
      if (pb == 0) {
        if (!is_v) offsets(g, pj);
        rows_of(is_v, is_v ? pj - 1 : pj, g.hk);
      }
      return true;
    };
    int slot = 0, par = 1;  // the first pass over the ring waits for nothing
    auto step = [&]() {
      if (++slot == NS) {
        slot = 0;
        par ^= 1;
      }
    };
    if constexpr (F32) {
      // a thread's four units of a piece are in registers: each is loaded for the next piece as soon as it is
      // split and stored for this one
      float x[4][8];
      const bool vec = TREE || a.vec;
      // fixed i: the row of a unit depends on the piece only through b, which a switch over few values resolves
      auto load = [&](int i) {
        const float *src = nullptr;
        if (!is_v) {
          src = (const float *)row_p[i];
        } else {
#pragma unroll
          for (int r = 0; r < NR; r++)
            if (r == unit_row(true, pb, i)) src = (const float *)row_p[r];
        }
        if (!src) {
#pragma unroll
          for (int k = 0; k < 8; k++) x[i][k] = 0.f;
        } else {
          src += unit_block(is_v, pb, i) * 64;
          if (vec) {
            *(float4 *)x[i] = *(const float4 *)src;
            *(float4 *)(x[i] + 4) = *(const float4 *)(src + 4);
          } else {
#pragma unroll
            for (int k = 0; k < 8; k++) x[i][k] = src[k];
          }
        }
      };
      float fk = 1.f, fv = 1.f;
      bool have = advance();
      if (have) {
#pragma unroll
        for (int i = 0; i < 4; i++) load(i);
      }
      while (have) {
        const bool v = is_v, first = (v ? pj - 1 : pj) == g.t0 && pb == 0;
        const int wi = si & 7;
        have = advance();
        int e = 0;
        if (first) {
          float mx = 0.f;
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) mx = fmaxf(mx, fabsf(x[i][k]));
          mx = warp_max(mx);
          named_bar(4, LD);
          if (lane == 0) c.amax[warp - 9] = mx;
          named_bar(4, LD);
#pragma unroll
          for (int i = 0; i < 8; i++) mx = fmaxf(mx, c.amax[i]);
          e = scale_exp(mx);
          (v ? fv : fk) = exp2_int(e);
        }
        const float f = v ? fv : fk;
        const int s_hi = slot;
        wait(&c.empty[slot], par);
        step();
        const int s_lo = slot;
        wait(&c.empty[slot], par);
        step();
        if (first && lt == 0) (v ? c.ve : c.ke)[wi] = e;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t at = unit_at(v, i);
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int k = 0; k < 4; k++) split2(x[i][2 * k] * f, x[i][2 * k + 1] * f, hi[k], lo[k]);
          *(uint4 *)(ring + s_hi * PIECE + at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *(uint4 *)(ring + s_lo * PIECE + at) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
          if (have) load(i);
        }
        fence_proxy_async_smem();
        mbar_arrive(&c.full[s_hi]);
        mbar_arrive(&c.full[s_lo]);
      }
    } else {
      constexpr int D = 5;  // pieces in flight per thread
      static_assert(D < NS, "a piece in flight needs its slot");
      int done = 0, issued = 0;
      auto finish = [&]() {  // this thread's part of the oldest piece in flight has landed
        fence_proxy_async_smem();
        mbar_arrive(&c.full[done % NS]);
        done++;
      };
      while (advance()) {
        wait(&c.empty[slot], par);
        const uint32_t base = smem_u32(ring + slot * PIECE);
        auto piece = [&](auto v_const, auto b_const) {  // both known: row_p stays in registers
          constexpr bool V = decltype(v_const)::value;
          constexpr int B = decltype(b_const)::value;
#pragma unroll
          for (int i = 0; i < NR; i++) {
            const T *src = row_p[unit_row(V, B, i)];
            const bool ok = src != nullptr;
            src = ok ? src + unit_block(V, B, i) * 64 : (const T *)(TREE ? a.kv.k : a.k);
            const uint32_t dst = base + unit_at(V, i);
            if (TREE || a.vec) {
              cp_async16(dst, src, ok);
            } else {
              T e[8];
#pragma unroll
              for (int k = 0; k < 8; k++) e[k] = ok ? src[k] : from_f<T>(0.f);
              const uint4 w = *(uint4 *)e;
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                           : "memory");
            }
          }
        };
        auto of_kind = [&](auto v_const) {
          if (NP == 1 || pb == 0) piece(v_const, std::integral_constant<int, 0>());
          else if (NP == 2 || pb == 1) piece(v_const, std::integral_constant<int, NP >= 2 ? 1 : 0>());
          else if (pb == 2) piece(v_const, std::integral_constant<int, NP >= 4 ? 2 : 0>());
          else piece(v_const, std::integral_constant<int, NP >= 4 ? 3 : 0>());
        };
        if (is_v) of_kind(std::true_type());
        else of_kind(std::false_type());
        cp_async_commit();
        issued++;
        step();
        if (issued - done > D) {
          cp_async_wait<D>();
          finish();
        }
      }
      cp_async_wait<0>();
      while (done < issued) finish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// Joins the parts of a row whose slots were split over CTAs: one warp per row,
// parts in CTA order.  Grid (sequence, kv head, groups of 8 rows).
template <int TY, int HD>
__global__ void __launch_bounds__(256) tc_combine_kernel(const __grid_constant__ AttnOp a) {
  using T = typename TypeOf<TY>::T;
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, s = blockIdx.x, hk = blockIdx.y, G = a.nh / a.nkv;
  const int item = blockIdx.z * 8 + (threadIdx.x >> 5);
  const TreeSeq q = tree_seq(a, s);
  if (item >= q.live * G) return;
  int64_t before = 0, total = 0;
  for (int i = lane; i < a.n_seq; i += 32) {
    const int64_t n = seq_units(a, i);
    total += n;
    if (i < s) before += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    total += __shfl_xor_sync(0xffffffffu, total, o);
  }
  const int C = a.n_cta, nt = tree_tiles(q.n), mts = (q.live * G + TC_ROWS - 1) / TC_ROWS;
  const int mt = item / TC_ROWS, r = item % TC_ROWS;
  const int64_t ua = before + (int64_t)(hk * mts + mt) * nt, ub = ua + nt;
  const int c0 = (int)(((ua + 1) * C - 1) / total), c1 = (int)((ub * C - 1) / total);
  if (c0 == c1) return;  // written by its CTA
  // (max, sum) of part c; an empty CTA has none
  auto part_row = [&](int cc) -> int64_t {
    const int64_t x0 = total * cc / C, x1 = total * (cc + 1) / C;
    return x0 == x1 ? -1 : ((int64_t)cc * 2 + (ua >= x0)) * a.part_rows + r;
  };
  float m = -INFINITY;
  for (int cc = c0 + lane; cc <= c1; cc += 32) {
    const int64_t p = part_row(cc);
    if (p >= 0) m = fmaxf(m, a.ml[2 * p]);
  }
  m = warp_max(m);
  constexpr int DL = HD / 32;
  float l = 0.f, acc[DL];
#pragma unroll
  for (int i = 0; i < DL; i++) acc[i] = 0.f;
  for (int cb = c0; cb <= c1; cb += 32) {
    const int64_t p = cb + lane <= c1 ? part_row(cb + lane) : -1;
    float w = 0.f, lp = 0.f;
    if (p >= 0) {
      const float mp = a.ml[2 * p];
      lp = a.ml[2 * p + 1];
      w = mp == -INFINITY ? 0.f : ex2(mp - m);
      if (lp != lp) w = 1.f;
    }
    l += warp_sum(w * lp);
    const int n = min(32, c1 - cb + 1);
#pragma unroll 4
    for (int i = 0; i < n; i++) {
      const int64_t pi = __shfl_sync(0xffffffffu, p, i);
      const float wi = __shfl_sync(0xffffffffu, w, i);
      if (pi < 0 || wi == 0.f) continue;
      const float *x = a.part + pi * HD + lane * DL;
#pragma unroll
      for (int d = 0; d < DL; d++) acc[d] = fmaf(wi, x[d], acc[d]);
    }
  }
  const int t = item / G, h = hk * G + item - t * G;
  const int64_t row = (int64_t)s * a.T + t;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bool bad = !(l < INFINITY);
  T *o = (T *)a.o + row * a.orow + h * a.ohead + lane * DL;
#pragma unroll
  for (int d = 0; d < DL; d++) {
    const float x = l == 0.f ? 0.f : acc[d] * inv;
    bad |= !(fabsf(x) < INFINITY);
    o[d] = from_f<T>(x);
  }
  if (__any_sync(0xffffffffu, bad)) exact_row<T, HD, true>(a, s, t, 0, (int)row, h);
}

// ------------------------------------------------------------------ host
namespace {

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled g_encode = nullptr;

// Rows [n_rows][nkv] of hd dims as [head][64-dim block][row][64], in boxes of box_rows rows x box_blocks blocks.
bool make_map(CUtensorMap *m, bool bf16, const void *p, int64_t row, int64_t head, int hd, int nkv, int n_rows,
              int box_rows, int box_blocks) {
  if (nkv == 1) head = hd;  // never used; must be a stride all the same
  const int64_t lim = (int64_t)1 << 39;
  if (!g_encode || (uintptr_t)p % 16 || row < 8 || head < 8 || row % 8 || head % 8 || row > lim || head > lim) return false;
  const cuuint64_t dims[4] = {64, (cuuint64_t)n_rows, (cuuint64_t)hd / 64, (cuuint64_t)nkv};
  const cuuint64_t strides[3] = {(cuuint64_t)row * 2, 128, (cuuint64_t)head * 2};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, (cuuint32_t)box_blocks, 1}, one[4] = {1, 1, 1, 1};
  return g_encode(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(p),
                  dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TY, int HD, bool TREE, bool TMA>
cudaError_t configure_one() {
  return cudaFuncSetAttribute(attn_tc_kernel<TY, HD, TREE, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              Geo<TY, HD>::SMEM);
}
template <int TY, int HD>
cudaError_t configure_hd() {
  if constexpr (TY != TY_F32) CW_TRY((configure_one<TY, HD, false, true>()));
  CW_TRY((configure_one<TY, HD, false, false>()));
  CW_TRY((configure_one<TY, HD, true, false>()));
  return carveout_max(tc_combine_kernel<TY, HD>);
}

template <int TY, int HD>
cudaError_t prompt_hd(AttnOp a, cudaStream_t st) {
  CUtensorMap mk, mv;
  const int64_t tiles = (int64_t)a.n_rows / TC_ROWS + a.n_seq;
  if (tiles * a.nh > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const dim3 grid((unsigned)(tiles * a.nh));
  using G = Geo<TY, HD>;
  if constexpr (TY != TY_F32) {
    if (make_map(&mk, TY == TY_BF16, a.k, a.krow, a.khead, HD, a.nkv, a.n_rows, TC_KEYS, 1) &&
        make_map(&mv, TY == TY_BF16, a.v, a.vrow, a.vhead, HD, a.nkv, a.n_rows, G::VK, G::CB))
      return launch_pdl(attn_tc_kernel<TY, HD, false, true>, grid, G::threads(true), G::SMEM, st, a, mk, mv);
  }
  memset(&mk, 0, sizeof mk);
  memset(&mv, 0, sizeof mv);
  const int al = TY == TY_F32 ? 4 : 8;
  a.vec = ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 && (a.krow | a.khead | a.vrow | a.vhead) % al == 0;
  return launch_pdl(attn_tc_kernel<TY, HD, false, false>, grid, G::threads(false), G::SMEM, st, a, mk, mv);
}

template <int TY, int HD>
cudaError_t tree_hd(const AttnOp &a, cudaStream_t st) {
  static const CUtensorMap none = {};
  using G = Geo<TY, HD>;
  CW_TRY(launch_pdl(attn_tc_kernel<TY, HD, true, false>, dim3(a.n_cta), G::threads(false), G::SMEM, st, a, none, none));
  if (tree_tiles(a.max_len) == 1) return cudaSuccess;  // no segment can be split
  return launch_pdl(tc_combine_kernel<TY, HD>, dim3(a.n_seq, a.nkv, (a.T * (a.nh / a.nkv) + 7) / 8), 256, 0, st, a);
}

template <int TY>
cudaError_t configure_ty() {
  CW_TRY((configure_hd<TY, 64>()));
  CW_TRY((configure_hd<TY, 128>()));
  return configure_hd<TY, 256>();
}
template <int TY>
cudaError_t prompt_ty(const AttnOp &a, int hd, cudaStream_t st) {
  return hd == 64 ? prompt_hd<TY, 64>(a, st) : hd == 128 ? prompt_hd<TY, 128>(a, st) : prompt_hd<TY, 256>(a, st);
}
template <int TY>
cudaError_t tree_ty(const AttnOp &a, int hd, cudaStream_t st) {
  return hd == 64 ? tree_hd<TY, 64>(a, st) : hd == 128 ? tree_hd<TY, 128>(a, st) : tree_hd<TY, 256>(a, st);
}

}  // namespace

cudaError_t tc_configure() {
  void *fn = nullptr;
  cudaDriverEntryPointQueryResult found;
  CW_TRY(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &found));
  if (found == cudaDriverEntryPointSuccess) g_encode = (EncodeTiled)fn;
  CW_TRY(configure_ty<TY_F32>());
  CW_TRY(configure_ty<TY_F16>());
  return configure_ty<TY_BF16>();
}

cudaError_t tc_prompt(const AttnOp &a, int type, int hd, cudaStream_t st) {
  if (type == CWEN_T_F32) return prompt_ty<TY_F32>(a, hd, st);
  return type == CWEN_T_F16 ? prompt_ty<TY_F16>(a, hd, st) : prompt_ty<TY_BF16>(a, hd, st);
}
cudaError_t tc_tree(const AttnOp &a, int type, int hd, cudaStream_t st) {
  if (type == CWEN_T_F32) return tree_ty<TY_F32>(a, hd, st);
  return type == CWEN_T_F16 ? tree_ty<TY_F16>(a, hd, st) : tree_ty<TY_BF16>(a, hd, st);
}

}  // namespace cw
