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
// work on one while the other's softmax runs); the warps from 9 on fill a ring of
// 16 KB pieces in the order in which the MMAs use them: K as 128 slots x 64
// dims, V as 8192/HD slots x HD dims in groups of 16 slots, both with 128-byte
// swizzle.  f16 and bf16 pieces go round four warps, each lane one tensor copy
// (TMA boxes of whole pages: K as many slots as a page holds in a power of two, V
// 16); pages that are no multiple of 16 slots and rows that TMA cannot address are
// copied 16 bytes a lane (or by element).
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
//
// Bounds and measurements (B200; a tile at head dim 256 is 2048 MMA clocks): a
// long bf16 prompt (16381 tokens in 9 sequences, 24 heads on 4 of 256) takes 1.07
// ms, 1.0 PFLOP/s of causal work, bound by the 128 KB of K and V that every SM
// draws from the L2 per tile; one token over 32767 bf16 slots 44 us (a bare load
// of its bytes 33 us); 9 f32 nodes over 32495 slots 120 us and f32 prompts of 4100
// tokens 0.95 ms, both bound by the loaders' split into parts.
#include <cuda.h>
#include <string.h>

#include <type_traits>

#include "attn_tc.cuh"

namespace cw {

namespace {

constexpr int PIECE = 16384;
constexpr int LOAD_WARPS = 4;  // f16, bf16
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
  static constexpr int LOADERS = F32 ? 256 : 32 * LOAD_WARPS, THREADS = 288 + LOADERS;
  // Tree: what a segment's start and end cost, in tiles.  31 ragged sequences of 8 kv heads of 128, to 12000 slots, a call
  // by itself: 295 us with 4, 272 with 6, 256 with 8 and 257 with 12 (one after another 270 with each); 4 heads of 256
  // one after another 214 with 4, 218 with 6; f32 (8 sequences) 197, 209, 209, 229 with 4, 6, 8, 12.
  static constexpr int SEG_COST = F32 || HD == 256 ? 4 : 8;
  static constexpr int VG = CB * 2048;       // 16 slots of a V piece: [block][16 slots][128 B]
};
// f32: tiles of a window.  Error against 64 bits of a 4100-token prompt and a 12000-token one: 3.1e-6 and 2.3e-6 with 4,
// 3.7e-6 with 8 (prompt), 4.9e-6 and 5.1e-6 with 16, 6.0e-6 and 1.3e-5 unbroken; a window's end costs about 20000 clocks.
constexpr int WIN = 8;
struct Ctl {
  uint64_t full[12], empty[12], s_full[2], p_ready[2], pv_done, q_full, o_free, o_done, drained, tail[LOAD_WARPS];
  int64_t u0, u1;
  int hk0, mt0, t00;
  uint32_t tmem;
  volatile int abort, bad;
  int s0, tile0, begin, end;
  unsigned badrows[4];
  float mref[TC_ROWS];
  float2 ml[2][TC_ROWS];
  uint32_t rowoff[4][TC_KEYS];  // f32, [tile mod 4]: rows of the slots
  // f32: exponents that Q rows, and a window's K and V, were multiplied by (the loaders run up to three windows ahead)
  int qe[TC_ROWS], ke[8], ve[8];
  float amax[8];
};
struct CtlF32 : Ctl {
  alignas(16) uint8_t stage[8][1024];
};

// Where one segment of work lies: the tiles [w0, w1) of a row tile's nt, and
// the window [t0, t1) of them at hand.
struct Seg {
  int s, hk, mt, t0, t1, nt, w0, w1;
  TreeSeq ts;
};

CW_HOST_DEV int tree_tiles(int n) { return (n + TC_KEYS - 1) / TC_KEYS; }
// Units of a segment: first seg_cost that stand for its fixed cost, then its tiles.
CW_DEV int seg_units(const AttnOp &a, int n) { return tree_tiles(n) + a.seg_cost; }
CW_DEV int64_t seq_units(const AttnOp &a, int s) {
  const TreeSeq q = tree_seq(a, s);
  const int G = a.nh / a.nkv;
  return q.live ? (int64_t)a.nkv * ((q.live * G + TC_ROWS - 1) / TC_ROWS) * seg_units(a, q.n) : 0;
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
    hk = c.hk0;
    mt = c.mt0;
    t0 = c.t00;
    left = c.u1 - c.u0;
  }
  CW_DEV bool next(const AttnOp &a, Seg &g) {
    while (step(a, g))
      if (g.t1 > g.t0) return true;  // units without tiles: another CTA's segment
    return false;
  }
  CW_DEV bool step(const AttnOp &a, Seg &g) {
    if (left <= 0) return false;
    const int G = a.nh / a.nkv;
    g.ts = tree_seq(a, s);
    while (g.ts.live == 0) g.ts = tree_seq(a, ++s);
    g.nt = tree_tiles(g.ts.n);
    g.s = s;
    g.hk = hk;
    g.mt = mt;
    const int end = (int)min((int64_t)seg_units(a, g.ts.n), t0 + left);  // units [t0, end) of the segment
    g.t0 = max(t0 - a.seg_cost, 0);
    g.t1 = max(end - a.seg_cost, 0);
    left -= end - t0;
    t0 = 0;
    if (end == seg_units(a, g.ts.n) && ++mt * TC_ROWS >= g.ts.live * G) {
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
// The exponent that brings a largest value into [2^8, 2^9).  Zeros say nothing of what follows: 2^8 leaves room for
// values to 255 in steps of 2^-33.  Non-finite values: 0.
CW_DEV int scale_exp(float amax) {
  if (!(amax < INFINITY)) return 0;
  if (!(amax > 1e-30f)) return 8;
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

// 32 rows of a warp, one per lane in registers, to their places in global memory: through shared memory, so that
// UNITS neighbouring lanes write 16-byte units of one row (32 different rows at once would cost 32 passes of the
// load/store unit).  stage: 32 x UNITS x 16 bytes of the warp.  dst: the lane's row; ok: whether it is there.
template <int UNITS, class E>
CW_DEV void flush_rows(uint8_t *stage, const uint32_t *x, E *dst, bool ok, bool vec) {
  constexpr int M = UNITS - 1, SH = UNITS == 4 ? 1 : 2, N = 16 / (int)sizeof(E);
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < UNITS; u++)
    *(uint4 *)(stage + (lane * UNITS + (u ^ ((lane >> SH) & M))) * 16) = make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < UNITS; i++) {
    const int r = (i * 32 + lane) / UNITS, u = lane & M;
    const uint4 w = *(const uint4 *)(stage + (r * UNITS + (u ^ ((r >> SH) & M))) * 16);
    E *d = (E *)__shfl_sync(0xffffffffu, (unsigned long long)dst, r) + u * N;
    if (!__shfl_sync(0xffffffffu, (int)ok, r)) continue;
    if (vec) {
      *(uint4 *)d = w;
    } else {
      const E *e = (const E *)&w;
#pragma unroll
      for (int k = 0; k < N; k++) d[k] = e[k];
    }
  }
  __syncwarp();
}
// The way back.
template <int UNITS>
CW_DEV void fetch_rows(uint8_t *stage, uint32_t *x, const float *src, bool ok, bool vec) {
  constexpr int M = UNITS - 1, SH = UNITS == 4 ? 1 : 2;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < UNITS; i++) {
    const int r = (i * 32 + lane) / UNITS, u = lane & M;
    const float *p = (const float *)__shfl_sync(0xffffffffu, (unsigned long long)src, r) + u * 4;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    if (__shfl_sync(0xffffffffu, (int)ok, r)) {
      if (vec) w = *(const float4 *)p;
      else w = make_float4(p[0], p[1], p[2], p[3]);
    }
    *(float4 *)(stage + (r * UNITS + (u ^ ((r >> SH) & M))) * 16) = w;
  }
  __syncwarp();
#pragma unroll
  for (int u = 0; u < UNITS; u++) {
    const uint4 w = *(const uint4 *)(stage + (lane * UNITS + (u ^ ((lane >> SH) & M))) * 16);
    x[4 * u] = w.x;
    x[4 * u + 1] = w.y;
    x[4 * u + 2] = w.z;
    x[4 * u + 3] = w.w;
  }
  __syncwarp();
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

// kbox: slots of a K box, 0 where tensor copies are not used (pages of no multiple of 16 slots, rows off 16 bytes).
// One token over 32767 bf16 slots: 44 us with them, 50-62 us with 16-byte copies by lanes, whose address arithmetic
// holds up the loaders.
template <int TY, int HD, bool TREE>
__global__ void __launch_bounds__(Geo<TY, HD>::THREADS, 1)
    attn_tc_kernel(const __grid_constant__ AttnOp a, const __grid_constant__ CUtensorMap mk,
                   const __grid_constant__ CUtensorMap mv, int kbox) {
  using G_ = Geo<TY, HD>;
  using T = typename TypeOf<TY>::T;
  constexpr bool F32 = TY == TY_F32, BF = TY == TY_BF16;
  constexpr int LD = G_::LOADERS;
  constexpr int CB = G_::CB, NP = G_::NP, VK = G_::VK, NS = G_::NS;
  constexpr int O_COL = 0, S_COL = 256;
  __shared__ typename std::conditional<F32, CtlF32, Ctl>::type c;
  extern __shared__ uint8_t dyn[];
  uint8_t *qs = (uint8_t *)(((uintptr_t)dyn + 1023) & ~(uintptr_t)1023);
  uint8_t *ring = qs + G_::Q_BYTES * (F32 ? 2 : 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int G = a.nh / a.nkv;

  if (warp == 8) tmem_alloc(&c.tmem, 512);
  if (tid == 0) {
    for (int i = 0; i < NS; i++) {
      mbar_init(&c.full[i], F32 ? LD : 1);
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
    for (int i = 0; i < LOAD_WARPS; i++) mbar_init(&c.tail[i], 1);
    mbar_fence_init();
    c.abort = 0;
    c.bad = 0;
  }
  if (tid < 4) c.badrows[tid] = 0;
  if (!F32 && kbox && tid == 9 * 32) {
    tma_prefetch_map(&mk);
    tma_prefetch_map(&mv);
  }
  pdl_wait();
  pdl_trigger();  // after the wait: the joining kernel may read the lengths before its own wait
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
          c.begin = b;
          c.end = e;
          c.tile0 = (int)(u0 - at);
          if constexpr (TREE) {
            const TreeSeq q = tree_seq(a, i);
            const int64_t rem = u0 - at;
            const int nt = seg_units(a, q.n), mts = (q.live * G + TC_ROWS - 1) / TC_ROWS;
            const int64_t x = rem <= 0x7fffffff ? (uint32_t)rem / (uint32_t)nt : rem / nt;
            c.t00 = (int)(rem - x * nt);
            c.mt0 = (int)x % mts;  // x < n_kv mts
            c.hk0 = (int)x / mts;
          }
          break;
        }
        at += n;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tm = c.tmem;
  if (c.u0 >= c.u1) {
    if (warp == 8) tmem_dealloc(tm, 512);
    return;
  }

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
        if constexpr (F32) {
          constexpr int UB = CB < 4 ? CB : 4;  // units on their way at once
#pragma unroll 1
          for (int i0 = tid; i0 < 128 * CB * 8; i0 += 256 * UB) {
            float x[UB][8];
#pragma unroll
            for (int j = 0; j < UB; j++) {
              const int i = i0 + 256 * j, rr = i / (CB * 8), u = i % (CB * 8);
              int64_t row;
              int h, t;
              const bool have = place(rr, row, h, t);
              const float *src = (const float *)a.q + (have ? row * a.qrow + h * a.qhead + u * 8 : 0);
#pragma unroll
              for (int k = 0; k < 8; k++) x[j][k] = 0.f;
              if (have && qvec) {
                *(float4 *)x[j] = *(const float4 *)src;
                *(float4 *)(x[j] + 4) = *(const float4 *)(src + 4);
              } else if (have) {
#pragma unroll
                for (int k = 0; k < 8; k++) x[j][k] = src[k];
              }
            }
#pragma unroll
            for (int j = 0; j < UB; j++) {
              const int i = i0 + 256 * j, rr = i / (CB * 8), u = i % (CB * 8);
              uint8_t *dst = qs + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4);
              float mx = 0.f;
#pragma unroll
              for (int k = 0; k < 8; k++) mx = fmaxf(mx, fabsf(x[j][k]));
#pragma unroll
              for (int k = 1; k < CB * 8; k <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, k));
              const int e = scale_exp(mx);
              const float f = a.scale < 0.f ? -exp2_int(e) : exp2_int(e);
              uint32_t hi[4], lo[4];
#pragma unroll
              for (int k = 0; k < 4; k++) split2(x[j][2 * k] * f, x[j][2 * k + 1] * f, hi[k], lo[k]);
              *(uint4 *)dst = make_uint4(hi[0], hi[1], hi[2], hi[3]);
              *(uint4 *)(dst + G_::Q_BYTES) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
              if (u == 0) c.qe[rr] = e;
            }
          }
        } else {
#pragma unroll 4
          for (int i = tid; i < 128 * CB * 8; i += 256) {
            const int rr = i / (CB * 8), u = i % (CB * 8);
            int64_t row;
            int h, t;
            const bool have = place(rr, row, h, t);
            uint8_t *dst = qs + (u >> 3) * 16384 + rr * 128 + (((u & 7) ^ (rr & 7)) << 4);
            const T *src = (const T *)a.q + (have ? row * a.qrow + h * a.qhead + u * 8 : 0);
            if (qvec) {
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
      // Q is read no more, but by another window of the segment
      uint8_t *const stage = qs + warp * 2048;
      if (warp_live) {
#pragma unroll 1
        for (int k = 0; k < HD / 64; k++) {
          const int col = wg * (HD / 2) + 32 * k;
          uint32_t x[32];
          tmem_ld32(tm + lane_base + O_COL + col, x);
          tmem_wait_ld();
          T *o = (T *)a.o + (have ? row * a.orow + h * a.ohead : 0) + col;
          if constexpr (F32) {
            float *dst = part ? part + col : (float *)o;
            const bool v4 = part || ovec;
            auto emit = [&](auto units, uint8_t *st) {
              constexpr int U = decltype(units)::value;
#pragma unroll
              for (int i = 0; i < 32; i += 4 * U) {
                uint32_t old[4 * U];
                float f[4 * U];
                if (!first) fetch_rows<U>(st, old, dst + i, have, v4);
#pragma unroll
                for (int d = 0; d < 4 * U; d++) {
                  f[d] = __uint_as_float(x[i + d]) * f_new;
                  if (!first) f[d] = fmaf(__uint_as_float(old[d]), f_old, f[d]);
                  f[d] = l == 0.f ? 0.f : f[d] * inv;
                  bad |= !(fabsf(f[d]) < INFINITY);
                }
                flush_rows<U>(st, (const uint32_t *)f, dst + i, have, v4);
              }
            };
            emit(std::integral_constant<int, 2>(), c.stage[warp]);
          } else {
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; i++) {
              f[i] = l == 0.f ? 0.f : __uint_as_float(x[i]) * inv;
              bad |= !(fabsf(f[i]) < INFINITY);
            }
            if (TREE && part) {
#pragma unroll
              for (int i = 0; i < 32; i += 16) flush_rows<4>(stage, (const uint32_t *)f + i, part + col + i, have, true);
            } else {
              uint32_t w[16];
#pragma unroll
              for (int i = 0; i < 16; i++) w[i] = pack2(BF, f[2 * i], f[2 * i + 1]);
              flush_rows<4>(stage, w, o, have, ovec);
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
      const uint32_t q_lo = sw128_lo(smem_u32(qs), 16), k_lo = sw128_lo(smem_u32(ring), 16), v_lo = sw128_lo(smem_u32(ring), 2048);
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
              tc_mma_ts_sw128(tm + O_COL, p + (F32 ? 32 * (ks >> 1) + 8 * (ks & 1) + 16 * lo : 8 * ks), vv + k * (G_::VG >> 4), I_O,
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
  } else if constexpr (!F32) {
    // ------------------------------------------------------------ loads, a piece per warp
    const int mine = warp - 9;
    int slot = 0, par = 1, turn = 0, tails = 0;  // the first pass over the ring waits for nothing
    // pool row (or prompt row) of a slot, -1: none
    auto row_of = [&](const Seg &g, int sl) -> int64_t {
      if constexpr (TREE) {
        if (sl >= g.ts.n) return -1;
        const int64_t r = cwp_row(a.kv.table + (int64_t)g.s * a.kv.stride, a.kv.stride, a.kv.n_pages, a.kv.page_size, sl);
        if (r < 0) {
          c.bad = 1;
          atomicOr(a.err, OPE_PAGE);
        }
        return r;
      } else {
        return pbegin + sl < pend ? pbegin + sl : -1;
      }
    };
    auto put = [&](const Seg &g, bool is_v, int tile, int b) {
      if (turn == mine) {
        wait(&c.empty[slot], par);
        uint8_t *dst = ring + slot * PIECE;
        const int n = TREE ? g.ts.n : pend - pbegin, sl0 = tile * TC_KEYS + (is_v ? b * VK : 0);
        if (kbox) {
          // a tile that ends inside: boxes with a slot at least, then zeros over the V rows behind the last slot
          // (whatever they hold meets zero weights, which must not make NaN); K there meets the mask
          const int step = is_v ? 16 : kbox, have = min(n - sl0, is_v ? VK : TC_KEYS);  // slots of the piece
          const int boxes = have <= 0 ? 0 : (have + step - 1) / step;
          const bool tail = is_v && have < VK;
          uint64_t *bar = tail ? &c.tail[mine] : &c.full[slot];
          if (lane == 0 && boxes) mbar_expect_tx(bar, boxes * (is_v ? G_::VG : step * 128));
          __syncwarp();
          if (lane < boxes) {
            int64_t r = row_of(g, sl0 + lane * step);
            if (r < 0) r = 0;  // a bad page: any rows do, exact_row comes after
            if (!is_v) tma_4d(dst + lane * step * 128, &mk, 0, (int)r, b, g.hk, bar);
            else tma_4d(dst + lane * G_::VG, &mv, 0, (int)r, 0, g.hk, bar);
          }
          if (tail) {
            if (boxes) {
              wait(bar, tails & 1);
              tails++;
            }
            constexpr int UR = HD / 8;
            for (int i = max(have, 0) * UR + lane; i < VK * UR; i += 32) {
              const int key = i / UR, u = i % UR;
              *(uint4 *)(dst + (key >> 4) * G_::VG + (u >> 3) * 2048 + (key & 15) * 128 + ((u & 7) << 4)) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&c.full[slot]);
          }
        } else {
          // rows a lane looks up (K, V); V: units of a row, rows a step
          constexpr int KL = TC_KEYS / 32, VL = VK / 32, UR = HD / 8, VR = 32 / UR;
          const T *base = (const T *)(TREE ? (is_v ? a.kv.v : a.kv.k) : (is_v ? a.v : a.k));
          const int64_t rs = TREE ? (int64_t)a.nkv * HD : is_v ? a.vrow : a.krow, hs = TREE ? HD : is_v ? a.vhead : a.khead;
          base += g.hk * hs;
          int64_t off[KL];
#pragma unroll
          for (int i = 0; i < KL; i++) {
            off[i] = -1;
            if (i < VL || !is_v) off[i] = row_of(g, sl0 + lane + 32 * i);
          }
#pragma unroll 1
          for (int i8 = 0; i8 < 4; i8++) {  // 8 units a lane at a time: the code runs rarely, and from a cold cache
            const int pick = is_v ? i8 * VR / 4 : i8;
            const int64_t mine_r = pick == 0 ? off[0] : pick == 1 ? off[1] : pick == 2 ? off[2] : off[3];
#pragma unroll
            for (int ii = 0; ii < 8; ii++) {
              const int i = i8 * 8 + ii;
              const int key = is_v ? i * VR + lane / UR : i * 4 + (lane >> 3), u = is_v ? lane % UR : b * 8 + (lane & 7);
              const int64_t r = __shfl_sync(0xffffffffu, mine_r, key & 31);
              const T *src = base + (r < 0 ? 0 : r * rs + u * 8);
              uint8_t *d = dst + (((u & 7) ^ (key & 7)) << 4) +
                           (is_v ? (key >> 4) * G_::VG + (u >> 3) * 2048 + (key & 15) * 128 : key * 128);
              if (TREE || a.vec) {
                cp_async16(smem_u32(d), src, r >= 0);
              } else {
                T e[8];
#pragma unroll
                for (int k = 0; k < 8; k++) e[k] = r >= 0 ? src[k] : from_f<T>(0.f);
                *(uint4 *)d = *(uint4 *)e;
              }
            }
          }
          cp_async_commit();
          cp_async_wait<0>();
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&c.full[slot]);
        }
      }
      if (++turn == LOAD_WARPS) turn = 0;
      if (++slot == NS) {
        slot = 0;
        par ^= 1;
      }
    };
    Seg g;
    while (next(g)) {
      if (TREE && g.ts.cut && lane == 0) atomicOr(a.err, OPE_PAGE);
      // K(t0), then K(j), V(j - 1), then V(t1 - 1)
      for (int j = g.t0; j <= g.t1; j++) {
        if (j < g.t1)
          for (int b = 0; b < NP; b++) put(g, false, j, b);
        if (j > g.t0)
          for (int b = 0; b < NP; b++) put(g, true, j - 1, b);
      }
    }
    if (c.abort) {  // copies may still be landing: a millisecond is far beyond any of them
      const long long t0 = cycles_now();
      while (cycles_now() - t0 < 2000000ll) {
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ loads, f32
    const int lt = tid - 288;
    // A thread takes 8-dim units of the rows lt/8, lt/8 + 32, ... of a tile: for K piece b the block b of all of
    // them, for V piece b every block of those in it.
    constexpr int RSTEP = LD / 8, NR = TC_KEYS / RSTEP, RV = VK / RSTEP;
    const int r0 = lt >> 3, u0 = lt & 7, swz = (u0 ^ (r0 & 7)) << 4;
    // unit i (of NR) of a piece: its row and its block, and its place in the piece
    auto unit_row = [&](bool is_v, int b, int i) { return is_v ? b * RV + i % RV : i; };
    auto unit_block = [&](bool is_v, int b, int i) { return is_v ? i / RV : b; };
    auto unit_at = [&](bool is_v, int i) {
      const int kr = r0 + (is_v ? i % RV : i) * RSTEP;
      return swz + (is_v ? (kr >> 4) * G_::VG + (i / RV) * 2048 + (kr & 15) * 128 : kr * 128);
    };
    constexpr uint32_t NONE = 0xffffffffu;
    uint32_t(*const rowoff)[TC_KEYS] = c.rowoff;
    // Rows of a tile's slots.  The table entries of a tile are read two tiles, and its rows are known one tile before
    // they are used, so that neither load is waited for.
    int entry = -1, page = -1;
    auto look = [&](const Seg &g, int tile) {
      const int sl = tile * TC_KEYS + lt;
      entry = -1;
      if constexpr (TREE) {
        if (tile < g.w1 && lt < TC_KEYS && sl < g.ts.n) {
          entry = (int)cwp_entry(a.kv.stride, a.kv.page_size, sl);
          if (entry >= 0) page = a.kv.table[(int64_t)g.s * a.kv.stride + entry];
        }
      }
    };
    auto note = [&](const Seg &g, int tile) {
      if (tile >= g.w1 || lt >= TC_KEYS) return;
      const int sl = tile * TC_KEYS + lt;
      uint32_t o = NONE;
      if constexpr (TREE) {
        if (sl < g.ts.n) {
          const int64_t x = entry < 0 ? -1 : cwp_row_in(page, entry, a.kv.n_pages, a.kv.page_size, sl);
          if (x >= 0) {
            o = (uint32_t)x;
          } else {
            c.bad = 1;
            atomicOr(a.err, OPE_PAGE);
          }
        }
      } else if (pbegin + sl < pend) {
        o = (uint32_t)(pbegin + sl);
      }
      rowoff[tile & 3][lt] = o;
    };
    // the row of unit i of a piece, and where the unit is
    auto row_at = [&](bool is_v, int tile, int b, int i) { return rowoff[tile & 3][r0 + unit_row(is_v, b, i) * RSTEP]; };
    auto source = [&](const Seg &g, bool is_v, uint32_t o, int b, int i) -> const T * {
      const int u = unit_block(is_v, b, i) * 64 + u0 * 8;
      if constexpr (TREE) return (const T *)(is_v ? a.kv.v : a.kv.k) + ((int64_t)o * a.nkv + g.hk) * HD + u;
      else return (const T *)(is_v ? a.v : a.k) + (int64_t)o * (is_v ? a.vrow : a.krow) + g.hk * (is_v ? a.vhead : a.khead) + u;
    };
    // to be called for the tiles [w0, w1) of a segment in order
    auto tile_rows = [&](const Seg &g, int tile) {
      if (tile == g.w0) {
        named_bar(4, LD);  // the segment before is through with rowoff
        if (TREE && g.ts.cut && lt == 0) atomicOr(a.err, OPE_PAGE);
        look(g, tile);
        note(g, tile);
        look(g, tile + 1);
      }
      note(g, tile + 1);
      look(g, tile + 2);
      named_bar(4, LD);
    };
    {
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
        if (pb == 0 && !is_v) tile_rows(g, pj);
        return true;
      };
      int slot = 0, par = 1;  // the first pass over the ring waits for nothing
      auto step = [&]() {
        if (++slot == NS) {
          slot = 0;
          par ^= 1;
        }
      };
      // a thread's four units of a piece are in registers; the next piece's are loaded while the MMAs take this one
      float x[4][8];
      unsigned gone = 0;  // units whose slot is not there: read from a row that is, made zero below
      auto load = [&]() {
        const int tile = is_v ? pj - 1 : pj;
        const float *src[4];
        gone = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t o = row_at(is_v, tile, pb, i);
          if (o == NONE) gone |= 1u << i;
          src[i] = (const float *)source(g, is_v, o == NONE ? (TREE ? 0 : pbegin) : o, pb, i);
        }
        if (a.vec == 2) {
#pragma unroll
          for (int i = 0; i < 4; i++) ld_global_f8(src[i], x[i]);
        } else if (a.vec) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            *(float4 *)x[i] = *(const float4 *)src[i];
            *(float4 *)(x[i] + 4) = *(const float4 *)(src[i] + 4);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 8; k++) x[i][k] = src[i][k];
        }
        if constexpr (TREE) {
          // one piece in registers does not cover the memory's latency: a 128-byte line a thread, of the tile that
          // comes next in K or in V, into the L2 (8 ragged sequences of 8 kv heads of 128, one token each 217 -> 198 us,
          // trees of 24 nodes 234 -> 227 us; the chain of 9 over 4 heads of 256 as before)
          if (tile + 1 < g.w1) {
            const uint32_t o = rowoff[(tile + 1) & 3][lt >> 1];
            if (o != NONE) {
              const float *line = (const float *)(is_v ? a.kv.v : a.kv.k) + ((int64_t)o * a.nkv + g.hk) * HD + (2 * pb + (lt & 1)) * 32;
              asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
            }
          }
        }
      };
      float fk = 1.f, fv = 1.f;
      bool have = advance();
      if (have) load();
      while (have) {
        const bool v = is_v, first = (v ? pj - 1 : pj) == g.t0 && pb == 0;
        const int wi = si & 7;
        have = advance();
        int e = 0;
        if (gone) {
#pragma unroll
          for (int i = 0; i < 4; i++)
            if ((gone >> i) & 1) {
#pragma unroll
              for (int k = 0; k < 8; k++) x[i][k] = 0.f;
            }
        }
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
        }
        fence_proxy_async_smem();  // waits for loads too: before the next ones
        mbar_arrive(&c.full[s_hi]);
        mbar_arrive(&c.full[s_lo]);
        if (have) load();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tm, 512);
  }
}

// Joins the parts of the rows whose slots were split over CTAs.  Grid
// (sequence, kv head, groups of `rows` rows); a CTA takes its rows one after
// another, its threads as groups of HD/4 that take every NG-th part of the row
// and four dims each, and adds the groups in order.
template <int TY, int HD>
__global__ void __launch_bounds__(256) tc_combine_kernel(const __grid_constant__ AttnOp a, int rows) {
  using T = typename TypeOf<TY>::T;
  constexpr int TG = HD / 4, NG = 256 / TG;
  __shared__ float w[TC_CTAS + 8];
  __shared__ float4 acc_s[256];
  __shared__ float red_m[8], red_l[8];
  pdl_trigger();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, s = blockIdx.x, hk = blockIdx.y, G = a.nh / a.nkv;
  const TreeSeq q = tree_seq(a, s);
  const int i0 = blockIdx.z * rows, i1 = min(q.live * G, i0 + rows);
  if (i0 >= i1) {
    pdl_wait();  // or a grid without rows would end before the kernel it follows
    return;
  }
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
  // first unit of CTA c: floor(total c / C)
  const int64_t tq = total / C;
  const int tr = (int)(total - tq * C);
  auto first_unit = [&](int cc) { return tq * cc + (tr * cc) / C; };
  pdl_wait();  // the lengths are older than the kernel before, which ends its own wait before this one starts
  int mt = -1, c0 = 0, c1 = 0;
  int64_t ua = 0;
  for (int item = i0; item < i1; item++) {
    if (item / TC_ROWS != mt) {
      mt = item / TC_ROWS;
      ua = before + (int64_t)(hk * mts + mt) * (nt + a.seg_cost) + a.seg_cost;  // the segment's first tile
      c0 = (int)(((ua + 1) * C - 1) / total);
      c1 = (int)(((ua + nt) * C - 1) / total);
    }
    if (c0 == c1) continue;  // written by its CTA
    const int r = item - mt * TC_ROWS, np = c1 - c0 + 1;
    // weight of part c0 + tid (an empty CTA has none; np <= TC_CTAS < 256)
    auto part_row = [&](int i) -> int64_t { return ((int64_t)(c0 + i) * 2 + (ua >= first_unit(c0 + i))) * a.part_rows + r; };
    float mp = -INFINITY, lp = 0.f;
    if (tid < np && first_unit(c0 + tid) != first_unit(c0 + tid + 1)) {
      const int64_t p = part_row(tid);
      mp = a.ml[2 * p];
      lp = a.ml[2 * p + 1];
    }
    const float mw = warp_max(mp);
    if (lane == 0) red_m[warp] = mw;
    __syncthreads();
    float m = red_m[0];
#pragma unroll
    for (int i = 1; i < 8; i++) m = fmaxf(m, red_m[i]);
    float wt = mp == -INFINITY ? 0.f : ex2(mp - m);
    if (lp != lp) wt = 1.f;
    if (tid < np) w[tid] = wt;
    const float lw = warp_sum(wt * lp);
    if (lane == 0) red_l[warp] = lw;
    __syncthreads();
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) l += red_l[i];
    const int g = tid / TG, d = (tid % TG) * 4;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = g; i < np; i += NG) {
      const float wi = w[i];
      if (wi != 0.f) {  // a part of no weight may never have been written
        const float4 x = *(const float4 *)(a.part + part_row(i) * HD + d);
        acc.x = fmaf(wi, x.x, acc.x);
        acc.y = fmaf(wi, x.y, acc.y);
        acc.z = fmaf(wi, x.z, acc.z);
        acc.w = fmaf(wi, x.w, acc.w);
      }
    }
    acc_s[tid] = acc;
    __syncthreads();
    const int t = item / G, h = hk * G + item - t * G;
    const int64_t row = (int64_t)s * a.T + t;
    bool bad = false;
    if (tid < TG) {
#pragma unroll
      for (int i = 1; i < NG; i++) {
        const float4 x = acc_s[tid + i * TG];
        acc.x += x.x;
        acc.y += x.y;
        acc.z += x.z;
        acc.w += x.w;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
      bad = !(l < INFINITY);
      T *o = (T *)a.o + row * a.orow + h * a.ohead + d;
#pragma unroll
      for (int i = 0; i < 4; i++) {
        bad |= !(fabsf(f[i]) < INFINITY);
        o[i] = from_f<T>(l == 0.f ? 0.f : f[i]);
      }
    }
    if (__syncthreads_or(bad) && warp == 0) exact_row<T, HD, true>(a, s, t, 0, (int)row, h);
  }
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

template <int TY, int HD>
cudaError_t configure_hd() {
  CW_TRY(cudaFuncSetAttribute(attn_tc_kernel<TY, HD, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<TY, HD>::SMEM));
  CW_TRY(cudaFuncSetAttribute(attn_tc_kernel<TY, HD, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo<TY, HD>::SMEM));
  return carveout_max(tc_combine_kernel<TY, HD>);
}

// Tensor maps of K and V; false where their rows cannot be addressed so.
template <int TY, int HD>
bool make_maps(CUtensorMap &mk, CUtensorMap &mv, const void *k, int64_t krow, int64_t khead, const void *v, int64_t vrow,
               int64_t vhead, int nkv, int n_rows, int kbox) {
  memset(&mk, 0, sizeof mk);
  memset(&mv, 0, sizeof mv);
  return TY != TY_F32 && kbox >= 16 && make_map(&mk, TY == TY_BF16, k, krow, khead, HD, nkv, n_rows, kbox, 1) &&
         make_map(&mv, TY == TY_BF16, v, vrow, vhead, HD, nkv, n_rows, 16, HD / 64);
}

template <int TY, int HD>
cudaError_t prompt_hd(AttnOp a, cudaStream_t st) {
  CUtensorMap mk, mv;
  using G = Geo<TY, HD>;
  const int64_t tiles = (int64_t)a.n_rows / TC_ROWS + a.n_seq;
  if (tiles * a.nh > 0x7fffffff) return cudaErrorInvalidConfiguration;
  const int al = TY == TY_F32 ? 4 : 8;
  a.vec = ((uintptr_t)a.k | (uintptr_t)a.v) % 16 == 0 && (a.krow | a.khead | a.vrow | a.vhead) % al == 0;
  if (a.vec && ((uintptr_t)a.k | (uintptr_t)a.v) % 32 == 0 && (a.krow | a.khead | a.vrow | a.vhead) % 8 == 0) a.vec = 2;
  const int kbox = make_maps<TY, HD>(mk, mv, a.k, a.krow, a.khead, a.v, a.vrow, a.vhead, a.nkv, a.n_rows, TC_KEYS) ? TC_KEYS : 0;
  return launch_pdl(attn_tc_kernel<TY, HD, false>, dim3((unsigned)(tiles * a.nh)), G::THREADS, G::SMEM, st, a, mk, mv, kbox);
}

template <int TY, int HD>
cudaError_t tree_hd(AttnOp a, cudaStream_t st) {
  CUtensorMap mk, mv;
  using G = Geo<TY, HD>;
  a.seg_cost = G::SEG_COST;
  a.vec = ((uintptr_t)a.kv.k | (uintptr_t)a.kv.v) % 32 == 0 ? 2 : 1;
  int kbox = a.kv.page_size & -a.kv.page_size;
  kbox = kbox > TC_KEYS ? TC_KEYS : kbox;
  const int64_t row = (int64_t)a.nkv * HD;
  if (!make_maps<TY, HD>(mk, mv, a.kv.k, row, HD, a.kv.v, row, HD, a.nkv, a.kv.n_pages * a.kv.page_size, kbox)) kbox = 0;
  CW_TRY(launch_pdl(attn_tc_kernel<TY, HD, true>, dim3(a.n_cta), G::THREADS, G::SMEM, st, a, mk, mv, kbox));
  if (tree_tiles(a.max_len) == 1) return cudaSuccess;  // no segment can be split
  // rows one after another in a CTA once there is more than a wave of them
  const int per = a.T * (a.nh / a.nkv);
  const int64_t want = ((int64_t)a.n_seq * a.nkv * per + 8 * a.n_cta - 1) / (8 * a.n_cta);
  const int rows = (int)(want < 1 ? 1 : want > per ? per : want);
  return launch_pdl(tc_combine_kernel<TY, HD>, dim3(a.n_seq, a.nkv, (per + rows - 1) / rows), 256, 0, st, a, rows);
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
