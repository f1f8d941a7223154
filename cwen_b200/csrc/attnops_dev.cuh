// Device pieces shared by the attention operators' kernels: the call's
// description, what a row sees, and the slow exact row.
#pragma once
#include "attnops.cuh"
#include "sm100.cuh"

namespace cw {

struct AttnOp {
  KvView kv;                  // tree: the paged cache
  const void *k, *v;          // prompt: rows of k and v
  int64_t krow, khead, vrow, vhead;
  const void *q;
  int64_t qrow, qhead;
  void *o;
  int64_t orow, ohead;
  const int *cu, *len, *n_node;
  const uint64_t *mask;
  int n_seq, n_rows, T, max_len, nh, nkv;
  float scale;
  int vec;                    // prompt: k and v rows are 16-byte aligned
  float *part, *ml;           // tree: partial outputs and their (max, sum)
  int part_rows, n_cta, seg_cost;
  int *err;
};

// One sequence of a tree call, cut to what the call may read.
struct TreeSeq {
  int len;    // committed slots
  int live;   // nodes whose rows are computed
  int n;      // slots in all
  bool cut;   // a length was out of range
};
CW_DEV TreeSeq tree_seq(const AttnOp &a, int s) {
  TreeSeq r;
  const int len = a.len[s];
  r.live = a.n_node ? min(max(a.n_node[s], 0), a.T) : a.T;
  r.cut = r.live > 0 && (len < 0 || (int64_t)len + r.live > a.max_len);
  const int l0 = len < 0 ? 0 : len;
  r.n = (int)min((int64_t)l0 + r.live, (int64_t)a.max_len);
  r.len = min(l0, r.n);
  return r;
}
// Nodes that row t sees, among those with a slot.
CW_DEV uint64_t tree_bits(const AttnOp &a, const TreeSeq &q, int s, int t) {
  const int nodes = q.n - q.len;
  const uint64_t have = nodes >= 64 ? ~0ull : (1ull << nodes) - 1;
  return have & (a.mask ? a.mask[(int64_t)s * a.T + t] : (t == 63 ? ~0ull : (2ull << t) - 1));
}
// The rows [b, e) of sequence s of a packed prompt, cut to the rows there are.
CW_DEV void prompt_seq(const AttnOp &a, int s, int &b, int &e) {
  b = min(max(a.cu[s], 0), a.n_rows);
  e = min(max(a.cu[s + 1], b), a.n_rows);
}

// One row by one warp, every place that the row does not see left out by a
// select: what the tiled kernels fall back to for rows whose tile met a
// non-finite value (a masked place times a zero weight would be NaN) or a bad
// page id.  Chunks of 32 slots: scores one slot per lane, then the weighted
// sum one dim per lane and 32-dim slice.  s, t: tree; b: the first row of the
// row's sequence (prompt).  -> out[row][h]
template <class T, int HD, bool TREE>
__device__ __noinline__ void exact_row(const AttnOp &a, int s, int t, int b, int row, int h) {
  constexpr int DL = HD / 32;
  const int lane = threadIdx.x & 31, hk = h / (a.nh / a.nkv);
  TreeSeq ts = {};
  uint64_t bits = 0;
  int n;
  if constexpr (TREE) {
    ts = tree_seq(a, s);
    bits = tree_bits(a, ts, s, t);
    n = ts.n;
  } else {
    n = row - b + 1;
  }
  const T *q = (const T *)a.q + row * a.qrow + h * a.qhead;
  float m = -INFINITY, l = 0.f, acc[DL];
#pragma unroll
  for (int i = 0; i < DL; i++) acc[i] = 0.f;
  for (int c0 = 0; c0 < n; c0 += 32) {
    const int j = c0 + lane;
    bool see = j < n;
    const T *kp = nullptr, *vp = nullptr;
    if constexpr (TREE) {
      if (see && j >= ts.len) see = (bits >> (j - ts.len)) & 1;
      if (see) {
        const int64_t r = cwp_row(a.kv.table + (int64_t)s * a.kv.stride, a.kv.stride, a.kv.n_pages, a.kv.page_size, j);
        see = r >= 0;
        if (see) {
          kp = (const T *)a.kv.k + (r * a.nkv + hk) * HD;
          vp = (const T *)a.kv.v + (r * a.nkv + hk) * HD;
        }
      }
    } else if (see) {
      kp = (const T *)a.k + (int64_t)(b + j) * a.krow + hk * a.khead;
      vp = (const T *)a.v + (int64_t)(b + j) * a.vrow + hk * a.vhead;
    }
    float sc = -INFINITY;
    if (see) {
      float d0 = 0.f;
      for (int d = 0; d < HD; d++) d0 = fmaf(to_f<T>(q[d]), to_f<T>(kp[d]), d0);
      sc = d0 * a.scale;
    }
    const float mn = fmaxf(m, warp_max(sc));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float corr = m == -INFINITY ? 0.f : expf(m - ref);
    const float e = see ? expf(sc - ref) : 0.f;
    l = fmaf(l, corr, warp_sum(e));
    m = mn;
#pragma unroll
    for (int i = 0; i < DL; i++) acc[i] *= corr;
    const unsigned live = __ballot_sync(0xffffffffu, see);
    for (int t2 = 0; t2 < 32; t2++) {
      if (!((live >> t2) & 1)) continue;
      const float p = __shfl_sync(0xffffffffu, e, t2);
      const T *vv = (const T *)__shfl_sync(0xffffffffu, (unsigned long long)vp, t2);
#pragma unroll
      for (int i = 0; i < DL; i++) acc[i] = fmaf(p, to_f<T>(vv[lane + 32 * i]), acc[i]);
    }
  }
  T *o = (T *)a.o + row * a.orow + h * a.ohead;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int i = 0; i < DL; i++) o[lane + 32 * i] = from_f<T>(l == 0.f ? 0.f : acc[i] * inv);
}

CW_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace cw
