// Rotary positions and the row operations of the paged cache.
//
// rope: for pair i < n_rot/2 of every head of row r, with the angle
//   a = 2 pi pos[r] turn[i],
//   (x0, x1) -> mscale (x0 cos a - x1 sin a, x0 sin a + x1 cos a);
// the head's other dims are copied.  The angle's turns are reduced to
// [-1/2, 1/2] in 64 bits (positions reach millions of radians), sine and cosine and
// the rotation are fp32.
// append: the same rotation on K rows on their way into the pages, V beside it.
// compact: the rows of an accepted path move down to consecutive slots.
//
// All three are bound by HBM (short calls by their launch).  Measured on B200:
// rope of 16384 rows of 32 x 128 bf16 50 us (5.4 TB/s); append of 32768 rows of
// 4 x 256, f32 into bf16, 91 us (4.4 TB/s: the look-ups of place and angle come
// before a CTA's first store); compaction of 64 sequences in 16 bf16 layers 39 us
// (5.7 TB/s).  Many small CTAs with one unit per thread in flight beat fewer with
// four (110-130 us for the append).
#include <math.h>
#include <string.h>

#include "attnops.cuh"

namespace cw {

constexpr int RT = 256;          // threads per CTA
constexpr int ROPE_TAB = 2048;   // (cos, sin) pairs a CTA keeps: its rows x n_rot/2

// V elements at p as floats / back: one 16- or 32-byte access when V > 1.
template <class T, int V>
CW_DEV void load_v(const T *p, float (&f)[V]) {
  if constexpr (V == 1) {
    f[0] = to_f<T>(*p);
  } else {
    constexpr int N = V * (int)sizeof(T) / 16;
    uint4 u[N];
#pragma unroll
    for (int i = 0; i < N; i++) u[i] = reinterpret_cast<const uint4 *>(p)[i];
    const T *e = reinterpret_cast<const T *>(u);
#pragma unroll
    for (int i = 0; i < V; i++) f[i] = to_f<T>(e[i]);
  }
}
template <class T, int V>
CW_DEV void store_v(T *p, const float (&f)[V]) {
  if constexpr (V == 1) {
    *p = from_f<T>(f[0]);
  } else {
    constexpr int N = V * (int)sizeof(T) / 16;
    uint4 u[N];
    T *e = reinterpret_cast<T *>(u);
#pragma unroll
    for (int i = 0; i < V; i++) e[i] = from_f<T>(f[i]);
#pragma unroll
    for (int i = 0; i < N; i++) reinterpret_cast<uint4 *>(p)[i] = u[i];
  }
}

struct RowsArgs {
  const void *x, *x2;        // rows to rotate; append: K, and V beside it
  int64_t xrow, xhead, vrow, vhead;
  void *y, *y2;              // rope: rows; append: the layer's K and V pools
  int64_t yrow, yhead;
  const int *pos;
  int n_rows, n_head, dim;
  int n_rot, inverse, in_place;
  // append
  const int *seq, *slot, *table;
  int stride, n_seq, n_pages, page_size;
  int *err;
};

// One unit of a head: a pair of V-vectors (half layout, i and i + n_rot/2),
// or one V-vector (interleaved pairs, or dims that only pass).
template <class S, class D, int V, bool HALF, bool ROT>
CW_DEV void do_unit(const S *x, D *y, int j, int pu, int n_rot, const float2 *cs) {
  if (ROT && j < pu) {
    if constexpr (HALF) {
      const int d = j * V, n2 = n_rot >> 1;
      float a[V], b[V], ra[V], rb[V];
      load_v<S, V>(x + d, a);
      load_v<S, V>(x + d + n2, b);
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float2 w = cs[d + i];
        ra[i] = a[i] * w.x - b[i] * w.y;
        rb[i] = a[i] * w.y + b[i] * w.x;
      }
      store_v<D, V>(y + d, ra);
      store_v<D, V>(y + d + n2, rb);
    } else if constexpr (V == 1) {
      const float a = to_f<S>(x[2 * j]), b = to_f<S>(x[2 * j + 1]);
      const float2 w = cs[j];
      y[2 * j] = from_f<D>(a * w.x - b * w.y);
      y[2 * j + 1] = from_f<D>(a * w.y + b * w.x);
    } else {
      float a[V], r[V];
      load_v<S, V>(x + j * V, a);
#pragma unroll
      for (int i = 0; i < V; i += 2) {
        const float2 w = cs[(j * V + i) >> 1];
        r[i] = a[i] * w.x - a[i + 1] * w.y;
        r[i + 1] = a[i] * w.y + a[i + 1] * w.x;
      }
      store_v<D, V>(y + j * V, r);
    }
  } else {
    const int d = (ROT ? n_rot : 0) + (j - (ROT ? pu : 0)) * V;
    float a[V];
    load_v<S, V>(x + d, a);
    store_v<D, V>(y + d, a);
  }
}

// Units of one head: the rotated ones (pu) and all of them.
template <int V, bool HALF>
CW_HOST_DEV int pair_units(int n_rot) { return HALF ? n_rot / 2 / V : (V == 1 ? n_rot / 2 : n_rot / V); }

// Grid (row groups of rb rows, segments of a row's units).
template <class S, class D, int V, bool HALF, bool APPEND>
__global__ void __launch_bounds__(RT) rows_kernel(const __grid_constant__ RowsArgs a,
                                                  const __grid_constant__ cwen_rope rope, int rb) {
  pdl_trigger();
  pdl_wait();
  __shared__ float2 tab[ROPE_TAB];
  __shared__ int64_t dst[RT];
  const int r0 = blockIdx.x * rb, nr = min(rb, a.n_rows - r0), n2 = a.n_rot >> 1;
  for (int i = threadIdx.x; i < nr * n2; i += RT) {
    const int r = i / n2, p = i - r * n2;
    double t = (double)a.pos[r0 + r] * rope.turn[p];
    t -= rint(t);
    float s, c;
    sincospif((float)(2.0 * t), &s, &c);
    tab[i] = make_float2(c * rope.mscale, (a.inverse ? -s : s) * rope.mscale);
  }
  if constexpr (APPEND) {
    for (int r = threadIdx.x; r < nr; r += RT) {
      const int q = a.seq[r0 + r];
      int64_t row = -1;
      if (q >= 0 && q < a.n_seq)
        row = cwp_row(a.table + (int64_t)q * a.stride, a.stride, a.n_pages, a.page_size, a.slot[r0 + r]);
      if (row < 0 && q >= 0) atomicOr(a.err, OPE_PAGE);  // q < 0: a padding row
      dst[r] = row;
    }
  }
  __syncthreads();
  const int pu = pair_units<V, HALF>(a.n_rot);
  const int uh = a.in_place ? pu : pu + (a.dim - a.n_rot) / V;  // units of a rotated head
  const int vu = a.dim / V;                                      // append: units of a V head
  const int upr = a.n_head * (APPEND ? uh + vu : uh);
  const int seg = gridDim.y == 1 ? upr : (upr + gridDim.y - 1) / gridDim.y;
  const int u0 = blockIdx.y * seg, nu = min(seg, upr - u0);
  if (nu <= 0) return;
  for (int i = threadIdx.x; i < nr * nu; i += RT) {
    const int r = i / nu, u = u0 + i - r * nu;
    const float2 *cs = tab + r * n2;
    if constexpr (APPEND) {
      const int64_t row = dst[r];
      if (row < 0) continue;
      if (u < a.n_head * uh) {
        const int h = u / uh;
        do_unit<S, D, V, HALF, true>((const S *)a.x + (r0 + r) * a.xrow + h * a.xhead,
                                     (D *)a.y + (row * a.n_head + h) * a.dim, u - h * uh, pu, a.n_rot, cs);
      } else {
        const int w = u - a.n_head * uh, h = w / vu;
        do_unit<S, D, V, HALF, false>((const S *)a.x2 + (r0 + r) * a.vrow + h * a.vhead,
                                      (D *)a.y2 + (row * a.n_head + h) * a.dim, w - h * vu, 0, 0, nullptr);
      }
    } else {
      const int h = u / uh;
      do_unit<S, D, V, HALF, true>((const S *)a.x + (r0 + r) * a.xrow + h * a.xhead,
                                   (D *)a.y + (r0 + r) * a.yrow + h * a.yhead, u - h * uh, pu, a.n_rot, cs);
    }
  }
}

// Moves of one sequence's accepted path.  Bit i of the path (node u) goes
// from slot len + u to len + i <= len + u, so in path order no source lies
// behind a destination: a thread that owns one 16-byte column of the rows
// makes its moves in order, loads of a group before its stores.
// Sixteen moves in flight: 36 us where eight took 54 (64 sequences, 16 layers).
constexpr int CT = 128, CG = 16;  // threads of a CTA; moves of a group
__global__ void __launch_bounds__(CT) compact_kernel(uint4 *k, uint4 *v, int n_layer, int64_t layer_cols, int cols,
                                                     const int *table, int stride, int n_pages, int page_size,
                                                     const int *len, const uint64_t *keep, int *len_out, int *err) {
  pdl_trigger();
  pdl_wait();
  __shared__ int64_t src[64], dst[64];
  __shared__ int n_moves;
  const int s = blockIdx.x;
  const uint64_t m = keep[s];
  const int n = len[s], np = __popcll(m);
  if (threadIdx.x < 32) {
    int base = 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int u = h * 32 + threadIdx.x, i = __popcll(m & ((1ull << u) - 1));  // node, its place in the path
      bool mv = false;
      int64_t a = -1, b = -1;
      if (((m >> u) & 1) && u != i) {
        const int *row = table + (int64_t)s * stride;
        a = n < 0 ? -1 : cwp_row(row, stride, n_pages, page_size, (int64_t)n + u);
        b = n < 0 ? -1 : cwp_row(row, stride, n_pages, page_size, (int64_t)n + i);
        mv = a >= 0 && b >= 0;
        if (!mv) atomicOr(err, OPE_PAGE);
      }
      const unsigned bal = __ballot_sync(0xffffffffu, mv);
      if (mv) {
        const int at = base + __popc(bal & ((1u << threadIdx.x) - 1));
        src[at] = a * cols;
        dst[at] = b * cols;
      }
      base += __popc(bal);
    }
    if (threadIdx.x == 0) {
      n_moves = base;
      if (len_out && blockIdx.y == 0 && blockIdx.z == 0) len_out[s] = n + np;
    }
  }
  __syncthreads();
  const int c = blockIdx.z * CT + threadIdx.x;
  if (c >= cols) return;
  const int layer = blockIdx.y >> 1;
  uint4 *p = ((blockIdx.y & 1) ? v : k) + layer * layer_cols + c;
  const int nm = n_moves;
  for (int i = 0; i < nm; i += CG) {
    uint4 w[CG];
#pragma unroll
    for (int j = 0; j < CG; j++)
      if (i + j < nm) w[j] = p[src[i + j]];
#pragma unroll
    for (int j = 0; j < CG; j++)
      if (i + j < nm) p[dst[i + j]] = w[j];
  }
}

int check_kv(const char *fn, const cwen_kv *c) {
  if (!c || !type_ok(c->type) || c->n_layer < 1 || c->n_layer > 1024 || c->n_pages < 1 || c->page_size < 1 ||
      c->page_size > 65536 || c->n_kv < 1 || c->n_kv > 256 || c->head_dim < 8 || c->head_dim > 512 ||
      c->head_dim % 8 || !c->k || !c->v || ((uintptr_t)c->k | (uintptr_t)c->v) % 16) {
    set_error("%s: need a cache of type F32/F16/BF16, 1..1024 layers, pages of 1..65536 slots, 1..256 kv heads of "
              "8..512 dims (a multiple of 8), 16-byte aligned pools", fn);
    return CWEN_EINVAL;
  }
  return CWEN_OK;
}

namespace {

bool rope_ok(const cwen_rope *r, int dim) { return r->n_rot >= 2 && r->n_rot <= 256 && r->n_rot % 2 == 0 && r->n_rot <= dim; }

template <class S, class D, int V, bool HALF, bool APPEND>
cudaError_t launch_rows_t(const RowsArgs &a, const cwen_rope &r, cudaStream_t st) {
  const int pu = pair_units<V, HALF>(a.n_rot), uh = a.in_place ? pu : pu + (a.dim - a.n_rot) / V;
  const int upr = a.n_head * (APPEND ? uh + a.dim / V : uh);
  // about four units a thread, eight where the rows' places are looked up first (32768 rows of 4 heads of 256, f32 into
  // bf16: 99 us against 111 us; rope of 16384 rows: 60 us with eight, 56 us with four); a CTA's rows bounded by its angle table and by dst[]
  int rb = (APPEND ? 8 : 4) * RT / (upr > 0 ? upr : 1);
  const int cap = a.n_rot ? ROPE_TAB / (a.n_rot / 2) : RT;
  rb = rb < 1 ? 1 : (rb > cap ? cap : rb);
  if (rb > RT) rb = RT;
  int segs = 1;
  // few rows: spread the CTAs' work until every SM has some
  const int groups = (a.n_rows + rb - 1) / rb;
  if (rb == 1 || groups < engine().n_sm) {
    const int want = (int)(((int64_t)rb * upr + 2 * RT - 1) / (2 * RT));
    segs = want < 1 ? 1 : (want > 1024 ? 1024 : want);
  }
  return launch_pdl(rows_kernel<S, D, V, HALF, APPEND>, dim3(groups, segs), RT, 0, st, a, r, rb);
}
template <class S, class D, int VW, bool APPEND>
cudaError_t launch_rows(const RowsArgs &a, const cwen_rope &r, bool vec, cudaStream_t st) {
  if (r.half) return vec ? launch_rows_t<S, D, VW, true, APPEND>(a, r, st) : launch_rows_t<S, D, 1, true, APPEND>(a, r, st);
  return vec ? launch_rows_t<S, D, VW, false, APPEND>(a, r, st) : launch_rows_t<S, D, 1, false, APPEND>(a, r, st);
}

}  // namespace

cudaError_t kvops_configure() { return cudaSuccess; }

}  // namespace cw

using namespace cw;

extern "C" {

int cwen_rope_init(cwen_rope *r, int n_rot, int half, double base, double factor, double orig_ctx, double beta_fast,
                   double beta_slow) {
  const bool ramp = beta_fast != 0.0 || beta_slow != 0.0;
  if (!r || n_rot < 2 || n_rot > 256 || n_rot % 2 || !(base > 0.0) || !(factor > 0.0) || isinf(base) || isinf(factor) ||
      (ramp && !(orig_ctx > 0.0 && beta_slow >= 0.0 && beta_fast > beta_slow && factor >= 1.0))) {
    set_error("cwen_rope_init: need an even n_rot in [2,256], base and factor > 0; by parts: orig_ctx > 0, "
              "beta_fast > beta_slow >= 0, factor >= 1");
    return CWEN_EINVAL;
  }
  memset(r, 0, sizeof *r);
  r->n_rot = n_rot;
  r->half = half != 0;
  r->mscale = 1.0f;
  const double two_pi = 6.283185307179586476925286766559;
  for (int i = 0; i < n_rot / 2; i++) {
    double t = pow(base, -2.0 * i / n_rot) / two_pi;
    if (ramp) {
      double g = (t * orig_ctx - beta_slow) / (beta_fast - beta_slow);
      g = g < 0.0 ? 0.0 : (g > 1.0 ? 1.0 : g);
      t *= g + (1.0 - g) / factor;
    } else {
      t /= factor;
    }
    r->turn[i] = t;
  }
  if (ramp) r->mscale = (float)(0.1 * log(factor) + 1.0);
  return CWEN_OK;
}

int cwen_cuda_rope(const cwen_rope *r, int type, int n_rows, int n_head, int head_dim, const void *x, int64_t xrow,
                   int64_t xhead, const int *pos, int inverse, void *y, int64_t yrow, int64_t yhead, void *stream) {
  if (!r || !type_ok(type) || n_rows < 0 || n_head < 1 || n_head > 4096 || head_dim < 2 || head_dim > 512 ||
      !rope_ok(r, head_dim) || !x || !y || !pos) {
    set_error("cwen_cuda_rope: need F32/F16/BF16 rows of 1..4096 heads of 2..512 dims, an even n_rot <= head_dim, "
              "non-null buffers");
    return CWEN_EINVAL;
  }
  if (x == y && (xrow != yrow || xhead != yhead)) {
    set_error("cwen_cuda_rope: in place the strides of x and y must be equal");
    return CWEN_EINVAL;
  }
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_rope: engine not initialised");
    return CWEN_ESTATE;
  }
  if (n_rows == 0) return CWEN_OK;
  OpDevice dev;
  CW_CHECK(dev.err);
  const int es = type_size(type), V = 16 / es;
  RowsArgs a = {};
  a.x = x; a.xrow = xrow; a.xhead = xhead;
  a.y = y; a.yrow = yrow; a.yhead = yhead;
  a.pos = pos; a.n_rows = n_rows; a.n_head = n_head; a.dim = head_dim;
  a.n_rot = r->n_rot; a.inverse = inverse != 0; a.in_place = x == y;
  const int part = r->half ? r->n_rot / 2 : r->n_rot;
  const bool vec = part % V == 0 && head_dim % V == 0 && ((uintptr_t)x | (uintptr_t)y) % 16 == 0 &&
                   (xrow | xhead | yrow | yhead) % V == 0;
  cudaStream_t st = stream ? (cudaStream_t)stream : E.stream;
  if (type == CWEN_T_F32) CW_CHECK((launch_rows<float, float, 4, false>(a, *r, vec, st)));
  else if (type == CWEN_T_F16) CW_CHECK((launch_rows<__half, __half, 8, false>(a, *r, vec, st)));
  else CW_CHECK((launch_rows<__nv_bfloat16, __nv_bfloat16, 8, false>(a, *r, vec, st)));
  E.prof.launches++;
  return CWEN_OK;
}

int cwen_cuda_kv_append(const cwen_kv *c, int layer, const int *table, int table_stride, int n_seq, int type,
                        int n_rows, const void *k, int64_t krow, int64_t khead, const void *v, int64_t vrow,
                        int64_t vhead, const int *seq, const int *slot, const cwen_rope *r, const int *pos,
                        void *stream) {
  int rc = check_kv("cwen_cuda_kv_append", c);
  if (rc) return rc;
  if (layer < 0 || layer >= c->n_layer || !table || table_stride < 1 || n_seq < 1 || n_rows < 0 || !k || !v || !seq ||
      !slot || (type != c->type && type != CWEN_T_F32) || (r && !rope_ok(r, c->head_dim))) {
    set_error("cwen_cuda_kv_append: need a layer of the cache, a table, rows of the cache's type or F32, seq and slot "
              "of every row, an even n_rot <= head_dim");
    return CWEN_EINVAL;
  }
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_kv_append: engine not initialised");
    return CWEN_ESTATE;
  }
  if (n_rows == 0) return CWEN_OK;
  OpDevice dev;
  CW_CHECK(dev.err);
  const int ss = type_size(type), ds = type_size(c->type), V = 16 / ds;
  static const cwen_rope none = {};
  const cwen_rope &rp = r ? *r : none;
  RowsArgs a = {};
  a.x = k; a.xrow = krow; a.xhead = khead;
  a.x2 = v; a.vrow = vrow; a.vhead = vhead;
  const int64_t off = (int64_t)layer * kv_layer_rows(c) * c->n_kv * c->head_dim * ds;
  a.y = (char *)c->k + off; a.y2 = (char *)c->v + off;
  a.pos = pos ? pos : slot; a.n_rows = n_rows; a.n_head = c->n_kv; a.dim = c->head_dim;
  a.n_rot = r ? r->n_rot : 0;
  a.seq = seq; a.slot = slot; a.table = table; a.stride = table_stride; a.n_seq = n_seq;
  a.n_pages = c->n_pages; a.page_size = c->page_size; a.err = E.op_err;
  const int part = rp.half ? a.n_rot / 2 : a.n_rot, al = 16 / ss < V ? 16 / ss : V;
  const bool vec = part % V == 0 && ((uintptr_t)k | (uintptr_t)v) % 16 == 0 && (krow | khead | vrow | vhead) % al == 0;
  cudaStream_t st = stream ? (cudaStream_t)stream : E.stream;
  if (c->type == CWEN_T_F32) CW_CHECK((launch_rows<float, float, 4, true>(a, rp, vec, st)));
  else if (c->type == CWEN_T_F16) {
    if (type == CWEN_T_F32) CW_CHECK((launch_rows<float, __half, 8, true>(a, rp, vec, st)));
    else CW_CHECK((launch_rows<__half, __half, 8, true>(a, rp, vec, st)));
  } else {
    if (type == CWEN_T_F32) CW_CHECK((launch_rows<float, __nv_bfloat16, 8, true>(a, rp, vec, st)));
    else CW_CHECK((launch_rows<__nv_bfloat16, __nv_bfloat16, 8, true>(a, rp, vec, st)));
  }
  E.prof.launches++;
  return CWEN_OK;
}

int cwen_cuda_kv_compact(const cwen_kv *c, const int *table, int table_stride, int n_seq, const int *len,
                         const uint64_t *keep, int *len_out, void *stream) {
  int rc = check_kv("cwen_cuda_kv_compact", c);
  if (rc) return rc;
  if (!table || table_stride < 1 || n_seq < 0 || !len || !keep || len_out == len) {
    set_error("cwen_cuda_kv_compact: need a table, len and keep of every sequence, len_out not len");
    return CWEN_EINVAL;
  }
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_kv_compact: engine not initialised");
    return CWEN_ESTATE;
  }
  if (n_seq == 0) return CWEN_OK;
  OpDevice dev;
  CW_CHECK(dev.err);
  const int cols = c->n_kv * c->head_dim * type_size(c->type) / 16;
  cudaStream_t st = stream ? (cudaStream_t)stream : E.stream;
  CW_CHECK(launch_pdl(compact_kernel, dim3(n_seq, 2 * c->n_layer, (cols + CT - 1) / CT), CT, 0, st, (uint4 *)c->k,
                      (uint4 *)c->v, c->n_layer, kv_layer_rows(c) * cols, cols, table, table_stride, c->n_pages,
                      c->page_size, len, keep, len_out, E.op_err));
  E.prof.launches++;
  return CWEN_OK;
}

int cwen_cuda_attn_status(void *stream) {
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_attn_status: engine not initialised");
    return CWEN_ESTATE;
  }
  OpDevice dev;
  CW_CHECK(dev.err);
  cudaStream_t st = stream ? (cudaStream_t)stream : E.stream;
  int flag = 0;
  CW_CHECK(cudaMemcpyAsync(&flag, E.op_err, sizeof flag, cudaMemcpyDeviceToHost, st));
  CW_CHECK(cudaStreamSynchronize(st));
  if (!flag) return CWEN_OK;
  CW_CHECK(cudaMemsetAsync(E.op_err, 0, sizeof flag, st));
  CW_CHECK(cudaStreamSynchronize(st));
  if (flag & OPE_WAIT) {
    set_error("attention operators: a bounded device wait gave up");
    return CWEN_ETIMEOUT;
  }
  set_error("attention operators: a sequence, slot, length or page id was out of range (its rows were left out)");
  return CWEN_ERANGE;
}

}  // extern "C"
