// Attention over packed prompts and over drafted trees on a paged cache.
//
//   o = sum_j p_j v_j,  p_j = exp(scale q.k_j - m) / sum, over the slots j the
// row sees: j <= i inside its sequence (prompt), or the committed slots and
// the nodes of its mask (tree).  A row that sees nothing gives zeros.
//
// First form: one warp per (row, head) with an online softmax over chunks of
// 32 slots, one slot per lane for the scores, then one slice of dims per lane
// for the weighted sum.
#include "attn_tc.cuh"

namespace cw {

template <class T, int HD, bool TREE>
__global__ void __launch_bounds__(128) attn_simple_kernel(const __grid_constant__ AttnOp a) {
  pdl_trigger();
  pdl_wait();
  const int64_t item = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int64_t n_items = (int64_t)(TREE ? a.n_seq * a.T : a.n_rows) * a.nh;
  if (item >= n_items) return;
  const int row = (int)(item / a.nh), h = (int)(item % a.nh);
  if constexpr (TREE) {
    const int s = row / a.T, t = row % a.T;
    const TreeSeq q = tree_seq(a, s);
    if (t >= q.live) return;
    bool bad = q.cut;
    for (int j = (threadIdx.x & 31) * a.kv.page_size; !bad && j < q.n; j += 32 * a.kv.page_size)
      bad = cwp_row(a.kv.table + (int64_t)s * a.kv.stride, a.kv.stride, a.kv.n_pages, a.kv.page_size, j) < 0;
    if (bad) atomicOr(a.err, OPE_PAGE);
    __syncwarp();
    exact_row<T, HD, true>(a, s, t, 0, row, h);
  } else {
    int lo = 0, hi = a.n_seq;  // the last sequence that begins at or before the row
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= row) lo = mid;
      else hi = mid;
    }
    int b, e;
    prompt_seq(a, lo, b, e);
    if (row < b || row >= e) return;
    exact_row<T, HD, false>(a, 0, 0, b, row, h);
  }
}

template <class T, bool TREE>
cudaError_t launch_simple(const AttnOp &a, int hd, cudaStream_t st) {
  const int64_t items = (int64_t)(TREE ? a.n_seq * a.T : a.n_rows) * a.nh;
  const dim3 grid((unsigned)((items + 3) / 4));
  if (hd == 64) return launch_pdl(attn_simple_kernel<T, 64, TREE>, grid, 128, 0, st, a);
  if (hd == 128) return launch_pdl(attn_simple_kernel<T, 128, TREE>, grid, 128, 0, st, a);
  return launch_pdl(attn_simple_kernel<T, 256, TREE>, grid, 128, 0, st, a);
}
template <bool TREE>
cudaError_t launch_attn_op(const AttnOp &a, int type, int hd, cudaStream_t st) {
  if (type == CWEN_T_F32) return launch_simple<float, TREE>(a, hd, st);
  return TREE ? tc_tree(a, type == CWEN_T_BF16, hd, st) : tc_prompt(a, type == CWEN_T_BF16, hd, st);
}

static bool heads_ok(int nh, int nkv, int hd) {
  return nkv >= 1 && nkv <= 256 && nh >= nkv && nh <= 4096 && nh % nkv == 0 && (hd == 64 || hd == 128 || hd == 256);
}

// Rows of one part of a split row tile.
static int part_rows(int T, int G) {
  const int64_t n = (int64_t)T * G;
  return n >= TC_ROWS ? TC_ROWS : (int)(n + 3) / 4 * 4;
}

cudaError_t attnops_configure() { return tc_configure(); }

}  // namespace cw

using namespace cw;

extern "C" {

int cwen_cuda_attn_prompt(int type, int n_seq, const int *cu, int n_rows, int n_head, int n_kv, int head_dim,
                          float scale, const void *q, int64_t qrow, int64_t qhead, const void *k, int64_t krow,
                          int64_t khead, const void *v, int64_t vrow, int64_t vhead, void *out, int64_t orow,
                          int64_t ohead, void *stream) {
  if (!type_ok(type) || n_seq < 0 || n_seq > 65535 || n_rows < 0 || !heads_ok(n_head, n_kv, head_dim) || !cu || !q ||
      !k || !v || !out) {
    set_error("cwen_cuda_attn_prompt: need F32/F16/BF16, at most 65535 sequences, n_head a multiple of n_kv, head_dim "
              "64, 128 or 256, non-null buffers");
    return CWEN_EINVAL;
  }
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_attn_prompt: engine not initialised");
    return CWEN_ESTATE;
  }
  if (n_seq == 0 || n_rows == 0) return CWEN_OK;
  OpDevice dev;
  CW_CHECK(dev.err);
  AttnOp a = {};
  a.k = k; a.v = v; a.krow = krow; a.khead = khead; a.vrow = vrow; a.vhead = vhead;
  a.q = q; a.qrow = qrow; a.qhead = qhead; a.o = out; a.orow = orow; a.ohead = ohead;
  a.cu = cu; a.n_seq = n_seq; a.n_rows = n_rows; a.nh = n_head; a.nkv = n_kv; a.scale = scale; a.err = E.op_err;
  CW_CHECK((launch_attn_op<false>(a, type, head_dim, stream ? (cudaStream_t)stream : E.stream)));
  E.prof.launches++;
  return CWEN_OK;
}

size_t cwen_cuda_attn_tree_ws(const cwen_kv *c, int n_seq, int T, int n_head) {
  (void)n_seq;  // the parts of a call are counted by CTAs, not by sequences
  if (!c || T < 1 || n_head < 1 || c->n_kv < 1 || c->head_dim < 1) return 0;
  return (size_t)TC_CTAS * 2 * part_rows(T, n_head / c->n_kv) * (c->head_dim + 2) * sizeof(float);
}

int cwen_cuda_attn_tree(const cwen_kv *c, int layer, const int *table, int table_stride, int n_seq, const int *len,
                        int max_len, int T, const int *n_node, const uint64_t *mask, int n_head, float scale,
                        const void *q, int64_t qrow, int64_t qhead, void *out, int64_t orow, int64_t ohead, void *ws,
                        size_t ws_bytes, void *stream) {
  int rc = check_kv("cwen_cuda_attn_tree", c);
  if (rc) return rc;
  if (layer < 0 || layer >= c->n_layer || !table || table_stride < 1 || n_seq < 0 || n_seq > 65535 || !len || T < 1 ||
      T > 64 || max_len < 1 || max_len > (1 << 30) || max_len > (int64_t)table_stride * c->page_size ||
      !heads_ok(n_head, c->n_kv, c->head_dim) || kv_layer_rows(c) > 0x7fffffff || !q || !out) {
    set_error("cwen_cuda_attn_tree: need a layer of the cache, a table, 1 <= T <= 64, 1 <= max_len <= table_stride * "
              "page_size, n_head a multiple of n_kv, head_dim 64, 128 or 256, fewer than 2^31 slots, non-null buffers");
    return CWEN_EINVAL;
  }
  if (!ws || ws_bytes < cwen_cuda_attn_tree_ws(c, n_seq, T, n_head) || (uintptr_t)ws % 16) {
    set_error("cwen_cuda_attn_tree: the workspace needs %zu bytes, 16-byte aligned",
              cwen_cuda_attn_tree_ws(c, n_seq, T, n_head));
    return CWEN_EINVAL;
  }
  Engine &E = engine();
  if (!E.live) {
    set_error("cwen_cuda_attn_tree: engine not initialised");
    return CWEN_ESTATE;
  }
  if (n_seq == 0) return CWEN_OK;
  OpDevice dev;
  CW_CHECK(dev.err);
  AttnOp a = {};
  const int64_t off = (int64_t)layer * kv_layer_rows(c) * c->n_kv * c->head_dim * type_size(c->type);
  a.kv.k = (const char *)c->k + off; a.kv.v = (const char *)c->v + off;
  a.kv.table = table; a.kv.stride = table_stride; a.kv.n_pages = c->n_pages; a.kv.page_size = c->page_size;
  a.q = q; a.qrow = qrow; a.qhead = qhead; a.o = out; a.orow = orow; a.ohead = ohead;
  a.len = len; a.n_node = n_node; a.mask = mask; a.n_seq = n_seq; a.T = T; a.max_len = max_len;
  a.nh = n_head; a.nkv = c->n_kv; a.scale = scale; a.err = E.op_err;
  a.part_rows = part_rows(T, n_head / c->n_kv);
  a.n_cta = E.n_sm < TC_CTAS ? E.n_sm : TC_CTAS;
  a.part = (float *)ws;
  a.ml = a.part + (size_t)TC_CTAS * 2 * a.part_rows * c->head_dim;
  CW_CHECK((launch_attn_op<true>(a, c->type, c->head_dim, stream ? (cudaStream_t)stream : E.stream)));
  E.prof.launches++;
  return CWEN_OK;
}

}  // extern "C"
