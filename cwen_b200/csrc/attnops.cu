// Attention over packed prompts and over drafted trees on a paged cache: the C
// ABI (include/cwen_cuda.h).  The kernels are in attn_tc.cu.
#include "attn_tc.cuh"

namespace cw {

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
  CW_CHECK(tc_prompt(a, type, head_dim, stream ? (cudaStream_t)stream : E.stream));
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
  CW_CHECK(tc_tree(a, c->type, c->head_dim, stream ? (cudaStream_t)stream : E.stream));
  E.prof.launches++;
  return CWEN_OK;
}

}  // extern "C"
