// Shared pieces of the attention operators on caller buffers (kvops.cu,
// attnops.cu): type conversion, the cache view a kernel takes by value,
// argument checks.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "engine.cuh"
#include "kvpage.h"

namespace cw {

// ---- element types ----
template <class T> CW_DEV float to_f(T v);
template <> CW_DEV float to_f<float>(float v) { return v; }
template <> CW_DEV float to_f<__half>(__half v) { return __half2float(v); }
template <> CW_DEV float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> CW_DEV T from_f(float v);
template <> CW_DEV float from_f<float>(float v) { return v; }
template <> CW_DEV __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> CW_DEV __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

inline int type_size(int t) { return t == CWEN_T_F32 ? 4 : 2; }
inline bool type_ok(int t) { return t == CWEN_T_F32 || t == CWEN_T_F16 || t == CWEN_T_BF16; }

// One layer of a cache pool and the table of its sequences.
struct KvView {
  const void *k, *v;  // the layer's [n_pages * page_size][n_kv][head_dim]
  const int *table;
  int stride, n_pages, page_size;
};

// Bits of the operators' device flag (Engine::op_err).
enum { OPE_PAGE = 1, OPE_WAIT = 2 };

// Runs a call on the engine's device, whatever the caller's current device is.
struct OpDevice {
  int prev = -1;
  cudaError_t err;
  OpDevice() {
    err = cudaGetDevice(&prev);
    if (err == cudaSuccess && prev != engine().device) err = cudaSetDevice(engine().device);
  }
  ~OpDevice() {
    if (prev >= 0 && prev != engine().device) cudaSetDevice(prev);
  }
};

// CWEN_OK, or CWEN_EINVAL with the message set.
int check_kv(const char *fn, const cwen_kv *c);
inline int64_t kv_layer_rows(const cwen_kv *c) { return (int64_t)c->n_pages * c->page_size; }

cudaError_t kvops_configure();
cudaError_t attnops_configure();

}  // namespace cw
