// pf_train.h -- operators of the training path: the layer-norm backward (pf_layernorm_bwd.cu),
// attention with a learned bias and its backward (pf_attention.cu), the relative-position bias and
// the gradient of its table (pf_relpos.cu).
#pragma once
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/pairformer_b200.h"
#include "pf_common.cuh"
#include "pf_tmap.h"

namespace pf {
namespace train {

// Lets kernel K take up to `most` bytes of dynamic shared memory, once per device. The limit is one per kernel and
// device for all host threads, so it is the largest that any call needs and never lowered: a limit set to each call's
// own size would fail another thread's larger launch.
template <auto K>
int room_for_shared(size_t most) {
  static std::atomic<unsigned long long> done{0};
  return once_per_device(done, [&]() -> int {
    PF_CUDA_TRY(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most));
    return PF_OK;
  });
}

size_t layernorm_bwd_ws_bytes(int64_t rows, int c, int dtype);
int layernorm_bwd(const void* x, const void* dy, const float* gamma, void* dx, float* dgamma, float* dbeta,
                  int64_t rows, int c, float eps, int dtype, void* ws, size_t ws_bytes, cudaStream_t st);

// Column sums of n rows of m values, in a fixed order: columns below m0 to out0, the others to out1.
int sum_rows(const float* part, int64_t n, int64_t m, float* out0, int64_t m0, float* out1, cudaStream_t st);

size_t attention_bwd_ws_bytes(const pf_attention_shape& s, bool shared_dbias);
int attention_fwd(const pf_attention_call& c, cudaStream_t st);
int attention_bwd(const pf_attention_call& c, void* ws, size_t ws_bytes, cudaStream_t st);

size_t relpos_bias_bwd_ws_bytes(int64_t n_rows, int64_t n_cols, int heads, int r_max, int s_max);
int relpos_bias(const void* w, int w_dtype, pf_token_ids ids, void* out, int64_t hs, int64_t rs, int dtype,
                int64_t row0, int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int r_max, int s_max,
                cudaStream_t st);
int relpos_bias_bwd(const void* dbias, int64_t hs, int64_t rs, int dtype, pf_token_ids ids, float* dw, int64_t row0,
                    int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int r_max, int s_max, void* ws,
                    size_t ws_bytes, cudaStream_t st);

}  // namespace train
}  // namespace pf
