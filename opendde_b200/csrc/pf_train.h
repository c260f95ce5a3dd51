// pf_train.h -- operators of the training path: the layer-norm backward (pf_layernorm_bwd.cu),
// attention with a learned bias and its backward (pf_attention.cu), the relative-position bias and
// the gradient of its table (pf_relpos.cu).
#pragma once
#include <cuda_runtime.h>
#include "../../include/pairformer_b200.h"

namespace pf {
namespace train {

size_t layernorm_bwd_ws_bytes(int64_t rows, int c, int dtype);
int layernorm_bwd(const void* x, const void* dy, const float* gamma, void* dx, float* dgamma, float* dbeta,
                  int64_t rows, int c, float eps, int dtype, void* ws, size_t ws_bytes, cudaStream_t st);

// out[i] = sum over n rows of part[row * m + i], in row order (fixed: the result does not depend on
// scheduling)
int sum_rows(const float* part, int64_t n, int64_t m, float* out, cudaStream_t st);

size_t attention_bwd_ws_bytes(const pf_attention_shape& s);
int attention_fwd(const pf_attention_shape& s, pf_head_view q, pf_head_view k, pf_head_view v, pf_bias_view bias,
                  pf_mask_view mask, pf_head_view o, float* stats, int16_t* o_lo, cudaStream_t st);
int attention_bwd(const pf_attention_shape& s, pf_head_view q, pf_head_view k, pf_head_view v, pf_bias_view bias,
                  pf_mask_view mask, pf_head_view o, const float* stats, const int16_t* o_lo, pf_head_view d_o,
                  pf_head_view dq, pf_head_view dk, pf_head_view dv, pf_bias_view dbias, void* ws, size_t ws_bytes,
                  cudaStream_t st);

size_t relpos_bias_bwd_ws_bytes(int64_t n_rows, int64_t n_cols, int heads, int r_max, int s_max);
int relpos_bias(const void* w, int w_dtype, pf_token_ids ids, void* out, int64_t hs, int64_t rs, int dtype,
                int64_t row0, int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int r_max, int s_max,
                cudaStream_t st);
int relpos_bias_bwd(const void* dbias, int64_t hs, int64_t rs, int dtype, pf_token_ids ids, float* dw, int64_t row0,
                    int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int r_max, int s_max, void* ws,
                    size_t ws_bytes, cudaStream_t st);

}  // namespace train
}  // namespace pf
