// pf_attention_bf16.cu -- the bf16 kernels of pf_attention.cuh.
#include "pf_attention.cuh"

namespace pf {
namespace train {
namespace attn {
int launch_bf16(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st) {
  return launch_dim<__nv_bfloat16>(kind, a, blocks, flops, st);
}
int rows_bf16(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st) {
  return launch_rows<__nv_bfloat16>(a, stats, o, lo, rows, st);
}
}  // namespace attn
}  // namespace train
}  // namespace pf
