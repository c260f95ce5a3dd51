// pf_attention_f32.cu -- the f32 kernels of pf_attention.cuh.
#include "pf_attention.cuh"

namespace pf {
namespace train {
namespace attn {
int launch_f32(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st) {
  return launch_dim<float>(kind, a, blocks, flops, st);
}
int rows_f32(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st) {
  return launch_rows<float>(a, stats, o, lo, rows, st);
}
}  // namespace attn
}  // namespace train
}  // namespace pf
