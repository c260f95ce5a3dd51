// pf_attention.cuh -- attention with a learned bias, forward and backward: the plan and what its parts
// share. Kernels: pf_attention_bf16.cu (tensor cores) and pf_attention_f32.cu; host: pf_attention.cu.
//
// For one batch entry b and head h (key head h / (H / KV)), with t_ij = scale q_i.k_j + bias_ij over
// the keys j that the mask leaves:
//   m_i = max_j t_ij,  l_i = sum_j exp(t_ij - m_i),  p_ij = exp(t_ij - m_i) / l_i,  o_i = sum_j p_ij v_j
//   D_i = do_i.o_i,  dp_ij = do_i.v_j,  ds_ij = p_ij (dp_ij - D_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i,  dbias = ds
// The forward is one pass over the keys with the running m and l. It keeps m and l (not m + log l:
// next to a bias of the type's lowest value log l would be lost) and, for bf16, the low half of o.
// The backward recomputes p from them tile by tile, so no [n_q, n_k] array but dbias is written:
//   rows   D and the row constants of p
//   dkv    one block per key tile, loops over the query heads of its key head and their queries
//   dq     one block per query tile, loops over the keys: dq, and dbias where it is no sum
//   dbias  a bias shared by the batch: one block per tile of the [n_q, n_k] plane loops over the batch
//          and adds ds in registers, so the sum has a fixed order and needs no atomics
//
// Precision: scores, softmax statistics, D, accumulators and the sum over a shared bias's batch are fp32
// in both storage types. bf16: in the backward p and ds are multiplied as sums of two
// bf16 values, so that a gradient is rounded once, to its own type. ds is a difference of dp and D, so an error of o
// would be its largest: the forward multiplies p as a sum of two bf16 values (three where the bias is
// fp32, whose gradient then keeps fp32's accuracy), D is formed from o before its rounding, and for
// that the forward keeps the 16 bits of o that the rounding dropped.
//
// Rows: a row that sees no key has m = -inf, l = 0; its o and gradients are 0. Masked keys are never
// read (their rows are zero-filled and their columns set to -inf), so NaN there does no harm. Where one
// key has all of a row's weight in fp32 (l and its p are exactly 1) its ds is set to 0, which it is to
// within 2^-24 of dp: a row with one visible key has no score gradient, and dp - D would leave rounding
// noise in its place.
#pragma once

#include "pf_common.cuh"
#include "pf_prof.h"
#include "pf_train.h"

namespace pf {
namespace train {
namespace attn {

constexpr int kThreads = 128;  // of a block

struct Heads {  // element (b, n, h, e) at p + b*bs + n*ns + h*hs + e
  const void* p;
  int64_t bs, ns, hs;
};

struct Args {
  Heads q, k, v, g;  // g: do
  void *o, *dq, *dk, *dv, *dbias;
  int64_t o_bs, o_ns, o_hs;  // o in the forward; the first gradient's strides otherwise
  int64_t dk_bs, dk_ns, dk_hs, dv_bs, dv_ns, dv_hs;
  const void* bias;
  int64_t b_bs, b_hs, b_rs;     // bias strides (batch stride 0: shared)
  int64_t db_bs, db_hs, db_rs;  // dbias strides
  int bias_f32, bias_vec, db_vec;  // storage, and whether groups of four keys are aligned
  const float* mask;
  int64_t m_bs, m_ks;
  float* stats;         // forward: m [B][H][n_q], then l
  int16_t* o_lo;        // [B][n_q][H][d]
  const float* rows;    // backward: four row constants for each of [B][H][n_q]
  int64_t rows_plane;   // B * H * n_q
  int64_t B, nq, nk;
  int H, KV, d;
  float scale;
  int vec_q, vec_k, vec_v, vec_g;  // 16-byte accesses allowed
  int64_t tiles;                   // tiles along the split axis of this launch
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool ok) {
  const int n = ok ? 16 : 0;  // the rest is zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

enum Kind { kFwd, kDq, kDkv, kDqDkv };

// One translation unit per storage type. launch_*: the forward, dq (with dbias of one batch entry per
// plane where a.dbias is set), dk and dv, or all three; dbias_*: the gradient of a shared bias, from `parts` partial
// planes [parts][H][n_q][n_k] in `part` where parts > 1; rows_*: the row constants, 16 bytes per row.
int launch_bf16(Kind kind, const Args& a, double flops, cudaStream_t st);
int launch_f32(Kind kind, const Args& a, double flops, cudaStream_t st);
int dbias_bf16(const Args& a, float* part, int parts, double flops, cudaStream_t st);
int dbias_f32(const Args& a, float* part, int parts, double flops, cudaStream_t st);
// dq and the gradient of a shared bias in one pass, where it fits; parts as for dbias_*
bool dq_plane_bf16_fits(int64_t nk, int d);
bool dq_plane_f32_fits(int64_t nk, int d);
int dq_plane_f32(const Args& a, float* part, int parts, double flops, cudaStream_t st);
int dq_plane_bf16(const Args& a, float* part, int parts, double flops, cudaStream_t st);
int rows_bf16(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st);
int rows_f32(const Args& a, const float* stats, Heads o, float* rows, cudaStream_t st);

}  // namespace attn
}  // namespace train
}  // namespace pf
