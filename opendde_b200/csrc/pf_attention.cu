// pf_attention.cu -- host side of attention with a learned bias (kernels: pf_attention.cuh).
#include "pf_attention.cuh"

namespace pf {
namespace train {
namespace {

using attn::Args;
using attn::Heads;

int launch(int dtype, attn::Kind kind, const Args& a, double flops, cudaStream_t st) {
  return dtype == PF_BF16 ? attn::launch_bf16(kind, a, flops, st) : attn::launch_f32(kind, a, flops, st);
}

template <int BT>
__global__ void __launch_bounds__(256) k_sum_planes(Args a, const float* __restrict__ part, int parts) {
  const int64_t n = (int64_t)a.H * a.nq * a.nk;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
    for (int p = 0; p < parts; ++p) s += part[p * n + i];
    const int64_t j = i % a.nk, hi = i / a.nk, h = hi / a.nq, q = hi - h * a.nq;
    const int64_t off = h * a.db_hs + q * a.db_rs + j;
    if (BT == 2)
      ((float*)a.dbias)[off] = s;
    else
      ((__nv_bfloat16*)a.dbias)[off] = __float2bfloat16_rn(s);
  }
}

int sum_planes(const Args& a, const float* part, int parts, cudaStream_t st) {
  const int64_t n = (int64_t)a.H * a.nq * a.nk, want = (n + 255) / 256;
  const unsigned blocks = (unsigned)(want < 148 * 8 ? want : 148 * 8);
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_sum_planes", 4.0 * n * (parts + 1), 'b');
    if (a.bias_f32)
      k_sum_planes<2><<<blocks, 256, 0, st>>>(a, part, parts);
    else
      k_sum_planes<1><<<blocks, 256, 0, st>>>(a, part, parts);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// How the gradient of a shared bias is computed: with dq in one pass (bf16: one block of 16 warps per SM; fp32:
// three blocks of four, or two above 256 keys), or by itself (as many blocks as run at a time), in `parts` parts
// of the batch.
struct SharedPlan {
  bool plane;
  int parts;
};
// Parts of at least four entries each for `blocks` blocks per part of which `fit` run at a time: the fewest waves
// of blocks per part (512 tokens, four heads, bf16: 9 parts of 32 blocks fill two waves to 97 %, 4 parts one to
// 86 %; 900 tokens: 480 blocks in one part would be two waves for the work of one), against what a part costs,
// a plane written and read and a block's first entry, about two and a half entries' work. `time`: in units
// of the work on a full machine.
int best_parts(int64_t blocks, int64_t fit, int64_t batch, double* time) {
  const int64_t most = batch / 4 < 1 ? 1 : batch / 4, cap = fit / blocks > 16 ? fit / blocks : 16;
  int best = 1;
  for (int64_t n = 1; n <= most && n <= cap; ++n) {
    const double waves = (double)((blocks * n + fit - 1) / fit);
    const double t = waves * fit / (double)(blocks * n) + (n > 1 ? 2.5 * n / (double)batch : 0.0);
    if (n == 1 || t < *time) *time = t, best = (int)n;
  }
  return best;
}
SharedPlan shared_plan(const pf_attention_shape& s) {
  if (s.n_q == 0 || s.n_k == 0 || s.batch == 0) return SharedPlan{false, 1};
  const bool bf16 = s.dtype == PF_BF16;
  double time = 0.0;
  if (bf16 ? attn::dq_plane_bf16_fits(s.n_k, s.head_dim) : attn::dq_plane_f32_fits(s.n_k, s.head_dim)) {
    const int fit = 148 * (bf16 ? 1 : (s.n_k <= 256 ? 3 : 2));
    const int n = best_parts((s.n_q + 63) / 64 * s.heads, fit, s.batch, &time);
    // where most of the machine would stay idle, the two passes are faster
    if (time < 1.7) return SharedPlan{true, n};
  }
  // tiles of the kernels and how many blocks an SM holds
  const int64_t rows = bf16 ? 128 : 64, keys = bf16 || s.head_dim <= 32 ? 64 : (s.head_dim <= 64 ? 32 : 16);
  const int64_t blocks = ((s.n_q + rows - 1) / rows) * ((s.n_k + keys - 1) / keys) * s.heads;
  return SharedPlan{false, best_parts(blocks, (s.head_dim <= 32 ? (bf16 ? 3 : 4) : 1) * 148, s.batch, &time)};
}

Heads heads(const pf_head_view& v) { return Heads{v.ptr, v.batch_stride, v.seq_stride, v.head_stride}; }

// 16-byte accesses: the base, every stride and the channels are whole 16-byte units
int whole16(const pf_head_view& v, const pf_attention_shape& s) {
  const int64_t e = s.dtype == PF_F32 ? 4 : 8;
  return (uintptr_t)v.ptr % 16 == 0 && v.batch_stride % e == 0 && v.seq_stride % e == 0 && v.head_stride % e == 0 &&
         s.head_dim % e == 0;
}

// four neighbouring keys as one access
int whole_quads(const pf_bias_view& v, int dtype) {
  return (uintptr_t)v.ptr % (dtype == PF_F32 ? 16 : 8) == 0 && v.batch_stride % 4 == 0 && v.head_stride % 4 == 0 &&
         v.row_stride % 4 == 0;
}

Args make_args(const pf_attention_call& c) {
  const pf_attention_shape& s = c.shape;
  const pf_head_view &q = c.q, &k = c.k, &v = c.v;
  const pf_bias_view& bias = c.bias;
  const pf_mask_view& mask = c.mask;
  Args a{};
  a.q = heads(q);
  a.k = heads(k);
  a.v = heads(v);
  a.vec_q = whole16(q, s);
  a.vec_k = whole16(k, s);
  a.vec_v = whole16(v, s);
  a.bias = bias.ptr;
  a.b_bs = bias.batch_stride;
  a.b_hs = bias.head_stride;
  a.b_rs = bias.row_stride;
  a.bias_f32 = s.bias_dtype == PF_F32;
  a.bias_vec = whole_quads(bias, s.bias_dtype);
  a.mask = mask.ptr;
  a.m_bs = mask.row_stride;
  a.m_ks = mask.col_stride;
  a.B = s.batch;
  a.nq = s.n_q;
  a.nk = s.n_k;
  a.H = s.heads;
  a.KV = s.kv_heads;
  a.d = s.head_dim;
  a.scale = s.scale;
  a.rows_plane = s.batch * s.heads * s.n_q;
  return a;
}

}  // namespace

int attention_fwd(const pf_attention_call& c, cudaStream_t st) {
  const pf_attention_shape& s = c.shape;
  Args a = make_args(c);
  a.o = c.o.ptr;
  a.o_bs = c.o.batch_stride;
  a.o_ns = c.o.seq_stride;
  a.o_hs = c.o.head_stride;
  a.stats = c.stats;
  a.o_lo = (int16_t*)c.o_lo;
  return launch(s.dtype, attn::kFwd, a, 4.0 * s.batch * s.heads * s.n_q * s.n_k * s.head_dim, st);
}

// The row constants (16 bytes per row), then the partial planes of a gradient that is summed over the batch.
size_t attention_bwd_ws_bytes(const pf_attention_shape& s, bool shared_dbias) {
  Arena ar(nullptr, 0);
  ar.take<float>((size_t)4 * s.batch * s.heads * s.n_q);
  if (shared_dbias && s.batch > 1) {
    const int parts = shared_plan(s).parts;
    if (parts > 1) ar.take<float>((size_t)parts * s.heads * s.n_q * s.n_k);
  }
  return ar.used;
}

int attention_bwd(const pf_attention_call& c, void* ws, size_t ws_bytes, cudaStream_t st) {
  const pf_attention_shape& s = c.shape;
  const pf_head_view &dq = c.dq, &dk = c.dk, &dv = c.dv;
  const pf_bias_view& dbias = c.dbias;
  Args a = make_args(c);
  a.g = heads(c.d_o);
  a.vec_g = whole16(c.d_o, s);
  Arena ar(ws, ws_bytes);
  float* rows = ar.take<float>((size_t)4 * a.rows_plane);
  a.rows = rows;
  const double pair = 2.0 * s.batch * s.heads * s.n_q * s.n_k * s.head_dim;
  if (a.rows_plane > 0)
    PF_TRY(s.dtype == PF_BF16 ? attn::rows_bf16(a, c.stats, heads(c.o), (const int16_t*)c.o_lo, rows, st)
                              : attn::rows_f32(a, c.stats, heads(c.o), rows, st));
  const bool shared = dbias.ptr && s.batch > 1 && dbias.batch_stride == 0;
  if (dbias.ptr) {
    a.db_bs = dbias.batch_stride;
    a.db_hs = dbias.head_stride;
    a.db_rs = dbias.row_stride;
    a.db_vec = whole_quads(dbias, s.bias_dtype);
  }
  if (dk.ptr) {
    a.dk = dk.ptr;
    a.dk_bs = dk.batch_stride;
    a.dk_ns = dk.seq_stride;
    a.dk_hs = dk.head_stride;
    a.dv = dv.ptr;
    a.dv_bs = dv.batch_stride;
    a.dv_ns = dv.seq_stride;
    a.dv_hs = dv.head_stride;
  }
  a.dq = dq.ptr;
  a.o_bs = dq.batch_stride;
  a.o_ns = dq.seq_stride;
  a.o_hs = dq.head_stride;
  const bool sum = shared && s.n_q > 0 && s.n_k > 0;
  const SharedPlan plan = sum ? shared_plan(s) : SharedPlan{false, 1};
  a.dbias = shared ? nullptr : dbias.ptr;
  const bool by_rows = (dq.ptr || a.dbias) && !plan.plane;
  if (by_rows || dk.ptr)
    PF_TRY(launch(s.dtype, !by_rows ? attn::kDkv : (dk.ptr ? attn::kDqDkv : attn::kDq), a,
                  (by_rows ? 3 * pair : 0.0) + (dk.ptr ? 4 * pair : 0.0), st));
  if (!sum) return PF_OK;
  a.dbias = dbias.ptr;
  float* part = plan.parts > 1 ? ar.take<float>((size_t)plan.parts * s.heads * s.n_q * s.n_k) : nullptr;
  if (!ar.ok()) return fail(PF_EWORKSPACE, "attention backward: workspace too small");
  if (plan.plane)
    PF_TRY(s.dtype == PF_BF16 ? attn::dq_plane_bf16(a, part, plan.parts, 3 * pair, st)
                              : attn::dq_plane_f32(a, part, plan.parts, 3 * pair, st));
  else
    PF_TRY(s.dtype == PF_BF16 ? attn::dbias_bf16(a, part, plan.parts, 2 * pair, st)
                              : attn::dbias_f32(a, part, plan.parts, 2 * pair, st));
  if (plan.parts > 1) return sum_planes(a, part, plan.parts, st);
  return PF_OK;
}

}  // namespace train
}  // namespace pf
