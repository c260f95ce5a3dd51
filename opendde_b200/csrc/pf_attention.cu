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

Args make_args(const pf_attention_shape& s, pf_head_view q, pf_head_view k, pf_head_view v, pf_bias_view bias,
               pf_mask_view mask) {
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

int attention_fwd(const pf_attention_shape& s, pf_head_view q, pf_head_view k, pf_head_view v, pf_bias_view bias,
                  pf_mask_view mask, pf_head_view o, float* stats, int16_t* o_lo, cudaStream_t st) {
  Args a = make_args(s, q, k, v, bias, mask);
  a.o = o.ptr;
  a.o_bs = o.batch_stride;
  a.o_ns = o.seq_stride;
  a.o_hs = o.head_stride;
  a.stats = stats;
  a.o_lo = o_lo;
  a.p_terms = bias.ptr && s.bias_dtype == PF_F32 ? 3 : 2;
  const double pair = 2.0 * s.batch * s.heads * s.n_q * s.n_k * s.head_dim;
  return launch(s.dtype, attn::kFwd, a, 2 * pair, st);
}

// The row constants (16 bytes per row), then the partial planes of a shared bias's gradient. Sized as if
// the bias were shared: a caller need not say.
size_t attention_bwd_ws_bytes(const pf_attention_shape& s) {
  Arena ar(nullptr, 0);
  ar.take<float>((size_t)4 * s.batch * s.heads * s.n_q);
  if (s.dtype == PF_BF16 && s.batch > 1) {
    const int parts = attn::dbias_parts_bf16(s.batch, s.n_q, s.n_k, s.heads);
    if (parts > 1) ar.take<float>((size_t)parts * s.heads * s.n_q * s.n_k);
  }
  return ar.used;
}

int attention_bwd(const pf_attention_shape& s, pf_head_view q, pf_head_view k, pf_head_view v, pf_bias_view bias,
                  pf_mask_view mask, pf_head_view o, const float* stats, const int16_t* o_lo, pf_head_view d_o,
                  pf_head_view dq, pf_head_view dk, pf_head_view dv, pf_bias_view dbias, void* ws,
                  size_t ws_bytes, cudaStream_t st) {
  Args a = make_args(s, q, k, v, bias, mask);
  a.g = heads(d_o);
  a.vec_g = whole16(d_o, s);
  Arena ar(ws, ws_bytes);
  float* rows = ar.take<float>((size_t)4 * a.rows_plane);
  a.rows = rows;
  const double pair = 2.0 * s.batch * s.heads * s.n_q * s.n_k * s.head_dim;
  if (a.rows_plane > 0)
    PF_TRY(s.dtype == PF_BF16 ? attn::rows_bf16(a, stats, heads(o), o_lo, rows, st)
                              : attn::rows_f32(a, stats, heads(o), rows, st));
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
    PF_TRY(launch(s.dtype, attn::kDkv, a, 4 * pair, st));
  }
  if (dq.ptr || (dbias.ptr && !shared)) {
    a.dq = dq.ptr;
    a.o_bs = dq.batch_stride;
    a.o_ns = dq.seq_stride;
    a.o_hs = dq.head_stride;
    a.dbias = shared ? nullptr : dbias.ptr;
    PF_TRY(launch(s.dtype, attn::kDq, a, 3 * pair, st));
  }
  if (shared && s.n_q > 0 && s.n_k > 0) {
    a.dbias = dbias.ptr;
    if (s.dtype == PF_F32) return attn::dbias_f32(a, 2 * pair, st);
    const int parts = attn::dbias_parts_bf16(s.batch, s.n_q, s.n_k, s.heads);
    float* part = parts > 1 ? ar.take<float>((size_t)parts * s.heads * s.n_q * s.n_k) : nullptr;
    if (!ar.ok()) return fail(PF_EWORKSPACE, "attention backward: workspace too small");
    return attn::dbias_bf16(a, part, parts, 2 * pair, st);
  }
  return PF_OK;
}

}  // namespace train
}  // namespace pf
