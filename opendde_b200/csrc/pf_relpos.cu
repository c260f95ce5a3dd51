// pf_relpos.cu -- the relative-position bias of attention heads and the gradient of its table.
//
// With the feature columns of a token pair (pf_relp.cuh: residue offset, token offset, same entity,
// symmetry-copy offset; each offset clipped to a bucket)
//   out[h, i, j] = W[h, res] + W[h, tok] + W[h, sym] + [same entity] W[h, ent]
//   dW[h, f]     = sum over the pairs (i, j) whose column f is set of dout[h, i, j]
// Both passes move the [H, rows, cols] plane once and are bound by that. A lane owns one column j
// and a warp walks down rows i, for kHeads heads at a time, so the indices of a pair are computed
// once for all of them. Down a column the buckets change rarely: the residue offset inside the
// window of 2 r_max + 1 rows around j, the others at chain ends. The forward keeps the current sums
// in registers and reads the table (shared memory) only when a column index changes; the backward
// adds runs of equal buckets in registers and flushes them when an index changes.
//
// The flush adds into the warp's own table in shared memory. Lanes that meet in one bucket are
// ordered by __match_any_sync and add one after the other, then the warps' tables and the blocks'
// partial tables are added in a fixed order: no atomics, equal inputs give equal bits.

#include "pf_common.cuh"
#include "pf_prof.h"
#include "pf_relp.cuh"
#include "pf_train.h"

namespace pf {
namespace train {
namespace {

constexpr int kRelWarps = 8;
constexpr int kRelRows = 64;  // rows of a block at most (their ids lie in shared memory)

struct RelArgs {
  pf_token_ids ids;
  int64_t row0, n_rows, col0, n_cols;
  int64_t hs, rs;  // head and row stride of the plane
  int heads, R, S, n_feat, rows_per_block;
};

struct TokId {
  int asym, res, ent, tok, sym;
};

__device__ __forceinline__ TokId load_id(const pf_token_ids& p, int64_t i) {
  return TokId{p.asym_id[i], p.residue_index[i], p.entity_id[i], p.token_index[i], p.sym_id[i]};
}

// a - b clipped to [-lim, lim], plus lim; the difference saturates, so no pair of ids wraps around
__device__ __forceinline__ int clip_diff(int a, int b, int lim) {
  int d;
  asm("sub.sat.s32 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return min(max(d, -lim), lim) + lim;
}

// The columns of one pair: the residue column, and the others packed (token column, symmetry column,
// same-entity bit; each column is below 2^12).
__device__ __forceinline__ void pair_cols(const TokId& i, const TokId& j, int R, int S, int& res, int& rest) {
  const bool chain = i.asym == j.asym, ent = i.ent == j.ent;
  res = chain ? clip_diff(i.res, j.res, R) : 2 * R + 1;
  const int tok = 2 * R + 2 + ((chain && i.res == j.res) ? clip_diff(i.tok, j.tok, R) : 2 * R + 1);
  const int sym = 4 * R + 5 + (ent ? clip_diff(i.sym, j.sym, S) : 2 * S + 1);
  rest = tok | (sym << 12) | ((ent ? 1 : 0) << 24);
}

template <class TW, class T, int G>
__global__ void __launch_bounds__(kRelWarps * 32) k_relpos_bias(RelArgs a, const TW* __restrict__ w, T* out) {
  extern __shared__ float tab[];  // [G][n_feat]
  __shared__ TokId rid[kRelRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = blockIdx.z * G, nh = min(G, a.heads - h0);
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_per_block;
  const int nr = (int)min((int64_t)a.rows_per_block, a.n_rows - r0);
  for (int i = threadIdx.x; i < G * a.n_feat; i += blockDim.x)
    tab[i] = i < nh * a.n_feat ? to_f(w[(int64_t)h0 * a.n_feat + i]) : 0.f;
  for (int i = threadIdx.x; i < nr; i += blockDim.x) rid[i] = load_id(a.ids, a.row0 + r0 + i);
  __syncthreads();
  const int64_t j = ((int64_t)blockIdx.x * kRelWarps + warp) * 32 + lane;
  if (j >= a.n_cols) return;
  const TokId cid = load_id(a.ids, a.col0 + j);
  int cur_res = -1, cur_rest = -1;
  float rest_v[G], val[G];
#pragma unroll
  for (int g = 0; g < G; ++g) rest_v[g] = val[g] = 0.f;
  T* o = out + (int64_t)h0 * a.hs + r0 * a.rs + j;
  for (int i = 0; i < nr; ++i, o += a.rs) {
    int res, rest;
    pair_cols(rid[i], cid, a.R, a.S, res, rest);
    if (res != cur_res || rest != cur_rest) {
      if (rest != cur_rest) {
        const int tok = rest & 0xfff, sym = (rest >> 12) & 0xfff;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float* t = tab + g * a.n_feat;
          rest_v[g] = t[tok] + t[sym] + ((rest >> 24) ? t[4 * a.R + 4] : 0.f);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) val[g] = tab[g * a.n_feat + res] + rest_v[g];
      cur_res = res;
      cur_rest = rest;
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (g < nh) o[(int64_t)g * a.hs] = from_f<T>(val[g]);
  }
}

// Adds each lane's G values to column f of the warp's table; lanes with pred == false add nothing.
// Every lane of the warp takes part.
template <int G>
__device__ __forceinline__ void flush(float* tab, int n_feat, bool pred, int f, const float* v) {
  const unsigned live = __ballot_sync(0xffffffffu, pred);
  if (live == 0) return;
  const unsigned same = __match_any_sync(0xffffffffu, pred ? f : -1);
  const unsigned lane = threadIdx.x & 31;
  const int rank = pred ? __popc(same & ((1u << lane) - 1u)) : 0;
  const int last = __reduce_max_sync(0xffffffffu, rank);
  for (int r = 0; r <= last; ++r) {
    if (pred && rank == r) {
#pragma unroll
      for (int g = 0; g < G; ++g) tab[g * n_feat + f] += v[g];
    }
    __syncwarp();
  }
}

template <class T, int G>
__global__ void __launch_bounds__(kRelWarps * 32) k_relpos_bias_bwd(RelArgs a, const T* __restrict__ dout,
                                                                    float* part) {
  extern __shared__ float tab[];  // [kRelWarps][G][n_feat]
  __shared__ TokId rid[kRelRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = blockIdx.z * G, nh = min(G, a.heads - h0);
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_per_block;
  const int nr = (int)min((int64_t)a.rows_per_block, a.n_rows - r0);
  const int per_warp = G * a.n_feat;
  for (int i = threadIdx.x; i < kRelWarps * per_warp; i += blockDim.x) tab[i] = 0.f;
  for (int i = threadIdx.x; i < nr; i += blockDim.x) rid[i] = load_id(a.ids, a.row0 + r0 + i);
  __syncthreads();
  float* mine = tab + warp * per_warp;
  const int64_t j = ((int64_t)blockIdx.x * kRelWarps + warp) * 32 + lane;
  const bool live = j < a.n_cols;
  const TokId cid = load_id(a.ids, a.col0 + (live ? j : 0));
  int cur_res = 0, cur_rest = 0;
  pair_cols(rid[0], cid, a.R, a.S, cur_res, cur_rest);
  // run: the sum since the residue column last changed; all: since the others last changed, without run
  float run[G], all[G];
#pragma unroll
  for (int g = 0; g < G; ++g) run[g] = all[g] = 0.f;
  auto flush_rest = [&](bool pred) {
    flush<G>(mine, a.n_feat, pred, cur_rest & 0xfff, all);
    flush<G>(mine, a.n_feat, pred, (cur_rest >> 12) & 0xfff, all);
    flush<G>(mine, a.n_feat, pred && (cur_rest >> 24), 4 * a.R + 4, all);
  };
  const T* p = dout + (int64_t)h0 * a.hs + r0 * a.rs + (live ? j : 0);
  constexpr int U = 4;  // rows in flight
  for (int i0 = 0; i0 < nr; i0 += U) {
    T x[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < G; ++g)
        x[u][g] = (live && i0 + u < nr && g < nh) ? p[(int64_t)(i0 + u) * a.rs + (int64_t)g * a.hs] : from_f<T>(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u < nr) {  // the same for the whole warp
        int res, rest;
        pair_cols(rid[i0 + u], cid, a.R, a.S, res, rest);
        const bool new_res = live && res != cur_res, new_rest = live && rest != cur_rest;
        if (__any_sync(0xffffffffu, new_res || new_rest)) {
          const bool out = new_res || new_rest;
          flush<G>(mine, a.n_feat, out, cur_res, run);
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (out) {
              all[g] += run[g];
              run[g] = 0.f;
            }
          if (__any_sync(0xffffffffu, new_rest)) {
            flush_rest(new_rest);
#pragma unroll
            for (int g = 0; g < G; ++g)
              if (new_rest) all[g] = 0.f;
          }
          cur_res = res;
          cur_rest = rest;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) run[g] += to_f(x[u][g]);
      }
    }
  }
  flush<G>(mine, a.n_feat, live, cur_res, run);
#pragma unroll
  for (int g = 0; g < G; ++g) all[g] += run[g];
  flush_rest(live);
  __syncthreads();
  // [row chunk x column strip][head][feature]
  float* dst = part + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * a.heads * a.n_feat + (int64_t)h0 * a.n_feat;
  for (int i = threadIdx.x; i < nh * a.n_feat; i += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kRelWarps; ++w) s += tab[w * per_warp + i];
    dst[i] = s;
  }
}

struct RelGrid {
  int G, rows_per_block;
  int64_t strips, chunks, groups;
};

// Four heads at a time where eight warps' tables for them fit in 64 KB of shared memory (r_max up to
// about 125), else one. Row chunks: about four blocks per SM, and not so short that the tables'
// zeroing and adding outweigh the rows.
RelGrid plan(int64_t n_rows, int64_t n_cols, int heads, int n_feat) {
  RelGrid p;
  p.G = n_feat <= 512 ? 4 : 1;
  p.strips = (n_cols + kRelWarps * 32 - 1) / (kRelWarps * 32);
  p.groups = (heads + p.G - 1) / p.G;
  const int64_t want = (148 * 4 + p.strips * p.groups - 1) / (p.strips * p.groups);
  int64_t per = (n_rows + want - 1) / want;
  per = per < 16 ? 16 : (per > kRelRows ? kRelRows : per);
  p.rows_per_block = (int)per;
  p.chunks = (n_rows + per - 1) / per;
  return p;
}

RelArgs rel_args(const RelGrid& p, pf_token_ids ids, int64_t row0, int64_t n_rows, int64_t col0, int64_t n_cols,
                 int64_t hs, int64_t rs, int heads, int R, int S) {
  return RelArgs{ids, row0, n_rows, col0, n_cols, hs, rs, heads, R, S, relp_n_feat(R, S), p.rows_per_block};
}

int check_grid(const RelGrid& p) {
  if (p.strips > 0x7fffffffll || p.chunks > 65535 || p.groups > 65535)
    return fail(PF_EUNSUPPORTED, "relative-position bias: tile too large");
  return PF_OK;
}

template <class TW, class T, int G>
int launch_fwd(const RelGrid& p, const RelArgs& a, const void* w, void* out, cudaStream_t st) {
  const size_t smem = (size_t)G * a.n_feat * sizeof(float);
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_relpos_bias", (double)a.heads * a.n_rows * a.n_cols * sizeof(T), 'b');
    k_relpos_bias<TW, T, G><<<dim3((unsigned)p.strips, (unsigned)p.chunks, (unsigned)p.groups), kRelWarps * 32, smem,
                              st>>>(a, (const TW*)w, (T*)out);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

template <class T, int G>
int launch_bwd(const RelGrid& p, const RelArgs& a, const void* dout, float* part, cudaStream_t st) {
  const size_t smem = (size_t)kRelWarps * G * a.n_feat * sizeof(float);
  auto* kern = k_relpos_bias_bwd<T, G>;
  if (smem > 40 * 1024)
    PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_relpos_bias_bwd", (double)a.heads * a.n_rows * a.n_cols * sizeof(T), 'b');
    kern<<<dim3((unsigned)p.strips, (unsigned)p.chunks, (unsigned)p.groups), kRelWarps * 32, smem, st>>>(
        a, (const T*)dout, part);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

}  // namespace

int relpos_bias(const void* w, int w_dtype, pf_token_ids ids, void* out, int64_t hs, int64_t rs, int dtype,
                int64_t row0, int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int R, int S,
                cudaStream_t st) {
  const RelGrid p = plan(n_rows, n_cols, heads, relp_n_feat(R, S));
  PF_TRY(check_grid(p));
  const RelArgs a = rel_args(p, ids, row0, n_rows, col0, n_cols, hs, rs, heads, R, S);
#define PF_REL(TW, T) return p.G == 4 ? launch_fwd<TW, T, 4>(p, a, w, out, st) : launch_fwd<TW, T, 1>(p, a, w, out, st)
  if (w_dtype == PF_F32) {
    if (dtype == PF_F32) PF_REL(float, float);
    PF_REL(float, __nv_bfloat16);
  }
  if (dtype == PF_F32) PF_REL(__nv_bfloat16, float);
  PF_REL(__nv_bfloat16, __nv_bfloat16);
#undef PF_REL
}

// One partial table per block of a head group; none where one block covers the tile.
size_t relpos_bias_bwd_ws_bytes(int64_t n_rows, int64_t n_cols, int heads, int R, int S) {
  if (n_rows == 0 || n_cols == 0) return 0;
  const RelGrid p = plan(n_rows, n_cols, heads, relp_n_feat(R, S));
  const int64_t n = p.strips * p.chunks;
  return n == 1 ? 0 : (size_t)n * heads * relp_n_feat(R, S) * sizeof(float);
}

int relpos_bias_bwd(const void* dbias, int64_t hs, int64_t rs, int dtype, pf_token_ids ids, float* dw, int64_t row0,
                    int64_t n_rows, int64_t col0, int64_t n_cols, int heads, int R, int S, void* ws, size_t,
                    cudaStream_t st) {
  const int n_feat = relp_n_feat(R, S);
  const RelGrid p = plan(n_rows, n_cols, heads, n_feat);
  PF_TRY(check_grid(p));
  const RelArgs a = rel_args(p, ids, row0, n_rows, col0, n_cols, hs, rs, heads, R, S);
  const int64_t n = p.strips * p.chunks;
  float* part = n == 1 ? dw : (float*)ws;
  if (dtype == PF_F32)
    PF_TRY((p.G == 4 ? launch_bwd<float, 4>(p, a, dbias, part, st) : launch_bwd<float, 1>(p, a, dbias, part, st)));
  else
    PF_TRY((p.G == 4 ? launch_bwd<__nv_bfloat16, 4>(p, a, dbias, part, st)
                     : launch_bwd<__nv_bfloat16, 1>(p, a, dbias, part, st)));
  return n == 1 ? PF_OK : sum_rows(part, n, (int64_t)heads * n_feat, dw, st);
}

}  // namespace train
}  // namespace pf
