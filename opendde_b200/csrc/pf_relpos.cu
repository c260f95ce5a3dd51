// pf_relpos.cu -- the relative-position bias of attention heads and the gradient of its table.
//
// With the feature columns of a token pair (pf_relp.cuh: residue offset, token offset, same entity,
// symmetry-copy offset; each offset clipped to a bucket)
//   out[h, i, j] = W[h, res] + W[h, tok] + W[h, sym] + [same entity] W[h, ent]
//   dW[h, f]     = sum over the pairs (i, j) whose column f is set of dout[h, i, j]
// Both passes move the [H, rows, cols] plane once and are bound by that. A lane owns one column j
// and a warp walks down rows i, for up to eight heads at a time, so the indices of a pair are computed
// once for all of them. Down a column the buckets change rarely: the residue offset inside the
// window of 2 r_max + 1 rows around j, the others at chain ends. The forward keeps the current sums
// in registers and reads the table (shared memory) only when a column index changes; the backward
// adds runs of equal buckets in registers and flushes them when an index changes.
//
// The flush adds into the warp's own table in shared memory. Lanes that meet in one bucket are
// ordered by __match_any_sync and add one after the other, then the warps' tables and the blocks'
// partial tables are added in a fixed order: no atomics, equal inputs give equal bits. 1536 tokens, 16
// heads, fp32: forward 36 us (4.2 TB/s), backward 85 us (the warps on the diagonal flush every row).

#include "pf_common.cuh"
#include "pf_prof.h"
#include "pf_relp.cuh"
#include "pf_train.h"

namespace pf {
namespace train {
namespace {

constexpr int kRelWarps = 8;
constexpr int kRelWaves = 4;
constexpr int kRelRows = 64;  // rows of a block at most (their ids lie in shared memory)

struct RelArgs {
  pf_token_ids ids;
  int64_t row0, n_rows, col0, n_cols;
  int64_t hs, rs;  // head and row stride of the plane
  int heads, R, S, n_feat, rows_per_block;
};

struct PairCols {
  int res, tok, sym;  // feature columns; sym carries the same-entity bit above them
};
constexpr int kEntBit = 1 << 16;  // above every column (at most 2048)
__device__ __forceinline__ PairCols pair_cols(const RelpIds& i, const RelpIds& j, int R, int S) {
  const RelpIndex x = relp_index(i, j, R, S);
  return PairCols{x.res, x.tok, x.chn + (x.same_ent ? kEntBit : 0)};
}

template <class TW, class T, int G>
__global__ void __launch_bounds__(kRelWarps * 32) k_relpos_bias(RelArgs a, const TW* __restrict__ w, T* out) {
  extern __shared__ float tab[];  // [G][n_feat]
  __shared__ RelpIds rid[kRelRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = blockIdx.z * G, nh = min(G, a.heads - h0);
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_per_block;
  const int nr = (int)min((int64_t)a.rows_per_block, a.n_rows - r0);
  for (int i = threadIdx.x; i < G * a.n_feat; i += blockDim.x)
    tab[i] = i < nh * a.n_feat ? to_f(w[(int64_t)h0 * a.n_feat + i]) : 0.f;
  for (int i = threadIdx.x; i < nr; i += blockDim.x) rid[i] = relp_ids(a.ids, a.row0 + r0 + i);
  __syncthreads();
  const int64_t j = ((int64_t)blockIdx.x * kRelWarps + warp) * 32 + lane;
  if (j >= a.n_cols) return;
  const RelpIds cid = relp_ids(a.ids, a.col0 + j);
  PairCols cur{-1, -1, -1};
  float rest_v[G], val[G];
#pragma unroll
  for (int g = 0; g < G; ++g) rest_v[g] = val[g] = 0.f;
  T* o = out + (int64_t)h0 * a.hs + r0 * a.rs + j;
  for (int i = 0; i < nr; ++i, o += a.rs) {
    const PairCols p = pair_cols(rid[i], cid, a.R, a.S);
    const bool new_rest = p.tok != cur.tok || p.sym != cur.sym;
    if (p.res != cur.res || new_rest) {
      if (new_rest) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float* t = tab + g * a.n_feat;
          rest_v[g] = t[p.tok] + t[p.sym & (kEntBit - 1)] + (p.sym & kEntBit ? t[4 * a.R + 4] : 0.f);
        }
      }
#pragma unroll
      for (int g = 0; g < G; ++g) val[g] = tab[g * a.n_feat + p.res] + rest_v[g];
      cur = p;
    }
#pragma unroll
    for (int g = 0; g < G; ++g)
      if (g < nh) o[(int64_t)g * a.hs] = from_f<T>(val[g]);
  }
}

// tab[g][f] += v[g]: all reads before the writes, which the compiler cannot know to be apart
template <int G>
__device__ __forceinline__ void add_column(float* tab, int n_feat, int f, const float* v) {
  float t[G];
#pragma unroll
  for (int g = 0; g < G; ++g) t[g] = tab[g * n_feat + f];
#pragma unroll
  for (int g = 0; g < G; ++g) tab[g * n_feat + f] = t[g] + v[g];
}

// Adds each lane's G values to column f of the warp's table; lanes with pred == false add nothing.
// Every lane of the warp takes part. Lanes that share a column add in lane order, or (all of them in
// one column: clipped offsets, other chains) through a butterfly.
template <int G>
__device__ __forceinline__ void flush(float* tab, int n_feat, bool pred, int f, const float* v) {
  const unsigned live = __ballot_sync(0xffffffffu, pred);
  if (live == 0) return;
  const unsigned lane = threadIdx.x & 31, before = live & ((1u << lane) - 1u);
  const bool head = before == 0;  // the first of them, where pred
  const int prev = __shfl_sync(0xffffffffu, f, head ? lane : 31 - __clz(before));
  const unsigned starts = __ballot_sync(0xffffffffu, pred && (head || f != prev));
  if ((starts & (starts - 1)) == 0) {  // one column for all
    float s[G];
#pragma unroll
    for (int g = 0; g < G; ++g) s[g] = warp_sum(pred ? v[g] : 0.f);
    if (pred && head) add_column<G>(tab, n_feat, f, s);
    __syncwarp();
    return;
  }
  int rank;  // among the lanes of its column
  if (__all_sync(0xffffffffu, !pred || head || f <= prev) || __all_sync(0xffffffffu, !pred || head || f >= prev)) {
    // In order, as down a chain: lanes of one column are neighbours. (Matching 32 different columns
    // against each other takes many times as long.)
    const int start = 31 - __clz(starts & (0xffffffffu >> (31 - lane)));
    rank = __popc(before) - __popc(live & ((1u << (start & 31)) - 1u));
    if (live == 0xffffffffu) {  // sums of neighbours, then one add per column
      float s[G];
#pragma unroll
      for (int g = 0; g < G; ++g) s[g] = v[g];
      for (int d = 1; __any_sync(0xffffffffu, rank >= d); d <<= 1) {
        const bool same = __shfl_down_sync(0xffffffffu, start, d) == start && lane + d < 32;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const float o = __shfl_down_sync(0xffffffffu, s[g], d);
          if (same) s[g] += o;
        }
      }
      if (rank == 0) add_column<G>(tab, n_feat, f, s);
      __syncwarp();
      return;
    }
  } else {
    const unsigned same = __match_any_sync(0xffffffffu, pred ? f : -1);
    rank = __popc(same & ((1u << lane) - 1u));
  }
  for (int r = 0; __any_sync(0xffffffffu, pred && rank >= r); ++r) {
    if (pred && rank == r) add_column<G>(tab, n_feat, f, v);
    __syncwarp();
  }
}

template <class T, int G>
__global__ void __launch_bounds__(kRelWarps * 32) k_relpos_bias_bwd(RelArgs a, const T* __restrict__ dout,
                                                                    float* part) {
  extern __shared__ float tab[];  // [kRelWarps][G][n_feat]
  __shared__ RelpIds rid[kRelRows];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int h0 = blockIdx.z * G, nh = min(G, a.heads - h0);
  const int64_t r0 = (int64_t)blockIdx.y * a.rows_per_block;
  const int nr = (int)min((int64_t)a.rows_per_block, a.n_rows - r0);
  const int per_warp = G * a.n_feat;
  for (int i = threadIdx.x; i < kRelWarps * per_warp; i += blockDim.x) tab[i] = 0.f;
  for (int i = threadIdx.x; i < nr; i += blockDim.x) rid[i] = relp_ids(a.ids, a.row0 + r0 + i);
  __syncthreads();
  float* mine = tab + warp * per_warp;
  const int64_t j = ((int64_t)blockIdx.x * kRelWarps + warp) * 32 + lane;
  const bool live = j < a.n_cols;
  const RelpIds cid = relp_ids(a.ids, a.col0 + (live ? j : 0));
  PairCols cur = pair_cols(rid[0], cid, a.R, a.S);
  // Sums since the residue column last changed, before that since the token column did, and before that
  // since the others did; a change flushes its own sum and the ones inside it.
  float run[G], tok[G], sym[G];
#pragma unroll
  for (int g = 0; g < G; ++g) run[g] = tok[g] = sym[g] = 0.f;
  auto flush_sym = [&](bool pred) {
    flush<G>(mine, a.n_feat, pred, cur.sym & (kEntBit - 1), sym);
    flush<G>(mine, a.n_feat, pred && (cur.sym & kEntBit), 4 * a.R + 4, sym);
  };
  const T* p = dout + (int64_t)h0 * a.hs + r0 * a.rs + (live ? j : 0);
  constexpr int U = G == 8 ? 4 : 8;  // rows in flight
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
        const PairCols c = pair_cols(rid[i0 + u], cid, a.R, a.S);
        const bool new_sym = live && c.sym != cur.sym, new_tok = new_sym || (live && c.tok != cur.tok),
                   new_res = new_tok || (live && c.res != cur.res);
        if (__any_sync(0xffffffffu, new_res)) {
          flush<G>(mine, a.n_feat, new_res, cur.res, run);
#pragma unroll
          for (int g = 0; g < G; ++g)
            if (new_res) {
              tok[g] += run[g];
              run[g] = 0.f;
            }
          if (__any_sync(0xffffffffu, new_tok)) {
            flush<G>(mine, a.n_feat, new_tok, cur.tok, tok);
#pragma unroll
            for (int g = 0; g < G; ++g)
              if (new_tok) {
                sym[g] += tok[g];
                tok[g] = 0.f;
              }
            if (__any_sync(0xffffffffu, new_sym)) {
              flush_sym(new_sym);
#pragma unroll
              for (int g = 0; g < G; ++g)
                if (new_sym) sym[g] = 0.f;
            }
          }
          if (live) cur = c;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) run[g] += to_f(x[u][g]);
      }
    }
  }
  flush<G>(mine, a.n_feat, live, cur.res, run);
#pragma unroll
  for (int g = 0; g < G; ++g) tok[g] += run[g];
  flush<G>(mine, a.n_feat, live, cur.tok, tok);
#pragma unroll
  for (int g = 0; g < G; ++g) sym[g] += tok[g];
  flush_sym(live);
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

// As many heads at a time as eight warps' tables leave room for in 64 KB of shared memory: eight up to
// 256 features (r_max up to 61), four up to 512, else one. Row chunks: about eight blocks per SM (two run
// at a time; the warps on the diagonal of a chain take several times as long as the others, and shorter
// chunks even that out: 16 rows 84 us, 32 rows 97 us at 1536 tokens and 16 heads), of at least four rows.
RelGrid plan(int64_t n_rows, int64_t n_cols, int heads, int n_feat) {
  RelGrid p;
  p.G = n_feat <= 256 && heads > 4 ? 8 : (n_feat <= 512 ? 4 : 1);
  p.strips = (n_cols + kRelWarps * 32 - 1) / (kRelWarps * 32);
  p.groups = (heads + p.G - 1) / p.G;
  int64_t want = 148 * kRelWaves * 2 / (p.strips * p.groups);
  want = want < 1 ? 1 : want;
  int64_t per = (n_rows + want - 1) / want;
  per = per < 4 ? 4 : (per > kRelRows ? kRelRows : per);
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
  PF_TRY((room_for_shared<k_relpos_bias_bwd<T, G>>(64 * 1024)));  // see plan()
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_relpos_bias_bwd", (double)a.heads * a.n_rows * a.n_cols * sizeof(T), 'b');
    k_relpos_bias_bwd<T, G><<<dim3((unsigned)p.strips, (unsigned)p.chunks, (unsigned)p.groups), kRelWarps * 32, smem,
                              st>>>(a, (const T*)dout, part);
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
#define PF_REL(TW, T)                                          \
  return p.G == 8   ? launch_fwd<TW, T, 8>(p, a, w, out, st)   \
         : p.G == 4 ? launch_fwd<TW, T, 4>(p, a, w, out, st)   \
                    : launch_fwd<TW, T, 1>(p, a, w, out, st)
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
  const int64_t m = (int64_t)heads * n_feat;
#define PF_REL(T)                                                  \
  PF_TRY((p.G == 8   ? launch_bwd<T, 8>(p, a, dbias, part, st)     \
          : p.G == 4 ? launch_bwd<T, 4>(p, a, dbias, part, st)     \
                     : launch_bwd<T, 1>(p, a, dbias, part, st)))
  if (dtype == PF_F32)
    PF_REL(float);
  else
    PF_REL(__nv_bfloat16);
#undef PF_REL
  return n == 1 ? PF_OK : sum_rows(part, n, m, dw, m, nullptr, st);
}

}  // namespace train
}  // namespace pf
