// pf_layernorm_bwd.cu -- the backward pass of the layer norm (pf_layernorm_fwd).
//
// With xh = (x - mean) * rstd and g = gamma * dy (rows of c channels):
//   dx     = rstd * (g - mean(g) - xh * mean(g * xh))
//   dgamma = sum over rows of dy * xh,   dbeta = sum over rows of dy
// Mean and rstd are recomputed from x, which the pass has to read anyway, so the forward keeps
// nothing. A row lies in the registers of L lanes (L a power of two up to a warp); one round of
// shuffles gives the mean, a second one the three sums of centred values (the variance is a sum of
// squares of x - mean, not a difference of moments, which a large mean would cancel).
//
// A warp walks over rows and keeps its lanes' share of dgamma and dbeta in registers; a block adds
// its warps' shares through shared memory and writes one partial row, and k_sum_rows adds the partial
// rows in a fixed order (no atomics: equal inputs give equal bits). Few rows are one cluster of blocks, which add
// their rows through distributed shared memory in the same launch.

#include <cooperative_groups.h>

#include "pf_common.cuh"
#include "pf_f32x2.cuh"
#include "pf_prof.h"
#include "pf_train.h"

namespace pf {
namespace train {
namespace {

// E consecutive channels of a row as one access: 16 bytes, or one element where rows are not whole
// aligned 16-byte vectors.
template <class T, int E>
struct Chunk;
template <>
struct Chunk<float, 4> {
  float4 r;
  __device__ void load(const float* p) { r = *reinterpret_cast<const float4*>(p); }
  __device__ void zero() { r = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ void get(float* f) const { f[0] = r.x, f[1] = r.y, f[2] = r.z, f[3] = r.w; }
  __device__ static void store(float* p, const float* f) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  }
};
template <>
struct Chunk<__nv_bfloat16, 8> {
  uint4 r;
  __device__ void load(const __nv_bfloat16* p) { r = *reinterpret_cast<const uint4*>(p); }
  __device__ void zero() { r = make_uint4(0, 0, 0, 0); }
  __device__ void get(float* f) const {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(w[i] << 16);
      f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
  __device__ static void store(__nv_bfloat16* p, const float* f) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <class T>
struct Chunk<T, 1> {
  T r;
  __device__ void load(const T* p) { r = *p; }
  __device__ void zero() { r = from_f<T>(0.f); }
  __device__ void get(float* f) const { f[0] = to_f(r); }
  __device__ static void store(T* p, const float* f) { *p = from_f<T>(f[0]); }
};

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

namespace cg = cooperative_groups;
constexpr int kWarps = 8;
constexpr int kRanks = 8;  // blocks of the cluster that takes few rows

// Blocks on an SM: two (128 registers) where a lane has up to 16 channels, and at 768 bf16 channels exactly; more
// channels need the registers of one block (two: 0.3 to 1.4 KB of spills; 30000 rows of 1024, bf16 109 against 59 us,
// fp32 115 against 70 us; 40000 rows of 768, fp32 137 against 82 us, but bf16 57 against 63 us; 30000 rows of 640
// bf16 56 against 53 us).
constexpr int blocks_per_sm(int channels, bool full) { return channels <= 16 || (full && channels <= 24) ? 2 : 1; }

// L lanes per row, V chunks of E channels per lane, U rows of a lane in flight; FULL: c = L V E.
template <class T, int E, int L, int V, int U, bool FULL>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm(V * E, FULL))
    k_layernorm_bwd(const T* x, const T* dy, const float* __restrict__ gamma, T* dx, float* dg_out, float* db_out,
                    int64_t part, int64_t rows, int c, float eps, int ranks) {
  constexpr int R = 32 / L;  // rows of a warp side by side
  constexpr int N = V * E / 2;  // channel pairs of a lane
  extern __shared__ float sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (L - 1), grp = lane / L;
  const int nv = c / E;
  const float inv_c = 1.f / (float)c;
  auto in = [&](int i) { return FULL || sub + (i / E) * L < nv; };       // element i of the lane exists
  auto channel = [&](int i) { return (sub + (i / E) * L) * E + i % E; };  // its channel
  F2 gw[N], ag[N], ab[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    gw[i] = F2(in(2 * i) ? (gamma ? gamma[channel(2 * i)] : 1.f) : 0.f,
               in(2 * i + 1) ? (gamma ? gamma[channel(2 * i + 1)] : 1.f) : 0.f);
    ag[i] = ab[i] = F2(0.f);
  }
  const int64_t step = (int64_t)gridDim.x * kWarps * R * U;
  for (int64_t base = ((int64_t)blockIdx.x * kWarps + warp) * R * U; base < rows; base += step) {
    Chunk<T, E> xr[U][V], gr[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + (int64_t)u * R + grp;
#pragma unroll
      for (int t = 0; t < V; ++t) {
        const int v = sub + t * L;
        if (row < rows && (FULL || v < nv)) {
          xr[u][t].load(x + row * c + (int64_t)v * E);
          gr[u][t].load(dy + row * c + (int64_t)v * E);
        } else {
          xr[u][t].zero();
          gr[u][t].zero();
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = base + (int64_t)u * R + grp;
      float f[V * E], g[V * E];
#pragma unroll
      for (int t = 0; t < V; ++t) {
        xr[u][t].get(f + t * E);
        gr[u][t].get(g + t * E);
      }
      F2 s0 = F2(f[0], f[1]);
#pragma unroll
      for (int i = 1; i < N; ++i) s0 = add2(s0, F2(f[2 * i], f[2 * i + 1]));
      const float mean = group_sum<L>(s0.sum()) * inv_c;
      const F2 nmean(-mean);
      F2 s1(0.f), s2(0.f), s3(0.f);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        F2 d = add2(F2(f[2 * i], f[2 * i + 1]), nmean);
        d.get(f[2 * i], f[2 * i + 1]);
        if (!FULL) {
          if (!in(2 * i)) f[2 * i] = 0.f;
          if (!in(2 * i + 1)) f[2 * i + 1] = 0.f;
          d = F2(f[2 * i], f[2 * i + 1]);
        }
        const F2 gg = mul2(F2(g[2 * i], g[2 * i + 1]), gw[i]);
        s1 = fma2(d, d, s1);
        s2 = add2(s2, gg);
        s3 = fma2(gg, d, s3);
      }
      const float q1 = group_sum<L>(s1.sum()), q2 = group_sum<L>(s2.sum()), q3 = group_sum<L>(s3.sum());
      // rows past the end are zero and add nothing, whatever eps is
      const float rstd = row < rows ? rsqrtf(q1 * inv_c + eps) : 0.f;
      // dx = rstd (g - mean(g)) - d rstd^3 mean(g d)
      const F2 r2(rstd), m1(-q2 * inv_c * rstd), m2(-q3 * inv_c * rstd * rstd * rstd);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const F2 d = F2(f[2 * i], f[2 * i + 1]), gy = F2(g[2 * i], g[2 * i + 1]);
        ag[i] = fma2(gy, mul2(d, r2), ag[i]);
        ab[i] = add2(ab[i], gy);
        fma2(d, m2, fma2(mul2(gy, gw[i]), r2, m1)).get(f[2 * i], f[2 * i + 1]);
      }
      if (dx && row < rows) {
#pragma unroll
        for (int t = 0; t < V; ++t) {
          const int v = sub + t * L;
          if (FULL || v < nv) Chunk<T, E>::store(dx + row * c + (int64_t)v * E, f + t * E);
        }
      }
    }
  }
  if (!dg_out && !db_out) return;
  // the warp's rows side by side, then the block's warps
  float a[2 * N], b[2 * N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    ag[i].get(a[2 * i], a[2 * i + 1]);
    ab[i].get(b[2 * i], b[2 * i + 1]);
  }
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) {
      a[i] += __shfl_xor_sync(0xffffffffu, a[i], o);
      b[i] += __shfl_xor_sync(0xffffffffu, b[i], o);
    }
  }
  if (grp == 0) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i)
      if (in(i)) {
        sm[(warp * 2) * c + channel(i)] = a[i];
        sm[(warp * 2 + 1) * c + channel(i)] = b[i];
      }
  }
  __syncthreads();
  const int64_t off = (int64_t)blockIdx.x * part;
  for (int i = threadIdx.x; i < c; i += kWarps * 32) {
    float sa = 0.f, sb = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      sa += sm[(w * 2) * c + i];
      sb += sm[(w * 2 + 1) * c + i];
    }
    if (ranks > 1) {
      sm[i] = sa;  // this thread alone has read column i
      sm[c + i] = sb;
    } else {
      if (dg_out) dg_out[off + i] = sa;
      if (db_out) db_out[off + i] = sb;
    }
  }
  if (ranks > 1) {  // the grid is one cluster: each block adds a share of the columns over all of them
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    const int share = (2 * c + ranks - 1) / ranks, i1 = min(2 * c, ((int)blockIdx.x + 1) * share);
    for (int i = blockIdx.x * share + threadIdx.x; i < i1; i += kWarps * 32) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < kRanks; ++r) s += *cluster.map_shared_rank(sm + i, r);
      if (i < c) {
        if (dg_out) dg_out[i] = s;
      } else {
        if (db_out) db_out[i - c] = s;
      }
    }
    cluster.sync();  // no block leaves while others read its sums
  }
}

// 32 columns by 32 row groups per block: group y adds rows y, y + 32, ..., then the groups are added.
// Columns below m0 go to out0, the others to out1.
__global__ void __launch_bounds__(1024) k_sum_rows(const float* __restrict__ part, int64_t n, int64_t m,
                                                   float* __restrict__ out0, int64_t m0, float* __restrict__ out1) {
  __shared__ float sm[32][33];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (i < m)
    for (int64_t r = threadIdx.y; r < n; r += 32) s += part[r * m + i];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  // warp y adds the groups of column y
  float v = sm[threadIdx.x][threadIdx.y];
  v = warp_sum(v);
  const int64_t j = (int64_t)blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && j < m) {
    if (j < m0)
      out0[j] = v;
    else
      out1[j - m0] = v;
  }
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Blocks of the row kernel for rows of `chunk` rows per block and step, `values` values of a lane in flight: a cluster
// of eight where the rows are few steps of it, up to four of 16 values, two of 32 (called and replayed, us, fp32: 64
// rows of 384 channels, one step, 18 and 4.7 against 21 to 25 and 6.2 in two launches; 128 rows of 1024, two steps, 20
// and 8 against 24 and 8; 1024 rows of 128, four steps, 18 and 8 against 21 and 6; 3500 rows of 37, 28 steps, 25 and
// 25 against 22 and 8); else enough warps to cover the rows, at most four blocks on each SM.
bool few_rows(int64_t rows, int chunk, int values) {
  const int steps = values > 16 ? 64 / values : 4;
  return rows <= (int64_t)steps * kRanks * chunk;
}
int64_t grid_blocks(int64_t rows, int rows_per_block) {
  const int64_t need = (rows + rows_per_block - 1) / rows_per_block, most = (int64_t)sm_count() * 4;
  return need < 1 ? 1 : (need < most ? need : most);
}

template <class T, int E, int L, int V, int U, bool FULL>
int launch(const T* x, const T* dy, const float* gamma, T* dx, float* dg, float* db, int64_t rows, int c, float eps,
           float* part, cudaStream_t st) {
  constexpr int rows_per_block = kWarps * (32 / L) * U;
  const bool cluster = (dg || db) && few_rows(rows, rows_per_block, U * V * E);
  const int64_t blocks = cluster ? kRanks : grid_blocks(rows, rows_per_block);  // more than one where sums are wanted
  const size_t smem = (size_t)kWarps * 2 * c * sizeof(float);
  constexpr auto* kern = k_layernorm_bwd<T, E, L, V, U, FULL>;
  PF_TRY(room_for_shared<kern>((size_t)kWarps * 2 * L * V * E * sizeof(float)));  // the instance's widest rows
  const int64_t m0 = dg ? c : 0, m = m0 + (db ? c : 0);  // a partial row: dgamma, then dbeta
  float* pg = cluster || !dg ? dg : part;
  float* pb = cluster || !db ? db : part + m0;
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_layernorm_bwd", 3.0 * (double)rows * c * sizeof(T), 'b');
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = kRanks, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(kWarps * 32);
    cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cfg.attrs = &attr, cfg.numAttrs = cluster ? 1 : 0;
    PF_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, x, dy, gamma, dx, pg, pb, m, rows, c, eps, cluster ? kRanks : 1));
  }
  PF_CHECK_LAUNCH();
  return cluster || m == 0 ? PF_OK : sum_rows(part, blocks, m, dg, m0, db, st);
}

template <class T, int E>
int dispatch(const T* x, const T* dy, const float* gamma, T* dx, float* dg, float* db, int64_t rows, int c, float eps,
             float* part, cudaStream_t st) {
  // two chunks per lane and few lanes per row: a row's four sums then take few shuffle steps
  const int nv = c / E;
#define PF_LN(L, V, U)                                                                        \
  return nv == L * V ? launch<T, E, L, V, U, true>(x, dy, gamma, dx, dg, db, rows, c, eps, part, st) \
                     : launch<T, E, L, V, U, false>(x, dy, gamma, dx, dg, db, rows, c, eps, part, st)
  if (nv <= 2) PF_LN(1, 2, 1);
  if (nv <= 4) PF_LN(2, 2, 1);
  if (nv <= 8) PF_LN(4, 2, 2);
  if (nv <= 16) PF_LN(8, 2, 2);
  if (nv <= 32) PF_LN(16, 2, 2);
  if (nv <= 64) PF_LN(32, 2, 2);
  if constexpr (E > 1) {
    if (nv <= 96) PF_LN(32, 3, 1);
  }
  if (nv <= 128) PF_LN(32, 4, 1);
  if constexpr (E < 8) {
    if (nv <= 256) PF_LN(32, 8, 1);
  }
  if constexpr (E == 1) {
    if (nv <= 512) PF_LN(32, 16, 1);
    if (nv <= 1024) PF_LN(32, 32, 1);
  }
#undef PF_LN
  return fail(PF_EINVAL_SHAPE, "layernorm backward: c=%d", c);
}

}  // namespace

int sum_rows(const float* part, int64_t n, int64_t m, float* out0, int64_t m0, float* out1, cudaStream_t st) {
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_sum_rows", 4.0 * (double)(n + 1) * m, 'b');
    k_sum_rows<<<(unsigned)((m + 31) / 32), dim3(32, 32), 0, st>>>(part, n, m, out0, m0, out1);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// Two partial rows (dgamma, dbeta) per block of the largest grid that these rows can have: every instance takes at
// least one row per warp and step.
size_t layernorm_bwd_ws_bytes(int64_t rows, int c, int) {
  return (size_t)grid_blocks(rows, kWarps) * 2 * c * sizeof(float);
}

int layernorm_bwd(const void* x, const void* dy, const float* gamma, void* dx, float* dgamma, float* dbeta,
                  int64_t rows, int c, float eps, int dtype, void* ws, size_t, cudaStream_t st) {
  const size_t esz = dtype == PF_F32 ? 4 : 2;
  const bool vec = (c * esz) % 16 == 0 && ((uintptr_t)x | (uintptr_t)dy | (uintptr_t)dx) % 16 == 0;
  float* part = (float*)ws;
  if (dtype == PF_F32) {
    const float *xf = (const float*)x, *df = (const float*)dy;
    return vec ? dispatch<float, 4>(xf, df, gamma, (float*)dx, dgamma, dbeta, rows, c, eps, part, st)
               : dispatch<float, 1>(xf, df, gamma, (float*)dx, dgamma, dbeta, rows, c, eps, part, st);
  }
  const __nv_bfloat16 *xh = (const __nv_bfloat16*)x, *dh = (const __nv_bfloat16*)dy;
  return vec ? dispatch<__nv_bfloat16, 8>(xh, dh, gamma, (__nv_bfloat16*)dx, dgamma, dbeta, rows, c, eps, part, st)
             : dispatch<__nv_bfloat16, 1>(xh, dh, gamma, (__nv_bfloat16*)dx, dgamma, dbeta, rows, c, eps, part, st);
}

}  // namespace train
}  // namespace pf
