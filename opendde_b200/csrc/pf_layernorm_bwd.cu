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
// rows in a fixed order (no atomics: equal inputs give equal bits). One block writes the result itself.

#include "pf_common.cuh"
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

constexpr int kWarps = 8;

// L lanes per row, V chunks of E channels per lane, U rows of a lane in flight.
template <class T, int E, int L, int V, int U>
__global__ void __launch_bounds__(kWarps * 32) k_layernorm_bwd(const T* x, const T* dy,
                                                               const float* __restrict__ gamma, T* dx, float* dg_out,
                                                               float* db_out, int64_t rows, int c, float eps) {
  constexpr int R = 32 / L;  // rows of a warp side by side
  extern __shared__ float sm[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int sub = lane & (L - 1), grp = lane / L;
  const int nv = c / E;
  const float inv_c = 1.f / (float)c;
  float gw[V * E], ag[V * E], ab[V * E];
#pragma unroll
  for (int t = 0; t < V; ++t)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int v = sub + t * L;
      gw[t * E + e] = v < nv ? (gamma ? gamma[v * E + e] : 1.f) : 0.f;
      ag[t * E + e] = ab[t * E + e] = 0.f;
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
        if (row < rows && v < nv) {
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
      float s0 = 0.f;
#pragma unroll
      for (int t = 0; t < V; ++t) {
        float f[E];
        xr[u][t].get(f);
#pragma unroll
        for (int e = 0; e < E; ++e) s0 += f[e];
      }
      const float mean = group_sum<L>(s0) * inv_c;
      float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
      for (int t = 0; t < V; ++t) {
        float f[E], g[E];
        xr[u][t].get(f);
        gr[u][t].get(g);
        const bool in = sub + t * L < nv;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = in ? f[e] - mean : 0.f, gg = g[e] * gw[t * E + e];
          s1 += d * d;
          s2 += gg;
          s3 += gg * d;
        }
      }
      s1 = group_sum<L>(s1);
      s2 = group_sum<L>(s2);
      s3 = group_sum<L>(s3);
      // rows past the end are zero and add nothing, whatever eps is
      const float rstd = row < rows ? rsqrtf(s1 * inv_c + eps) : 0.f;
      const float m1 = s2 * inv_c, m2 = s3 * inv_c * rstd * rstd;
#pragma unroll
      for (int t = 0; t < V; ++t) {
        float f[E], g[E], o[E];
        xr[u][t].get(f);
        gr[u][t].get(g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float d = f[e] - mean;
          o[e] = (g[e] * gw[t * E + e] - m1 - d * m2) * rstd;
          ag[t * E + e] += g[e] * (d * rstd);  // rows past the end have dy = 0
          ab[t * E + e] += g[e];
        }
        const int v = sub + t * L;
        if (dx && row < rows && v < nv) Chunk<T, E>::store(dx + row * c + (int64_t)v * E, o);
      }
    }
  }
  if (!dg_out && !db_out) return;
  // the warp's rows side by side, then the block's warps
#pragma unroll
  for (int i = 0; i < V * E; ++i) {
#pragma unroll
    for (int o = L; o < 32; o <<= 1) {
      ag[i] += __shfl_xor_sync(0xffffffffu, ag[i], o);
      ab[i] += __shfl_xor_sync(0xffffffffu, ab[i], o);
    }
  }
  if (grp == 0) {
#pragma unroll
    for (int t = 0; t < V; ++t) {
      const int v = sub + t * L;
      if (v < nv)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          sm[(warp * 2) * c + v * E + e] = ag[t * E + e];
          sm[(warp * 2 + 1) * c + v * E + e] = ab[t * E + e];
        }
    }
  }
  __syncthreads();
  const int64_t part = (int64_t)blockIdx.x * c;
  for (int i = threadIdx.x; i < c; i += kWarps * 32) {
    float a = 0.f, b = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      a += sm[(w * 2) * c + i];
      b += sm[(w * 2 + 1) * c + i];
    }
    if (dg_out) dg_out[part + i] = a;
    if (db_out) db_out[part + i] = b;
  }
}

// 32 columns by 8 row groups per block: group y adds rows y, y + 8, ..., then the groups are added.
__global__ void __launch_bounds__(256) k_sum_rows(const float* __restrict__ part, int64_t n, int64_t m,
                                                  float* __restrict__ out) {
  __shared__ float sm[8][33];
  const int64_t i = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (i < m)
    for (int64_t r = threadIdx.y; r < n; r += 8) s += part[r * m + i];
  sm[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && i < m) {
#pragma unroll
    for (int y = 1; y < 8; ++y) s += sm[y][threadIdx.x];
    out[i] = s;
  }
}

int sm_count() {
  int dev = 0, n = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev);
  return n;
}

// Blocks of the row kernel: enough warps to cover the rows, at most four blocks on each SM.
int64_t grid_blocks(int64_t rows, int rows_per_block) {
  const int64_t need = (rows + rows_per_block - 1) / rows_per_block, most = (int64_t)sm_count() * 4;
  return need < 1 ? 1 : (need < most ? need : most);
}

template <class T, int E, int L, int V, int U>
int launch(const T* x, const T* dy, const float* gamma, T* dx, float* dg, float* db, int64_t rows, int c, float eps,
           float* part, cudaStream_t st) {
  const int64_t blocks = grid_blocks(rows, kWarps * (32 / L) * U);
  const size_t smem = (size_t)kWarps * 2 * c * sizeof(float);
  auto* kern = k_layernorm_bwd<T, E, L, V, U>;
  if (smem > 48 * 1024) PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  const bool direct = blocks == 1;
  float* pg = direct ? dg : (dg ? part : nullptr);
  float* pb = direct ? db : (db ? part + blocks * c : nullptr);
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_layernorm_bwd", 3.0 * (double)rows * c * sizeof(T), 'b');
    kern<<<(unsigned)blocks, kWarps * 32, smem, st>>>(x, dy, gamma, dx, pg, pb, rows, c, eps);
  }
  PF_CHECK_LAUNCH();
  if (direct) return PF_OK;
  if (dg) PF_TRY(sum_rows(pg, blocks, c, dg, st));
  if (db) PF_TRY(sum_rows(pb, blocks, c, db, st));
  return PF_OK;
}

template <class T, int E>
int dispatch(const T* x, const T* dy, const float* gamma, T* dx, float* dg, float* db, int64_t rows, int c, float eps,
             float* part, cudaStream_t st) {
  const int nv = c / E;
#define PF_LN(L, V, U) return launch<T, E, L, V, U>(x, dy, gamma, dx, dg, db, rows, c, eps, part, st)
  if (nv <= 1) PF_LN(1, 1, 2);
  if (nv <= 2) PF_LN(2, 1, 2);
  if (nv <= 4) PF_LN(4, 1, 2);
  if (nv <= 8) PF_LN(8, 1, 2);
  if (nv <= 16) PF_LN(16, 1, 2);
  if (nv <= 32) PF_LN(32, 1, 2);
  if (nv <= 64) PF_LN(32, 2, 1);
  if (nv <= 96) PF_LN(32, 3, 1);
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

int sum_rows(const float* part, int64_t n, int64_t m, float* out, cudaStream_t st) {
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_sum_rows", 4.0 * (double)(n + 1) * m, 'b');
    k_sum_rows<<<(unsigned)((m + 31) / 32), dim3(32, 8), 0, st>>>(part, n, m, out);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// Two partial rows (dgamma, dbeta) per block of the largest grid; the size depends on the channel
// count alone, and a problem of one block needs none of it.
size_t layernorm_bwd_ws_bytes(int64_t, int c, int) { return (size_t)sm_count() * 4 * 2 * c * sizeof(float); }

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
