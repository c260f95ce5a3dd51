// pf_attention_f32.cu -- the fp32 kernels of pf_attention.cuh: a stationary tile of 64 rows (16 per warp)
// against streamed tiles of BN rows that cp.async double-buffers in shared memory, with FFMA.

#include "pf_attention.cuh"
#include "pf_f32x2.cuh"

namespace pf {
namespace train {
namespace attn {
namespace {

constexpr int BM = kWarps * 16;  // rows of a stationary tile

// ---------------------------------------------------------------- tiles

template <int DP>
struct Pitch {
  static constexpr int value = DP + 4;  // rows shifted by 16 bytes: no bank conflicts
};

__device__ __forceinline__ bool key_seen(const Args& a, int64_t b, int64_t j) {
  return a.mask == nullptr || a.mask[b * a.m_bs + j * a.m_ks] != 0.f;
}

// Rows [r0, r0 + ROWS) of (b, h) into shared memory, zero past n and d, and where MASKED for masked keys.
template <int DP, int ROWS, bool MASKED>
__device__ __forceinline__ void load_tile(float* sm, const Args& a, const Heads& s, int vec, int64_t b, int h, int64_t r0,
                                          int64_t n) {
  constexpr int P = Pitch<DP>::value, E = 4, CH = DP / E;
  const float* base = (const float*)s.p + b * s.bs + (int64_t)h * s.hs;
  if (vec) {
#pragma unroll
    for (int i = threadIdx.x; i < ROWS * CH; i += kThreads) {
      const int r = i / CH, c = (i - r * CH) * E;
      const int64_t row = r0 + r;
      bool ok = row < n && c < a.d;
      if (MASKED && ok) ok = key_seen(a, b, row);
      cp_async16(smem_addr(sm + r * P + c), ok ? base + row * s.ns + c : base, ok);
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * DP; i += kThreads) {
      const int r = i / DP, c = i - r * DP;
      const int64_t row = r0 + r;
      bool ok = row < n && c < a.d;
      if (MASKED && ok) ok = key_seen(a, b, row);
      sm[r * P + c] = ok ? base[row * s.ns + c] : 0.f;
    }
  }
}

// Which of the BN keys from j0 on are visible, as bits (the same in every lane of a warp).
template <int BN>
__device__ __forceinline__ uint64_t seen_bits(const Args& a, int64_t b, int64_t j0) {
  const int lane = threadIdx.x & 31;
  uint64_t bits = 0;
#pragma unroll
  for (int i = 0; i < BN / 32; ++i) {
    const int64_t j = j0 + i * 32 + lane;
    const bool ok = j < a.nk && key_seen(a, b, j);
    bits |= (uint64_t)__ballot_sync(0xffffffffu, ok) << (32 * i);
  }
  return bits;
}
template <int BN>
__device__ __forceinline__ bool all_seen(uint64_t bits) {
  return bits == (BN == 64 ? ~0ull : (1ull << (BN & 63)) - 1ull);
}

// ---------------------------------------------------------------- products
// Register layout of a 16 x 8n accumulator (both types): lane (g, t) = (lane / 4, lane % 4) holds
// c[n][0..1] = row g, columns 8n + 2t, +1 and c[n][2..3] = row g + 8, the same columns.

template <int DP, int BN>
struct Prod {
  static constexpr int P = Pitch<DP>::value;
  // c = a b^T; pairs hold the sums over even and odd depths
  static __device__ void nt(float (&c)[BN / 8][4], const float* a, const float* b) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    F2 s[BN / 8][4];
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = F2(0.f);
#pragma unroll 4
    for (int k = 0; k < DP; k += 4) {
      const float4 a0 = *reinterpret_cast<const float4*>(a + g * P + k);
      const float4 a1 = *reinterpret_cast<const float4*>(a + (g + 8) * P + k);
      const F2 a0l(a0.x, a0.y), a0h(a0.z, a0.w), a1l(a1.x, a1.y), a1h(a1.z, a1.w);
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) {
        const float4 b0 = *reinterpret_cast<const float4*>(b + (n * 8 + 2 * t) * P + k);
        const float4 b1 = *reinterpret_cast<const float4*>(b + (n * 8 + 2 * t + 1) * P + k);
        const F2 b0l(b0.x, b0.y), b0h(b0.z, b0.w), b1l(b1.x, b1.y), b1h(b1.z, b1.w);
        s[n][0] = fma2(a0h, b0h, fma2(a0l, b0l, s[n][0]));
        s[n][1] = fma2(a0h, b1h, fma2(a0l, b1l, s[n][1]));
        s[n][2] = fma2(a1h, b0h, fma2(a1l, b0l, s[n][2]));
        s[n][3] = fma2(a1h, b1h, fma2(a1l, b1l, s[n][3]));
      }
    }
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) c[n][e] = s[n][e].sum();
  }
  // acc += p b; p goes through the warp's scratch rows [16][BN + 4]
  static __device__ void nn(float (&acc)[DP / 8][4], const float (&p)[BN / 8][4], float* sc, const float* b) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int Q = BN + 4;
    __syncwarp();
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) {
      *reinterpret_cast<float2*>(sc + g * Q + n * 8 + 2 * t) = make_float2(p[n][0], p[n][1]);
      *reinterpret_cast<float2*>(sc + (g + 8) * Q + n * 8 + 2 * t) = make_float2(p[n][2], p[n][3]);
    }
    __syncwarp();
    F2 s[DP / 8][2];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      s[n][0] = F2(acc[n][0], acc[n][1]);
      s[n][1] = F2(acc[n][2], acc[n][3]);
    }
#pragma unroll 2
    for (int k = 0; k < BN; k += 4) {
      const float4 a0 = *reinterpret_cast<const float4*>(sc + g * Q + k);
      const float4 a1 = *reinterpret_cast<const float4*>(sc + (g + 8) * Q + k);
      const float x0[4] = {a0.x, a0.y, a0.z, a0.w}, x1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const F2 y0(x0[u]), y1(x1[u]);
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          const float2 v = *reinterpret_cast<const float2*>(b + (k + u) * P + n * 8 + 2 * t);
          s[n][0] = fma2(y0, F2(v.x, v.y), s[n][0]);
          s[n][1] = fma2(y1, F2(v.x, v.y), s[n][1]);
        }
      }
    }
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      s[n][0].get(acc[n][0], acc[n][1]);
      s[n][1].get(acc[n][2], acc[n][3]);
    }
  }
};

// ---------------------------------------------------------------- shared-memory plan

template <int DP, int BN>
struct Smem {
  static constexpr int P = Pitch<DP>::value;
  static constexpr int kStat = BM * P, kStream = BN * P;  // elements
  static constexpr int kScratch = kWarps * 16 * (BN + 4);
  // nstat stationary tiles, nstream streamed tiles (double-buffered), the products' scratch rows
  static size_t bytes(int nstat, int nstream) {
    return ((size_t)nstat * kStat + 2 * (size_t)nstream * kStream + kScratch) * sizeof(float);
  }
};

// ---------------------------------------------------------------- scores

__device__ __forceinline__ float ld_bias1(const Args& a, int64_t off) {
  return a.bias_f32 ? ((const float*)a.bias)[off] : __bfloat162float(((const __nv_bfloat16*)a.bias)[off]);
}

// x[n][i] = scale * x[n][i] + bias of rows (i0 + g, i0 + g + 8), keys j0 + 8n + 2t (+1); only visible
// keys of real rows are read.
template <int BN>
__device__ __forceinline__ void add_bias(float (&x)[BN / 8][4], const Args& a, int64_t b, int h, int64_t i0,
                                         int64_t j0, uint64_t bits) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int n = 0; n < BN / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[n][e] *= a.scale;
  if (a.bias == nullptr) return;
  const bool full = all_seen<BN>(bits) && a.bias_vec;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = i0 + g + 8 * r;
    if (i >= a.nq) continue;
    const int64_t off = b * a.b_bs + (int64_t)h * a.b_hs + i * a.b_rs + j0 + 2 * t;
    if (full && a.bias_f32) {
      const float* p = (const float*)a.bias + off;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) {
        const float2 v = *reinterpret_cast<const float2*>(p + n * 8);
        x[n][2 * r] += v.x;
        x[n][2 * r + 1] += v.y;
      }
    } else if (full) {
      const __nv_bfloat16* p = (const __nv_bfloat16*)a.bias + off;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) {
        const uint32_t v = *reinterpret_cast<const uint32_t*>(p + n * 8);
        x[n][2 * r] += __uint_as_float(v << 16);
        x[n][2 * r + 1] += __uint_as_float(v & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if ((bits >> (n * 8 + 2 * t + e)) & 1) x[n][2 * r + e] += ld_bias1(a, off + n * 8 + e);
    }
  }
}

template <int BN>
__device__ __forceinline__ void hide(float (&x)[BN / 8][4], uint64_t bits) {
  if (all_seen<BN>(bits)) return;
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int n = 0; n < BN / 8; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (!((bits >> (n * 8 + 2 * t + e)) & 1)) x[n][e] = x[n][2 + e] = -INFINITY;
}

// p and, in dp's place, ds (see the head of the file)
template <int BN>
__device__ __forceinline__ void prob_ds_rows(float (&s)[BN / 8][4], float (&dp)[BN / 8][4], const float* m,
                                             const float* c, const float* D, const float* peak) {
#pragma unroll
  for (int n = 0; n < BN / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = expf(s[n][e] - m[e >> 1]) * c[e >> 1];
      s[n][e] = p;
      dp[n][e] = peak[e >> 1] != 0.f && p == 1.f ? 0.f : p * (dp[n][e] - D[e >> 1]);
    }
}

template <int DP>
__device__ __forceinline__ void store_rows(void* out, int64_t off, int64_t ns, int64_t i0, int64_t n, int d,
                                           const float (&acc)[DP / 8][4], float f0, float f1) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = i0 + g + 8 * r;
    if (i >= n) continue;
    float* p = (float*)out + off + i * ns;
    const float f = r ? f1 : f0;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = c * 8 + 2 * t + e;
        if (col < d) p[col] = acc[c][2 * r + e] * f;
      }
  }
}

// ---------------------------------------------------------------- forward

template <int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_fwd(Args a) {
  using M = Prod<DP, BN>;
  using S = Smem<DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sq = (float*)raw;
  float* sk = sq + S::kStat;           // [2]
  float* sv = sk + 2 * S::kStream;     // [2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* sc = sv + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int h = (int)(id % a.H), kh = h / (a.H / a.KV);
  const int64_t b = id / a.H;
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16;
  const int64_t nt = (a.nk + BN - 1) / BN;
  load_tile<DP, BM, false>(sq, a, a.q, a.vec_q, b, h, i0, a.nq);
  auto issue = [&](int64_t kt) {
    const int s = (int)(kt & 1);
    load_tile<DP, BN, true>(sk + s * S::kStream, a, a.k, a.vec_k, b, kh, kt * BN, a.nk);
    load_tile<DP, BN, true>(sv + s * S::kStream, a, a.v, a.vec_v, b, kh, kt * BN, a.nk);
    cp_commit();
  };
  float acc[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  if (nt > 0) issue(0);
  for (int64_t kt = 0; kt < nt; ++kt) {
    const uint64_t bits = seen_bits<BN>(a, b, kt * BN);
    cp_wait<0>();
    __syncthreads();
    if (kt + 1 < nt) issue(kt + 1);
    if (bits == 0 || w0 >= a.nq) continue;  // nothing to see, or a warp past the end
    const int s = (int)(kt & 1);
    float x[BN / 8][4];
    M::nt(x, sq + warp * 16 * S::P, sk + s * S::kStream);
    add_bias<BN>(x, a, b, h, w0, kt * BN, bits);
    hide<BN>(x, bits);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float mx = m[r];
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) mx = fmaxf(mx, fmaxf(x[n][2 * r], x[n][2 * r + 1]));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float base = mx == -INFINITY ? 0.f : mx;  // nothing seen yet: every p is 0
      const float corr = expf(m[r] - base);
      m[r] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = expf(x[n][2 * r + e] - base);
          x[n][2 * r + e] = p;
          sum += p;
        }
      l[r] = l[r] * corr + sum;
#pragma unroll
      for (int n = 0; n < DP / 8; ++n) {
        acc[n][2 * r] *= corr;
        acc[n][2 * r + 1] *= corr;
      }
    }
    M::nn(acc, x, sc, sv + s * S::kStream);
  }
  cp_commit();
  cp_wait<0>();
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
    const int64_t i = w0 + g + 8 * r;
    if (i >= a.nq) continue;
    if (a.stats && t == 0) {
      const int64_t at = (b * a.H + h) * a.nq + i;
      a.stats[at] = m[r];
      a.stats[a.rows_plane + at] = l[r];
    }
    float* o = (float*)a.o + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = c * 8 + 2 * t + e;
        if (col < a.d) o[col] = acc[c][2 * r + e] * inv;
      }
  }
}

// ---------------------------------------------------------------- backward

// Eight lanes per row (b, i, h): D, and {m, 1 / l, peak, D}; peak = 1 where one key has all of
// the row's weight in fp32 (l = 1).
__global__ void __launch_bounds__(256) k_rows(Args a, const float* __restrict__ stats, Heads o,
                                              float4* __restrict__ rows) {
  const int sub = threadIdx.x & 7;
  const int64_t r = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool live = r < a.rows_plane;
  const int64_t rr = live ? r : 0;
  const int h = (int)(rr % a.H);
  const int64_t bi = rr / a.H, b = bi / a.nq, i = bi - b * a.nq;
  const float* po = (const float*)o.p + b * o.bs + i * o.ns + (int64_t)h * o.hs;
  const float* pg = (const float*)a.g.p + b * a.g.bs + i * a.g.ns + (int64_t)h * a.g.hs;
  float s = 0.f;
  if (live)
    for (int e = sub; e < a.d; e += 8) s += po[e] * pg[e];
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  if (!live || sub) return;
  const int64_t at = (b * a.H + h) * a.nq + i;
  const float m = stats[at], l = stats[a.rows_plane + at];
  const bool none = l == 0.f;
  rows[at] = make_float4(none ? INFINITY : m, none ? 0.f : 1.f / l, l == 1.f ? 1.f : 0.f, none ? 0.f : s);
}

struct RowConst {
  float m[2], c[2], peak[2], D[2];
};
__device__ __forceinline__ RowConst row_const(const Args& a, int64_t b, int h, int64_t i0) {
  const int g = (threadIdx.x & 31) >> 2;
  RowConst r;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = i0 + g + 8 * k;
    const float4 v = i < a.nq ? ((const float4*)a.rows)[(b * a.H + h) * a.nq + i] : make_float4(INFINITY, 0.f, 0.f, 0.f);
    r.m[k] = v.x, r.c[k] = v.y, r.peak[k] = v.z, r.D[k] = v.w;
  }
  return r;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// ds of the warp's rows to dbias (real rows, keys below nk)
template <int BN>
__device__ __forceinline__ void store_dbias(const Args& a, int64_t b, int h, int64_t i0, int64_t j0,
                                            const float (&ds)[BN / 8][4]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const bool full = j0 + BN <= a.nk && a.db_vec;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = i0 + g + 8 * r;
    if (i >= a.nq) continue;
    const int64_t off = b * a.db_bs + (int64_t)h * a.db_hs + i * a.db_rs + j0 + 2 * t;
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) {
      if (full) {
        if (a.bias_f32)
          *reinterpret_cast<float2*>((float*)a.dbias + off + n * 8) = make_float2(ds[n][2 * r], ds[n][2 * r + 1]);
        else
          *reinterpret_cast<uint32_t*>((__nv_bfloat16*)a.dbias + off + n * 8) =
              pack2(ds[n][2 * r], ds[n][2 * r + 1]);
      } else {
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (j0 + n * 8 + 2 * t + e < a.nk) {
            if (a.bias_f32)
              ((float*)a.dbias)[off + n * 8 + e] = ds[n][2 * r + e];
            else
              ((__nv_bfloat16*)a.dbias)[off + n * 8 + e] = __float2bfloat16_rn(ds[n][2 * r + e]);
          }
      }
    }
  }
}

// dq of one query tile; dbias too where a.dbias is set (one batch entry per bias plane).
template <int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dq(Args a) {
  using M = Prod<DP, BN>;
  using S = Smem<DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sq = (float*)raw;
  float* sg = sq + S::kStat;
  float* sk = sg + S::kStat;        // [2]
  float* sv = sk + 2 * S::kStream;  // [2]
  const int warp = threadIdx.x >> 5;
  float* sc = sv + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int h = (int)(id % a.H), kh = h / (a.H / a.KV);
  const int64_t b = id / a.H;
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16;
  const int64_t nt = (a.nk + BN - 1) / BN;
  load_tile<DP, BM, false>(sq, a, a.q, a.vec_q, b, h, i0, a.nq);
  load_tile<DP, BM, false>(sg, a, a.g, a.vec_g, b, h, i0, a.nq);
  auto issue = [&](int64_t kt) {
    const int s = (int)(kt & 1);
    load_tile<DP, BN, true>(sk + s * S::kStream, a, a.k, a.vec_k, b, kh, kt * BN, a.nk);
    load_tile<DP, BN, true>(sv + s * S::kStream, a, a.v, a.vec_v, b, kh, kt * BN, a.nk);
    cp_commit();
  };
  float acc[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  const RowConst rc = row_const(a, b, h, w0);
  if (nt > 0) issue(0);
  for (int64_t kt = 0; kt < nt; ++kt) {
    const uint64_t bits = seen_bits<BN>(a, b, kt * BN);
    cp_wait<0>();
    __syncthreads();
    if (kt + 1 < nt) issue(kt + 1);
    const int s = (int)(kt & 1);
    float x[BN / 8][4], y[BN / 8][4];
    if (w0 >= a.nq) continue;  // a warp past the end
    if (bits == 0) {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
    } else {
      M::nt(x, sq + warp * 16 * S::P, sk + s * S::kStream);
      M::nt(y, sg + warp * 16 * S::P, sv + s * S::kStream);
      add_bias<BN>(x, a, b, h, w0, kt * BN, bits);
      hide<BN>(x, bits);
      prob_ds_rows<BN>(x, y, rc.m, rc.c, rc.D, rc.peak);
      M::nn(acc, y, sc, sk + s * S::kStream);
    }
    if (a.dbias) store_dbias<BN>(a, b, h, w0, kt * BN, y);
  }
  cp_commit();
  cp_wait<0>();
  if (a.dq)
    store_rows<DP>(a.dq, b * a.o_bs + (int64_t)h * a.o_hs, a.o_ns, w0, a.nq, a.d, acc, a.scale, a.scale);
}

// dk and dv of one key tile: the transposed scores, keys down the rows.
template <int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dkv(Args a) {
  using M = Prod<DP, BN>;
  using S = Smem<DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sk = (float*)raw;
  float* sv = sk + S::kStat;
  float* sq = sv + S::kStat;        // [2]
  float* sg = sq + 2 * S::kStream;  // [2]
  __shared__ float4 cst[2][BN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* sc = sg + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int kh = (int)(id % a.KV), group = a.H / a.KV;
  const int64_t b = id / a.KV;
  const int64_t j0 = tile * BM, w0 = j0 + warp * 16;
  const int64_t per = (a.nq + BN - 1) / BN, nt = per * group;
  load_tile<DP, BM, true>(sk, a, a.k, a.vec_k, b, kh, j0, a.nk);
  load_tile<DP, BM, true>(sv, a, a.v, a.vec_v, b, kh, j0, a.nk);
  auto issue = [&](int64_t it) {
    const int s = (int)(it & 1), h = kh * group + (int)(it / per);
    const int64_t i0 = (it % per) * BN;
    load_tile<DP, BN, false>(sq + s * S::kStream, a, a.q, a.vec_q, b, h, i0, a.nq);
    load_tile<DP, BN, false>(sg + s * S::kStream, a, a.g, a.vec_g, b, h, i0, a.nq);
    cp_commit();
    for (int c = threadIdx.x; c < BN; c += kThreads) {
      const int64_t i = i0 + c;
      cst[s][c] = i < a.nq ? ((const float4*)a.rows)[(b * a.H + h) * a.nq + i] : make_float4(INFINITY, 0.f, 0.f, 0.f);
    }
  };
  bool seen[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t j = w0 + g + 8 * r;
    seen[r] = j < a.nk && key_seen(a, b, j);
  }
  float dk[DP / 8][4], dv[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;
  const bool any = __syncthreads_or(seen[0] || seen[1]);
  if (any && nt > 0) {
    issue(0);
    for (int64_t it = 0; it < nt; ++it) {
      const int s = (int)(it & 1), h = kh * group + (int)(it / per);
      const int64_t i0 = (it % per) * BN;
      cp_wait<0>();
      __syncthreads();
      if (it + 1 < nt) issue(it + 1);
      if (w0 >= a.nk) continue;  // a warp past the end
      float x[BN / 8][4], y[BN / 8][4];
      M::nt(x, sk + warp * 16 * S::P, sq + s * S::kStream);
      M::nt(y, sv + warp * 16 * S::P, sg + s * S::kStream);
      const int64_t off = b * a.b_bs + (int64_t)h * a.b_hs + w0 + g;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = n * 8 + 2 * t + e;
          const float4 rc = cst[s][c];
          const bool row = i0 + c < a.nq;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v = x[n][2 * r + e] * a.scale;
            if (a.bias && seen[r] && row) v += ld_bias1(a, off + (i0 + c) * a.b_rs + 8 * r);
            const float p = expf((seen[r] ? v : -INFINITY) - rc.x) * rc.y;
            x[n][2 * r + e] = p;
            y[n][2 * r + e] = rc.z != 0.f && p == 1.f ? 0.f : p * (y[n][2 * r + e] - rc.w);
          }
        }
      M::nn(dv, x, sc, sg + s * S::kStream);
      M::nn(dk, y, sc, sq + s * S::kStream);
    }
  }
  cp_commit();
  cp_wait<0>();
  store_rows<DP>(a.dk, b * a.dk_bs + (int64_t)kh * a.dk_hs, a.dk_ns, w0, a.nk, a.d, dk, a.scale, a.scale);
  store_rows<DP>(a.dv, b * a.dv_bs + (int64_t)kh * a.dv_hs, a.dv_ns, w0, a.nk, a.d, dv, 1.f, 1.f);
}

// dbias of one 64 x BN tile of the plane of head h, summed over a part of the batch: the result where there
// is one part, else an fp32 partial plane.
template <int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dbias(Args a, float* part, int parts) {
  using M = Prod<DP, BN>;
  using S = Smem<DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  float* sm[2] = {(float*)raw, (float*)raw + 2 * S::kStat + 2 * S::kStream};  // q, do, k, v of two batch entries
  const int warp = threadIdx.x >> 5;
  int64_t id = blockIdx.x;
  const int64_t nkt = (a.nk + BN - 1) / BN;
  const int64_t kt = id % nkt;
  id /= nkt;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int h = (int)(id % a.H), kh = h / (a.H / a.KV), pt = (int)(id / a.H);
  const int64_t b0 = a.B * pt / parts, b1 = a.B * (pt + 1) / parts;
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16, j0 = kt * BN;
  auto issue = [&](int64_t b) {
    float* p = sm[b & 1];
    load_tile<DP, BM, false>(p, a, a.q, a.vec_q, b, h, i0, a.nq);
    load_tile<DP, BM, false>(p + S::kStat, a, a.g, a.vec_g, b, h, i0, a.nq);
    load_tile<DP, BN, true>(p + 2 * S::kStat, a, a.k, a.vec_k, b, kh, j0, a.nk);
    load_tile<DP, BN, true>(p + 2 * S::kStat + S::kStream, a, a.v, a.vec_v, b, kh, j0, a.nk);
    cp_commit();
  };
  float acc[BN / 8][4];
#pragma unroll
  for (int n = 0; n < BN / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  if (b0 < b1) issue(b0);
  for (int64_t b = b0; b < b1; ++b) {
    const uint64_t bits = seen_bits<BN>(a, b, j0);
    cp_wait<0>();
    __syncthreads();
    if (b + 1 < b1) issue(b + 1);
    if (bits == 0 || w0 >= a.nq) continue;
    const float* p = sm[b & 1];
    const RowConst rc = row_const(a, b, h, w0);
    float x[BN / 8][4], y[BN / 8][4];
    M::nt(x, p + warp * 16 * S::P, p + 2 * S::kStat);
    M::nt(y, p + S::kStat + warp * 16 * S::P, p + 2 * S::kStat + S::kStream);
    add_bias<BN>(x, a, 0, h, w0, j0, bits);
    hide<BN>(x, bits);
    prob_ds_rows<BN>(x, y, rc.m, rc.c, rc.D, rc.peak);
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] += y[n][e];
  }
  cp_commit();
  cp_wait<0>();
  if (parts == 1) {
    store_dbias<BN>(a, 0, h, w0, j0, acc);
  } else {
    Args w = a;  // the part's plane in dbias's place
    w.dbias = part;
    w.bias_f32 = 1;
    w.db_vec = (a.nk & 3) == 0;
    w.db_rs = a.nk;
    w.db_hs = a.nq * a.nk;
    w.db_bs = a.H * a.nq * a.nk;
    store_dbias<BN>(w, pt, h, w0, j0, acc);
  }
}

// ---------------------------------------------------------------- launches

template <class F, class... X>
int go(F* kern, size_t smem, int64_t blocks, const char* name, double flops, cudaStream_t st, X... x) {
  if (blocks == 0) return PF_OK;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: %lld tiles are too many", (long long)blocks);
  if (smem > 40 * 1024)
    PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  {
    PF_LAUNCH_SCOPE_WORK(st, name, flops, 'f');
    kern<<<(unsigned)blocks, kThreads, smem, st>>>(x...);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

template <int DP>
int launch_t(Kind kind, Args a, double flops, cudaStream_t st) {
  constexpr int BN = 32;
  using S = Smem<DP, BN>;
  a.tiles = ((kind == kDkv ? a.nk : a.nq) + BM - 1) / BM;
  const int64_t blocks = a.tiles * (kind == kDkv ? a.KV : a.H) * a.B;
  if (kind == kFwd) return go(k_attn_fwd<DP, BN>, S::bytes(1, 2), blocks, "k_attn_fwd", flops, st, a);
  if (kind == kDq) return go(k_attn_dq<DP, BN>, S::bytes(2, 2), blocks, "k_attn_dq", flops, st, a);
  return go(k_attn_dkv<DP, BN>, S::bytes(2, 2), blocks, "k_attn_dkv", flops, st, a);
}
template <int DP>
int launch_db(Args a, float* part, int parts, double flops, cudaStream_t st) {
  constexpr int BN = 32;
  a.tiles = (a.nq + BM - 1) / BM;
  return go(k_attn_dbias<DP, BN>, Smem<DP, BN>::bytes(4, 2), a.tiles * ((a.nk + BN - 1) / BN) * a.H * parts,
            "k_attn_dbias", flops, st, a, part, parts);
}

}  // namespace

int launch_f32(Kind kind, const Args& a, double flops, cudaStream_t st) {
  if (a.d <= 32) return launch_t<32>(kind, a, flops, st);
  if (a.d <= 64) return launch_t<64>(kind, a, flops, st);
  if (a.d <= 96) return launch_t<96>(kind, a, flops, st);
  return launch_t<128>(kind, a, flops, st);
}
int dbias_f32(const Args& a, float* part, int parts, double flops, cudaStream_t st) {
  if (a.d <= 32) return launch_db<32>(a, part, parts, flops, st);
  if (a.d <= 64) return launch_db<64>(a, part, parts, flops, st);
  if (a.d <= 96) return launch_db<96>(a, part, parts, flops, st);
  return launch_db<128>(a, part, parts, flops, st);
}
int rows_f32(const Args& a, const float* stats, Heads o, float* rows, cudaStream_t st) {
  const int64_t blocks = (a.rows_plane + 31) / 32;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: too many rows");
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_rows", (8.0 * a.d + 24.0) * (double)a.rows_plane, 'b');
    k_rows<<<(unsigned)blocks, 256, 0, st>>>(a, stats, o, (float4*)rows);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

}  // namespace attn
}  // namespace train
}  // namespace pf
