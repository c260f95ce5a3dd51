// pf_attention.cuh -- attention with a learned bias, forward and backward, by tiles (both storage
// types); included by pf_attention_bf16.cu and pf_attention_f32.cu, dispatched by pf_attention.cu.
//
// For one batch entry b and head h (key head h / (H / KV)), with t_ij = scale q_i.k_j + bias_ij over
// the keys j that the mask leaves:
//   m_i = max_j t_ij,  l_i = sum_j exp(t_ij - m_i),  p_ij = exp(t_ij - m_i) / l_i,  o_i = sum_j p_ij v_j
//   D_i = do_i.o_i,  dp_ij = do_i.v_j,  ds_ij = p_ij (dp_ij - D_i)
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i,  dbias = ds
// The forward is one pass over the keys with the running m and l. It keeps m and l (not m + log l:
// next to a bias of the type's lowest value log l would be lost) and the low half of o (below).
// The backward recomputes p from them tile by tile, so no [n_q, n_k] array but dbias is written:
//   k_attn_rows   D and the row constants of p
//   k_attn_dkv    one block per key tile, loops over the query heads of its key head and their queries:
//                 computes the transposed scores, so that p^T and ds^T are the left operands of dv, dk
//   k_attn_dq     one block per query tile, loops over the keys: dq, and dbias where it has no sum
//   k_attn_dbias  a bias shared by the batch: one block per tile of the [n_q, n_k] plane loops over the
//                 batch and adds ds in registers, so the sum has a fixed order and needs no atomics
// All four multiply a stationary tile of 64 rows (16 per warp) with streamed tiles of BN rows that
// cp.async double-buffers in shared memory.
//
// Arithmetic: bf16 operands go through m16n8k16 tensor-core products with fp32 accumulation; in the
// backward p and ds are rounded to bf16 as operands of the second product (one rounding of the operand's
// own type), all else -- scores, softmax statistics, D, the sum over a shared bias's batch, accumulators --
// is fp32. fp32 operands use FFMA on the same register layout. ds is a difference of dp and D, so an
// error of o would be its largest: the forward multiplies p as a sum of two bf16 values (three where the
// bias is fp32, whose gradient then keeps fp32's accuracy), D is formed from o before its rounding, and
// for that the forward keeps the 16 bits of o that the rounding dropped.
//
// Rows: a row that sees no key has m = -inf, l = 0; its o and gradients are 0. Masked keys are never
// read (their rows are zero-filled), so NaN there does no harm; their bias is not used either. Where p
// is exactly 1 in fp32, ds is set to 0: a row with one visible key has none, and dp - D would leave
// rounding noise in its place.
#pragma once

#include "pf_common.cuh"
#include "pf_prof.h"
#include "pf_train.h"

namespace pf {
namespace train {
namespace attn {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int BM = kWarps * 16;  // rows of a stationary tile

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
  int bias_f32, bias_vec, db_vec;  // storage, and whether pairs of keys are aligned
  const float* mask;
  int64_t m_bs, m_ks;
  float* stats;         // forward: m [B][H][n_q], then l
  int16_t* o_lo;        // [B][n_q][H][d]
  const float* rows;    // backward: m', c, D, each [B][H][n_q]
  int64_t rows_plane;   // B * H * n_q
  int64_t B, nq, nk;
  int H, KV, d;
  float scale;
  int vec_q, vec_k, vec_v, vec_g;  // 16-byte accesses allowed
  int p_terms;                     // forward, bf16: bf16 values that p is split into
  int64_t tiles;                   // tiles along the split axis of this launch
};

// ---------------------------------------------------------------- tiles

template <class T, int DP>
struct Pitch {
  static constexpr int value = DP + 16 / (int)sizeof(T);  // rows shifted by 16 bytes: no bank conflicts
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

__device__ __forceinline__ bool key_seen(const Args& a, int64_t b, int64_t j) {
  return a.mask == nullptr || a.mask[b * a.m_bs + j * a.m_ks] != 0.f;
}

// Rows [r0, r0 + ROWS) of (b, h) into shared memory, zero past n and d, and where MASKED for masked keys.
template <class T, int DP, int ROWS, bool MASKED>
__device__ __forceinline__ void load_tile(T* sm, const Args& a, const Heads& s, int vec, int64_t b, int h, int64_t r0,
                                          int64_t n) {
  constexpr int P = Pitch<T, DP>::value, E = 16 / (int)sizeof(T), CH = DP / E;
  const T* base = (const T*)s.p + b * s.bs + (int64_t)h * s.hs;
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
      sm[r * P + c] = ok ? base[row * s.ns + c] : from_f<T>(0.f);
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

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <class T, int DP, int BN>
struct Prod;

template <int DP, int BN>
struct Prod<__nv_bfloat16, DP, BN> {
  using T = __nv_bfloat16;
  static constexpr int P = Pitch<T, DP>::value;
  struct Stat {  // the warp's 16 rows of a stationary tile as left operands
    uint32_t a[DP / 16][4];
  };
  static __device__ void fetch(Stat& s, const T* sm) {
    const int lane = threadIdx.x & 31;
    const uint32_t base = smem_addr(sm + (lane & 15) * P + (lane >> 4) * 8);
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) ldsm4(s.a[k], base + k * 32);
  }
  // c[16 x BN] = a[16 x DP] b[BN x DP]^T
  static __device__ void nt(float (&c)[BN / 8][4], const Stat& s, const T*, const T* b) {
    const int lane = threadIdx.x & 31;
    const uint32_t base = smem_addr(b + ((lane & 7) + ((lane >> 4) & 1) * 8) * P + ((lane >> 3) & 1) * 8);
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int n = 0; n < BN / 16; ++n) {
        uint32_t r[4];
        ldsm4(r, base + (n * 16 * P + k * 16) * 2);
        mma_bf16(c[2 * n], s.a[k], r[0], r[1]);
        mma_bf16(c[2 * n + 1], s.a[k], r[2], r[3]);
      }
  }
  // acc[16 x DP] += p[16 x BN] b[BN x DP]
  static __device__ void nn(float (&acc)[DP / 8][4], const float (&p)[BN / 8][4], T*, const T* b) {
    const int lane = threadIdx.x & 31;
    const uint32_t base = smem_addr(b + (lane & 15) * P + (lane >> 4) * 8);
#pragma unroll
    for (int k = 0; k < BN / 16; ++k) {
      const uint32_t a[4] = {pack_bf16(p[2 * k][0], p[2 * k][1]), pack_bf16(p[2 * k][2], p[2 * k][3]),
                             pack_bf16(p[2 * k + 1][0], p[2 * k + 1][1]), pack_bf16(p[2 * k + 1][2], p[2 * k + 1][3])};
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        uint32_t r[4];
        ldsm4_t(r, base + (k * 16 * P + n * 16) * 2);
        mma_bf16(acc[2 * n], a, r[0], r[1]);
        mma_bf16(acc[2 * n + 1], a, r[2], r[3]);
      }
    }
  }
  // the same with p as a sum of `terms` bf16 values (8 bits each)
  static __device__ void nn_split(float (&acc)[DP / 8][4], const float (&p)[BN / 8][4], T*, const T* b, int terms) {
    const int lane = threadIdx.x & 31;
    const uint32_t base = smem_addr(b + (lane & 15) * P + (lane >> 4) * 8);
#pragma unroll
    for (int k = 0; k < BN / 16; ++k) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = p[2 * k + (e >> 2)][e & 3];
      for (int term = 0; term < terms; ++term) {
        uint32_t a[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          a[e] = pack_bf16(x[2 * e], x[2 * e + 1]);
          x[2 * e] -= __uint_as_float(a[e] << 16);
          x[2 * e + 1] -= __uint_as_float(a[e] & 0xffff0000u);
        }
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
          uint32_t r[4];
          ldsm4_t(r, base + (k * 16 * P + n * 16) * 2);
          mma_bf16(acc[2 * n], a, r[0], r[1]);
          mma_bf16(acc[2 * n + 1], a, r[2], r[3]);
        }
      }
    }
  }
};

template <int DP, int BN>
struct Prod<float, DP, BN> {
  using T = float;
  static constexpr int P = Pitch<T, DP>::value;
  struct Stat {};
  static __device__ void fetch(Stat&, const T*) {}
  static __device__ void nt(float (&c)[BN / 8][4], const Stat&, const T* a, const T* b) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) c[n][0] = c[n][1] = c[n][2] = c[n][3] = 0.f;
#pragma unroll 4
    for (int k = 0; k < DP; k += 4) {
      const float4 a0 = *reinterpret_cast<const float4*>(a + g * P + k);
      const float4 a1 = *reinterpret_cast<const float4*>(a + (g + 8) * P + k);
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) {
        const float4 b0 = *reinterpret_cast<const float4*>(b + (n * 8 + 2 * t) * P + k);
        const float4 b1 = *reinterpret_cast<const float4*>(b + (n * 8 + 2 * t + 1) * P + k);
        c[n][0] += a0.x * b0.x + a0.y * b0.y + a0.z * b0.z + a0.w * b0.w;
        c[n][1] += a0.x * b1.x + a0.y * b1.y + a0.z * b1.z + a0.w * b1.w;
        c[n][2] += a1.x * b0.x + a1.y * b0.y + a1.z * b0.z + a1.w * b0.w;
        c[n][3] += a1.x * b1.x + a1.y * b1.y + a1.z * b1.z + a1.w * b1.w;
      }
    }
  }
  static __device__ void nn_split(float (&acc)[DP / 8][4], const float (&p)[BN / 8][4], T* sc, const T* b, int) {
    nn(acc, p, sc, b);
  }
  // p goes through the warp's scratch rows [16][BN + 4]
  static __device__ void nn(float (&acc)[DP / 8][4], const float (&p)[BN / 8][4], T* sc, const T* b) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    constexpr int Q = BN + 4;
    __syncwarp();
#pragma unroll
    for (int n = 0; n < BN / 8; ++n) {
      *reinterpret_cast<float2*>(sc + g * Q + n * 8 + 2 * t) = make_float2(p[n][0], p[n][1]);
      *reinterpret_cast<float2*>(sc + (g + 8) * Q + n * 8 + 2 * t) = make_float2(p[n][2], p[n][3]);
    }
    __syncwarp();
#pragma unroll 2
    for (int k = 0; k < BN; k += 4) {
      const float4 a0 = *reinterpret_cast<const float4*>(sc + g * Q + k);
      const float4 a1 = *reinterpret_cast<const float4*>(sc + (g + 8) * Q + k);
      const float x0[4] = {a0.x, a0.y, a0.z, a0.w}, x1[4] = {a1.x, a1.y, a1.z, a1.w};
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int n = 0; n < DP / 8; ++n) {
          const float2 v = *reinterpret_cast<const float2*>(b + (k + u) * P + n * 8 + 2 * t);
          acc[n][0] += x0[u] * v.x;
          acc[n][1] += x0[u] * v.y;
          acc[n][2] += x1[u] * v.x;
          acc[n][3] += x1[u] * v.y;
        }
    }
  }
};

// ---------------------------------------------------------------- shared-memory plan

template <class T, int DP, int BN>
struct Smem {
  static constexpr int P = Pitch<T, DP>::value;
  static constexpr int kStat = BM * P, kStream = BN * P;  // elements
  static constexpr int kScratch = sizeof(T) == 4 ? kWarps * 16 * (BN + 4) : 0;
  // nstat stationary tiles, nstream streamed tiles (double-buffered), the products' scratch rows
  static size_t bytes(int nstat, int nstream) {
    return ((size_t)nstat * kStat + 2 * (size_t)nstream * kStream + kScratch) * sizeof(T);
  }
};

// ---------------------------------------------------------------- scores

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T>
__device__ __forceinline__ float exp_shift(float t, float m) {  // exp(t - m)
  if (sizeof(T) == 4) return expf(t - m);
  // t - m first: with the type's lowest value as t and m, t * log2(e) would overflow
  return ex2((t - m) * 1.4426950408889634f);
}

// The row constant beside m: 1 / l (fp32), or -log2 l folded into the exponent (bf16).
template <class T>
__device__ __forceinline__ float prob(float t, float m, float c) {
  if (sizeof(T) == 4) return expf(t - m) * c;
  return ex2(fmaf(t - m, 1.4426950408889634f, c));
}

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
template <class T, int BN>
__device__ __forceinline__ void prob_ds_rows(float (&s)[BN / 8][4], float (&dp)[BN / 8][4], const float* m,
                                             const float* c, const float* D) {
#pragma unroll
  for (int n = 0; n < BN / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = prob<T>(s[n][e], m[e >> 1], c[e >> 1]);
      s[n][e] = p;
      dp[n][e] = p == 1.f ? 0.f : p * (dp[n][e] - D[e >> 1]);
    }
}

template <class T, int DP>
__device__ __forceinline__ void store_rows(void* out, int64_t off, int64_t ns, int64_t i0, int64_t n, int d,
                                           const float (&acc)[DP / 8][4], float f0, float f1) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = i0 + g + 8 * r;
    if (i >= n) continue;
    T* p = (T*)out + off + i * ns;
    const float f = r ? f1 : f0;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = c * 8 + 2 * t + e;
        if (col < d) p[col] = from_f<T>(acc[c][2 * r + e] * f);
      }
  }
}

// ---------------------------------------------------------------- forward

template <class T, int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_fwd(Args a) {
  using M = Prod<T, DP, BN>;
  using S = Smem<T, DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  T* sq = (T*)raw;
  T* sk = sq + S::kStat;           // [2]
  T* sv = sk + 2 * S::kStream;     // [2]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  T* sc = sv + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int h = (int)(id % a.H), kh = h / (a.H / a.KV);
  const int64_t b = id / a.H;
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16;
  const int64_t nt = (a.nk + BN - 1) / BN;
  load_tile<T, DP, BM, false>(sq, a, a.q, a.vec_q, b, h, i0, a.nq);
  auto issue = [&](int64_t kt) {
    const int s = (int)(kt & 1);
    load_tile<T, DP, BN, true>(sk + s * S::kStream, a, a.k, a.vec_k, b, kh, kt * BN, a.nk);
    load_tile<T, DP, BN, true>(sv + s * S::kStream, a, a.v, a.vec_v, b, kh, kt * BN, a.nk);
    cp_commit();
  };
  float acc[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  typename M::Stat fq;
  if (nt > 0) issue(0);
  for (int64_t kt = 0; kt < nt; ++kt) {
    const uint64_t bits = seen_bits<BN>(a, b, kt * BN);
    cp_wait<0>();
    __syncthreads();
    if (kt == 0) M::fetch(fq, sq + warp * 16 * S::P);
    if (kt + 1 < nt) issue(kt + 1);
    if (bits == 0) continue;  // the same for the whole block
    const int s = (int)(kt & 1);
    float x[BN / 8][4];
    M::nt(x, fq, sq + warp * 16 * S::P, sk + s * S::kStream);
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
      const float corr = exp_shift<T>(m[r], base);
      m[r] = mx;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float p = exp_shift<T>(x[n][2 * r + e], base);
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
    M::nn_split(acc, x, sc, sv + s * S::kStream, a.p_terms);
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
    T* o = (T*)a.o + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
    int16_t* lo = a.o_lo ? a.o_lo + ((b * a.nq + i) * a.H + h) * a.d : nullptr;
#pragma unroll
    for (int c = 0; c < DP / 8; ++c)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int col = c * 8 + 2 * t + e;
        if (col >= a.d) continue;
        const float v = acc[c][2 * r + e] * inv;
        const T y = from_f<T>(v);
        o[col] = y;
        if (sizeof(T) == 2 && lo) {
          // fp32 bits of o less those of its bf16 rounding: o is their sum again (a tie that rounds
          // down would need one more than 16 bits hold and loses the last bit; NaN keeps none)
          const int diff = (int)(__float_as_uint(v) - __float_as_uint(to_f(y)));
          lo[col] = v == v ? (int16_t)min(diff, 32767) : (int16_t)0;
        }
      }
  }
}

// ---------------------------------------------------------------- backward

// D and the row constants: eight lanes per row (b, i, h).
template <class T>
__global__ void __launch_bounds__(256) k_attn_rows(Args a, const float* __restrict__ stats, Heads o,
                                                   const int16_t* __restrict__ lo, float* __restrict__ rows) {
  const int sub = threadIdx.x & 7;
  const int64_t r = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);
  const bool live = r < a.rows_plane;
  const int64_t rr = live ? r : 0;
  const int h = (int)(rr % a.H);
  const int64_t bi = rr / a.H, b = bi / a.nq, i = bi - b * a.nq;
  const T* po = (const T*)o.p + b * o.bs + i * o.ns + (int64_t)h * o.hs;
  const T* pg = (const T*)a.g.p + b * a.g.bs + i * a.g.ns + (int64_t)h * a.g.hs;
  float s = 0.f;
  if (live)
    for (int e = sub; e < a.d; e += 8) {
      float v = to_f(po[e]);
      if (sizeof(T) == 2 && v == v) v = __uint_as_float(__float_as_uint(v) + (int)lo[rr * a.d + e]);
      s += v * to_f(pg[e]);
    }
  s += __shfl_xor_sync(0xffffffffu, s, 1);
  s += __shfl_xor_sync(0xffffffffu, s, 2);
  s += __shfl_xor_sync(0xffffffffu, s, 4);
  if (!live || sub) return;
  const int64_t at = (b * a.H + h) * a.nq + i;
  const float m = stats[at], l = stats[a.rows_plane + at];
  const bool none = l == 0.f;  // sees nothing: p = exp(t - inf) = 0
  rows[at] = none ? INFINITY : m;
  rows[a.rows_plane + at] = none ? 0.f : (sizeof(T) == 4 ? 1.f / l : -log2f(l));
  rows[2 * a.rows_plane + at] = none ? 0.f : s;
}

struct RowConst {
  float m[2], c[2], D[2];
};
__device__ __forceinline__ RowConst row_const(const Args& a, int64_t b, int h, int64_t i0) {
  const int g = (threadIdx.x & 31) >> 2;
  RowConst r;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t i = i0 + g + 8 * k, at = (b * a.H + h) * a.nq + i;
    const bool ok = i < a.nq;
    r.m[k] = ok ? a.rows[at] : INFINITY;
    r.c[k] = ok ? a.rows[a.rows_plane + at] : 0.f;
    r.D[k] = ok ? a.rows[2 * a.rows_plane + at] : 0.f;
  }
  return r;
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
              pack_bf16(ds[n][2 * r], ds[n][2 * r + 1]);
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
template <class T, int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dq(Args a) {
  using M = Prod<T, DP, BN>;
  using S = Smem<T, DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  T* sq = (T*)raw;
  T* sg = sq + S::kStat;
  T* sk = sg + S::kStat;        // [2]
  T* sv = sk + 2 * S::kStream;  // [2]
  const int warp = threadIdx.x >> 5;
  T* sc = sv + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int h = (int)(id % a.H), kh = h / (a.H / a.KV);
  const int64_t b = id / a.H;
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16;
  const int64_t nt = (a.nk + BN - 1) / BN;
  load_tile<T, DP, BM, false>(sq, a, a.q, a.vec_q, b, h, i0, a.nq);
  load_tile<T, DP, BM, false>(sg, a, a.g, a.vec_g, b, h, i0, a.nq);
  auto issue = [&](int64_t kt) {
    const int s = (int)(kt & 1);
    load_tile<T, DP, BN, true>(sk + s * S::kStream, a, a.k, a.vec_k, b, kh, kt * BN, a.nk);
    load_tile<T, DP, BN, true>(sv + s * S::kStream, a, a.v, a.vec_v, b, kh, kt * BN, a.nk);
    cp_commit();
  };
  float acc[DP / 8][4];
#pragma unroll
  for (int n = 0; n < DP / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  const RowConst rc = row_const(a, b, h, w0);
  typename M::Stat fq, fg;
  if (nt > 0) issue(0);
  for (int64_t kt = 0; kt < nt; ++kt) {
    const uint64_t bits = seen_bits<BN>(a, b, kt * BN);
    cp_wait<0>();
    __syncthreads();
    if (kt == 0) {
      M::fetch(fq, sq + warp * 16 * S::P);
      M::fetch(fg, sg + warp * 16 * S::P);
    }
    if (kt + 1 < nt) issue(kt + 1);
    const int s = (int)(kt & 1);
    float x[BN / 8][4], y[BN / 8][4];
    if (bits == 0) {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.f;
    } else {
      M::nt(x, fq, sq + warp * 16 * S::P, sk + s * S::kStream);
      M::nt(y, fg, sg + warp * 16 * S::P, sv + s * S::kStream);
      add_bias<BN>(x, a, b, h, w0, kt * BN, bits);
      hide<BN>(x, bits);
      prob_ds_rows<T, BN>(x, y, rc.m, rc.c, rc.D);
      M::nn(acc, y, sc, sk + s * S::kStream);
    }
    if (a.dbias) store_dbias<BN>(a, b, h, w0, kt * BN, y);
  }
  cp_commit();
  cp_wait<0>();
  if (a.dq)
    store_rows<T, DP>(a.dq, b * a.o_bs + (int64_t)h * a.o_hs, a.o_ns, w0, a.nq, a.d, acc, a.scale, a.scale);
}

// dk and dv of one key tile: the transposed scores, keys down the rows.
template <class T, int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dkv(Args a) {
  using M = Prod<T, DP, BN>;
  using S = Smem<T, DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  T* sk = (T*)raw;
  T* sv = sk + S::kStat;
  T* sq = sv + S::kStat;        // [2]
  T* sg = sq + 2 * S::kStream;  // [2]
  __shared__ float cst[2][3][BN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  T* sc = sg + 2 * S::kStream + warp * 16 * (BN + 4);
  int64_t id = blockIdx.x;
  const int64_t tile = id % a.tiles;
  id /= a.tiles;
  const int kh = (int)(id % a.KV), group = a.H / a.KV;
  const int64_t b = id / a.KV;
  const int64_t j0 = tile * BM, w0 = j0 + warp * 16;
  const int64_t per = (a.nq + BN - 1) / BN, nt = per * group;
  load_tile<T, DP, BM, true>(sk, a, a.k, a.vec_k, b, kh, j0, a.nk);
  load_tile<T, DP, BM, true>(sv, a, a.v, a.vec_v, b, kh, j0, a.nk);
  auto issue = [&](int64_t it) {
    const int s = (int)(it & 1), h = kh * group + (int)(it / per);
    const int64_t i0 = (it % per) * BN;
    load_tile<T, DP, BN, false>(sq + s * S::kStream, a, a.q, a.vec_q, b, h, i0, a.nq);
    load_tile<T, DP, BN, false>(sg + s * S::kStream, a, a.g, a.vec_g, b, h, i0, a.nq);
    cp_commit();
    for (int c = threadIdx.x; c < BN; c += kThreads) {
      const int64_t i = i0 + c, at = (b * a.H + h) * a.nq + i;
      const bool ok = i < a.nq;
      cst[s][0][c] = ok ? a.rows[at] : INFINITY;
      cst[s][1][c] = ok ? a.rows[a.rows_plane + at] : 0.f;
      cst[s][2][c] = ok ? a.rows[2 * a.rows_plane + at] : 0.f;
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
  typename M::Stat fk, fv;
  if (any && nt > 0) {
    issue(0);
    for (int64_t it = 0; it < nt; ++it) {
      const int s = (int)(it & 1), h = kh * group + (int)(it / per);
      const int64_t i0 = (it % per) * BN;
      cp_wait<0>();
      __syncthreads();
      if (it == 0) {
        M::fetch(fk, sk + warp * 16 * S::P);
        M::fetch(fv, sv + warp * 16 * S::P);
      }
      if (it + 1 < nt) issue(it + 1);
      float x[BN / 8][4], y[BN / 8][4];
      M::nt(x, fk, sk + warp * 16 * S::P, sq + s * S::kStream);
      M::nt(y, fv, sv + warp * 16 * S::P, sg + s * S::kStream);
      const int64_t off = b * a.b_bs + (int64_t)h * a.b_hs + w0 + g;
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int c = n * 8 + 2 * t + e;
          const float m = cst[s][0][c], k = cst[s][1][c], D = cst[s][2][c];
          const bool row = i0 + c < a.nq;
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float v = x[n][2 * r + e] * a.scale;
            if (a.bias && seen[r] && row) v += ld_bias1(a, off + (i0 + c) * a.b_rs + 8 * r);
            const float p = prob<T>(seen[r] ? v : -INFINITY, m, k);
            x[n][2 * r + e] = p;
            y[n][2 * r + e] = p == 1.f ? 0.f : p * (y[n][2 * r + e] - D);
          }
        }
      M::nn(dv, x, sc, sg + s * S::kStream);
      M::nn(dk, y, sc, sq + s * S::kStream);
    }
  }
  cp_commit();
  cp_wait<0>();
  store_rows<T, DP>(a.dk, b * a.dk_bs + (int64_t)kh * a.dk_hs, a.dk_ns, w0, a.nk, a.d, dk, a.scale, a.scale);
  store_rows<T, DP>(a.dv, b * a.dv_bs + (int64_t)kh * a.dv_hs, a.dv_ns, w0, a.nk, a.d, dv, 1.f, 1.f);
}

// dbias of one 64 x BN tile of the plane of head h, summed over the batch.
template <class T, int DP, int BN>
__global__ void __launch_bounds__(kThreads) k_attn_dbias(Args a) {
  using M = Prod<T, DP, BN>;
  using S = Smem<T, DP, BN>;
  extern __shared__ __align__(16) unsigned char raw[];
  T* sm[2] = {(T*)raw, (T*)raw + 2 * S::kStat + 2 * S::kStream};  // q, do, k, v of two batch entries
  const int warp = threadIdx.x >> 5;
  int64_t id = blockIdx.x;
  const int64_t nkt = (a.nk + BN - 1) / BN;
  const int64_t kt = id % nkt;
  id /= nkt;
  const int64_t tile = id % a.tiles;
  const int h = (int)(id / a.tiles), kh = h / (a.H / a.KV);
  const int64_t i0 = tile * BM, w0 = i0 + warp * 16, j0 = kt * BN;
  auto issue = [&](int64_t b) {
    T* p = sm[b & 1];
    load_tile<T, DP, BM, false>(p, a, a.q, a.vec_q, b, h, i0, a.nq);
    load_tile<T, DP, BM, false>(p + S::kStat, a, a.g, a.vec_g, b, h, i0, a.nq);
    load_tile<T, DP, BN, true>(p + 2 * S::kStat, a, a.k, a.vec_k, b, kh, j0, a.nk);
    load_tile<T, DP, BN, true>(p + 2 * S::kStat + S::kStream, a, a.v, a.vec_v, b, kh, j0, a.nk);
    cp_commit();
  };
  float acc[BN / 8][4];
#pragma unroll
  for (int n = 0; n < BN / 8; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
  issue(0);
  for (int64_t b = 0; b < a.B; ++b) {
    const uint64_t bits = seen_bits<BN>(a, b, j0);
    cp_wait<0>();
    __syncthreads();
    if (b + 1 < a.B) issue(b + 1);
    if (bits == 0) continue;
    const T* p = sm[b & 1];
    typename M::Stat fq, fg;
    M::fetch(fq, p + warp * 16 * S::P);
    M::fetch(fg, p + S::kStat + warp * 16 * S::P);
    const RowConst rc = row_const(a, b, h, w0);
    float x[BN / 8][4], y[BN / 8][4];
    M::nt(x, fq, p + warp * 16 * S::P, p + 2 * S::kStat);
    M::nt(y, fg, p + S::kStat + warp * 16 * S::P, p + 2 * S::kStat + S::kStream);
    add_bias<BN>(x, a, 0, h, w0, j0, bits);
    hide<BN>(x, bits);
    prob_ds_rows<T, BN>(x, y, rc.m, rc.c, rc.D);
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] += y[n][e];
  }
  cp_wait<0>();
  store_dbias<BN>(a, 0, h, w0, j0, acc);
}

// ---------------------------------------------------------------- launches

enum Kind { kFwd, kDq, kDkv, kDbias };

template <class T, int DP, int BN>
int launch_kind(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st) {
  using S = Smem<T, DP, BN>;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: %lld tiles are too many", (long long)blocks);
  void (*kern)(Args) = nullptr;
  size_t smem = 0;
  const char* name = nullptr;
  switch (kind) {
    case kFwd: kern = k_attn_fwd<T, DP, BN>; smem = S::bytes(1, 2); name = "k_attn_fwd"; break;
    case kDq: kern = k_attn_dq<T, DP, BN>; smem = S::bytes(2, 2); name = "k_attn_dq"; break;
    case kDkv: kern = k_attn_dkv<T, DP, BN>; smem = S::bytes(2, 2); name = "k_attn_dkv"; break;
    case kDbias: kern = k_attn_dbias<T, DP, BN>; smem = S::bytes(4, 2); name = "k_attn_dbias"; break;
  }
  if (smem > 40 * 1024)
    PF_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  {
    PF_LAUNCH_SCOPE_WORK(st, name, flops, 'f');
    kern<<<(unsigned)blocks, kThreads, smem, st>>>(a);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// The rows of a streamed tile: 64 where two score tiles and the accumulators fit in registers, else 32.
template <class T>
int launch_dim(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st) {
  constexpr int N1 = sizeof(T) == 2 ? 64 : 32;
  if (a.d <= 32) return launch_kind<T, 32, N1>(kind, a, blocks, flops, st);
  if (a.d <= 64) return launch_kind<T, 64, N1>(kind, a, blocks, flops, st);
  if (a.d <= 96) return launch_kind<T, 96, 32>(kind, a, blocks, flops, st);
  return launch_kind<T, 128, 32>(kind, a, blocks, flops, st);
}
inline int stream_rows(int dtype, int d) { return dtype == PF_BF16 && d <= 64 ? 64 : 32; }

template <class T>
int launch_rows(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st) {
  const int64_t blocks = (a.rows_plane + 31) / 32;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: too many rows");
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_rows", (2.0 * sizeof(T) * a.d + 20.0) * (double)a.rows_plane, 'b');
    k_attn_rows<T><<<(unsigned)blocks, 256, 0, st>>>(a, stats, o, lo, rows);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// one translation unit per storage type
int launch_bf16(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st);
int launch_f32(Kind kind, const Args& a, int64_t blocks, double flops, cudaStream_t st);
int rows_bf16(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st);
int rows_f32(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st);

}  // namespace attn
}  // namespace train
}  // namespace pf
