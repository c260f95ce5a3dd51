// pf_attention_tc.cuh -- building blocks of the tensor-core attention kernels (pf_attention_bf16.cu,
// pf_attention_f32.cu): swizzled shared tiles and their ldmatrix addresses, products, visible keys, bias
// fragments, scores. See pf_attention_bf16.cu for the layout.
#pragma once
#include <cooperative_groups.h>

#include <type_traits>

#include "pf_attention.cuh"
#include "pf_f32x2.cuh"

namespace pf {
namespace train {
namespace attn {
namespace {

using bf16 = __nv_bfloat16;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kTile = 64;  // rows of a streamed tile

// ---------------------------------------------------------------- shared tiles

template <int DP>
struct Tile {
  static constexpr int RB = DP == 96 ? 256 : DP * 2;  // bytes of a row
  static constexpr int CH = DP / 8;                   // 16-byte chunks in use
  static __device__ __forceinline__ int swz(int row) {
    return DP == 32 ? ((row >> 1) & 3) ^ ((row >> 3) & 1) : (row & 7) ^ (((row >> 3) & 1) << 1);
  }
  static __device__ __forceinline__ uint32_t off(int row, int ch) { return row * RB + ((ch ^ swz(row)) << 4); }
};

// A lane's row address inside a block of 16 rows for one ldmatrix.x4 pattern.
template <int DP>
struct LaneAddr {
  uint32_t rb, v;
  __device__ __forceinline__ LaneAddr(int row, int ch) : rb(row * Tile<DP>::RB), v(ch ^ Tile<DP>::swz(row)) {}
  // rows 16 blk.. of the tile at `base`, chunks 2 pair, 2 pair + 1
  __device__ __forceinline__ uint32_t at(uint32_t base, int blk, int pair) const {
    return base + blk * 16 * Tile<DP>::RB + rb + (((uint32_t)(2 * pair) ^ v) << 4);
  }
};
__device__ __forceinline__ int perm_row(int r, int half) { return 4 * (r >> 1) + (r & 1) + 2 * half; }
// left operand, natural rows
template <int DP>
__device__ __forceinline__ LaneAddr<DP> lane_a() {
  const int l = threadIdx.x & 31;
  return LaneAddr<DP>(l & 15, l >> 4);
}
// right operand with the depth along the row (keys are its columns, permuted)
template <int DP>
__device__ __forceinline__ LaneAddr<DP> lane_b() {
  const int l = threadIdx.x & 31;
  return LaneAddr<DP>(perm_row(l & 7, l >> 4), (l >> 3) & 1);
}
// right operand with the depth down the rows (transposing load): permuted keys, or natural rows
template <int DP>
__device__ __forceinline__ LaneAddr<DP> lane_bt() {
  const int l = threadIdx.x & 31;
  return LaneAddr<DP>(perm_row(l & 7, (l >> 3) & 1), l >> 4);
}
template <int DP>
__device__ __forceinline__ LaneAddr<DP> lane_bn() {
  const int l = threadIdx.x & 31;
  return LaneAddr<DP>(l & 15, l >> 4);
}

__device__ __forceinline__ void ldsm4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
// the same at a constant offset from the address
template <int OFF>
__device__ __forceinline__ void ldsm4i(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF));
}
template <int OFF>
__device__ __forceinline__ void ldsm4_ti(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4+%5];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr), "n"(OFF));
}
// f(0) .. f(N - 1) with constant arguments
template <int N, int I = 0, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    unrolled<N, I + 1>(f);
  }
}
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// the first product of a sum
__device__ __forceinline__ void mma0(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float lo_f(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_f(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// Rows [r0, r0 + ROWS) of (b, h), zero past n and d and where `live` has no bit for a row (tiles of 64).
template <int DP, int ROWS>
__device__ __forceinline__ void load_rows(uint32_t sm, const bf16* base, int64_t ns, int vec, int64_t r0, int64_t n,
                                          int d, uint64_t live) {
  constexpr int CH = Tile<DP>::CH;
  if (vec) {
#pragma unroll
    for (int i = threadIdx.x; i < ROWS * CH; i += kThreads) {
      const int r = i / CH, c = i - r * CH;
      const bool ok = r0 + r < n && c * 8 < d && ((live >> (r & 63)) & 1);
      cp_async16(sm + Tile<DP>::off(r, c), ok ? base + (r0 + r) * ns + c * 8 : base, ok);
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * DP; i += kThreads) {
      const int r = i / DP, c = i - r * DP;
      const bool ok = r0 + r < n && c < d && ((live >> (r & 63)) & 1);
      const bf16 x = ok ? base[(r0 + r) * ns + c] : from_f<bf16>(0.f);
      asm volatile("st.shared.b16 [%0], %1;" ::"r"(sm + Tile<DP>::off(r, c >> 3) + (c & 7) * 2),
                   "h"(*reinterpret_cast<const unsigned short*>(&x))
                   : "memory");
    }
  }
}
__device__ __forceinline__ const bf16* head_base(const Heads& s, int64_t b, int h) {
  return (const bf16*)s.p + b * s.bs + (int64_t)h * s.hs;
}

// One operand's tiles of 64 rows, one after the other: a thread keeps its place in the tile, so a tile costs
// an add and a copy for each of its chunks.
template <int DP>
struct Stream {
  static constexpr int CH = Tile<DP>::CH;
  static constexpr bool kPlain = kThreads % CH == 0;  // else rows and chunks of a thread change from pass to pass
  static constexpr int RP = kThreads / CH, PASSES = kPlain ? kTile / RP : 1;
  const bf16* base;
  const char* p;
  int64_t ns, step, r0, n;
  uint32_t dst;
  int row, d, vec;
  bool col;
  // rows r0, r0 + 64, ... of `base`, which has n
  __device__ __forceinline__ Stream(const bf16* base, int64_t ns, int vec, int64_t r0, int64_t n, int d)
      : base(base), ns(ns), r0(r0), n(n), d(d), vec(vec && kPlain) {
    row = threadIdx.x / CH;
    const int c = threadIdx.x - row * CH;
    p = (const char*)(base + (r0 + row) * ns + c * 8);
    step = RP * ns * 2;
    dst = Tile<DP>::off(row, c);
    col = c * 8 < d;
  }
  // rows without a bit in `live`, which has none past the end, are zero
  __device__ __forceinline__ void next(uint32_t sm, uint64_t live, int vec16) {
    if (vec) {
      const uint32_t half[2] = {(uint32_t)live, (uint32_t)(live >> 32)};
#pragma unroll
      for (int j = 0; j < PASSES; ++j) {
        const bool ok = col && ((half[j * RP / 32] >> (row + j * RP % 32)) & 1);
        // 128 channels: rows 8 apart differ in one bit of the swizzle
        const uint32_t at = DP == 128 ? (dst ^ ((j & 1) << 5)) : dst;
        cp_async16(sm + at + j * RP * Tile<DP>::RB, p + j * step, ok);
      }
      p += PASSES * step;
    } else {
      load_rows<DP, kTile>(sm, base, ns, vec16, r0, n, d, live);
    }
    r0 += kTile;
  }
};
__device__ __forceinline__ uint64_t first_bits(int64_t n) { return n >= 64 ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1); }

// ---------------------------------------------------------------- visible keys

// Mask values of keys j0 + lane and j0 + 32 + lane (0 past the end), read a tile ahead of their use.
__device__ __forceinline__ float2 seen_raw(const Args& a, int64_t b, int64_t j0) {
  const int64_t j = j0 + (threadIdx.x & 31);
  float2 r;
  if (a.mask) {
    const float* m = a.mask + b * a.m_bs;
    r.x = j < a.nk ? m[j * a.m_ks] : 0.f;
    r.y = j + 32 < a.nk ? m[(j + 32) * a.m_ks] : 0.f;
  } else {
    r.x = j < a.nk ? 1.f : 0.f;
    r.y = j + 32 < a.nk ? 1.f : 0.f;
  }
  return r;
}
__device__ __forceinline__ uint64_t seen_ballot(float2 r) {
  return (uint64_t)__ballot_sync(0xffffffffu, r.x != 0.f) |
         ((uint64_t)__ballot_sync(0xffffffffu, r.y != 0.f) << 32);
}

// ---------------------------------------------------------------- bias fragments
// BT: 0 no bias, 1 bf16, 2 fp32. Four neighbouring keys of one row.

template <int BT>
struct Bias4 {
  uint32_t w[BT == 2 ? 4 : (BT == 1 ? 2 : 1)];
};
template <int BT>
__device__ __forceinline__ const char* bias_row(const Args& a, int64_t b, int h, int64_t i) {
  if (BT == 0) return nullptr;
  return (const char*)a.bias + (b * a.b_bs + (int64_t)h * a.b_hs + i * a.b_rs) * (BT == 2 ? 4 : 2);
}
// keys j .. j + 3, the first of them at p; `fast`: all exist and are aligned together
template <int BT>
__device__ __forceinline__ void bias_get(Bias4<BT>& r, const char* p, int64_t j, int64_t nk, bool fast) {
  if (BT == 1) {
    if (fast) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      r.w[0] = v.x, r.w[1] = v.y;
    } else {
      const unsigned short* q = (const unsigned short*)p;
      const int left = (int)(nk - j < 4 ? nk - j : 4);
      uint32_t e[4];
      if (left == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = q[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = i < left ? q[i] : 0;
      }
      r.w[0] = e[0] | (e[1] << 16), r.w[1] = e[2] | (e[3] << 16);
    }
  } else if (BT == 2) {
    if (fast) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    } else {
      const uint32_t* q = (const uint32_t*)p;
      const int left = (int)(nk - j < 4 ? nk - j : 4);
      if (left == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = q[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) r.w[i] = i < left ? q[i] : 0;
      }
    }
  }
}
// the same of the row at p
template <int BT>
__device__ __forceinline__ void bias_load(Bias4<BT>& r, const char* p, int64_t j, int64_t nk, bool fast) {
  bias_get<BT>(r, p + j * (BT == 2 ? 4 : 2), j, nk, fast);
}
template <int BT>
__device__ __forceinline__ float bias_val(const Bias4<BT>& r, int i) {
  if (BT == 1) return (i & 1) ? hi_f(r.w[i >> 1]) : lo_f(r.w[i >> 1]);
  if (BT == 2) return __uint_as_float(r.w[i]);
  return 0.f;
}
// Scores of two neighbouring columns, scale * s + bias, s in natural units (next to a bias of the type's lowest
// value a factor log2(e) would overflow).
template <int BT>
__device__ __forceinline__ void score2(float* x, F2 scale, const Bias4<BT>& r, int n) {
  const F2 s = F2(x[0], x[1]);
  const F2 y = BT == 0 ? mul2(s, scale) : fma2(s, scale, F2(bias_val<BT>(r, 2 * n), bias_val<BT>(r, 2 * n + 1)));
  y.get(x[0], x[1]);
}
// p of two neighbouring columns from their scores: exp(t - m) / l with nm = -m, c = -log2 l
__device__ __forceinline__ F2 prob2(const float* x, F2 nm, F2 c) {
  const F2 y = fma2(add2(F2(x[0], x[1]), nm), F2(kLog2e), c);
  float p0, p1;
  y.get(p0, p1);
  return F2(ex2(p0), ex2(p1));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// one row's four columns of a group as the products leave them, x[0][2r..] then x[1][2r..]: keys j .. j + 3,
// the first of them at p
template <int BT>
__device__ __forceinline__ void put_bias4(char* p, int64_t j, int64_t nk, bool fast, float v0, float v1, float v2,
                                          float v3) {
  if (BT == 2) {
    float* q = (float*)p;
    if (fast) {
      *reinterpret_cast<float4*>(q) = make_float4(v0, v1, v2, v3);
    } else {
      if (j < nk) q[0] = v0;
      if (j + 1 < nk) q[1] = v1;
      if (j + 2 < nk) q[2] = v2;
      if (j + 3 < nk) q[3] = v3;
    }
  } else {
    bf16* q = (bf16*)p;
    if (fast) {
      *reinterpret_cast<uint2*>(q) = make_uint2(pack_bf16(v0, v1), pack_bf16(v2, v3));
    } else {
      if (j < nk) q[0] = __float2bfloat16_rn(v0);
      if (j + 1 < nk) q[1] = __float2bfloat16_rn(v1);
      if (j + 2 < nk) q[2] = __float2bfloat16_rn(v2);
      if (j + 3 < nk) q[3] = __float2bfloat16_rn(v3);
    }
  }
}
// the same of the row at p
template <int BT>
__device__ __forceinline__ void store_bias4(const Args& a, char* p, int64_t j, bool fast, float v0, float v1, float v2,
                                            float v3) {
  put_bias4<BT>(p + j * (BT == 2 ? 4 : 2), j, a.nk, fast, v0, v1, v2, v3);
}

// 8 consecutive accumulator columns of a row, two per lane
__device__ __forceinline__ void store_pair(bf16* p, int col, int d, bool vec, float v0, float v1) {
  if (vec) {
    if (col < d) *reinterpret_cast<uint32_t*>(p + col) = pack_bf16(v0, v1);
  } else {
    if (col < d) p[col] = __float2bfloat16_rn(v0);
    if (col + 1 < d) p[col + 1] = __float2bfloat16_rn(v1);
  }
}
__device__ __forceinline__ bool pair_ok(const void* p, int64_t bs, int64_t ns, int64_t hs, int d) {
  return ((uintptr_t)p & 3) == 0 && ((bs | ns | hs | d) & 1) == 0;
}

// ---------------------------------------------------------------- dk, dv of a cluster

// `blocks` blocks of kernel K with `cluster` of them to a cluster (1: none) and `smem` bytes of shared memory, of
// which other calls take `most` at most.
template <auto K, class... X>
int go(size_t smem, size_t most, int64_t blocks, int cluster, const char* name, double flops, cudaStream_t st, X... x) {
  if (blocks == 0) return PF_OK;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: %lld tiles are too many", (long long)blocks);
  PF_TRY(room_for_shared<K>(most));
  {
    PF_LAUNCH_SCOPE_WORK(st, name, flops, 'f');
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)blocks), cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cfg.attrs = &attr, cfg.numAttrs = cluster > 1 ? 1 : 0;
    PF_CUDA_TRY(cudaLaunchKernelEx(&cfg, K, x...));
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

// The blocks of a cluster that the query heads of a key head are shared out to: a power of two up to eight, where
// there is room for them next to dq's blocks (computed or not: the same bits either way), two blocks on each SM.
// 3 x 301 queries by 517 keys, 2 key heads of 4 query heads each, bf16, one term of p and ds, with dq: 44 us in one
// block, 37 us in two, 38 us in four.
inline int dkv_ranks(const Args& a, int64_t blocks, int64_t dq_blocks) {
  int ranks = 1;
  while (ranks < 8 && a.H / a.KV % (2 * ranks) == 0 && 2 * ranks * blocks + dq_blocks <= 2 * 148) ranks *= 2;
  return ranks;
}

// The sum over the cluster's blocks, in their order, of x and y (a warp's 16 keys each, as the products leave
// them): each block adds a share of the 64 keys from all blocks' shared memory and passes them to store(which,
// key, channel, v0, v1).
template <int DP, class Store>
__device__ __forceinline__ void sum_ranks(unsigned char* raw, const float (&x)[DP / 8][4], const float (&y)[DP / 8][4],
                                          int ranks, int rank, Store store) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  float* red = (float*)raw;  // [2][64][DP]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  __syncthreads();  // the tiles are done with
#pragma unroll
  for (int r = 0; r < 2; ++r)
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      float* p = red + (warp * 16 + perm_row(g, r)) * DP + n * 8 + 2 * t;
      *reinterpret_cast<float2*>(p) = make_float2(x[n][2 * r], x[n][2 * r + 1]);
      *reinterpret_cast<float2*>(p + 64 * DP) = make_float2(y[n][2 * r], y[n][2 * r + 1]);
    }
  cluster.sync();
  const int keys = 64 / ranks;
  for (int i = threadIdx.x; i < keys * DP; i += kThreads) {  // pairs of channels
    const int c = i % (DP / 2) * 2, k = i / (DP / 2), which = k / keys, row = rank * keys + k % keys;
    float2 s = make_float2(0.f, 0.f);
    for (int q = 0; q < ranks; ++q) {
      const float2 v = *cluster.map_shared_rank(reinterpret_cast<float2*>(red + (which * 64 + row) * DP + c), q);
      s.x += v.x, s.y += v.y;
    }
    store(which, row, c, s.x, s.y);
  }
  cluster.sync();  // no block leaves while others read its sums
}

// ---------------------------------------------------------------- tensor memory as thread-private storage

__device__ __forceinline__ void tmem_ld8(uint32_t addr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(addr));
}
// the wait takes the loaded registers along, so that no use of them moves above it
__device__ __forceinline__ void tmem_wait8(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

}  // namespace
}  // namespace attn
}  // namespace train
}  // namespace pf
