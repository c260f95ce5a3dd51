// pf_attention_f32.cu -- the fp32 kernels of pf_attention.cuh, on the bf16 tensor cores.
//
// An fp32 value is the sum of three bf16 values of 8 bits each (its rounding, the rounding of what is
// left, and the rest), so a product of two fp32 operands is the sum of six bf16 products whose order is
// 2^0, 2^-8, 2^-8, 2^-16, 2^-16, 2^-16; the three left out are below 2^-24 of the product. The tensor
// cores add in fp32 but cut off below the last bit of the running sum, which over a long sum would
// pile up: the small products are added apart from the large ones, and the second product (with p or
// ds) restarts from zero for every 16 columns and is added to the accumulators by rounded fp32
// additions. Against the FFMA form of the same kernels, which the multiply-adds bound at 128 per clock
// and SM (149 rows of 149 tokens, 12 heads of 32, forward plus backward: 1.9 ms), six products at 1024
// per clock and SM are 1.3 times as many, with a quarter of the instructions (0.76 ms; 0.55 ms of products).
// An infinity splits into an infinity and a NaN: at a visible place it gives NaN. The third value of an operand
// below 2^-110 falls under bf16's least step, 2^-133 (which the products keep): half of that is its error, and a
// gradient whose operands are all of 2^-116 is 1e-5 off.
//
// The layout is that of pf_attention_bf16.cu, with every tile in three planes. The streamed tiles are read
// into registers a tile ahead, split, and stored to the other buffer after the products of the current
// one. 16 stationary rows per warp, four warps to a block.

#include "pf_attention_tc.cuh"
#include "pf_sm100.cuh"

namespace pf {
namespace train {
namespace attn {
namespace {

// Rows of a streamed tile: four 16-byte loads per thread and operand.
template <int DP>
struct Split {
  static constexpr int KT = 2048 / DP;
  static constexpr int RB = Tile<DP>::RB;
  static constexpr int kPlane = KT * RB;   // bytes of a streamed plane
  static constexpr int kTile3 = 3 * kPlane;
  static constexpr int kStatPlane = 64 * RB, kStat3 = 3 * kStatPlane;
};

__device__ __forceinline__ void split4(const float4& v, uint2 (&w)[3]) {
  float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    w[p].x = pack_bf16(x[0], x[1]);
    w[p].y = pack_bf16(x[2], x[3]);
    if (p < 2) {
      fma2(F2(lo_f(w[p].x), hi_f(w[p].x)), F2(-1.f), F2(x[0], x[1])).get(x[0], x[1]);
      fma2(F2(lo_f(w[p].y), hi_f(w[p].y)), F2(-1.f), F2(x[2], x[3])).get(x[2], x[3]);
    }
  }
}

// A thread's place in the tiles of KT rows of one operand: four 16-byte loads, rows `row` + RP i.
template <int DP>
struct Place {
  static constexpr int CH = DP / 4, RP = kThreads / CH;
  int row, col;
  uint32_t dst;
  __device__ __forceinline__ Place() {
    row = threadIdx.x / CH;
    col = (threadIdx.x - row * CH) * 4;
    dst = Tile<DP>::off(row, col >> 3) + (col & 7) * 2;
  }
  // the offset of load i: rows RP apart have the same swizzle (32 channels) or differ in one bit of it
  __device__ __forceinline__ uint32_t at(int i) const {
    const uint32_t x = DP == 32 ? 0 : (DP == 64 ? (i & 1) * 2 : (i & 1) * 4 + (i >> 1) * 2);
    return (dst ^ (x << 4)) + i * RP * Tile<DP>::RB;
  }
};

// A tile on its way: read, then split and stored.
template <int DP>
struct Ahead {
  using P = Place<DP>;
  float4 v[4];
  // rows r0.. of `base`; those without a bit in `live`, which has none past the end, are zero
  __device__ __forceinline__ void read(const P& at, const float* base, int64_t ns, int vec, int64_t r0, int d,
                                       uint64_t live) {
    const float* p = base + (r0 + at.row) * ns + at.col;
    const uint64_t mine = at.col < d ? live >> at.row : 0;
    const uint32_t half[2] = {(uint32_t)mine, (uint32_t)(mine >> 32)};
    const int64_t step = ns * P::RP;
#pragma unroll
    for (int i = 0; i < 4; ++i, p += step) {
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if ((half[i * P::RP / 32] >> (i * P::RP % 32)) & 1) {
        if (vec) {
          v[i] = *reinterpret_cast<const float4*>(p);
        } else {
          v[i].x = p[0];
          if (at.col + 1 < d) v[i].y = p[1];
          if (at.col + 2 < d) v[i].z = p[2];
          if (at.col + 3 < d) v[i].w = p[3];
        }
      }
    }
  }
  template <int PLANE>
  __device__ __forceinline__ void store(const P& at, uint32_t sm) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint2 w[3];
      split4(v[i], w);
      const uint32_t to = sm + at.at(i);
      unrolled<3>([&](auto Q) {
        constexpr int p = decltype(Q)::value;
        asm volatile("st.shared.v2.b32 [%0+%3], {%1, %2};" ::"r"(to), "r"(w[p].x), "r"(w[p].y), "n"(p * PLANE)
                     : "memory");
      });
    }
  }
};
// 64 rows at once
template <int DP>
__device__ __forceinline__ void load_stat(const Place<DP>& at, uint32_t sm, const float* base, int64_t ns, int vec,
                                          int64_t r0, int d, uint64_t live) {
  using S = Split<DP>;
#pragma unroll 1
  for (int r = 0; r < 64; r += S::KT) {
    Ahead<DP> t;
    t.read(at, base, ns, vec, r0 + r, d, live >> r);
    t.template store<S::kStatPlane>(at, sm + r * S::RB);
  }
}
__device__ __forceinline__ const float* head_f(const Heads& s, int64_t b, int h) {
  return (const float*)s.p + b * s.bs + (int64_t)h * s.hs;
}

// x (16 rows by 16 columns) = a b^T over the channels: the lane's addresses of the operands' first planes for each
// 16 channels, PA and PB bytes between the planes
template <int KS, int PA, int PB>
__device__ __forceinline__ void nt3(float (&x)[2][4], const uint32_t (&aa)[KS], const uint32_t (&ba)[KS]) {
  float lo[2][4];
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    uint32_t a[3][4], b[3][4];
    unrolled<3>([&](auto P) {
      constexpr int p = decltype(P)::value;
      ldsm4i<p * PA>(a[p], aa[k]);
      ldsm4i<p * PB>(b[p], ba[k]);
    });
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (k == 0) {
        mma0(lo[n], a[2], b[0][2 * n], b[0][2 * n + 1]);
        mma0(x[n], a[0], b[0][2 * n], b[0][2 * n + 1]);
      } else {
        mma(lo[n], a[2], b[0][2 * n], b[0][2 * n + 1]);
        mma(x[n], a[0], b[0][2 * n], b[0][2 * n + 1]);
      }
      mma(lo[n], a[1], b[1][2 * n], b[1][2 * n + 1]);
      mma(lo[n], a[0], b[2][2 * n], b[2][2 * n + 1]);
      mma(lo[n], a[1], b[0][2 * n], b[0][2 * n + 1]);
      mma(lo[n], a[0], b[1][2 * n], b[1][2 * n + 1]);
    }
  }
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r)
      add2(F2(x[n][2 * r], x[n][2 * r + 1]), F2(lo[n][2 * r], lo[n][2 * r + 1])).get(x[n][2 * r], x[n][2 * r + 1]);
}
// acc += p b for 16 columns of p in three terms: the lane's addresses of b's first plane for each 16 channels
template <int NB, int PB>
__device__ __forceinline__ void nn3(float (&acc)[NB][4], const uint32_t (&pa)[3][4], const uint32_t (&ba)[NB / 2]) {
#pragma unroll
  for (int c = 0; c < NB / 2; ++c) {
    uint32_t b[3][4];
    unrolled<3>([&](auto P) {
      constexpr int p = decltype(P)::value;
      ldsm4_ti<p * PB>(b[p], ba[c]);
    });
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      float s[4];
      mma0(s, pa[2], b[0][2 * n], b[0][2 * n + 1]);
      mma(s, pa[1], b[1][2 * n], b[1][2 * n + 1]);
      mma(s, pa[0], b[2][2 * n], b[2][2 * n + 1]);
      mma(s, pa[1], b[0][2 * n], b[0][2 * n + 1]);
      mma(s, pa[0], b[1][2 * n], b[1][2 * n + 1]);
      mma(s, pa[0], b[0][2 * n], b[0][2 * n + 1]);
      float* d = acc[2 * c + n];
      add2(F2(d[0], d[1]), F2(s[0], s[1])).get(d[0], d[1]);
      add2(F2(d[2], d[3]), F2(s[2], s[3])).get(d[2], d[3]);
    }
  }
}
template <int DP>
__device__ __forceinline__ void addresses(uint32_t (&to)[DP / 16], const LaneAddr<DP>& l, uint32_t base, int blk) {
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) to[k] = l.at(base, blk, k);
}
// 16 x 16 values in accumulator layout as left operands in three terms (left as their remainder)
__device__ __forceinline__ void split_a(float (&x)[2][4], uint32_t (&pa)[3][4]) {
#pragma unroll
  for (int p = 0; p < 3; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* v = &x[i >> 1][2 * (i & 1)];
      pa[p][i] = pack_bf16(v[0], v[1]);
      if (p < 2) fma2(F2(lo_f(pa[p][i]), hi_f(pa[p][i])), F2(-1.f), F2(v[0], v[1])).get(v[0], v[1]);
    }
}

// `hidden` in place of the columns without a bit
__device__ __forceinline__ void hide16(float (&x)[2][4], uint32_t bits, float hidden = -INFINITY) {
  if (bits == 0xffffu) return;
  const int t = threadIdx.x & 3;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (!((bits >> (4 * t + 2 * n + e)) & 1)) x[n][e] = x[n][2 + e] = hidden;
}

__device__ __forceinline__ void store2f(float* p, int col, int d, bool vec, float v0, float v1) {
  if (vec) {
    if (col < d) *reinterpret_cast<float2*>(p + col) = make_float2(v0, v1);
  } else {
    if (col < d) p[col] = v0;
    if (col + 1 < d) p[col + 1] = v1;
  }
}
__device__ __forceinline__ bool pair_ok_f(const void* p, int64_t bs, int64_t ns, int64_t hs, int d) {
  return ((uintptr_t)p & 7) == 0 && ((bs | ns | hs | d) & 1) == 0;
}
template <int KT>
__device__ __forceinline__ uint64_t tile_bits(float2 raw) {
  return seen_ballot(raw) & (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
}

// ---------------------------------------------------------------- forward

template <int DP, int BT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? 3 : 1) k_fwd(Args a) {
  using S = Split<DP>;
  constexpr int KT = S::KT, KS = DP / 16, NB = DP / 8, HB = KT < 32 ? KT : 32, GQ = HB / 16;
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sq = smem_addr(raw), sk = sq + S::kStat3, sv = sk + 2 * S::kTile3;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>(), lt = lane_bt<DP>();
  unsigned id = blockIdx.x;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV);
  const int64_t b = id / a.H, w0 = (int64_t)tile * 64 + warp * 16;
  const int nt = (int)((a.nk + KT - 1) / KT);
  const float *bk = head_f(a.k, b, kh), *bv = head_f(a.v, b, kh);
  const char* brow[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    brow[r] = bias_row<BT>(a, b, h, i < a.nq ? i : a.nq - 1);
  }
  const F2 scale(a.scale);
  float acc[NB][4], mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
  uint64_t bits = tile_bits<KT>(seen_raw(a, b, 0));
  Ahead<DP> pk, pv;
  const Place<DP> place;
  load_stat<DP>(place, sq, head_f(a.q, b, h), a.q.ns, a.vec_q, (int64_t)tile * 64, a.d,
                first_bits(a.nq - (int64_t)tile * 64));
  pk.read(place, bk, a.k.ns, a.vec_k, 0, a.d, bits);
  pv.read(place, bv, a.v.ns, a.vec_v, 0, a.d, bits);
  pk.template store<S::kPlane>(place, sk);
  pv.template store<S::kPlane>(place, sv);
  uint32_t qa[KS];
  addresses<DP>(qa, la, sq, warp);
  for (int kt = 0; kt < nt; ++kt) {
    const uint64_t next = tile_bits<KT>(seen_raw(a, b, (int64_t)(kt + 1) * KT));
    __syncthreads();
    if (kt + 1 < nt) {
      pk.read(place, bk, a.k.ns, a.vec_k, (int64_t)(kt + 1) * KT, a.d, next);
      pv.read(place, bv, a.v.ns, a.vec_v, (int64_t)(kt + 1) * KT, a.d, next);
    }
    if (bits != 0 && w0 < a.nq) {
      const uint32_t tk = sk + (kt & 1) * S::kTile3, tv = sv + (kt & 1) * S::kTile3;
#pragma unroll 1
      for (int hb = 0; hb < KT / HB; ++hb) {
        const int64_t j0 = (int64_t)kt * KT + hb * HB;
        const uint32_t hbits = (uint32_t)(bits >> (HB * hb));
        if ((hbits & (HB == 32 ? ~0u : 0xffffu)) == 0) continue;  // no visible key
        float x[GQ][2][4];
#pragma unroll
        for (int q = 0; q < GQ; ++q) {
          Bias4<BT> br[2];
          const bool fast = a.bias_vec && j0 + q * 16 + 16 <= a.nk;
#pragma unroll
          for (int r = 0; r < 2; ++r) bias_load<BT>(br[r], brow[r], j0 + q * 16 + 4 * t, a.nk, fast);
          uint32_t ba[KS];
          addresses<DP>(ba, lb, tk, hb * GQ + q);
          nt3<KS, S::kStatPlane, S::kPlane>(x[q], qa, ba);
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) score2<BT>(&x[q][n][2 * r], scale, br[r], n);
          hide16(x[q], (hbits >> (16 * q)) & 0xffffu);
        }
        float nm[2];
        bool grew = false;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float v = mx[r];
#pragma unroll
          for (int q = 0; q < GQ; ++q)
#pragma unroll
            for (int n = 0; n < 2; ++n) v = max3(v, x[q][n][2 * r], x[q][n][2 * r + 1]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          nm[r] = v;
          grew |= v != mx[r];
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float corr = nm[r] == mx[r] ? 1.f : ex2((mx[r] - nm[r]) * kLog2e);
            mx[r] = nm[r];
            sum[r] *= corr;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              acc[n][2 * r] *= corr;
              acc[n][2 * r + 1] *= corr;
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const F2 neg(mx[r] == -INFINITY ? 0.f : -mx[r]);  // nothing seen yet: every p is 0
          F2 s(0.f);
#pragma unroll
          for (int q = 0; q < GQ; ++q)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const F2 p = prob2(&x[q][n][2 * r], neg, F2(0.f));
              p.get(x[q][n][2 * r], x[q][n][2 * r + 1]);
              s = add2(s, p);
            }
          sum[r] += s.sum();
        }
#pragma unroll
        for (int q = 0; q < GQ; ++q) {
          uint32_t pa[3][4];
          split_a(x[q], pa);
          uint32_t ba[KS];
          addresses<DP>(ba, lt, tv, hb * GQ + q);
          nn3<NB, S::kPlane>(acc, pa, ba);
        }
      }
    }
    if (kt + 1 < nt) {
      pk.template store<S::kPlane>(place, sk + ((kt + 1) & 1) * S::kTile3);
      pv.template store<S::kPlane>(place, sv + ((kt + 1) & 1) * S::kTile3);
    }
    bits = next;
  }
  const bool vec = pair_ok_f(a.o, a.o_bs, a.o_ns, a.o_hs, a.d);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float l = sum[r];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int64_t i = w0 + r * 8 + g;
    if (i >= a.nq) continue;
    if (a.stats && t == 0) {
      const int64_t at = (b * a.H + h) * a.nq + i;
      a.stats[at] = mx[r];
      a.stats[a.rows_plane + at] = l;
    }
    float* o = (float*)a.o + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
#pragma unroll
    for (int n = 0; n < NB; ++n) store2f(o, n * 8 + 2 * t, a.d, vec, acc[n][2 * r] * inv, acc[n][2 * r + 1] * inv);
  }
}

// ---------------------------------------------------------------- row constants

// D, and {m, -log2 l, peak, -D} of the rows (b, h, i), i fastest; peak = 1 where one key has all of the
// row's weight in fp32 (l = 1). L lanes per row, four channels each (VEC: as one access).
template <int L, bool VEC>
__global__ void __launch_bounds__(256) k_rows(Args a, const float* __restrict__ stats, Heads o,
                                              float4* __restrict__ rows) {
  const int sub = threadIdx.x & (L - 1);
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const bool live = at < a.rows_plane;
  const int64_t r = live ? at : 0, bh = r / a.nq, i = r - bh * a.nq, b = bh / a.H;
  const int h = (int)(bh - b * a.H), c = sub * 4;
  const float* po = head_f(o, b, h) + i * o.ns + c;
  const float* pg = head_f(a.g, b, h) + i * a.g.ns + c;
  float s = 0.f;
  if (VEC) {
    if (live && c < a.d) {
      const float4 x = *reinterpret_cast<const float4*>(po), y = *reinterpret_cast<const float4*>(pg);
      s = x.x * y.x + x.y * y.y + x.z * y.z + x.w * y.w;
    }
  } else if (live) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (c + e < a.d) s += po[e] * pg[e];
  }
#pragma unroll
  for (int k = 1; k < L; k <<= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (!live || sub) return;
  const float m = stats[at], l = stats[a.rows_plane + at];
  const bool none = l == 0.f;
  rows[at] = make_float4(none ? INFINITY : m, none ? 0.f : -log2f(l), l == 1.f ? 1.f : 0.f, none ? 0.f : -s);
}

// p from scores and ds in dp's place
__device__ __forceinline__ void prob_ds(float (&x)[2][4], float (&y)[2][4], const F2 (&nmx)[2], const F2 (&lg)[2],
                                        const F2 (&nd)[2], bool peaked) {
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const F2 p = prob2(&x[n][2 * r], nmx[r], lg[r]);
      p.get(x[n][2 * r], x[n][2 * r + 1]);
      mul2(p, add2(F2(y[n][2 * r], y[n][2 * r + 1]), nd[r])).get(y[n][2 * r], y[n][2 * r + 1]);
    }
  if (peaked) {
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (x[n][e] == 1.f) y[n][e] = 0.f;
  }
}

// ---------------------------------------------------------------- dq (and dbias)

// dq of rows [64 tile, 64 tile + 64) of (b, h). dbias of the entry is written where a.dbias is set; PLANE: added to
// the sums of the entries before, eight words of tensor memory per lane for each 16 keys, from tm0.
template <int DP, int BT, bool PLANE>
__device__ __forceinline__ void dq_rows(const Args& a, int64_t b, int h, unsigned tile, uint32_t tm0) {
  using S = Split<DP>;
  constexpr int KT = S::KT, KS = DP / 16, NB = DP / 8;
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sq = smem_addr(raw), sg = sq + S::kStat3, sk = sg + S::kStat3, sv = sk + 2 * S::kTile3;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>(), lt = lane_bt<DP>();
  const int kh = h / (a.H / a.KV);
  const int64_t w0 = (int64_t)tile * 64 + warp * 16;
  const bool put = BT && !PLANE && a.dbias;
  const int nt = (int)((a.nk + KT - 1) / KT);
  const float *bk = head_f(a.k, b, kh), *bv = head_f(a.v, b, kh);
  const char* brow[2];
  char* drow[2];
  F2 nmx[2], lg[2], nd[2];
  bool peaked = false;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g, ic = i < a.nq ? i : a.nq - 1;
    brow[r] = bias_row<BT>(a, b, h, ic);
    drow[r] = (put && i < a.nq)
                  ? (char*)a.dbias + (b * a.db_bs + (int64_t)h * a.db_hs + i * a.db_rs) * (BT == 2 ? 4 : 2)
                  : nullptr;
    const float4 c = ((const float4*)a.rows)[(b * a.H + h) * a.nq + ic];
    nmx[r] = F2(-c.x), lg[r] = F2(c.y), nd[r] = F2(c.w);
    peaked |= c.z != 0.f;
  }
  peaked = __any_sync(0xffffffffu, peaked);
  const F2 scale(a.scale);
  float acc[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
  uint64_t bits = tile_bits<KT>(seen_raw(a, b, 0));
  Ahead<DP> pk, pv;
  const Place<DP> place;
  const uint64_t rows = first_bits(a.nq - (int64_t)tile * 64);
  load_stat<DP>(place, sq, head_f(a.q, b, h), a.q.ns, a.vec_q, (int64_t)tile * 64, a.d, rows);
  load_stat<DP>(place, sg, head_f(a.g, b, h), a.g.ns, a.vec_g, (int64_t)tile * 64, a.d, rows);
  pk.read(place, bk, a.k.ns, a.vec_k, 0, a.d, bits);
  pv.read(place, bv, a.v.ns, a.vec_v, 0, a.d, bits);
  pk.template store<S::kPlane>(place, sk);
  pv.template store<S::kPlane>(place, sv);
  uint32_t qa[KS], ga[KS];
  addresses<DP>(qa, la, sq, warp);
  addresses<DP>(ga, la, sg, warp);
  for (int kt = 0; kt < nt; ++kt) {
    const uint64_t next = tile_bits<KT>(seen_raw(a, b, (int64_t)(kt + 1) * KT));
    __syncthreads();
    if (kt + 1 < nt) {
      pk.read(place, bk, a.k.ns, a.vec_k, (int64_t)(kt + 1) * KT, a.d, next);
      pv.read(place, bv, a.v.ns, a.vec_v, (int64_t)(kt + 1) * KT, a.d, next);
    }
    if (w0 < a.nq && (bits != 0 || put)) {
      const uint32_t tk = sk + (kt & 1) * S::kTile3, tv = sv + (kt & 1) * S::kTile3;
#pragma unroll 1
      for (int q = 0; q < KT / 16; ++q) {
        const int64_t j0 = (int64_t)kt * KT + q * 16;
        const uint32_t qbits = (uint32_t)(bits >> (16 * q)) & 0xffffu;
        if (qbits == 0 && (!put || j0 >= a.nk)) continue;  // no visible key, and nothing to write
        Bias4<BT> br[2];
        const bool whole = j0 + 16 <= a.nk;
#pragma unroll
        for (int r = 0; r < 2; ++r) bias_load<BT>(br[r], brow[r], j0 + 4 * t, a.nk, a.bias_vec && whole);
        float x[2][4], y[2][4];
        uint32_t ba[KS];
        addresses<DP>(ba, lb, tk, q);
        nt3<KS, S::kStatPlane, S::kPlane>(x, qa, ba);
        addresses<DP>(ba, lb, tv, q);
        nt3<KS, S::kStatPlane, S::kPlane>(y, ga, ba);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, br[r], n);
        hide16(x, qbits);
        prob_ds(x, y, nmx, lg, nd, peaked);
        hide16(y, qbits, 0.f);  // a hidden key's ds is 0, whatever do holds
        if (PLANE) {
          uint32_t tm[8];
          const uint32_t at = tm0 + (uint32_t)(kt * (KT / 16) + q) * 8;
          tmem_ld8(at, tm);
          tmem_wait8(tm);
#pragma unroll
          for (int i = 0; i < 8; i += 2) {
            float s0, s1;
            add2(F2(__uint_as_float(tm[i]), __uint_as_float(tm[i + 1])), F2(y[i >> 2][i & 3], y[i >> 2][(i & 3) + 1]))
                .get(s0, s1);
            tm[i] = __float_as_uint(s0), tm[i + 1] = __float_as_uint(s1);
          }
          tmem_st8(at, tm);
          if (!a.dq) continue;
        }
        if (put)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (drow[r])
              store_bias4<BT>(a, drow[r], j0 + 4 * t, a.db_vec && whole, y[0][2 * r], y[0][2 * r + 1], y[1][2 * r],
                              y[1][2 * r + 1]);
        uint32_t da[3][4];
        split_a(y, da);
        addresses<DP>(ba, lt, tk, q);
        nn3<NB, S::kPlane>(acc, da, ba);
      }
    }
    if (kt + 1 < nt) {
      pk.template store<S::kPlane>(place, sk + ((kt + 1) & 1) * S::kTile3);
      pv.template store<S::kPlane>(place, sv + ((kt + 1) & 1) * S::kTile3);
    }
    bits = next;
  }
  if (!a.dq) return;
  const bool vec = pair_ok_f(a.dq, a.o_bs, a.o_ns, a.o_hs, a.d);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    if (i >= a.nq) continue;
    float* o = (float*)a.dq + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
#pragma unroll
    for (int n = 0; n < NB; ++n)
      store2f(o, n * 8 + 2 * t, a.d, vec, acc[n][2 * r] * a.scale, acc[n][2 * r + 1] * a.scale);
  }
}

template <int DP, int BT>
__device__ __forceinline__ void dq_block(const Args& a, unsigned id, int64_t tiles) {
  const unsigned tile = id % (unsigned)tiles;
  id /= (unsigned)tiles;
  if (id / a.H < a.B)  // else it makes up a whole cluster
    dq_rows<DP, BT, false>(a, id / a.H, id % a.H, tile, 0);
}

// dq and the gradient of a bias that the batch shares in one pass (see k_dq_plane of the bf16 kernels): a block
// takes 64 rows of one head through a part of the batch, and its rows of the plane lie in tensor memory, 128
// columns for up to 256 keys (three blocks per SM) or 256 for up to 512 (two). Next to dq and dbias apart this
// saves two of five products: 149 rows of 149 tokens, 12 heads, 0.28 ms against 0.48 ms.
constexpr int kPlaneKeys = 512;

template <int BT>
__global__ void __launch_bounds__(kThreads, 3) k_dq_plane(Args a, float* part, int parts, int tcols, int tptr_at) {
  extern __shared__ __align__(128) unsigned char raw[];
  uint32_t* tptr = (uint32_t*)(raw + tptr_at);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned id = blockIdx.x;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, pt = id / a.H;
  const int64_t b0 = a.B * pt / parts, b1 = a.B * (pt + 1) / parts;
  const int64_t w0 = (int64_t)tile * 64 + warp * 16;
  const int groups = (int)((a.nk + 15) / 16);
  if (warp == 0) {
    sm100::tmem_alloc(smem_addr(tptr), tcols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tbase = *tptr, tm0 = tbase + ((uint32_t)(warp * 32) << 16);
  const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
  for (int q = 0; q < groups; ++q) tmem_st8(tm0 + q * 8, zero);
  sm100::tmem_st_wait();
  for (int64_t b = b0; b < b1; ++b) {
    if (b > b0) __syncthreads();  // the last entry's tiles are done with
    dq_rows<32, BT, true>(a, b, h, tile, tm0);
    sm100::tmem_st_wait();
  }
  for (int q = 0; q < groups; ++q) {
    uint32_t tm[8];
    __syncwarp();
    tmem_ld8(tm0 + q * 8, tm);
    tmem_wait8(tm);
    const int64_t j = (int64_t)q * 16 + 4 * t;
    const bool whole = (int64_t)q * 16 + 16 <= a.nk;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + r * 8 + g;
      if (i >= a.nq) continue;
      const float v0 = __uint_as_float(tm[2 * r]), v1 = __uint_as_float(tm[2 * r + 1]),
                  v2 = __uint_as_float(tm[4 + 2 * r]), v3 = __uint_as_float(tm[5 + 2 * r]);
      if (parts == 1)
        store_bias4<BT>(a, (char*)a.dbias + ((int64_t)h * a.db_hs + i * a.db_rs) * (BT == 2 ? 4 : 2), j,
                        a.db_vec && whole, v0, v1, v2, v3);
      else
        store_bias4<2>(a, (char*)(part + (((int64_t)pt * a.H + h) * a.nq + i) * a.nk), j, (a.nk & 3) == 0 && whole, v0,
                       v1, v2, v3);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  if (warp == 0) sm100::tmem_dealloc(tbase, tcols);
}

// ---------------------------------------------------------------- dk, dv

template <int DP, int BT>
__device__ __forceinline__ void dkv_block(const Args& a, unsigned id, int64_t tiles, int rank, int ranks) {
  using S = Split<DP>;
  constexpr int KT = S::KT, KS = DP / 16, NB = DP / 8;
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sk = smem_addr(raw), sv = sk + S::kStat3, sq = sv + S::kStat3, sg = sq + 2 * S::kTile3;
  float4* cst = (float4*)(raw + 2 * S::kStat3 + 4 * S::kTile3);  // [2][KT]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>(), ln = lane_bn<DP>();
  const unsigned tile = id % (unsigned)tiles;
  id /= (unsigned)tiles;
  const int kh = id % a.KV, group = a.H / a.KV, heads = group / ranks, h0 = kh * group + rank * heads;
  const int64_t b = id / a.KV, j0 = (int64_t)tile * 64, w0 = j0 + warp * 16;
  const int per = (int)((a.nq + KT - 1) / KT), nt = per * heads;
  const uint64_t live = seen_ballot(seen_raw(a, b, j0));
  const uint32_t mine = (uint32_t)(live >> (warp * 16)) & 0xffffu;
  const bool bfast = a.bias_vec && w0 + 16 <= a.nk;
  const F2 scale(a.scale);
  float dk[NB][4], dv[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;
  if (live != 0 && nt > 0) {
    Ahead<DP> pq, pg;
    const Place<DP> place;
    float4 pc = make_float4(0.f, 0.f, 0.f, 0.f);
    auto read = [&](int it) {
      const int h = h0 + it / per;
      const int64_t i0 = (int64_t)(it % per) * KT;
      const uint64_t rows = first_bits(a.nq - i0) & (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
      pq.read(place, head_f(a.q, b, h), a.q.ns, a.vec_q, i0, a.d, rows);
      pg.read(place, head_f(a.g, b, h), a.g.ns, a.vec_g, i0, a.d, rows);
      // a row past the end has p = 0
      if (threadIdx.x < KT)
        pc = i0 + threadIdx.x < a.nq ? ((const float4*)a.rows)[(b * a.H + h) * a.nq + i0 + threadIdx.x]
                                     : make_float4(INFINITY, 0.f, 0.f, 0.f);
    };
    auto store = [&](int it) {
      pq.template store<S::kPlane>(place, sq + (it & 1) * S::kTile3);
      pg.template store<S::kPlane>(place, sg + (it & 1) * S::kTile3);
      if (threadIdx.x < KT) cst[(it & 1) * KT + threadIdx.x] = pc;
    };
    load_stat<DP>(place, sk, head_f(a.k, b, kh), a.k.ns, a.vec_k, j0, a.d, live);
    load_stat<DP>(place, sv, head_f(a.v, b, kh), a.v.ns, a.vec_v, j0, a.d, live);
    uint32_t ka[KS], va[KS];
    addresses<DP>(ka, lb, sk, warp);
    addresses<DP>(va, lb, sv, warp);
    read(0);
    store(0);
    for (int it = 0; it < nt; ++it) {
      __syncthreads();
      if (it + 1 < nt) read(it + 1);
      if (mine != 0) {
        const int h = h0 + it / per;
        const int64_t i0 = (int64_t)(it % per) * KT;
        const uint32_t tq = sq + (it & 1) * S::kTile3, tg = sg + (it & 1) * S::kTile3;
#pragma unroll 1
        for (int blk = 0; blk < KT / 16; ++blk) {
          if (i0 + blk * 16 >= a.nq) break;
          Bias4<BT> br[2];
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int64_t i = i0 + blk * 16 + r * 8 + g;
            bias_load<BT>(br[r], bias_row<BT>(a, b, h, i < a.nq ? i : a.nq - 1), w0 + 4 * t, a.nk, bfast);
          }
          float x[2][4], y[2][4];
          uint32_t aa[KS];
          addresses<DP>(aa, la, tq, blk);
          nt3<KS, S::kPlane, S::kStatPlane>(x, aa, ka);
          addresses<DP>(aa, la, tg, blk);
          nt3<KS, S::kPlane, S::kStatPlane>(y, aa, va);
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, br[r], n);
          hide16(x, mine);
          const float4 c[2] = {cst[(it & 1) * KT + blk * 16 + g], cst[(it & 1) * KT + blk * 16 + 8 + g]};
          const F2 nmx[2] = {F2(-c[0].x), F2(-c[1].x)}, lg[2] = {F2(c[0].y), F2(c[1].y)},
                   nd[2] = {F2(c[0].w), F2(c[1].w)};
          prob_ds(x, y, nmx, lg, nd, __any_sync(0xffffffffu, c[0].z != 0.f || c[1].z != 0.f));
          uint32_t u[3][4], w[3][4];
          split_a(x, u);
#pragma unroll
          for (int p = 0; p < 3; ++p) {  // 8 x 8 blocks transposed, the two off the diagonal changing places
            w[p][0] = transpose8(u[p][0]), w[p][2] = transpose8(u[p][1]);
            w[p][1] = transpose8(u[p][2]), w[p][3] = transpose8(u[p][3]);
          }
          addresses<DP>(aa, ln, tg, blk);
          nn3<NB, S::kPlane>(dv, w, aa);
          split_a(y, u);
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            w[p][0] = transpose8(u[p][0]), w[p][2] = transpose8(u[p][1]);
            w[p][1] = transpose8(u[p][2]), w[p][3] = transpose8(u[p][3]);
          }
          addresses<DP>(aa, ln, tq, blk);
          nn3<NB, S::kPlane>(dk, w, aa);
        }
      }
      if (it + 1 < nt) store(it + 1);
    }
  }
  const bool vk = pair_ok_f(a.dk, a.dk_bs, a.dk_ns, a.dk_hs, a.d), vv = pair_ok_f(a.dv, a.dv_bs, a.dv_ns, a.dv_hs, a.d);
  if (ranks > 1) {
    float* pk = (float*)a.dk + b * a.dk_bs + (int64_t)kh * a.dk_hs + j0 * a.dk_ns;
    float* pv = (float*)a.dv + b * a.dv_bs + (int64_t)kh * a.dv_hs + j0 * a.dv_ns;
    sum_ranks<DP>(raw, dk, dv, ranks, rank, [&](int which, int row, int c, float v0, float v1) {
      if (j0 + row >= a.nk) return;
      if (which == 0)
        store2f(pk + row * a.dk_ns, c, a.d, vk, v0 * a.scale, v1 * a.scale);
      else
        store2f(pv + row * a.dv_ns, c, a.d, vv, v0, v1);
    });
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t j = w0 + perm_row(g, r);  // row g + 8 r of the block holds this key
    if (j >= a.nk) continue;
    float* ok = (float*)a.dk + b * a.dk_bs + (int64_t)kh * a.dk_hs + j * a.dk_ns;
    float* ov = (float*)a.dv + b * a.dv_bs + (int64_t)kh * a.dv_hs + j * a.dv_ns;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      store2f(ok, n * 8 + 2 * t, a.d, vk, dk[n][2 * r] * a.scale, dk[n][2 * r + 1] * a.scale);
      store2f(ov, n * 8 + 2 * t, a.d, vv, dv[n][2 * r], dv[n][2 * r + 1]);
    }
  }
}

// dk and dv in the first blocks, dq in the others (either may be none): where neither fills the machine they
// run side by side.
template <int DP, int BT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? 3 : 1) k_dqkv(Args a, unsigned dkv_blocks, int ranks) {
  if (blockIdx.x < dkv_blocks)
    dkv_block<DP, BT>(a, blockIdx.x / ranks, (a.nk + 63) / 64, blockIdx.x % ranks, ranks);
  else
    dq_block<DP, BT>(a, blockIdx.x - dkv_blocks, (a.nq + 63) / 64);
}

// ---------------------------------------------------------------- dbias shared by the batch

// A 64 x KT tile of one head's plane, summed over the batch entries of a part (see k_dbias of the bf16
// kernels). One buffer: other blocks of the SM work while this one reads its next entry.
template <int DP, int BT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? 4 : 1) k_dbias(Args a, float* part, int parts) {
  using S = Split<DP>;
  constexpr int KT = S::KT, KS = DP / 16, GQ = KT / 16;
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sq = smem_addr(raw), sg = sq + S::kStat3, sk = sg + S::kStat3, sv = sk + S::kTile3;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>();
  unsigned id = blockIdx.x;
  const unsigned nkt = (unsigned)((a.nk + KT - 1) / KT);
  const unsigned kt = id % nkt;
  id /= nkt;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV), pt = id / a.H;
  const int64_t b0 = a.B * pt / parts, b1 = a.B * (pt + 1) / parts;
  const int64_t i0 = (int64_t)tile * 64, w0 = i0 + warp * 16, j0 = (int64_t)kt * KT;
  const char* brow[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    brow[r] = bias_row<BT>(a, 0, h, i < a.nq ? i : a.nq - 1);
  }
  const F2 scale(a.scale);
  const Place<DP> place;
  uint32_t qa[KS], ga[KS];
  addresses<DP>(qa, la, sq, warp);
  addresses<DP>(ga, la, sg, warp);
  float acc[GQ][2][4];
#pragma unroll
  for (int q = 0; q < GQ; ++q)
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[q][n][e] = 0.f;
  for (int64_t b = b0; b < b1; ++b) {
    const uint64_t bits = tile_bits<KT>(seen_raw(a, b, j0));
    if (bits == 0) continue;  // the same for the whole block
    __syncthreads();
    load_stat<DP>(place, sq, head_f(a.q, b, h), a.q.ns, a.vec_q, i0, a.d, first_bits(a.nq - i0));
    load_stat<DP>(place, sg, head_f(a.g, b, h), a.g.ns, a.vec_g, i0, a.d, first_bits(a.nq - i0));
    Ahead<DP> pk, pv;
    pk.read(place, head_f(a.k, b, kh), a.k.ns, a.vec_k, j0, a.d, bits);
    pv.read(place, head_f(a.v, b, kh), a.v.ns, a.vec_v, j0, a.d, bits);
    pk.template store<S::kPlane>(place, sk);
    pv.template store<S::kPlane>(place, sv);
    F2 nmx[2], lg[2], nd[2];
    bool peaked = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + r * 8 + g;
      const float4 c = ((const float4*)a.rows)[(b * a.H + h) * a.nq + (i < a.nq ? i : a.nq - 1)];
      nmx[r] = F2(-c.x), lg[r] = F2(c.y), nd[r] = F2(c.w);
      peaked |= c.z != 0.f;
    }
    peaked = __any_sync(0xffffffffu, peaked);
    __syncthreads();
    if (w0 >= a.nq) continue;
#pragma unroll
    for (int q = 0; q < GQ; ++q) {
      if (((uint32_t)(bits >> (16 * q)) & 0xffffu) == 0) continue;  // no visible key
      Bias4<BT> br[2];
      const bool fast = a.bias_vec && j0 + q * 16 + 16 <= a.nk;
#pragma unroll
      for (int r = 0; r < 2; ++r) bias_load<BT>(br[r], brow[r], j0 + q * 16 + 4 * t, a.nk, fast);
      float x[2][4], y[2][4];
      uint32_t ba[KS];
      addresses<DP>(ba, lb, sk, q);
      nt3<KS, S::kStatPlane, S::kPlane>(x, qa, ba);
      addresses<DP>(ba, lb, sv, q);
      nt3<KS, S::kStatPlane, S::kPlane>(y, ga, ba);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, br[r], n);
      hide16(x, (uint32_t)(bits >> (16 * q)) & 0xffffu);
      prob_ds(x, y, nmx, lg, nd, peaked);
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float* d = &acc[q][n][2 * r];
          add2(F2(d[0], d[1]), F2(y[n][2 * r], y[n][2 * r + 1])).get(d[0], d[1]);
        }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    if (i >= a.nq) continue;
#pragma unroll
    for (int q = 0; q < GQ; ++q) {
      const int64_t j = j0 + q * 16 + 4 * t;
      const bool whole = j0 + q * 16 + 16 <= a.nk;
      const float v0 = acc[q][0][2 * r], v1 = acc[q][0][2 * r + 1], v2 = acc[q][1][2 * r], v3 = acc[q][1][2 * r + 1];
      if (parts == 1)
        store_bias4<BT>(a, (char*)a.dbias + ((int64_t)h * a.db_hs + i * a.db_rs) * (BT == 2 ? 4 : 2), j,
                        a.db_vec && whole, v0, v1, v2, v3);
      else
        store_bias4<2>(a, (char*)(part + (((int64_t)pt * a.H + h) * a.nq + i) * a.nk), j, (a.nk & 3) == 0 && whole, v0,
                       v1, v2, v3);
    }
  }
}

// ---------------------------------------------------------------- launches

template <int DP, int BT>
int launch_t(Kind kind, Args a, double flops, cudaStream_t st) {
  using S = Split<DP>;
  const int64_t tq = (a.nq + 63) / 64, tk = (a.nk + 63) / 64;
  if (kind == kFwd) {
    a.tiles = tq;
    constexpr size_t smem = S::kStat3 + 4 * S::kTile3;
    return go<k_fwd<DP, BT>>(smem, smem, tq * a.H * a.B, 1, "k_attn_fwd", flops, st, a);
  }
  const int64_t bq = kind == kDkv ? 0 : tq * a.H * a.B, bkv = kind == kDq ? 0 : tk * a.KV * a.B;
  const int ranks = bkv == 0 ? 1 : dkv_ranks(a, bkv, tq * a.H * a.B);
  const int64_t bk = bkv * ranks, blocks = (bk + bq + ranks - 1) / ranks * ranks;
  constexpr size_t smem = 2 * S::kStat3 + 4 * S::kTile3 + 2 * S::KT * 16;
  return go<k_dqkv<DP, BT>>(smem, smem, blocks, ranks,
                            kind == kDq ? "k_attn_dq" : (kind == kDkv ? "k_attn_dkv" : "k_attn_dqkv"), flops, st, a,
                            (unsigned)bk, ranks);
}
template <int DP, int BT>
int launch_db(Args a, float* part, int parts, double flops, cudaStream_t st) {
  using S = Split<DP>;
  a.tiles = (a.nq + 63) / 64;
  constexpr size_t smem = 2 * S::kStat3 + 2 * S::kTile3;
  return go<k_dbias<DP, BT>>(smem, smem, a.tiles * ((a.nk + S::KT - 1) / S::KT) * a.H * parts, 1, "k_attn_dbias", flops,
                             st, a, part, parts);
}

template <int BT>
int launch_plane(Args a, float* part, int parts, double flops, cudaStream_t st) {
  using S = Split<32>;
  const int tcols = a.nk <= 256 ? 128 : 256;
  constexpr int tiles = 2 * S::kStat3 + 4 * S::kTile3;
  // room for as many blocks as tensor memory holds
  constexpr size_t most = 100 * 1024;
  const size_t smem = tcols == 128 ? tiles + 16 : most;
  a.tiles = (a.nq + 63) / 64;
  return go<k_dq_plane<BT>>(smem, most, a.tiles * a.H * parts, 1, "k_attn_dq_plane", flops, st, a, part, parts, tcols,
                            tiles);
}

}  // namespace

#define PF_ATT_DIM(FN, BT, ...)                    \
  do {                                             \
    if (a.d <= 32) return FN<32, BT>(__VA_ARGS__); \
    if (a.d <= 64) return FN<64, BT>(__VA_ARGS__); \
    return FN<128, BT>(__VA_ARGS__);               \
  } while (0)

int launch_f32(Kind kind, const Args& a, double flops, cudaStream_t st) {
  if (!a.bias) PF_ATT_DIM(launch_t, 0, kind, a, flops, st);
  if (a.bias_f32) PF_ATT_DIM(launch_t, 2, kind, a, flops, st);
  PF_ATT_DIM(launch_t, 1, kind, a, flops, st);
}
int dbias_f32(const Args& a, float* part, int parts, double flops, cudaStream_t st) {
  if (a.bias_f32) PF_ATT_DIM(launch_db, 2, a, part, parts, flops, st);
  PF_ATT_DIM(launch_db, 1, a, part, parts, flops, st);
}
bool dq_plane_f32_fits(int64_t nk, int d) { return d <= 32 && nk <= kPlaneKeys; }
int dq_plane_f32(const Args& a, float* part, int parts, double flops, cudaStream_t st) {
  return a.bias_f32 ? launch_plane<2>(a, part, parts, flops, st) : launch_plane<1>(a, part, parts, flops, st);
}
int rows_f32(const Args& a, const float* stats, Heads o, float* rows, cudaStream_t st) {
  const int lanes = a.d <= 32 ? 8 : (a.d <= 64 ? 16 : 32);
  const int64_t blocks = (a.rows_plane * lanes + 255) / 256;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: too many rows");
  const bool vec = a.vec_g && (uintptr_t)o.p % 16 == 0 && ((o.bs | o.ns | o.hs) & 3) == 0;
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_rows", (8.0 * a.d + 24.0) * (double)a.rows_plane, 'b');
    auto* kern = lanes == 8    ? (vec ? k_rows<8, true> : k_rows<8, false>)
                 : lanes == 16 ? (vec ? k_rows<16, true> : k_rows<16, false>)
                               : (vec ? k_rows<32, true> : k_rows<32, false>);
    kern<<<(unsigned)blocks, 256, 0, st>>>(a, stats, o, (float4*)rows);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

}  // namespace attn
}  // namespace train
}  // namespace pf
