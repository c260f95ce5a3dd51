// pf_attention_bf16.cu -- the bf16 kernels of pf_attention.cuh on warp-level tensor-core products.
//
// Work of one warp: 16 or 32 query rows against groups of 16 keys (forward, dq, dbias), or 16 keys
// against groups of 16 queries (dk, dv); four warps to a block, streamed tiles of 64 rows
// double-buffered by cp.async. For the heads of 24 and 32 channels of this package a 16 x 16 block of
// scores costs two to four products of depth 32 next to 256 exponentials, so the kernels are bound by
// the issue of products, exponentials and the arithmetic around them, not by memory: 768 rows of 768
// tokens, four heads, forward 1.5 ms, dk and dv 2.4 ms, dq with dbias 2.5 ms (0.6, 1.2 and 0.8 ms of products).
//
// Columns of a group of 16 keys are permuted so that a lane's four columns are four neighbouring keys
// (lane t of a quad: keys 4t..4t+3 in place of 2t, 2t+1, 2t+8, 2t+9): a bias row is then read, and a
// dbias row written, 8 (bf16) or 16 (fp32) bytes at a time in full 32-byte sectors. The permutation is
// in the row addresses of ldmatrix alone. Shared rows are whole (no padding) with their 16-byte chunks
// XOR-swizzled so that natural and permuted row sets are both free of bank conflicts.
//
// dk and dv need the transposed p and ds as left operands; the scores are computed with queries down
// the rows all the same (the bias is read along its rows) and each 8 x 8 block is transposed in
// registers by movmatrix.

#include "pf_attention_tc.cuh"
#include "pf_sm100.cuh"

namespace pf {
namespace train {
namespace attn {
namespace {

// ---------------------------------------------------------------- forward

// Tiles that are wholly visible and inside, with aligned bias rows, take the body without any checks
// (FAST): the checks would be half of its instructions.
template <int DP, int BT, int MT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? (MT == 1 ? 4 : 3) : 2) k_fwd(Args a) {
  using S = Tile<DP>;
  constexpr int QR = 64 * MT, KS = DP / 16, NB = DP / 8, RB = S::RB, BS = BT == 2 ? 4 : 2;
  constexpr int TERMS = BT == 2 ? 3 : 2;  // bf16 values that p is split into (see the head of pf_attention.cuh)
  constexpr int kV = 2 * kTile * RB;      // from a K tile to its V tile
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sq = smem_addr(raw), sk = sq + QR * RB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  unsigned id = blockIdx.x;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV);
  const int64_t b = id / a.H, nk = a.nk;
  const int64_t i0 = (int64_t)tile * QR, w0 = i0 + warp * 16 * MT;
  const int nt = (int)((nk + kTile - 1) / kTile);
  const int bvec = a.bias_vec;
  const bool work = w0 < a.nq;  // else a warp past the end
  load_rows<DP, QR>(sq, head_base(a.q, b, h), a.q.ns, a.vec_q, i0, a.nq, a.d, ~0ull);
  Stream<DP> ks(head_base(a.k, b, kh), a.k.ns, a.vec_k, 0, nk, a.d), vs(head_base(a.v, b, kh), a.v.ns, a.vec_v, 0, nk, a.d);
  auto issue = [&](int kt, uint64_t live) {
    const uint32_t s = sk + (kt & 1) * kTile * RB;
    ks.next(s, live, a.vec_k);
    vs.next(s + kV, live, a.vec_v);
    cp_commit();
  };
  uint32_t ka[KS], va[KS];
  {
    const LaneAddr<DP> lb = lane_b<DP>(), lt = lane_bt<DP>();
#pragma unroll
    for (int k = 0; k < KS; ++k) ka[k] = lb.at(sk, 0, k), va[k] = lt.at(sk + kV, 0, k);
  }
  const char* bp[MT][2];  // the lane's first key of the tile, in its rows
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + m * 16 + r * 8 + g;
      bp[m][r] = BT ? bias_row<BT>(a, b, h, i < a.nq ? i : a.nq - 1) + 4 * t * BS : nullptr;  // such rows are not stored
    }
  Bias4<BT> ring[2][MT][2];
  // group q of the tile at key j0 (4 and on: of the next one)
  auto fetch = [&](int slot, int q, int64_t j0, bool fast) {
    if (BT == 0) return;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) bias_get<BT>(ring[slot][m][r], bp[m][r] + q * 16 * BS, j0 + q * 16 + 4 * t, nk, fast);
  };
  const F2 scale(a.scale);
  float acc[MT][NB][4], mx[MT][2], sum[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
    mx[m][0] = mx[m][1] = -INFINITY;
    sum[m][0] = sum[m][1] = 0.f;
  }
  uint32_t fq[MT][KS][4];
  uint64_t bits = seen_ballot(seen_raw(a, b, 0));
  if (nt > 0) issue(0, bits);
  float2 rawm = seen_raw(a, b, kTile);
  auto body = [&](auto mode, int64_t j0, uint32_t off, bool nf) {
    constexpr bool FAST = decltype(mode)::value;
    uint32_t kc[KS], vc[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) kc[k] = ka[k] + off, vc[k] = va[k] + off;
#pragma unroll 1
    for (int hb = 0; hb < 2; ++hb) {  // 32 keys
      float x[MT][4][4];
      unrolled<2>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r[4];
          ldsm4i<q * 16 * RB>(r, kc[k]);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            if (k == 0) {
              mma0(x[m][2 * q], fq[m][k], r[0], r[1]);
              mma0(x[m][2 * q + 1], fq[m][k], r[2], r[3]);
            } else {
              mma(x[m][2 * q], fq[m][k], r[0], r[1]);
              mma(x[m][2 * q + 1], fq[m][k], r[2], r[3]);
            }
          }
        }
      });
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 2; ++r) score2<BT>(&x[m][2 * q + n][2 * r], scale, ring[q][m][r], n);
        fetch(q, 2 * hb + q + 2, j0, hb == 0 ? FAST || (bvec && j0 + (q + 3) * 16 <= nk) : nf);
      }
      if (!FAST) {
        const uint32_t hbits = (uint32_t)(bits >> (32 * hb));
        if (hbits != 0xffffffffu) {
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const uint32_t mine = hbits >> (16 * q + 4 * t);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (!((mine >> (2 * n + e)) & 1))
#pragma unroll
                  for (int m = 0; m < MT; ++m) x[m][2 * q + n][e] = x[m][2 * q + n][2 + e] = -INFINITY;
          }
        }
      }
      bool grew = false;
      float nm[MT][2];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float v = mx[m][r];
#pragma unroll
          for (int n = 0; n < 4; ++n) v = max3(v, x[m][n][2 * r], x[m][n][2 * r + 1]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          nm[m][r] = v;
          grew |= v != mx[m][r];
        }
      if (__any_sync(0xffffffffu, grew)) {  // rare after the first tiles
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float corr = nm[m][r] == mx[m][r] ? 1.f : ex2((mx[m][r] - nm[m][r]) * kLog2e);
            mx[m][r] = nm[m][r];
            sum[m][r] *= corr;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
              acc[m][n][2 * r] *= corr;
              acc[m][n][2 * r + 1] *= corr;
            }
          }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const F2 neg(mx[m][r] == -INFINITY ? 0.f : -mx[m][r]);  // nothing seen yet: every p is 0
          F2 s2;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const F2 p = prob2(&x[m][n][2 * r], neg, F2(0.f));
            p.get(x[m][n][2 * r], x[m][n][2 * r + 1]);
            s2 = n == 0 ? p : add2(s2, p);
          }
          sum[m][r] += s2.sum();
        }
      unrolled<2>([&](auto Q) {
        constexpr int q = decltype(Q)::value;
        uint32_t f[KS][4];
#pragma unroll
        for (int c = 0; c < KS; ++c) ldsm4_ti<q * 16 * RB>(f[c], vc[c]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t pa[TERMS][4];
#pragma unroll
          for (int term = 0; term < TERMS; ++term)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float* v = &x[m][2 * q + (i >> 1)][2 * (i & 1)];
              pa[term][i] = pack_bf16(v[0], v[1]);
              if (term + 1 < TERMS) fma2(F2(lo_f(pa[term][i]), hi_f(pa[term][i])), F2(-1.f), F2(v[0], v[1])).get(v[0], v[1]);
            }
#pragma unroll
          for (int c = 0; c < KS; ++c)
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              float* d = acc[m][2 * c + n];
              if (BT == 2) {
                // the products cut off below the last bit of their sum: start from zero, small terms first,
                // and add the group by rounded additions
                float part[4];
                mma0(part, pa[TERMS - 1], f[c][2 * n], f[c][2 * n + 1]);
#pragma unroll
                for (int term = TERMS - 2; term >= 0; --term) mma(part, pa[term], f[c][2 * n], f[c][2 * n + 1]);
                add2(F2(d[0], d[1]), F2(part[0], part[1])).get(d[0], d[1]);
                add2(F2(d[2], d[3]), F2(part[2], part[3])).get(d[2], d[3]);
              } else {
#pragma unroll
                for (int term = 0; term < TERMS; ++term) mma(d, pa[term], f[c][2 * n], f[c][2 * n + 1]);
              }
            }
        }
      });
#pragma unroll
      for (int k = 0; k < KS; ++k) kc[k] += 32 * RB, vc[k] += 32 * RB;
    }
  };
  if (work) {
    fetch(0, 0, 0, bvec && 16 <= nk);
    fetch(1, 1, 0, bvec && 32 <= nk);
  }
  for (int kt = 0; kt < nt; ++kt) {
    const uint64_t next = seen_ballot(rawm);
    const int64_t j0 = (int64_t)kt * kTile;
    cp_wait<0>();
    __syncthreads();
    if (kt == 0) {
      const LaneAddr<DP> la = lane_a<DP>();
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < KS; ++k) ldsm4(fq[m][k], la.at(sq, warp * MT + m, k));
    }
    if (kt + 1 < nt) issue(kt + 1, next);
    rawm = seen_raw(a, b, j0 + 2 * kTile);
    if (work) {
      const bool nf = bvec && j0 + kTile + 32 <= nk;  // the next tile's first two groups
      const uint32_t off = (kt & 1) * kTile * RB;
      if (bits == ~0ull && (BT == 0 || bvec)) {
        body(std::true_type{}, j0, off, nf);
      } else if (bits != 0) {
        body(std::false_type{}, j0, off, nf);
      } else {  // no visible key
        fetch(0, 4, j0, nf);
        fetch(1, 5, j0, nf);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) bp[m][0] += kTile * BS, bp[m][1] += kTile * BS;
    }
    bits = next;
  }
  cp_commit();
  cp_wait<0>();
  const bool vec = pair_ok(a.o, a.o_bs, a.o_ns, a.o_hs, a.d);
  const bool lo_vec = (a.d & 1) == 0;
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float l = sum[m][r];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int64_t i = w0 + m * 16 + r * 8 + g;
      if (i >= a.nq) continue;
      if (a.stats && t == 0) {
        const int64_t at = (b * a.H + h) * a.nq + i;
        a.stats[at] = mx[m][r];
        a.stats[a.rows_plane + at] = l;
      }
      bf16* o = (bf16*)a.o + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
      int16_t* lo = a.o_lo ? a.o_lo + ((b * a.nq + i) * a.H + h) * a.d : nullptr;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int col = n * 8 + 2 * t;
        const float v0 = acc[m][n][2 * r] * inv, v1 = acc[m][n][2 * r + 1] * inv;
        store_pair(o, col, a.d, vec, v0, v1);
        if (lo) {
          // fp32 bits of o less those of its bf16 rounding: o is their sum again (a tie that rounds down
          // would need one more than 16 bits hold and loses the last bit; NaN keeps none)
          const uint32_t w = pack_bf16(v0, v1);
          const int d0 = min((int)(__float_as_uint(v0) - (w << 16)), 32767);
          const int d1 = min((int)(__float_as_uint(v1) - (w & 0xffff0000u)), 32767);
          const int16_t l0 = v0 == v0 ? (int16_t)d0 : (int16_t)0, l1 = v1 == v1 ? (int16_t)d1 : (int16_t)0;
          if (lo_vec) {
            if (col < a.d) *reinterpret_cast<short2*>(lo + col) = make_short2(l0, l1);
          } else {
            if (col < a.d) lo[col] = l0;
            if (col + 1 < a.d) lo[col + 1] = l1;
          }
        }
      }
    }
}

// ---------------------------------------------------------------- row constants

// D, and {m, -log2 l, peak, -D} of the rows (b, h, i), i fastest; peak = 1 where one key has all of the
// row's weight in fp32 (l = 1). L lanes per row, eight channels each (VEC: as one access of o, its low
// halves and do).
template <int L, bool VEC>
__global__ void __launch_bounds__(256) k_rows(Args a, const float* __restrict__ stats, Heads o,
                                              const int16_t* __restrict__ lo, float4* __restrict__ rows) {
  const int sub = threadIdx.x & (L - 1);
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) / L;
  const bool live = at < a.rows_plane;
  const int64_t r = live ? at : 0, bh = r / a.nq, i = r - bh * a.nq, b = bh / a.H;
  const int h = (int)(bh - b * a.H), c = sub * 8;
  const bf16* po = head_base(o, b, h) + i * o.ns + c;
  const bf16* pg = head_base(a.g, b, h) + i * a.g.ns + c;
  const int16_t* pl = lo + ((b * a.nq + i) * a.H + h) * a.d + c;
  float s = 0.f;
  if (VEC) {
    if (live && c < a.d) {
      const uint4 vo = *reinterpret_cast<const uint4*>(po), vg = *reinterpret_cast<const uint4*>(pg),
                  vl = *reinterpret_cast<const uint4*>(pl);
      const uint32_t wo[4] = {vo.x, vo.y, vo.z, vo.w}, wg[4] = {vg.x, vg.y, vg.z, vg.w}, wl[4] = {vl.x, vl.y, vl.z, vl.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float a0 = lo_f(wo[k]), a1 = hi_f(wo[k]);
        const int l0 = (int)(wl[k] << 16) >> 16, l1 = (int)wl[k] >> 16;
        s += (a0 == a0 ? __uint_as_float(__float_as_uint(a0) + l0) : a0) * lo_f(wg[k]);
        s += (a1 == a1 ? __uint_as_float(__float_as_uint(a1) + l1) : a1) * hi_f(wg[k]);
      }
    }
  } else if (live) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < a.d) {
        float v = to_f(po[e]);
        if (v == v) v = __uint_as_float(__float_as_uint(v) + (int)pl[e]);
        s += v * to_f(pg[e]);
      }
  }
#pragma unroll
  for (int k = 1; k < L; k <<= 1) s += __shfl_xor_sync(0xffffffffu, s, k);
  if (!live || sub) return;
  const float m = stats[at], l = stats[a.rows_plane + at];
  const bool none = l == 0.f;  // sees nothing: p = exp(t - inf) = 0
  rows[at] = make_float4(none ? INFINITY : m, none ? 0.f : -log2f(l), l == 1.f ? 1.f : 0.f, none ? 0.f : -s);
}

// bf16 values that p and ds are split into as operands of the second product, whatever the size of the problem: 16
// bits of them, so that a gradient is the fp32 one rounded once (1e-4 from the rounded fp64 value, 2-norm). One
// value would leave 2.7e-3 there, and take 2.0 instead of 2.4 ms for dk and dv and 2.3 instead of 2.5 ms for dq and
// dbias of 768 rows of 768 tokens, four heads.
constexpr int kTerms = 2;
// 16 x 16 values in accumulator layout as left operands (left as what the last term drops)
__device__ __forceinline__ void split_terms(uint32_t (&da)[kTerms][4], float (&y)[2][4]) {
#pragma unroll
  for (int term = 0; term < kTerms; ++term)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float* v = &y[i >> 1][2 * (i & 1)];
      da[term][i] = pack_bf16(v[0], v[1]);
      if (term + 1 < kTerms) fma2(F2(lo_f(da[term][i]), hi_f(da[term][i])), F2(-1.f), F2(v[0], v[1])).get(v[0], v[1]);
    }
}

// ---------------------------------------------------------------- dq (and dbias of one batch entry)

template <int DP, int BT>
__device__ __forceinline__ void dq_block(const Args& a, unsigned id, int64_t tiles) {
  using S = Tile<DP>;
  constexpr int QR = 64, KS = DP / 16, NB = DP / 8, RB = S::RB, BS = BT == 2 ? 4 : 2;
  constexpr int kV = 2 * kTile * RB;  // from a K tile to its V tile
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sq = smem_addr(raw), sg = sq + QR * RB, sk = sg + QR * RB;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const unsigned tile = id % (unsigned)tiles;
  id /= (unsigned)tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV);
  const int64_t b = id / a.H, nk = a.nk;
  if (b >= a.B) return;  // makes up a whole cluster
  const int64_t i0 = (int64_t)tile * QR, w0 = i0 + warp * 16;
  const int nt = (int)((nk + kTile - 1) / kTile);
  const int bvec = a.bias_vec;
  const bool work = w0 < a.nq, put = BT && a.dbias != nullptr;
  load_rows<DP, QR>(sq, head_base(a.q, b, h), a.q.ns, a.vec_q, i0, a.nq, a.d, ~0ull);
  load_rows<DP, QR>(sg, head_base(a.g, b, h), a.g.ns, a.vec_g, i0, a.nq, a.d, ~0ull);
  Stream<DP> ks(head_base(a.k, b, kh), a.k.ns, a.vec_k, 0, nk, a.d), vs(head_base(a.v, b, kh), a.v.ns, a.vec_v, 0, nk, a.d);
  auto issue = [&](int kt, uint64_t live) {
    const uint32_t s = sk + (kt & 1) * kTile * RB;
    ks.next(s, live, a.vec_k);
    vs.next(s + kV, live, a.vec_v);
    cp_commit();
  };
  uint32_t ka[KS], ta[KS];
  {
    const LaneAddr<DP> lb = lane_b<DP>(), lt = lane_bt<DP>();
#pragma unroll
    for (int k = 0; k < KS; ++k) ka[k] = lb.at(sk, 0, k), ta[k] = lt.at(sk, 0, k);
  }
  const char* bp[2];  // the lane's first key of the tile, in its rows of the bias and of dbias
  char* dp[2];
  F2 nmx[2], lg[2], nd[2];
  bool peaked = false;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g, ic = i < a.nq ? i : a.nq - 1;
    bp[r] = BT ? bias_row<BT>(a, b, h, ic) + 4 * t * BS : nullptr;
    dp[r] = (put && i < a.nq) ? (char*)a.dbias + (b * a.db_bs + (int64_t)h * a.db_hs + i * a.db_rs + 4 * t) * BS : nullptr;
    const float4 c = ((const float4*)a.rows)[(b * a.H + h) * a.nq + ic];
    nmx[r] = F2(-c.x), lg[r] = F2(c.y), nd[r] = F2(c.w);
    peaked |= c.z != 0.f;
  }
  peaked = __any_sync(0xffffffffu, peaked);
  // what the body without checks needs of the warp's rows
  const bool plain = !peaked && (BT == 0 || bvec) && (!put || (a.db_vec && w0 + 16 <= a.nq));
  Bias4<BT> ring[2][2];
  auto fetch = [&](int slot, int q, int64_t j0, bool fast) {
    if (BT == 0) return;
#pragma unroll
    for (int r = 0; r < 2; ++r) bias_get<BT>(ring[slot][r], bp[r] + q * 16 * BS, j0 + q * 16 + 4 * t, nk, fast);
  };
  const F2 scale(a.scale);
  float acc[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
  uint32_t fq[KS][4], fg[KS][4];
  uint64_t bits = seen_ballot(seen_raw(a, b, 0));
  if (nt > 0) issue(0, bits);
  float2 rawm = seen_raw(a, b, kTile);
  auto body = [&](auto mode, int64_t j0, uint32_t off, bool nf) {
    constexpr bool FAST = decltype(mode)::value;
    uint32_t kc[KS], tc[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) kc[k] = ka[k] + off, tc[k] = ta[k] + off;
#pragma unroll 1
    for (int hb = 0; hb < 2; ++hb) {
      unrolled<2>([&](auto Q) {  // 16 keys
        constexpr int q = decltype(Q)::value;
        float x[2][4], y[2][4];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r[4], u[4];
          ldsm4i<q * 16 * RB>(r, kc[k]);
          ldsm4i<q * 16 * RB + kV>(u, kc[k]);
          if (k == 0) {
            mma0(x[0], fq[k], r[0], r[1]);
            mma0(x[1], fq[k], r[2], r[3]);
            mma0(y[0], fg[k], u[0], u[1]);
            mma0(y[1], fg[k], u[2], u[3]);
          } else {
            mma(x[0], fq[k], r[0], r[1]);
            mma(x[1], fq[k], r[2], r[3]);
            mma(y[0], fg[k], u[0], u[1]);
            mma(y[1], fg[k], u[2], u[3]);
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, ring[q][r], n);
        fetch(q, 2 * hb + q + 2, j0, hb == 0 ? FAST || (bvec && j0 + (q + 3) * 16 <= nk) : nf);
        if (!FAST) {
          const uint32_t mine = (uint32_t)(bits >> (32 * hb + 16 * q + 4 * t));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((mine >> (2 * n + e)) & 1)) x[n][e] = x[n][2 + e] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const F2 p = prob2(&x[n][2 * r], nmx[r], lg[r]);
            if (!FAST) p.get(x[n][2 * r], x[n][2 * r + 1]);
            mul2(p, add2(F2(y[n][2 * r], y[n][2 * r + 1]), nd[r])).get(y[n][2 * r], y[n][2 * r + 1]);
          }
        if (!FAST && peaked) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (x[n][e] == 1.f) y[n][e] = 0.f;
        }
        if (!FAST) {  // a hidden key's ds is 0, whatever do holds
          const uint32_t mine = (uint32_t)(bits >> (32 * hb + 16 * q + 4 * t));
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((mine >> (2 * n + e)) & 1)) y[n][e] = y[n][2 + e] = 0.f;
        }
        if (put) {
          const int64_t j = j0 + hb * 32 + q * 16 + 4 * t;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (FAST || dp[r])
              put_bias4<BT>(dp[r] + (hb * 32 + q * 16) * BS, j, nk, FAST || (a.db_vec && j0 + hb * 32 + q * 16 + 16 <= nk),
                            y[0][2 * r], y[0][2 * r + 1], y[1][2 * r], y[1][2 * r + 1]);
        }
        uint32_t da[kTerms][4];
        split_terms(da, y);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          uint32_t f[4];
          ldsm4_ti<q * 16 * RB>(f, tc[c]);
#pragma unroll
          for (int term = 0; term < kTerms; ++term) {
            mma(acc[2 * c], da[term], f[0], f[1]);
            mma(acc[2 * c + 1], da[term], f[2], f[3]);
          }
        }
      });
#pragma unroll
      for (int k = 0; k < KS; ++k) kc[k] += 32 * RB, tc[k] += 32 * RB;
    }
  };
  if (work) {
    fetch(0, 0, 0, bvec && 16 <= nk);
    fetch(1, 1, 0, bvec && 32 <= nk);
  }
  for (int kt = 0; kt < nt; ++kt) {
    const uint64_t next = seen_ballot(rawm);
    const int64_t j0 = (int64_t)kt * kTile;
    cp_wait<0>();
    __syncthreads();
    if (kt == 0) {
      const LaneAddr<DP> la = lane_a<DP>();
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        ldsm4(fq[k], la.at(sq, warp, k));
        ldsm4(fg[k], la.at(sg, warp, k));
      }
    }
    if (kt + 1 < nt) issue(kt + 1, next);
    rawm = seen_raw(a, b, j0 + 2 * kTile);
    if (work) {
      const bool nf = bvec && j0 + kTile + 32 <= nk;  // the next tile's first two groups
      const uint32_t off = (kt & 1) * kTile * RB;
      if (bits == ~0ull && plain) {
        body(std::true_type{}, j0, off, nf);
      } else if (bits != 0 || put) {
        body(std::false_type{}, j0, off, nf);
      } else {  // no visible key
        fetch(0, 4, j0, nf);
        fetch(1, 5, j0, nf);
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        bp[r] += kTile * BS;
        if (dp[r]) dp[r] += kTile * BS;
      }
    }
    bits = next;
  }
  cp_commit();
  cp_wait<0>();
  if (!a.dq) return;
  const bool vec = pair_ok(a.dq, a.o_bs, a.o_ns, a.o_hs, a.d);
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    if (i >= a.nq) continue;
    bf16* o = (bf16*)a.dq + b * a.o_bs + (int64_t)h * a.o_hs + i * a.o_ns;
#pragma unroll
    for (int n = 0; n < NB; ++n)
      store_pair(o, n * 8 + 2 * t, a.d, vec, acc[n][2 * r] * a.scale, acc[n][2 * r + 1] * a.scale);
  }
}

// ---------------------------------------------------------------- dk, dv

// 16 keys per warp (32 need 168 registers where 16 need 128, and three blocks on an SM are slower than four:
// 768 tokens 2.5 against 2.4 ms); HOLD: their fragments stay in registers.
template <int DP, int BT>
__device__ __forceinline__ void dkv_block(const Args& a, unsigned id, int64_t tiles, int rank, int ranks) {
  using S = Tile<DP>;
  constexpr int KR = 64, KS = DP / 16, NB = DP / 8, RB = S::RB, BS = BT == 2 ? 4 : 2;
  constexpr bool HOLD = DP <= 64;
  constexpr int kG = 2 * kTile * RB;  // from a Q tile to its dO tile
  extern __shared__ __align__(128) unsigned char raw[];
  const uint32_t sk = smem_addr(raw), sv = sk + KR * RB, sq = sv + KR * RB, sc = sq + 2 * kG;
  const float4* cst = (const float4*)(raw + (sc - sk));  // [2][64]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> lb = lane_b<DP>();
  const unsigned tile = id % (unsigned)tiles;
  id /= (unsigned)tiles;
  const int kh = id % a.KV, group = a.H / a.KV;
  const int64_t b = id / a.KV, nq = a.nq;
  const int64_t j0 = (int64_t)tile * KR, w0 = j0 + warp * 16;
  const int per = (int)((nq + kTile - 1) / kTile);
  const uint64_t live = seen_ballot(seen_raw(a, b, j0));  // visible keys of the block
  load_rows<DP, 64>(sk, head_base(a.k, b, kh), a.k.ns, a.vec_k, j0, a.nk, a.d, live);
  load_rows<DP, 64>(sv, head_base(a.v, b, kh), a.v.ns, a.vec_v, j0, a.nk, a.d, live);
  constexpr uint32_t kAll = 0xffffu;
  const uint32_t mine = (uint32_t)(live >> (warp * 16)) & kAll;  // and of the warp
  const bool bfast = a.bias_vec && w0 + 16 <= a.nk;
  const bool plain = mine == kAll && (BT == 0 || bfast);  // the body without checks
  uint32_t qa[KS], ta[KS];
  {
    const LaneAddr<DP> la = lane_a<DP>(), ln = lane_bn<DP>();
#pragma unroll
    for (int k = 0; k < KS; ++k) qa[k] = la.at(sq, 0, k), ta[k] = ln.at(sq, 0, k);
  }
  const F2 scale(a.scale);
  float dk[NB][4], dv[NB][4];
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) dk[n][e] = dv[n][e] = 0.f;
  uint32_t fk[HOLD ? KS : 1][4], fv[HOLD ? KS : 1][4];
  Bias4<BT> ring[2][2];
  const char* bp[2] = {nullptr, nullptr};  // the lane's first key in rows g, g + 8 of the block that is read next
  const int64_t bstep = a.b_rs * 16 * BS;
  auto fetch = [&](int slot, int64_t i0, bool fast) {  // rows i0 .. i0 + 15; 0 past the end
    if (BT == 0) return;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool row = fast || i0 + 8 * r + g < nq;
      if (row) {
        bias_get<BT>(ring[slot][r], bp[r], w0 + 4 * t, a.nk, fast || bfast);
      } else {
#pragma unroll
        for (int w = 0; w < (BT == 2 ? 4 : (BT == 1 ? 2 : 1)); ++w) ring[slot][r].w[w] = 0;
      }
      bp[r] += bstep;
    }
  };
  auto body = [&](auto mode, int64_t i0, int s, bool nf) {
    constexpr bool FAST = decltype(mode)::value;
    const uint32_t off = s * kTile * RB;
    uint32_t qc[KS], tc[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) qc[k] = qa[k] + off, tc[k] = ta[k] + off;
#pragma unroll 1
    for (int hb = 0; hb < 2; ++hb) {
      unrolled<2>([&](auto B) {  // 16 queries
        constexpr int blk = decltype(B)::value;
        float x[2][4], y[2][4];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t fq[4], fg[4];
          ldsm4i<blk * 16 * RB>(fq, qc[k]);
          ldsm4i<blk * 16 * RB + kG>(fg, qc[k]);
          uint32_t rk[4], rv[4];
          if (HOLD) {
#pragma unroll
            for (int i = 0; i < 4; ++i) rk[i] = fk[k][i], rv[i] = fv[k][i];
          } else {
            ldsm4(rk, lb.at(sk, warp, k));
            ldsm4(rv, lb.at(sv, warp, k));
          }
          if (k == 0) {
            mma0(x[0], fq, rk[0], rk[1]);
            mma0(x[1], fq, rk[2], rk[3]);
            mma0(y[0], fg, rv[0], rv[1]);
            mma0(y[1], fg, rv[2], rv[3]);
          } else {
            mma(x[0], fq, rk[0], rk[1]);
            mma(x[1], fq, rk[2], rk[3]);
            mma(y[0], fg, rv[0], rv[1]);
            mma(y[1], fg, rv[2], rv[3]);
          }
        }
        const float4 c[2] = {cst[s * kTile + hb * 32 + blk * 16 + g], cst[s * kTile + hb * 32 + blk * 16 + 8 + g]};
        const F2 nmx[2] = {F2(-c[0].x), F2(-c[1].x)}, lg[2] = {F2(c[0].y), F2(c[1].y)}, nd[2] = {F2(c[0].w), F2(c[1].w)};
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, ring[blk][r], n);
        fetch(blk, i0 + hb * 32 + blk * 16 + 32, hb == 0 ? FAST : nf);
        if (!FAST) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((mine >> (4 * t + 2 * n + e)) & 1)) x[n][e] = x[n][2 + e] = -INFINITY;
        }
        const bool peaked = __any_sync(0xffffffffu, c[0].z != 0.f || c[1].z != 0.f);
        uint32_t pa[kTerms][4], da[kTerms][4];
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float p[2], ds[2];
            const F2 p2 = prob2(&x[n][2 * r], nmx[r], lg[r]);
            p2.get(p[0], p[1]);
            mul2(p2, add2(F2(y[n][2 * r], y[n][2 * r + 1]), nd[r])).get(ds[0], ds[1]);
            if (peaked) {
              if (p[0] == 1.f) ds[0] = 0.f;
              if (p[1] == 1.f) ds[1] = 0.f;
            }
#pragma unroll
            for (int term = 0; term < kTerms; ++term) {
              const uint32_t a = pack_bf16(p[0], p[1]), c = pack_bf16(ds[0], ds[1]);
              pa[term][2 * r + n] = transpose8(a);
              da[term][2 * r + n] = transpose8(c);
              if (term + 1 < kTerms) {
                fma2(F2(lo_f(a), hi_f(a)), F2(-1.f), F2(p[0], p[1])).get(p[0], p[1]);
                fma2(F2(lo_f(c), hi_f(c)), F2(-1.f), F2(ds[0], ds[1])).get(ds[0], ds[1]);
              }
            }
          }
#pragma unroll
        for (int n = 0; n < KS; ++n) {
          uint32_t fg[4], fq[4];
          ldsm4_ti<blk * 16 * RB + kG>(fg, tc[n]);
          ldsm4_ti<blk * 16 * RB>(fq, tc[n]);
#pragma unroll
          for (int term = 0; term < kTerms; ++term) {
            mma(dv[2 * n], pa[term], fg[0], fg[1]);
            mma(dv[2 * n + 1], pa[term], fg[2], fg[3]);
            mma(dk[2 * n], da[term], fq[0], fq[1]);
            mma(dk[2 * n + 1], da[term], fq[2], fq[3]);
          }
        }
      });
#pragma unroll
      for (int k = 0; k < KS; ++k) qc[k] += 32 * RB, tc[k] += 32 * RB;
    }
  };
  if (live != 0 && per > 0) {
    int it = 0;
    const int heads = group / ranks, first = rank * heads;
    for (int hh = first; hh < first + heads; ++hh) {
      const int h = kh * group + hh;
      Stream<DP> qs(head_base(a.q, b, h), a.q.ns, a.vec_q, 0, nq, a.d), gs(head_base(a.g, b, h), a.g.ns, a.vec_g, 0, nq, a.d);
      const float4* pr = (const float4*)a.rows + (b * a.H + h) * nq;
      auto issue = [&](int qt, int s) {
        const uint64_t rows = first_bits(nq - (int64_t)qt * kTile);
        qs.next(sq + s * kTile * RB, rows, a.vec_q);
        gs.next(sq + kG + s * kTile * RB, rows, a.vec_g);
        if (threadIdx.x < kTile) {
          const int64_t i = (int64_t)qt * kTile + threadIdx.x;
          cp_async16(sc + (s * kTile + threadIdx.x) * 16, i < nq ? pr + i : pr, i < nq);
        }
        cp_commit();
      };
      if (hh > first) __syncthreads();  // the last head's tiles are done with
      issue(0, it & 1);
      if (BT) {
#pragma unroll
        for (int r = 0; r < 2; ++r) bp[r] = bias_row<BT>(a, b, h, 8 * r + g) + (w0 + 4 * t) * BS;
      }
      fetch(0, 0, false);
      fetch(1, 16, false);
      for (int qt = 0; qt < per; ++qt, ++it) {
        const int s = it & 1;
        cp_wait<0>();
        __syncthreads();
        if (HOLD && it == 0) {
#pragma unroll
          for (int k = 0; k < (HOLD ? KS : 1); ++k) {
            ldsm4(fk[k], lb.at(sk, warp, k));
            ldsm4(fv[k], lb.at(sv, warp, k));
          }
        }
        if (qt + 1 < per) issue(qt + 1, s ^ 1);
        if (mine == 0) continue;  // none of the warp's keys is visible
        const int64_t i0 = (int64_t)qt * kTile;
        const bool nf = plain && i0 + kTile + 32 <= nq;  // the next tile's first two blocks
        if (plain && i0 + kTile <= nq)
          body(std::true_type{}, i0, s, nf);
        else
          body(std::false_type{}, i0, s, nf);
      }
    }
  }
  cp_commit();
  cp_wait<0>();
  const bool vk = pair_ok(a.dk, a.dk_bs, a.dk_ns, a.dk_hs, a.d), vv = pair_ok(a.dv, a.dv_bs, a.dv_ns, a.dv_hs, a.d);
  if (ranks > 1) {
    bf16* pk = (bf16*)a.dk + b * a.dk_bs + (int64_t)kh * a.dk_hs + j0 * a.dk_ns;
    bf16* pv = (bf16*)a.dv + b * a.dv_bs + (int64_t)kh * a.dv_hs + j0 * a.dv_ns;
    sum_ranks<DP>(raw, dk, dv, ranks, rank, [&](int which, int row, int c, float v0, float v1) {
      if (j0 + row >= a.nk) return;
      if (which == 0)
        store_pair(pk + row * a.dk_ns, c, a.d, vk, v0 * a.scale, v1 * a.scale);
      else
        store_pair(pv + row * a.dv_ns, c, a.d, vv, v0, v1);
    });
    return;
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t j = w0 + perm_row(g, r);  // row g + 8 r of the block holds this key
    if (j >= a.nk) continue;
    bf16* ok = (bf16*)a.dk + b * a.dk_bs + (int64_t)kh * a.dk_hs + j * a.dk_ns;
    bf16* ov = (bf16*)a.dv + b * a.dv_bs + (int64_t)kh * a.dv_hs + j * a.dv_ns;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      store_pair(ok, n * 8 + 2 * t, a.d, vk, dk[n][2 * r] * a.scale, dk[n][2 * r + 1] * a.scale);
      store_pair(ov, n * 8 + 2 * t, a.d, vv, dv[n][2 * r], dv[n][2 * r + 1]);
    }
  }
}

// dk and dv in the first blocks, dq in the others (either may be none): where neither fills the machine they
// run side by side.
template <int DP, int BT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? 4 : 2) k_dqkv(Args a, unsigned dkv_blocks, int ranks) {
  if (blockIdx.x < dkv_blocks)
    dkv_block<DP, BT>(a, blockIdx.x / ranks, (a.nk + 63) / 64, blockIdx.x % ranks, ranks);
  else
    dq_block<DP, BT>(a, blockIdx.x - dkv_blocks, (a.nq + 63) / 64);
}

// ---------------------------------------------------------------- dbias shared by the batch

// A 128 x 64 tile of one head's plane, summed over the batch entries of a part; with one part the
// result is written, else an fp32 partial plane [part][H][n_q][n_k] that k_sum_planes adds up.
template <int DP, int BT>
__global__ void __launch_bounds__(kThreads, DP == 32 ? 3 : 1) k_dbias(Args a, float* part, int parts) {
  using S = Tile<DP>;
  constexpr int MT = 2, QR = 128, KS = DP / 16;
  constexpr bool HOLD = DP == 32;
  extern __shared__ __align__(128) unsigned char raw[];
  constexpr int kStage = (2 * QR + 2 * kTile) * S::RB + QR * 16;
  const uint32_t s0 = smem_addr(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>();
  unsigned id = blockIdx.x;
  const unsigned nkt = (unsigned)((a.nk + kTile - 1) / kTile);
  const unsigned kt = id % nkt;
  id /= nkt;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV);
  const int p = id / a.H;
  const int64_t b0 = a.B * p / parts, b1 = a.B * (p + 1) / parts;
  const int64_t i0 = (int64_t)tile * QR, w0 = i0 + warp * 16 * MT, j0 = (int64_t)kt * kTile;
  auto issue = [&](int64_t b, uint64_t live) {
    const uint32_t q = s0 + (int)(b & 1) * kStage, gr = q + QR * S::RB, k = gr + QR * S::RB, v = k + kTile * S::RB,
                   c = v + kTile * S::RB;
    load_rows<DP, QR>(q, head_base(a.q, b, h), a.q.ns, a.vec_q, i0, a.nq, a.d, ~0ull);
    load_rows<DP, QR>(gr, head_base(a.g, b, h), a.g.ns, a.vec_g, i0, a.nq, a.d, ~0ull);
    load_rows<DP, kTile>(k, head_base(a.k, b, kh), a.k.ns, a.vec_k, j0, a.nk, a.d, live);
    load_rows<DP, kTile>(v, head_base(a.v, b, kh), a.v.ns, a.vec_v, j0, a.nk, a.d, live);
    const int64_t i = i0 + threadIdx.x;  // kThreads == QR
    const float4* pr = (const float4*)a.rows + (b * a.H + h) * a.nq;
    cp_async16(c + threadIdx.x * 16, i < a.nq ? pr + i : pr, i < a.nq);
    cp_commit();
  };
  const char* brow[MT][2];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + m * 16 + r * 8 + g;
      brow[m][r] = bias_row<BT>(a, 0, h, i < a.nq ? i : a.nq - 1);
    }
  const bool fast = a.bias_vec && j0 + kTile <= a.nk;
  const F2 scale(a.scale);
  float acc[MT][8][4];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[m][n][e] = 0.f;
  uint64_t bits = b0 < b1 ? seen_ballot(seen_raw(a, b0, j0)) : 0;
  if (b0 < b1) issue(b0, bits);
  float2 rawm = b0 + 1 < b1 ? seen_raw(a, b0 + 1, j0) : make_float2(0.f, 0.f);
  for (int64_t b = b0; b < b1; ++b) {
    const uint64_t next = seen_ballot(rawm);
    cp_wait<0>();
    __syncthreads();
    if (b + 1 < b1) issue(b + 1, next);
    rawm = b + 2 < b1 ? seen_raw(a, b + 2, j0) : make_float2(0.f, 0.f);
    if (bits == 0 || w0 >= a.nq) {
      bits = next;
      continue;
    }
    const uint32_t tq = s0 + (int)(b & 1) * kStage, tg = tq + QR * S::RB, tk = tg + QR * S::RB,
                   tv = tk + kTile * S::RB;
    const float4* cst = (const float4*)(raw + (int)(b & 1) * kStage + (2 * QR + 2 * kTile) * S::RB);
    uint32_t fq[HOLD ? MT : 1][HOLD ? KS : 1][4], fg[HOLD ? MT : 1][HOLD ? KS : 1][4];
    if (HOLD) {
#pragma unroll
      for (int m = 0; m < (HOLD ? MT : 1); ++m)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          ldsm4(fq[m][k], la.at(tq, warp * MT + m, k));
          ldsm4(fg[m][k], la.at(tg, warp * MT + m, k));
        }
    }
    F2 nmx[MT][2], lg[MT][2], nd[MT][2];
    bool peaked = false;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float4 c = cst[warp * 16 * MT + m * 16 + r * 8 + g];
        nmx[m][r] = F2(-c.x), lg[m][r] = F2(c.y), nd[m][r] = F2(c.w);
        peaked |= c.z != 0.f;
      }
    peaked = __any_sync(0xffffffffu, peaked);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      Bias4<BT> br[MT][2];  // the same every batch entry: from L1
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 2; ++r) bias_load<BT>(br[m][r], brow[m][r], j0 + q * 16 + 4 * t, a.nk, fast);
      float x[MT][2][4], y[MT][2][4];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        uint32_t r[4], u[4];
        ldsm4(r, lb.at(tk, q, k));
        ldsm4(u, lb.at(tv, q, k));
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          uint32_t rq[4], rg[4];
          if (HOLD) {
#pragma unroll
            for (int i = 0; i < 4; ++i) rq[i] = fq[m][k][i], rg[i] = fg[m][k][i];
          } else {
            ldsm4(rq, la.at(tq, warp * MT + m, k));
            ldsm4(rg, la.at(tg, warp * MT + m, k));
          }
          if (k == 0) {
            mma0(x[m][0], rq, r[0], r[1]);
            mma0(x[m][1], rq, r[2], r[3]);
            mma0(y[m][0], rg, u[0], u[1]);
            mma0(y[m][1], rg, u[2], u[3]);
          } else {
            mma(x[m][0], rq, r[0], r[1]);
            mma(x[m][1], rq, r[2], r[3]);
            mma(y[m][0], rg, u[0], u[1]);
            mma(y[m][1], rg, u[2], u[3]);
          }
        }
      }
      const uint32_t qbits = (uint32_t)(bits >> (16 * q)) & 0xffffu;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float* v = &x[m][n][2 * r];
            float* d = &acc[m][2 * q + n][2 * r];
            score2<BT>(v, scale, br[m][r], n);
            if (qbits != 0xffffu) {
              if (!((qbits >> (4 * t + 2 * n)) & 1)) v[0] = -INFINITY;
              if (!((qbits >> (4 * t + 2 * n + 1)) & 1)) v[1] = -INFINITY;
            }
            const F2 p = prob2(v, nmx[m][r], lg[m][r]);
            F2 dl = add2(F2(y[m][n][2 * r], y[m][n][2 * r + 1]), nd[m][r]);
            if (peaked) {
              float p0, p1, d0, d1;
              p.get(p0, p1);
              dl.get(d0, d1);
              dl = F2(p0 == 1.f ? 0.f : d0, p1 == 1.f ? 0.f : d1);
            }
            fma2(p, dl, F2(d[0], d[1])).get(d[0], d[1]);
          }
    }
    bits = next;
  }
  cp_commit();
  cp_wait<0>();
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + m * 16 + r * 8 + g;
      if (i >= a.nq) continue;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int64_t j = j0 + q * 16 + 4 * t;
        const float v0 = acc[m][2 * q][2 * r], v1 = acc[m][2 * q][2 * r + 1], v2 = acc[m][2 * q + 1][2 * r],
                    v3 = acc[m][2 * q + 1][2 * r + 1];
        if (parts == 1)
          store_bias4<BT>(a, (char*)a.dbias + ((int64_t)h * a.db_hs + i * a.db_rs) * (BT == 2 ? 4 : 2), j,
                          a.db_vec && j0 + q * 16 + 16 <= a.nk, v0, v1, v2, v3);
        else
          store_bias4<2>(a, (char*)(part + (((int64_t)p * a.H + h) * a.nq + i) * a.nk), j,
                         (a.nk & 3) == 0 && j0 + q * 16 + 16 <= a.nk, v0, v1, v2, v3);
      }
    }
}

// ---------------------------------------------------------------- dq and a shared dbias in one pass

// The gradient of a bias that the batch shares is a sum over the batch, dq a sum over the keys: one pass
// can do both if a block keeps its rows of the [n_q, n_k] plane while it walks over the batch. A block of
// 16 warps takes 64 rows by all keys of one head and a part of the batch: warp w rows 16 (w % 4).. and
// the w / 4-th quarter of the keys. Its share of the plane, 16 rows by n_k / 4 keys in fp32, lies in tensor
// memory as thread-private storage (128 words per thread: up to 1024 keys); a group of 16 keys costs one
// eight-word load, four packed adds and one store. All keys and values of a batch entry are in shared
// memory, double-buffered (up to 832 keys of 32 channels), so warps run freely between two entries; the
// quarters' dq are added through shared memory. Next to dq and dbias apart this saves two of five products
// and one of two exponentials per score (768 rows of 768 tokens, four heads: 2.5 ms; apart, 900 rows of 900, 1.6
// times the scores: 6.8 ms). It is bound by instruction issue.
constexpr int kPlaneThreads = 512;
constexpr int kPlaneKeys = 832;

struct PlaneSmem {  // byte offsets
  int kv, q, cst, vis, end;
  __host__ __device__ explicit PlaneSmem(int nkp) {
    const int one = 2 * nkp * 64, red = 4 * 64 * 36 * 4;  // keys and values; the quarters' dq
    kv = one > red ? one : red;
    q = 2 * kv;
    cst = q + 2 * 2 * 64 * 64;
    vis = cst + 2 * 64 * 16;
    end = vis + 3 * 32 * 4 + 16;
  }
};

template <int BT>
__global__ void __launch_bounds__(kPlaneThreads, 1) k_dq_plane(Args a, float* part, int parts, int G, int tcols) {
  constexpr int DP = 32, KS = 2, NB = 4, BS = BT == 2 ? 4 : 2;
  using S = Tile<DP>;
  extern __shared__ __align__(128) unsigned char raw[];
  const int nkp = (int)((a.nk + 31) / 32) * 32;
  const PlaneSmem L(nkp);
  const uint32_t s0 = smem_addr(raw);
  uint32_t* vis = (uint32_t*)(raw + L.vis);  // [3][32] words of visible keys
  uint32_t* tptr = vis + 96;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rg = warp & 3, sl = warp >> 2;
  const LaneAddr<DP> la = lane_a<DP>(), lb = lane_b<DP>(), lt = lane_bt<DP>();
  unsigned id = blockIdx.x;
  const unsigned tile = id % (unsigned)a.tiles;
  id /= (unsigned)a.tiles;
  const int h = id % a.H, kh = h / (a.H / a.KV);
  const int pt = id / a.H;
  const int64_t b0 = a.B * pt / parts, b1 = a.B * (pt + 1) / parts;
  const int64_t i0 = (int64_t)tile * 64, w0 = i0 + rg * 16;
  const int words = nkp / 32;

  if (warp == 0) {
    sm100::tmem_alloc(smem_addr(tptr), tcols);
    sm100::tmem_relinquish();
  }
  auto see = [&](int64_t b) {  // the words of entry b
    for (int w = warp; w < words; w += 16) {
      const int64_t j = w * 32 + lane;
      const unsigned m = __ballot_sync(0xffffffffu, j < a.nk && (!a.mask || a.mask[b * a.m_bs + j * a.m_ks] != 0.f));
      if (lane == 0) vis[(int)(b % 3) * 32 + w] = m;
    }
  };
  auto issue = [&](int64_t b) {
    const uint32_t* v = vis + (int)(b % 3) * 32;
    const uint32_t sk = s0 + (int)(b & 1) * L.kv, sv = sk + nkp * S::RB, sq = s0 + L.q + (int)(b & 1) * 8192,
                   sg = sq + 4096;
    const bf16 *pk = head_base(a.k, b, kh), *pv = head_base(a.v, b, kh), *pq = head_base(a.q, b, h),
               *pg = head_base(a.g, b, h);
    const int row = threadIdx.x >> 2, c = threadIdx.x & 3;
    const uint32_t dst = S::off(row, c);  // rows 128 apart have the same swizzle
    const bool col = c * 8 < a.d;
    auto keys = [&](uint32_t sm, const bf16* p, int64_t ns, int vec) {
      if (vec) {
        const char* q = (const char*)(p + row * ns + c * 8);
        const int64_t step = ns * 256;
        for (int r = row; r < nkp; r += 128, q += step, sm += 128 * S::RB)
          cp_async16(sm + dst, q, col && ((v[r >> 5] >> (r & 31)) & 1));  // no bits past the end
      } else {
        for (int i = threadIdx.x; i < nkp * DP; i += kPlaneThreads) {
          const int r = i / DP, e = i % DP;
          const bool ok = e < a.d && ((v[r >> 5] >> (r & 31)) & 1);
          const bf16 x = ok ? p[r * ns + e] : from_f<bf16>(0.f);
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(sm + S::off(r, e >> 3) + (e & 7) * 2),
                       "h"(*reinterpret_cast<const unsigned short*>(&x))
                       : "memory");
        }
      }
    };
    auto queries = [&](uint32_t sm, const bf16* p, int64_t ns, int vec) {
      if (vec) {
        if (row < 64) cp_async16(sm + dst, p + (i0 + row) * ns + c * 8, col && i0 + row < a.nq);
      } else {
        for (int i = threadIdx.x; i < 64 * DP; i += kPlaneThreads) {
          const int r = i / DP, e = i % DP;
          const bf16 x = e < a.d && i0 + r < a.nq ? p[(i0 + r) * ns + e] : from_f<bf16>(0.f);
          asm volatile("st.shared.b16 [%0], %1;" ::"r"(sm + S::off(r, e >> 3) + (e & 7) * 2),
                       "h"(*reinterpret_cast<const unsigned short*>(&x))
                       : "memory");
        }
      }
    };
    keys(sk, pk, a.k.ns, a.vec_k);
    keys(sv, pv, a.v.ns, a.vec_v);
    queries(sq, pq, a.q.ns, a.vec_q);
    queries(sg, pg, a.g.ns, a.vec_g);
    if (threadIdx.x < 64) {
      const int64_t i = i0 + threadIdx.x;
      const float4* pr = (const float4*)a.rows + (b * a.H + h) * a.nq;
      cp_async16(s0 + L.cst + (int)(b & 1) * 1024 + threadIdx.x * 16, i < a.nq ? pr + i : pr, i < a.nq);
    }
    cp_commit();
  };
  if (b0 < b1) see(b0);
  if (b0 + 1 < b1) see(b0 + 1);
  const int q0 = sl * G;  // the warp's groups: q0 .. q0 + G - 1, in pairs
  const char* brow[2];    // the lane's first key of the first pair
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int64_t i = w0 + r * 8 + g;
    brow[r] = bias_row<BT>(a, 0, h, i < a.nq ? i : a.nq - 1) + (q0 * 16 + 4 * t) * BS;
  }
  Bias4<BT> ring[2][2];
  auto fetch = [&](int u, const char* const (&p)[2], int64_t j, bool fast) {  // group u of the pair at key j
#pragma unroll
    for (int r = 0; r < 2; ++r) bias_get<BT>(ring[u][r], p[r] + u * 16 * BS, j + u * 16 + 4 * t, a.nk, fast);
  };
  auto inside = [&](int64_t j) { return a.bias_vec && j + 32 <= a.nk; };
  fetch(0, brow, q0 * 16, inside(q0 * 16));
  fetch(1, brow, q0 * 16, inside(q0 * 16));
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tbase = *tptr;
  const uint32_t tm0 = tbase + ((uint32_t)(rg * 32) << 16) + q0 * 8;
  {
    const uint32_t zero[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int q = 0; q < G; ++q) tmem_st8(tm0 + q * 8, zero);
    sm100::tmem_st_wait();
  }
  if (b0 < b1) issue(b0);
  const F2 scale(a.scale);
  for (int64_t b = b0; b < b1; ++b) {
    cp_wait<0>();
    __syncthreads();
    if (b + 1 < b1) issue(b + 1);
    if (b + 2 < b1) see(b + 2);
    const uint32_t* v = vis + (int)(b % 3) * 32;
    const uint32_t sk = s0 + (int)(b & 1) * L.kv, sv = sk + nkp * S::RB, sq = s0 + L.q + (int)(b & 1) * 8192,
                   sg = sq + 4096;
    const float4* cst = (const float4*)(raw + L.cst + (int)(b & 1) * 1024);
    uint32_t fq[KS][4], fg[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      ldsm4(fq[k], la.at(sq, rg, k));
      ldsm4(fg[k], la.at(sg, rg, k));
    }
    F2 nmx[2], lg[2], nd[2];
    bool peaked = false;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float4 c = cst[rg * 16 + r * 8 + g];
      nmx[r] = F2(-c.x), lg[r] = F2(c.y), nd[r] = F2(c.w);
      peaked |= c.z != 0.f;
    }
    peaked = __any_sync(0xffffffffu, peaked);
    float acc[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
    uint32_t ka[KS], ta[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k) ka[k] = lb.at(sk, q0, k), ta[k] = lt.at(sk, q0, k);
    const uint32_t dv = sv - sk;
    uint32_t tm_at = tm0;
    const char* bp[2] = {brow[0], brow[1]};
    auto pair = [&](auto mode, uint32_t bits, int64_t nj, bool nf) {
      constexpr bool FAST = decltype(mode)::value;
      unrolled<2>([&](auto U) {
        constexpr int u = decltype(U)::value;
        uint32_t tm[8];
        tmem_ld8(tm_at + u * 8, tm);
        float x[2][4], y[2][4];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t r[4], w[4];
          ldsm4i<u * 16 * S::RB>(r, ka[k]);
          ldsm4i<u * 16 * S::RB>(w, ka[k] + dv);
          if (k == 0) {
            mma0(x[0], fq[k], r[0], r[1]);
            mma0(x[1], fq[k], r[2], r[3]);
            mma0(y[0], fg[k], w[0], w[1]);
            mma0(y[1], fg[k], w[2], w[3]);
          } else {
            mma(x[0], fq[k], r[0], r[1]);
            mma(x[1], fq[k], r[2], r[3]);
            mma(y[0], fg[k], w[0], w[1]);
            mma(y[1], fg[k], w[2], w[3]);
          }
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) score2<BT>(&x[n][2 * r], scale, ring[u][r], n);
        fetch(u, bp, nj, nf);
        if (!FAST) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (!((bits >> (u * 16 + 4 * t + 2 * n + e)) & 1)) x[n][e] = x[n][2 + e] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const F2 p = prob2(&x[n][2 * r], nmx[r], lg[r]);
            if (!FAST) p.get(x[n][2 * r], x[n][2 * r + 1]);
            mul2(p, add2(F2(y[n][2 * r], y[n][2 * r + 1]), nd[r])).get(y[n][2 * r], y[n][2 * r + 1]);
          }
        if (!FAST && peaked) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (x[n][e] == 1.f) y[n][e] = 0.f;
        }
        tmem_wait8(tm);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float s, s1;
          add2(F2(__uint_as_float(tm[2 * i]), __uint_as_float(tm[2 * i + 1])),
               F2(y[i >> 1][2 * (i & 1)], y[i >> 1][2 * (i & 1) + 1]))
              .get(s, s1);
          tm[2 * i] = __float_as_uint(s), tm[2 * i + 1] = __float_as_uint(s1);
        }
        tmem_st8(tm_at + u * 8, tm);
        uint32_t da[kTerms][4];
        split_terms(da, y);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
          uint32_t f[4];
          ldsm4_ti<u * 16 * S::RB>(f, ta[c]);
#pragma unroll
          for (int term = 0; term < kTerms; ++term) {
            mma(acc[2 * c], da[term], f[0], f[1]);
            mma(acc[2 * c + 1], da[term], f[2], f[3]);
          }
        }
      });
    };
#pragma unroll 1
    for (int qq = 0; qq < G; qq += 2) {
      const int word = (q0 + qq) >> 1;
      const uint32_t bits = word < words ? v[word] : 0;
      const bool last = qq + 2 >= G;  // the next entry starts over with the same bias
#pragma unroll
      for (int r = 0; r < 2; ++r) bp[r] = last ? brow[r] : bp[r] + 32 * BS;
      const int64_t nj = (int64_t)(q0 + (last ? 0 : qq + 2)) * 16;
      const bool nf = inside(nj);
      if (w0 < a.nq) {
        if (bits == 0xffffffffu && !peaked) {
          pair(std::true_type{}, bits, nj, nf);
        } else if (bits != 0) {
          pair(std::false_type{}, bits, nj, nf);
        } else {  // no visible key
          fetch(0, bp, nj, nf);
          fetch(1, bp, nj, nf);
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) ka[k] += 32 * S::RB, ta[k] += 32 * S::RB;
      tm_at += 16;
    }
    sm100::tmem_st_wait();
    if (a.dq) {
      __syncthreads();  // entry b's keys and values are done with
      float* red = (float*)(raw + (int)(b & 1) * L.kv);
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          *reinterpret_cast<float2*>(red + (sl * 64 + rg * 16 + r * 8 + g) * 36 + n * 8 + 2 * t) =
              make_float2(acc[n][2 * r], acc[n][2 * r + 1]);
      __syncthreads();
      const int row = threadIdx.x >> 3, c0 = (threadIdx.x & 7) * 4;
      float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const float4 x = *reinterpret_cast<const float4*>(red + (s * 64 + row) * 36 + c0);
        o[0] += x.x, o[1] += x.y, o[2] += x.z, o[3] += x.w;
      }
      if (i0 + row < a.nq) {
        bf16* p = (bf16*)a.dq + b * a.o_bs + (int64_t)h * a.o_hs + (i0 + row) * a.o_ns;
        const bool vec = pair_ok(a.dq, a.o_bs, a.o_ns, a.o_hs, a.d);
        store_pair(p, c0, a.d, vec, o[0] * a.scale, o[1] * a.scale);
        store_pair(p, c0 + 2, a.d, vec, o[2] * a.scale, o[3] * a.scale);
      }
    }
  }
  cp_commit();
  cp_wait<0>();
  // the plane: as k_dbias writes it
  for (int q = 0; q < G; ++q) {
    const int64_t j = (int64_t)(q0 + q) * 16 + 4 * t;
    uint32_t tm[8];
    __syncwarp();
    tmem_ld8(tm0 + q * 8, tm);
    tmem_wait8(tm);
    if ((int64_t)(q0 + q) * 16 >= a.nk) continue;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const int64_t i = w0 + r * 8 + g;
      if (i >= a.nq) continue;
      const float v0 = __uint_as_float(tm[2 * r]), v1 = __uint_as_float(tm[2 * r + 1]),
                  v2 = __uint_as_float(tm[4 + 2 * r]), v3 = __uint_as_float(tm[5 + 2 * r]);
      const bool whole = (int64_t)(q0 + q) * 16 + 16 <= a.nk;
      if (parts == 1)
        store_bias4<BT>(a, (char*)a.dbias + ((int64_t)h * a.db_hs + i * a.db_rs) * (BT == 2 ? 4 : 2), j,
                        a.db_vec && whole, v0, v1, v2, v3);
      else
        store_bias4<2>(a, (char*)(part + (((int64_t)pt * a.H + h) * a.nq + i) * a.nk), j, (a.nk & 3) == 0 && whole,
                       v0, v1, v2, v3);
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::tc_fence_after();
  if (warp == 0) sm100::tmem_dealloc(tbase, tcols);
}

// ---------------------------------------------------------------- launches

template <int DP, int BT>
int launch_t(Kind kind, Args a, double flops, cudaStream_t st) {
  constexpr size_t RB = Tile<DP>::RB;
  const int64_t tq = (a.nq + 63) / 64, tk = (a.nk + 63) / 64;
  if (kind == kFwd) {
    // two row blocks per warp where the accumulators leave room for them and there are blocks enough (768 rows
    // of 768 tokens: 1.5 against 1.7 ms)
    if constexpr (DP == 32) {
      const int64_t t2 = (a.nq + 127) / 128;
      if (t2 * a.H * a.B >= 3 * 148) {
        a.tiles = t2;
        constexpr size_t smem = (128 + 4 * kTile) * RB;
        return go<k_fwd<DP, BT, 2>>(smem, smem, t2 * a.H * a.B, 1, "k_attn_fwd", flops, st, a);
      }
    }
    a.tiles = tq;
    constexpr size_t smem = (64 + 4 * kTile) * RB;
    return go<k_fwd<DP, BT, 1>>(smem, smem, tq * a.H * a.B, 1, "k_attn_fwd", flops, st, a);
  }
  const int64_t bq = kind == kDkv ? 0 : tq * a.H * a.B, bkv = kind == kDq ? 0 : tk * a.KV * a.B;
  constexpr size_t smem = (128 + 4 * kTile) * RB + 2048;
  const char* name = kind == kDq ? "k_attn_dq" : (kind == kDkv ? "k_attn_dkv" : "k_attn_dqkv");
  const int ranks = bkv == 0 ? 1 : dkv_ranks(a, bkv, tq * a.H * a.B);
  const int64_t bk = bkv * ranks, blocks = (bk + bq + ranks - 1) / ranks * ranks;
  return go<k_dqkv<DP, BT>>(smem, smem, blocks, ranks, name, flops, st, a, (unsigned)bk, ranks);
}

template <int DP, int BT>
int launch_db(Args a, float* part, int parts, double flops, cudaStream_t st) {
  constexpr size_t smem = 2 * ((size_t)(256 + 128) * Tile<DP>::RB + 2048);
  a.tiles = (a.nq + 127) / 128;
  return go<k_dbias<DP, BT>>(smem, smem, a.tiles * ((a.nk + 63) / 64) * a.H * parts, 1, "k_attn_dbias", flops, st, a,
                             part, parts);
}

template <int BT>
int launch_plane(Args a, float* part, int parts, double flops, cudaStream_t st) {
  const int nkp = (int)((a.nk + 31) / 32) * 32;  // whole pairs of groups
  const int G = ((nkp / 16 + 3) / 4 + 1) / 2 * 2;  // groups of a quarter, an even number
  int tcols = 32;
  while (tcols < 4 * G * 8) tcols *= 2;
  a.tiles = (a.nq + 63) / 64;
  const int64_t blocks = a.tiles * a.H * parts;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: %lld tiles are too many", (long long)blocks);
  const int smem = PlaneSmem(nkp).end;
  PF_TRY(room_for_shared<k_dq_plane<BT>>(PlaneSmem(kPlaneKeys).end));
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_dq_plane", flops, 'f');
    k_dq_plane<BT><<<(unsigned)blocks, kPlaneThreads, smem, st>>>(a, part, parts, G, tcols);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

}  // namespace

#define PF_ATT_DIM(FN, BT, ...)                    \
  do {                                             \
    if (a.d <= 32) return FN<32, BT>(__VA_ARGS__); \
    if (a.d <= 64) return FN<64, BT>(__VA_ARGS__); \
    if (a.d <= 96) return FN<96, BT>(__VA_ARGS__); \
    return FN<128, BT>(__VA_ARGS__);               \
  } while (0)

int launch_bf16(Kind kind, const Args& a, double flops, cudaStream_t st) {
  if (!a.bias) PF_ATT_DIM(launch_t, 0, kind, a, flops, st);
  if (a.bias_f32) PF_ATT_DIM(launch_t, 2, kind, a, flops, st);
  PF_ATT_DIM(launch_t, 1, kind, a, flops, st);
}

int dbias_bf16(const Args& a, float* part, int parts, double flops, cudaStream_t st) {
  if (a.bias_f32) PF_ATT_DIM(launch_db, 2, a, part, parts, flops, st);
  PF_ATT_DIM(launch_db, 1, a, part, parts, flops, st);
}

bool dq_plane_bf16_fits(int64_t nk, int d) { return d <= 32 && nk <= kPlaneKeys; }
int dq_plane_bf16(const Args& a, float* part, int parts, double flops, cudaStream_t st) {
  return a.bias_f32 ? launch_plane<2>(a, part, parts, flops, st) : launch_plane<1>(a, part, parts, flops, st);
}

int rows_bf16(const Args& a, const float* stats, Heads o, const int16_t* lo, float* rows, cudaStream_t st) {
  const int lanes = a.d <= 32 ? 4 : (a.d <= 64 ? 8 : 16);
  const int64_t blocks = (a.rows_plane * lanes + 255) / 256;
  if (blocks > 0x7fffffffll) return fail(PF_EUNSUPPORTED, "attention: too many rows");
  const bool vec = a.vec_g && ((uintptr_t)o.p | (uintptr_t)lo) % 16 == 0 && ((o.bs | o.ns | o.hs) & 7) == 0;
  {
    PF_LAUNCH_SCOPE_WORK(st, "k_attn_rows", (6.0 * a.d + 24.0) * (double)a.rows_plane, 'b');
    auto* kern = lanes == 4   ? (vec ? k_rows<4, true> : k_rows<4, false>)
                 : lanes == 8 ? (vec ? k_rows<8, true> : k_rows<8, false>)
                              : (vec ? k_rows<16, true> : k_rows<16, false>);
    kern<<<(unsigned)blocks, 256, 0, st>>>(a, stats, o, lo, (float4*)rows);
  }
  PF_CHECK_LAUNCH();
  return PF_OK;
}

}  // namespace attn
}  // namespace train
}  // namespace pf
