// Single-query decode attention over a 4-bit cache (vt_int4.cuh), on the persistent schedule of vt_attn_flat.cu:
// flat tile list, cost-balanced shares, published piece states, merge by the last ticket holder.
//
// Mathematics.  With u = nibble in 0 .. 15, s = e4m3 group scale, S = head scale (both products of the stored row):
//   logit[t, h] = scale S_k sum_G s_k[t, G] ( sum_{d in G} u_k[t, d] q[h, d]  -  8 sum_{d in G} q[h, d] )
//   O[h, d in G] = S_v ( sum_t p[t, h] s_v[t, G] u_v[t, d]  -  8 sum_t p[t, h] s_v[t, G] )
// so the nibbles enter the matrix products as they are and every scale is applied to a number per (token, group), not
// per element: the K scale to the four partial logits, the V scale to the probabilities.  The two "- 8" terms are the
// start value of the logit accumulators and one extra product row per group.
//
// Nibble -> f16 without a conversion: a nibble in bits 0-3 of a half is the subnormal u 2^-24, in bits 4-7 u 2^-20,
// both exact operands.  One AND per pair of nibbles makes a fragment register; the factor 16 between the two
// positions is taken out of Q (K side) or of the finished output rows (V side).  Per 8 nibbles: 1 PRMT, 1 shift, 4 AND.
//   K fragment: lane (r4, c4) owns bytes [16 c4, +16) of its two token rows, i.e. of every group dims 8 c4 .. 8 c4 + 7;
//     half-register pairs (dim 8 c4 + j, 8 c4 + 4 + j) are MMA k indices (2 c4, 2 c4 + 1), j = 2 a in step a's lower
//     half, 2 a + 1 in its upper half.
//   V fragment: lane r4 owns bytes [8 r4, +8) of its four token rows, four dims of every group; accumulator tile
//     2 G + a holds dims 32 G + 4 r4 + 2 a (fragment row r4) and + 1 (row r4 + 8).
// Tokens are permuted among a warp's 16 fragment rows so that both load patterns are free of bank conflicts at the
// row pitch of the cache (544, 272, 144 or 80 bytes): the tile is copied as it lies in memory.
//
// P carries the V scale in f16 (11 bits), times 64 so that small probabilities stay normal; the sums are fp32.
// Roofline: HBM.  Bytes per (token, kv head): 2 x 68 (72 / 80 with 2 / 1 heads in a unit).
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_int4.cuh"
#include "vt_kernels.h"
#include "vt_mma.cuh"
#include "vt_mma_f8.cuh"
#include "vt_attn_flat_sched.cuh"

namespace vt {
namespace {

constexpr int kCWarps = 8;                 // consumer warps = heads of a unit x token sub-rows of a tile
constexpr int kThreads4 = kCWarps * 32;
constexpr int kRingBudget = 106000;        // two CTAs per SM with their tables
constexpr int kBaseCacheMaxBatch4 = 256;
constexpr float kPScaleLog2 = 6.f;         // P is carried times 2^6

template <int U>
struct Cfg4 {
  static constexpr int R = kCWarps / U;                 // warps that share a head, each on its own 16 tokens
  static constexpr int UB = int4_unit_bytes(U);
  static constexpr int SUBS = U >= 4 ? 2 : 1;           // 16-token steps per warp and tile
  static constexpr int TOK = 16 * R * SUBS;             // tokens per tile
  static constexpr int kTile = TOK * UB;                // K tile, then V tile
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = kRingBudget / kStage;
  static_assert(kStages >= 3, "ring too shallow");
};

// 2^x to about 2 ulp; 0 for -inf.  (Below 2^-126 it flushes to 0, far under what a probability contributes.)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// fragment row -> token of the warp's 16 (see the header: conflict-free at the pitch of U heads)
template <int U>
__device__ __forceinline__ int token_of_row(int row) {
  const int i = row & 7;
  if (U == 8)    // pitch 136 words = 8 mod 32
    return static_cast<int>((0x53427160u >> (4 * i)) & 15u) + (row & 8);
  return static_cast<int>((0xA684E2C0u >> (4 * i)) & 15u) + (row >> 3);   // pitches 68, 36, 20 words = 4 mod 16 (odd x 4)
}

// D = A B, accumulator starting at zero
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

template <int NB>
struct WarpAttn4 {
  uint32_t qb[NB][4][2][2];   // [group][step][k half]
  float qoff[NB][4][2];       // -8 sum q over the group, per column
  float qmul[NB][2];          // partial logits -> log2 domain
  float o[NB][8][4];
  float corr[NB][4];          // row G: 8 sum p s_v[G]
  float mrun[NB][2], lrun[NB][2];

  __device__ __forceinline__ static int dim_of(int mb, int half, int r4) {
    return 32 * (mb >> 1) + 4 * r4 + 2 * (mb & 1) + half;
  }

  __device__ __forceinline__ void start(const __nv_bfloat16 *qrow, int g, float sl2, int lane) {
    const int r4 = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int head = nb * 8 + r4;
      float q[4][8], amax = 0.f;
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (head < g) w = __ldg(reinterpret_cast<const uint4 *>(qrow + head * kHeadDim + 32 * G + 8 * c4));
        Unpack<false>::run(w, q[G]);
#pragma unroll
        for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(q[G][e]));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      // A power of two brings the head's largest element into [2^14, 2^15): bf16 values are then exact in f16 down
      // to 2^-25 of it, also after the division by 16 of the upper nibble positions.
      const int ex = static_cast<int>((__float_as_uint(amax) >> 23) & 255u);
      const float f = (ex == 0 || ex == 255) ? 1.f : __uint_as_float(static_cast<uint32_t>(min(268 - ex, 254)) << 23);
      float sum[4];
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        sum[G] = 0.f;
#pragma unroll
        for (int a = 0; a < 2; ++a) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int j = 2 * a + k;
            const float m = k ? f * 0.0625f : f;
            const uint32_t w = pack_f16(q[G][j] * m, q[G][4 + j] * m);
            qb[nb][G][a][k] = w;
            sum[G] += (f16_lo(w) + f16_hi(w)) * (k ? 16.f : 1.f);
          }
        }
        sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], 1);
        sum[G] += __shfl_xor_sync(0xffffffffu, sum[G], 2);
      }
      const float mul = sl2 * (16777216.f / f);   // 2^24 of the nibbles, 1 / f of Q
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int src = (2 * c4 + e) * 4;
#pragma unroll
        for (int G = 0; G < 4; ++G) qoff[nb][G][e] = __shfl_sync(0xffffffffu, sum[G], src) * -4.76837158203125e-7f;   // -8 2^-24
        qmul[nb][e] = __shfl_sync(0xffffffffu, mul, src);
        mrun[nb][e] = -INFINITY;
        lrun[nb][e] = 0.f;
      }
#pragma unroll
      for (int mb = 0; mb < 8; ++mb) o[nb][mb][0] = o[nb][mb][1] = o[nb][mb][2] = o[nb][mb][3] = 0.f;
      corr[nb][0] = corr[nb][1] = corr[nb][2] = corr[nb][3] = 0.f;
    }
  }

  // Partial logits of 16 tokens per group of dims, joined with the group scales: s[nb][token ta: heads 2 c4, + 1; tb: ..].
  template <int U>
  __device__ __forceinline__ void logits(float (&s)[NB][4], const unsigned char *kt, int sc, int ta, int tb, int c4) const {
    constexpr int UB = Cfg4<U>::UB;
    float acc[NB][4][4];
    const uint4 ka = *reinterpret_cast<const uint4 *>(kt + ta * UB + 16 * c4);
    const uint4 kb = *reinterpret_cast<const uint4 *>(kt + tb * UB + 16 * c4);
    const uint32_t wsa = *reinterpret_cast<const uint32_t *>(kt + ta * UB + sc);
    const uint32_t wsb = *reinterpret_cast<const uint32_t *>(kt + tb * UB + sc);
#pragma unroll
    for (int G = 0; G < 4; ++G) {
      const uint32_t sel = (G & 1) ? 0x7632u : 0x5410u;
      uint32_t xa = G < 2 ? prmt(ka.x, ka.z, sel) : prmt(ka.y, ka.w, sel);
      uint32_t xb = G < 2 ? prmt(kb.x, kb.z, sel) : prmt(kb.y, kb.w, sel);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t f[4] = {xa & 0x000f000fu, xb & 0x000f000fu, xa & 0x00f000f0u, xb & 0x00f000f0u};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          if (a == 0) mma_f16_zero(acc[nb][G], f, qb[nb][G][0][0], qb[nb][G][0][1]);
          else mma_f16(acc[nb][G], f, qb[nb][G][1][0], qb[nb][G][1][1]);
        }
        xa >>= 8;
        xb >>= 8;
      }
    }
    const uint32_t a01 = e4m3x2_to_f16x2(wsa), a23 = e4m3x2_to_f16x2(wsa >> 16);
    const uint32_t b01 = e4m3x2_to_f16x2(wsb), b23 = e4m3x2_to_f16x2(wsb >> 16);
    const float ga[4] = {f16_lo(a01), f16_hi(a01), f16_lo(a23), f16_hi(a23)};
    const float gb[4] = {f16_lo(b01), f16_hi(b01), f16_lo(b23), f16_hi(b23)};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // the "- 8" of a group is added to its sum here, on the FMA pipe: as the start value of the accumulators it
      // costs a move per register on the ALU pipe, which is the busy one
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        const float x0 = acc[nb][G][0] + qoff[nb][G][0], x1 = acc[nb][G][1] + qoff[nb][G][1];
        const float x2 = acc[nb][G][2] + qoff[nb][G][0], x3 = acc[nb][G][3] + qoff[nb][G][1];
        s[nb][0] = G ? fmaf(ga[G], x0, s[nb][0]) : ga[G] * x0;
        s[nb][1] = G ? fmaf(ga[G], x1, s[nb][1]) : ga[G] * x1;
        s[nb][2] = G ? fmaf(gb[G], x2, s[nb][2]) : gb[G] * x2;
        s[nb][3] = G ? fmaf(gb[G], x3, s[nb][3]) : gb[G] * x3;
      }
    }
  }

  // O^T += V^T . (s_v P)^T over 16 tokens; pb = P^T as a B operand.
  template <int U>
  __device__ __forceinline__ void values(const uint32_t (&pb)[NB][2], const unsigned char *vt, int sc, int n_tok, int r4, int c4) {
    constexpr int UB = Cfg4<U>::UB;
    const int t0 = token_of_row<U>(2 * c4), t1 = token_of_row<U>(2 * c4 + 1);
    const int t2 = token_of_row<U>(2 * c4 + 8), t3 = token_of_row<U>(2 * c4 + 9);
    const uint2 v0 = *reinterpret_cast<const uint2 *>(vt + t0 * UB + 8 * r4);
    const uint2 v1 = *reinterpret_cast<const uint2 *>(vt + t1 * UB + 8 * r4);
    const uint2 v2 = *reinterpret_cast<const uint2 *>(vt + t2 * UB + 8 * r4);
    const uint2 v3 = *reinterpret_cast<const uint2 *>(vt + t3 * UB + 8 * r4);
    uint32_t w0 = *reinterpret_cast<const uint32_t *>(vt + t0 * UB + sc);
    uint32_t w1 = *reinterpret_cast<const uint32_t *>(vt + t1 * UB + sc);
    uint32_t w2 = *reinterpret_cast<const uint32_t *>(vt + t2 * UB + sc);
    uint32_t w3 = *reinterpret_cast<const uint32_t *>(vt + t3 * UB + sc);
    if (n_tok < 16) {   // what lies past the context is stale and may be NaN as a scale; its P is 0
      w0 = t0 < n_tok ? w0 : 0u;
      w1 = t1 < n_tok ? w1 : 0u;
      w2 = t2 < n_tok ? w2 : 0u;
      w3 = t3 < n_tok ? w3 : 0u;
    }
    // per pair of tokens the scale bytes of groups (0, 1) and (2, 3), interleaved
    const uint32_t y01[2] = {prmt(w0, w1, 0x5140u), prmt(w0, w1, 0x7362u)};
    const uint32_t y23[2] = {prmt(w2, w3, 0x5140u), prmt(w2, w3, 0x7362u)};
#pragma unroll
    for (int G = 0; G < 4; ++G) {
      const uint32_t s01 = e4m3x2_to_f16x2((G & 1) ? y01[G >> 1] >> 16 : y01[G >> 1]);
      const uint32_t s23 = e4m3x2_to_f16x2((G & 1) ? y23[G >> 1] >> 16 : y23[G >> 1]);
      uint32_t b0[NB], b1[NB];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&pb[nb][0]), *reinterpret_cast<const __half2 *>(&s01));
        const __half2 y = __hmul2(*reinterpret_cast<const __half2 *>(&pb[nb][1]), *reinterpret_cast<const __half2 *>(&s23));
        b0[nb] = *reinterpret_cast<const uint32_t *>(&x);
        b1[nb] = *reinterpret_cast<const uint32_t *>(&y);
      }
      const uint32_t eight = r4 == G ? 0x00080008u : 0u;   // 8 x 2^-24 in fragment row G
      const uint32_t fc[4] = {eight, 0u, eight, 0u};
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) mma_f16(corr[nb], fc, b0[nb], b1[nb]);
      const uint32_t psel = (G & 1) ? 0x7632u : 0x5410u;
      uint32_t x01 = G < 2 ? prmt(v0.x, v1.x, psel) : prmt(v0.y, v1.y, psel);
      uint32_t x23 = G < 2 ? prmt(v2.x, v3.x, psel) : prmt(v2.y, v3.y, psel);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t f[4] = {x01 & 0x000f000fu, x01 & 0x00f000f0u, x23 & 0x000f000fu, x23 & 0x00f000f0u};
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_f16(o[nb][2 * G + a], f, b0[nb], b1[nb]);
        x01 >>= 8;
        x23 >>= 8;
      }
    }
  }

  // One tile of this warp: SUBS x 16 tokens, `stride` tokens apart.  kt / vt = the head's K / V bytes of the first
  // token, sc = offset of the scale words from there, n_tok > 0 = tokens from that one to the end of the context.
  template <int U, bool LOG>
  __device__ __forceinline__ void tile(const unsigned char *kt, const unsigned char *vt, int sc, int n_tok, int lane, float *lg,
                                       int g) {
    constexpr int SUBS = Cfg4<U>::SUBS, STEP = 16 * Cfg4<U>::R, UB = Cfg4<U>::UB;
    const int r4 = lane >> 2, c4 = lane & 3;
    const int ta = token_of_row<U>(r4), tb = token_of_row<U>(r4 + 8);
    float s[SUBS][NB][4];
#pragma unroll
    for (int i = 0; i < SUBS; ++i) logits<U>(s[i], kt + i * STEP * UB, sc, ta, tb, c4);
    // ---- online softmax (rows = tokens ta, tb; columns = heads 2 c4, 2 c4 + 1) ----
    uint32_t pb[SUBS][NB][2];
    float fac[NB][2];
    bool any_up = false;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int i = 0; i < SUBS; ++i) {
        float(&x)[4] = s[i][nb];
        x[0] *= qmul[nb][0];
        x[1] *= qmul[nb][1];
        x[2] *= qmul[nb][0];
        x[3] *= qmul[nb][1];
        const bool va = ta + i * STEP < n_tok, vb = tb + i * STEP < n_tok;
        if (n_tok < (SUBS - 1) * STEP + 16) {   // the context ends in this tile
          x[0] = va ? x[0] : -INFINITY;
          x[1] = va ? x[1] : -INFINITY;
          x[2] = vb ? x[2] : -INFINITY;
          x[3] = vb ? x[3] : -INFINITY;
        }
        if constexpr (LOG) {
          const int head = nb * 8 + 2 * c4;
          float *pa = lg + (ta + i * STEP) * g + head, *pt = lg + (tb + i * STEP) * g + head;
          if (head + 1 < g) {   // head is even, and so is g here: 8-byte aligned
            if (va) *reinterpret_cast<float2 *>(pa) = make_float2(x[0], x[1]);
            if (vb) *reinterpret_cast<float2 *>(pt) = make_float2(x[2], x[3]);
          } else if (head < g) {
            if (va) *pa = x[0];
            if (vb) *pt = x[2];
          }
        }
        mx0 = fmaxf(mx0, fmaxf(x[0], x[2]));
        mx1 = fmaxf(mx1, fmaxf(x[1], x[3]));
      }
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
      }
      // the running "maximum" sits 6 below the true one, which carries P times 2^6 through sums, states and merges
      const float mn0 = fmaxf(mrun[nb][0], mx0 - kPScaleLog2), mn1 = fmaxf(mrun[nb][1], mx1 - kPScaleLog2);
      fac[nb][0] = ex2(mrun[nb][0] - mn0);   // the first token is valid, so mn is finite
      fac[nb][1] = ex2(mrun[nb][1] - mn1);
      any_up |= (mn0 > mrun[nb][0]) | (mn1 > mrun[nb][1]);
      mrun[nb][0] = mn0;
      mrun[nb][1] = mn1;
      lrun[nb][0] *= fac[nb][0];
      lrun[nb][1] *= fac[nb][1];
#pragma unroll
      for (int i = 0; i < SUBS; ++i) {
        const float(&x)[4] = s[i][nb];
        const float p00 = ex2(x[0] - mn0), p01 = ex2(x[1] - mn1), p10 = ex2(x[2] - mn0), p11 = ex2(x[3] - mn1);
        lrun[nb][0] += p00 + p10;
        lrun[nb][1] += p01 + p11;
        pb[i][nb][0] = movmatrix_trans(pack_f16(p00, p01));
        pb[i][nb][1] = movmatrix_trans(pack_f16(p10, p11));
      }
    }
    if (__any_sync(0xffffffffu, any_up)) {
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int mb = 0; mb < 8; ++mb) {
          o[nb][mb][0] *= fac[nb][0]; o[nb][mb][1] *= fac[nb][1];
          o[nb][mb][2] *= fac[nb][0]; o[nb][mb][3] *= fac[nb][1];
        }
        corr[nb][0] *= fac[nb][0]; corr[nb][1] *= fac[nb][1];
      }
    }
#pragma unroll
    for (int i = 0; i < SUBS; ++i) values<U>(pb[i], vt + i * STEP * UB, sc, n_tok - i * STEP, r4, c4);
  }

  // Row sums over the lanes, the "- 8" correction and the powers of two: afterwards o and lrun are what the
  // other engines publish (the head scale of V is applied by the merge).
  __device__ __forceinline__ void finish(int lane) {
    const int c4 = lane & 3;
    constexpr float kLo = 16777216.f;   // 2^24 of the nibbles; row r4 + 8 holds upper nibbles: a sixteenth
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        lrun[nb][0] += __shfl_xor_sync(0xffffffffu, lrun[nb][0], off);
        lrun[nb][1] += __shfl_xor_sync(0xffffffffu, lrun[nb][1], off);
      }
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        const float c0 = __shfl_sync(0xffffffffu, corr[nb][0], 4 * G + c4);
        const float c1 = __shfl_sync(0xffffffffu, corr[nb][1], 4 * G + c4);
#pragma unroll
        for (int a = 0; a < 2; ++a) {
          float(&x)[4] = o[nb][2 * G + a];
          x[0] = (x[0] - c0) * kLo;
          x[1] = (x[1] - c1) * kLo;
          x[2] = (x[2] * 0.0625f - c0) * kLo;
          x[3] = (x[3] * 0.0625f - c1) * kLo;
        }
      }
    }
  }

  template <int ROW>
  __device__ __forceinline__ void store(float *dst, int lane, int g) const {
    const int r4 = lane >> 2, c4 = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int head = nb * 8 + 2 * c4 + e;
        if (head >= g) continue;
#pragma unroll
        for (int mb = 0; mb < 8; ++mb) {
          dst[head * ROW + dim_of(mb, 0, r4)] = o[nb][mb][e];
          dst[head * ROW + dim_of(mb, 1, r4)] = o[nb][mb][2 + e];
        }
        if (r4 == 0) {
          dst[head * ROW + 128] = mrun[nb][e];
          dst[head * ROW + 129] = lrun[nb][e];
        }
      }
    }
  }
};

// Where a warp's copies stand: the tile to fetch next.  In shared memory: it is needed once per tile, registers always.
struct Cursor {
  const char *k, *v;         // the unit's rows of the piece's sequence
  long long tau;             // position of the piece after this one
  int tile, tile_end, seq_len, pad;
};

// ring | barriers | cursors | flags | prefix[batch + 1] | lens[batch] | (pad to 8) | kbase[batch] | vbase[batch]
__host__ __device__ constexpr int meta_ints4(int batch) { return ((2 * batch + 1 + 4) + 1) / 2 * 2; }
template <int U>
constexpr int smem_bytes4(int batch) {
  return Cfg4<U>::kStages * (Cfg4<U>::kStage + 16) + kCWarps * static_cast<int>(sizeof(Cursor)) + meta_ints4(batch) * 4 + (batch <= kBaseCacheMaxBatch4 ? batch * 16 : 0);
}

template <int U, int NB, bool LOG>
__global__ void __launch_bounds__(kThreads4, NB == 1 ? 2 : 1) attn_int4_kernel(AttnParams p) {
  using C = Cfg4<U>;
  constexpr int R = C::R, UB = C::UB, TOK = C::TOK, HEADS = NB * 8;
  extern __shared__ __align__(128) unsigned char smem[];
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kStages * C::kStage);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Cursor &cur = reinterpret_cast<Cursor *>(bars + 2 * C::kStages)[warp];
  int *flags = reinterpret_cast<int *>(reinterpret_cast<Cursor *>(bars + 2 * C::kStages) + kCWarps);
  int *prefix = flags + 4;
  int *lens = prefix + p.batch + 1;
  const bool cache_bases = p.batch <= kBaseCacheMaxBatch4;
  unsigned long long *kbase_s = reinterpret_cast<unsigned long long *>(flags + meta_ints4(p.batch));
  unsigned long long *vbase_s = kbase_s + p.batch;
  const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + C::kStages), ring0 = smem_u32(smem);

  const int g = p.h / p.kvh, slabs = p.kvh / U;
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full0 + 8 * s, kCWarps);
      mbar_init(empty0 + 8 * s, kCWarps);
    }
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < p.batch; i += kThreads4) {
    int len = max(p.seq_lens[i], 0);
    if constexpr (LOG) len = min(len, p.logit_rows);   // the logits have room for no more
    lens[i] = len;
    prefix[i + 1] = len > 0 ? ((len + TOK - 1) / TOK + kBoundaryCost) * slabs : 0;
    if (cache_bases) {
      const int64_t slot = p.slot_ids[i];
      kbase_s[i] = p.k_table[slot];
      vbase_s[i] = p.v_table[slot];
    }
  }
  __syncthreads();
  if (warp == 0) {
    int carry = 0;
    for (int base = 0; base < p.batch; base += 32) {
      const int i = base + lane;
      int v = i < p.batch ? prefix[i + 1] : 0;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, v, off);
        if (lane >= off) v += n;
      }
      if (i < p.batch) prefix[i + 1] = carry + v;
      carry += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) prefix[0] = 0;
  }
  __syncthreads();
  pdl_launch_dependents();
  const long long total = prefix[p.batch];
  const int n_ctas = static_cast<int>(min(static_cast<long long>(gridDim.x), total));
  const bool active = static_cast<int>(blockIdx.x) < n_ctas;
  const long long tau0 = active ? total * blockIdx.x / n_ctas : 0;
  const long long tau1 = active ? total * (blockIdx.x + 1) / n_ctas : 0;
  const int64_t row_bytes = static_cast<int64_t>(slabs) * UB;

  // ---------------- copies ----------------
  // Every warp fetches an eighth of the rows of the CTA's next tile into its ring stage, `n` tiles into the share, once
  // all warps are done with what the stage held; false when a bounded wait ran out.  A single-unit cache is contiguous
  // over tokens: one copy of K and one of V.  Otherwise a row of the unit (80 to 544 bytes) is one copy, a lane each.
  const uint64_t policy = l2_policy_evict_first();
  const auto fetch = [&](int n) -> bool {
    if (cur.tile >= cur.tile_end) {
      long long tau = cur.tau;
      Piece pc{};
      while (tau < tau1) {
        pc = locate(prefix, p.batch, slabs, tau, tau1);
        tau += pc.advance;
        if (pc.tile_end > pc.tile_begin) break;
      }
      __syncwarp();
      if (lane == 0) {
        cur.tau = tau;
        cur.tile = pc.tile_begin;
        cur.tile_end = pc.tile_end;
        if (pc.tile_end > pc.tile_begin) {
          const int64_t slot = p.slot_ids[pc.b];
          cur.k = reinterpret_cast<const char *>(cache_bases ? kbase_s[pc.b] : p.k_table[slot]) + pc.slab * UB;
          cur.v = reinterpret_cast<const char *>(cache_bases ? vbase_s[pc.b] : p.v_table[slot]) + pc.slab * UB;
          cur.seq_len = lens[pc.b];
        }
      }
      __syncwarp();
      if (cur.tile >= cur.tile_end) return true;   // the share is fetched
    }
    constexpr int ROWS = TOK / kCWarps;
    const int tile = cur.tile, s = n % C::kStages;
    const int t0 = tile * TOK + warp * ROWS, nt = min(max(cur.seq_len - t0, 0), ROWS);
    const int64_t src = t0 * row_bytes;
    const char *kb = cur.k + src, *vb = cur.v + src;
    if (n >= C::kStages && !mbar_wait(empty0 + 8 * s, ((n / C::kStages) - 1) & 1)) {
      if (lane == 0) atomicExch(p.status, kKernelErrMagic);
      return false;
    }
    const uint32_t dst = ring0 + s * C::kStage + warp * ROWS * UB;
    __syncwarp();
    if (lane == 0) {
      cur.tile = tile + 1;
      mbar_arrive_expect_tx(full0 + 8 * s, 2u * nt * UB);
    }
    __syncwarp();
    if (slabs == 1) {
      if (lane < 2 && nt > 0) bulk_g2s_hint(dst + lane * C::kTile, lane ? vb : kb, nt * UB, full0 + 8 * s, policy);
    } else {
      const int row = lane & 15;
      static_assert(ROWS <= 16, "a lane per row of K and of V");
      if (row < nt)
        bulk_g2s_hint(dst + (lane >> 4) * C::kTile + row * UB, (lane >> 4 ? vb : kb) + row * row_bytes, UB, full0 + 8 * s, policy);
    }
    return true;
  };
  bool failed = false;
  if (lane == 0) {
    cur.tau = tau0;
    cur.tile = cur.tile_end = 0;
  }
  __syncwarp();
  for (int n = 0; n < C::kStages - 1; ++n) failed |= !fetch(n);

  // ---------------- consumer warps ----------------
  const int hs = warp % U, rr = warp / U;
  const float sl2_base = p.scale * 1.4426950408889634f;
  const int tid = threadIdx.x;
  __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(p.out);
  if (blockIdx.x == 0) {   // sequences without context produce zeros; nobody owns a tile of theirs
    for (int b = 0; b < p.batch; ++b)
      if (prefix[b + 1] == prefix[b]) {
        for (int i = tid; i < p.h * kHeadDim; i += kCWarps * 32) out[b * p.out_stride + i] = __float2bfloat16(0.f);
        if (p.lse)
          for (int i = tid; i < p.h; i += kCWarps * 32) p.lse[b * p.h + i] = -INFINITY;
      }
  }
  int it = 0;
  bool first_piece = true;
  for (long long tau = tau0; tau < tau1;) {
    const Piece pc = locate(prefix, p.batch, slabs, tau, tau1);
    if (pc.tile_end <= pc.tile_begin) {
      tau += pc.advance;
      continue;
    }
    const int seq_len = lens[pc.b];
    const int kv_head = pc.slab * U + hs;
    const int64_t append_off = p.new_key ? p.byte_off[pc.b] : -1;
    if (p.overlap == 2) pdl_wait_prior_grid();
    WarpAttn4<NB> st;
    st.start(static_cast<const __nv_bfloat16 *>(p.q) + pc.b * p.q_stride + kv_head * g * kHeadDim, g,
             sl2_base * p.k_scale[kv_head], lane);
    float *lg = nullptr;
    if constexpr (LOG) lg = p.logits + (static_cast<size_t>(pc.b) * p.kvh + kv_head) * p.logit_rows * g;
    for (int tile = pc.tile_begin; tile < pc.tile_end; ++tile, ++it) {
      const int s = it % C::kStages;
      // the stage of the tile before this one, which the other warps are likely done with
      if (!failed && !fetch(it + C::kStages - 1)) failed = true;
      if (!failed && !mbar_wait(full0 + 8 * s, (it / C::kStages) & 1)) failed = true;
      if (failed) continue;
      unsigned char *kt = smem + s * C::kStage + hs * 64, *vt = kt + C::kTile;
      const int sc = U * 64 + hs * 4 - hs * 64;
      const int t0 = tile * TOK;
      const int fresh = seq_len - 1 - t0;   // position of the newest token in the tile
      bool wrote = false;
      if (append_off >= 0 && fresh < TOK && (fresh / 16) % R == rr) {
        // Fused step: this warp owns the newest token's row of its kv head.  The copy brought whatever the range
        // held; quantise the step's row over it, in the stage and in the range.
        char *kd, *vd;
        if (cache_bases) {
          kd = reinterpret_cast<char *>(kbase_s[pc.b]);
          vd = reinterpret_cast<char *>(vbase_s[pc.b]);
        } else {
          const int64_t slot = p.slot_ids[pc.b];
          kd = reinterpret_cast<char *>(p.k_table[slot]);
          vd = reinterpret_cast<char *>(p.v_table[slot]);
        }
        const int64_t dst = append_off + pc.slab * UB + hs * 64;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(kv ? p.new_value : p.new_key) +
                                     pc.b * (kv ? p.new_value_stride : p.new_key_stride) + kv_head * kHeadDim + lane * 4;
          const uint2 w = __ldg(reinterpret_cast<const uint2 *>(src));
          const float x[4] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
          uint32_t bits, s8;
          quantise4(x, (kv ? p.v_scale : p.k_scale)[kv_head], &bits, &s8);
          unsigned char *row = (kv ? vt : kt) + fresh * UB;
          char *far = (kv ? vd : kd) + dst;
          const int at = 8 * (lane & 7) + 2 * (lane >> 3);
          *reinterpret_cast<uint16_t *>(row + at) = static_cast<uint16_t>(bits);
          *reinterpret_cast<uint16_t *>(far + at) = static_cast<uint16_t>(bits);
          if ((lane & 7) == 0) {
            row[sc + (lane >> 3)] = static_cast<unsigned char>(s8);
            far[sc + (lane >> 3)] = static_cast<char>(s8);
          }
        }
        __syncwarp();
        wrote = true;
      }
      const int n_tok = seq_len - t0 - 16 * rr;
      if (n_tok > 0)
        st.template tile<U, LOG>(kt + 16 * rr * UB, vt + 16 * rr * UB, sc, n_tok, lane,
                                 LOG ? lg + static_cast<size_t>(t0 + 16 * rr) * g : nullptr, g);
      if (wrote) fence_proxy_async();   // before the copy engine refills the stage
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * s);
    }
    st.finish(lane);

    const bool whole = pc.tile_begin == 0 && pc.tile_end == pc.tiles_in_stream;
    if (R == 1 && whole) {
      const int r4 = lane >> 2, c4 = lane & 3;
      const float vs = p.v_scale[kv_head];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int head = nb * 8 + 2 * c4 + e;
          if (head < g) {
            const float inv = vs / st.lrun[nb][e];
            const int hq = kv_head * g + head;
            __nv_bfloat16 *dst = out + pc.b * p.out_stride + hq * kHeadDim;
#pragma unroll
            for (int mb = 0; mb < 8; ++mb)   // dims d, d + 1 are the two fragment rows
              *reinterpret_cast<uint32_t *>(dst + WarpAttn4<NB>::dim_of(mb, 0, r4)) =
                  pack_bf16(st.o[nb][mb][e] * inv, st.o[nb][mb][2 + e] * inv);
            if (r4 == 0) write_stats(p, pc.b * p.h + hq, st.mrun[nb][e], st.lrun[nb][e]);
          }
        }
      }
    } else {
      if (p.overlap) pdl_wait_prior_grid();
      float *slot_base = p.fl_part + (static_cast<size_t>(blockIdx.x) * 2 + (first_piece ? 0 : 1)) * kCWarps * HEADS * kPartRow;
      st.template store<kPartRow>(slot_base + warp * HEADS * kPartRow, lane, g);
      __threadfence();
      named_bar_sync(1, kCWarps * 32);
      const int c_first = owner_of(pc.stream_begin + kBoundaryCost, total, n_ctas);
      const int c_last = owner_of(pc.stream_end - 1, total, n_ctas);
      if (tid == 0) {
        unsigned *ctr = p.fl_count + pc.b * slabs + pc.slab;
        const unsigned old = atomicAdd(ctr, 1u);
        const int last = old + 1 == static_cast<unsigned>(c_last - c_first + 1);
        if (last) *ctr = 0u;
        flags[0] = last;
      }
      named_bar_sync(1, kCWarps * 32);
      const bool merger = flags[0] != 0;
      named_bar_sync(1, kCWarps * 32);
      if (merger) {
        merge_stream<kCWarps, U, R, HEADS, true, false>(p, pc, total, n_ctas, c_first, c_last, warp, lane, g);
        if (R > 1) named_bar_sync(1, kCWarps * 32);   // this CTA's next piece may publish to the slot just read
      }
    }
    first_piece = false;
    tau += pc.advance;
  }
  if (failed && lane == 0) atomicExch(p.status, kKernelErrMagic);
}

template <int U, int NB, bool LOG>
int launch4(const AttnParams &p_in, cudaStream_t stream) {
  AttnParams p = p_in;
  p.n_ctas = (NB == 1 ? 2 : 1) * kFlatSms;
  const int smem = smem_bytes4<U>(p.batch);
  static SmemOptIn opt_in;
  if (!opt_in.ensure(attn_int4_kernel<U, NB, LOG>, smem)) return VT_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.n_ctas);
  cfg.blockDim = dim3(kThreads4);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.overlap ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, attn_int4_kernel<U, NB, LOG>, p) == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

template <int U>
int launch_u(const AttnParams &p, cudaStream_t stream) {
  const bool nb1 = p.h / p.kvh <= 8;
  if (p.logits) return nb1 ? launch4<U, 1, true>(p, stream) : launch4<U, 2, true>(p, stream);
  return nb1 ? launch4<U, 1, false>(p, stream) : launch4<U, 2, false>(p, stream);
}

}  // namespace

int launch_attn_int4(const AttnParams &p, cudaStream_t stream) {
  switch (int4_unit(p.kvh)) {
    case 8: return launch_u<8>(p, stream);
    case 4: return launch_u<4>(p, stream);
    case 2: return launch_u<2>(p, stream);
    default: return launch_u<1>(p, stream);
  }
}

}  // namespace vt
