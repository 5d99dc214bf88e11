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
// Measured: 32 sequences of 16k-32k rows, 32/8 heads (869 MB): 205 us, 4.2 TB/s; without the copies it takes 195, the
// integer unit is 54 % busy: the unpacking bounds it.  64 sequences of 1k-4k rows, 32/32 heads (726 MB): 213 us; one q
// head per kv head leaves seven of the eight columns of every product empty.  One sequence of 700 rows, 32/8 heads: 20 us.
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_int4.cuh"
#include "vt_kernels.h"
#include "vt_mma.cuh"
#include "vt_mma_f8.cuh"
#include "vt_attn_flat_sched.cuh"
#include "vt_umma.cuh"

namespace vt {
namespace {

constexpr int kCWarps = 8;                 // consumer warps = heads of a unit x token sub-rows of a tile
constexpr int kThreads4 = kCWarps * 32;
constexpr int kRingBudget = 106000;        // two CTAs per SM with their tables
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
__host__ __device__ constexpr int token_of_row(int row) {
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
  float o[NB][8][4];
  float corr[NB][4];          // row G: 8 sum p s_v[G]
  float mrun[NB][2], lrun[NB][2];

  __device__ __forceinline__ static int dim_of(int mb, int half, int r4) {
    return 32 * (mb >> 1) + 4 * r4 + 2 * (mb & 1) + half;
  }

  // Per pair of q heads of the warp, in shared memory (ten registers the tile loop would spill): -8 sum q of every group,
  // and the factor from partial logits to the log2 domain.
  static constexpr int kQRow = 6;   // pairs of floats: 4 offsets, factor, pad
  static constexpr int kQFloats = NB * 4 * kQRow * 2;

  __device__ __forceinline__ void start(const __nv_bfloat16 *qrow, int g, float sl2, int lane, float *qs) {
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
      if (c4 == 0) {
        float *mine = qs + (head >> 1) * kQRow * 2 + (head & 1);
#pragma unroll
        for (int G = 0; G < 4; ++G) mine[2 * G] = sum[G] * -4.76837158203125e-7f;   // -8 2^-24
        mine[8] = sl2 * (16777216.f / f);   // 2^24 of the nibbles, 1 / f of Q
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        mrun[nb][e] = -INFINITY;
        lrun[nb][e] = 0.f;
      }
#pragma unroll
      for (int mb = 0; mb < 8; ++mb) o[nb][mb][0] = o[nb][mb][1] = o[nb][mb][2] = o[nb][mb][3] = 0.f;
      corr[nb][0] = corr[nb][1] = corr[nb][2] = corr[nb][3] = 0.f;
    }
    __syncwarp();
  }

  // Partial logits of 16 tokens per group of dims, joined with the group scales: s[nb][token ta: heads 2 c4, + 1; tb: ..].
  template <int U>
  __device__ __forceinline__ void logits(float (&s)[NB][4], const unsigned char *kt, int sc, const int4 &at, int c4, const float *qs) const {
    constexpr int DB = Cfg4<U>::UB * token_of_row<U>(8);   // from fragment row r4 to r4 + 8
    float acc[NB][4][4];
    const uint4 ka = *reinterpret_cast<const uint4 *>(kt + at.x);
    const uint4 kb = *reinterpret_cast<const uint4 *>(kt + at.x + DB);
    const uint32_t wsa = *reinterpret_cast<const uint32_t *>(kt + at.y + sc);
    const uint32_t wsb = *reinterpret_cast<const uint32_t *>(kt + at.y + DB + sc);
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
    // pairs (scale, scale) for the two heads of a column pair
    const uint64_t ga[4] = {f2_pack(f16_lo(a01), f16_lo(a01)), f2_pack(f16_hi(a01), f16_hi(a01)), f2_pack(f16_lo(a23), f16_lo(a23)),
                            f2_pack(f16_hi(a23), f16_hi(a23))};
    const uint64_t gb[4] = {f2_pack(f16_lo(b01), f16_lo(b01)), f2_pack(f16_hi(b01), f16_hi(b01)), f2_pack(f16_lo(b23), f16_lo(b23)),
                            f2_pack(f16_hi(b23), f16_hi(b23))};
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // The "- 8" of a group is added to its sum here, on the FMA pipe (two lanes an instruction): as the start value of
      // the accumulators it costs a move per register on the ALU pipe, which is the busy one.
      const uint64_t *qp = reinterpret_cast<const uint64_t *>(qs) + (nb * 4 + c4) * kQRow;
      uint64_t sa = 0, sb = 0;
#pragma unroll
      for (int G = 0; G < 4; ++G) {
        const uint64_t off = qp[G];
        const uint64_t xa = f2_add(f2_pack(acc[nb][G][0], acc[nb][G][1]), off), xb = f2_add(f2_pack(acc[nb][G][2], acc[nb][G][3]), off);
        sa = G ? f2_fma(ga[G], xa, sa) : f2_mul(ga[G], xa);
        sb = G ? f2_fma(gb[G], xb, sb) : f2_mul(gb[G], xb);
      }
      f2_unpack(f2_mul(sa, qp[4]), s[nb][0], s[nb][1]);
      f2_unpack(f2_mul(sb, qp[4]), s[nb][2], s[nb][3]);
    }
  }

  // O^T += V^T . (s_v P)^T over 16 tokens; pb = P^T as a B operand.
  template <int U>
  __device__ __forceinline__ void values(const uint32_t (&pb)[NB][2], const unsigned char *vt, int sc, int n_tok, const int4 &at, int r4) {
    constexpr int UB = Cfg4<U>::UB, DB = UB * token_of_row<U>(8);
    const int o0 = at.z, o1 = at.w;
    const uint2 v0 = *reinterpret_cast<const uint2 *>(vt + o0 + 8 * r4);
    const uint2 v1 = *reinterpret_cast<const uint2 *>(vt + o1 + 8 * r4);
    const uint2 v2 = *reinterpret_cast<const uint2 *>(vt + o0 + DB + 8 * r4);
    const uint2 v3 = *reinterpret_cast<const uint2 *>(vt + o1 + DB + 8 * r4);
    uint32_t w0 = *reinterpret_cast<const uint32_t *>(vt + o0 + sc);
    uint32_t w1 = *reinterpret_cast<const uint32_t *>(vt + o1 + sc);
    uint32_t w2 = *reinterpret_cast<const uint32_t *>(vt + o0 + DB + sc);
    uint32_t w3 = *reinterpret_cast<const uint32_t *>(vt + o1 + DB + sc);
    if (n_tok < 16) {   // what lies past the context is stale and may be NaN as a scale; its P is 0
      const int end = n_tok * UB;
      w0 = o0 < end ? w0 : 0u;
      w1 = o1 < end ? w1 : 0u;
      w2 = o0 + DB < end ? w2 : 0u;
      w3 = o1 + DB < end ? w3 : 0u;
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
  __device__ __forceinline__ void tile(const unsigned char *kt, const unsigned char *vt, int sc, int n_tok, int lane, const float *qs, const int4 &at, float *lg,
                                       int g) {
    constexpr int SUBS = Cfg4<U>::SUBS, STEP = 16 * Cfg4<U>::R, UB = Cfg4<U>::UB;
    const int r4 = lane >> 2, c4 = lane & 3;
    float s[SUBS][NB][4];
#pragma unroll
    for (int i = 0; i < SUBS; ++i) logits<U>(s[i], kt + i * STEP * UB, sc, at, c4, qs);
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
        const bool ragged = n_tok < (SUBS - 1) * STEP + 16;   // the context ends in this tile
        int ta = 0, tb = 0;
        if (LOG || ragged) { ta = at.y / UB; tb = ta + token_of_row<U>(8); }
        const bool va = ta + i * STEP < n_tok, vb = tb + i * STEP < n_tok;
        if (ragged) {
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
    for (int i = 0; i < SUBS; ++i) values<U>(pb[i], vt + i * STEP * UB, sc, n_tok - i * STEP, at, r4);
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

// What is needed once per piece is kept in shared memory, because registers held over the tile loop are the scarce
// resource (spills go to an L1 that the rings leave 20 KB of: a handful of reloads per tile cost 200 of 440 us).
struct PieceRec {
  const char *k, *v;               // the unit's rows of the piece's sequence
  int b, slab, tile_begin, tile_end, tiles, seq_len;   // as Piece; tiles = of the whole stream
  int stream_begin, stream_end;
};
constexpr int kPieces = 32;        // pieces looked up at a time; a share of more (many one-tile sequences) goes in rounds
struct FreshRow { uint32_t w[2][32]; };   // fused step: a warp's lanes' 16 bits and scale byte (<< 16) of the newest K and V row

// ring | barriers | pieces | fresh rows | q statistics | fragment offsets | flags | prefix[batch + 1] | lens[batch]
__host__ __device__ constexpr int meta_ints4(int batch) { return ((2 * batch + 1 + 4) + 1) / 2 * 2; }
template <int U, int NB>
struct Layout4 {
  static constexpr int kBars = Cfg4<U>::kStages * Cfg4<U>::kStage;
  static constexpr int kPiece = kBars + Cfg4<U>::kStages * 16;
  static constexpr int kFresh = kPiece + kPieces * static_cast<int>(sizeof(PieceRec));
  static constexpr int kQ = kFresh + kCWarps * static_cast<int>(sizeof(FreshRow));
  static constexpr int kAt = kQ + kCWarps * WarpAttn4<NB>::kQFloats * 4;      // per lane: fragment offsets in a tile
  static constexpr int kMeta = kAt + 32 * 16;                                 // 4 ints: total positions, CTAs, pieces of the share
  static constexpr int bytes(int batch) { return kMeta + meta_ints4(batch) * 4; }
  static_assert(kPiece % 8 == 0 && kQ % 16 == 0 && kAt % 16 == 0 && kMeta % 8 == 0, "alignment");
};

// Merging the pieces of a stream.  Every warp publishes its own state (the scratch layout of merge_stream) and draws a
// ticket of its kv head; whoever draws the last one merges, so the heads of a stream are merged side by side by whichever
// CTAs finish last.  A stream cut into many states is merged in two levels: groups of about sqrt(states), each by the
// warp that completes it, into the state of the group's first piece; then the groups.  Whole call with one and with two
// levels: 2 sequences of 28k rows, 32/8 heads, 65 and 41 us; 3 of 20k-27k, 8/2 heads (four warps a head), 109 and 32;
// 2 of 1.7k, 8/1 heads (eight warps a head), 60 and 29.
struct MergeArgs {
  int b, kv_head, first, count, step, per;   // pieces first, first + step, ... (count of them), `per` states each
  int c_first, slot0;                        // the stream's first piece and its scratch slot
};

// I q heads at a time, J states of each in flight, the first before the weights are known.  final: the result; otherwise
// the merged state goes to the first piece's first row.  One warp alone issues an instruction every few cycles, so what
// counts is their number: a lane works out where one state lies and the others take it from there by a shuffle (with the
// division in every load 22 states of 4 heads took 21 us).  Rows of heads behind the last and the repeated last state
// are read along, and left out or weighted 0.
template <int U, int HEADS, int I, int J>
__device__ __forceinline__ void merge_states(const AttnParams &p, const MergeArgs &a, bool final, int lane, int g) {
  const int n_src = a.count * a.per, hh = a.kv_head % U;
  const auto state_at = [&](int i) {   // in floats; the scratch holds below 2^25
    const int q = i / a.per, c = a.first + q * a.step, r = i - q * a.per;
    const int slot = c * 2 + (c == a.c_first ? a.slot0 : 0);
    return (slot * kCWarps + r * U + hh) * (HEADS * kPartRow);
  };
  const float vsc = __ldg(p.v_scale + a.kv_head);
  float *const part = p.fl_part;
  for (int h0 = 0; h0 < g; h0 += I) {
    const float *const mine = part + h0 * kPartRow + lane * 4;
    float M[I], L[I];
    float4 acc[I];
#pragma unroll
    for (int k = 0; k < I; ++k) {
      M[k] = -INFINITY;
      L[k] = 0.f;
      acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int s0 = 0; s0 < n_src; s0 += 32) {
      const int cnt = min(32, n_src - s0);
      const int at = state_at(s0 + min(lane, cnt - 1));
      float2 ml[I];
#pragma unroll
      for (int k = 0; k < I; ++k) {
        ml[k] = __ldcg(reinterpret_cast<const float2 *>(part + at + (h0 + k) * kPartRow + 128));
        if (lane >= cnt) ml[k] = make_float2(-INFINITY, 0.f);
      }
      float4 v[J][I];
      const auto fetch = [&](int j0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float *src = mine + __shfl_sync(0xffffffffu, at, j0 + j);
#pragma unroll
          for (int k = 0; k < I; ++k) v[j][k] = __ldcg(reinterpret_cast<const float4 *>(src + k * kPartRow));
        }
      };
      fetch(0);
      float w[I];   // weight of state s0 + lane
#pragma unroll
      for (int k = 0; k < I; ++k) {
        float mx = ml[k].x;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float Mn = fmaxf(M[k], mx), f = M[k] == -INFINITY ? 0.f : ex2(M[k] - Mn);
        w[k] = ml[k].x == -INFINITY ? 0.f : ex2(ml[k].x - Mn);
        float sum = w[k] * ml[k].y;
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        L[k] = L[k] * f + sum;
        acc[k].x *= f; acc[k].y *= f; acc[k].z *= f; acc[k].w *= f;
        M[k] = Mn;
      }
#pragma unroll 1
      for (int j0 = 0; j0 < cnt; j0 += J) {
        if (j0 > 0) fetch(j0);
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
          for (int k = 0; k < I; ++k) {
            const float y = __shfl_sync(0xffffffffu, w[k], j0 + j);   // 0 behind the last state
            acc[k].x = fmaf(y, v[j][k].x, acc[k].x); acc[k].y = fmaf(y, v[j][k].y, acc[k].y);
            acc[k].z = fmaf(y, v[j][k].z, acc[k].z); acc[k].w = fmaf(y, v[j][k].w, acc[k].w);
          }
      }
    }
    __syncwarp();   // every lane has read the rows of these heads
#pragma unroll
    for (int k = 0; k < I; ++k) {
      if (h0 + k >= g) continue;
      if (final) {
        const int hq = a.kv_head * g + h0 + k;
        const float inv = vsc / L[k];
        uint2 packed;
        packed.x = pack_bf16(acc[k].x * inv, acc[k].y * inv);
        packed.y = pack_bf16(acc[k].z * inv, acc[k].w * inv);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(p.out) + a.b * p.out_stride + hq * kHeadDim + lane * 4) = packed;
        if (lane == 0) write_stats(p, a.b * p.h + hq, M[k], L[k]);
      } else {
        float *dst = part + state_at(0) + (h0 + k) * kPartRow;
        *reinterpret_cast<float4 *>(dst + lane * 4) = acc[k];
        if (lane == 0) *reinterpret_cast<float2 *>(dst + 128) = make_float2(M[k], L[k]);
      }
    }
  }
}
template <int U, int HEADS>
__device__ __noinline__ void merge_any(const AttnParams &p, const MergeArgs &a, bool final, int lane, int g) {
  if (g == 1) merge_states<U, HEADS, 1, 16>(p, a, final, lane, g);
  else if (g == 2) merge_states<U, HEADS, 2, 8>(p, a, final, lane, g);
  else merge_states<U, HEADS, 4, 4>(p, a, final, lane, g);
}

// owner_of with a division of 32 bits where that is enough (64 bits: some 300 cycles each, between a state and its merge).
__device__ __forceinline__ int owner4(int tau, int total, int n_ctas) {
  const unsigned long long x = static_cast<unsigned long long>(tau + 1) * n_ctas - 1;
  return static_cast<int>(x >> 32 ? x / total : static_cast<unsigned>(x) / static_cast<unsigned>(total));
}

// One ticket for the whole warp, whose stores come before it; true for the last of `n`, which also clears the counter.
__device__ __forceinline__ bool last_ticket(unsigned *ctr, int n, int lane) {
  __syncwarp();
  int last = 0;
  if (lane == 0) {   // the fence covers the stores of the lanes it has met
    __threadfence();
    last = atomicAdd(ctr, 1u) + 1 == static_cast<unsigned>(n);
    if (last) *ctr = 0u;   // clean for the next launch
    __threadfence();
  }
  return __shfl_sync(0xffffffffu, last, 0);
}

// Called by every warp after it has published its state of piece `c` of stream [c_first, c_last].
constexpr int kOneLevel = 48;   // states; a second level costs its tickets and its start, about 4 us, which 22 states do not repay (19 and 20 us)
template <int U, int R, int HEADS>
__device__ __noinline__ void publish(const AttnParams &p, int b, int kv_head, int c, int c_first, int c_last, int slot0, int lane, int g) {
  const int pieces = c_last - c_first + 1, hh = kv_head % U;
  unsigned *ctr = p.fl_count + b * p.kvh + kv_head;
  MergeArgs a{b, kv_head, c_first, pieces, 1, R, c_first, slot0};
  int n = pieces * R;
  if (n > kOneLevel) {
    const int size = (static_cast<int>(sqrtf(static_cast<float>(n))) + R - 1) / R;   // pieces per group
    const int k = (c - c_first) / size, lead = c_first + k * size;
    const size_t slot = static_cast<size_t>(lead) * 2 + (lead == c_first ? slot0 : 0);
    a.first = lead;
    a.count = min(size, c_last + 1 - lead);
    if (!last_ticket(p.fl_group + slot * kCWarps + hh, a.count * R, lane)) return;
    merge_any<U, HEADS>(p, a, false, lane, g);
    a.first = c_first;
    a.count = n = (pieces + size - 1) / size;
    a.step = size;
    a.per = 1;
  }
  if (last_ticket(ctr, n, lane)) merge_any<U, HEADS>(p, a, true, lane, g);
}

// Looks up the next pieces of positions [meta[3], end), one warp for the CTA: meta[2] = how many that hold tiles, meta[3]
// = position behind them.
template <int UB>
__device__ __noinline__ void look_up(const AttnParams &p, PieceRec *rec, int *meta, int slabs, int end, int lane) {
  const int *prefix = meta + 4, *lens = prefix + p.batch + 1;
  int n = 0, tau = meta[3];
  while (tau < end && n < kPieces) {
    const Piece pc = locate(prefix, p.batch, slabs, tau, end);
    tau += pc.advance;
    if (pc.tile_end <= pc.tile_begin) continue;   // only phantom positions of this stream fall into the share
    if (lane == 0) {
      PieceRec &r = rec[n];
      r.b = pc.b; r.slab = pc.slab; r.tile_begin = pc.tile_begin; r.tile_end = pc.tile_end; r.tiles = pc.tiles_in_stream;
      r.seq_len = lens[pc.b];
      r.stream_begin = static_cast<int>(pc.stream_begin); r.stream_end = static_cast<int>(pc.stream_end);
    }
    ++n;
  }
  __syncwarp();
  for (int i = lane; i < n; i += 32) {   // the ranges' addresses, all pieces at once
    const int64_t slot = p.slot_ids[rec[i].b];
    rec[i].k = reinterpret_cast<const char *>(p.k_table[slot]) + rec[i].slab * UB;
    rec[i].v = reinterpret_cast<const char *>(p.v_table[slot]) + rec[i].slab * UB;
  }
  if (lane == 0) { meta[2] = n; meta[3] = tau; }
}

// Fused step: quantises the step's row of this warp's head, stores it into the ranges and leaves the lanes' bits in ws.
template <int U>
__device__ __noinline__ void append_row(const AttnParams &p, FreshRow &out, const PieceRec &pc, int hs, int64_t off, int lane) {
  const int kv_head = pc.slab * U + hs, at = 8 * (lane & 7) + 2 * (lane >> 3);
  for (int kv = 0; kv < 2; ++kv) {
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(kv ? p.new_value : p.new_key) +
                               pc.b * (kv ? p.new_value_stride : p.new_key_stride) + kv_head * kHeadDim + lane * 4;
    const uint2 w = __ldg(reinterpret_cast<const uint2 *>(src));
    const float x[4] = {bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
    uint32_t bits, s8;
    quantise4(x, (kv ? p.v_scale : p.k_scale)[kv_head], &bits, &s8);
    char *far = const_cast<char *>(kv ? pc.v : pc.k) + off;   // the unit's bytes of the row
    *reinterpret_cast<uint16_t *>(far + hs * 64 + at) = static_cast<uint16_t>(bits);
    if ((lane & 7) == 0) far[U * 64 + hs * 4 + (lane >> 3)] = static_cast<char>(s8);
    out.w[kv][lane] = bits | s8 << 16;
  }
  __syncwarp();
}

__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {   // does not suspend
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}

// Fetches tile `tile` of a piece into ring stage s; the whole warp calls it.  `use` = how often the stage was filled
// before.  1: done, 0: the stage is still in use and `wait` is false, -1: a bounded wait ran out.  A single-unit cache is
// contiguous over tokens: one copy of K and one of V.  Otherwise a row of the unit (80 to 544 bytes) is one copy.
template <int U>
__device__ __forceinline__ int fetch_tile(const AttnParams &p, unsigned char *smem, const PieceRec &pc, int tile, int s, int use,
                                          int slabs, int lane, bool wait) {
  using C = Cfg4<U>;
  constexpr int UB = C::UB;
  const uint32_t bar = smem_u32(smem) + C::kStages * C::kStage + 8 * s;   // full; the empty ones follow
  if (use > 0) {
    const uint32_t empty = bar + 8 * C::kStages, parity = (use - 1) & 1;
    if (!wait) {
      if (!__all_sync(0xffffffffu, mbar_test(empty, parity))) return 0;
    } else if (!__all_sync(0xffffffffu, mbar_wait(empty, parity))) {
      if (lane == 0) atomicExch(p.status, kKernelErrMagic);
      return -1;
    }
  }
  const int t0 = tile * C::TOK, nt = min(pc.seq_len - t0, C::TOK);
  const int64_t src = static_cast<int64_t>(t0) * (slabs * UB);
  const char *kb = pc.k + src, *vb = pc.v + src;
  const uint32_t dst = smem_u32(smem) + s * C::kStage;
  const uint64_t policy = l2_policy_evict_first();
  if (lane == 0) mbar_arrive_expect_tx(bar, 2u * nt * UB);
  __syncwarp();
  if (slabs == 1) {
    if (lane == 0) {
      bulk_g2s_hint(dst, kb, nt * UB, bar, policy);
      bulk_g2s_hint(dst + C::kTile, vb, nt * UB, bar, policy);
    }
  } else {
    for (int row = lane; row < nt; row += 32) {
      bulk_g2s_hint(dst + row * UB, kb + static_cast<int64_t>(row) * (slabs * UB), UB, bar, policy);
      bulk_g2s_hint(dst + C::kTile + row * UB, vb + static_cast<int64_t>(row) * (slabs * UB), UB, bar, policy);
    }
  }
  return 1;
}

// Moves a copy position `n` tiles on in the list of pieces.
__device__ __forceinline__ void next_copy(const PieceRec *rec, int pieces, int &piece, int &tile, int n) {
  tile += n;
  while (piece < pieces && tile >= rec[piece].tile_end) {
    const int over = tile - rec[piece].tile_end;
    ++piece;
    if (piece < pieces) tile = rec[piece].tile_begin + over;
  }
}

// Piece `now` of the CTA's share, the `it`-th tile on: attention, then either the result or a published state and a
// ticket.  Bit 0: a bounded wait ran out; bit 1: a state was published.  A function of its own, with no calls inside: what
// the compiler would otherwise keep on the stack across the merge it reloads in the tile loop.
template <int U, int NB, bool LOG>
__device__ __noinline__ int run_piece(const AttnParams &p, int now, int it, int state, int &copy_piece, int &copy_tile) {
  using C = Cfg4<U>;
  using S = Layout4<U, NB>;
  constexpr int R = C::R, UB = C::UB, TOK = C::TOK, HEADS = NB * 8;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hs = warp % U, rr = warp / U;      // head of the unit, token sub-row
  float *qs = reinterpret_cast<float *>(smem + S::kQ) + warp * WarpAttn4<NB>::kQFloats;
  const int *meta = reinterpret_cast<const int *>(smem + S::kMeta);
  const uint32_t full0 = smem_u32(smem + S::kBars), empty0 = full0 + 8 * C::kStages;
  const int g = p.h / p.kvh, slabs = p.kvh / U;
  const PieceRec *rec = reinterpret_cast<const PieceRec *>(smem + S::kPiece);
  const PieceRec &pc = rec[now];
  bool failed = state & 1;
  const bool fresh = state & 2;   // this warp overlays the newest token's row; bit 2: the CTA's first piece
  WarpAttn4<NB> st;
  {
    const int kv_head = pc.slab * U + hs;
    st.start(static_cast<const __nv_bfloat16 *>(p.q) + pc.b * p.q_stride + kv_head * g * kHeadDim, g,
             p.scale * 1.4426950408889634f * p.k_scale[kv_head], lane, qs);
  }
  int left = pc.seq_len - pc.tile_begin * TOK;   // tokens from the tile's first to the end of the context
  for (int tiles = pc.tile_end - pc.tile_begin; tiles > 0; --tiles, ++it, left -= TOK) {
    const int s = it % C::kStages;
    // Warp n % 8 fetches tile n, into the stage of the tile before this one: now if all warps are done with that, else
    // after this tile.
    const int n = it + C::kStages - 1;
    const bool mine = (n & (kCWarps - 1)) == warp && copy_piece < meta[2];
    int fetched = 1;
    if (mine && !failed) fetched = fetch_tile<U>(p, smem, rec[copy_piece], copy_tile, n % C::kStages, n / C::kStages, slabs, lane, false);
    if (!failed && !mbar_wait(full0 + 8 * s, (it / C::kStages) & 1)) failed = true;
    if (failed) continue;
    unsigned char *kt = smem + s * C::kStage + hs * 64;
    constexpr int kSc = U * 64;   // scale words from the unit's first byte
    const bool overlay = fresh && left <= TOK;
    if (overlay) {   // the copy brought whatever the range held in the newest row's place
      const int at = 8 * (lane & 7) + 2 * (lane >> 3);
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        const uint32_t w = reinterpret_cast<const FreshRow *>(smem + S::kFresh)[warp].w[kv][lane];
        unsigned char *row = kt + kv * C::kTile + (left - 1) * UB;
        *reinterpret_cast<uint16_t *>(row + at) = static_cast<uint16_t>(w);
        if ((lane & 7) == 0) row[kSc - hs * 60 + (lane >> 3)] = static_cast<unsigned char>(w >> 16);
      }
      __syncwarp();
    }
    const int n_tok = left - 16 * rr;
    if (n_tok > 0) {
      float *lg = nullptr;
      if constexpr (LOG)
        lg = p.logits + ((static_cast<size_t>(pc.b) * p.kvh + pc.slab * U + hs) * p.logit_rows + (pc.seq_len - n_tok)) * g;
      st.template tile<U, LOG>(kt + 16 * rr * UB, kt + C::kTile + 16 * rr * UB, kSc - hs * 60, n_tok, lane, qs,
                               reinterpret_cast<const int4 *>(smem + S::kAt)[lane], lg, g);
    }
    if (overlay) fence_proxy_async();   // before the copy engine refills the stage
    __syncwarp();
    if (lane == 0) mbar_arrive(empty0 + 8 * s);
    if (fetched == 0 && fetch_tile<U>(p, smem, rec[copy_piece], copy_tile, n % C::kStages, n / C::kStages, slabs, lane, true) < 0)
      failed = true;
    if (mine) next_copy(rec, meta[2], copy_piece, copy_tile, kCWarps);
  }
  st.finish(lane);

  const int kv_head = pc.slab * U + hs;
  const bool whole = pc.tile_begin == 0 && pc.tile_end == pc.tiles;
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
          __nv_bfloat16 *dst = static_cast<__nv_bfloat16 *>(p.out) + pc.b * p.out_stride + hq * kHeadDim;
#pragma unroll
          for (int mb = 0; mb < 8; ++mb)   // dims d, d + 1 are the two fragment rows
            *reinterpret_cast<uint32_t *>(dst + WarpAttn4<NB>::dim_of(mb, 0, r4)) =
                pack_bf16(st.o[nb][mb][e] * inv, st.o[nb][mb][2 + e] * inv);
          if (r4 == 0) write_stats(p, pc.b * p.h + hq, st.mrun[nb][e], st.lrun[nb][e]);
        }
      }
    }
  } else {
    if (p.overlap) pdl_wait_prior_grid();   // the scratch is shared with the previous launch
    float *slot_base = p.fl_part + (static_cast<size_t>(blockIdx.x) * 2 + (state & 4 ? 0 : 1)) * kCWarps * HEADS * kPartRow;
    st.template store<kPartRow>(slot_base + warp * HEADS * kPartRow, lane, g);
    return (failed ? 1 : 0) | 2;
  }
  return failed ? 1 : 0;
}

template <int U, int NB, bool LOG>
__global__ void __launch_bounds__(kThreads4, NB == 1 ? 2 : 1) attn_int4_kernel(const __grid_constant__ AttnParams p) {
  using C = Cfg4<U>;
  using S = Layout4<U, NB>;
  constexpr int R = C::R, UB = C::UB, TOK = C::TOK, HEADS = NB * 8;
  extern __shared__ __align__(128) unsigned char smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int hs = warp % U, rr = warp / U;      // head of the unit, token sub-row
  int *meta = reinterpret_cast<int *>(smem + S::kMeta);
  int *prefix = meta + 4, *lens = prefix + p.batch + 1;
  PieceRec *rec = reinterpret_cast<PieceRec *>(smem + S::kPiece);
  const uint32_t full0 = smem_u32(smem + S::kBars), empty0 = full0 + 8 * C::kStages;
  const int g = p.h / p.kvh, slabs = p.kvh / U;
  if (threadIdx.x < 32)   // K row's part, K scales, V rows 2 c4 and 2 c4 + 1 (without the lane's 8 bytes)
    reinterpret_cast<int4 *>(smem + S::kAt)[lane] =
        make_int4(token_of_row<U>(lane >> 2) * UB + 16 * (lane & 3), token_of_row<U>(lane >> 2) * UB,
                  token_of_row<U>(2 * (lane & 3)) * UB, token_of_row<U>(2 * (lane & 3) + 1) * UB);
  if (threadIdx.x == 32) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(full0 + 8 * s, 1);
      mbar_init(empty0 + 8 * s, kCWarps);
    }
    mbar_fence_init();
  }
  for (int i = threadIdx.x; i < p.batch; i += kThreads4) {
    int len = max(p.seq_lens[i], 0);
    if constexpr (LOG) len = min(len, p.logit_rows);   // the logits have room for no more
    lens[i] = len;
    prefix[i + 1] = len > 0 ? ((len + TOK - 1) / TOK + kBoundaryCost) * slabs : 0;
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
    if (lane == 0) {
      prefix[0] = 0;
      const int n_ctas = min(static_cast<int>(gridDim.x), carry);
      meta[0] = carry;
      meta[1] = n_ctas;
      meta[3] = static_cast<int>(blockIdx.x) < n_ctas ? static_cast<int>(static_cast<long long>(carry) * blockIdx.x / n_ctas) : 0;
    }
  }
  __syncthreads();
  pdl_launch_dependents();
  const int end = static_cast<int>(blockIdx.x) < meta[1] ? static_cast<int>(static_cast<long long>(meta[0]) * (blockIdx.x + 1) / meta[1]) : 0;

  if (blockIdx.x == 0) {   // sequences without context produce zeros; nobody owns a tile of theirs
    for (int b = 0; b < p.batch; ++b)
      if (prefix[b + 1] == prefix[b]) {
        for (int i = threadIdx.x; i < p.h * kHeadDim; i += kThreads4)
          static_cast<__nv_bfloat16 *>(p.out)[b * p.out_stride + i] = __float2bfloat16(0.f);
        if (p.lse)
          for (int i = threadIdx.x; i < p.h; i += kThreads4) p.lse[b * p.h + i] = -INFINITY;
      }
  }
  bool failed = false, first = true, more = true;
  int it = 0;   // tiles of the share so far
  while (more) {
    if (warp == 0) look_up<UB>(p, rec, meta, slabs, end, lane);
    __syncthreads();
    const int pieces = meta[2];
    int copy_piece = 0, copy_tile = rec[0].tile_begin;
    const int ahead = (warp - it) & (kCWarps - 1);   // warp n % 8 fetches tile n
    next_copy(rec, pieces, copy_piece, copy_tile, ahead);
    if (ahead < C::kStages - 1 && copy_piece < pieces) {
      const int n = it + ahead;
      failed |= fetch_tile<U>(p, smem, rec[copy_piece], copy_tile, n % C::kStages, n / C::kStages, slabs, lane, true) < 0;
      next_copy(rec, pieces, copy_piece, copy_tile, kCWarps);
    }
    for (int now = 0; now < pieces; ++now) {
      const PieceRec &pc = rec[now];
      if (p.overlap == 2) pdl_wait_prior_grid();
      const int64_t append_off = p.new_key ? p.byte_off[pc.b] : -1;
      const bool fresh = append_off >= 0 && pc.tile_end == pc.tiles && ((pc.seq_len - 1) % TOK / 16) % R == rr;
      if (fresh)   // this warp owns the newest token's row of its head
        append_row<U>(p, reinterpret_cast<FreshRow *>(smem + S::kFresh)[warp], pc, hs, append_off, lane);
      const int got = run_piece<U, NB, LOG>(p, now, it, (failed ? 1 : 0) | (fresh ? 2 : 0) | (first ? 4 : 0), copy_piece, copy_tile);
      failed = got & 1;
      first = false;
      it += pc.tile_end - pc.tile_begin;
      if (got & 2) {
        const int total = meta[0], n_ctas = meta[1], c_first = owner4(pc.stream_begin + kBoundaryCost, total, n_ctas);
        // the stream is its first CTA's first piece iff it already runs where that CTA's share begins
        const int slot0 = static_cast<long long>(pc.stream_begin) * n_ctas <= static_cast<long long>(total) * c_first ? 0 : 1;
        publish<U, R, HEADS>(p, pc.b, pc.slab * U + hs, blockIdx.x, c_first, owner4(pc.stream_end - 1, total, n_ctas), slot0, lane, g);
      }
      // a stream that lies wholly in this CTA's share used slot 1, as the next piece may
      if (R > 1 && pc.tile_begin == 0 && pc.tile_end == pc.tiles) named_bar_sync(1, kCWarps * 32);
    }
    more = meta[3] < end;
    __syncthreads();   // the list and its end are read no more
  }
}

template <int U, int NB, bool LOG>
int launch4(const AttnParams &p_in, cudaStream_t stream) {
  AttnParams p = p_in;
  p.n_ctas = (NB == 1 ? 2 : 1) * kFlatSms;
  const int smem = Layout4<U, NB>::bytes(p.batch);
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
