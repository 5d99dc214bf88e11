// The 4-bit KV cache format, shared by the append, the read-back and the attention kernels.
//
// One token's row holds all kv heads of the rank, in units of U heads (U = 8, 4, 2 or 1, the largest that divides
// kvh).  A unit is U x 64 bytes of nibbles followed by U x 4 bytes of group scales, zero-padded to 16 bytes: 544,
// 272, 144 or 80 bytes.  Every row therefore starts on a 16-byte boundary and a run of rows of a single-unit cache
// is one contiguous bulk copy, the same property the bf16 and fp8 rows have.
//   dim 32 G + 4 r + j  ->  byte 8 r + 2 G + (j >> 1) of the head's 64 bytes, low nibble for even j
//   group G (32 dims)   ->  e4m3 scale byte G of the head's 4
//   element = (nibble - 8) * e4m3 * scale[kv_head],  nibble - 8 in [-7, 7]
// The nibble order is the attention kernel's: the 8 bytes [8 r, 8 r + 8) give the lane that owns fragment row r four
// dims of each of the four groups, so that one accumulator tile (16 dims) lies inside one group (see vt_attn_int4.cu).
// scale[kv_head] is the frozen per-head scale of the fp8 cache (amax / 448); a group's e4m3 scale is its own amax / 7
// in units of that, at most 64 for values inside the calibrated range, so seven times that range is representable.
#pragma once
#include "vt_device.cuh"

namespace vt {

__host__ __device__ constexpr int int4_unit(int kvh) {
  return kvh % 8 == 0 ? 8 : kvh % 4 == 0 ? 4 : kvh % 2 == 0 ? 2 : 1;
}
__host__ __device__ constexpr int int4_unit_bytes(int u) { return 64 * u + (4 * u + 15) / 16 * 16; }
__host__ __device__ constexpr int int4_row_bytes(int kvh) {
  return kvh / int4_unit(kvh) * int4_unit_bytes(int4_unit(kvh));
}
// byte offsets of a head's nibbles and of its scale word inside a row
__host__ __device__ constexpr int int4_head_offset(int kvh, int head) {
  const int u = int4_unit(kvh);
  return head / u * int4_unit_bytes(u) + head % u * 64;
}
__host__ __device__ constexpr int int4_scale_offset(int kvh, int head) {
  const int u = int4_unit(kvh);
  return head / u * int4_unit_bytes(u) + 64 * u + head % u * 4;
}

__device__ __forceinline__ float e4m3_to_float(uint32_t byte) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<unsigned short>(byte)));
  return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xffffu)));
}

// One warp quantises one head's row of one token: lane l brings dims 4 l .. 4 l + 3 (group l / 8) and gets back their
// 16 bits, byte 8 (l % 8) + 2 (l / 8) of the head, and its group's scale byte.  IEEE divisions, so that the stored
// bits are those of the definition: s8 = e4m3(amax / (7 S)) saturating, q = clamp(round(x / (s8 S)), -7, 7).  NaN
// elements become 0 and do not enter amax; infinities saturate; a group with step 0 is all zero.
__device__ __forceinline__ void quantise4(const float (&x)[4], float head_scale, uint32_t *bits, uint32_t *scale_byte) {
  float amax = fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3])));   // fmaxf drops NaN
  amax = fmaxf(amax, 0.f);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const uint32_t s8 = float2_to_e4m3x2(__fdiv_rn(amax, __fmul_rn(7.0f, head_scale)), 0.f) & 0xffu;
  const float step = __fmul_rn(e4m3_to_float(s8), head_scale);
  uint32_t b = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    int q = 0;
    if (step > 0.f && x[j] == x[j]) q = static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x[j], step)), -7.f), 7.f));
    b |= static_cast<uint32_t>(q + 8) << (4 * j);
  }
  *bits = b;
  *scale_byte = step > 0.f ? s8 : 0u;
}

}  // namespace vt
