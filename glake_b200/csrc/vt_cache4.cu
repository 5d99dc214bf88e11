// Writing and reading back quantised KV ranges outside the attention kernels: the 4-bit append
// (reshape_and_cache with kv dtype int4) and the read-back of a quantised cache as dense bf16 rows.
//
// Bytes per (row, kv head): append reads 512 (K and V, bf16) and writes 136; read-back the reverse.  HBM is the bound
// only if the arithmetic stays small, about 14 instructions per element at the copy bandwidth.  Hence eight lanes per
// (row, head) with 16 elements each, the group maximum on packed bf16, and one multiplication by 1 / step per element
// in place of a division (append_int4_kernel), with the loads a round ahead; 8 x 4096 rows of 8 heads: append 44 us (3.9
// TB/s), read-back 33 us (5.1 TB/s), against 140 and 44 with one warp per (row, head) and a division per element.  What
// bounds the append is instruction issue (82 % busy), the integer unit (60 %) the read-back.
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_int4.cuh"
#include "vt_kernels.h"
#include "vt_mma.cuh"

namespace vt {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = kThreads / 8;   // (row, head) pairs a CTA works on at once

// Division by the number of kv heads: n / d for n < 2^32 / d.
struct FastDiv {
  uint32_t d, m;
  explicit FastDiv(int n) : d(n), m(n == 1 ? 0u : static_cast<uint32_t>((1ull << 32) / n) + 1u) {}
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return d == 1 ? n : __umulhi(n, m); }
};

__device__ __forceinline__ uint32_t absmax_bf16x2(uint32_t a, uint32_t b) {   // NaN wins
  const __nv_bfloat162 x = __hmax2_nan(__habs2(*reinterpret_cast<const __nv_bfloat162 *>(&a)),
                                       __habs2(*reinterpret_cast<const __nv_bfloat162 *>(&b)));
  return *reinterpret_cast<const uint32_t *>(&x);
}

// Codes of 16 elements for one step, four to the low 16 bits of a word (the bits above are junk).  q = round(x / step)
// as the rounding of x times the rounded reciprocal, taken exactly inside an FMA: that product is within 2e-6 of the
// quotient (below 7.5 in magnitude for a scale that did not saturate), so the result is that of the IEEE division
// except where it comes within 1e-5 of a tie.  False then, and for a step whose reciprocal is no normal number.
__device__ __forceinline__ bool codes_fast(const float (&x)[16], float step, uint32_t (&c)[4]) {
  constexpr float kMagic = 12582920.f;   // 1.5 2^23 + 8: the low bits of x inv + kMagic are q + 8
  const float inv = step > 0.f ? __frcp_rn(step) : 0.f;
  float worst = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t t[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float r = __fmaf_rn(x[4 * i + j], inv, kMagic);
      worst = fmaxf(worst, fabsf(__fmaf_rn(x[4 * i + j], inv, -__fsub_rn(r, kMagic))));
      t[j] = __float_as_uint(r);
    }
    c[i] = t[0] + t[1] * 16u + t[2] * 256u + t[3] * 4096u;   // kMagic's other bits lie above bit 16
  }
  return worst < 0.49999f && !(step > 0.f && step < 1.18e-38f);
}
// The code of one element, by definition.  (By value: an array handed over would live in local memory in every round.)
__device__ __noinline__ uint32_t code_exact(float x, float step) {
  int q = 0;
  if (step > 0.f && x == x) q = static_cast<int>(fminf(fmaxf(rintf(__fdiv_rn(x, step)), -7.f), 7.f));
  return static_cast<uint32_t>(q + 8);
}

// Eight lanes per (row, kv head, K or V): lane 2 G + p brings dims 32 G + 16 p .. + 15, i.e. the codes of group G for
// the pieces r = 4 p .. 4 p + 3, and after a 4 x 4 transposition among the lanes of equal p stores all of piece
// r = 4 p + G (8 bytes).  grid: (batch, row blocks); rows_per_cta 1 for decode.
__global__ void __launch_bounds__(kThreads) append_int4_kernel(AppendParams p, int rows_per_cta, bool vec_ok, FastDiv kvh_div) {
  const int i = blockIdx.x;
  const int64_t off = p.byte_off[i];
  if (off < 0) return;   // padded entry
  const bool decode = p.max_seq_len == 1;
  const int n_rows = decode ? 1 : p.seq_lens[i];
  const int t0 = blockIdx.y * rows_per_cta;
  if (t0 >= n_rows) return;
  const int t1 = min(t0 + rows_per_cta, n_rows);
  const int64_t slot = p.slot_ids[i];
  const int64_t row_bytes = int4_row_bytes(p.kvh);
  const int lane = threadIdx.x & 31, l8 = lane & 7, G = l8 >> 1, half = l8 & 1;
  const int64_t src0 = decode ? i : static_cast<int64_t>(p.cache_seq_lens[i]);
  const uint32_t items = static_cast<uint32_t>(t1 - t0) * p.kvh * 2;
  char *const base[2] = {reinterpret_cast<char *>(p.k_table[slot]) + off, reinterpret_cast<char *>(p.v_table[slot]) + off};
  const int u = int4_unit(p.kvh), ub = int4_unit_bytes(u), ushift = __ffs(u) - 1;
  // A round's 32 bytes and head scale are loaded one round ahead.  Whole warps go round together: lanes past the last
  // item work on it again and do not store.
  struct Item { uint32_t w[8]; float head_scale; int head, kv, t; };
  const auto load = [&](uint32_t first, Item &it) {
    const uint32_t n = min(first + (lane >> 3), items - 1);
    const uint32_t rest = kvh_div.div(n);
    it.head = n - rest * p.kvh;
    it.kv = rest & 1;
    it.t = t0 + (rest >> 1);
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(it.kv ? p.value : p.key) +
                               (src0 + it.t) * (it.kv ? p.value_stride : p.key_stride) + it.head * kHeadDim + l8 * 16;
    if (vec_ok) {
      const uint4 a = __ldcs(reinterpret_cast<const uint4 *>(src)), b = __ldcs(reinterpret_cast<const uint4 *>(src) + 1);
      it.w[0] = a.x; it.w[1] = a.y; it.w[2] = a.z; it.w[3] = a.w; it.w[4] = b.x; it.w[5] = b.y; it.w[6] = b.z; it.w[7] = b.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        it.w[e] = __bfloat16_as_ushort(src[2 * e]) | static_cast<uint32_t>(__bfloat16_as_ushort(src[2 * e + 1])) << 16;
    }
    it.head_scale = __ldg((it.kv ? p.v_scale : p.k_scale) + it.head);
  };
  Item next;
  uint32_t first = threadIdx.x / 32 * 4;
  if (first < items) load(first, next);
  for (; first < items; first += kItems) {
    const Item cur = next;
    if (first + kItems < items) load(first + kItems, next);
    const uint32_t(&w)[8] = cur.w;
    const int head = cur.head, kv = cur.kv, t = cur.t;
    const uint32_t mine = first + (lane >> 3);
    float x[16];
#pragma unroll
    for (int e = 0; e < 8; ++e) { x[2 * e] = bf16_lo(w[e]); x[2 * e + 1] = bf16_hi(w[e]); }
    uint32_t m = absmax_bf16x2(absmax_bf16x2(absmax_bf16x2(w[0], w[1]), absmax_bf16x2(w[2], w[3])),
                               absmax_bf16x2(absmax_bf16x2(w[4], w[5]), absmax_bf16x2(w[6], w[7])));
    m = absmax_bf16x2(m, __shfl_xor_sync(0xffffffffu, m, 1));
    float amax = bf16_hi(absmax_bf16x2(m, m << 16));
    const bool odd = __any_sync(0xffffffffu, amax != amax);
    if (odd) {   // some element is NaN: the maximum of the others
      amax = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) amax = fmaxf(amax, fabsf(x[e]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    }
    const float head_scale = cur.head_scale;
    uint32_t s8 = float2_to_e4m3x2(__fdiv_rn(amax, __fmul_rn(7.0f, head_scale)), 0.f) & 0xffu;
    const float step = __fmul_rn(e4m3_to_float(s8), head_scale);
    if (!(step > 0.f)) s8 = 0u;
    uint32_t c[4];
    const bool sure = codes_fast(x, step, c);
    if (odd || !sure || s8 >= 0x7eu) {   // NaN, a near tie, a saturated scale
#pragma unroll
      for (int e = 0; e < 4; ++e)
        c[e] = code_exact(x[4 * e], step) | code_exact(x[4 * e + 1], step) << 4 | code_exact(x[4 * e + 2], step) << 8 |
               code_exact(x[4 * e + 3], step) << 12;
    }
    // transposition: word of group G, piece i -> words of piece G
    const uint32_t a = __byte_perm(c[0], c[1], 0x5410), b = __byte_perm(c[2], c[3], 0x5410);
    const bool upper = (G & 2) != 0, odd_group = (G & 1) != 0;
    const uint32_t got = __shfl_xor_sync(0xffffffffu, upper ? a : b, 4);
    const uint32_t lo_g = upper ? got : a, hi_g = upper ? b : got;   // groups G & 1 and (G & 1) + 2, pieces 2 (G >> 1), + 1
    const uint32_t even_p = __byte_perm(lo_g, hi_g, 0x5410), odd_p = __byte_perm(lo_g, hi_g, 0x7632);
    const uint32_t other = __shfl_xor_sync(0xffffffffu, odd_group ? even_p : odd_p, 2);
    const uint32_t g0 = odd_group ? other : even_p, g1 = odd_group ? odd_p : other;   // groups (0, 2) and (1, 3) of piece G
    uint32_t sw = s8 << (8 * G);
    sw |= __shfl_xor_sync(0xffffffffu, sw, 2);
    sw |= __shfl_xor_sync(0xffffffffu, sw, 4);
    if (mine < items) {
      char *unit = base[kv] + t * row_bytes + (head >> ushift) * ub;
      const int hh = head & (u - 1);
      *reinterpret_cast<uint2 *>(unit + hh * 64 + 8 * (4 * half + G)) =
          make_uint2(__byte_perm(g0, g1, 0x5410), __byte_perm(g0, g1, 0x7632));
      if (l8 == 0) *reinterpret_cast<uint32_t *>(unit + 64 * u + 4 * hh) = sw;
    }
  }
}

// Rows [0, seq_lens[i]) of entry i's ranges as bf16 rows row_start[i] .. of k_out / v_out: eight lanes per (row, head),
// 16 dims each.  The product nibble * e4m3 is exact, the product with the head's scale is rounded to fp32 and the
// result once to bf16.
template <bool INT4>
__global__ void __launch_bounds__(kThreads) dequant_kernel(KvDequantParams p, int rows_per_cta, FastDiv kvh_div) {
  const int i = blockIdx.x;
  const int n_rows = min(p.seq_lens[i], p.max_seq_len);   // the caller made room for no more
  const int t0 = blockIdx.y * rows_per_cta;
  if (t0 >= n_rows) return;
  const int t1 = min(t0 + rows_per_cta, n_rows);
  const int64_t slot = p.slot_ids[i];
  const int64_t out0 = p.row_start[i];
  const int64_t row_bytes = INT4 ? int4_row_bytes(p.kvh) : p.kvh * kHeadDim;
  const int l8 = threadIdx.x & 7;
  const int u = int4_unit(p.kvh), ub = int4_unit_bytes(u), ushift = __ffs(u) - 1;
  const uint32_t items = static_cast<uint32_t>(t1 - t0) * p.kvh;
#pragma unroll 1
  for (int kv = 0; kv < 2; ++kv) {
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(kv ? p.v_out : p.k_out);
    if (!out) continue;
    const char *base = reinterpret_cast<const char *>(kv ? p.v_table[slot] : p.k_table[slot]);
    const float *scale = kv ? p.v_scale : p.k_scale;
    struct Item { uint4 w; uint32_t sw; float sc; uint32_t r; int head; };
    const auto load = [&](uint32_t n, Item &it) {
      it.r = kvh_div.div(n);
      it.head = n - it.r * p.kvh;
      const char *row = base + (t0 + static_cast<int>(it.r)) * row_bytes;
      if constexpr (INT4) {
        const char *unit = row + (it.head >> ushift) * ub;
        const int hh = it.head & (u - 1);
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(unit + hh * 64) + l8);   // piece l8: four dims of every group
        it.w = make_uint4(w.x, w.y, 0, 0);
        it.sw = __ldg(reinterpret_cast<const uint32_t *>(unit + 64 * u) + hh);
      } else {
        it.w = __ldcs(reinterpret_cast<const uint4 *>(row + it.head * kHeadDim) + l8);
      }
      it.sc = __ldg(scale + it.head);
    };
    // two items a round, the next round's in flight
    constexpr int N = 2;
    Item next[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((threadIdx.x >> 3) + k * kItems < items) load((threadIdx.x >> 3) + k * kItems, next[k]);
    for (uint32_t first = threadIdx.x >> 3; first < items; first += N * kItems) {
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const uint32_t n = first + k * kItems;
        if (n >= items) break;
        const Item cur = next[k];
        if (n + N * kItems < items) load(n + N * kItems, next[k]);
        __nv_bfloat16 *dst = out + ((out0 + t0 + static_cast<int>(cur.r)) * p.kvh + cur.head) * kHeadDim;
        if constexpr (INT4) {
          float s8[4];
          e4m3x4_to_float(cur.sw, s8);
#pragma unroll
          for (int G = 0; G < 4; ++G) {
            const uint32_t x = (G & 2 ? cur.w.y : cur.w.x) >> (16 * (G & 1));
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // 2^23 + nibble as a float, less 2^23 + 8
              const float q = __uint_as_float(((x >> (4 * j)) & 15u) | 0x4b000000u) - 8388616.f;
              f[j] = __fmul_rn(q * s8[G], cur.sc);
            }
            *reinterpret_cast<uint2 *>(dst + 32 * G + 4 * l8) = make_uint2(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]));
          }
        } else {
          float f[16];
          Unpack<true>::run(cur.w, f);
          uint32_t o[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) o[j] = pack_bf16(__fmul_rn(f[2 * j], cur.sc), __fmul_rn(f[2 * j + 1], cur.sc));
          uint4 *q = reinterpret_cast<uint4 *>(dst + 16 * l8);
          q[0] = make_uint4(o[0], o[1], o[2], o[3]);
          q[1] = make_uint4(o[4], o[5], o[6], o[7]);
        }
      }
    }
  }
}

// Rows per CTA: 128 (row, head) items, four rounds of the CTA, but fewer while that leaves less than four CTAs per SM;
// grid.y holds 65 535 blocks.
int rows_of_cta(int batch, int items_per_row, int max_seq_len) {
  const int64_t rows = static_cast<int64_t>(batch) * max_seq_len;
  const int64_t spread = rows / (4 * kFlatSms);
  const int most = std::max(1, 128 / items_per_row), least = std::max(1, kItems / items_per_row);
  return std::max<int>((max_seq_len + 65534) / 65535, static_cast<int>(std::min<int64_t>(most, std::max<int64_t>(least, spread))));
}

}  // namespace

int launch_append_int4(const AppendParams &p, cudaStream_t stream) {
  if (p.batch == 0) return VT_OK;
  const bool decode = p.max_seq_len == 1;
  const int rows_per_cta = decode ? 1 : rows_of_cta(p.batch, 2 * p.kvh, p.max_seq_len);
  const dim3 grid(p.batch, decode ? 1 : (p.max_seq_len + rows_per_cta - 1) / rows_per_cta);
  const bool vec_ok = ((reinterpret_cast<uintptr_t>(p.key) | reinterpret_cast<uintptr_t>(p.value)) & 15) == 0 &&
                      (p.key_stride % 8) == 0 && (p.value_stride % 8) == 0;
  append_int4_kernel<<<grid, kThreads, 0, stream>>>(p, rows_per_cta, vec_ok, FastDiv(p.kvh));
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

int launch_kv_dequant(const KvDequantParams &p, int kv_dtype, cudaStream_t stream) {
  const int max_seq_len = p.max_seq_len;
  if (p.batch == 0 || max_seq_len <= 0) return VT_OK;
  const int rows = rows_of_cta(p.batch, p.kvh, max_seq_len);
  const dim3 grid(p.batch, (max_seq_len + rows - 1) / rows);
  if (kv_dtype == VT_KV_INT4)
    dequant_kernel<true><<<grid, kThreads, 0, stream>>>(p, rows, FastDiv(p.kvh));
  else
    dequant_kernel<false><<<grid, kThreads, 0, stream>>>(p, rows, FastDiv(p.kvh));
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
