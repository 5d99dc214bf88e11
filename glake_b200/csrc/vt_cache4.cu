// Writing and reading back quantised KV ranges outside the attention kernels: the 4-bit append
// (reshape_and_cache with kv dtype int4) and the read-back of a quantised cache as dense bf16 rows.
//
// Bytes per (row, kv head): append reads 512 (K and V, bf16) and writes 136; read-back the reverse.  Both are bound by
// HBM for prompts; the arithmetic (one division per element and two per group) hides behind the loads.
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_int4.cuh"
#include "vt_kernels.h"

namespace vt {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

// One warp per (row, kv head, K or V).  grid: (batch, row blocks); rows_per_cta 1 for decode.
__global__ void __launch_bounds__(kThreads) append_int4_kernel(AppendParams p, int rows_per_cta, bool vec_ok) {
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
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t src0 = decode ? i : static_cast<int64_t>(p.cache_seq_lens[i]);
  const int items = (t1 - t0) * p.kvh * 2;
  for (int it = warp; it < items; it += kWarps) {
    const int head = it % p.kvh, rest = it / p.kvh;
    const int kv = rest & 1, t = t0 + (rest >> 1);
    const __nv_bfloat16 *src = static_cast<const __nv_bfloat16 *>(kv ? p.value : p.key) +
                               (src0 + t) * (kv ? p.value_stride : p.key_stride) + head * kHeadDim + lane * 4;
    float x[4];
    if (vec_ok) {
      const uint2 w = __ldg(reinterpret_cast<const uint2 *>(src));
      x[0] = bf16_lo(w.x); x[1] = bf16_hi(w.x); x[2] = bf16_lo(w.y); x[3] = bf16_hi(w.y);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = __bfloat162float(src[j]);
    }
    uint32_t bits, s8;
    quantise4(x, (kv ? p.v_scale : p.k_scale)[head], &bits, &s8);
    char *row = reinterpret_cast<char *>(kv ? p.v_table[slot] : p.k_table[slot]) + off + t * row_bytes;
    *reinterpret_cast<uint16_t *>(row + int4_head_offset(p.kvh, head) + 8 * (lane & 7) + 2 * (lane >> 3)) =
        static_cast<uint16_t>(bits);
    if ((lane & 7) == 0) row[int4_scale_offset(p.kvh, head) + (lane >> 3)] = static_cast<char>(s8);
  }
}

// Rows [0, seq_lens[i]) of entry i's ranges as bf16 rows row_start[i] .. of k_out / v_out.  A thread makes 8 dims
// (16 bytes of output).  The product nibble * e4m3 is exact, the product with the head's scale is rounded to fp32 and
// the result once to bf16.
template <bool INT4>
__global__ void __launch_bounds__(kThreads) dequant_kernel(KvDequantParams p, int rows_per_cta) {
  const int i = blockIdx.x;
  const int n_rows = min(p.seq_lens[i], p.max_seq_len);   // the caller made room for no more
  const int t0 = blockIdx.y * rows_per_cta;
  if (t0 >= n_rows) return;
  const int t1 = min(t0 + rows_per_cta, n_rows);
  const int64_t slot = p.slot_ids[i];
  const int64_t out0 = p.row_start[i];
  const int vec_per_row = p.kvh * (kHeadDim / 8);
  const int64_t row_bytes = INT4 ? int4_row_bytes(p.kvh) : p.kvh * kHeadDim;
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    uint4 *out = static_cast<uint4 *>(kv ? p.v_out : p.k_out);
    if (!out) continue;
    const char *base = reinterpret_cast<const char *>(kv ? p.v_table[slot] : p.k_table[slot]);
    const float *scale = kv ? p.v_scale : p.k_scale;
    for (int idx = threadIdx.x; idx < (t1 - t0) * vec_per_row; idx += kThreads) {
      const int t = t0 + idx / vec_per_row, v = idx % vec_per_row;
      const int head = v / (kHeadDim / 8), c8 = v % (kHeadDim / 8);   // dims 8 c8 .. 8 c8 + 7
      const char *row = base + t * row_bytes;
      const float sc = scale[head];
      float f[8];
      if constexpr (INT4) {
        const int G = c8 >> 2, r = (c8 & 3) * 2;                      // pieces r and r + 1 of group G
        const char *hp = row + int4_head_offset(p.kvh, head) + 8 * r + 2 * G;
        const uint32_t a = *reinterpret_cast<const uint16_t *>(hp), b = *reinterpret_cast<const uint16_t *>(hp + 8);
        const float s8 = e4m3_to_float(static_cast<unsigned char>(row[int4_scale_offset(p.kvh, head) + G]));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = __fmul_rn(static_cast<float>(static_cast<int>((a >> (4 * j)) & 15u) - 8) * s8, sc);
          f[4 + j] = __fmul_rn(static_cast<float>(static_cast<int>((b >> (4 * j)) & 15u) - 8) * s8, sc);
        }
      } else {
        const uint2 w = *reinterpret_cast<const uint2 *>(row + head * kHeadDim + c8 * 8);
        e4m3x4_to_float(w.x, f);
        e4m3x4_to_float(w.y, f + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __fmul_rn(f[j], sc);
      }
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
        o[j] = *reinterpret_cast<const uint32_t *>(&h);
      }
      out[(out0 + t) * vec_per_row + v] = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
}

}  // namespace

int launch_append_int4(const AppendParams &p, cudaStream_t stream) {
  if (p.batch == 0) return VT_OK;
  const bool decode = p.max_seq_len == 1;
  const int rows_per_cta = decode ? 1 : std::max(8, (p.max_seq_len + 65534) / 65535);   // grid.y holds 65 535
  const dim3 grid(p.batch, decode ? 1 : (p.max_seq_len + rows_per_cta - 1) / rows_per_cta);
  const bool vec_ok = ((reinterpret_cast<uintptr_t>(p.key) | reinterpret_cast<uintptr_t>(p.value)) & 7) == 0 &&
                      (p.key_stride % 4) == 0 && (p.value_stride % 4) == 0;
  append_int4_kernel<<<grid, kThreads, 0, stream>>>(p, rows_per_cta, vec_ok);
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

int launch_kv_dequant(const KvDequantParams &p, int kv_dtype, cudaStream_t stream) {
  const int max_seq_len = p.max_seq_len;
  if (p.batch == 0 || max_seq_len <= 0) return VT_OK;
  const int rows = std::max(16, (max_seq_len + 65534) / 65535);
  const dim3 grid(p.batch, (max_seq_len + rows - 1) / rows);
  if (kv_dtype == VT_KV_INT4)
    dequant_kernel<true><<<grid, kThreads, 0, stream>>>(p, rows);
  else
    dequant_kernel<false><<<grid, kThreads, 0, stream>>>(p, rows);
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
