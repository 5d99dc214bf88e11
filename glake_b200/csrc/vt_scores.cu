// Accumulated attention weights: what a cached row has received from the queries so far.
//   scores[slot, kv head, t] += sum over the kv head's q heads of softmax(scale q K^T)[t]
//
// Decode (accumulate_kernel): the attention kernels write every logit they compute and the (max, sum) of every
// (entry, q head); this kernel turns them into weights.  The weight of a row needs the sum over ALL rows, which no CTA
// of the attention launch knows while it holds the logits, so a second pass is needed either way; re-reading K for it
// would cost 256 bytes per (row, kv head), the logits cost 8 g.  Bytes: 4 g + 8 per (row, kv head).
// Measured, whole call: bf16, 8 sequences of 512-2048 rows, 32/32 heads 41 us; 32 of 4k-16k, 8/1 heads 49; fp8, 64 of
// 2k-8k, 32/8 heads 158, of which the accumulation 6, 9 and 13 (it starts while the attention kernel drains).
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_kernels.h"

namespace vt {
namespace {

constexpr int kAccThreads = 256;
constexpr int kAccTokens = 4;   // tokens per thread

// grid: (entry x kv head, blocks of 1024 tokens)
template <int G>
__global__ void __launch_bounds__(kAccThreads) accumulate_kernel(ScoreParams p) {
  pdl_wait_prior_grid();   // the attention kernel in front: everything below is its output or follows it
  const int b = blockIdx.x / p.kvh, head = blockIdx.x % p.kvh;
  const int len = min(p.seq_lens[b], p.logit_rows);
  const int t0 = blockIdx.y * kAccThreads * kAccTokens + threadIdx.x;
  if (t0 >= len) return;
  const float *lg = p.logits + (static_cast<size_t>(b) * p.kvh + head) * p.logit_rows * G;
  float *dst = p.scores + p.slot_ids[b] * p.slot_stride + head * p.head_stride;
  float m[G], inv[G];
#pragma unroll
  for (int j = 0; j < G; ++j) {
    const float2 s = *reinterpret_cast<const float2 *>(p.ml + 2 * ((static_cast<size_t>(b) * p.kvh + head) * G + j));
    m[j] = s.x;
    inv[j] = 1.f / s.y;
  }
#pragma unroll
  for (int i = 0; i < kAccTokens; ++i) {
    const int t = t0 + i * kAccThreads;
    if (t < len) {
      float x[G], w = 0.f;
      const float *src = lg + static_cast<size_t>(t) * G;
      if constexpr (G >= 4) {
#pragma unroll
        for (int j = 0; j < G; j += 4) *reinterpret_cast<float4 *>(x + j) = __ldcs(reinterpret_cast<const float4 *>(src + j));
      } else if constexpr (G == 2) {
        *reinterpret_cast<float2 *>(x) = __ldcs(reinterpret_cast<const float2 *>(src));
      } else {
        x[0] = __ldcs(src);
      }
#pragma unroll
      for (int j = 0; j < G; ++j) w = fmaf(exp2f(x[j] - m[j]), inv[j], w);
      // one addition per row and call when the slots of a call differ; a slot named twice still sums up
      atomicAdd(dst + t, w);
    }
  }
}

}  // namespace

int launch_accumulate(const ScoreParams &p, int g, int max_seq_len, cudaStream_t stream) {
  const dim3 grid(p.batch * p.kvh, (max_seq_len + kAccThreads * kAccTokens - 1) / (kAccThreads * kAccTokens));
  bool ok;
  switch (g) {
    case 1: ok = launch_dependent(accumulate_kernel<1>, grid, kAccThreads, 0, stream, p); break;
    case 2: ok = launch_dependent(accumulate_kernel<2>, grid, kAccThreads, 0, stream, p); break;
    case 4: ok = launch_dependent(accumulate_kernel<4>, grid, kAccThreads, 0, stream, p); break;
    case 8: ok = launch_dependent(accumulate_kernel<8>, grid, kAccThreads, 0, stream, p); break;
    case 16: ok = launch_dependent(accumulate_kernel<16>, grid, kAccThreads, 0, stream, p); break;
    default: return VT_ERR_UNSUPPORTED;
  }
  return ok ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
