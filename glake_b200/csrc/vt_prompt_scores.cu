// Attention weights of a prompt's last queries, summed per cached row: what decides which rows of a prompt are kept.
//   scores[slot, kv head, t] += sum over the last w = min(window, q_len) queries i and the kv head's q heads of
//                               softmax_t(scale q_i K^T)[t],   query i seeing rows t <= n - w + i
//
// The rows of the problem are the w x g (query, q head) pairs of one kv head; V is not read.  A row's weights need its
// maximum and sum over all keys first, so the logits are computed twice: keeping them would move 4 bytes per (row, key)
// each way, more time than the second product takes.
//   stats_kernel   per (entry, kv head, run of keys): running (max, sum) of every row over the run
//   columns_kernel the same run again: combines the runs' statistics, adds exp2(s - max) / sum over the rows
// A CTA holds a tile of 64 keys in shared memory; warp w takes row blocks w, w + 8, ... of 16 rows, with Q fragments
// read from global memory (L1) per block.  Bound: tensor pipe, 2 x 2 x 128 flop per (row, key).
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_kernels.h"
#include "vt_mma.cuh"

namespace vt {
namespace {

constexpr int kPsThreads = 256;
constexpr int kPsWarps = kPsThreads / 32;
constexpr int kPsKeys = 64;                   // keys per tile
constexpr int kPsPitch = 256 + 16;            // bytes; ldmatrix rows fall into distinct banks

// Loads 64 rows of a head into shared memory (rows past the end as zeros).
__device__ __forceinline__ void load_keys(unsigned char *tile, const char *base, int64_t row_bytes, int t0, int n) {
  for (int i = threadIdx.x; i < kPsKeys * 16; i += kPsThreads) {
    const int r = i >> 4, c = i & 15;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (t0 + r < n) v = __ldg(reinterpret_cast<const uint4 *>(base + (t0 + r) * row_bytes) + c);
    *reinterpret_cast<uint4 *>(tile + r * kPsPitch + c * 16) = v;
  }
}

struct RowBlock {
  uint32_t q[8][4];   // A fragments: rows r4, r4 + 8 of the block
  int last[2];        // last key of the two rows; -1: no such row
};

// Rows are (query i, q head j) = i * g + j of this kv head.
__device__ __forceinline__ void load_rows(RowBlock &rb, const PromptScoreParams &p, int b, int head, int block, int n,
                                          int w, int lane) {
  const int g = p.h / p.kvh, r4 = lane >> 2, c4 = lane & 3;
  const __nv_bfloat16 *src[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int row = block * 16 + r4 + 8 * e;
    const bool there = row < w * g;
    const int i = there ? row / g : 0, j = there ? row % g : 0;
    rb.last[e] = there ? n - w + i : -1;
    src[e] = static_cast<const __nv_bfloat16 *>(p.q) +
             (static_cast<int64_t>(p.q_start[b]) + p.q_lens[b] - w + i) * p.q_stride + (head * g + j) * kHeadDim;
  }
#pragma unroll
  for (int ks = 0; ks < 8; ++ks) {
#pragma unroll
    for (int k = 0; k < 4; ++k)   // a0: row r4, k 2 c4; a1: row r4 + 8; a2, a3: k + 8
      rb.q[ks][k] = __ldg(reinterpret_cast<const uint32_t *>(src[k & 1] + ks * 16 + 2 * c4 + (k >> 1) * 8));
  }
}

// Logits (log2 domain, masked to -inf) of the block's rows against the 64 keys: s[nb][..] = key 8 nb + 2 c4 + {0, 1}.
__device__ __forceinline__ void block_logits(float (&s)[8][4], const RowBlock &rb, uint32_t tile, int t0, float sl2, int lane) {
  const int c4 = lane & 3;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
  const uint32_t at = tile + (lane & 7) * kPsPitch + (lane >> 3) * 16;
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) {
#pragma unroll
    for (int ks = 0; ks < 8; ks += 2) {   // one ldmatrix brings the B fragments of two k steps
      uint32_t k[4];
      ldmatrix_x4(at + nb * 8 * kPsPitch + ks * 32, k);
      mma_bf16(s[nb], rb.q[ks], k[0], k[1]);
      mma_bf16(s[nb], rb.q[ks + 1], k[2], k[3]);
    }
  }
#pragma unroll
  for (int nb = 0; nb < 8; ++nb) {
    const int t = t0 + 8 * nb + 2 * c4;
    s[nb][0] = t <= rb.last[0] ? s[nb][0] * sl2 : -INFINITY;
    s[nb][1] = t + 1 <= rb.last[0] ? s[nb][1] * sl2 : -INFINITY;
    s[nb][2] = t <= rb.last[1] ? s[nb][2] * sl2 : -INFINITY;
    s[nb][3] = t + 1 <= rb.last[1] ? s[nb][3] * sl2 : -INFINITY;
  }
}

struct Run {
  int b, head, n, w, t_begin, t_end;
  const char *base;
  int64_t row_bytes;
};
__device__ __forceinline__ bool locate_run(const PromptScoreParams &p, Run &r) {
  r.b = blockIdx.x / p.kvh;
  r.head = blockIdx.x % p.kvh;
  r.n = min(max(p.seq_lens[r.b], 0), p.max_seq_len);
  r.w = min(min(p.window, p.q_lens[r.b]), r.n);
  r.t_begin = blockIdx.y * p.run_keys;
  r.t_end = min(r.t_begin + p.run_keys, r.n);
  if (r.w <= 0 || r.t_begin >= r.t_end) return false;
  r.row_bytes = static_cast<int64_t>(p.kvh) * kHeadDim * 2;
  r.base = reinterpret_cast<const char *>(p.k_table[(p.range_ids ? p.range_ids : p.slot_ids)[r.b]]) + r.head * kHeadDim * 2;
  return true;
}

__global__ void __launch_bounds__(kPsThreads) stats_kernel(PromptScoreParams p) {
  __shared__ __align__(16) unsigned char tile[kPsKeys * kPsPitch];
  Run r;
  if (!locate_run(p, r)) return;
  const int g = p.h / p.kvh, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r4 = lane >> 2;
  const int blocks = (r.w * g + 15) / 16;
  const float sl2 = p.scale * 1.4426950408889634f;
  float2 *ml = p.ml + (static_cast<int64_t>(blockIdx.x) * p.runs + blockIdx.y) * p.rows;
  // row blocks in rounds of one per warp, the run's keys streamed once per round
  for (int b0 = 0; b0 < blocks; b0 += kPsWarps) {
    const int block = b0 + warp;
    RowBlock rb;
    load_rows(rb, p, r.b, r.head, block, r.n, r.w, lane);
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    for (int t0 = r.t_begin; t0 < r.t_end; t0 += kPsKeys) {
      __syncthreads();
      load_keys(tile, r.base, r.row_bytes, t0, r.t_end);
      __syncthreads();
      if (block >= blocks) continue;
      float s[8][4];
      block_logits(s, rb, smem_u32(tile), t0, sl2, lane);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = m[e];
#pragma unroll
        for (int nb = 0; nb < 8; ++nb) mx = fmaxf(mx, fmaxf(s[nb][2 * e], s[nb][2 * e + 1]));
        if (mx > -INFINITY) {   // per lane: the four lanes of a row are joined at the end
          float sum = l[e] * exp2f(m[e] - mx);
#pragma unroll
          for (int nb = 0; nb < 8; ++nb) sum += exp2f(s[nb][2 * e] - mx) + exp2f(s[nb][2 * e + 1] - mx);
          l[e] = sum;
          m[e] = mx;
        }
      }
    }
    if (block < blocks) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mx = m[e];
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        float sum = mx > -INFINITY ? l[e] * exp2f(m[e] - mx) : 0.f;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const int row = block * 16 + r4 + 8 * e;
        if ((lane & 3) == 0 && row < r.w * g) ml[row] = make_float2(mx, sum);
      }
    }
  }
}

__global__ void __launch_bounds__(kPsThreads) columns_kernel(PromptScoreParams p) {
  __shared__ __align__(16) unsigned char tile[kPsKeys * kPsPitch];
  __shared__ float part[kPsWarps][kPsKeys];
  extern __shared__ float2 final_ml[];   // (max, 1 / sum) of every row
  Run r;
  if (!locate_run(p, r)) return;
  const int g = p.h / p.kvh, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r4 = lane >> 2, c4 = lane & 3;
  const int rows = r.w * g, blocks = (rows + 15) / 16;
  const float sl2 = p.scale * 1.4426950408889634f;
  const int runs = (r.n + p.run_keys - 1) / p.run_keys;
  const float2 *ml = p.ml + static_cast<int64_t>(blockIdx.x) * p.runs * p.rows;
  for (int row = threadIdx.x; row < blocks * 16; row += kPsThreads) {
    float m = -INFINITY, l = 0.f;
    if (row < rows) {
      for (int i = 0; i < runs; ++i) m = fmaxf(m, ml[static_cast<int64_t>(i) * p.rows + row].x);
      for (int i = 0; i < runs; ++i) {
        const float2 x = ml[static_cast<int64_t>(i) * p.rows + row];
        if (x.y > 0.f) l = fmaf(x.y, exp2f(x.x - m), l);
      }
    }
    final_ml[row] = row < rows ? make_float2(m, 1.f / l) : make_float2(0.f, 0.f);
  }
  float *dst = p.scores + p.slot_ids[r.b] * p.slot_stride + r.head * p.head_stride;
  const bool one_round = blocks <= kPsWarps;
  RowBlock rb;
  if (one_round) load_rows(rb, p, r.b, r.head, warp, r.n, r.w, lane);
  for (int t0 = r.t_begin; t0 < r.t_end; t0 += kPsKeys) {
    __syncthreads();
    load_keys(tile, r.base, r.row_bytes, t0, r.t_end);
    __syncthreads();
    float col[8][2];
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) col[nb][0] = col[nb][1] = 0.f;
    for (int block = warp; block < blocks; block += kPsWarps) {
      if (!one_round) load_rows(rb, p, r.b, r.head, block, r.n, r.w, lane);
      float s[8][4];
      block_logits(s, rb, smem_u32(tile), t0, sl2, lane);
      const float2 a = final_ml[block * 16 + r4], c = final_ml[block * 16 + r4 + 8];
#pragma unroll
      for (int nb = 0; nb < 8; ++nb) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          col[nb][e] = fmaf(exp2f(s[nb][e] - a.x), a.y, col[nb][e]);
          col[nb][e] = fmaf(exp2f(s[nb][2 + e] - c.x), c.y, col[nb][e]);
        }
      }
    }
#pragma unroll
    for (int nb = 0; nb < 8; ++nb) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float x = col[nb][e];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (r4 == 0) part[warp][8 * nb + 2 * c4 + e] = x;
      }
    }
    __syncthreads();
    if (threadIdx.x < kPsKeys && t0 + static_cast<int>(threadIdx.x) < r.t_end) {
      float x = 0.f;
#pragma unroll
      for (int k = 0; k < kPsWarps; ++k) x += part[k][threadIdx.x];
      atomicAdd(dst + t0 + threadIdx.x, x);   // one addition per row when the slots of a call differ
    }
  }
}

}  // namespace

// Keys per run: enough CTAs for two waves of resident ones, whole tiles, at most 256 runs.
int prompt_run_keys(int batch, int kvh, int max_seq_len) {
  const int pairs = std::max(1, batch * kvh);
  const int runs = std::min(256, std::max(1, (4 * kFlatSms + pairs - 1) / pairs));
  const int keys = (std::max(max_seq_len, 1) + runs - 1) / runs;
  return (keys + kPsKeys - 1) / kPsKeys * kPsKeys;
}

int launch_prompt_scores(const PromptScoreParams &p, cudaStream_t stream) {
  const dim3 grid(p.batch * p.kvh, p.runs);
  const int smem = (p.rows + 15) / 16 * 16 * static_cast<int>(sizeof(float2));
  static SmemOptIn opt_in;
  if (!opt_in.ensure(columns_kernel, smem)) return VT_ERR_CUDA;
  stats_kernel<<<grid, kPsThreads, 0, stream>>>(p);
  columns_kernel<<<grid, kPsThreads, smem, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
