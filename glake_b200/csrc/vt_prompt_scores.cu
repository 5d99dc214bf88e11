// Attention weights of a prompt's last queries, summed per cached row: what decides which rows of a prompt are kept.
//   scores[slot, kv head, t] += sum over the last w = min(window, q_len) queries i and the kv head's q heads of
//                               softmax_t(scale q_i K^T)[t],   query i seeing rows t <= n - w + i
//
// The rows of the problem are the w x g (query, q head) pairs of one kv head, in blocks of 128; V is not read.  A row's
// weights need its maximum and sum over all keys first, so the logits are computed twice: keeping them would move 4
// bytes per (row, key) each way, more time than the second product takes.
//   pass 1   D = Q K^T, TMEM lane = row: running (max, sum) of every row over the CTA's run of keys, in one thread each
//   pass 2   D = K Q^T, TMEM lane = key: sum over the rows of exp2(s - (max + log2 sum)), again in one thread
// so neither pass needs a reduction across lanes.  One CTA of eight warps per (entry, kv head, run of keys); a tile is 128
// keys, fetched with cp.async into the 128-byte swizzle, two stages; one thread issues the eight tcgen05.mma of a tile into
// one of two 128-column accumulators, which warps 0-3 and 4-7 read (half the columns each) while the next tile multiplies.
// Bound: the exponentials, one per (row, key) and pass (16 per clock and SM); 96 KB and 256 TMEM columns, two CTAs per SM.
// 4 x 16384 keys, 8 kv heads, 128 rows each: 88 us (44 a pass; the exponential unit 42 % busy); the same two passes on
// mma.sync with shuffles: 366 us.  A tile takes 2.7 us whatever the order of loads, products and arithmetic: refilling a
// stage before the tile's arithmetic 88.7, multiplying the next tile under it 86.3, sixteen warps a CTA 90.9.
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_kernels.h"
#include "vt_umma.cuh"

namespace vt {
namespace {

constexpr int kPsThreads = 256;
constexpr int kPsKeys = 128;                    // keys per tile
constexpr int kPsRows = 128;                    // rows per block
constexpr int kPsSlab = 128 * 128;              // 64 dims of 128 rows
constexpr int kPsRunKeys = 1024;                // most keys per run: their sums are kept in shared memory
constexpr int kPsStages = 2;
constexpr int kPsSmem = 1024 + 2 * kPsSlab + kPsStages * 2 * kPsSlab + kPsRows * 8 + 2 * kPsRunKeys * 4;
constexpr uint32_t kPsCols = 256;

__device__ __forceinline__ void cp_async16_fill(uint32_t dst, const void *src, bool there) {   // zeros when not there
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}

template <int PASS>
__global__ void __launch_bounds__(kPsThreads, 2) prompt_scores_kernel(PromptScoreParams p) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t base_s = (smem_u32(smem_raw) + 1023u) & ~1023u;
  unsigned char *sm = smem_raw + (base_s - smem_u32(smem_raw));
  const uint32_t q_s = base_s, k_s = q_s + 2 * kPsSlab;
  float2 *half_ml = reinterpret_cast<float2 *>(sm + 2 * kPsSlab + kPsStages * 2 * kPsSlab);   // pass 1: of warps 4-7
  float *ref = reinterpret_cast<float *>(half_ml);                                            // pass 2: max + log2 sum per row
  float *sums = reinterpret_cast<float *>(half_ml + kPsRows);                                 // pass 2: [2][run keys]
  __shared__ __align__(8) uint64_t bars[2];
  __shared__ uint32_t tmem_slot;
  const uint32_t bar = smem_u32(bars);

  const int b = blockIdx.x / p.kvh, head = blockIdx.x % p.kvh;
  const int n = min(max(p.seq_lens[b], 0), p.max_seq_len);
  const int q_len = p.q_lens[b], w = min(min(p.window, q_len), n);
  const int t_begin = blockIdx.y * p.run_keys, t_end = min(t_begin + p.run_keys, n);
  const int g = p.h / p.kvh, rows = w * g;
  const int block0 = PASS == 1 ? blockIdx.z : 0, block1 = PASS == 1 ? block0 + 1 : (rows + kPsRows - 1) / kPsRows;
  if (w <= 0 || t_begin >= t_end || block0 * kPsRows >= rows) return;   // whole CTA: nothing allocated yet
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wg = warp >> 2, lane_row = (warp & 3) * 32 + lane;          // this thread's TMEM lane
  const int tiles = (t_end - t_begin + kPsKeys - 1) / kPsKeys;
  // the sign goes into Q; a scale of 0 stays positive, so that masked logits stay -inf
  const float sl2 = fmaxf(fabsf(p.scale) * 1.4426950408889634f, 1e-30f);
  const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
  const int64_t row_bytes = static_cast<int64_t>(p.kvh) * kHeadDim * 2;
  const char *keys = reinterpret_cast<const char *>(p.k_table[(p.range_ids ? p.range_ids : p.slot_ids)[b]]) + head * kHeadDim * 2;

  if (tid == 0) {
    mbar_init(bar, 1);
    mbar_init(bar + 8, 1);
    mbar_fence_init();
  }
  if (warp == 0) {
    tmem_alloc(smem_u32(&tmem_slot), kPsCols);
    tmem_relinquish();
  }
  if constexpr (PASS == 2)
    for (int i = tid; i < 2 * p.run_keys; i += kPsThreads) sums[i] = 0.f;
  tcgen05_fence_before();
  __syncthreads();
  tcgen05_fence_after();
  if constexpr (PASS == 1) pdl_launch_dependents();   // pass 2 sets up while the last runs finish
  const uint32_t tmem = tmem_slot, my_lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);

  const auto fetch = [&](int j) {   // tile j of the run into its stage: 128 rows of 256 bytes
    const uint32_t dst = k_s + (j & 1) * 2 * kPsSlab;
    const int part = tid & 15, t0 = t_begin + j * kPsKeys;
#pragma unroll
    for (int i = 0; i < kPsKeys * 16 / kPsThreads; ++i) {
      const int r = (tid >> 4) + i * (kPsThreads / 16);
      const bool there = t0 + r < t_end;
      cp_async16_fill(dst + (part >> 3) * kPsSlab + sw128_offset(r, part & 7), keys + (there ? t0 + r : t_begin) * row_bytes + part * 16,
                      there);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  bool ok = true;
  int done = 0;   // blocks so far
  for (int block = block0; block < block1; ++block) {
    const int row0 = block * kPsRows, block_rows = min(kPsRows, rows - row0);
    const int cols = (block_rows + 31) / 32 * 32;                       // pass 2: columns multiplied and read
    fetch(0);
    {   // Q rows of the block (zeros behind the last), and what pass 2 subtracts from their logits
      const int r = tid >> 1, half = tid & 1;
      const bool there = r < block_rows;
      const int row = there ? row0 + r : 0, i = row / g, j = row - i * g;
      const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const __nv_bfloat16 *>(p.q) +
                                                         (static_cast<int64_t>(p.q_start[b]) + q_len - w + i) * p.q_stride +
                                                         (head * g + j) * kHeadDim + half * 64);
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (there) v = __ldg(src + c);
        v.x ^= flip; v.y ^= flip; v.z ^= flip; v.w ^= flip;
        *reinterpret_cast<uint4 *>(sm + half * kPsSlab + sw128_offset(r, c)) = v;
      }
      if constexpr (PASS == 2) {
        pdl_wait_prior_grid();   // the statistics of pass 1
        float m = -INFINITY, l = 0.f;
        if (there) {   // two threads of a row share its runs
          const int runs = (n + p.run_keys - 1) / p.run_keys;
          const float2 *ml = p.ml + static_cast<int64_t>(blockIdx.x) * p.runs * p.rows + row;
#pragma unroll 4
          for (int k = half; k < runs; k += 2) {
            const float2 x = __ldcg(ml + static_cast<int64_t>(k) * p.rows);
            const float mn = fmaxf(m, x.x);
            if (x.y > 0.f) l = l * ex2_approx(m - mn) + x.y * ex2_approx(x.x - mn);
            m = x.y > 0.f ? mn : m;
          }
        }
        const float m2 = __shfl_xor_sync(0xffffffffu, m, 1), l2 = __shfl_xor_sync(0xffffffffu, l, 1);
        const float mn = fmaxf(m, m2);
        const float sum = (l > 0.f ? l * ex2_approx(m - mn) : 0.f) + (l2 > 0.f ? l2 * ex2_approx(m2 - mn) : 0.f);
        if (half == 0) ref[r] = there ? mn + log2f(sum) : INFINITY;     // a row that is not there weighs 0
      }
    }
    float m = -INFINITY, l = 0.f;                                       // pass 1
    const int row = row0 + lane_row;
    const int last = n - w + row / g;                                   // pass 1: last key of this thread's row
    const bool idle = PASS == 1 && (warp & 3) * 32 >= block_rows;       // no row in this warp's lanes
    for (int j = 0; j <= tiles; ++j) {
      if (j < tiles) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        fence_proxy_async_smem();
      }
      tcgen05_fence_before();
      __syncthreads();   // tile j is in shared memory, accumulator j & 1 has been read by everybody
      if (tid == 0 && j < tiles) {
        tcgen05_fence_after();
        const uint32_t k_tile = k_s + (j & 1) * 2 * kPsSlab;
        const uint32_t idesc = umma_idesc_bf16_f32(128, PASS == 1 ? kPsKeys : cols, false, false);
#pragma unroll
        for (int kk = 0; kk < 8; ++kk) {
          const uint32_t off = (kk >> 2) * kPsSlab + (kk & 3) * 32;
          const uint64_t dq = umma_desc_sw128(q_s + off, 0, 1024), dk = umma_desc_sw128(k_tile + off, 0, 1024);
          umma_bf16(tmem + (j & 1) * 128, PASS == 1 ? dq : dk, PASS == 1 ? dk : dq, idesc, kk > 0);
        }
        umma_commit(bar + 8 * (j & 1));
      }
      if (j > 0 && ok) {   // the product of tile j - 1; the barrier's earlier phases are those of the blocks before
        const int k = j - 1, before = (k & 1) ? done * (tiles / 2) : done * ((tiles + 1) / 2);
        ok = __all_sync(0xffffffffu, mbar_wait(bar + 8 * (k & 1), (before + (k >> 1)) & 1));
      }
      if (j + 1 < tiles) fetch(j + 1);   // into the stage that product has read
      if (j == 0 || !ok || idle) continue;
      tcgen05_fence_after();
      const int t0 = t_begin + (j - 1) * kPsKeys;
      const uint32_t acc = my_lanes + ((j - 1) & 1) * 128;
      if constexpr (PASS == 1) {
        float x[64];
        {
          uint32_t v0[32], v1[32];
          tmem_ld_32x32b_x32(acc + wg * 64, v0);
          tmem_ld_32x32b_x32(acc + wg * 64 + 32, v1);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            x[i] = __uint_as_float(v0[i]);
            x[32 + i] = __uint_as_float(v1[i]);
          }
        }
        const int c0 = t0 + wg * 64, lim = min(last, t_end - 1);
        if (c0 + 63 > lim) {
#pragma unroll
          for (int i = 0; i < 64; ++i) x[i] = c0 + i <= lim ? x[i] : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 64; i += 2) mx = max3(mx, x[i], x[i + 1]);
        mx = mx == -INFINITY ? mx : mx * sl2;
        const float mn = fmaxf(m, mx);
        if (mn > -INFINITY) {
          const uint64_t sl2_2 = f2_pack(sl2, sl2), ref2 = f2_pack(-mn, -mn);
          uint64_t s0 = f2_pack(l * ex2_approx(m - mn), 0.f), s1 = f2_pack(0.f, 0.f);
#pragma unroll
          for (int i = 0; i < 64; i += 4) {
            float a0, a1, a2, a3;
            f2_unpack(f2_fma(f2_pack(x[i], x[i + 1]), sl2_2, ref2), a0, a1);
            f2_unpack(f2_fma(f2_pack(x[i + 2], x[i + 3]), sl2_2, ref2), a2, a3);
            s0 = f2_add(s0, f2_pack(ex2_approx(a0), ex2_approx(a1)));
            s1 = f2_add(s1, f2_pack(ex2_approx(a2), ex2_approx(a3)));
          }
          float a, c;
          f2_unpack(f2_add(s0, s1), a, c);
          l = a + c;
          m = mn;
        }
      } else {
        // key t0 + lane_row; column = row of the block; rows from first_row on see the key
        const int t = t0 + lane_row;
        const int first_row = max(0, t - (n - w)) * g - row0;
        const bool ragged = t0 + kPsKeys - 1 > n - w;
        uint64_t s0 = f2_pack(0.f, 0.f), s1 = s0;
        for (int c0 = wg * 32; c0 < cols; c0 += 64) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(acc + c0, v);
          tmem_ld_wait();
          if (ragged) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = c0 + i >= first_row ? v[i] : 0xff800000u;
          }
          const uint64_t sl2_2 = f2_pack(sl2, sl2);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            const float4 r = *reinterpret_cast<const float4 *>(ref + c0 + i);
            float a0, a1, a2, a3;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sl2_2, f2_pack(-r.x, -r.y)), a0, a1);
            f2_unpack(f2_fma(f2_pack(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), sl2_2, f2_pack(-r.z, -r.w)), a2, a3);
            s0 = f2_add(s0, f2_pack(ex2_approx(a0), ex2_approx(a1)));
            s1 = f2_add(s1, f2_pack(ex2_approx(a2), ex2_approx(a3)));
          }
        }
        float a, c;
        f2_unpack(f2_add(s0, s1), a, c);
        if (t < t_end) sums[wg * p.run_keys + (t - t_begin)] += a + c;
      }
    }
    ++done;
    if constexpr (PASS == 1) {
      if (wg == 1) half_ml[lane_row] = make_float2(m, l);
      __syncthreads();
      if (wg == 0 && lane_row < block_rows) {
        const float2 o = half_ml[lane_row];
        const float mn = fmaxf(m, o.x);
        const float sum = (l > 0.f ? l * ex2_approx(m - mn) : 0.f) + (o.y > 0.f ? o.y * ex2_approx(o.x - mn) : 0.f);
        p.ml[(static_cast<int64_t>(blockIdx.x) * p.runs + blockIdx.y) * p.rows + row] = make_float2(mn, sum);
      }
    }
    __syncthreads();   // Q and the references are read no more
  }
  if constexpr (PASS == 2) {
    float *dst = p.scores + p.slot_ids[b] * p.slot_stride + head * p.head_stride;
    for (int t = t_begin + tid; t < t_end; t += kPsThreads)   // one addition per row when the slots of a call differ
      atomicAdd(dst + t, sums[t - t_begin] + sums[p.run_keys + t - t_begin]);
  }
  tcgen05_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, kPsCols);
  if (!ok && lane == 0) atomicExch(p.status, kKernelErrMagic);
}

}  // namespace

// Keys per run: the number of tiles that keeps the two resident CTAs of every SM busy in the fewest tile times, a CTA's
// start counted as one and a half.
int prompt_run_keys(int batch, int kvh, int max_seq_len) {
  const int64_t pairs = std::max<int64_t>(1, static_cast<int64_t>(batch) * kvh);
  const int tiles = (std::max(max_seq_len, 1) + kPsKeys - 1) / kPsKeys;
  int best = 1;
  double best_cost = 1e30;
  for (int t = 1; t <= kPsRunKeys / kPsKeys; ++t) {
    const int64_t ctas = pairs * ((tiles + t - 1) / t);
    const double cost = static_cast<double>((ctas + 2 * kFlatSms - 1) / (2 * kFlatSms)) * (t + 1.5);
    if (cost < best_cost) { best_cost = cost; best = t; }
  }
  return best * kPsKeys;
}

int launch_prompt_scores(const PromptScoreParams &p, cudaStream_t stream) {
  static SmemOptIn opt1, opt2;
  if (!opt1.ensure(prompt_scores_kernel<1>, kPsSmem) || !opt2.ensure(prompt_scores_kernel<2>, kPsSmem)) return VT_ERR_CUDA;
  const int blocks = (p.rows + kPsRows - 1) / kPsRows;
  prompt_scores_kernel<1><<<dim3(p.batch * p.kvh, p.runs, blocks), kPsThreads, kPsSmem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return VT_ERR_CUDA;
  return launch_dependent(prompt_scores_kernel<2>, dim3(p.batch * p.kvh, p.runs), kPsThreads, kPsSmem, stream, p) ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
