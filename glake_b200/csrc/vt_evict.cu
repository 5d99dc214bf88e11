// Eviction of cached rows by accumulated attention weight.
//
// Per (sequence, kv head) with n > budget rows: the first `sink` and the last `recent` rows stay, and of the rest the
// budget - sink - recent heaviest, equal weights going to the lower row.  The kept rows keep their order and move to
// the front of the range, so that the tail of the range stays the recent window and the next eviction needs no
// record of positions.
//
// select_kernel: one CTA per (sequence, kv head).  Radix selection (11 + 11 + 10 bits of the order-preserving integer
//   of the weight) finds the key of the last row that fits and how many rows with that key do; then every warp walks
//   its run of rows once, ranks by ballots and writes the kept row numbers and the compacted weights.  Weights are
//   held in shared memory when they fit (45 056 rows), so memory sees them once; also what makes scores_out == scores safe.
// move_kernel: a chunk of kept rows per CTA, through registers.  In place, a destination row may still be the source
//   of an earlier destination (kept[i] >= i).  Chunks draw their number from a counter, load all their rows,
//   raise a flag, and store after the flags of the earlier chunks of the same head whose sources reach into their
//   destination.  A chunk only ever waits for chunks with lower numbers, which have started and raise their flag
//   without waiting, so the order of the blocks does not matter; the wait is bounded all the same.
// Roofline: HBM.  4 bytes of weight read and written per row, kept rows read and written once.
// 16 sequences of 7k-32k rows, 8 kv heads, to 8192 rows a head (bf16): selection 33 us, bound by its passes over shared
// memory (128 CTAs), move 175 us (6.1 TB/s).  The move launched while the selection still ran made the whole slower (245
// against 211 us): its waiting CTAs take the place of the selection's.
#include <algorithm>

#include "../../include/vtensor.h"
#include "vt_device.cuh"
#include "vt_int4.cuh"
#include "vt_kernels.h"

namespace vt {
namespace {

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelSmemRows = 45056;   // with the ballots and the histogram: 201 KB
constexpr int kMoveThreads = 256;
constexpr uint32_t kNoKey = 0xffffffffu;

// Order-preserving unsigned key; -0 equals +0, NaN counts as -inf.
__device__ __forceinline__ uint32_t weight_key(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

constexpr int kSelList = 2048;

struct SelectState {
  int hist[2048];
  uint32_t list[kSelList];   // keys that share the first digit's prefix, when they are few
  int listed;
  int warp_sum[kSelWarps];
  int warp_gt[kSelWarps], warp_eq[kSelWarps];
  uint32_t prefix;   // digits fixed so far
  int want;          // rows still to take among those with this prefix
};

// Digit of the want-th largest element in hist[bins]; leaves st.want = how many to take from that digit's rows.
__device__ __forceinline__ void pick_digit(SelectState &st, int bins, int shift) {
  // thread t owns bins - 1 - t, ... descending: 2 bins per thread for 2048, 1 for 1024
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = bins / kSelThreads;
  int mine[2] = {0, 0}, sum = 0;
  for (int i = 0; i < per; ++i) {
    mine[i] = st.hist[bins - 1 - (tid * per + i)];
    sum += mine[i];
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) st.warp_sum[warp] = inc;
  __syncthreads();
  const int want = st.want;
  int before = 0;
  for (int w = 0; w < warp; ++w) before += st.warp_sum[w];
  int above = before + inc - sum;   // rows in higher digits than this thread's
  __syncthreads();
  for (int i = 0; i < per; ++i) {
    if (above < want && want <= above + mine[i]) {
      st.prefix |= static_cast<uint32_t>(bins - 1 - (tid * per + i)) << shift;
      st.want = want - above;
    }
    above += mine[i];
  }
  __syncthreads();
}

// The rows to keep of one (sequence, head) with n > budget.  HELD: the weights are in shared memory (`held`, loaded here);
// otherwise every pass reads them from memory again.  ballots: two words per 32 rows (above the limit | equal to it).
template <bool HELD>
__device__ __forceinline__ void select_rows(const EvictParams &p, SelectState &st, float *held, uint2 *ballots, const float *src, float *dst,
                                            int32_t *kept, int n) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int lo = p.sink, hi = n - p.recent;   // rows that may go
  const int need = p.budget - p.sink - p.recent;
  const auto weight = [&](int t) { return HELD ? held[t] : __ldcg(src + t); };
  for (int i = tid; i < 2048; i += kSelThreads) st.hist[i] = 0;
  if (tid == 0) { st.prefix = 0; st.want = need; st.listed = 0; }
  __syncthreads();
  // the weights come in and the first digit (sign, exponent, two bits) is counted on the way
#pragma unroll 4
  for (int t = tid; t < n; t += kSelThreads) {
    const float x = __ldcg(src + t);
    if (HELD) held[t] = x;
    if (t >= lo && t < hi) atomicAdd(&st.hist[weight_key(x) >> 21], 1);
  }
  __syncthreads();
  uint32_t limit = kNoKey;   // rows with a key above stay; `ties` of those equal to it
  int ties = 0;
  if (need > 0) {
    pick_digit(st, 2048, 21);
    for (int i = tid; i < 2048; i += kSelThreads) st.hist[i] = 0;
    const uint32_t first = st.prefix;
    __syncthreads();
#pragma unroll 4
    for (int t = lo + tid; t < hi; t += kSelThreads) {
      const uint32_t key = weight_key(weight(t));
      if ((key & 0xffe00000u) == first) {
        atomicAdd(&st.hist[(key >> 10) & 2047u], 1);
        const int at = atomicAdd(&st.listed, 1);
        if (at < kSelList) st.list[at] = key;
      }
    }
    __syncthreads();
    pick_digit(st, 2048, 10);
    for (int i = tid; i < 1024; i += kSelThreads) st.hist[i] = 0;
    const uint32_t second = st.prefix;
    const int listed = st.listed;
    __syncthreads();
    if (listed <= kSelList) {
      for (int i = tid; i < listed; i += kSelThreads)
        if ((st.list[i] & 0xfffffc00u) == second) atomicAdd(&st.hist[st.list[i] & 1023u], 1);
    } else {
#pragma unroll 4
      for (int t = lo + tid; t < hi; t += kSelThreads) {
        const uint32_t key = weight_key(weight(t));
        if ((key & 0xfffffc00u) == second) atomicAdd(&st.hist[key & 1023u], 1);
      }
    }
    __syncthreads();
    pick_digit(st, 1024, 0);
    limit = st.prefix;
    ties = st.want;
  }
  // Every warp owns a run of rows: count by ballots (kept in shared memory while there is room), scan over the warps, write.
  const int run = (n + kSelThreads - 1) / kSelThreads * 32;
  const int r0 = min(warp * run, n), r1 = min(r0 + run, n);
  const auto rank = [&](int t) {
    bool stays = false, tie = false;
    if (t < r1) {
      if (t < lo || t >= hi) {
        stays = true;
      } else if (need > 0) {
        const uint32_t key = weight_key(weight(t));
        stays = key > limit;
        tie = key == limit;
      }
    }
    return make_uint2(__ballot_sync(0xffffffffu, stays), __ballot_sync(0xffffffffu, tie));
  };
  int gt = 0, eq = 0;
#pragma unroll 4
  for (int t = r0; t < r1; t += 32) {
    const uint2 b = rank(t + lane);
    if (HELD && lane == 0) ballots[t >> 5] = b;
    gt += __popc(b.x);
    eq += __popc(b.y);
  }
  if (lane == 0) { st.warp_gt[warp] = gt; st.warp_eq[warp] = eq; }
  __syncthreads();
  gt = eq = 0;
  for (int w = 0; w < warp; ++w) { gt += st.warp_gt[w]; eq += st.warp_eq[w]; }
  const bool write_now = HELD || src != dst;
  const unsigned below = (1u << lane) - 1u;
#pragma unroll 4
  for (int t = r0; t < r1; t += 32) {
    const uint2 b = HELD ? ballots[t >> 5] : rank(t + lane);
    const bool s = (b.x >> lane) & 1u, e = (b.y >> lane) & 1u;
    const int my_eq = eq + __popc(b.y & below);
    if (s || (e && my_eq < ties)) {
      const int at = gt + __popc(b.x & below) + min(my_eq, ties);
      kept[at] = t + lane;
      if (write_now) dst[at] = weight(t + lane);
    }
    gt += __popc(b.x);
    eq += __popc(b.y);
  }
  __syncthreads();
  if (!write_now) {
    // Too long for shared memory and in place: 1024 kept weights at a time, in order; a weight's destination is
    // never behind its source, so what a later step reads has not been written.
    for (int t0 = 0; t0 < p.budget; t0 += kSelThreads) {
      const int t = t0 + tid;
      const float x = t < p.budget ? __ldcg(src + kept[t]) : 0.f;
      __syncthreads();
      if (t < p.budget) dst[t] = x;
      __syncthreads();
    }
  }
  for (int t = p.budget + tid; t < n; t += kSelThreads) dst[t] = 0.f;
}

__global__ void __launch_bounds__(kSelThreads) select_kernel(EvictParams p) {
  extern __shared__ __align__(16) float held[];
  __shared__ SelectState st;
  const int b = blockIdx.x / p.kvh, head = blockIdx.x % p.kvh, tid = threadIdx.x;
  const int n = min(max(p.seq_lens[b], 0), p.max_seq_len);
  const int64_t row0 = p.slot_ids[b] * p.slot_stride + head * p.head_stride;
  const float *src = p.scores + row0;
  float *dst = p.scores_out + row0;
  int32_t *kept = p.kept + static_cast<int64_t>(blockIdx.x) * p.budget;
  for (int c = tid; c < p.chunks; c += kSelThreads) p.flags[static_cast<int64_t>(blockIdx.x) * p.chunks + c] = 0;
  if (blockIdx.x == 0 && tid == 0) *p.ticket = 0;
  if (n <= p.budget) {   // everything stays
    for (int t = tid; t < p.budget; t += kSelThreads) kept[t] = t < n ? t : -1;
    if (src != dst)
      for (int t = tid; t < n; t += kSelThreads) dst[t] = src[t];
    return;
  }
  uint2 *ballots = reinterpret_cast<uint2 *>(held + (p.held_rows + 3) / 4 * 4);
  if (n <= p.held_rows)
    select_rows<true>(p, st, held, ballots, src, dst, kept, n);
  else
    select_rows<false>(p, st, held, ballots, src, dst, kept, n);
}

// VEC 16-byte vectors of a row and head: 16 bf16, 8 fp8, 4 for the 4-bit cache, which has a 4-byte scale word beside.
template <int VEC, bool INT4>
__global__ void __launch_bounds__(kMoveThreads) move_kernel(EvictParams p) {
  constexpr int ROWS = kMoveRegs * kMoveThreads / VEC;   // rows per chunk
  constexpr int PER = kMoveThreads / VEC;                // rows of one register
  __shared__ int ticket_s;
  if (threadIdx.x == 0) ticket_s = atomicAdd(p.ticket, 1);
  __syncthreads();
  const int heads = p.batch * p.kvh;
  const int chunk = ticket_s / heads, bh = ticket_s % heads;
  const int b = bh / p.kvh, head = bh % p.kvh;
  const int n = min(max(p.seq_lens[b], 0), p.max_seq_len);
  if (n <= p.budget) return;   // nothing of this head moves, and nobody waits for it
  const int32_t *kept = p.kept + static_cast<int64_t>(bh) * p.budget;
  const int c0 = chunk * ROWS, rows = min(ROWS, p.budget - c0);
  const int64_t slot = p.slot_ids[b];
  char *const base[2] = {reinterpret_cast<char *>(p.k_table[slot]), reinterpret_cast<char *>(p.v_table[slot])};
  const int64_t row_bytes = INT4 ? int4_row_bytes(p.kvh) : p.kvh * (VEC * 16);
  const int64_t head_off = INT4 ? int4_head_offset(p.kvh, head) : head * (VEC * 16);
  const int vec = threadIdx.x % VEC, r0 = threadIdx.x / VEC;
  // last source of an earlier chunk: this thread's chunk to look at, in flight with the rows
  const int end0 = static_cast<int>(threadIdx.x) < chunk ? kept[threadIdx.x * ROWS + ROWS - 1] : -1;
  uint4 x[2][kMoveRegs];
  uint32_t word[2] = {0u, 0u};
  bool moves[kMoveRegs];
  bool word_moves = false;
  uint32_t seen = 0u;   // depends on every word loaded
#pragma unroll
  for (int i = 0; i < kMoveRegs; ++i) {
    const int r = i * PER + r0;
    const int from = r < rows ? kept[c0 + r] : 0;
    moves[i] = r < rows && from != c0 + r;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
      x[kv][i] = make_uint4(0, 0, 0, 0);
      if (moves[i]) x[kv][i] = __ldcg(reinterpret_cast<const uint4 *>(base[kv] + from * row_bytes + head_off) + vec);
    }
  }
  if constexpr (INT4) {
    static_assert(ROWS == kMoveThreads, "one scale word per thread");
    const int from = threadIdx.x < rows ? kept[c0 + threadIdx.x] : 0;
    word_moves = threadIdx.x < rows && from != c0 + static_cast<int>(threadIdx.x);
    if (word_moves) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        word[kv] = __ldcg(reinterpret_cast<const uint32_t *>(base[kv] + from * row_bytes + int4_scale_offset(p.kvh, head)));
      seen = word[0] ^ word[1];
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveRegs; ++i)
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) seen ^= x[kv][i].x ^ x[kv][i].y ^ x[kv][i].z ^ x[kv][i].w;
  // The barrier's operand needs every loaded word, so behind it all rows of the chunk have arrived; a fence in every
  // thread says the same and cost a fifth of the kernel's time.
  int *flags = p.flags + static_cast<int64_t>(bh) * p.chunks;
  __syncthreads_or(seen == 0x9e3779b9u);
  if (threadIdx.x == 0) asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flags + chunk), "r"(1) : "memory");
  // earlier chunks whose last source is not in front of this chunk's destination
  bool ok = true;
  for (int c = threadIdx.x; c < chunk && ok; c += kMoveThreads) {
    const int end = c == static_cast<int>(threadIdx.x) ? end0 : kept[c * ROWS + ROWS - 1];
    if (end < c0) continue;
    unsigned long long t0 = 0;
    for (uint32_t it = 0;; ++it) {
      uint32_t f;
      asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(f) : "l"(flags + c) : "memory");
      if (f) break;
      if (it == 0) t0 = global_timer_ns();
      else if (global_timer_ns() - t0 > kWaitLimitNs || it > kWaitLimit) { ok = false; break; }
    }
  }
  if (!ok) atomicExch(p.status, kKernelErrMagic);
  if (__syncthreads_or(!ok)) return;
#pragma unroll
  for (int i = 0; i < kMoveRegs; ++i)
    if (moves[i]) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        reinterpret_cast<uint4 *>(base[kv] + (c0 + i * PER + r0) * row_bytes + head_off)[vec] = x[kv][i];
    }
  if constexpr (INT4) {
    if (word_moves) {
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        *reinterpret_cast<uint32_t *>(base[kv] + (c0 + static_cast<int>(threadIdx.x)) * row_bytes +
                                      int4_scale_offset(p.kvh, head)) = word[kv];
    }
  }
}

}  // namespace

int evict_chunk_rows(int kv_dtype) {
  return kMoveRegs * kMoveThreads / (kv_dtype == VT_KV_BF16 ? 16 : kv_dtype == VT_KV_FP8_E4M3 ? 8 : 4);
}

int launch_evict(const EvictParams &p_in, int kv_dtype, cudaStream_t stream) {
  EvictParams p = p_in;
  p.held_rows = std::min(p.max_seq_len, kSelSmemRows);
  static SmemOptIn opt_in;
  const int smem = (p.held_rows + 3) / 4 * 16 + (p.held_rows / 32 + 1) * static_cast<int>(sizeof(uint2));
  if (!opt_in.ensure(select_kernel, smem)) return VT_ERR_CUDA;
  const int heads = p.batch * p.kvh;
  select_kernel<<<heads, kSelThreads, smem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return VT_ERR_CUDA;
  const int grid = heads * p.chunks;
  if (kv_dtype == VT_KV_BF16)
    move_kernel<16, false><<<grid, kMoveThreads, 0, stream>>>(p);
  else if (kv_dtype == VT_KV_FP8_E4M3)
    move_kernel<8, false><<<grid, kMoveThreads, 0, stream>>>(p);
  else
    move_kernel<4, true><<<grid, kMoveThreads, 0, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? VT_OK : VT_ERR_CUDA;
}

}  // namespace vt
