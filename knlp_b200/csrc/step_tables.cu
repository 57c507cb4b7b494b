// Tables of a serving step from the requests' lengths: query offsets, lengths after the step,
// the cache blocks the step takes from the free list, their block-table entries, and position
// and cache slot of every new token.
//
//   fresh_s  = blocks(ctx_s + new_s) - blocks(ctx_s),  blocks(n) = min(ceil(n / block_size), max_blocks)
//   table[s, blocks(ctx_s) + j] = free[head + sum_{r<s} fresh_r + j],   0 <= j < fresh_s
//   token i of request s: position ctx_s + i, slot = table[s, pos / bs] * bs + pos % bs
//
// What bounds it: latency.  A step of 32 requests moves 5 KB (3.5 us on the device); 1024 prompts
// with 1.0 Mi tokens write 17 MB (15 us, 2.6 us at the copy rate: the blocks' scans).  ONE launch
// without any communication between blocks: every block scans the lengths of all requests itself
// (8 bytes each, from L2), in chunks of kChunk, and serves the tokens and fresh table entries of
// its own share that fall into the chunk.  A token finds its request by bisection in shared
// memory; its slot comes from the free list directly when the block is fresh, so that no block
// reads a table entry that another one writes.

#include "serve.cuh"

namespace knlp {
namespace {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;
constexpr int kChunk = kThreads * kPerThread;  // requests scanned at a time
constexpr int kTokensPerBlock = 1024;
// Lengths and token sums saturate here: a corrupt length gives useless tables, but every
// prefix stays monotone and every index inside its row.
constexpr int kMost = 1 << 30;

__device__ __forceinline__ int add_most(int a, int b) { return min(a + b, kMost); }

struct StepArgs {
  const int32_t* ctx;
  const int32_t* fresh_tokens;
  int32_t* table;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* free_blocks;
  int64_t n_free;
  const int32_t* free_head;
  int n_seqs, block_size;
  int64_t n_slots;
  int32_t* query_start_loc;
  int32_t* seq_lens;
  int64_t* slot_mapping;
  int64_t* positions;
  int32_t* blocks_taken;
};

__global__ void __launch_bounds__(kThreads) step_tables_kernel(StepArgs a) {
  __shared__ int s_end[kChunk];    // tokens of the chunk's requests up to and with this one
  __shared__ int s_fresh[kChunk];  // fresh blocks, the same
  __shared__ int s_ctx[kChunk];
  __shared__ int s_warp[2][kThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bs = a.block_size;
  const int64_t head = a.free_head ? max(*a.free_head, 0) : 0;
  auto blocks_of = [&](int n) { return min(n / bs + (n % bs != 0), a.max_blocks); };
  // id of the j-th block the step takes; -1 behind the end of the free list
  auto taken = [&](int64_t j) { return head + j < a.n_free ? a.free_blocks[head + j] : -1; };

  const int64_t tok_lo = static_cast<int64_t>(blockIdx.x) * kTokensPerBlock;
  const int64_t tok_hi = min(tok_lo + kTokensPerBlock, a.n_slots);
  int64_t tok_base = 0, fresh_base = 0;  // totals of the chunks before
  for (int s0 = 0; s0 < a.n_seqs; s0 += kChunk) {
    int tk[kPerThread], fr[kPerThread], sum_t = 0, sum_f = 0;
    const int i0 = s0 + tid * kPerThread;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int i = i0 + k;
      const int c = i < a.n_seqs ? min(max(a.ctx[i], 0), kMost - 1) : 0;
      const int n = i < a.n_seqs ? min(max(a.fresh_tokens[i], 0), kMost - 1) : 0;
      s_ctx[tid * kPerThread + k] = c;
      sum_t = add_most(sum_t, n);
      sum_f += blocks_of(c + n) - blocks_of(c);
      tk[k] = sum_t;
      fr[k] = sum_f;
    }
    int inc_t = sum_t, inc_f = sum_f;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int t = __shfl_up_sync(~0u, inc_t, d), f = __shfl_up_sync(~0u, inc_f, d);
      if (lane >= d) inc_t = add_most(inc_t, t), inc_f += f;
    }
    if (lane == 31) s_warp[0][warp] = inc_t, s_warp[1][warp] = inc_f;
    __syncthreads();
    int off_t = __shfl_up_sync(~0u, inc_t, 1), off_f = __shfl_up_sync(~0u, inc_f, 1);
    if (lane == 0) off_t = off_f = 0;
    int all_t = 0, all_f = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) off_t = add_most(off_t, s_warp[0][w]), off_f += s_warp[1][w];
      all_t = add_most(all_t, s_warp[0][w]);
      all_f += s_warp[1][w];
    }
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      s_end[tid * kPerThread + k] = add_most(off_t, tk[k]);
      s_fresh[tid * kPerThread + k] = off_f + fr[k];
    }
    __syncthreads();
    const int n_here = min(kChunk, a.n_seqs - s0);

    // lengths and offsets: one block per chunk writes them
    if (s0 / kChunk % gridDim.x == blockIdx.x) {
      for (int i = tid; i < n_here; i += kThreads) {
        const int n = s_end[i] - (i ? s_end[i - 1] : 0);
        a.query_start_loc[s0 + i + 1] = static_cast<int32_t>(tok_base + s_end[i]);
        a.seq_lens[s0 + i] = s_ctx[i] + n;
      }
    }
    // first index i of the chunk with ends[i] > v
    auto find = [&](const int* ends, int v) {
      int lo = 0, hi = n_here - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (ends[mid] > v) hi = mid; else lo = mid + 1;
      }
      return lo;
    };
    // fresh table entries, in runs of kThreads dealt to the blocks in turn
    const int64_t first_run = fresh_base / kThreads;
    const unsigned skip = (blockIdx.x + gridDim.x - static_cast<unsigned>(first_run % gridDim.x)) % gridDim.x;
    for (int64_t run = first_run + skip; run * kThreads < fresh_base + all_f; run += gridDim.x) {
      const int64_t j = run * kThreads + tid;
      if (j < fresh_base || j >= fresh_base + all_f) continue;
      const int v = static_cast<int>(j - fresh_base);
      const int i = find(s_fresh, v);
      const int e = blocks_of(s_ctx[i]) + v - (i ? s_fresh[i - 1] : 0);
      a.table[static_cast<int64_t>(s0 + i) * a.bt_stride + e] = taken(j);
    }
    // tokens of this block's share
    const int64_t lo = max(tok_lo, tok_base), hi = min(tok_hi, tok_base + all_t);
    for (int64_t t = lo + tid; t < hi; t += kThreads) {
      const int v = static_cast<int>(t - tok_base);
      const int i = find(s_end, v);
      const int c = s_ctx[i];
      const int pos = c + v - (i ? s_end[i - 1] : 0);
      const int e = pos / bs, first = blocks_of(c);
      int id = -1;
      if (e < first) {
        id = a.table[static_cast<int64_t>(s0 + i) * a.bt_stride + e];
      } else if (e < a.max_blocks) {
        id = taken(fresh_base + (i ? s_fresh[i - 1] : 0) + e - first);
      }
      a.slot_mapping[t] = id < 0 ? -1 : static_cast<int64_t>(id) * bs + (pos - e * bs);
      if (a.positions) a.positions[t] = pos;
    }
    tok_base += all_t;
    fresh_base += all_f;
    __syncthreads();
  }
  // padding behind the last token
  for (int64_t t = max(tok_lo, tok_base) + tid; t < tok_hi; t += kThreads) {
    a.slot_mapping[t] = -1;
    if (a.positions) a.positions[t] = 0;
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.query_start_loc[0] = 0;
    *a.blocks_taken = static_cast<int32_t>(fresh_base);
  }
}

}  // namespace

int launch_step_tables(const int32_t* ctx, const int32_t* fresh_tokens, int32_t* table,
                       int64_t bt_stride, int max_blocks, const int32_t* free_blocks,
                       int64_t n_free, const int32_t* free_head, int n_seqs, int block_size,
                       int64_t n_slots, int32_t* query_start_loc, int32_t* seq_lens,
                       int64_t* slot_mapping, int64_t* positions, int32_t* blocks_taken,
                       cudaStream_t st) {
  StepArgs a{ctx, fresh_tokens, table, bt_stride, max_blocks, free_blocks, n_free, free_head,
             n_seqs, block_size, n_slots, query_start_loc, seq_lens, slot_mapping, positions,
             blocks_taken};
  const int64_t blocks = (n_slots + kTokensPerBlock - 1) / kTokensPerBlock;
  step_tables_kernel<<<static_cast<unsigned>(blocks < 1 ? 1 : blocks), kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? KNLP_OK : KNLP_ERR_LAUNCH;
}

}  // namespace knlp
