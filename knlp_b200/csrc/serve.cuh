// Launch functions of the serving-step operators: step tables, attention of several query
// tokens per sequence, token scores.
#pragma once

#include "common.cuh"

namespace knlp {

// api.cu: argument check of one plane, and the SM count of the current device.
int check_plane(const knlp_kv_plane* p, bool unquantized_k);
int sm_count();

struct ExtendArgs {
  const void* q;
  int q_dtype;
  int64_t q_stride[2];
  Plane k, v;
  const int32_t* block_table;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* seq_lens;
  const int32_t* query_start_loc;
  int64_t num_blocks;
  int n_seqs, n_tokens, n_q_heads, n_kv_heads, head_dim, block_size;
  float scale;
  bool causal;
  void* out;
  int out_dtype;
  int64_t out_row_stride;
  float* lse;
};

// Cached tokens of a sequence, at most what its table row can hold.
__device__ __forceinline__ int extend_length(const ExtendArgs& a, int seq) {
  const int64_t most = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const int n = max(a.seq_lens[seq], 0);
  return n < most ? n : static_cast<int>(most);
}

// New tokens of a sequence and its first query row, kept inside the query whatever the offsets.
__device__ __forceinline__ int extend_rows(const ExtendArgs& a, int seq, int* first) {
  const int lo = min(max(a.query_start_loc[seq], 0), a.n_tokens);
  const int hi = min(max(a.query_start_loc[seq + 1], 0), a.n_tokens);
  *first = lo;
  return max(hi - lo, 0);
}

// Tensor-core kernel (extend_plan.cu, extend_mma.cuh).  Returns KNLP_OK, 1 if the layout is not
// one it addresses (nothing launched), < 0 on error.
int launch_extend_mma(const ExtendArgs& a, int max_query_len, int max_seq_len, float* ws,
                      int64_t ws_floats, int n_sms, cudaStream_t st);
int64_t extend_workspace_floats(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads,
                                int head_dim, int n_sms);
// Device-side status word shared by the kernels with bounded waits (decode_mma.cu).
int* decode_status_ptr();

int launch_extend_generic(const ExtendArgs& a, cudaStream_t st);

int launch_step_tables(const int32_t* ctx, const int32_t* fresh_tokens, int32_t* table,
                       int64_t bt_stride, int max_blocks, const int32_t* free_blocks,
                       int64_t n_free, const int32_t* free_head, int n_seqs, int block_size,
                       int64_t n_slots, int32_t* query_start_loc, int32_t* seq_lens,
                       int64_t* slot_mapping, int64_t* positions, int32_t* blocks_taken,
                       cudaStream_t st);

int launch_token_score(const void* logits, int dtype, int64_t row_stride, const int64_t* ids,
                       int n_rows, int vocab, int top_k, float* logprob, float* entropy,
                       int32_t* rank, int64_t* top_ids, float* top_logprobs, int n_sms,
                       cudaStream_t st);

}  // namespace knlp
