// C ABI of the serving-step operators: argument validation and dispatch.

#include "serve.cuh"

using namespace knlp;

namespace {

bool dtype_ok(int dt) { return dt == KNLP_F32 || dt == KNLP_F16 || dt == KNLP_BF16; }

}  // namespace

extern "C" {

int knlp_b200_extend_workspace(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads,
                               int head_dim, int64_t* workspace_floats_out) {
  if (!workspace_floats_out) return KNLP_ERR_NULL;
  if (n_seqs < 0 || n_tokens < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads)
    return KNLP_ERR_SHAPE;
  if (head_dim != 32 && head_dim != 64 && head_dim != 128 && head_dim != 256) return KNLP_ERR_SHAPE;
  *workspace_floats_out = extend_workspace_floats(n_seqs, n_tokens, n_q_heads, n_kv_heads, head_dim, sm_count());
  return KNLP_OK;
}

int knlp_b200_extend_attention(const void* query, int q_dtype, const int64_t q_stride[2],
                               const knlp_kv_plane* k_plane, const knlp_kv_plane* v_plane,
                               const int32_t* block_table, int64_t bt_stride, int max_blocks,
                               const int32_t* seq_lens, const int32_t* query_start_loc,
                               int64_t num_blocks, int n_seqs, int n_tokens, int n_q_heads,
                               int n_kv_heads, int head_dim, int block_size, int max_query_len,
                               int max_seq_len, float softmax_scale, float* workspace,
                               int64_t workspace_floats, void* out, int out_dtype,
                               int64_t out_row_stride, float* lse, unsigned flags, void* stream) {
  if (!query || !q_stride || !block_table || !seq_lens || !query_start_loc || !workspace || !out)
    return KNLP_ERR_NULL;
  if (q_dtype != KNLP_F16 && q_dtype != KNLP_BF16) return KNLP_ERR_DTYPE;
  if (!dtype_ok(out_dtype)) return KNLP_ERR_DTYPE;
  if (flags & ~(KNLP_EXTEND_FORCE_GENERIC | KNLP_EXTEND_FULL)) return KNLP_ERR_MODE;
  int64_t need = 0;
  int rc = knlp_b200_extend_workspace(n_seqs, n_tokens, n_q_heads, n_kv_heads, head_dim, &need);
  if (rc) return rc;
  if (block_size <= 0 || max_blocks <= 0 || num_blocks <= 0) return KNLP_ERR_SHAPE;
  if (n_q_heads > 65535) return KNLP_ERR_SHAPE;
  if (!(softmax_scale > 0.0f) || max_query_len < 0 || max_seq_len < 0) return KNLP_ERR_SHAPE;
  if (workspace_floats < need) return KNLP_ERR_WORKSPACE;
  if (out_row_stride < head_dim) return KNLP_ERR_STRIDE;
  rc = check_plane(k_plane, true);
  if (rc) return rc;
  rc = check_plane(v_plane, false);
  if (rc) return rc;
  if ((k_plane->mode == KNLP_KV_F16 && q_dtype != KNLP_F16) ||
      (k_plane->mode == KNLP_KV_BF16 && q_dtype != KNLP_BF16))
    return KNLP_ERR_MODE;
  if (n_seqs == 0 || n_tokens == 0) return KNLP_OK;
  ExtendArgs a{};
  a.q = query;
  a.q_dtype = q_dtype;
  a.q_stride[0] = q_stride[0];
  a.q_stride[1] = q_stride[1];
  a.k = make_plane(k_plane);
  a.v = make_plane(v_plane);
  a.block_table = block_table;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  a.seq_lens = seq_lens;
  a.query_start_loc = query_start_loc;
  a.num_blocks = num_blocks;
  a.n_seqs = n_seqs;
  a.n_tokens = n_tokens;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.scale = softmax_scale;
  a.causal = !(flags & KNLP_EXTEND_FULL);
  a.out = out;
  a.out_dtype = out_dtype;
  a.out_row_stride = out_row_stride;
  a.lse = lse;
  if (!(flags & KNLP_EXTEND_FORCE_GENERIC)) {
    rc = launch_extend_mma(a, max_query_len, max_seq_len, workspace, workspace_floats, sm_count(),
                           static_cast<cudaStream_t>(stream));
    if (rc <= 0) return rc;  // launched, or failed for good
  }
  return launch_extend_generic(a, static_cast<cudaStream_t>(stream));
}

int knlp_b200_build_step(const int32_t* context_lens, const int32_t* query_lens,
                         int32_t* block_table, int64_t bt_stride, int max_blocks,
                         const int32_t* free_blocks, int64_t n_free, const int32_t* free_head,
                         int n_seqs, int block_size, int64_t n_slots, int32_t* query_start_loc,
                         int32_t* seq_lens, int64_t* slot_mapping, int64_t* positions,
                         int32_t* blocks_taken, void* stream) {
  if (!query_start_loc || !blocks_taken) return KNLP_ERR_NULL;
  if (n_seqs < 0 || n_slots < 0 || n_free < 0 || block_size <= 0 || max_blocks <= 0)
    return KNLP_ERR_SHAPE;
  if (n_slots >= (1 << 30) || max_blocks > (1 << 20)) return KNLP_ERR_TOO_LARGE;
  if (n_seqs && (!context_lens || !query_lens || !block_table || !seq_lens)) return KNLP_ERR_NULL;
  if ((n_free && !free_blocks) || (n_slots && !slot_mapping)) return KNLP_ERR_NULL;
  if (bt_stride < max_blocks && n_seqs > 1) return KNLP_ERR_STRIDE;  // rows that overlap
  return launch_step_tables(context_lens, query_lens, block_table, bt_stride, max_blocks,
                            free_blocks, n_free, free_head, n_seqs, block_size, n_slots,
                            query_start_loc, seq_lens, slot_mapping, positions, blocks_taken,
                            static_cast<cudaStream_t>(stream));
}

int knlp_b200_token_score(const void* logits, int dtype, int64_t row_stride,
                          const int64_t* token_ids, int n_rows, int vocab, int top_k,
                          float* logprob, float* entropy, int32_t* rank, int64_t* top_ids,
                          float* top_logprobs, void* stream) {
  if (!dtype_ok(dtype)) return KNLP_ERR_DTYPE;
  if (n_rows < 0 || vocab <= 0 || top_k < 0 || top_k > vocab) return KNLP_ERR_SHAPE;
  if (top_k > KNLP_MAX_TOP || n_rows > (1 << 27) || vocab > (1 << 30)) return KNLP_ERR_TOO_LARGE;
  if (n_rows == 0) return KNLP_OK;
  if (!logits || !token_ids || !logprob || !entropy || !rank) return KNLP_ERR_NULL;
  if (top_k && (!top_ids || !top_logprobs)) return KNLP_ERR_NULL;
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == KNLP_F32 ? 4 : 2)) return KNLP_ERR_STRIDE;
  return launch_token_score(logits, dtype, row_stride, token_ids, n_rows, vocab, top_k, logprob,
                            entropy, rank, top_ids, top_logprobs, sm_count(),
                            static_cast<cudaStream_t>(stream));
}

}  // extern "C"
