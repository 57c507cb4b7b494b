// Stride-generic attention of several query tokens per sequence over the packed cache, on the
// CUDA cores: any strides and alignment, head_dim 32 / 64 / 128 / 256, any number of q heads per
// kv head, every K / V mode.  It serves the layouts that the tensor-core kernel does not address
// and is the in-library cross-check of that kernel.
//
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over j < limit(i); with ctx = len - n_new,
//   limit(i) = ctx + i + 1 (causal) or len
//
// Mapping: grid (query token, kv head x q-head group); 4 warps take the visible tokens
// round-robin, a lane owns head_dim / 32 elements of every row, the group's q heads share each
// row read; the warps' states (m, l, o) are merged through shared memory.  Everything is fp32.

#include "plane_row.cuh"
#include "serve.cuh"

namespace knlp {
namespace {

constexpr int kWarps = 4;

// The sequence that holds token t: first s with starts[s + 1] > t.  -1: none.
__device__ __forceinline__ int sequence_of(const int32_t* starts, int n_seqs, int t) {
  if (t < starts[0] || t >= starts[n_seqs]) return -1;
  int lo = 0, hi = n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  return lo;
}

template <int EPL, int QH>
__global__ void __launch_bounds__(kWarps * 32)
extend_generic_kernel(const ExtendArgs a, int n_rep, int q_groups) {
  const int tok = blockIdx.x;
  const int kvh = blockIdx.y / q_groups, qg = blockIdx.y % q_groups;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int P = a.block_size;
  const int seq = sequence_of(a.query_start_loc, a.n_seqs, tok);
  if (seq < 0) return;  // a row behind the last sequence stays as it is
  int first;
  const int n_new = extend_rows(a, seq, &first);
  const int len = extend_length(a, seq);
  const int end = a.causal ? min(len, max(a.seq_lens[seq] - n_new + tok - first + 1, 0)) : len;

  const int h_first = qg * QH;
  float q[QH][EPL], m[QH], l[QH], acc[QH][EPL];
#pragma unroll
  for (int h = 0; h < QH; ++h) {
    const int hr = h_first + h;
    const int qh = kvh * n_rep + (hr < n_rep ? hr : 0);
    const int64_t base = tok * a.q_stride[0] + qh * a.q_stride[1] + lane * EPL;
    m[h] = -INFINITY;
    l[h] = 0.0f;
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
      q[h][i] = load_elem_rt(a.q, base + i, a.q_dtype) * a.scale;
      acc[h][i] = 0.0f;
    }
  }

  for (int t = warp; t < end; t += kWarps) {
    int64_t blk = a.block_table[seq * a.bt_stride + t / P];
    blk = blk < 0 ? 0 : (blk >= a.num_blocks ? a.num_blocks - 1 : blk);
    const int off = t % P;
    float kv[EPL];
    auto load = [&](const Plane& p) {
      load_row<EPL>(p, p.codes + blk * p.cs[0] + off * p.cs[1] + kvh * p.cs[2],
                    p.scales + blk * p.ss[0] + off * p.ss[1] + kvh * p.ss[2],
                    p.zeros ? p.zeros + blk * p.zs[0] + off * p.zs[1] + kvh * p.zs[2] : nullptr,
                    lane, kv);
    };
    load(a.k);
    float s[QH];
#pragma unroll
    for (int h = 0; h < QH; ++h) {
      float dot = 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) dot = fmaf(q[h][i], kv[i], dot);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
      s[h] = dot;
    }
    load(a.v);
#pragma unroll
    for (int h = 0; h < QH; ++h) {
      const float m_new = fmaxf(m[h], s[h]);
      // a score of -inf weighs nothing, also while there is no other one (-inf - -inf)
      const float alpha = m[h] == m_new ? 1.0f : __expf(m[h] - m_new);
      const float pr = s[h] == -INFINITY ? 0.0f : __expf(s[h] - m_new);
      l[h] = l[h] * alpha + pr;
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[h][i] = acc[h][i] * alpha + pr * kv[i];
      m[h] = m_new;
    }
  }

  __shared__ float sm_m[kWarps][QH], sm_l[kWarps][QH], sm_o[kWarps][QH][EPL * 32];
#pragma unroll
  for (int h = 0; h < QH; ++h) {
    if (lane == 0) sm_m[warp][h] = m[h], sm_l[warp][h] = l[h];
#pragma unroll
    for (int i = 0; i < EPL; ++i) sm_o[warp][h][lane * EPL + i] = acc[h][i];
  }
  __syncthreads();
  for (int h = warp; h < QH; h += kWarps) {
    const int hr = h_first + h;
    if (hr >= n_rep) break;
    float mm = -INFINITY, ll = 0.0f, o[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) o[i] = 0.0f;
    for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, sm_m[w][h]);
    for (int w = 0; w < kWarps; ++w) {
      const float wgt = sm_l[w][h] > 0.0f ? __expf(sm_m[w][h] - mm) : 0.0f;
      ll += sm_l[w][h] * wgt;
#pragma unroll
      for (int i = 0; i < EPL; ++i) o[i] += sm_o[w][h][lane * EPL + i] * wgt;
    }
    const float inv = ll > 0.0f ? 1.0f / ll : 0.0f;
    const int64_t row = static_cast<int64_t>(tok) * a.n_q_heads + kvh * n_rep + hr;
#pragma unroll
    for (int i = 0; i < EPL; ++i)
      store_elem_rt(a.out, row * a.out_row_stride + lane * EPL + i, o[i] * inv, a.out_dtype);
    if (a.lse && lane == 0) a.lse[row] = ll > 0.0f ? mm + logf(ll) : -INFINITY;
  }
}

template <int EPL>
int launch_epl(const ExtendArgs& a, cudaStream_t st) {
  const int n_rep = a.n_q_heads / a.n_kv_heads;
  if (n_rep == 1) {
    extend_generic_kernel<EPL, 1><<<dim3(a.n_tokens, a.n_kv_heads), kWarps * 32, 0, st>>>(a, n_rep, 1);
  } else {
    const int qg = (n_rep + 3) / 4;
    extend_generic_kernel<EPL, 4><<<dim3(a.n_tokens, a.n_kv_heads * qg), kWarps * 32, 0, st>>>(a, n_rep, qg);
  }
  return cudaGetLastError() == cudaSuccess ? KNLP_OK : KNLP_ERR_LAUNCH;
}

}  // namespace

int launch_extend_generic(const ExtendArgs& a, cudaStream_t st) {
  switch (a.head_dim) {
    case 32: return launch_epl<1>(a, st);
    case 64: return launch_epl<2>(a, st);
    case 128: return launch_epl<4>(a, st);
    case 256: return launch_epl<8>(a, st);
    default: return KNLP_ERR_SHAPE;
  }
}

}  // namespace knlp
