// Scores of given tokens from logits: log probability, entropy of the distribution, rank of the
// token, and the k largest logits with their log probabilities.  Per row x of V logits:
//
//   m = max x,  l = sum e^(x-m),  w = sum e^(x-m) (x-m)
//   logprob(t) = (x_t - m) - ln l,   entropy = ln l - w / l,   rank = 1 + #{i : x_i > x_t}
//
// What bounds it: the logits are read once (2 or 4 bytes each) against one exp2 and about seven
// more instructions: fp32 rows run at 5.3 TB/s without alternatives, bf16 rows at 3.5 (2047 rows
// of 50257 with 8 alternatives: 68 us, 3.0 TB/s), by instruction issue.  A thread keeps (m, l, w)
// of its own share online, in base-2 units; they are merged at the end: with d = m_old - m, l' = l
// 2^d and w' = (w + d l) 2^d.
//
// The k largest come from the same pass: the k-th largest of the kGroups group maxima (a group =
// a few threads' shares) is a bound that at least k elements reach, and hardly more than k do.
// Only the shares whose maximum reaches it are read again (from L2), the elements that reach
// the bound are collected and ordered by counting.  Equal logits go by the lower index; where
// ties or a lopsided row overflow the collection, slower exact paths follow (below).  NaN counts
// as the largest value, as in torch.
//
// Blocks of 256 threads: the ranking at a row's end runs under other rows' reading (512 threads:
// 83 us on the same case).  A row is served by a cluster of 1, 2, 4 or 8 blocks, each with a
// slice; the first block merges through distributed shared memory.  More than one block pays while
// rows x slices leave SMs without work (launch_token_score).

#include <cooperative_groups.h>

#include "pair_math.cuh"
#include "serve.cuh"

namespace cg = cooperative_groups;

namespace knlp {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kGroups = kThreads / 2;  // shares of two neighbouring threads
constexpr int kCap = 1024;             // collected candidates of one slice
constexpr int kMaxTop = KNLP_MAX_TOP;
constexpr int kMaxParts = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

static_assert(kMaxParts * kMaxTop <= kCap, "");

struct ScoreArgs {
  const void* logits;
  int64_t row_stride;
  const int64_t* ids;
  int vocab, top_k, slice;
  float* logprob;
  float* entropy;
  int32_t* rank;
  int64_t* top_ids;
  float* top_logprobs;
};

// max that keeps a NaN of either side
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Exponent of 2^.. for a difference of logits that is <= 0.  Differences are formed before they
// are scaled (masks may be the type's lowest value, whose product with log2 e overflows); -1e4
// stands for every exponent that gives 0, so that a masked logit adds 0 and not 0 * inf.
constexpr float kNothing = -1e4f;
__device__ __forceinline__ float exponent(float diff) { return max_nan(diff * kLog2e, kNothing); }

// Order of the values: NaN above +inf, -0 equal to +0.
__device__ __forceinline__ uint32_t order(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
// Value and index in one key: the larger value first, then the lower index.
__device__ __forceinline__ uint64_t key_of(float x, int i) {
  return static_cast<uint64_t>(order(x)) << 32 | static_cast<uint32_t>(~i);
}
__device__ __forceinline__ int index_of(uint64_t key) { return ~static_cast<uint32_t>(key); }

struct Stats {
  float m, l, w;  // maximum; sums in base 2 relative to it
  int above;      // elements larger than the given token's
  __device__ __forceinline__ void merge(const Stats& o) {
    above += o.above;
    const float mm = max_nan(m, o.m);
    // a side without a finite element has l = w = 0 and nothing to shift
    const float d0 = m == mm ? 0.0f : exponent(m - mm), d1 = o.m == mm ? 0.0f : exponent(o.m - mm);
    const float e0 = exp2f(d0), e1 = exp2f(d1);
    const float w0 = l == 0.0f ? 0.0f : (w + d0 * l) * e0;
    const float w1 = o.l == 0.0f ? 0.0f : (o.w + d1 * o.l) * e1;
    w = w0 + w1;
    l = l * e0 + o.l * e1;
    m = mm;
  }
};

// Statistics of `width` neighbouring lanes, in all of them.
__device__ __forceinline__ void merge_lanes(Stats& s, int width) {
  for (int d = width / 2; d; d >>= 1) {
    Stats o;
    o.m = __shfl_xor_sync(~0u, s.m, d);
    o.l = __shfl_xor_sync(~0u, s.l, d);
    o.w = __shfl_xor_sync(~0u, s.w, d);
    o.above = __shfl_xor_sync(~0u, s.above, d);
    s.merge(o);
  }
}

template <int DT>
struct Vec;  // 16 bytes of logits
template <>
struct Vec<KNLP_F32> {
  static constexpr int n = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    f[0] = __uint_as_float(v.x), f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z), f[3] = __uint_as_float(v.w);
  }
};
template <>
struct Vec<KNLP_F16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
      f[2 * i] = p.x, f[2 * i + 1] = p.y;
    }
  }
};
template <>
struct Vec<KNLP_BF16> {
  static constexpr int n = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* f) {
    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = __uint_as_float(u[i] << 16);
      f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
};

// A thread's running statistics: its sums in two halves, for paired arithmetic.
struct Running {
  float m = -INFINITY;
  uint64_t l = 0, w = 0;
  int above = 0;
  __device__ __forceinline__ Stats total() const {
    float l0, l1, w0, w1;
    unpack2(l, l0, l1);
    unpack2(w, w0, w1);
    return {m, l0 + l1, w0 + w1, above};
  }
};

// N (even) values, or one (the other half of its pair a masked logit).
template <int N>
__device__ __forceinline__ void take(Running& s, const float* f, float given) {
  float c = f[0];
#pragma unroll
  for (int i = 1; i < N; ++i) c = max_nan(c, f[i]);
  if (!(c <= s.m)) {  // also for a NaN, which then stays
    if (s.m != -INFINITY) {
      const float d = exponent(s.m - c), e = exp2f(d);
      s.w = mul2(fma2(pack2(d, d), s.l, s.w), pack2(e, e));
      s.l = mul2(s.l, pack2(e, e));
    }
    s.m = max_nan(s.m, c);
  }
  if (s.m == -INFINITY) return;
  const uint64_t off = pack2(-s.m, -s.m), scale = pack2(kLog2e, kLog2e);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    float t0, t1, e0, e1;
    unpack2(mul2(add2(pack2(f[i], i + 1 < N ? f[i + 1] : -INFINITY), off), scale), t0, t1);
    t0 = max_nan(t0, kNothing), t1 = max_nan(t1, kNothing);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(t0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(t1));
    s.l = add2(s.l, pack2(e0, e1));
    s.w = fma2(pack2(e0, e1), pack2(t0, t1), s.w);
  }
  if (!(c <= given)) {
#pragma unroll
    for (int i = 0; i < N; ++i) s.above += f[i] > given;
  }
}

struct Shared {
  Stats warp[kWarps];
  Stats all;  // of this slice
  uint64_t cand[kCap];    // candidates of the slice, then the lists of all slices
  uint64_t top[kMaxTop];  // this slice's k best keys, 0 where it has fewer elements
  uint32_t group[kGroups];  // order() of the group maxima
  int hot[kThreads];
  uint64_t best[kWarps];
  uint64_t merged[kMaxTop];
  uint32_t bound;
  int n_cand, n_strict, n_hot, ties;
  int tie_warp[kWarps];
};

// Walks one thread's share of a slice: single elements up to the first 16-byte boundary, whole
// vectors thread by thread, single elements behind the last one.
template <int DT>
struct Slice {
  static constexpr int N = Vec<DT>::n;
  static constexpr int kSize = 16 / N;
  const char* base;  // first element
  int first, n;      // its index in the row, elements
  int head, vecs;    // elements before the vectors, number of vectors

  __device__ Slice(const void* row, int first_, int n_) : first(first_), n(n_) {
    base = static_cast<const char*>(row) + static_cast<int64_t>(first) * kSize;
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(base) & 15);
    head = min(off ? (16 - off) / kSize : 0, n);
    vecs = (n - head) / N;
  }
  __device__ __forceinline__ float at(int i) const { return load_elem<DT>(base, i); }
  __device__ __forceinline__ uint4 vec(int v) const {
    return __ldg(reinterpret_cast<const uint4*>(base + head * kSize) + v);
  }
  // index in the slice of the thread's single element before / behind the vectors, or -1
  __device__ __forceinline__ int single(int t, int which) const {
    if (which == 0) return t < head ? t : -1;
    const int i = head + vecs * N + t;
    return i < n ? i : -1;
  }
};

// Elements of the slice that pass `f(value, index)` offered to every thread of the block,
// over the shares listed in hot.
template <int DT, class F>
__device__ __forceinline__ void over_hot(const Slice<DT>& s, const int* hot, int n_hot, F f) {
  const int per = (s.vecs + kThreads - 1) / kThreads;  // vectors of a share, rounded up
  for (int w = threadIdx.x; w < n_hot * per; w += kThreads) {
    // neighbouring threads take neighbouring shares of one vector row: the hot list is sorted
    // by nothing in particular, but what it lists of one row lies within 8 KB
    const int v = hot[w % n_hot] + w / n_hot * kThreads;
    if (v >= s.vecs) continue;
    float x[Vec<DT>::n];
    Vec<DT>::unpack(s.vec(v), x);
#pragma unroll
    for (int i = 0; i < Vec<DT>::n; ++i) f(x[i], s.head + v * Vec<DT>::n + i);
  }
  if (threadIdx.x < n_hot) {
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int i = s.single(hot[threadIdx.x], which);
      if (i >= 0) f(s.at(i), i);
    }
  }
}

// The k best keys of the slice into sh.top.  share_max: maximum of the caller's share.
template <int DT>
__device__ void top_of_slice(Shared& sh, const Slice<DT>& s, int k, float share_max) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid < kMaxTop) sh.top[tid] = 0;
  if (tid == 0) sh.n_cand = sh.n_strict = sh.n_hot = sh.ties = 0;
  float g = share_max;
  g = max_nan(g, __shfl_xor_sync(~0u, g, 1));
  if ((tid & 1) == 0) sh.group[tid >> 1] = order(g);
  __syncthreads();
  // the k-th largest group maximum (k <= kMaxTop < kGroups)
  if (tid < kGroups) {
    const uint32_t mine = sh.group[tid];
    int before = 0;
#pragma unroll 8
    for (int i = 0; i < kGroups; ++i) before += sh.group[i] > mine || (sh.group[i] == mine && i < tid);
    if (before == k - 1) sh.bound = mine;
  }
  __syncthreads();
  const uint32_t bound = sh.bound;
  if (order(share_max) >= bound) sh.hot[atomicAdd(&sh.n_hot, 1)] = tid;
  __syncthreads();
  const int n_hot = sh.n_hot;
  over_hot<DT>(s, sh.hot, n_hot, [&](float x, int i) {
    if (order(x) >= bound) {
      const int c = atomicAdd(&sh.n_cand, 1);
      if (c < kCap) sh.cand[c] = key_of(x, s.first + i);
    }
  });
  __syncthreads();
  int n = sh.n_cand;
  if (n > kCap) {
    // Too many, as a rule because many elements equal the bound (a masked row, coarse types).
    // Those above it, then the first of the equal ones in the order of their index.
    __syncthreads();
    over_hot<DT>(s, sh.hot, n_hot, [&](float x, int i) {
      if (order(x) > bound) {
        const int c = atomicAdd(&sh.n_strict, 1);
        if (c < kCap - kMaxTop) sh.cand[c] = key_of(x, s.first + i);
      }
    });
    __syncthreads();
    n = sh.n_strict;
    if (n <= kCap - kMaxTop) {
      for (int i0 = 0; i0 < s.n && sh.ties < k; i0 += kThreads) {
        const int i = i0 + tid;
        const float x = i < s.n ? s.at(i) : 0.0f;
        const bool tie = i < s.n && order(x) == bound;
        const unsigned vote = __ballot_sync(~0u, tie);
        if (lane == 0) sh.tie_warp[warp] = __popc(vote);
        __syncthreads();
        int at = sh.ties + __popc(vote & ((1u << lane) - 1)), all = 0;
        for (int w = 0; w < kWarps; ++w) {
          if (w < warp) at += sh.tie_warp[w];
          all += sh.tie_warp[w];
        }
        if (tie && at < k) sh.cand[n + at] = key_of(x, s.first + i);
        __syncthreads();
        if (tid == 0) sh.ties += all;
        __syncthreads();
      }
      n += min(sh.ties, k);
    } else {
      // A row whose large values crowd in a few shares: the best key below the last, k times.
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        uint64_t b = 0;
        for (int i = tid; i < s.n; i += kThreads) {
          const uint64_t key = key_of(s.at(i), s.first + i);
          if (key < last && key > b) b = key;
        }
        for (int d = 16; d; d >>= 1) {
          const uint64_t o = __shfl_xor_sync(~0u, b, d);
          b = o > b ? o : b;
        }
        if (lane == 0) sh.best[warp] = b;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w) b = sh.best[w] > b ? sh.best[w] : b;
        if (tid == 0) sh.top[j] = b;
        last = b;
        __syncthreads();
      }
      return;
    }
    __syncthreads();
  }
  for (int i = tid; i < n; i += kThreads) {
    const uint64_t mine = sh.cand[i];
    int before = 0;
    for (int j = 0; j < n; ++j) before += sh.cand[j] > mine;
    if (before < k) sh.top[before] = mine;
  }
  __syncthreads();
}

template <int DT>
__global__ void __launch_bounds__(kThreads) token_score_kernel(ScoreArgs a) {
  __shared__ Shared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int part = cluster.block_rank(), parts = cluster.num_blocks();
  const int64_t row = blockIdx.x / parts;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int N = Vec<DT>::n;
  const char* x = static_cast<const char*>(a.logits) + row * a.row_stride * (16 / N);
  const int lo = min(part * a.slice, a.vocab), hi = min(lo + a.slice, a.vocab);
  const Slice<DT> s(x, lo, hi - lo);
  const int64_t id = a.ids[row];
  const bool known = id >= 0 && id < a.vocab;
  const float given = known ? load_elem<DT>(x, id) : INFINITY;

  Running run;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int i = s.single(tid, which);
    if (i >= 0) {
      const float f = s.at(i);
      take<1>(run, &f, given);
    }
  }
  int v = tid;
  for (; v + 3 * kThreads < s.vecs; v += 4 * kThreads) {
    uint4 u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = s.vec(v + j * kThreads);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float f[N];
      Vec<DT>::unpack(u[j], f);
      take<N>(run, f, given);
    }
  }
  for (; v < s.vecs; v += kThreads) {
    float f[N];
    Vec<DT>::unpack(s.vec(v), f);
    take<N>(run, f, given);
  }

  const float share_max = run.m;
  Stats st = run.total();
  merge_lanes(st, 32);
  if (lane == 0) sh.warp[warp] = st;
  if (a.top_k) top_of_slice<DT>(sh, s, a.top_k, share_max);
  __syncthreads();
  if (warp == 0) {
    Stats all = sh.warp[lane % kWarps];
    merge_lanes(all, kWarps);
    if (lane == 0) sh.all = all;
  }
  cluster.sync();
  if (part == 0) {
    if (warp == 0) {
      Stats all = cluster.map_shared_rank(&sh, lane % parts)->all;
      merge_lanes(all, parts);
      if (lane == 0) sh.warp[0] = all;
    }
    const int n = parts * a.top_k;  // <= kCap
    for (int i = tid; i < n; i += kThreads) sh.cand[i] = cluster.map_shared_rank(&sh, i / a.top_k)->top[i % a.top_k];
    __syncthreads();
    const Stats t = sh.warp[0];
    const bool empty = t.m == -INFINITY;  // no logit above -inf: no token has a probability
    const float log_sum = empty ? 0.0f : kLn2 * log2f(t.l);
    auto logprob = [&](float v) { return empty ? v : (v - t.m) - log_sum; };
    if (tid == 0) {
      a.logprob[row] = known ? logprob(given) : id < 0 ? 0.0f : NAN;
      a.entropy[row] = empty ? 0.0f : log_sum - kLn2 * (t.w / t.l);
      a.rank[row] = known ? t.above + 1 : 0;
    }
    for (int i = tid; i < n; i += kThreads) {
      const uint64_t mine = sh.cand[i];
      int before = 0;
      for (int j = 0; j < n; ++j) before += sh.cand[j] > mine;
      if (before < a.top_k && mine) sh.merged[before] = mine;
    }
    __syncthreads();
    if (tid < a.top_k) {
      const int i = index_of(sh.merged[tid]);
      a.top_ids[row * a.top_k + tid] = i;
      a.top_logprobs[row * a.top_k + tid] = logprob(load_elem<DT>(x, i));
    }
  }
  cluster.sync();  // the other blocks' shared memory stays until the first one has read it
}

}  // namespace

int launch_token_score(const void* logits, int dtype, int64_t row_stride, const int64_t* ids,
                       int n_rows, int vocab, int top_k, float* logprob, float* entropy,
                       int32_t* rank, int64_t* top_ids, float* top_logprobs, int n_sms,
                       cudaStream_t st) {
  // Slices while they find idle SMs: with two blocks per SM 128 rows of 128256 bf16 logits take 20.5
  // us (2 slices each), with eight 29.6 us (8 slices): a block's own ranking does not get shorter.
  int parts = 1;
  while (parts < kMaxParts && n_rows * parts * 2 <= n_sms * 2 && vocab / (parts * 2) >= 4096)
    parts *= 2;
  const int slice = ((vocab + parts - 1) / parts + 7) / 8 * 8;
  ScoreArgs a{logits, row_stride, ids, vocab, top_k, slice, logprob, entropy, rank, top_ids,
              top_logprobs};
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(n_rows) * parts);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t rc = dtype == KNLP_F32   ? cudaLaunchKernelEx(&cfg, token_score_kernel<KNLP_F32>, a)
                   : dtype == KNLP_F16 ? cudaLaunchKernelEx(&cfg, token_score_kernel<KNLP_F16>, a)
                                       : cudaLaunchKernelEx(&cfg, token_score_kernel<KNLP_BF16>, a);
  if (rc != cudaSuccess) {
    cudaGetLastError();
    return KNLP_ERR_LAUNCH;
  }
  return KNLP_OK;
}

}  // namespace knlp
