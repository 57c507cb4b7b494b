// Host side of the tensor-core extend attention, the kernel that plans its work on the GPU, and
// the kernel that merges the pieces of split rows.
//
// Work: the packed query rows (token x group head) of a sequence are cut into tiles of 256, each
// with the cached tokens it can see; a last tile of at most 32 rows goes to the kernel for few
// rows (extend_few.cuh), the others to the one for many (extend_mma.cuh).  A tile's range of cached
// tokens may be cut into pieces that different CTAs serve and a last kernel merges.  The lengths
// live on the GPU, so a block per kernel plans there (4 us): it counts the tiles, weighs a dozen
// piece lengths by the rounds that the resulting items need on the machine, and writes the list of
// pieces, longest first.  Items are (piece, kv head), heads innermost: the CTAs that serve the heads
// of one piece run at the same time and share the 32-byte sectors in which the scales of several
// heads lie.  A CTA's items are dealt out back and forth; sorted so, four prompts of 1500-3900
// tokens take 694 us, in the order of the sequences 723 us.

#include "extend_launch.cuh"

namespace knlp {
namespace extend {
namespace {

constexpr int kPlanThreads = 512;
constexpr int kCandidates = kPlanThreads / 32;
constexpr int kMaxRows = 2 * kRows;
constexpr int kSharedSeqs = 1024, kSharedTiles = 2048;
// Time of an item in units of one 128 x 128 tile of one stream: what it costs besides its tiles
// (query in, result out, an empty pipeline at both ends), and of the merging launch.
constexpr float kItemCost = 4.0f, kMergeCost = 5.0f;

// Sizes of a kernel's lists.
struct Bounds {
  int64_t tiles, entries, parts;  // parts: rows of partial results
  Bounds(bool few, int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads, int n_sms) {
    const int64_t rows = static_cast<int64_t>(n_tokens) * (n_q_heads / n_kv_heads);
    tiles = rows / (few ? few::kFewRows : kMaxRows) + n_seqs;
    entries = 2 * tiles + 16 * static_cast<int64_t>(n_sms) / n_kv_heads + 2;
    // every row in pieces, up to a few tiles per SM
    const int64_t all = static_cast<int64_t>(n_tokens) * n_q_heads * 64;
    const int64_t most = static_cast<int64_t>(n_sms) * (few ? 8 * few::kFewRows : 3 * kMaxRows);
    parts = all < most ? all : most;
  }
};

struct Tile {
  int seq, row0, rows, kv;  // kv: tiles of cached tokens
  __device__ float cost() const { return rows > kRows ? 2.0f * kv : 1.0f * kv; }
  // pieces of at most `c` units, none shorter than two tiles (one per stream)
  __device__ int pieces(float c) const {
    const int most = rows > kRows ? kv : kv / 2;
    return max(1, min(most, static_cast<int>(ceilf(cost() / c))));
  }
};

// What a batch is cut into.
struct Cut {
  bool few_rows;  // the list of the kernel for few rows
  bool only_few;  // all rows go there, 32 at a time; else in tiles of 256, and what is left over
  // Tiles of a sequence with that many rows.
  __device__ int tiles_of(int64_t rows) const {
    if (only_few) return few_rows ? static_cast<int>((rows + few::kFewRows - 1) / few::kFewRows) : 0;
    const int rest = static_cast<int>(rows % kMaxRows);
    const bool few = rest > 0 && rest <= few::kFewRows;
    return few_rows ? few : static_cast<int>(rows / kMaxRows) + (rest > 0 && !few);
  }
  // First row of a tile, the i-th of its sequence.
  __device__ int row0(int64_t rows, int i) const {
    return only_few ? i * few::kFewRows : few_rows ? static_cast<int>(rows / kMaxRows) * kMaxRows : i * kMaxRows;
  }
  __device__ int most() const { return few_rows ? few::kFewRows : kMaxRows; }
};

__device__ Tile tile_at(const ExtendArgs& a, const Cut& cut, int rep, const int* base, int t) {
  int lo = 0, hi = a.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (base[mid + 1] > t) hi = mid; else lo = mid + 1;
  }
  int first;
  const int n = extend_rows(a, lo, &first), len = extend_length(a, lo);
  Tile x;
  x.seq = lo;
  x.row0 = cut.row0(static_cast<int64_t>(n) * rep, t - base[lo]);
  x.rows = min(cut.most(), n * rep - x.row0);
  const int last = (x.row0 + x.rows - 1) / rep;
  const int seen = a.causal ? max(min(a.seq_lens[lo] - n + last + 1, len), 0) : len;
  x.kv = (seen + kTile - 1) / kTile;
  return x;
}
// Exclusive prefix sums of N values over the block, and their totals.
template <int N>
__device__ void scan(int (&v)[N], int (&total)[N], int (*sh)[kPlanThreads / 32]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) inc[i] = v[i];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int o = __shfl_up_sync(~0u, inc[i], d);
      if (lane >= d) inc[i] += o;
    }
  __syncthreads();
  if (lane == 31)
    for (int i = 0; i < N; ++i) sh[i][warp] = inc[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int off = 0, all = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) {
      if (w < warp) off += sh[i][w];
      all += sh[i][w];
    }
    v[i] = off + inc[i] - v[i];
    total[i] = all;
  }
}

// A kernel's lists in the workspace.
struct Lists {
  int max_entries, max_tiles;
  int64_t max_parts;
  int* base;  // first tile of each sequence
  Plan* plan;
  Entry* entries;
  Split* splits;
};

__global__ void __launch_bounds__(kPlanThreads)
extend_plan_kernel(const __grid_constant__ ExtendArgs a, int rep, int n_ctas, bool only_few, bool whole,
                   const __grid_constant__ Lists many, const __grid_constant__ Lists few) {
  const Cut how{blockIdx.x == 1, only_few};  // a block per kernel
  const Lists& to = how.few_rows ? few : many;
  // small batches are planned out of shared memory: every step of it is a latency
  __shared__ int sh_base[kSharedSeqs + 1];
  __shared__ int2 sh_tiles[kSharedTiles];  // (kv, rows)
  int* const base = a.n_seqs <= kSharedSeqs ? sh_base : to.base;
  __shared__ int sh[4][kPlanThreads / 32];
  __shared__ float sh_cost[kCandidates], sh_piece[kCandidates], sh_worst[kCandidates];
  __shared__ int sh_at[kPlanThreads];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = a.n_kv_heads;

  int n_tiles = 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += kPlanThreads) {
    const int s = s0 + tid;
    int first, v[1] = {0}, total[1];
    if (s < a.n_seqs) {
      v[0] = how.tiles_of(static_cast<int64_t>(extend_rows(a, s, &first)) * rep);
    }
    scan(v, total, sh);
    if (s < a.n_seqs) base[s] = n_tiles + v[0];
    n_tiles += total[0];
  }
  if (tid == 0) base[a.n_seqs] = n_tiles;
  __syncthreads();
  n_tiles = min(n_tiles, to.max_tiles);  // more only for offsets that are not ascending

  float cost = 0.0f;
  for (int t = tid; t < n_tiles; t += kPlanThreads) {
    const Tile x = tile_at(a, how, rep, base, t);
    cost += x.cost();
    if (t < kSharedTiles) sh_tiles[t] = make_int2(x.kv, x.rows);
  }
  // a tile as far as its cost goes
  auto size_of = [&](int t) {
    if (t >= kSharedTiles) return tile_at(a, how, rep, base, t);
    Tile x{};
    x.kv = sh_tiles[t].x, x.rows = sh_tiles[t].y;
    return x;
  };
#pragma unroll
  for (int d = 16; d; d >>= 1) cost += __shfl_xor_sync(~0u, cost, d);
  if (lane == 0) sh_cost[warp] = cost;
  __syncthreads();
  cost = 0.0f;
  for (int w = 0; w < kCandidates; ++w) cost += sh_cost[w];
  __syncthreads();

  // A candidate per warp: pieces of 1 / f of a CTA's equal share, or none (warp 0).
  const float share = cost * heads / n_ctas;
  const float piece = warp == 0 || whole ? 1e30f : fmaxf(share / (warp < 8 ? 0.5f * warp + 0.5f : warp - 3), 2.0f);
  float worst = 0.0f;
  int items = 0;
  int64_t parts = 0;
  for (int t = lane; t < n_tiles; t += 32) {
    const Tile x = size_of(t);
    const int n = x.pieces(piece);
    items += n;
    worst = fmaxf(worst, x.cost() / n);
    if (n > 1) parts += static_cast<int64_t>(n) * x.rows;
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    worst = fmaxf(worst, __shfl_xor_sync(~0u, worst, d));
    items += __shfl_xor_sync(~0u, items, d);
    parts += __shfl_xor_sync(~0u, parts, d);
  }
  if (lane == 0) {
    items *= heads;
    parts *= heads;
    const int rounds = (items + n_ctas - 1) / n_ctas;
    // writing and reading a partial row takes about 2e-3 of a unit on the whole machine
    float est = fmaxf(rounds * (items ? cost * heads / items + kItemCost : 0.0f), worst + kItemCost) +
                (parts ? kMergeCost + 1e-3f * parts : 0.0f);
    if (parts > to.max_parts) est = 1e30f;
    if (warp == 0) est = fminf(est, 1e29f);  // always possible
    sh_cost[warp] = est;
    sh_piece[warp] = piece;
    sh_worst[warp] = worst;
  }
  __syncthreads();
  int best = 0;
  for (int w = 1; w < kCandidates; ++w)
    if (sh_cost[w] < sh_cost[best]) best = w;
  const float c = sh_piece[best];

  // Where the pieces of each length begin, longest first, by counting: kPlanThreads classes.
  const float per_class = (kPlanThreads - 1) / fmaxf(sh_worst[best], 1.0f);
  auto class_of = [&](const Tile& x, int n) {
    return kPlanThreads - 1 - min(kPlanThreads - 1, static_cast<int>(x.cost() / n * per_class));
  };
  sh_at[tid] = 0;
  __syncthreads();
  for (int t = tid; t < n_tiles; t += kPlanThreads) {
    const Tile x = size_of(t);
    const int n = x.pieces(c);
    atomicAdd(&sh_at[class_of(x, n)], n);
  }
  __syncthreads();
  int first[1] = {sh_at[tid]}, all[1];
  scan(first, all, sh);
  sh_at[tid] = first[0];
  __syncthreads();

  int n_entries = 0, n_splits = 0, n_parts = 0, n_rows = 0;
  for (int t0 = 0; t0 < n_tiles; t0 += kPlanThreads) {
    const int t = t0 + tid;
    Tile x{};
    int n = 0;
    if (t < n_tiles) {
      x = tile_at(a, how, rep, base, t);
      n = x.pieces(c);
    }
    const int cut = n > 1 ? x.rows * heads : 0;
    int v[4] = {n, n > 1, n * cut, cut}, total[4];
    scan(v, total, sh);
    const int e0 = n ? atomicAdd(&sh_at[class_of(x, n)], n) : 0, part = n_parts + v[2];
    for (int i = 0; i < n && e0 + i < to.max_entries; ++i) {
      const int lo = static_cast<int>(static_cast<int64_t>(x.kv) * i / n);
      const int hi = static_cast<int>(static_cast<int64_t>(x.kv) * (i + 1) / n);
      to.entries[e0 + i] = {x.seq, x.row0, x.rows, lo, hi, n > 1 ? part + i * cut : -1, 0, 0};
    }
    if (n > 1) to.splits[n_splits + v[1]] = {x.seq, x.row0, x.rows, n, part, n_rows + v[3], 0, 0};
    n_entries += total[0];
    n_splits += total[1];
    n_parts += total[2];
    n_rows += total[3];
  }
  if (tid == 0) *to.plan = {min(n_entries, to.max_entries), n_splits, n_rows, 0};
}

// Merge of split rows, a warp per row: with M = max m_p and w_p = 2^(m_p - M),
// o = sum w_p o_p / sum w_p l_p.  It moves a few MB; what it costs is the launch.
constexpr int kMergeThreads = 256;
template <int D>
__global__ void __launch_bounds__(kMergeThreads)
extend_merge_kernel(const __grid_constant__ Params many, const __grid_constant__ Params few) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const ExtendArgs& a = many.a;
  const int lane = threadIdx.x & 31, heads = a.n_kv_heads;
  constexpr int E = D / 32;
  const int n_many = many.plan->split_rows, n_all = n_many + few.plan->split_rows;
  for (int i = (blockIdx.x * kMergeThreads + threadIdx.x) >> 5; i < n_all; i += gridDim.x * (kMergeThreads / 32)) {
    const Params& p = i < n_many ? many : few;
    const int g = i < n_many ? i : i - n_many;
    int lo = 0, hi = p.plan->n_splits - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.splits[mid].first <= g) lo = mid; else hi = mid - 1;
    }
    const Split s = p.splits[lo];
    const int head = (g - s.first) / s.rows, r = (g - s.first) - head * s.rows;
    const float* row = p.parts + (static_cast<int64_t>(s.part) + static_cast<int64_t>(head) * s.rows + r) * (D + 4);
    const int64_t step = static_cast<int64_t>(heads) * s.rows * (D + 4);
    float m = -INFINITY;
    for (int i = lane; i < s.pieces; i += 32) m = fmaxf(m, row[i * step + D]);
#pragma unroll
    for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    float l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    for (int i0 = 0; i0 < s.pieces; i0 += 32) {
      float w = 0.0f;
      if (i0 + lane < s.pieces) {
        const float mp = row[(i0 + lane) * step + D];
        w = mp == m ? 1.0f : exp2f(mp - m);
        l += w * row[(i0 + lane) * step + D + 1];
      }
      const int n = min(32, s.pieces - i0);
#pragma unroll 4
      for (int i = 0; i < n; ++i) {
        const float wi = __shfl_sync(~0u, w, i);
        const float* src = row + (i0 + i) * step + lane * E;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(wi, src[e], o[e]);
      }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) l += __shfl_xor_sync(~0u, l, d);
    const float inv = l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
    int first;
    extend_rows(a, s.seq, &first);
    const int flat = s.row0 + r, tok = flat / p.rep;
    const int64_t out_row = (static_cast<int64_t>(first) + tok) * a.n_q_heads + head * p.rep + (flat - tok * p.rep);
#pragma unroll
    for (int e = 0; e < E; ++e)
      store_elem_rt(a.out, out_row * a.out_row_stride + lane * E + e, o[e] * inv, a.out_dtype);
    if (a.lse && lane == 0) a.lse[out_row] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
  }
}

// Whether every cp.async and vector access of the kernel is aligned on this plane.
bool plane_aligned(const Plane& p, int head_dim) {
  for (int i = 0; i < 3; ++i)
    if (p.cs[i] % 16) return false;
  if (reinterpret_cast<uintptr_t>(p.codes) % 16) return false;
  if (p.mode == KNLP_KV_F16 || p.mode == KNLP_KV_BF16) return true;
  const int bytes = head_dim / 32 * 2;
  auto rows = [&](const __half* base, const int64_t* stride) {
    if (reinterpret_cast<uintptr_t>(base) % bytes) return false;
    for (int i = 0; i < 3; ++i)
      if (stride[i] * 2 % bytes) return false;
    return true;
  };
  return rows(p.scales, p.ss) && (p.mode != KNLP_KV_INT4_ASYM || rows(p.zeros, p.zs));
}

int launch_modes(const Params& p, const Params& few, bool only_few, int grid, cudaStream_t st) {
  const int k = p.a.k.mode == KNLP_KV_BF16 ? kRaw : p.a.k.mode, v = p.a.v.mode;
  if (k == KNLP_KV_INT4_ASYM && v == KNLP_KV_INT4_ASYM) return launch_extend_pair<KNLP_KV_INT4_ASYM, KNLP_KV_INT4_ASYM>(p, few, only_few, grid, st);
  if (k == KNLP_KV_INT4_SYM && v == KNLP_KV_INT4_SYM) return launch_extend_pair<KNLP_KV_INT4_SYM, KNLP_KV_INT4_SYM>(p, few, only_few, grid, st);
  if (k == KNLP_KV_INT8_G32 && v == KNLP_KV_INT4_ASYM) return launch_extend_pair<KNLP_KV_INT8_G32, KNLP_KV_INT4_ASYM>(p, few, only_few, grid, st);
  if (k == KNLP_KV_INT8_G32 && v == KNLP_KV_INT4_SYM) return launch_extend_pair<KNLP_KV_INT8_G32, KNLP_KV_INT4_SYM>(p, few, only_few, grid, st);
  if (k == KNLP_KV_INT8_G32 && v == KNLP_KV_INT8_G32) return launch_extend_pair<KNLP_KV_INT8_G32, KNLP_KV_INT8_G32>(p, few, only_few, grid, st);
  if (k == kRaw && v == KNLP_KV_INT4_ASYM) return launch_extend_pair<kRaw, KNLP_KV_INT4_ASYM>(p, few, only_few, grid, st);
  if (k == kRaw && v == KNLP_KV_INT4_SYM) return launch_extend_pair<kRaw, KNLP_KV_INT4_SYM>(p, few, only_few, grid, st);
  if (k == kRaw && v == KNLP_KV_INT8_G32) return launch_extend_pair<kRaw, KNLP_KV_INT8_G32>(p, few, only_few, grid, st);
  return 1;
}

bool pair_built(int k, int v) {
  const bool raw = k == KNLP_KV_F16 || k == KNLP_KV_BF16;
  return raw || k == KNLP_KV_INT8_G32 || k == v;
}

// Workspace, in ints / floats, for each kernel: plan, first tile of each sequence, pieces, splits,
// partial rows.
struct Sizes {
  Bounds bounds[2];
  int64_t at[2], entries_at[2], splits_at[2], parts_at[2], floats = 0;
  Sizes(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads, int head_dim, int n_sms)
      : bounds{{false, n_seqs, n_tokens, n_q_heads, n_kv_heads, n_sms}, {true, n_seqs, n_tokens, n_q_heads, n_kv_heads, n_sms}} {
    for (int i = 0; i < 2; ++i) {
      at[i] = floats;
      entries_at[i] = at[i] + (4 + n_seqs + 1 + 3) / 4 * 4;
      splits_at[i] = entries_at[i] + bounds[i].entries * 8;
      parts_at[i] = splits_at[i] + bounds[i].tiles * 8;
      floats = parts_at[i] + bounds[i].parts * (head_dim + 4);
    }
    floats += 4;  // alignment of the start
  }
};

}  // namespace
}  // namespace extend

int64_t extend_workspace_floats(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads,
                                int head_dim, int n_sms) {
  return extend::Sizes(n_seqs, n_tokens, n_q_heads, n_kv_heads, head_dim, n_sms).floats;
}

int launch_extend_mma(const ExtendArgs& a, int max_query_len, int max_seq_len, float* ws,
                      int64_t ws_floats, int n_sms, cudaStream_t st) {
  using namespace extend;
  if (a.head_dim != 64 && a.head_dim != 128) return 1;
  if (!pair_built(a.k.mode, a.v.mode)) return 1;
  if (!plane_aligned(a.k, a.head_dim) || !plane_aligned(a.v, a.head_dim)) return 1;
  const int out_size = a.out_dtype == KNLP_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(a.q) % 16 || a.q_stride[0] % 8 || a.q_stride[1] % 8) return 1;
  if (reinterpret_cast<uintptr_t>(a.out) % 16 || a.out_row_stride * out_size % 16) return 1;
  if (static_cast<int64_t>(a.n_tokens) * a.n_q_heads > (1 << 30)) return 1;
  const uintptr_t mis = reinterpret_cast<uintptr_t>(ws) % 16;
  if (mis % 4) return KNLP_ERR_STRIDE;
  if (mis) ws += (16 - mis) / 4;
  const Sizes z(a.n_seqs, a.n_tokens, a.n_q_heads, a.n_kv_heads, a.head_dim, n_sms);
  if (ws_floats < z.floats) return KNLP_ERR_WORKSPACE;
  Params p[2]{};
  Lists lists[2];
  for (int i = 0; i < 2; ++i) {
    Lists& l = lists[i];
    l.max_entries = static_cast<int>(z.bounds[i].entries);
    l.max_tiles = static_cast<int>(z.bounds[i].tiles);
    l.max_parts = z.bounds[i].parts;
    l.plan = reinterpret_cast<Plan*>(ws + z.at[i]);
    l.base = reinterpret_cast<int*>(ws + z.at[i] + 4);
    l.entries = reinterpret_cast<Entry*>(ws + z.entries_at[i]);
    l.splits = reinterpret_cast<Split*>(ws + z.splits_at[i]);
    p[i].a = a;
    p[i].plan = l.plan;
    p[i].entries = l.entries;
    p[i].splits = l.splits;
    p[i].parts = ws + z.parts_at[i];
    p[i].status = decode_status_ptr();
    if (!p[i].status) return KNLP_ERR_NO_DEVICE;
    p[i].rep = a.n_q_heads / a.n_kv_heads;
    p[i].block_shift = -1;
    for (int b = 0; b < 31; ++b)
      if (a.block_size == 1 << b) p[i].block_shift = b;
  }
  // The host's bounds save launches; the plan keeps to what is launched, so bounds that are too
  // small cost time, never rows or tokens.  Up to 32 rows per sequence: the kernel for many rows is
  // left out and longer sequences are cut into 32s.  Up to three tiles of cached tokens: pieces
  // are not made and the merge is left out.
  const bool only_few = static_cast<int64_t>(max_query_len < a.n_tokens ? max_query_len : a.n_tokens) * p[0].rep <= few::kFewRows;
  const bool whole = max_seq_len <= 3 * kTile;
  extend_plan_kernel<<<2, kPlanThreads, 0, st>>>(a, p[0].rep, n_sms, only_few, whole, lists[0], lists[1]);
  if (cudaGetLastError() != cudaSuccess) return KNLP_ERR_LAUNCH;
  const int rc = launch_modes(p[0], p[1], only_few, n_sms, st);
  if (rc != KNLP_OK) return rc > 0 ? KNLP_ERR_MODE : rc;
  if (whole) return KNLP_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(2 * n_sms);
  cfg.blockDim = dim3(kMergeThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = a.head_dim == 64 ? cudaLaunchKernelEx(&cfg, extend_merge_kernel<64>, p[0], p[1])
                                           : cudaLaunchKernelEx(&cfg, extend_merge_kernel<128>, p[0], p[1]);
  if (err != cudaSuccess) {
    cudaGetLastError();
    return KNLP_ERR_LAUNCH;
  }
  return KNLP_OK;
}

}  // namespace knlp
