// The extend attention of few query rows (at most 32 per kv head: single tokens, drafted tokens),
// on the fifth-generation tensor cores with the cached TOKENS on M and the rows on N:
//
//   S^T = K Q^T  (128 tokens x 32 rows),   P^T = exp2(c S^T - m),   O^T += V^T P^T  (head_dim x 32),
//   l += 1 P^T  (a product with ones: every lane of the accumulator holds the column sums)
//
// What bounds it: a tile of 128 tokens is 20 KB, 890 cycles at the SM's share of the measured
// bandwidth, and 32 K values to convert; measured 2200 cycles a tile with 65 % of the issue slots
// taken (3-8 new tokens x 16 sequences on 8-32 K cached tokens, 32/8 heads of 128, INT4: 175 us,
// 2.1 TB/s).  With rows on M, as the kernel for many rows has them, 3/4 of the products and of the
// softmax lanes serve nothing, on two of its eight softmax warps: the same case takes 280 us there.
// Here a tile's products take 3 x 320 tensor cycles at N = 32 and eight warps share its exponentials.
//
// One CTA per SM, 28 warps of at most 72 registers:
//   warps 0-3, 4-7  softmax, a thread per token of the tile; the second warpgroup has the upper
//                   half of the rows (in groups of eight).  Then the result, a thread per column
//                   of O, the rows dealt out to both
//   warps 8-23      dequantization: two warpgroups for K, two for V, every other tile each
//   warps 24, 25    issue the scores (four buffers, ahead of the softmax), the outputs
// Two operand slots per plane, each filled by its own warpgroup.  P^T goes through shared memory
// (64 bytes per token, 64-byte swizzle).
//
// The maximum of a row is spread over the lanes, so it is not formed per tile: a tile uses the
// reference m that it finds, one vote says whether any score exceeds it by 2^8, and only then
// (always in an item's first tile) the tile's maxima are taken and O and l rescaled.
#pragma once

#include "extend_mma.cuh"

namespace knlp {
namespace extend {
namespace few {

constexpr int kFewRows = 32;
constexpr int kFewThreads = 28 * 32;
constexpr int kScoreBuffers = 4;
constexpr float kLowest = -8192.0f;  // of scores in powers of two; sums with it keep 2^-11

// TMEM columns: four buffers of S^T, O^T, l, and a tile of ones (fp16 pairs) as an operand.
constexpr int kTmemO = kScoreBuffers * kFewRows, kTmemL = kTmemO + kFewRows, kTmemOnes = kTmemL + kFewRows;
constexpr int kTmemColumns = 256;
static_assert(kTmemOnes + kTile / 2 <= kTmemColumns, "");

template <int KM, int VM, int D>
struct FewLayout {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kK = KM == kRaw ? 0 : PlaneTile<KM, D>::kBytes, kV = PlaneTile<VM, D>::kBytes;
  static constexpr int kQ = 0;
  static constexpr int kP = kFewRows * D * 2;
  static constexpr int kKV = kP + kTile * kFewRows * 2;  // K slots 0, 1, V slots 0, 1
  static constexpr int kStageK = kKV + 4 * kTileBytes;
  static constexpr int kRoom = 232448 - 1024 - kMiscBytes - kStageK;
  // stages of a warpgroup: as many as fit, V's (or K's) second one if only one of them does
  static constexpr int kBoth = kRoom / (2 * (kK + kV)) < 4 ? kRoom / (2 * (kK + kV)) : 4;
  static constexpr int kLeft = kRoom - kBoth * 2 * (kK + kV);
  static constexpr int kMoreK = kBoth < 4 && kK && kLeft >= 2 * kK;
  static constexpr int kStagesK = kK ? kBoth + kMoreK : 0;
  static constexpr int kStagesV = kBoth + (kBoth < 4 && kK && !kMoreK && kLeft >= 2 * kV);
  static_assert(kBoth >= 1, "a stage of each warpgroup has to fit");
  static constexpr int kStageV = kStageK + 2 * kStagesK * kK;
  static constexpr int kMisc = (kStageV + 2 * kStagesV * kV + 127) / 128 * 128;
  static constexpr int kBytes = kMisc + kMiscBytes + 1024;
  static_assert(kBytes <= 232448, "shared memory of an SM");
};

struct FewMisc {
  uint64_t full[2][2], empty[2][2];  // [plane][slot]
  uint64_t q_full, s_full[kScoreBuffers], s_free[kScoreBuffers], p_full, p_free, o_full;
  uint32_t tmem;
  int abort;
  // per query row
  alignas(16) float off[kFewRows];  // -m, the reference of its exponents; read as float4
  float delta[kFewRows], factor[kFewRows];  // what a rescaling adds to m, 2^-delta
  float most[4][kFewRows];  // maxima of the warps
  int limit[kFewRows];      // cached tokens that it attends to
  int64_t out_row[kFewRows];
  BadList bad[kBadLists];
};
static_assert(sizeof(FewMisc) <= kMiscBytes, "");

constexpr uint32_t kProbsHigh = 512 >> 4 | 1u << 14 | 4u << 29;  // 64-byte swizzle, 8 tokens 512 bytes

// D (+)= A B with A in shared memory and B in shared memory; HB: high word of B's descriptor.
template <int OFFA, int OFFB, uint32_t HB>
__device__ __forceinline__ void mma_ss2(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b32 x, y;\n.reg .b64 da, db;\n"
      "add.u32 x, %1, %5;\nadd.u32 y, %2, %6;\n"
      "mov.b64 da, {x, %7};\nmov.b64 db, {y, %8};\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "n"(OFFA), "n"(OFFB), "n"(kOperandHigh), "n"(HB) : "memory");
}
// The same with A in TMEM.
template <int COL, int OFFB, uint32_t HB>
__device__ __forceinline__ void mma_ts2(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b32 x, y;\n.reg .b64 db;\n"
      "add.u32 x, %1, %5;\nadd.u32 y, %2, %6;\n"
      "mov.b64 db, {y, %7};\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "n"(COL), "n"(OFFB), "n"(HB) : "memory");
}
constexpr uint32_t kAisMn = 1u << 15;  // instruction descriptor: A is MN-major

// Of a warpgroup of the softmax, and of both.
__device__ __forceinline__ bool any_of_128(int id, bool x) {
  uint32_t r;
  asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbarrier.cta.red.or.pred q, %2, 128, p;\nselp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"(static_cast<uint32_t>(x)), "r"(id) : "memory");
  return r;
}
__device__ __forceinline__ void sync_128(int id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void sync_256() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Every other tile of a plane, counted over all items, by one warpgroup into its own slot.  The
// warpgroups of a plane, and planes of one mode, run the same code (see produce).
template <class L, int MODE, int D, int STAGES>
__device__ __forceinline__ void few_produce(const Params& p, char* sm, FewMisc& mi, int n_items, int side, int phase, int w, int lane) {
  using T = PlaneTile<MODE, D>;
  constexpr int kStages = STAGES;
  char* const stages = sm + (side ? L::kStageV : L::kStageK) + phase * kStages * T::kBytes;
  char* const to = sm + L::kKV + (side * 2 + phase) * L::kTileBytes;
  const int row = w * 32 + lane;
  Copies<MODE, D, 2> copies(p, side ? p.a.v : p.a.k, n_items, w, lane, phase);
  for (int i = 0; i < kStages; ++i) copies.next(stages + i * T::kBytes);
  uint32_t count = 0, use = 0, stage = 0;
  int serial = 0;
  for (int r = 0, ki; (ki = item_of(r)) < n_items; ++r) {
    const Item it(p, ki);
    const int n = it.tiles();
    if (n == 0) continue;
    BadList& bad = mi.bad[serial % kBadLists];
    if (side) {
      if (phase == 0 && row == 0) bad.clear();
      asm volatile("bar.sync 3, 256;" ::: "memory");  // both warpgroups of V
    }
    for (int j = (count & 1) != phase; j < n; j += 2, ++use) {
      if constexpr (kStages == 0) {
        mbar_wait(&mi.empty[side][phase], (use + 1) & 1, &mi.abort, p.status);
        copies.next(to);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        char* const from = stages + stage * T::kBytes;
        if constexpr (T::kQuant) {
          if (side && any_not_finite<MODE, D>(from, row)) bad.note<MODE, D>(from, row, (it.e.tile0 + j) * kTile + row);
        }
        mbar_wait(&mi.empty[side][phase], (use + 1) & 1, &mi.abort, p.status);
        dequantize_row<MODE, D>(from, to, row);
      }
      fence_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&mi.full[side][phase]);
      if constexpr (kStages > 0) {
        copies.next(stages + stage * T::kBytes);
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
    }
    count += n;
    ++serial;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int KM, int VM, int D>
__global__ void __launch_bounds__(kFewThreads, 1) extend_few_kernel(const __grid_constant__ Params p) {
  using L = FewLayout<KM, VM, D>;
  extern __shared__ char smem_raw[];
  char* sm = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  FewMisc& mi = *reinterpret_cast<FewMisc*>(sm + L::kMisc);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const ExtendArgs& a = p.a;

  if (tid == 0) {
    for (int s = 0; s < 2; ++s)
      for (int i = 0; i < 2; ++i) mbar_init(&mi.full[s][i], 4), mbar_init(&mi.empty[s][i], 1);
    for (int i = 0; i < kScoreBuffers; ++i) mbar_init(&mi.s_full[i], 1), mbar_init(&mi.s_free[i], 8);
    mbar_init(&mi.q_full, 8);
    mbar_init(&mi.p_full, 8);
    mbar_init(&mi.p_free, 1);
    mbar_init(&mi.o_full, 1);
    mi.abort = 0;
    for (int i = 0; i < kBadLists; ++i) mi.bad[i].clear();
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 24) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&mi.tmem)), "n"(kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = mi.tmem;
  const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
  if (warp < 4) {
    uint32_t ones[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) ones[i] = 0x3c003c00u;
#pragma unroll
    for (int i = 0; i < kTile / 2; i += 16) tmem_st16(tmem + lanes + kTmemOnes + i, ones);
    tmem_wait_st();
  }
  fence_before();
  __syncthreads();
  fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_items = p.plan->n_entries * a.n_kv_heads;
  auto wait = [&](uint64_t* b, uint32_t phase) { mbar_wait(b, phase & 1, &mi.abort, p.status); };

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax and results
    const float c = a.scale * kLog2e;
    const int wg = warp >> 2, tok128 = tid & 127, bar = 4 + wg;
    uint32_t count = 0, n_o = 0;  // tiles, items with tiles so far
    for (int r = 0, k; (k = item_of(r)) < n_items; ++r) {
      const Item it(p, k);
      const int rows = it.e.rows, n = it.tiles();
      sync_256();  // the last item's tables and query are not in use any more
      if (tid < kFewRows) {
        const int flat = it.e.row0 + tid, tok = flat / p.rep;
        mi.limit[tid] = tid >= rows ? 0 : a.causal ? max(min(it.ctx + tok + 1, it.len), 0) : it.len;
        mi.out_row[tid] = (static_cast<int64_t>(it.first) + tok) * a.n_q_heads + it.head * p.rep + (flat - tok * p.rep);
        mi.off[tid] = 0.0f;
      }
      if (n) {
        constexpr int kPer = D / 8;  // 16-byte chunks of a row
#pragma unroll
        for (int i0 = 0; i0 < kFewRows * kPer; i0 += 256) {
          const int i = i0 + tid, r = i / kPer, chunk = i % kPer;
          uint4 v = make_uint4(0, 0, 0, 0);
          if (r < rows) {
            const int f = it.e.row0 + r, t = f / p.rep;
            const int64_t off = (static_cast<int64_t>(it.first) + t) * a.q_stride[0] +
                                (static_cast<int64_t>(it.head) * p.rep + (f - t * p.rep)) * a.q_stride[1];
            v = reinterpret_cast<const uint4*>(static_cast<const char*>(a.q) + 2 * off)[chunk];
          }
          *reinterpret_cast<uint4*>(sm + L::kQ + (chunk >> 3) * (kFewRows * 128) + r * 128 +
                                    (((chunk & 7) ^ (r & 7)) << 4)) = query_operand<KM>(v, a.q_dtype);
        }
        fence_smem();
      }
      sync_256();
      if (n && lane == 0) mbar_arrive(&mi.q_full);
      // the fewest tokens that a row attends to: tiles below it need no mask
      const int least = __reduce_min_sync(~0u, lane < rows ? mi.limit[lane] : 0x7fffffff);
      // this warpgroup's rows: `mine` from `from` on, in groups of eight
      const int groups = (rows + 7) / 8, lower = (groups + 1) / 2;
      const int from = wg * lower * 8, mine = wg ? groups - lower : lower;
      const int held = min(rows - from, mine * 8);

      // The scores of the next tile are on their way while this one's P is handed over.
      constexpr int kMine = kFewRows / 2;
      float s[kMine];
      auto ask = [&](uint32_t tile) {
        const uint32_t b = tile % kScoreBuffers;
        wait(&mi.s_full[b], tile / kScoreBuffers);
        fence_after();
        tmem_ld16(tmem + lanes + b * kFewRows + from, reinterpret_cast<uint32_t*>(s));
      };
      if (n) ask(count);
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++count) {
        const int token = (it.e.tile0 + j) * kTile + tok128;
        tmem_wait_ld16(reinterpret_cast<uint32_t*>(s));
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&mi.s_free[count % kScoreBuffers]);
        uint32_t pk[kMine / 2];
        if (mine) {
          if ((it.e.tile0 + j + 1) * kTile > least) {
#pragma unroll
            for (int x = 0; x < kMine; ++x) s[x] = token < mi.limit[from + x] ? s[x] : -INFINITY;
          }
          float top = -INFINITY;
#pragma unroll
          for (int g = 0; g < kMine / 8; ++g) {
            if (g >= mine) break;
            const float4 o0 = *reinterpret_cast<const float4*>(&mi.off[from + g * 8]);
            const float4 o1 = *reinterpret_cast<const float4*>(&mi.off[from + g * 8 + 4]);
            const float o[8] = {o0.x, o0.y, o0.z, o0.w, o1.x, o1.y, o1.z, o1.w};
#pragma unroll
            for (int x = 0; x < 8; ++x) s[g * 8 + x] = fmaf(s[g * 8 + x], c, o[x]);
#pragma unroll
            for (int x = 0; x < 8; x += 2) top = max3(top, s[g * 8 + x], s[g * 8 + x + 1]);
          }
          if (any_of_128(bar, j == 0 || top > kGrow)) {
            // maxima of the tile's columns, relative to the references
#pragma unroll
            for (int x = 0; x < kMine; ++x) {
              if (x >= held) break;
              float v;
              asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(v) : "f"(s[x]));
              if (lane == 0) mi.most[warp & 3][from + x] = v;
            }
            sync_128(bar);
            if (tok128 < mine * 8) {
              const int x = from + tok128;
              float v = -INFINITY;
              if (tok128 < held) v = fmaxf(fmaxf(mi.most[0][x], mi.most[1][x]), fmaxf(mi.most[2][x], mi.most[3][x]));
              // a row whose scores are all -inf so far: a real one will lie above its reference
              const float first = v > -INFINITY ? v : tok128 < held ? kLowest : 0.0f;
              const float by = j == 0 ? first : fmaxf(v, 0.0f);
              mi.delta[x] = by;
              mi.factor[x] = exp2f(-by);
              mi.off[x] -= by;
            }
            sync_128(bar);
            if (j > 0) {
              wait(&mi.p_free, count - 1);  // the outputs so far are done
              fence_after();
#pragma unroll 1
              for (int x0 = 0; x0 < mine * 8; x0 += 4) {
#pragma unroll 1
                for (int acc = kTmemO; acc <= kTmemL; acc += kFewRows) {
                  uint32_t o[4];
                  tmem_ld4(tmem + lanes + acc + from + x0, o);
                  tmem_wait_ld4(o);
#pragma unroll
                  for (int x = 0; x < 4; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * mi.factor[from + x0 + x]);
                  tmem_st4(tmem + lanes + acc + from + x0, o);
                }
              }
              tmem_wait_st();
            }
#pragma unroll
            for (int x = 0; x < kMine; ++x)
              if (x < mine * 8) s[x] -= mi.delta[from + x];
          }
#pragma unroll
          for (int g = 0; g < kMine / 8; ++g) {
            if (g >= mine) break;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              float p0, p1;
              asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(s[g * 8 + 2 * x]));
              asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(s[g * 8 + 2 * x + 1]));
              pk[g * 4 + x] = as_u32(__floats2half2_rn(p0, p1));
            }
          }
        }
        if (j + 1 < n) ask(count + 1);
        wait(&mi.p_free, count + 1);  // the product with the last tile's P is done
#pragma unroll
        for (int g = 0; g < kMine / 8; ++g) {
          if (g >= mine) break;
          *reinterpret_cast<uint4*>(sm + L::kP + tok128 * 64 + (((from / 8 + g) ^ ((tok128 >> 1) & 3)) << 4)) =
              make_uint4(pk[g * 4], pk[g * 4 + 1], pk[g * 4 + 2], pk[g * 4 + 3]);
        }
        fence_smem();
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&mi.p_full);
      }

      // a thread per column of O as the accumulator has it, 4 rows at a time, dealt out to the warpgroups
      if (n) {
        wait(&mi.o_full, n_o);
        fence_after();
      }
      const BadList& bad = mi.bad[n_o % kBadLists];
      constexpr bool kPaired = VM == KNLP_KV_INT4_SYM || VM == KNLP_KV_INT4_ASYM;
      const int d = kPaired ? (tok128 & ~7) + ((tok128 >> 1) & 3) + 4 * (tok128 & 1) : tok128;
      const bool direct = it.e.part < 0;
      float* part = p.parts + (static_cast<int64_t>(it.e.part) + static_cast<int64_t>(it.head) * rows) * (D + 4);
#pragma unroll 1
      for (int x0 = wg * 4; x0 < rows; x0 += 8) {
        uint32_t ou[4], lu[4];
        if (n) {
          tmem_ld4(tmem + lanes + kTmemO + x0, ou);
          tmem_ld4(tmem + lanes + kTmemL + x0, lu);
          tmem_wait_ld4(ou);
          tmem_wait_ld4(lu);
        } else {
#pragma unroll
          for (int x = 0; x < 4; ++x) ou[x] = lu[x] = 0;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = x0 + x;
          if (row >= rows) break;
          const float l = __uint_as_float(lu[x]);
          float v = __uint_as_float(ou[x]);
          if (direct) v *= l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
          if (n && bad.count && bad.hits(mi.limit[row], d / 32)) v = NAN;  // never in a healthy cache
          if (direct) {
            if (tok128 < D) store_elem_rt(a.out, mi.out_row[row] * a.out_row_stride + d, v, a.out_dtype);
            if (tok128 == row && a.lse) a.lse[mi.out_row[row]] = l == 0.0f ? -INFINITY : kLn2 * (log2f(l) - mi.off[row]);
          } else {
            if (tok128 < D) part[row * (D + 4) + d] = v;
            // a piece that holds nothing for the row does not weigh
            if (tok128 == row) part[row * (D + 4) + D] = l == 0.0f ? -INFINITY : -mi.off[row], part[row * (D + 4) + D + 1] = l;
          }
        }
      }
      fence_before();
      n_o += n > 0;
    }
  } else if (warp < 24) {
    const int wg = (warp - 8) >> 2;  // K, K, V, V
    if constexpr (KM == VM && L::kStagesK == L::kStagesV) {
      few_produce<L, KM, D, L::kStagesK>(p, sm, mi, n_items, wg >> 1, wg & 1, warp & 3, lane);
    } else {
      if (wg < 2) few_produce<L, KM, D, L::kStagesK>(p, sm, mi, n_items, 0, wg, warp & 3, lane);
      else few_produce<L, VM, D, L::kStagesV>(p, sm, mi, n_items, 1, wg - 2, warp & 3, lane);
    }
  } else if (warp < 26) {
    // ---------------------------------------------------------------- matrix products
    auto wait_warp = [&](uint64_t* x, uint32_t phase) { mbar_wait_warp(x, phase & 1, &mi.abort, p.status); };
    const uint32_t tm = uniform(tmem);
    const int n_all = uniform(n_items);
    uint32_t count = 0, n_q = 0;
    for (int r = 0, k; (k = item_of(r)) < n_all; ++r) {
      const Item it(p, k);
      const int n = uniform(it.tiles());
      if (n == 0) continue;
      if (warp == 24) {
        const uint32_t idesc = product(kTile, kFewRows, KM == kRaw && a.k.mode == KNLP_KV_BF16, false);
        const uint32_t q = operand(smem_addr(sm + L::kQ), 16);
        wait_warp(&mi.q_full, n_q++);
        fence_after();
        for (int j = 0; j < n; ++j, ++count) {
          const uint32_t b = count % kScoreBuffers, slot = count & 1;
          const uint32_t kk = operand(smem_addr(sm + L::kKV), 16) + slot * (L::kTileBytes >> 4);
          wait_warp(&mi.full[0][slot], count >> 1);
          wait_warp(&mi.s_free[b], count / kScoreBuffers + 1);
          fence_after();
          if (elect()) {
            auto step = [&](auto i) {
              constexpr int s = decltype(i)::value;
              mma_ss2<((s >> 2) * (kTile * 128) + (s & 3) * 32) / 16, ((s >> 2) * (kFewRows * 128) + (s & 3) * 32) / 16, kOperandHigh>(
                  tm + b * kFewRows, kk, q, idesc, s > 0);
            };
            step(Int<0>{}), step(Int<1>{}), step(Int<2>{}), step(Int<3>{});
            if constexpr (D == 128) step(Int<4>{}), step(Int<5>{}), step(Int<6>{}), step(Int<7>{});
            commit(&mi.s_full[b]);
            commit(&mi.empty[0][slot]);
          }
          __syncwarp();
        }
      } else {
        constexpr uint32_t idesc_o = product(128, kFewRows, false, true) | kAisMn, idesc_l = product(128, kFewRows, false, true);
        const uint32_t pr = operand(smem_addr(sm + L::kP), 16);
        for (int j = 0; j < n; ++j, ++count) {
          const uint32_t slot = count & 1;
          // head_dim 64: the upper 64 rows of M repeat the lower ones (a block stride of 0)
          const uint32_t v = operand(smem_addr(sm + L::kKV) + 2 * L::kTileBytes, D == 128 ? kTile * 128 : 0) + slot * (L::kTileBytes >> 4);
          wait_warp(&mi.full[1][slot], count >> 1);
          wait_warp(&mi.p_full, count);
          fence_after();
          if (elect()) {
            auto step = [&](auto i) {
              constexpr int s = decltype(i)::value;
              mma_ss2<s * 2048 / 16, s * 1024 / 16, kProbsHigh>(tm + kTmemO, v, pr, idesc_o, j > 0 || s > 0);
              mma_ts2<s * 8, s * 1024 / 16, kProbsHigh>(tm + kTmemL, tm + kTmemOnes, pr, idesc_l, j > 0 || s > 0);
            };
            step(Int<0>{}), step(Int<1>{}), step(Int<2>{}), step(Int<3>{});
            step(Int<4>{}), step(Int<5>{}), step(Int<6>{}), step(Int<7>{});
            commit(&mi.p_free);
            commit(&mi.empty[1][slot]);
            if (j + 1 == n) commit(&mi.o_full);
          }
          __syncwarp();
        }
      }
    }
  }
  __syncwarp();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 24)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kTmemColumns) : "memory");
}

}  // namespace few
}  // namespace extend
}  // namespace knlp
