// Attention of several query tokens per sequence over the packed cache, on the fifth-generation
// tensor cores (tcgen05, accumulators in TMEM).
//
//   S = Q K^T,  P = exp2(c S - m),  O += P V   per 128 query rows x 128 cached tokens, online
//   maximum m and sum l per row;  o = O / l.  A query row is one (token, q head) of a kv head's
//   group, so all q heads of the group share every dequantized K / V tile.
//
// What bounds it: a 128 x 128 tile costs 2 x 512 tensor cycles at head_dim 128 and 1024 cycles of
// the SM's 16 ex2 per cycle; measured, the chain of a softmax step (TMEM load, maximum,
// exponentials, TMEM store, hand-over) beside them: 4096 new tokens at 28 000 cached ones, 32/8
// heads of 128, INT4: 2.19 ms, 910 TFLOP/s, 49 % tensor pipe, 49 % special function unit, 59 % issue slots.  Work
// items and their split over CTAs: extend_plan.cu.
//
// One CTA per SM (it owns all 512 TMEM columns), 20 warps whose registers are dealt out by
// setmaxnreg (2 x 136 + 2 x 80 + 48 = 5 x 96 a lane):
//   warps 0-3, 4-7   two softmax streams, a thread per query row, 64 cached tokens at a time.  An
//                    item of more than 128 rows gives each stream its own 128 rows over the
//                    same K / V tiles; a smaller one gives both streams the same rows and a
//                    half of every tile, and their states are merged at the end.  S has two
//                    buffers per stream: the next scores are made under the softmax
//   warps 8-11 (K),  dequantization: packed rows are staged with cp.async a few tiles ahead, turned
//   12-15 (V)        into fp16 and written as swizzled tensor-core operands into a ring of three
//                    tiles (K, V alternating).  An unquantized K tile is copied into the ring
//   warps 16, 17     (18, 19 idle) issue a stream's products: S = Q K^T from shared memory,
//                    O += P V with P read from TMEM, where it overlays its S
//
// Roundings, all chosen for the tensor cores' fp16 inputs: dequantized K and V, P and (from bf16)
// Q are rounded to fp16, 2^-11 relative each; products accumulate in fp32, m, l and O are fp32.
// fp16 is used instead of bf16 because its 2^-11 keeps the result within a bf16 rounding of the
// 64-bit one, and dequantized values fit its range (codes x an fp16 scale).  An unquantized K
// plane enters the product as it is stored.
//
// INT4 codes leave a 32-bit word as (n0, n4), (n1, n5), (n2, n6), (n3, n7): pairing nibbles four
// apart takes one AND-OR each.  K keeps that order in the operand and Q is permuted alike; V
// keeps it too and the output columns are put back in order when they are stored.
//
// Every wait on a barrier is bounded: when one runs out, the CTA raises the status word and stops
// waiting (its results are then wrong, its control flow and addresses stay as they are).
#pragma once

#include "pair_math.cuh"
#include "serve.cuh"

namespace knlp {
namespace extend {

constexpr int kRows = 128;   // query rows of a stream
constexpr int kTile = 128;   // cached tokens of a K / V tile
constexpr int kStep = 64;    // of a softmax step
constexpr int kRing = 3;
constexpr int kThreads = 20 * 32;
constexpr int kMiscBytes = 2048;
constexpr int kBadLists = 4, kBadMost = 15;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// O is rescaled only when a row's maximum has grown by more than this (in powers of two): P
// then stays below 2^8, far inside fp16, and most tiles skip the pass over O.
constexpr float kGrow = 8.0f;

// Modes of a plane inside the kernel: KNLP_KV_* with both unquantized K types as kRaw.
constexpr int kRaw = KNLP_KV_F16;

// A piece of work: query rows [row0, row0 + rows) of a sequence (a row = token x group head),
// tiles [tile0, tile1) of its cached tokens, for each of the kv heads in turn.
struct Entry {
  int seq, row0, rows, tile0, tile1;
  int part;  // first row in the partial buffer of kv head 0, or -1: the piece is the whole range
  int pad0, pad1;
};

// A tile of rows whose range was cut: pieces lie at part + (piece * heads + head) * rows.
struct Split {
  int seq, row0, rows, pieces, part;
  int first;  // rows x heads of the splits before
  int pad0, pad1;
};

struct Plan {
  int n_entries, n_splits, split_rows, pad;
};

struct Params {
  ExtendArgs a;
  const Plan* plan;
  const Entry* entries;
  const Split* splits;
  float* parts;  // rows of head_dim + 4 floats: o (relative to 2^m), m, l, -, -
  int* status;
  int rep;          // q heads per kv head
  int block_shift;  // log2 of the block size, -1 if it is no power of two
};

template <int MODE, int D>
struct PlaneTile {
  static constexpr bool kQuant = MODE != kRaw;
  static constexpr int kRowBytes = MODE == kRaw ? 2 * D : MODE == KNLP_KV_INT8_G32 ? D : D / 2;
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kScaleBytes = D / 32 * 2;
  static constexpr int kScaleAt = kTile * kRowBytes;
  static constexpr int kZeroAt = kScaleAt + (kQuant ? kTile * kScaleBytes : 0);
  static constexpr int kBytes = kZeroAt + (MODE == KNLP_KV_INT4_ASYM ? kTile * kScaleBytes : 0);
  // position of a 16-byte chunk in its row, such that eight rows' equal chunks hit all banks
  static __device__ __forceinline__ int at(int row, int chunk) {
    constexpr int n = kChunks;
    const int f = n >= 8 ? row & 7 : (row / (8 / (n < 8 ? n : 8))) & (n - 1);
    return row * kRowBytes + ((chunk ^ f) << 4);
  }
};

template <int KM, int VM, int D>
struct Layout {
  static constexpr int kTileBytes = kTile * D * 2;  // one fp16 operand tile, also a Q tile
  static constexpr int kRoom = 232448 - 1024 - kMiscBytes - (2 + kRing) * kTileBytes;
  static constexpr int kK = KM == kRaw ? 0 : PlaneTile<KM, D>::kBytes, kV = PlaneTile<VM, D>::kBytes;
  static constexpr int kBoth = kRoom / (kK + kV) < 5 ? kRoom / (kK + kV) : 5;
  static constexpr int kLeft = kRoom - kBoth * (kK + kV);
  static constexpr int kStagesK = kK == 0 ? 0 : kBoth + (kBoth < 5 && kLeft >= kK);
  static constexpr int kStagesV = kBoth + (kBoth < 5 && kLeft - (kStagesK - kBoth) * kK >= kV && kK != 0);
  static_assert(kBoth >= 1, "a plane tile of each kind has to fit");
  static constexpr int kQ = 0;
  static constexpr int kRingAt = 2 * kTileBytes;
  static constexpr int kStageK = kRingAt + kRing * kTileBytes;
  static constexpr int kStageV = kStageK + kStagesK * kK;
  static constexpr int kMisc = (kStageV + kStagesV * kV + 127) / 128 * 128;
  static constexpr int kBytes = kMisc + kMiscBytes + 1024;  // 1024 for the alignment of the base
  static_assert(kBytes <= 232448, "shared memory of an SM");
};

template <int N>
struct Int {
  static constexpr int value = N;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint64_t* b, int n) {
  asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(smem_addr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(smem_addr(b)) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
      "selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok) : "r"(smem_addr(b)), "r"(parity) : "memory");
  return ok;
}
// Waits for the phase, at most about two seconds; then, or once another wait of the CTA has
// given up, returns at once with the CTA's abort flag and the status word set.
__device__ __forceinline__ void mbar_wait_long(uint64_t* b, uint32_t parity, volatile int* abort,
                                            int* status) {
  uint64_t t0, t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t0));
  while (!mbar_try(b, parity)) {
    if (*abort) return;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    if (t - t0 > 2000000000ull) {
      *abort = 1;
      atomicExch(status, 1);
      return;
    }
  }
}
__device__ __forceinline__ void mbar_wait(uint64_t* b, uint32_t parity, int* abort, int* status) {
  if (!mbar_try(b, parity)) mbar_wait_long(b, parity, abort, status);
}

// A value that all lanes hold, in a uniform register: descriptors made from it need no moves.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __reduce_or_sync(~0u, x); }
// The same wait for a converged warp, with a uniform branch.
__device__ __forceinline__ void mbar_wait_warp(uint64_t* b, uint32_t parity, int* abort, int* status) {
  if (!__all_sync(~0u, mbar_try(b, parity))) {
    mbar_wait_long(b, parity, abort, status);
    __syncwarp();
  }
}

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(b)) : "memory");
}

// 32 TMEM columns of the warp's 32 lanes, a lane's row per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// The wait names the registers of the load, so that no use of them moves above it.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :: "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Shared-memory operand descriptor, 128-byte swizzle, groups of eight 128-byte rows 1024 bytes
// apart.  K-major operands (Q, K): a row per query row / token.  MN-major operand (V as stored, a
// row per token): `lead` bytes between blocks of 64 columns.  Only the low word varies.
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t addr, int lead) {
  return addr >> 4 | static_cast<uint32_t>(lead >> 4) << 16;
}
// Instruction descriptor: fp32 accumulator, fp16 or bf16 inputs, B optionally MN-major.
__host__ __device__ constexpr uint32_t product(int m, int n, bool bf16, bool b_mn) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (b_mn ? 1u << 16 : 0u) |
         static_cast<uint32_t>(n >> 3) << 17 | static_cast<uint32_t>(m >> 4) << 24;
}
// D (+)= A B, both operands in shared memory at OFF 16-byte units behind a and b.  The
// descriptors are put together here: kept outside they would not fit the warp's registers.
template <int OFF>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b32 x, y;\n.reg .b64 da, db;\n"
      "add.u32 x, %1, %5;\nadd.u32 y, %2, %5;\n"
      "mov.b64 da, {x, %6};\nmov.b64 db, {y, %6};\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "n"(OFF), "n"(kOperandHigh) : "memory");
}
// The same with A in TMEM, at COL columns behind a.
template <int COL, int OFF>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\n.reg .b32 x, y;\n.reg .b64 db;\n"
      "add.u32 x, %1, %7;\nadd.u32 y, %2, %5;\n"
      "mov.b64 db, {y, %6};\nsetp.ne.u32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [x], db, %3, p;\n}"
      ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(acc)), "n"(OFF), "n"(kOperandHigh), "n"(COL) : "memory");
}

// One lane of the converged warp.
__device__ __forceinline__ bool elect() {
  uint32_t e;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(e));
  return e;
}

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool there) {
  const int n = there ? BYTES : 0;  // what is not there is filled with zeros
  if constexpr (BYTES == 16) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  } else {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
  }
}

__device__ __forceinline__ __half2 as_half2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld16(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
      :: "memory");
}
__device__ __forceinline__ void tmem_ld4(uint32_t addr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t addr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};"
               ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld4(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]) :: "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Eight 4-bit codes as fp16 integers, in the order (n0 n4)(n1 n5)(n2 n6)(n3 n7), less 8 when
// symmetric.  A nibble under the exponent of 1024 is 1024 + n (or + 16 n one nibble up); the
// subtraction and the scaling by 1/16 are exact.
template <bool SYM>
__device__ __forceinline__ void nibbles(uint32_t w, __half2* h) {
  const __half2 low = as_half2(SYM ? 0xe408e408u : 0xe400e400u);   // -1024 (- 8)
  const __half2 high = as_half2(SYM ? 0xd480d480u : 0xd400d400u);  // -64 (- 8)
  const __half2 sixteenth = as_half2(0x2c002c00u);
  const uint32_t w8 = w >> 8;
  h[0] = __hadd2(as_half2((w & 0x000f000fu) | 0x64006400u), low);
  h[1] = __hfma2(as_half2((w & 0x00f000f0u) | 0x64006400u), sixteenth, high);
  h[2] = __hadd2(as_half2((w8 & 0x000f000fu) | 0x64006400u), low);
  h[3] = __hfma2(as_half2((w8 & 0x00f000f0u) | 0x64006400u), sixteenth, high);
}

// One row of a staged plane tile as an operand row: 16-byte chunk c of a 64-column box goes to
// chunk c ^ (row & 7).  A value is rounded once, from code x scale (+ zero) to fp16.
template <int MODE, int D>
__device__ __forceinline__ void dequantize_row(const char* stage, char* tile, int row) {
  using P = PlaneTile<MODE, D>;
  auto put = [&](int chunk, uint4 v) {  // chunk: 8 elements of the row
    *reinterpret_cast<uint4*>(tile + (chunk >> 3) * (kTile * 128) + row * 128 +
                              (((chunk & 7) ^ (row & 7)) << 4)) = v;
  };
  {
    constexpr int G = D / 32;
    __half2 s[G / 2], z[G / 2];
#pragma unroll
    for (int g = 0; g < G / 2; ++g) {
      s[g] = reinterpret_cast<const __half2*>(stage + P::kScaleAt + row * P::kScaleBytes)[g];
      if constexpr (MODE == KNLP_KV_INT4_ASYM)
        z[g] = reinterpret_cast<const __half2*>(stage + P::kZeroAt + row * P::kScaleBytes)[g];
    }
    auto pick = [](const __half2* v, int g) { return g & 1 ? __high2half2(v[g >> 1]) : __low2half2(v[g >> 1]); };
#pragma unroll
    for (int c = 0; c < P::kChunks; ++c) {
      const int g = MODE == KNLP_KV_INT8_G32 ? c >> 1 : c;
      const uint4 w = *reinterpret_cast<const uint4*>(stage + P::at(row, c));
      const __half2 sc = pick(s, g);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
      if constexpr (MODE == KNLP_KV_INT8_G32) {  // 16 codes, half a group
        const __half2 bias = as_half2(0xe480e480u);  // -1152: the codes are biased by 128
        uint32_t o[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = u[i] ^ 0x80808080u;
          o[2 * i] = as_u32(__hmul2(__hadd2(as_half2(__byte_perm(x, 0x64646464u, 0x4140)), bias), sc));
          o[2 * i + 1] = as_u32(__hmul2(__hadd2(as_half2(__byte_perm(x, 0x64646464u, 0x4342)), bias), sc));
        }
        put(2 * c, make_uint4(o[0], o[1], o[2], o[3]));
        put(2 * c + 1, make_uint4(o[4], o[5], o[6], o[7]));
      } else {  // 32 codes, one group
        __half2 zc;
        if constexpr (MODE == KNLP_KV_INT4_ASYM) zc = pick(z, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          __half2 h[4];
          nibbles<MODE == KNLP_KV_INT4_SYM>(u[i], h);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (MODE == KNLP_KV_INT4_ASYM) h[k] = __hfma2(h[k], sc, zc);
            else h[k] = __hmul2(h[k], sc);
          }
          put(4 * c + i, make_uint4(as_u32(h[0]), as_u32(h[1]), as_u32(h[2]), as_u32(h[3])));
        }
      }
    }
  }
}

// Whether a scale or zero-point of a staged V row is not finite (x * 0 is then NaN).
template <int MODE, int D>
__device__ __forceinline__ bool any_not_finite(const char* stage, int row) {
  using P = PlaneTile<MODE, D>;
  __half2 t = __float2half2_rn(0.0f);
#pragma unroll
  for (int g = 0; g < D / 64; ++g) {
    t = __hfma2(reinterpret_cast<const __half2*>(stage + P::kScaleAt + row * P::kScaleBytes)[g], __float2half2_rn(0.0f), t);
    if constexpr (MODE == KNLP_KV_INT4_ASYM)
      t = __hfma2(reinterpret_cast<const __half2*>(stage + P::kZeroAt + row * P::kScaleBytes)[g], __float2half2_rn(0.0f), t);
  }
  return !__hbeq2(t, t);
}

// The groups that are concerned, as a mask.
template <int MODE, int D>
__device__ __forceinline__ int not_finite(const char* stage, int row) {
  using P = PlaneTile<MODE, D>;
  int mask = 0;
#pragma unroll
  for (int g = 0; g < D / 32; ++g) {
    uint16_t u = *reinterpret_cast<const uint16_t*>(stage + P::kScaleAt + row * P::kScaleBytes + 2 * g);
    bool bad = (u & 0x7c00) == 0x7c00;
    if constexpr (MODE == KNLP_KV_INT4_ASYM) {
      u = *reinterpret_cast<const uint16_t*>(stage + P::kZeroAt + row * P::kScaleBytes + 2 * g);
      bad |= (u & 0x7c00) == 0x7c00;
    }
    mask |= bad << g;
  }
  return mask;
}

// Eight elements of a query row as the product with a K operand of mode KM wants them: fp16 beside
// dequantized K, in the order of the nibbles beside 4-bit K.
template <int KM>
__device__ __forceinline__ uint4 query_operand(uint4 v, int dtype) {
  if constexpr (KM != kRaw) {
    if (dtype == KNLP_BF16) {
      uint32_t* u = &v.x;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        u[j] = as_u32(__floats2half2_rn(__uint_as_float(u[j] << 16), __uint_as_float(u[j] & 0xffff0000u)));
    }
  }
  if constexpr (KM == KNLP_KV_INT4_SYM || KM == KNLP_KV_INT4_ASYM) {
    v = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632),
                   __byte_perm(v.y, v.w, 0x5410), __byte_perm(v.y, v.w, 0x7632));
  }
  return v;
}

// A CTA's item of a round.  The list is sorted by length, longest first, and dealt out back and
// forth, so that a CTA's sum is even.
__device__ __forceinline__ int item_of(int r) {
  const int g = gridDim.x, b = blockIdx.x;
  return r * g + (r & 1 ? g - 1 - b : b);
}

// Geometry of an item that every role derives for itself.
struct Item {
  Entry e;
  int head, n, len, ctx, first;  // new tokens, cached tokens, len - n, first query row (token)
  __device__ Item(const Params& p, int k) {
    const int heads = p.a.n_kv_heads;
    const int4* src = reinterpret_cast<const int4*>(p.entries + k / heads);
    const int4 x = src[0], y = src[1];
    e = {x.x, x.y, x.z, x.w, y.x, y.y, 0, 0};
    head = k % heads;
    n = extend_rows(p.a, e.seq, &first);
    len = extend_length(p.a, e.seq);
    ctx = p.a.seq_lens[e.seq] - n;
  }
  __device__ int tiles() const { return e.tile1 - e.tile0; }
  __device__ bool pair() const { return e.rows > kRows; }  // each stream has rows of its own
  // steps of 64 tokens that each stream takes
  __device__ int steps() const { return pair() ? 2 * tiles() : tiles(); }
};

// Copies of one plane's tiles by a warpgroup, item after item: warp w copies rows 32 w .. 32 w + 31
// of every tile, a lane looks up one row's block, a tile before it is needed.  EVERY 2: only the
// tiles of the parity `phase`, counted over all items.
template <int MODE, int D, int EVERY>
struct Copies {
  using T = PlaneTile<MODE, D>;
  const Params& p;
  const Plane& pl;
  const int n_items, w, lane, phase;
  int round = 0, tile = 0, tile1 = 0, len = 0, block = 0, off = 0;
  uint32_t count = 0;  // tiles of the items so far
  const int32_t* table = nullptr;
  const char* head_codes = nullptr;
  int64_t head_scales = 0, head_zeros = 0;
  bool there = false, pending;  // pending: a tile is looked up

  __device__ __forceinline__ Copies(const Params& p_, const Plane& plane, int n_items_, int w_, int lane_, int phase_)
      : p(p_), pl(plane), n_items(n_items_), w(w_), lane(lane_), phase(phase_) {
    pending = look_up();
  }
  __device__ __forceinline__ bool look_up() {
    for (int k; tile >= tile1 && (k = item_of(round)) < n_items; ++round) {  // the first tile of the next item that has any
      const Item it(p, k);
      tile = it.e.tile0, tile1 = it.e.tile1, len = it.len;
      if constexpr (EVERY == 2) {
        tile += (count & 1) != phase;
        count += it.tiles();
      }
      table = p.a.block_table + it.e.seq * p.a.bt_stride;
      head_codes = reinterpret_cast<const char*>(pl.codes) + it.head * pl.cs[2];
      if constexpr (T::kQuant) {
        head_scales = it.head * pl.ss[2];
        head_zeros = it.head * pl.zs[2];
      }
    }
    if (tile >= tile1) return false;
    const int t = tile * kTile + w * 32 + lane;
    there = t < len;
    const int e = p.block_shift >= 0 ? t >> p.block_shift : t / p.a.block_size;
    off = t - e * p.a.block_size;
    block = there ? table[e] : 0;
    tile += EVERY;
    return true;
  }
  // The looked-up tile to `dst`, a stage (or the operand itself, unquantized), as one group of
  // asynchronous copies; then the look-up of the next.
  __device__ __forceinline__ void next(char* dst) {
    if (pending) {
      const int row = w * 32 + lane;
      const int64_t b = block < 0 ? 0 : block >= p.a.num_blocks ? p.a.num_blocks - 1 : block;
      const char* src = there ? head_codes + b * pl.cs[0] + off * pl.cs[1] : nullptr;
      const uint32_t lo = static_cast<uint32_t>(reinterpret_cast<uint64_t>(src));
      const uint32_t hi = static_cast<uint32_t>(reinterpret_cast<uint64_t>(src) >> 32);
      constexpr int n = T::kChunks, at_once = 32 / n;
      const int chunk = lane % n;
#pragma unroll
      for (int i = 0; i < 32; i += at_once) {
        const int r = i + lane / n;
        const uint64_t from = static_cast<uint64_t>(__shfl_sync(~0u, hi, r)) << 32 | __shfl_sync(~0u, lo, r);
        const int rr = w * 32 + r;
        const uint32_t to = smem_addr(dst) + (T::kQuant ? T::at(rr, chunk)
                                                        : (chunk >> 3) * (kTile * 128) + rr * 128 + (((chunk & 7) ^ (rr & 7)) << 4));
        copy_async<16>(to, from ? reinterpret_cast<const char*>(from) + chunk * 16 : head_codes, from != 0);
      }
      if constexpr (T::kQuant) {
        const int64_t so = there ? head_scales + b * pl.ss[0] + off * pl.ss[1] : 0;
        copy_async<T::kScaleBytes>(smem_addr(dst + T::kScaleAt + row * T::kScaleBytes), pl.scales + so, there);
        if constexpr (T::kBytes > T::kZeroAt) {
          const int64_t zo = there ? head_zeros + b * pl.zs[0] + off * pl.zs[1] : 0;
          copy_async<T::kScaleBytes>(smem_addr(dst + T::kZeroAt + row * T::kScaleBytes), pl.zeros + zo, there);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    pending = pending && look_up();
  }
};

// Tokens of an item whose V is not finite in some groups.  Such a value would reach rows that do
// not attend to its token (as 0 x NaN): the groups are zeroed in the stage and noted, and the
// rows that do attend to the token are made NaN at the end.
struct BadList {
  int count;
  int2 at[kBadMost + 1];  // (token, mask of groups); the last one: from this token on
  __device__ __forceinline__ void clear() {
    count = 0;
    at[kBadMost] = make_int2(0x7fffffff, 0);
  }
  template <int MODE, int D>
  __device__ __forceinline__ void note(char* stage, int row, int token) {
    using T = PlaneTile<MODE, D>;
    const int bad = not_finite<MODE, D>(stage, row);
    for (int g = 0; g < D / 32; ++g) {
      if (!(bad >> g & 1)) continue;
      *reinterpret_cast<uint16_t*>(stage + T::kScaleAt + row * T::kScaleBytes + 2 * g) = 0;
      if constexpr (T::kBytes > T::kZeroAt)
        *reinterpret_cast<uint16_t*>(stage + T::kZeroAt + row * T::kScaleBytes + 2 * g) = 0;
    }
    const int i = atomicAdd(&count, 1);
    if (i < kBadMost) {
      at[i] = make_int2(token, bad);
    } else {  // more than the list holds
      atomicMin(&at[kBadMost].x, token);
      atomicOr(&at[kBadMost].y, bad);
    }
  }
  // whether a row that attends to `limit` tokens sees such a value in the group
  __device__ __forceinline__ bool hits(int limit, int group) const {
    bool hit = false;
    for (int i = 0; i < min(count, kBadMost + 1); ++i) hit |= limit > at[i].x && (at[i].y >> group & 1);
    return hit;
  }
};

struct Misc {
  uint64_t ring_full[kRing];
  uint64_t ring_empty[2][kRing];  // a K tile, a V tile in the slot has been used
  uint64_t q_full;
  uint64_t s_full[2][2], p_full[2][2];  // [stream][buffer]
  uint64_t o_step[2], o_full[2];        // a product with V, the item's last one, is done
  uint32_t tmem;
  int abort;
  float m[kRows], l[kRows];  // second stream's state when both serve the same rows
  BadList bad[kBadLists];    // by item
};
static_assert(sizeof(Misc) <= kMiscBytes, "");

// One plane's tiles (side 0: K, 1: V) by a warpgroup: a lane converts one row of every tile, and
// only lanes of the same warp read what a lane has copied.  Planes of one mode run the same code:
// the instruction cache is what several warpgroups of unrolled code compete for.
template <class L, int MODE, int D, int STAGES>
__device__ __forceinline__ void produce(const Params& p, char* sm, Misc& mi, int n_items, int side,
                                        int w, int lane) {
  using T = PlaneTile<MODE, D>;
  constexpr int kStages = STAGES;
  char* const stages = sm + (side ? L::kStageV : L::kStageK);
  const int row = w * 32 + lane;
  Copies<MODE, D, 1> copies(p, side ? p.a.v : p.a.k, n_items, w, lane, 0);
  for (int i = 0; i < kStages; ++i) copies.next(stages + i * T::kBytes);
  uint32_t done = side, stage = 0;  // done: number of the plane tile in the ring's order
  // The slot's use before this one, always the other plane's, has to be over.
  auto wait_empty = [&]() {
    const uint32_t others = (done / kRing + 1) / 2;  // uses of this slot by the other plane
    mbar_wait(&mi.ring_empty[1 - side][done % kRing], (others + 1) & 1, &mi.abort, p.status);
  };
  int serial = 0;
  for (int r = 0, ki; (ki = item_of(r)) < n_items; ++r) {
    const Item it(p, ki);
    if (it.tiles() == 0) continue;
    BadList& bad = mi.bad[serial % kBadLists];
    if (side) {
      if (row == 0) bad.clear();
      asm volatile("bar.sync 3, 128;" ::: "memory");
    }
    for (int j = 0; j < it.tiles(); ++j, done += 2) {
      char* const to = sm + L::kRingAt + done % kRing * L::kTileBytes;
      if constexpr (kStages == 0) {
        wait_empty();
        copies.next(to);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      } else {
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        char* const from = stages + stage * T::kBytes;
        if constexpr (T::kQuant) {
          if (side && any_not_finite<MODE, D>(from, row)) bad.note<MODE, D>(from, row, (it.e.tile0 + j) * kTile + row);
        }
        wait_empty();
        dequantize_row<MODE, D>(from, to, row);
      }
      fence_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&mi.ring_full[done % kRing]);
      if constexpr (kStages > 0) {
        copies.next(stages + stage * T::kBytes);
        stage = stage + 1 == kStages ? 0 : stage + 1;
      }
    }
    ++serial;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

template <int KM, int VM, int D>
__global__ void __launch_bounds__(kThreads, 1) extend_mma_kernel(const __grid_constant__ Params p) {
  using L = Layout<KM, VM, D>;
  extern __shared__ char smem_raw[];
  char* sm = smem_raw + ((1024 - (smem_addr(smem_raw) & 1023)) & 1023);
  Misc& mi = *reinterpret_cast<Misc*>(sm + L::kMisc);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const ExtendArgs& a = p.a;

  if (tid == 0) {
    for (int i = 0; i < kRing; ++i) mbar_init(&mi.ring_full[i], 4), mbar_init(&mi.ring_empty[0][i], 2), mbar_init(&mi.ring_empty[1][i], 2);
    mbar_init(&mi.q_full, 8);
    for (int w = 0; w < 2; ++w) {
      for (int x = 0; x < 2; ++x) mbar_init(&mi.s_full[w][x], 1), mbar_init(&mi.p_full[w][x], 4);
      mbar_init(&mi.o_step[w], 1);
      mbar_init(&mi.o_full[w], 1);
    }
    mi.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid < kBadLists) mi.bad[tid].clear();
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&mi.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = mi.tmem;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int n_items = p.plan->n_entries * a.n_kv_heads;
  const bool raw_bf16 = KM == kRaw && a.k.mode == KNLP_KV_BF16;
#define KNLP_REGISTERS(what, n) asm volatile("setmaxnreg." what ".sync.aligned.u32 " #n ";")
  auto wait = [&](uint64_t* b, uint32_t phase) { mbar_wait(b, phase & 1, &mi.abort, p.status); };

  if (warp < 8) {
    // ---------------------------------------------------------------- softmax streams
    KNLP_REGISTERS("inc", 136);
    const int w = warp >> 2, row = tid & 127;  // row: of the stream's 128
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // the warp's 32 TMEM lanes
    const uint32_t t_s = tmem + lanes + w * 2 * kStep, t_o = tmem + lanes + 256 + w * D;
    const float c = a.scale * kLog2e;
    uint32_t count = 0, n_o = 0;  // steps, items so far
    int serial = 0;
    // A thread's row of an item, derived anew behind the tiles: it would not fit the registers
    // beside S.
    struct Row {
      int local, flat, tok, limit;
      bool valid, active;  // of the thread; of its warp
      __device__ Row(const Params& p, const Item& it, int w, int row) {
        const int first = it.pair() ? w * kRows : 0;
        local = first + row;
        valid = local < it.e.rows;
        active = first + (row & ~31) < it.e.rows;
        flat = it.e.row0 + local;
        tok = flat / p.rep;
        limit = !valid ? 0 : p.a.causal ? max(min(it.ctx + tok + 1, it.len), 0) : it.len;
      }
    };
    for (int r = 0, k; (k = item_of(r)) < n_items; ++r) {
      float m = -INFINITY, l = 0.0f;
      {
      const Item it(p, k);
      const int steps = it.steps();
      const Row rw(p, it, w, row);
      const int limit = rw.limit;
      const bool active = rw.active;
      const int whole = __reduce_min_sync(~0u, rw.valid ? limit : 0x7fffffff);  // of the warp's rows

      asm volatile("bar.sync 1, 256;" ::: "memory");  // nobody reads the Q area any more
      if (it.tiles() && (w == 0 || it.pair())) {
        // Q tile: D/8 lanes copy a row, 16 bytes each; a lane works out the place of one row, and
        // eight loads are in flight
        constexpr int kPer = D / 8, kAtOnce = 32 / kPer;
        char* q = sm + L::kQ + w * L::kTileBytes;
        const int r0 = (warp & 3) * 32, chunk = lane % kPer;
        const int f = rw.flat, t = rw.tok;
        const char* mine = nullptr;
        if (rw.valid)
          mine = static_cast<const char*>(a.q) + 2 * ((static_cast<int64_t>(it.first) + t) * a.q_stride[0] +
                                                      (static_cast<int64_t>(it.head) * p.rep + (f - t * p.rep)) * a.q_stride[1]);
        const uint32_t lo = static_cast<uint32_t>(reinterpret_cast<uint64_t>(mine));
        const uint32_t hi = static_cast<uint32_t>(reinterpret_cast<uint64_t>(mine) >> 32);
#pragma unroll 1
        for (int i0 = 0; i0 < 32; i0 += 8 * kAtOnce) {
          uint4 v[8];
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int r = i0 + x * kAtOnce + lane / kPer;
            const uint64_t from = static_cast<uint64_t>(__shfl_sync(~0u, hi, r)) << 32 | __shfl_sync(~0u, lo, r);
            v[x] = from ? reinterpret_cast<const uint4*>(from)[chunk] : make_uint4(0, 0, 0, 0);
          }
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int r = r0 + i0 + x * kAtOnce + lane / kPer;
            *reinterpret_cast<uint4*>(q + (chunk >> 3) * (kRows * 128) + r * 128 +
                                      (((chunk & 7) ^ (r & 7)) << 4)) = query_operand<KM>(v[x], a.q_dtype);
          }
        }
        fence_smem();
      }
      __syncwarp();
      if (it.tiles() && lane == 0) mbar_arrive(&mi.q_full);

      const int ahead = it.pair() ? kStep : kTile;
      int base = it.e.tile0 * kTile + (it.pair() ? 0 : w * kStep);
#pragma unroll 1
      for (int i = 0; i < steps; ++i, ++count, base += ahead) {
        const uint32_t t_b = t_s + (count & 1) * kStep;
        wait(&mi.s_full[w][count & 1], count >> 1);
        fence_after();
        {
          if (active) {
            float x0[32], x1[32];
            tmem_ld32(t_b, reinterpret_cast<uint32_t*>(x0));
            tmem_ld32(t_b + 32, reinterpret_cast<uint32_t*>(x1));
            tmem_wait_ld(reinterpret_cast<uint32_t*>(x0));
            tmem_wait_ld(reinterpret_cast<uint32_t*>(x1));
            if (base + kStep > whole) {  // some row of the warp ends inside the step
              const int seen = limit - base;
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                x0[x] = x < seen ? x0[x] : -INFINITY;
                x1[x] = 32 + x < seen ? x1[x] : -INFINITY;
              }
            }
            float mx[4] = {x0[0], x0[1], x1[0], x1[1]};
#pragma unroll
            for (int x = 2; x < 32; x += 4) {
              mx[0] = max3(mx[0], x0[x], x0[x + 1]);
              mx[2] = max3(mx[2], x1[x], x1[x + 1]);
              if (x + 2 < 32) {
                mx[1] = max3(mx[1], x0[x + 2], x0[x + 3]);
                mx[3] = max3(mx[3], x1[x + 2], x1[x + 3]);
              }
            }
            const float m_new = fmaxf(m, fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c);
            if (__any_sync(~0u, m_new > m + kGrow)) {
              const float f = m_new == m ? 1.0f : exp2f(m - m_new);
              m = m_new;
              l *= f;
              if (i > 0) {  // O has the steps before, once the last product is done
                wait(&mi.o_step[w], count - 1);
                fence_after();
#pragma unroll 1
                for (int col = 0; col < D; col += 16) {
                  uint32_t o[16];
                  tmem_ld16(t_o + col, o);
                  tmem_wait_ld16(o);
#pragma unroll
                  for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                  tmem_st16(t_o + col, o);
                }
              }
            }
            const float off = m == -INFINITY ? 0.0f : -m;
            const uint64_t c2 = pack2(c, c), off2 = pack2(off, off);
            uint64_t sum[2] = {0, 0};
            auto weights = [&](int chunk, const float* x) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                float y0, y1, p0, p1;
                unpack2(fma2(pack2(x[2 * e], x[2 * e + 1]), c2, off2), y0, y1);
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p0) : "f"(y0));
                asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p1) : "f"(y1));
                sum[e & 1] = add2(sum[e & 1], pack2(p0, p1));
                pk[e] = as_u32(__floats2half2_rn(p0, p1));
              }
              tmem_st16(t_b + chunk * 16, pk);  // P overlays S, which is in registers by now
            };
            weights(0, x0);
            weights(1, x1);
            float l0, l1;
            unpack2(add2(sum[0], sum[1]), l0, l1);
            l += l0 + l1;
            tmem_wait_st();
          }
          fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&mi.p_full[w][count & 1]);
        }
      }

      }
      // ---- epilogue
      const Item it(p, k);
      const int steps = it.steps();
      const auto [local, flat, tok, limit, valid, active] = Row(p, it, w, row);
      if (steps) {
        wait(&mi.o_full[w], n_o++);
        fence_after();
      }
      float* swap = reinterpret_cast<float*>(sm + L::kQ);  // [column][row] of the second stream
      const bool merge = !it.pair() && steps > 0;
      if (merge && w == 1) {
        if (active) {
#pragma unroll 1  // run once per item: straight-line code would come from memory, not from the cache
          for (int i = 0; i < D; i += 32) {
            uint32_t o[32];
            tmem_ld32(t_o + i, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int x = 0; x < 32; ++x) swap[(i + x) * kRows + row] = __uint_as_float(o[x]);
          }
          mi.m[row] = m;
          mi.l[row] = l;
        }
        fence_before();
      }
      if (merge) asm volatile("bar.sync 2, 256;" ::: "memory");
      if (active && (w == 0 || it.pair())) {
        float f0 = 1.0f, f1 = 0.0f;
        if (merge) {
          const float m1 = mi.m[row], mm = fmaxf(m, m1);
          f0 = m == mm ? 1.0f : exp2f(m - mm);
          f1 = m1 == mm ? 1.0f : exp2f(m1 - mm);
          l = l * f0 + mi.l[row] * f1;
          m = mm;
        }
        const bool direct = it.e.part < 0;
        const float inv = !direct ? 1.0f : l > 0.0f ? 1.0f / l : l == 0.0f ? 0.0f : l;
        const BadList& bad = mi.bad[serial % kBadLists];
        const int h = flat - tok * p.rep;
        const int64_t out_row = (static_cast<int64_t>(it.first) + tok) * a.n_q_heads + it.head * p.rep + h;
        float* part = direct ? nullptr
                             : p.parts + (static_cast<int64_t>(it.e.part) + static_cast<int64_t>(it.head) * it.e.rows + local) * (D + 4);
#pragma unroll 1
        for (int i = 0; i < D; i += 32) {
          float o[32];
          if (steps) {
            tmem_ld32(t_o + i, reinterpret_cast<uint32_t*>(o));
            tmem_wait_ld(reinterpret_cast<uint32_t*>(o));
          } else {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = 0.0f;
          }
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            if (merge) o[x] = o[x] * f0 + swap[(i + x) * kRows + row] * f1;
            o[x] *= inv;
          }
          if (bad.count && bad.hits(limit, i / 32)) {  // never in a healthy cache
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = NAN;
          }
          if (!valid) continue;
          float v[32];  // in the order of the head dimension
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            constexpr bool kPaired = VM == KNLP_KV_INT4_SYM || VM == KNLP_KV_INT4_ASYM;
            v[x] = o[kPaired ? (x & ~7) + 2 * (x & 3) + ((x >> 2) & 1) : x];
          }
          if (!direct) {
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(part + i + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          } else if (a.out_dtype == KNLP_F32) {
            float* dst = static_cast<float*>(a.out) + out_row * a.out_row_stride + i;
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(dst + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          } else {
            uint16_t* dst = static_cast<uint16_t*>(a.out) + out_row * a.out_row_stride + i;
            uint32_t u[16];
#pragma unroll
            for (int x = 0; x < 16; ++x) {
              if (a.out_dtype == KNLP_F16) {
                u[x] = as_u32(__floats2half2_rn(v[2 * x], v[2 * x + 1]));
              } else {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * x], v[2 * x + 1]);
                u[x] = *reinterpret_cast<const uint32_t*>(&b);
              }
            }
#pragma unroll
            for (int x = 0; x < 16; x += 4)
              *reinterpret_cast<uint4*>(dst + 2 * x) = make_uint4(u[x], u[x + 1], u[x + 2], u[x + 3]);
          }
        }
        if (valid) {
          if (!direct) {
            part[D] = m;
            part[D + 1] = l;
          } else if (a.lse) {
            a.lse[out_row] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
          }
        }
      }
      fence_before();
      serial += it.tiles() > 0;
    }
  } else if (warp < 16) {
    KNLP_REGISTERS("dec", 80);
    if constexpr (KM == VM && L::kStagesK == L::kStagesV) {
      produce<L, KM, D, L::kStagesK>(p, sm, mi, n_items, (warp - 8) >> 2, warp & 3, lane);
    } else {
      if (warp < 12) produce<L, KM, D, L::kStagesK>(p, sm, mi, n_items, 0, warp & 3, lane);
      else produce<L, VM, D, L::kStagesV>(p, sm, mi, n_items, 1, warp & 3, lane);
    }
  } else {
    // ---------------------------------------------------------------- matrix products
    KNLP_REGISTERS("dec", 48);
    if (warp < 18) {
      // A warp per stream; all of it follows the items and waits, one lane issues.
      const int w = warp - 16;
      const uint32_t q_at = operand(smem_addr(sm + L::kQ), 16);
      const uint32_t k_at = operand(smem_addr(sm + L::kRingAt), 16);
      const uint32_t v_at = operand(smem_addr(sm + L::kRingAt), kTile * 128);
      const uint32_t idesc_s = product(kRows, kStep, raw_bf16, false);
      constexpr uint32_t idesc_o = product(kRows, D, false, true);
      auto wait_warp = [&](uint64_t* x, uint32_t phase) { mbar_wait_warp(x, phase & 1, &mi.abort, p.status); };
      const int n_all = uniform(n_items);
      const uint32_t tm = uniform(tmem);
      uint32_t used = 0, n_q = 0, count = 0;
      // S buffer b = Q tile qt x half a K tile
      auto scores = [&](int b, int qt, uint32_t slot, int half, bool last_use) {
        const uint32_t q = q_at + (qt * L::kTileBytes >> 4);
        const uint32_t kk = k_at + (slot * L::kTileBytes >> 4) + half * (kStep * 128 >> 4);
        const uint32_t d = tm + (w * 2 + b) * kStep;
        if (elect()) {
          auto step = [&](auto i) {
            constexpr int n = decltype(i)::value;
            mma_ss<((n >> 2) * (kTile * 128) + (n & 3) * 32) / 16>(d, q, kk, idesc_s, n > 0);
          };
          step(Int<0>{}), step(Int<1>{}), step(Int<2>{}), step(Int<3>{});
          if constexpr (D == 128) step(Int<4>{}), step(Int<5>{}), step(Int<6>{}), step(Int<7>{});
          commit(&mi.s_full[w][b]);
          if (last_use) commit(&mi.ring_empty[0][slot]);
        }
        __syncwarp();
      };
      // O (+)= P in buffer b x half a V tile
      auto values = [&](int b, uint32_t slot, int half, bool acc, bool last_use, bool last) {
        const uint32_t v = v_at + (slot * L::kTileBytes >> 4) + half * (kStep * 128 >> 4);
        const uint32_t d = tm + 256 + w * D, pr = tm + (w * 2 + b) * kStep;
        if (elect()) {
          auto step = [&](auto i, bool add) {
            constexpr int n = decltype(i)::value;
            mma_ts<n * 8, n * 2048 / 16>(d, pr, v, idesc_o, add);
          };
          step(Int<0>{}, acc), step(Int<1>{}, true), step(Int<2>{}, true), step(Int<3>{}, true);
          commit(&mi.o_step[w]);
          if (last_use) commit(&mi.ring_empty[1][slot]);
          if (last) commit(&mi.o_full[w]);
        }
        __syncwarp();
      };
      auto ready = [&](uint32_t x) {  // plane tile x of the ring
        wait_warp(&mi.ring_full[x % kRing], x / kRing);
        fence_after();
        return x % kRing;
      };
      for (int r = 0, k; (k = item_of(r)) < n_all; ++r) {
        const Item it(p, k);
        const int n = uniform(it.tiles());
        if (n == 0) continue;
        wait_warp(&mi.q_full, n_q++);
        fence_after();
        // Step i: its output, then the scores of step i + 2.  Of a pair both streams use the same
        // half tiles, else each its half of every tile.
        const bool pair = uniform(it.pair());
        const int steps = pair ? 2 * n : n;
        for (int i = -2; i < steps; ++i) {
          if (i >= 0) {
            const uint32_t slot = ready(used + 2 * (pair ? i >> 1 : i) + 1);
            const int b = (count + i) & 1;
            wait_warp(&mi.p_full[w][b], (count + i) >> 1);
            fence_after();
            values(b, slot, pair ? i & 1 : w, i > 0, !pair || (i & 1), i + 1 == steps);
          }
          const int x = i + 2;
          if (x < steps) {
            const uint32_t slot = ready(used + 2 * (pair ? x >> 1 : x));
            scores((count + x) & 1, pair ? w : 0, slot, pair ? x & 1 : w, !pair || (x & 1));
          }
        }
        count += steps;
        used += 2 * n;
      }
    }
    __syncwarp();
  }
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 16)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

#undef KNLP_REGISTERS

}  // namespace extend
}  // namespace knlp
