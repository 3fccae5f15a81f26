// h24_ce.cu -- softmax cross entropy of a head's product without its logits.
//
//   z[t][v] = sum_k x[t][k] W[v][k],  lse[t] = log sum_v exp(z[t][v])
//   loss[t] = lse[t] - z[t][y_t]
//   d[t][v] = softmax(z[t])[v] - [v = y_t]
//   dx[t]   = g_t sum_v d[t][v] W[v],   dW[v] = sum_t g_t d[t][v] x[t]
//
// x and W are fp16 or bf16, products exact, sums fp32.  Tokens whose target is
// ignored are left out: the others' rows are copied together first (a pass of
// 4 bytes an element, which also gives rows that TMA can read), so a masked
// token costs nothing and what stands in its row does not matter.
//
// All four products run in one kernel, ce_gemm_kernel: persistent pairs of CTAs
// on 256 x 256 tiles (tcgen05.mma.cta_group::2, operands by TMA into a ring of
// stages of 128 k, two accumulators in TMEM, eight epilogue warps a CTA), each
// operand K-major or MN-major as it lies in memory, so nothing is transposed.
//   forward: the logits' tiles end in a maximum and a sum of exponentials a row
//     (a TMEM lane, so a thread, holds a row);
//   backward: the vocabulary goes by in pieces.  A piece's logits are computed
//     again and end as d in 16 bits; its part of dx (added up in fp32) and its
//     rows of dW are products with d.  One launch holds a piece's gradients and
//     the logits of the next piece, the long tiles first and each pair of SMs
//     taking the next one as it is ready.
// Up to 128 tokens are the tiles' columns instead, so that a tile holds 256 rows
// of the weights whatever the tokens.
//
// d is rounded to the operands' type (half a step, 2^-8 relative in bf16), as
// the tensor cores want it; in fp16 it is held times 2^15, so that probabilities
// down to 2^-39 keep their place.
//
// Many tokens are bound by what an SM takes from L2: 64 KB a stage and CTA, for
// 1,024 cycles of the tensor cores, at some 54 of 64 bytes a cycle.  [8192,1920] x
// [50688,1920] bf16: the loss 1,037 us (1.54 PFLOP/s, 0.92 of the measured burst),
// its gradients 3.4 ms (three products, 1.41 PFLOP/s; 1.2 to 1.3 under the power
// cap, with the loss 5.1 ms a step).  Few are bound by the head's bytes: one token
// and [50688,1920] 38 us of tiles (5.1 TB/s).
#include "h24_tile.cuh"

#include <limits.h>

#include <type_traits>

namespace h24 {
namespace {

constexpr int kTileM = 256;      // rows of a pair's tile, 128 a CTA
constexpr int kTileN = 256;      // its columns at most
constexpr int kTileK = 128;      // k of a stage
constexpr int kChunk = 64;       // a 128-byte swizzle row of 16-bit elements
constexpr int kOperand = 128 * kTileK * 2;  // bytes of a CTA's share of an operand's stage
constexpr int kBox = kOperand / 2;  // one load: 128 rows x 64 k (K-major) or 128 k x 64 columns (MN-major)
constexpr int kRing = 6 * kOperand;  // bytes of the ring of stages
constexpr int kMaxStages = 5;
constexpr int kHead = 1024;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 320;    // warp 0 loads, warp 1 issues MMAs, warps 2-9 read TMEM
constexpr int kBlockPitch = 33;  // fp32 of a row of an epilogue warp's 32 x 32 block
constexpr int kBlockBytes = 32 * kBlockPitch * 4;
constexpr int kSmem = 1024 + kHead + kRing + kEpiWarps * kBlockBytes;
static_assert(kSmem <= 227 * 1024, "shared memory");
constexpr int kBackBf16 = 32, kBackHalf = 11;  // (bf16, fp16)
// k blocks at most of a logit's sum in the tensor cores, in slices of one length.
template <bool kBf16, bool kForward, bool kFew>
__device__ __forceinline__ int slice_blocks(int nkb) {
  constexpr int kMost = !kForward ? (kBf16 ? kBackBf16 : kBackHalf) : kFew ? (kBf16 ? 2 : 1) : kBf16 ? 8 : 4;
  const int n = (nkb + kMost - 1) / kMost;
  return (nkb + n - 1) / n;
}
// The same of a gradient's sum, over the vocabulary (dx: each of its slices has an
// output of its own) or over the tokens (dW).
constexpr int kSumBf16 = 1024, kSumHalf = 256;
template <bool kBf16>
__device__ __forceinline__ int sum_blocks(int nkb) {
  constexpr int kMost = kBf16 ? kSumBf16 : kSumHalf;
  const int n = max(1, (nkb + kMost - 1) / kMost);
  return (nkb + n - 1) / n;
}
constexpr int kMaxJobs = 3;
constexpr int kGroupM = 32;      // row tiles that run through the vocabulary together
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -INFINITY;

enum Kind { kLoss, kProb, kStates, kHeadRows };

// One product of a launch.  Rows and sums over tokens go by the number of kept
// tokens, which only the device knows.
struct Job {
  int kind;
  bool swap;         // the weights' rows (kStates: columns) are the tile's rows, the tokens, at most 128, its columns
  int n_total, bn;   // columns, of which a tile takes bn
  int m_total;       // rows (kHeadRows, swap); the other kinds' rows are the tokens
  int k_total;       // length of the sum (kHeadRows: the tokens)
  int split;         // slices of the sum, each with its own output (kStates)
  int v0;            // first vocabulary row of the piece
  bool add;          // kStates: onto what is there
  void *out;
  int64_t pitch;     // elements between the output's rows
  int64_t plane;     // elements between the slices' outputs
};

struct GemmArgs {
  CUtensorMap map[2 * kMaxJobs];  // A and B of each job
  Job job[kMaxJobs];
  int jobs;
  int vocab;
  int stages, stage_a, stage_b;  // of the ring; bytes of A and of B in a stage
  int *next_tile;      // counts the tiles that pairs have taken beyond their first; null: each takes its turn
  const int *kept;     // number of tokens with a loss; null: the tokens' own rows are read, `tokens` of them
  int tokens;
  const int64_t *labels;  // of the tokens, where kept is null
  unsigned *ticket;       // set to 0, where kept is null
  const int *target;   // of each kept token
  const float *lse;    // of each kept token
  const float *own;    // d at each kept token's target, times what its row of d is held times
  float *z_target;
  float2 *parts;       // kLoss: maximum and sum of half a tile's columns
  int64_t part_pitch;
  const float *scale;  // kHeadRows: factor of the sum
  const float *log_factor; // log2 of what each kept token's row of d is held times; null: prob_log2 for all
  float prob_log2;
  int row_bytes;       // kHeadRows: rows of the output lie on 32, 16 or 2 bytes
  int *err;
};

// Numbers of tiles handed on within a pair.  No slot is waited for: the loading
// thread is at most a ring (5 k blocks, a tile has one at least) and two
// accumulators ahead of the warp that is last to read, 8 tiles.
constexpr int kSlots = 16;

struct PairHead {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
  uint64_t slot_full[kSlots];
  int slot[kSlots];
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(PairHead) <= kHead, "head");

// Shared-memory descriptor of an MN-major operand with the 128-byte swizzle:
// boxes of 64 columns (128 bytes) x 128 k, 16 KB apart; groups of 8 k 1,024
// bytes apart.
__device__ __forceinline__ uint64_t mn_desc(uint32_t addr) {
  return tile_desc(addr) | (uint64_t(kBox >> 4) << 16);
}

// Instruction descriptor: kind::f16, D fp32, A and B of one 16-bit type, each
// K-major (0) or MN-major (1), M = 256.
__device__ __forceinline__ uint32_t f16_idesc(bool bf16, int a_mn, int b_mn, int n) {
  const uint32_t type = bf16 ? 1u : 0u;
  return (1u << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(a_mn) << 15) |
         (static_cast<uint32_t>(b_mn) << 16) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(kTileM >> 4) << 24);
}

__device__ __forceinline__ void mma_f16_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}

struct Tile {
  int job, m, n, cols;  // first row, first column, columns (a multiple of 32)
  int kb, nkb, slice;   // k blocks
};

__device__ __forceinline__ bool rows_known(const Job &j) { return j.kind == kHeadRows || j.swap; }
__device__ __forceinline__ bool a_is_mn(const Job &j) { return j.kind == kHeadRows || (j.swap && j.kind == kStates); }
__device__ __forceinline__ bool b_is_mn(const Job &j) { return j.kind == kHeadRows || (!j.swap && j.kind == kStates); }

__device__ __forceinline__ int tiles_of(const Job &j, int kept) {
  if (j.swap && kept == 0) return 0;
  const int rows = rows_known(j) ? j.m_total : kept;
  return (rows + kTileM - 1) / kTileM * ((j.n_total + j.bn - 1) / j.bn) * j.split;
}

__device__ __forceinline__ Tile tile_at(const GemmArgs &a, int kept, int idx) {
  Tile t;
  t.job = 0;
  for (; t.job + 1 < a.jobs; ++t.job) {
    const int c = tiles_of(a.job[t.job], kept);
    if (idx < c) break;
    idx -= c;
  }
  const Job &j = a.job[t.job];
  const int nt = (j.n_total + j.bn - 1) / j.bn;
  const int mt = ((rows_known(j) ? j.m_total : kept) + kTileM - 1) / kTileM;
  int m, n;
  t.slice = 0;
  if (j.kind == kLoss || j.kind == kProb) {
    // Up to 32 row tiles side by side, so that these rows stay in L2 while the
    // vocabulary passes once.
    const int group = idx / (kGroupM * nt), g = min(kGroupM, mt - group * kGroupM);
    const int at = idx - group * kGroupM * nt;
    n = at / g;
    m = group * kGroupM + at - n * g;
  } else {
    // All columns of a row tile side by side: d, the larger operand, passes once.
    n = idx % nt;
    const int rest = idx / nt;
    t.slice = rest / mt;
    m = rest - t.slice * mt;
  }
  t.m = m * kTileM;
  t.n = n * j.bn;
  t.cols = min(j.bn, (j.n_total - t.n + 31) / 32 * 32);
  const int kblocks = ((j.kind == kHeadRows ? kept : j.k_total) + kTileK - 1) / kTileK;
  t.kb = static_cast<int>(static_cast<int64_t>(kblocks) * t.slice / j.split);
  t.nkb = static_cast<int>(static_cast<int64_t>(kblocks) * (t.slice + 1) / j.split) - t.kb;
  return t;
}

__device__ __forceinline__ void store32B(void *p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void load32B(const void *p, uint32_t (&w)[8]) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p)
               : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}
template <bool kBf16>
__device__ __forceinline__ uint16_t pack1(float a) {
  if constexpr (kBf16) return __bfloat16_as_ushort(__float2bfloat16_rn(a));
  return __half_as_ushort(__float2half_rn(a));
}

// What an epilogue thread does with 32 columns of its row.  `c` is the column
// within the tile; r the sums.
struct RowState {
  bool live;
  float lse;     // kProb
  float log2f;   // kProb: log2 of what the row of d is held times
  float own;     // kProb: the target's d, times that
  int target;    // the target's column of the tile (any number where it is elsewhere)
  int limit;     // columns of the tile that the vocabulary has
  float m, s, z; // kLoss, few tokens: running maximum, sum of exponentials, the target's logit
  bool found;
};

// The maximum that exponents are taken from.  2^((z - m) log2 e) is 1 where z is the
// maximum, with no rounding that would grow from join to join (z log2 e less a
// rounded m log2 e is off by as much as that rounding: 2^-24 of the logit each
// time, and a certain token's loss got below 0), so a sum is never below 1.
__device__ __forceinline__ float exp_base(float m) { return m == kNegInf ? 0.f : m; }

__device__ __forceinline__ void loss_chunk(RowState &st, int c, const float (&z)[32]) {
  float top = kNegInf;
  if (c + 32 <= st.limit) {
#pragma unroll
    for (int j = 0; j < 32; ++j) top = fmaxf(top, z[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < st.limit) top = fmaxf(top, z[j]);
  }
  const float m = fmaxf(st.m, top);
  const float base = exp_base(m);
  float s0 = st.s * exp2_fast((st.m - base) * kLog2e), s1 = 0.f;  // (2^-inf is 0)
  if (c + 32 <= st.limit) {
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      s0 += exp2_fast((z[j] - base) * kLog2e);
      s1 += exp2_fast((z[j + 1] - base) * kLog2e);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (c + j < st.limit) s0 += exp2_fast((z[j] - base) * kLog2e);
  }
  st.s = s0 + s1;
  st.m = m;
  const int at = st.target - c;
  if (static_cast<unsigned>(at) < 32u) {
    st.found = true;
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j == at) st.z = z[j];
  }
}

__device__ __forceinline__ void prob_row(const GemmArgs &a, int row, RowState &st) {
  st.lse = a.lse[row];
  st.log2f = a.log_factor ? a.log_factor[row] : a.prob_log2;
  st.own = a.own[row];
}

// The target's d is p - 1, which of a certain token's p would keep nothing but
// roundings; it comes from the loss instead, as expm1(-loss).
template <bool kBf16>
__device__ __forceinline__ void prob_chunk(const RowState &st, uint16_t *out, int c, const float (&z)[32]) {
  float d[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) d[j] = exp2_fast(fmaf(z[j] - st.lse, kLog2e, st.log2f));
  const int at = st.target - c;
  if (static_cast<unsigned>(at) < 32u) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j == at) d[j] = st.own;
  }
  if (!st.live || c + 32 > st.limit) {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (!st.live || c + j >= st.limit) d[j] = 0.f;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = pack2<kBf16>(d[16 * h + 2 * j], d[16 * h + 2 * j + 1]);
    store32B(out + c + 16 * h, w);
  }
}

__device__ __forceinline__ void states_chunk(bool add, float *out, const float (&z)[32]) {
  uint32_t w[4][8];
  if (add) {
#pragma unroll
    for (int h = 0; h < 4; ++h) load32B(out + 8 * h, w[h]);
  }
#pragma unroll
  for (int h = 0; h < 4; ++h) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      w[h][j] = __float_as_uint(add ? __uint_as_float(w[h][j]) + z[8 * h + j] : z[8 * h + j]);
    store32B(out + 8 * h, w[h]);
  }
}

// The order in which a pair of CTAs takes tiles.  Where tiles differ in length,
// a pair takes the next one when it is ready for it: the first CTA's loading
// thread counts it off in global memory and hands its number to the other warps
// of both CTAs.  The list has the long tiles first.  (The gradients of [1024,1152]
// x [50688,1152] take 323 us so, 393 with each pair in its turn.)
struct Turn {
  const GemmArgs &a;
  PairHead &H;
  bool counting;
  int tiles, n;
  volatile int *abort;

  // The next tile's number, or -1: for a warp, or (kThread) for one thread of it.
  template <bool kThread>
  __device__ __forceinline__ int take(int before, int first, int step) {
    if (!counting) {
      const int idx = before < 0 ? first : before + step;
      return idx < tiles ? idx : -1;
    }
    const int s = n % kSlots;
    const bool ok = bar_wait(&H.slot_full[s], n / kSlots & 1, abort, a.err);
    if (kThread ? !ok : !__all_sync(0xffffffffu, ok)) return -1;
    ++n;
    return *const_cast<volatile int *>(&H.slot[s]);
  }
  // The same for the thread that counts.
  __device__ __forceinline__ int give(int before, int counted, int first, int step) {
    int idx = before < 0 ? first : counting ? step + counted : before + step;
    if (idx >= tiles) idx = -1;
    if (!counting) return idx;
    const int s = n++ % kSlots;
    // The other CTA's slot is written and its barrier told of the bytes by one
    // asynchronous store, so that its readers need no more than for a load's bytes.
    const uint32_t bar = cluster_addr(&H.slot_full[s], 1);
    asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], 4;" ::"r"(bar) : "memory");
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u32 [%0], %1, [%2];" ::"r"(
                     cluster_addr(&H.slot[s], 1)),
                 "r"(idx), "r"(bar)
                 : "memory");
    *const_cast<volatile int *>(&H.slot[s]) = idx;
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(&H.slot_full[s])) : "memory");
    return idx;
  }
};

// Forward: the loss's tiles alone, of many tokens or of few.  The tensor cores
// cut off what falls below a sum's last place where they add to it, so a long sum
// shrinks: z of 7,680 k by 8e-6 of itself in bf16, 1.4e-5 in fp16 (measured:
// 1.7e-8 and 3e-8 to 5e-8 for each 16 k), which shows in an fp32 loss.  The
// forward pass therefore sums 1,024 k at most there, in fp16 512, and these sums
// rounded to nearest in registers: about 1e-6 whatever the length.  Shorter
// slices cost time, since reading a tile's TMEM takes 1,400 cycles (256 k: 2e-7,
// and [8192,1920] x [50688,1920] 1,405 us where 1,024 k take 1,037).  The narrower
// tiles of few tokens wait for HBM, and 256 and 128 k cost nothing there.
// The backward pass's probabilities are rounded to 16 bits, and the one entry that
// is a difference comes from the loss: slices of 4,096 k, in fp16 1,408, keep z
// to 4.4e-6 of itself, so a probability of a logit of 30 to 2^-13, where half a
// step is 2^-9 and 2^-12.  The gradients' own sums are cut at 131,072 terms, in
// fp16 at 32,768: terms of one sign lose 1.4e-4 and 1e-4 of their sum, where half a
// step of the result is 2e-3 and 2.4e-4 at least.
//
// kFew: up to 128 tokens, the columns of the tiles of logits and of dx.  kLong: what
// is summed in several slices, for which an epilogue thread holds 128 of them: in
// the forward pass the logits, in the backward pass those where k is longer than a
// slice, or they and dW where the tokens are (a step of [140000,1024] x
// [20000,1024] in bf16: 22.1 ms, 19.4 without).  (Within one kernel for all the
// gradients of [1024,1152] x [50688,1152] took 567 us, 479 so; the spills of the
// long kernels cost a step of [8192,1920] x [50688,1920] in fp16 5.1 ms instead of
// 4.8, and of [1024,7680] x [50688,7680] in bf16 nothing.)
enum Long { kNone, kLogits, kTokens };
template <bool kBf16, bool kForward, bool kFew, Long kLong>
__global__ void __launch_bounds__(kThreads, 1) ce_gemm_kernel(const __grid_constant__ GemmArgs a) {
  extern __shared__ uint8_t ce_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(ce_raw) + 1023) & ~uintptr_t(1023));
  PairHead &H = *reinterpret_cast<PairHead *>(smem);
  uint8_t *stages = smem + kHead;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int rank = static_cast<int>(blockIdx.x) & 1;
  const int first = static_cast<int>(blockIdx.x) >> 1, step = static_cast<int>(gridDim.x) >> 1;
  const int stage_bytes = a.stage_a + a.stage_b;
  volatile int *abort = &H.abort;

  if (t == 0) {
    for (int s = 0; s < a.stages; ++s) {
      bar_init(&H.full[s], 1);
      bar_init(&H.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      bar_init(&H.acc_full[s], 1);
      bar_init(&H.acc_empty[s], 2 * kEpiWarps);
    }
    for (int s = 0; s < kSlots; ++s) {
      bar_init(&H.slot_full[s], 1);
    }
    bar_init(&H.drain, 1);
    H.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    for (int i = 0; i < 2 * a.jobs; ++i) asm volatile("prefetch.tensormap [%0];" ::"l"(&a.map[i]) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&H.tmem)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync_all();  // both CTAs' barriers stand
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = H.tmem;
  pdl_enter();
  const int kept = a.kept ? *a.kept : a.tokens;
  if (kForward && kFew && a.ticket && blockIdx.x == 0 && t == 0) *a.ticket = 0;
  int tiles = 0;
  for (int j = 0; j < a.jobs; ++j) tiles += tiles_of(a.job[j], kept);
  Turn turn{a, H, a.next_tile != nullptr && kept > 0, tiles, 0, abort};  // (without a token no tile has a k block)

  if (warp == 0) {
    if (lane == 0) {
      asm volatile("fence.proxy.async;" ::: "memory");  // the rows were written by ordinary stores
      int s = 0, counted = 0;
      uint32_t ph = 0;
      for (int idx = -1;;) {
        if (rank == 0) {
          idx = turn.give(idx, counted, first, step);
          if (idx < 0) break;
          if (turn.counting) counted = atomicAdd(a.next_tile, 1);  // (its result is wanted after this tile's loads)
        } else {
          idx = turn.take<true>(idx, first, step);
          if (idx < 0) break;
        }
        const Tile tl = tile_at(a, kept, idx);
        const Job &j = a.job[tl.job];
        const CUtensorMap *ma = &a.map[2 * tl.job], *mb = ma + 1;
        const int half = tl.cols / 2, chunks = (half + kChunk - 1) / kChunk;
        const bool a_mn = a_is_mn(j), b_mn = b_is_mn(j);
        const uint32_t bytes = kOperand + (b_mn ? chunks * kBox : j.bn / 2 * 2 * kTileK);
        // Where the rows of the weights start: with the tile's rows, with the sum, or with its columns.
        const int a_row = j.swap && j.kind != kStates ? j.v0 : 0, a_k = j.swap && j.kind == kStates ? j.v0 : 0;
        const int b_row = !j.swap && !b_mn ? j.v0 : 0, b_k = !j.swap && j.kind == kStates ? j.v0 : 0;
        const int am = tl.m + rank * (kTileM / 2), bn = tl.n + rank * half;
        for (int i = 0; i < tl.nkb; ++i) {
          if (!bar_wait(&H.empty[s], ph ^ 1, abort, a.err)) goto loaded;
          uint8_t *sa = stages + s * stage_bytes, *sb = sa + a.stage_a;
          const int k = (tl.kb + i) * kTileK;
          // The first CTA's barrier counts the bytes of both; its phase cannot
          // end before its own arrival here.
          const uint32_t bar = cluster_addr(&H.full[s], 0);
          if (rank == 0) bar_expect(&H.full[s], 2 * bytes);
          if (a_mn) {
            tma_load_pair(ma, sa, bar, am, a_k + k);
            tma_load_pair(ma, sa + kBox, bar, am + kChunk, a_k + k);
          } else {
            tma_load_pair(ma, sa, bar, k, a_row + am);
            tma_load_pair(ma, sa + kBox, bar, k + kChunk, a_row + am);
          }
          if (b_mn) {
            for (int c = 0; c < chunks; ++c) tma_load_pair(mb, sb + c * kBox, bar, bn + c * kChunk, b_k + k);
          } else {
            tma_load_pair(mb, sb, bar, k, b_row + bn);
            tma_load_pair(mb, sb + a.stage_b / 2, bar, k + kChunk, b_row + bn);
          }
          if (++s == a.stages) s = 0, ph ^= 1;
        }
      }
    loaded:
      if (*abort) {  // copies in flight land long before this
        const unsigned long long t1 = now_ns();
        while (now_ns() - t1 < 20000000ull) {
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      int s = 0, acc = 0;
      uint32_t ph = 0, acc_ph = 0;
      bool ok = true;
      for (int idx = -1; ok;) {
        idx = turn.take<false>(idx, first, step);
        if (idx < 0) break;
        const Tile tl = tile_at(a, kept, idx);
        const Job &j = a.job[tl.job];
        const bool a_mn = a_is_mn(j), b_mn = b_is_mn(j);
        const uint32_t idesc = f16_idesc(kBf16, a_mn, b_mn, tl.cols);
        // 16 k are 32 bytes of a K-major row, 16 rows of 128 bytes of an MN-major
        // box; 64 k are a box of the one, half a box of the other.
        const uint64_t step_a = a_mn ? 2048 >> 4 : 32 >> 4, half_a = a_mn ? 8192 >> 4 : kBox >> 4;
        const uint64_t step_b = b_mn ? 2048 >> 4 : 32 >> 4, half_b = b_mn ? 8192 >> 4 : a.stage_b >> 5;
        const int slice = kForward || (kLong != kNone && j.kind == kProb) ? slice_blocks<kBf16, kForward, kFew>(tl.nkb)
                          : kLong == kTokens && j.kind == kHeadRows       ? sum_blocks<kBf16>(tl.nkb)
                                                                          : 0x7fffffff;
        for (int i = 0, at = 0; i < max(tl.nkb, 1); ++i) {  // (at: within a slice)
          if (at == 0) {
            ok = __all_sync(0xffffffffu, bar_wait(&H.acc_empty[acc], acc_ph ^ 1, abort, a.err));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          }
          if (tl.nkb == 0) break;
          ok = __all_sync(0xffffffffu, bar_wait(&H.full[s], ph, abort, a.err));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t st = su32(stages) + static_cast<uint32_t>(s * stage_bytes);
          const uint64_t ad = a_mn ? mn_desc(st) : tile_desc(st);
          const uint64_t bd = b_mn ? mn_desc(st + a.stage_a) : tile_desc(st + a.stage_a);
#pragma unroll
          for (int k = 0; k < kTileK / 16; ++k)
            mma_f16_pair(tmem + acc * kTileN, ad + k / 4 * half_a + k % 4 * step_a, bd + k / 4 * half_b + k % 4 * step_b,
                         idesc, at > 0 || k > 0);
          mma_commit_pair(&H.empty[s]);
          if (++s == a.stages) s = 0, ph ^= 1;
          if (++at == slice && i + 1 < tl.nkb) {
            mma_commit_pair(&H.acc_full[acc]);
            if (++acc == 2) acc = 0, acc_ph ^= 1;
            at = 0;
          }
        }
        if (!ok) break;
        mma_commit_pair(&H.acc_full[acc]);
        if (++acc == 2) acc = 0, acc_ph ^= 1;
      }
      // No MMA of the pair is left when this arrives (the last sync below holds
      // the other CTA until then).
      asm volatile(
          "{\n\t.reg .pred e;\n\t"
          "elect.sync _|e, 0xffffffff;\n\t"
          "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(su32(&H.drain))
          : "memory");
      bar_wait(&H.drain, 0, abort, a.err, false);
    }
  } else {
    // The warp's number from lane 0: the compiler then keeps what follows from
    // it, the column addresses above all, in uniform registers.
    const int uwarp = __shfl_sync(0xffffffffu, warp, 0);
    const int quarter = uwarp & 3, part = (uwarp - 2) >> 2;  // TMEM lanes, and first or second part of the columns
    const uint32_t ta = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    float *turned = reinterpret_cast<float *>(stages + kRing) + (uwarp - 2) * 32 * kBlockPitch;
    constexpr int kWordPitch = 17;  // the same of 16-bit elements
    uint32_t *words = reinterpret_cast<uint32_t *>(turned);
    int acc = 0;
    uint32_t ph = 0;
    // An accumulator is free once both CTAs' warps have read it.  (The arrival
    // tells of reads of TMEM and of nothing in memory: its release at the scope of
    // the cluster would wait for the tile's stores to arrive in L2.)
    auto release = [&] {
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr(&H.acc_empty[acc], 0))
                     : "memory");
      if (++acc == 2) acc = 0, ph ^= 1;
    };
    // The bits of the logits of a tile's columns c0 + 32 q: a slice of k after the
    // other.  The first slice's loads are in flight together.
    auto gather = [&](auto &sum, int nkb, int slice, int c0, int c1) {
      constexpr int Q = sizeof(sum) / sizeof(sum[0]);
      for (int i = 0; i < nkb; i += slice) {
        if (!__all_sync(0xffffffffu, bar_wait(&H.acc_full[acc], ph, abort, a.err))) return false;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t d = ta + acc * kTileN + c0;
        __syncwarp();
        if (i == 0) {
#pragma unroll
          for (int q = 0; q < Q; ++q)
            if (c0 + 32 * q < c1) tmem_ask32(d + 32 * q, sum[q]);
#pragma unroll
          for (int q = 0; q < Q; ++q) tmem_wait32(sum[q]);
        } else {
#pragma unroll
          for (int q = 0; q < Q; ++q) {
            if (c0 + 32 * q >= c1) break;
            int r[32];
            tmem_ask32(d + 32 * q, r);
            tmem_wait32(r);
#pragma unroll
            for (int k = 0; k < 32; ++k)
              sum[q][k] = __float_as_int(__int_as_float(sum[q][k]) + __int_as_float(r[k]));
          }
        }
        release();
      }
      return true;
    };
    RowState few[2];  // of this lane's tokens where they are the tiles' columns: kept from tile to tile
    int few_target[2];
    if (kFew) {
      const Job &j = a.job[a.job[0].swap ? 0 : a.jobs - 1];
      const int mid = (j.bn / 2 + 31) / 32 * 32;
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int token = (part ? mid : 0) + 32 * q + lane;
        RowState &st = few[q];
        st.live = token < kept && token < (part ? j.bn : mid);
        st.lse = st.log2f = st.own = 0.f;
        if (!kForward && st.live) prob_row(a, token, st);
        few_target[q] = -1;
        if (st.live) {
          const int64_t label = a.labels ? a.labels[token] : a.target[token];
          few_target[q] = label >= 0 && label < a.vocab ? static_cast<int>(label) : -1;
        }
        st.m = kNegInf;
        st.s = st.z = 0.f;
        st.found = false;
      }
    }
    for (int idx = -1;;) {
      idx = turn.take<false>(idx, first, step);
      if (idx < 0) break;
      const Tile tl = tile_at(a, kept, idx);
      const Job &j = a.job[tl.job];
      const int mid = (tl.cols / 2 + 31) / 32 * 32, c0 = part ? mid : 0, c1 = part ? tl.cols : mid;
      if (kForward && !kFew) {  // (asked for ahead of the wait)
        const int row = tl.m + rank * (kTileM / 2) + quarter * 32 + lane;
        few_target[0] = row < kept ? a.target[row] : -1;
      }
      if (kFew && (kForward || j.swap)) {
        // A lane holds a row of the weights and the columns are tokens: 32 x 32 of
        // them turn in shared memory, and each lane goes on with a token's row.
        const int row0 = tl.m + rank * (kTileM / 2) + quarter * 32;
        const bool logits = kForward || (kLong != kNone && j.kind == kProb);
        int sum[kLong != kNone ? 2 : 1][32];
        if (logits) {
          if (!gather(sum, tl.nkb, slice_blocks<kBf16, kForward, kFew>(tl.nkb), c0, c1)) break;
        } else {
          if (!__all_sync(0xffffffffu, bar_wait(&H.acc_full[acc], ph, abort, a.err))) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int c = c0 + 32 * q, token = c + lane;
          if (c >= c1) break;
          float z[32];
          __syncwarp();
          if (logits) {
#pragma unroll
            for (int i = 0; i < 32; ++i) turned[lane * kBlockPitch + i] = __int_as_float(sum[kLong != kNone ? q : 0][i]);
          } else {
            int r[32];
            tmem_ask32(ta + acc * kTileN + c, r);
            tmem_wait32(r);
#pragma unroll
            for (int i = 0; i < 32; ++i) turned[lane * kBlockPitch + i] = __int_as_float(r[i]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 32; ++i) z[i] = turned[i * kBlockPitch + lane];
          RowState &st = few[q];
          st.target = st.live ? few_target[q] - (j.v0 + row0) : 0x7fffffff;
          st.limit = a.vocab - (j.v0 + row0);
          if (kForward) {
            loss_chunk(st, 0, z);
          } else if (j.kind == kProb) {
            prob_chunk<kBf16>(st, static_cast<uint16_t *>(j.out) + token * j.pitch + row0, 0, z);
          } else if (st.live && row0 < j.pitch) {
            states_chunk(j.add, static_cast<float *>(j.out) + tl.slice * j.plane + token * j.pitch + row0, z);
          }
        }
        if (!logits) release();
        continue;
      }
      if constexpr (kForward && !kFew) {
        int sum[4][32];
        if (!gather(sum, tl.nkb, slice_blocks<kBf16, kForward, kFew>(tl.nkb), c0, c1)) break;
        auto z = [&](int q, int k) -> float { return __int_as_float(sum[q][k]); };
        const int limit = a.vocab - tl.n;
        if (c1 > limit || c0 + 128 > c1) {  // columns that are not there
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c0 + 32 * q + k >= min(c1, limit)) sum[q][k] = __float_as_int(kNegInf);
        }
        // Four chains each, of the 128 columns' maximum and sum.
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          top[q] = z(q, 0);
#pragma unroll
          for (int k = 1; k < 32; ++k) top[q] = fmaxf(top[q], z(q, k));
        }
        const float m = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])), base = exp_base(m);
        float part_sum[4] = {};
#pragma unroll
        for (int k = 0; k < 32; ++k)
#pragma unroll
          for (int q = 0; q < 4; ++q) part_sum[q] += exp2_fast((z(q, k) - base) * kLog2e);
        const int row = tl.m + rank * (kTileM / 2) + quarter * 32 + lane;
        if (row < kept) {
          a.parts[(static_cast<int64_t>(tl.n / j.bn) * 2 + part) * a.part_pitch + row] =
              make_float2(m, (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]));
          const int at = few_target[0] - tl.n - c0;
          if (at >= 0 && at < c1 - c0) {
            float own = 0.f;
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (at == 32 * q + k) own = z(q, k);
            a.z_target[row] = own;
          }
        }
        continue;
      }
      const int row0 = tl.m + rank * (kTileM / 2) + quarter * 32, row = row0 + lane;
      RowState st;
      st.live = row < (j.kind == kHeadRows ? j.m_total : kept);
      st.target = 0x7fffffff;
      st.lse = st.log2f = st.own = 0.f;
      st.limit = a.vocab - (j.v0 + tl.n);
      st.m = kNegInf;
      st.s = st.z = 0.f;
      st.found = false;
      if (!kFew && j.kind == kProb && st.live) {
        st.target = a.target[row] - (j.v0 + tl.n);
        prob_row(a, row, st);
      }
      const float scale = j.kind == kHeadRows ? *a.scale : 1.f;
      const int kind = j.kind, left0 = j.n_total - tl.n;
      const int64_t pitch = j.pitch;
      const bool add = j.add;
      uint16_t *out16 = static_cast<uint16_t *>(j.out) + (kind == kProb ? row : j.v0 + static_cast<int64_t>(row)) * pitch + tl.n;
      float *out32 = static_cast<float *>(j.out) + tl.slice * j.plane + row * pitch + tl.n;
      auto head_chunk = [&](int c, const int (&r)[32]) {
        float z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = __int_as_float(r[i]) * scale;
        const int left = left0 - c;
        if (a.row_bytes == 2) {
          // A lane holds a row.  Turned, a warp writes 32 columns of a row at a
          // time (the gradients of [333,1153] x [50257,1153] in 133 us; with padded
          // rows in scratch and a copy of them behind it 111 + 40, in words of two
          // elements shifted by one in odd rows 172, from the row's lane 203).
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 16; ++i) words[lane * kWordPitch + i] = pack2<kBf16>(z[2 * i], z[2 * i + 1]);
          __syncwarp();
          const int rows = min(32, j.m_total - row0);
          const uint16_t *from = reinterpret_cast<const uint16_t *>(words) + lane;
          uint16_t *to = out16 + c + lane - lane * pitch;
          if (lane < left && rows == 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i, to += pitch) *to = from[2 * kWordPitch * i];
          } else if (lane < left) {
            for (int i = 0; i < rows; ++i, to += pitch) *to = from[2 * kWordPitch * i];
          }
          return;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack2<kBf16>(z[16 * h + 2 * i], z[16 * h + 2 * i + 1]);
          uint16_t *to = out16 + c + 16 * h;
          if (a.row_bytes == 32) {
            if (st.live && 16 * h < left) store32B(to, w);
          } else {
            if (st.live && 16 * h < left) *reinterpret_cast<uint4 *>(to) = make_uint4(w[0], w[1], w[2], w[3]);
            if (st.live && 16 * h + 8 < left) *reinterpret_cast<uint4 *>(to + 8) = make_uint4(w[4], w[5], w[6], w[7]);
          }
        }
      };
      auto chunk = [&](int c, const int (&r)[32]) {
        if (kind == kHeadRows) return head_chunk(c, r);
        float z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = __int_as_float(r[i]);
        if (!kFew && kind == kProb) {
          prob_chunk<kBf16>(st, out16, c, z);
        } else if (st.live) {
          states_chunk(add, out32 + c, z);
        }
      };
      if (!kFew && ((kLong != kNone && kind == kProb) || (kLong == kTokens && kind == kHeadRows && kept > 0))) {
        int sum[4][32];
        const int slice = kind == kProb ? slice_blocks<kBf16, kForward, kFew>(tl.nkb) : sum_blocks<kBf16>(tl.nkb);
        if (!gather(sum, tl.nkb, slice, c0, c1)) break;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if (c0 + 32 * q >= c1) break;
          if (kLong == kTokens && kind == kHeadRows) {
            head_chunk(c0 + 32 * q, sum[q]);
          } else {
            float z[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) z[i] = __int_as_float(sum[q][i]);
            prob_chunk<kBf16>(st, out16, c0 + 32 * q, z);
          }
        }
        continue;
      }
      if (!__all_sync(0xffffffffu, bar_wait(&H.acc_full[acc], ph, abort, a.err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (int c = c0; c < c1; c += 32) {
        int r[32];
        __syncwarp();
        tmem_ask32(ta + acc * kTileN + c, r);
        tmem_wait32(r);
        if (tl.nkb == 0) {  // an empty sum has no MMA
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
        chunk(c, r);
      }
      release();
    }
    if (kForward && kFew) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int token = (part ? (a.job[0].bn / 2 + 31) / 32 * 32 : 0) + 32 * q + lane;
        if (!few[q].live) continue;
        a.parts[(static_cast<int64_t>(blockIdx.x) * 4 + quarter) * a.part_pitch + token] = make_float2(few[q].m, few[q].s);
        if (few[q].found) a.z_target[token] = few[q].z;
      }
    }
  }
  __syncwarp();
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while the other may signal it
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ---------------------------------------------------------------------------
// Rows: which tokens have a loss, and their states side by side
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

// What the forward pass leaves for the backward pass: the number of kept
// tokens, each token's target (kNoTarget: not in the vocabulary, kIgnored), and
// by the kept tokens' places the log of the sum of exponentials and the loss.
constexpr int kNoTarget = -1, kIgnored = -2;
struct State {
  int *kept, *target;
  float *lse, *loss;
};
State state_at(const int32_t *state, int64_t tokens) {
  int32_t *p = const_cast<int32_t *>(state);  // (only the forward pass writes it)
  return {p, p + 1, reinterpret_cast<float *>(p + 1 + tokens), reinterpret_cast<float *>(p + 1 + 2 * tokens)};
}

// 8 elements at a row's element c (a multiple of 8) of x, from any alignment;
// zeros past the row's end.
struct RowSource {
  const uint16_t *x;
  int64_t stride;
  int tokens, in;
  bool vec;  // rows lie on 16 bytes
  __device__ __forceinline__ uint4 load(int64_t r, int c) const {
    const uint16_t *p = x + r * stride + c;
    if (vec) return __ldg(reinterpret_cast<const uint4 *>(p));
    return load16_any(reinterpret_cast<const int8_t *>(p), 2 * (in - c), reinterpret_cast<const int8_t *>(x),
                      reinterpret_cast<const int8_t *>(x + (tokens - 1) * stride + in));
  }
};

struct RowsArgs {
  RowSource x;
  const int64_t *labels;
  const int *counts;  // kept tokens of each block, or null
  int64_t ignore;
  int vocab;
  State st;
  int *token, *target;  // of each place
  uint16_t *rows;  // copied states, `pitch` elements a row
  int64_t pitch;
  float *loss;     // of each token, or null
  unsigned *ticket;
  int per_block;
};

__device__ __forceinline__ int block_sum(int v, int *red) {
  v = __reduce_add_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  int sum = 0;
  for (int w = 0; w < kRowThreads / 32; ++w) sum += red[w];
  __syncthreads();
  return sum;
}

// The place of the thread's token among the block's kept ones, and their number.
__device__ __forceinline__ int block_place(bool keep, int *count, int *warp_base) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned votes = __ballot_sync(0xffffffffu, keep);
  if (lane == 0) warp_base[warp] = __popc(votes);
  __syncthreads();
  int at = __popc(votes & ((1u << lane) - 1));
  *count = 0;
  for (int w = 0; w < kRowThreads / 32; ++w) {
    if (w < warp) at += warp_base[w];
    *count += warp_base[w];
  }
  return at;
}

// What each block of a row kernel needs of all tokens, by the tokens of a block:
// how many are kept, and the largest |g| of the kept ones.  Up to 16,384 tokens the
// row kernels' blocks look at all tokens themselves, which costs less than one
// launch more; with 2^20 it made 0.5 ms of [1048576,64] x [256,64]'s loss (1.8 ms)
// and 9 ms of its gradients with a factor for each token (14.8).
constexpr int64_t kGroupedTokens = 16384;
struct GroupArgs {
  const int64_t *labels;  // forward: the targets as they are given
  int64_t ignore;
  const int *target;      // backward: the state's
  const float *dloss;     // null: no tops
  int64_t dloss_stride;
  RowSource x;            // of tops with the states' sizes; x null: without
  int64_t tokens;
  int per_block;
  int *counts, *tops;
};

// A token's factor as m * 2^power: m, never below 0, in [1, 2) and held in d
// before its rounding, in fp16 in [1/2, 1): there d is held times 2^15, and p may
// come out above 1 by what its logit's sum was cut off (4e-4 of a logit of -100),
// so that a factor up to 2 would leave fp16's range.  Zeros, infinities and NaN are
// all in m, and have no say in what the others are relative to.
struct Factor {
  float m, sign;
  int power;
  bool real;
  __device__ Factor(float g, bool bf16) {
    m = fabsf(g);
    sign = copysignf(1.f, g);
    power = 0;
    real = m > 0.f && m < INFINITY;
    if (!real) return;
    m = frexpf(m, &power);
    if (bf16) {
      m *= 2.f;
      --power;
    }
  }
};
constexpr int kNoTop = INT_MIN;

__device__ __forceinline__ int block_max(int v, int *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int w = 0; w < kRowThreads / 32; ++w) v = max(v, red[w]);
  __syncthreads();
  return v;
}

// (tops: of bf16 where there are no sizes, of fp16 with them)
__global__ void __launch_bounds__(kRowThreads) ce_groups_kernel(const GroupArgs a) {
  __shared__ int red[kRowThreads / 32];
  __shared__ unsigned size[kRowThreads];
  pdl_enter();
  const int t = threadIdx.x;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.per_block, r = r0 + t;
  const bool mine = t < a.per_block && r < a.tokens;
  const bool kept = mine && (a.labels ? __ldg(a.labels + r) != a.ignore : __ldg(a.target + r) != kIgnored);
  const int count = block_sum(kept, red);
  if (t == 0) a.counts[blockIdx.x] = count;
  if (!a.dloss) return;
  const bool sizes = a.x.x != nullptr;
  const Factor f(kept ? __ldg(a.dloss + r * a.dloss_stride) : 0.f, !sizes);
  int top = f.real ? f.power : kNoTop;
  if (sizes) {
    // The largest finite magnitude of each row, as bits.
    size[t] = f.real ? 0 : ~0u;
    __syncthreads();
    const int rows = static_cast<int>(min(static_cast<int64_t>(a.per_block), a.tokens - r0)), vecs = (a.x.in + 7) / 8;
    for (int i = t; i < rows * vecs; i += kRowThreads) {
      const int row = i / vecs;
      if (size[row] == ~0u) continue;
      const uint4 v = a.x.load(r0 + row, 8 * (i - row * vecs));
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      unsigned most = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned h = w[k / 2] >> (16 * (k & 1)) & 0x7fffu;
        if (h < 0x7c00u) most = max(most, h);
      }
      if (most > *const_cast<volatile unsigned *>(&size[row])) atomicMax(&size[row], most);
    }
    __syncthreads();
    if (f.real) {
      int e;
      const float most = __half2float(__ushort_as_half(static_cast<uint16_t>(size[t])));
      frexpf(most, &e);
      top = most > 0.f ? f.power + e : kNoTop;
    }
  }
  top = block_max(top, red);
  if (t == 0) a.tops[blockIdx.x] = top;
}

// Block b takes tokens b * per_block on.  It counts the kept tokens before its
// own, so the places are those of the tokens' order whatever the blocks' order
// is (the targets, 8 bytes a token, lie in L2; of many tokens it adds the blocks' counts).
__global__ void __launch_bounds__(kRowThreads) ce_rows_kernel(const RowsArgs a) {
  __shared__ int red[kRowThreads / 32], warp_base[kRowThreads / 32], from[kRowThreads];
  pdl_enter();
  const int t = threadIdx.x;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.per_block;
  int before = 0, count;
  if (a.counts)
    for (int i = t; i < static_cast<int>(blockIdx.x); i += kRowThreads) before += __ldg(a.counts + i);
  else
    for (int64_t i = t; i < r0; i += kRowThreads) before += __ldg(a.labels + i) != a.ignore;
  before = block_sum(before, red);
  // per_block is at most the number of threads.
  const int64_t r = r0 + t;
  const bool mine = t < a.per_block && r < a.x.tokens;
  const int64_t label = mine ? __ldg(a.labels + r) : a.ignore;
  const bool keep = mine && label != a.ignore;
  const int at = block_place(keep, &count, warp_base);
  const int target = !keep ? kIgnored : label >= 0 && label < a.vocab ? static_cast<int>(label) : kNoTarget;
  if (mine) {
    a.st.target[r] = target;
    if (!keep && a.loss) a.loss[r] = 0.f;
  }
  if (keep) {
    from[at] = t;
    a.target[before + at] = target;
    a.token[before + at] = static_cast<int>(r);
  }
  __syncthreads();
  const int vecs = (a.x.in + 7) / 8;
  uint4 *out = reinterpret_cast<uint4 *>(a.rows + before * a.pitch);
#pragma unroll 4
  for (int i = t; i < count * vecs; i += kRowThreads) {
    const int row = i / vecs, c = i - row * vecs;
    out[row * (a.pitch / 8) + c] = a.x.load(r0 + from[row], 8 * c);
  }
  if (blockIdx.x + 1 == gridDim.x && t == 0) {
    *a.st.kept = before + count;
    *a.ticket = 0;
  }
}

struct BackRowsArgs {
  RowSource x;
  State st;
  uint16_t *rows;    // copied states
  uint16_t *scaled;  // the same times their factor's power of two (for dW), or null
  int *place;        // of each token among the kept ones (-1: ignored)
  int *target;       // of each kept token
  float *own;        // and d there, times what its row of d is held times
  float *log_factor; // log2 of the rest of each kept token's factor, in fp16 times 2^15; null: g is the same for all
  float *power;      // each token's power of two, signed, in fp16 over 2^15
  int64_t pitch;
  const float *dloss;
  int64_t dloss_stride;
  const int *counts; // kept tokens of each block's tokens, or null
  const int *tops;   // and the power that their scaled states are relative to
  bool mean;
  float *scale;      // [0] factor of dW, [1] factor of dx where g is the same for all
  int *counters;     // of the launches that follow, set to 0
  int n_counters;
  int per_block;
};

// The copies of the backward pass.  A token's own factor is cut in two.  m goes
// into its row of d, and is rounded with it: no rounding more, and d's relative
// error is the one it has without.  The power of two goes into dx at the end, and
// for dW into the token's states.  bf16 has fp32's range for that: the powers are
// relative to the largest, and the states exact.  fp16 has not: relative to the
// largest factor, a state of 1 keeps 8 bits at a ratio of 2^-16 and none from 2^-25
// on, and a row of dW that only such tokens feed is off by as much.  There the
// powers are such that the largest state times its factor comes to lie below 2^15,
// and what is cut off is 2^-40 of that: less than half of dW's own smallest step
// wherever that product, times a d of one, is in fp16's range itself.  (A launch
// more and a pass over x for its sizes: 3 us of the step of [16,512] x [5000,512].)
template <bool kBf16>
__global__ void __launch_bounds__(kRowThreads) ce_back_rows_kernel(const BackRowsArgs a) {
  __shared__ float powers[kRowThreads];
  __shared__ int red[kRowThreads / 32], warp_base[kRowThreads / 32], places[kRowThreads];
  pdl_enter();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int kept = *a.st.kept;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * a.per_block;
  const bool each = a.log_factor != nullptr;
  int before = 0, count, top = kNoTop;
  if (a.counts) {
    for (int i = t; i < static_cast<int>(gridDim.x); i += kRowThreads) {
      if (i < static_cast<int>(blockIdx.x)) before += __ldg(a.counts + i);
      if (a.scaled) top = max(top, __ldg(a.tops + i));
    }
  } else {
    for (int64_t i = t; i < (a.scaled ? a.x.tokens : r0); i += kRowThreads) {
      if (__ldg(a.st.target + i) == kIgnored) continue;
      if (i < r0) ++before;
      if (a.scaled) {
        const Factor f(__ldg(a.dloss + i * a.dloss_stride), kBf16);
        if (f.real) top = max(top, f.power);
      }
    }
  }
  before = block_sum(before, red);
  if (a.scaled) top = block_max(top, red);
  // The scaled states are those of a factor of 2^unit.
  const int prob_power = kBf16 ? 0 : 15, unit = top == kNoTop ? 0 : top - prob_power;
  // The thread's token: its place, its target's d (see prob_chunk), its factor.
  const int64_t r = r0 + t;
  const bool mine = t < a.per_block && r < a.x.tokens;
  const int target = mine ? __ldg(a.st.target + r) : kIgnored;
  const bool keep = target != kIgnored;
  const int place = before + block_place(keep, &count, warp_base);
  places[t] = keep ? place : -1;
  if (mine) a.place[r] = places[t];
  if (keep) {
    float held = static_cast<float>(1 << prob_power);
    if (each) {
      const Factor f(__ldg(a.dloss + r * a.dloss_stride), kBf16);
      held *= f.m;
      a.log_factor[place] = log2f(held);
      a.power[r] = ldexpf(f.sign, f.power - prob_power);
      // (At most 2^39 where a state is not 0; one of zeros stays 0.)
      powers[t] = f.real ? ldexpf(f.sign, min(f.power - unit, 64)) : f.sign;
    }
    a.target[place] = target;
    // (With an infinite factor the row is no number: NaN at the target, so that dW is loud.)
    a.own[place] = held < INFINITY ? held * expm1f(-__ldg(a.st.loss + place)) : NAN;
  }
  __syncthreads();
  const int rows = static_cast<int>(min(static_cast<int64_t>(a.per_block), a.x.tokens - r0)), vecs = (a.x.in + 7) / 8;
#pragma unroll 2
  for (int i = t; i < rows * vecs; i += kRowThreads) {
    const int row = i / vecs, c = i - row * vecs;
    const int at = places[row];
    if (at < 0) continue;
    const uint4 v = a.x.load(r0 + row, 8 * c);
    reinterpret_cast<uint4 *>(a.rows + at * a.pitch)[c] = v;
    if (!a.scaled) continue;
    const float g = powers[row];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint16_t lo = static_cast<uint16_t>(w[k]), hi = static_cast<uint16_t>(w[k] >> 16);
      const float x0 = kBf16 ? __bfloat162float(__ushort_as_bfloat16(lo)) : __half2float(__ushort_as_half(lo));
      const float x1 = kBf16 ? __bfloat162float(__ushort_as_bfloat16(hi)) : __half2float(__ushort_as_half(hi));
      o[k] = pack2<kBf16>(x0 * g, x1 * g);
    }
    reinterpret_cast<uint4 *>(a.scaled + at * a.pitch)[c] = make_uint4(o[0], o[1], o[2], o[3]);
  }
  if (blockIdx.x + 1 == gridDim.x) {
    for (int i = t; i < a.n_counters; i += kRowThreads) a.counters[i] = 0;
    // The sums over tokens run in steps of 128: zeros up to there.
    const int end = (kept + kTileK - 1) / kTileK * kTileK;
    uint16_t *rows = a.scaled ? a.scaled : a.rows;
    for (int r = kept + warp; r < end; r += kRowThreads / 32)
      for (int c = lane; c < a.x.in; c += 32) rows[r * a.pitch + c] = 0;
    if (t == 0) {
      const float g = each ? ldexpf(1.f, unit - prob_power)
                           : (a.mean ? a.dloss[0] / static_cast<float>(kept) : a.dloss[0]) / static_cast<float>(1 << prob_power);
      a.scale[0] = kept ? g : 0.f;
      a.scale[1] = g;
    }
  }
}

// 8 elements from S words and H halves into two neighbouring 16-byte blocks.
template <int S, bool H>
__device__ __forceinline__ uint4 shifted(uint4 x, uint4 y) {
  const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = H ? __funnelshift_r(v[S + i], v[S + i + 1], 16) : v[S + i];
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// The head's rows at any pitch and alignment, copied to rows of `pitch`
// elements on 16 bytes, a warp a row: [50257,1153] 41 us for 232 MB, where the
// general copy by vectors of the int8 product, whose shifts differ from thread
// to thread, took 59.  What stands past a row's end is not read.
__global__ void __launch_bounds__(kRowThreads) ce_copy_head_kernel(const uint16_t *w, int64_t stride, int64_t rows,
                                                                   int in, uint16_t *out, int64_t pitch) {
  pdl_enter();
  const int lane = threadIdx.x & 31, vecs = (in + 7) / 8;
  const int8_t *lo = reinterpret_cast<const int8_t *>(w);
  const int8_t *hi = reinterpret_cast<const int8_t *>(w + (rows - 1) * stride + in);
  for (int64_t r = blockIdx.x * static_cast<int64_t>(kRowThreads / 32) + (threadIdx.x >> 5); r < rows;
       r += static_cast<int64_t>(gridDim.x) * (kRowThreads / 32)) {
    const int8_t *p = reinterpret_cast<const int8_t *>(w + r * stride);
    const uint32_t off = offset16(p);
    uint4 *to = reinterpret_cast<uint4 *>(out + r * pitch);
    if (p - off < lo || p - off + (vecs + 1) * 16 > hi) {  // blocks that reach past the matrix
      for (int c = lane; c < vecs; c += 32) to[c] = load16_any(p + 16 * c, 2 * in - 16 * c, lo, hi);
      continue;
    }
    const uint4 *from = reinterpret_cast<const uint4 *>(p - off);
    constexpr int U = 4;
    for (int c0 = lane; c0 < vecs; c0 += 32 * U) {
      uint4 x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = min(c0 + 32 * u, vecs - 1);
        x[u] = __ldg(from + c);
        y[u] = __ldg(from + c + 1);
      }
      auto put = [&](auto f) {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (c0 + 32 * u < vecs) to[c0 + 32 * u] = f(x[u], y[u]);
      };
      switch (off >> 1) {  // (the same for the warp)
        case 0: put([](uint4 a, uint4 b) { return shifted<0, false>(a, b); }); break;
        case 1: put([](uint4 a, uint4 b) { return shifted<0, true>(a, b); }); break;
        case 2: put([](uint4 a, uint4 b) { return shifted<1, false>(a, b); }); break;
        case 3: put([](uint4 a, uint4 b) { return shifted<1, true>(a, b); }); break;
        case 4: put([](uint4 a, uint4 b) { return shifted<2, false>(a, b); }); break;
        case 5: put([](uint4 a, uint4 b) { return shifted<2, true>(a, b); }); break;
        case 6: put([](uint4 a, uint4 b) { return shifted<3, false>(a, b); }); break;
        default: put([](uint4 a, uint4 b) { return shifted<3, true>(a, b); }); break;
      }
    }
  }
}

// ---------------------------------------------------------------------------
// The loss from the tiles' maxima and sums
// ---------------------------------------------------------------------------
struct CombineArgs {
  State st;
  const float2 *parts;
  int64_t part_pitch;
  int n_parts;
  const float *z_target;
  const int *token, *target;
  float *row_loss;   // by place (sum, mean)
  float *loss;       // of each token, or the one value
  int reduction;     // H24_REDUCE_*
  unsigned *ticket;
  // Where the tokens' own rows were multiplied (few tokens): the state is made here.
  const int64_t *labels;
  int64_t ignore;
  int tokens, vocab;
};
constexpr int kCombineRows = 4;  // 32 bytes of neighbouring parts; one row a block where tokens are few

template <int ROWS>
__global__ void __launch_bounds__(kRowThreads) ce_combine_kernel(const CombineArgs a) {
  __shared__ float2 red[kRowThreads / 32][ROWS];
  __shared__ double sums[kRowThreads / 32];
  __shared__ bool last;
  pdl_enter();
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const bool own = ROWS == 1 && a.labels;  // rows by token, not by place
  int kept, place = 0, n_mean = 0;
  bool known = true, keep = true;
  if (own) {
    const bool counts = t < a.tokens && a.labels[t] != a.ignore;  // (at most 128 tokens)
    const int64_t label = a.labels[blockIdx.x];
    keep = label != a.ignore;
    known = label >= 0 && label < a.vocab;
    place = __syncthreads_count(counts && t < static_cast<int>(blockIdx.x));
    const int total = __syncthreads_count(counts);
    kept = a.tokens;
    if (t == 0) {
      a.st.target[blockIdx.x] = !keep ? kIgnored : known ? static_cast<int>(label) : kNoTarget;
      if (blockIdx.x == 0) *a.st.kept = total;
      if (!keep && a.reduction == H24_REDUCE_NONE) a.loss[blockIdx.x] = 0.f;
      if (!keep && a.reduction != H24_REDUCE_NONE) a.row_loss[blockIdx.x] = 0.f;
    }
    n_mean = total;
  } else {
    kept = *a.st.kept;
    n_mean = kept;
  }
  const int r = t % ROWS;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + r;
  auto join = [](float2 &p, float2 q) {
    const float m = fmaxf(p.x, q.x), base = exp_base(m);
    p.y = p.y * exp2_fast((p.x - base) * kLog2e) + q.y * exp2_fast((q.x - base) * kLog2e);
    p.x = m;
  };
  float2 p = make_float2(kNegInf, 0.f);
  if (row < kept) {
#pragma unroll 8
    for (int i = t / ROWS; i < a.n_parts; i += kRowThreads / ROWS)
      join(p, __ldg(a.parts + i * a.part_pitch + row));
  }
  for (int o = 16; o >= ROWS; o >>= 1)
    join(p, make_float2(__shfl_xor_sync(0xffffffffu, p.x, o), __shfl_xor_sync(0xffffffffu, p.y, o)));
  if (lane < ROWS) red[warp][lane] = p;
  __syncthreads();
  if (t < ROWS && row < kept && keep) {
    for (int w = 1; w < kRowThreads / 32; ++w) join(p, red[w][t]);
    // A target outside the vocabulary has no loss: NaN, here and in the gradients.
    if (!own) known = a.target[row] >= 0;
    const float rest = known ? logf(p.y) : __int_as_float(0x7fffffff), lse = p.x + rest;
    const float loss = known ? (p.x - a.z_target[row]) + rest : rest;  // (both parts are 0 or more)
    a.st.lse[own ? place : row] = lse;
    a.st.loss[own ? place : row] = loss;
    if (a.reduction == H24_REDUCE_NONE)
      a.loss[own ? row : a.token[row]] = loss;
    else
      a.row_loss[row] = loss;
  }
  if (a.reduction == H24_REDUCE_NONE) return;
  // The block that is last to finish adds up all rows, in an order of its own
  // threads: the same for every call.
  __threadfence();
  __syncthreads();
  if (t == 0) last = atomicAdd(a.ticket, 1u) + 1 == gridDim.x;
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0.0;
#pragma unroll 8
  for (int i = t; i < kept; i += kRowThreads) sum += static_cast<double>(__ldcg(a.row_loss + i));
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) sums[warp] = sum;
  __syncthreads();
  if (t == 0) {
    sum = 0.0;
    for (int w = 0; w < kRowThreads / 32; ++w) sum += sums[w];
    *a.loss = static_cast<float>(a.reduction == H24_REDUCE_MEAN ? sum / n_mean : sum);
  }
}

// ---------------------------------------------------------------------------
// dx from the slices' sums
// ---------------------------------------------------------------------------
struct StatesArgs {
  const int *place;
  const float *acc;
  int64_t pitch, plane;
  int slices;
  int64_t tokens;
  int in;
  const float *scale;
  const float *power;  // a factor for each token, or null: scale[1]
  uint16_t *out;
  bool vec;            // out's rows lie on 16 bytes
};

template <bool kBf16>
__global__ void __launch_bounds__(kRowThreads) ce_states_kernel(const StatesArgs a) {
  pdl_enter();
  const int groups = (a.in + 7) / 8;
  const int64_t total = a.tokens * groups;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kRowThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kRowThreads) {
    const int64_t r = i / groups;
    const int c = static_cast<int>(i - r * groups) * 8;
    const int place = __ldg(a.place + r);
    float v[8] = {};
    if (place >= 0) {
      // (The rows of acc are padded to 32 columns.)
      const float *p = a.acc + place * a.pitch + c;
#pragma unroll 4
      for (int s = 0; s < a.slices; ++s, p += a.plane) {
        const float4 x = __ldcs(reinterpret_cast<const float4 *>(p)), y = __ldcs(reinterpret_cast<const float4 *>(p) + 1);
        v[0] += x.x, v[1] += x.y, v[2] += x.z, v[3] += x.w;
        v[4] += y.x, v[5] += y.y, v[6] += y.z, v[7] += y.w;
      }
      const float g = a.power ? a.power[r] : a.scale[1];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] *= g;
    }
    uint16_t *out = a.out + r * a.in + c;
    if (a.vec) {
      *reinterpret_cast<uint4 *>(out) = make_uint4(pack2<kBf16>(v[0], v[1]), pack2<kBf16>(v[2], v[3]),
                                                   pack2<kBf16>(v[4], v[5]), pack2<kBf16>(v[6], v[7]));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c + j < a.in) out[j] = pack1<kBf16>(v[j]);
    }
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Bytes of d for one piece of the vocabulary, and the columns that it has at
// least: with many tokens narrow pieces cost more in dx's fp32 sums, which are
// read and written for each, and leave too few tiles of dW (with 192 MiB alone
// [131072,1920] x [50688,1920] took 108 ms a step, 86 so; [262144,1024] x
// [4096,1024] 29 and 9.0).
constexpr int64_t kPieceBytes = int64_t(192) << 20, kPieceCols = 4096;

// Map of a matrix of 16-bit elements [rows][cols], row pitch `pitch` elements,
// in boxes of 64 columns x box_rows with the 128-byte swizzle.
bool map16(CUtensorMap *map, const void *base, int64_t rows, int64_t cols, int64_t pitch, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch) * 2};
  const cuuint32_t box[2] = {kChunk, static_cast<cuuint32_t>(box_rows)}, es[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void *>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
int64_t cdiv(int64_t n, int64_t by) { return (n + by - 1) / by; }

// Pool scratch that is freed on the stream when the call is through with it.
struct Scratch {
  cudaStream_t s;
  uint8_t *base = nullptr;
  int64_t used = 0;
  explicit Scratch(cudaStream_t stream) : s(stream) {}
  ~Scratch() {
    if (base) cudaFreeAsync(base, s);
  }
  // Offsets are given out first, then one block is allocated.
  int64_t take(int64_t bytes) {
    const int64_t at = used;
    used += up(bytes, 256);
    return at;
  }
  int allocate(const Tables *T) {
    H24_CUDA_TRY(cudaMallocFromPoolAsync(reinterpret_cast<void **>(&base), static_cast<size_t>(used > 0 ? used : 256),
                                         T->pool, s));
    return H24_OK;
  }
  template <typename P>
  P *at(int64_t offset) const {
    return reinterpret_cast<P *>(base + offset);
  }
};

template <auto kernel>
int launch_gemm(GemmArgs a, int64_t tiles, cudaStream_t s) {
  H24_CUDA_TRY(allow_smem<kernel>(kSmem));
  // Where all tiles have few tokens, B is small and the ring has more stages.
  a.stage_a = kOperand;
  a.stage_b = 0;
  for (int i = 0; i < a.jobs; ++i) {
    const int need = a.job[i].swap ? a.job[i].bn / 2 * 2 * kTileK : kOperand;
    a.stage_b = need > a.stage_b ? need : a.stage_b;
  }
  a.stages = kRing / (a.stage_a + a.stage_b);
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < 1 ? 1 : tiles < kPairs ? tiles : kPairs)));
  cfg.blockDim = dim3(kThreads);
  // All of the SM's shared memory: the pair takes all TMEM columns, so nothing
  // that waits for columns may be resident beside it.
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = 2;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  H24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a));
  count_launches(1);
  return H24_OK;
}

// Columns of the logits' tiles: 256, fewer where that leaves pairs of SMs without one.
int logits_bn(int64_t tokens, int64_t vocab) {
  int bn = kTileN;
  while (bn > 64 && cdiv(tokens, kTileM) * cdiv(vocab, bn) < kPairs) bn /= 2;
  return bn;
}

// Up to 128 tokens are the columns of the tiles of logits and of dx, not their
// rows: 256 rows of which few are there would cost more of the tensor cores than
// the weights' bytes cost of HBM (one token and [50688,1920]: 44 us, 38 so).
bool few_tokens(int64_t tokens) { return tokens <= 128; }

// Rows of a block of the row kernels: the blocks fill the GPU four times at most.
int rows_per_block(int64_t tokens) {
  const int64_t per = cdiv(tokens, 592);
  return static_cast<int>(per > kRowThreads ? kRowThreads : per);
}

bool rows_on_16(const void *p, int64_t pitch, int64_t cols) { return aligned16(p) && pitch % 8 == 0 && cols % 8 == 0; }

// W as TMA can read it: itself, or a copy with rows on 16 bytes.
int readable_head(const CeArgs &c, const Scratch &sc, int64_t copy_at, const void **w, int64_t *pitch) {
  *w = c.w;
  *pitch = c.w_stride;
  if (copy_at < 0) return H24_OK;
  *w = sc.at<void>(copy_at);
  *pitch = up(c.in, 8);
  H24_CUDA_TRY(launch_pdl(ce_copy_head_kernel, dim3(wave_grid(cdiv(c.vocab, kRowThreads / 32), 8)), dim3(kRowThreads),
                          sc.s, static_cast<const uint16_t *>(c.w), c.w_stride, c.vocab, static_cast<int>(c.in),
                          sc.at<uint16_t>(copy_at), *pitch));
  count_launches(1);
  return H24_OK;
}
bool head_readable(const CeArgs &c) { return aligned16(c.w) && c.w_stride % 8 == 0 && c.w_stride >= c.in; }

}  // namespace

int launch_ce_forward(const Tables *T, const CeArgs &c, const int64_t *labels, int64_t ignore, float *loss,
                      int32_t *state, cudaStream_t s) {
  const bool bf16 = c.dtype == H24_DTYPE_BF16;
  const bool swap = few_tokens(c.tokens);
  const int bn = swap ? static_cast<int>(up(c.tokens, 32)) : logits_bn(c.tokens, c.vocab);
  // Tiles, and the parts of a token's sum that they leave: one for each half of a
  // tile's columns, or for each warp of the grid that has its tokens.
  const int64_t n_tiles = cdiv(c.vocab, swap ? kTileM : bn), m_tiles = swap ? 1 : cdiv(c.tokens, kTileM);
  const int64_t n_parts = swap ? 8 * (n_tiles < kPairs ? n_tiles : kPairs) : 2 * n_tiles;
  const int64_t pitch = up(c.in, 8), part_pitch = up(c.tokens, kCombineRows);
  Scratch sc(s);
  const int64_t rows_at = sc.take((c.tokens + kTileK) * pitch * 2), token_at = sc.take(c.tokens * 4);
  const int64_t target_at = sc.take(c.tokens * 4);
  const int64_t zt_at = sc.take(c.tokens * 4), loss_at = sc.take(c.tokens * 4), ticket_at = sc.take(4);
  const int64_t parts_at = sc.take(n_parts * part_pitch * 8);
  const int64_t w_at = head_readable(c) ? -1 : sc.take(c.vocab * pitch * 2);
  const int per_block = rows_per_block(c.tokens);
  const int64_t row_blocks = cdiv(c.tokens, per_block);
  const int64_t counts_at = c.tokens > kGroupedTokens ? sc.take(row_blocks * 4) : -1;
  int rc = sc.allocate(T);
  if (rc != H24_OK) return rc;
  const State st = state_at(state, c.tokens);
  // Few tokens whose rows TMA can read are multiplied as they lie, the ignored
  // ones among them (they cost nothing more, and a column is a token's own); their
  // places are counted with the loss.  That spares a kernel of three.
  const bool own = swap && aligned16(c.x) && c.x_stride % 8 == 0 && c.x_stride >= c.in;
  RowsArgs r{};
  r.x = {static_cast<const uint16_t *>(c.x), c.x_stride, static_cast<int>(c.tokens), static_cast<int>(c.in),
         rows_on_16(c.x, c.x_stride, c.in)};
  r.labels = labels;
  r.ignore = ignore;
  r.vocab = static_cast<int>(c.vocab);
  r.st = st;
  r.token = sc.at<int>(token_at);
  r.target = sc.at<int>(target_at);
  r.rows = sc.at<uint16_t>(rows_at);
  r.pitch = pitch;
  r.loss = c.reduction == H24_REDUCE_NONE ? loss : nullptr;
  r.ticket = sc.at<unsigned>(ticket_at);
  r.per_block = per_block;
  if (counts_at >= 0) {
    GroupArgs q{};
    q.labels = labels;
    q.ignore = ignore;
    q.tokens = c.tokens;
    q.per_block = per_block;
    q.counts = sc.at<int>(counts_at);
    r.counts = q.counts;
    H24_CUDA_TRY(launch_pdl(ce_groups_kernel, dim3(static_cast<unsigned>(row_blocks)), dim3(kRowThreads), s, q));
    count_launches(1);
  }
  if (!own) {
    H24_CUDA_TRY(launch_pdl(ce_rows_kernel, dim3(static_cast<unsigned>(row_blocks)), dim3(kRowThreads), s, r));
    count_launches(1);
  }
  const void *w;
  int64_t w_pitch;
  if ((rc = readable_head(c, sc, w_at, &w, &w_pitch)) != H24_OK) return rc;

  GemmArgs g{};
  // A and B: the tokens' states and the head, or the other way round.
  if (!map16(&g.map[swap], own ? c.x : r.rows, c.tokens, c.in, own ? c.x_stride : pitch, swap ? bn / 2 : kTileM / 2) ||
      !map16(&g.map[!swap], w, c.vocab, c.in, w_pitch, swap ? kTileM / 2 : bn / 2))
    return fail(H24_ERR_CUDA, "linear_ce_forward: cuTensorMapEncodeTiled failed");
  g.jobs = 1;
  g.job[0].kind = kLoss;
  g.job[0].swap = swap;
  g.job[0].n_total = swap ? bn : static_cast<int>(c.vocab);
  g.job[0].m_total = static_cast<int>(c.vocab);
  g.job[0].bn = bn;
  g.job[0].k_total = static_cast<int>(c.in);
  g.job[0].split = 1;
  g.vocab = static_cast<int>(c.vocab);
  g.kept = own ? nullptr : st.kept;
  g.tokens = static_cast<int>(c.tokens);
  g.labels = own ? labels : nullptr;
  g.ticket = own ? r.ticket : nullptr;
  g.target = r.target;
  g.z_target = sc.at<float>(zt_at);
  g.parts = sc.at<float2>(parts_at);
  g.part_pitch = part_pitch;
  g.err = T->err;
  const int64_t tiles = m_tiles * n_tiles;
  if (swap)
    rc = bf16 ? launch_gemm<ce_gemm_kernel<true, true, true, kLogits>>(g, tiles, s)
              : launch_gemm<ce_gemm_kernel<false, true, true, kLogits>>(g, tiles, s);
  else
    rc = bf16 ? launch_gemm<ce_gemm_kernel<true, true, false, kLogits>>(g, tiles, s)
              : launch_gemm<ce_gemm_kernel<false, true, false, kLogits>>(g, tiles, s);
  if (rc != H24_OK) return rc;

  CombineArgs cb{};
  cb.st = st;
  cb.parts = g.parts;
  cb.part_pitch = part_pitch;
  cb.n_parts = static_cast<int>(n_parts);
  cb.z_target = g.z_target;
  cb.token = r.token;
  cb.target = r.target;
  cb.row_loss = sc.at<float>(loss_at);
  cb.loss = loss;
  cb.reduction = c.reduction;
  cb.ticket = r.ticket;
  cb.labels = own ? labels : nullptr;
  cb.ignore = ignore;
  cb.tokens = static_cast<int>(c.tokens);
  cb.vocab = static_cast<int>(c.vocab);
  if (swap)
    H24_CUDA_TRY(launch_pdl(ce_combine_kernel<1>, dim3(static_cast<unsigned>(c.tokens)), dim3(kRowThreads), s, cb));
  else
    H24_CUDA_TRY(launch_pdl(ce_combine_kernel<kCombineRows>, dim3(static_cast<unsigned>(cdiv(c.tokens, kCombineRows))),
                            dim3(kRowThreads), s, cb));
  count_launches(1);
  return H24_OK;
}

namespace {

// How the backward pass cuts its work.
struct BackPlan {
  int64_t piece;   // vocabulary rows of a piece, a multiple of 256
  int64_t pieces;
  int split;       // slices of a dx tile's sum
};
BackPlan back_plan(const CeArgs &c, bool want_states, bool want_head) {
  BackPlan p;
  const int64_t rows = up(c.tokens, kTileM);
  const int64_t most = kPieceBytes / (rows * 2) / kTileN * kTileN;
  p.pieces = cdiv(c.vocab, most < kPieceCols ? kPieceCols : most);
  p.piece = up(cdiv(c.vocab, p.pieces), kTileN);
  p.pieces = cdiv(c.vocab, p.piece);
  // A dx tile sums over a whole piece.  Slices of it where that is more than a
  // third of what a pair of SMs does in a launch.
  const int64_t kb = cdiv(p.pieces > 1 ? p.piece : c.vocab, kTileK), m_tiles = rows / kTileM, n_tiles = cdiv(c.in, kTileN);  // (few tokens: the same count)
  int64_t work = m_tiles * n_tiles * kb;
  if (want_head) work += cdiv(p.piece, kTileM) * n_tiles * cdiv(c.tokens, kTileK);
  if (p.pieces > 1) work += m_tiles * cdiv(p.piece, kTileN) * cdiv(c.in, kTileK);
  int64_t split = want_states ? cdiv(3 * kb * kPairs, work) : 1;
  const int64_t least = want_states ? cdiv(kb, c.dtype == H24_DTYPE_BF16 ? kSumBf16 : kSumHalf) : 1;  // (12 at most)
  if (split < least) split = least;
  if (split > kb) split = kb;
  if (split > 32) split = 32;
  p.split = static_cast<int>(split);
  return p;
}

}  // namespace

int launch_ce_backward(const Tables *T, const CeArgs &c, const float *dloss, int64_t dloss_stride, const int32_t *state,
                       void *dx, void *dw, cudaStream_t s) {
  const bool bf16 = c.dtype == H24_DTYPE_BF16, each = c.reduction == H24_REDUCE_NONE;
  const BackPlan plan = back_plan(c, dx != nullptr, dw != nullptr);
  const int64_t pitch = up(c.in, 8), rows = up(c.tokens, kTileM), acc_pitch = up(c.in, 32);
  Scratch sc(s);
  const int64_t rows_at = sc.take((c.tokens + kTileK) * pitch * 2);
  const int64_t scaled_at = each && dw ? sc.take((c.tokens + kTileK) * pitch * 2) : -1;
  const int64_t token_at = sc.take((each ? 5 : 3) * c.tokens * 4);  // words of each token
  const int per_block = rows_per_block(c.tokens);
  const int64_t row_blocks = cdiv(c.tokens, per_block);
  const bool sizes = scaled_at >= 0 && !bf16;
  const int64_t groups_at = c.tokens > kGroupedTokens || sizes ? sc.take(2 * row_blocks * 4) : -1;
  const int64_t scale_at = sc.take(8), counters_at = sc.take((plan.pieces + 1) * 4);
  const int64_t w_at = head_readable(c) ? -1 : sc.take(c.vocab * pitch * 2);
  const int64_t acc_at = dx ? sc.take(plan.split * c.tokens * acc_pitch * 4) : -1;
  const int64_t d_pitch = plan.piece, d_bytes = rows * d_pitch * 2;
  const int64_t d_at = sc.take(d_bytes), d2_at = plan.pieces > 1 ? sc.take(d_bytes) : d_at;
  int rc = sc.allocate(T);
  if (rc != H24_OK) return rc;
  const State st = state_at(state, c.tokens);

  BackRowsArgs r{};
  r.x = {static_cast<const uint16_t *>(c.x), c.x_stride, static_cast<int>(c.tokens), static_cast<int>(c.in),
         rows_on_16(c.x, c.x_stride, c.in)};
  r.st = st;
  r.rows = sc.at<uint16_t>(rows_at);
  r.scaled = scaled_at < 0 ? nullptr : sc.at<uint16_t>(scaled_at);
  r.place = sc.at<int>(token_at);
  r.target = r.place + c.tokens;
  r.own = sc.at<float>(token_at) + 2 * c.tokens;
  r.log_factor = each ? r.own + c.tokens : nullptr;
  r.power = each ? r.own + 2 * c.tokens : nullptr;
  r.pitch = pitch;
  r.dloss = dloss;
  r.dloss_stride = dloss_stride;
  r.mean = c.reduction == H24_REDUCE_MEAN;
  r.scale = sc.at<float>(scale_at);
  r.counters = sc.at<int>(counters_at);
  r.n_counters = static_cast<int>(plan.pieces + 1);
  r.per_block = per_block;
  if (groups_at >= 0) {
    GroupArgs q{};
    q.target = st.target;
    q.dloss = scaled_at >= 0 ? dloss : nullptr;
    if (sizes) q.x = r.x;
    q.dloss_stride = dloss_stride;
    q.tokens = c.tokens;
    q.per_block = per_block;
    q.counts = sc.at<int>(groups_at);
    q.tops = q.counts + row_blocks;
    r.counts = q.counts;
    r.tops = q.tops;
    H24_CUDA_TRY(launch_pdl(ce_groups_kernel, dim3(static_cast<unsigned>(row_blocks)), dim3(kRowThreads), s, q));
    count_launches(1);
  }
  H24_CUDA_TRY(launch_pdl(bf16 ? ce_back_rows_kernel<true> : ce_back_rows_kernel<false>,
                          dim3(static_cast<unsigned>(row_blocks)), dim3(kRowThreads), s, r));
  count_launches(1);
  const void *w;
  int64_t w_pitch;
  if ((rc = readable_head(c, sc, w_at, &w, &w_pitch)) != H24_OK) return rc;

  GemmArgs base{};
  base.vocab = static_cast<int>(c.vocab);
  base.kept = st.kept;
  base.target = r.target;
  base.lse = st.lse;
  base.own = r.own;
  base.scale = r.scale;
  base.prob_log2 = bf16 ? 0.f : 15.f;
  base.log_factor = r.log_factor;
  base.row_bytes = c.in % 16 == 0 && (reinterpret_cast<uintptr_t>(dw) & 31) == 0 ? 32 : c.in % 8 == 0 && aligned16(dw) ? 16 : 2;
  base.err = T->err;
  const int64_t rows_alloc = c.tokens + kTileK;
  const uint16_t *head_rows = r.scaled ? r.scaled : r.rows;
  const int bn_in = static_cast<int>(c.in >= kTileN ? kTileN : up(c.in, 32));
  const bool swap = few_tokens(c.tokens), long_k = cdiv(c.in, kTileK) > (bf16 ? kBackBf16 : kBackHalf);
  const bool long_tokens = dw && cdiv(c.tokens, kTileK) > (bf16 ? kSumBf16 : kSumHalf);
  const int bn_few = static_cast<int>(up(c.tokens, 32));
  const int64_t d_rows = swap ? bn_few : rows;  // rows of d that are written
  for (int64_t i = 0; i <= plan.pieces; ++i) {
    // The gradients of piece i - 1 beside the logits of piece i.
    GemmArgs g = base;
    g.next_tile = r.counters + i;
    bool ok = true;
    int64_t tiles = 0;
    int64_t longest = 0;
    if (i > 0) {
      const int64_t v0 = (i - 1) * plan.piece, v = c.vocab - v0 < plan.piece ? c.vocab - v0 : plan.piece;
      uint16_t *d = sc.at<uint16_t>(i & 1 ? d_at : d2_at);
      auto add_states = [&] {
        if (!dx) return;
        Job &j = g.job[g.jobs];
        j.kind = kStates;
        j.swap = swap;
        j.n_total = swap ? bn_few : static_cast<int>(c.in);
        j.m_total = static_cast<int>(c.in);
        j.bn = swap ? bn_few : bn_in;
        j.k_total = static_cast<int>(v);
        // (Each slice has a k block; a shorter last piece adds to fewer of them.)
        j.split = static_cast<int>(cdiv(v, kTileK) < plan.split ? cdiv(v, kTileK) : plan.split);
        j.v0 = static_cast<int>(v0);
        j.add = i > 1;
        j.out = sc.at<float>(acc_at);
        j.pitch = acc_pitch;
        j.plane = c.tokens * acc_pitch;
        ok = ok && map16(&g.map[2 * g.jobs + swap], d, d_rows, plan.piece, d_pitch, swap ? bn_few / 2 : kTileM / 2) &&
             map16(&g.map[2 * g.jobs + !swap], w, c.vocab, c.in, w_pitch, kTileK);
        tiles += rows / kTileM * cdiv(c.in, bn_in) * plan.split;
        ++g.jobs;
      };
      auto add_head = [&] {
        if (!dw) return;
        Job &j = g.job[g.jobs];
        j.kind = kHeadRows;
        j.n_total = static_cast<int>(c.in);
        j.bn = bn_in;
        j.m_total = static_cast<int>(v);
        j.split = 1;
        j.v0 = static_cast<int>(v0);
        j.out = dw;
        j.pitch = c.in;
        ok = ok && map16(&g.map[2 * g.jobs], d, d_rows, plan.piece, d_pitch, kTileK) &&
             map16(&g.map[2 * g.jobs + 1], head_rows, rows_alloc, c.in, pitch, kTileK);
        tiles += cdiv(v, kTileM) * cdiv(c.in, bn_in);
        ++g.jobs;
      };
      longest = cdiv(c.tokens, kTileK);
      if (longest > cdiv(v, kTileK) / plan.split) {
        add_head();
        add_states();
      } else {
        add_states();
        add_head();
      }
    }
    if (i < plan.pieces) {
      const int64_t v0 = i * plan.piece, v = c.vocab - v0 < plan.piece ? c.vocab - v0 : plan.piece;
      Job &j = g.job[g.jobs];
      j.kind = kProb;
      j.swap = swap;
      j.n_total = swap ? bn_few : static_cast<int>(up(v, kTileK));
      j.m_total = static_cast<int>(v);
      j.bn = swap ? bn_few : plan.pieces > 1 ? kTileN : logits_bn(c.tokens, c.vocab);
      j.k_total = static_cast<int>(c.in);
      j.split = 1;
      j.v0 = static_cast<int>(v0);
      j.out = sc.at<uint16_t>(i & 1 ? d2_at : d_at);
      j.pitch = d_pitch;
      ok = ok && map16(&g.map[2 * g.jobs + swap], r.rows, c.tokens, c.in, pitch, swap ? bn_few / 2 : kTileM / 2) &&
           map16(&g.map[2 * g.jobs + !swap], w, c.vocab, c.in, w_pitch, swap ? kTileM / 2 : j.bn / 2);
      tiles += swap ? cdiv(v, kTileM) : rows / kTileM * cdiv(j.n_total, j.bn);
      ++g.jobs;
    }
    if (!ok) return fail(H24_ERR_CUDA, "linear_ce_backward: cuTensorMapEncodeTiled failed");
    auto launch = [&](auto few, auto several) {
      constexpr bool kFew = decltype(few)::value;
      constexpr Long kLong = decltype(several)::value;
      return bf16 ? launch_gemm<ce_gemm_kernel<true, false, kFew, kLong>>(g, tiles, s)
                  : launch_gemm<ce_gemm_kernel<false, false, kFew, kLong>>(g, tiles, s);
    };
    constexpr std::integral_constant<Long, kNone> none;
    constexpr std::integral_constant<Long, kLogits> logits;
    constexpr std::integral_constant<Long, kTokens> both;
    rc = swap          ? (long_k ? launch(std::true_type(), logits) : launch(std::true_type(), none))
         : long_tokens ? launch(std::false_type(), both)
         : long_k      ? launch(std::false_type(), logits)
                       : launch(std::false_type(), none);
    if (rc != H24_OK) return rc;
  }
  if (dx) {
    StatesArgs o{};
    o.place = r.place;
    o.acc = sc.at<float>(acc_at);
    o.pitch = acc_pitch;
    o.plane = c.tokens * acc_pitch;
    o.slices = plan.split;
    o.tokens = c.tokens;
    o.in = static_cast<int>(c.in);
    o.scale = r.scale;
    o.power = r.power;
    o.out = static_cast<uint16_t *>(dx);
    o.vec = rows_on_16(dx, c.in, c.in);
    const int64_t blocks = cdiv(c.tokens * cdiv(c.in, 8), kRowThreads);
    H24_CUDA_TRY(launch_pdl(bf16 ? ce_states_kernel<true> : ce_states_kernel<false>, dim3(wave_grid(blocks, 8)),
                            dim3(kRowThreads), s, o));
    count_launches(1);
  }
  return H24_OK;
}

}  // namespace h24
