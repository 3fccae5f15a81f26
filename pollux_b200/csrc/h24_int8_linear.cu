// h24_int8_linear.cu -- product of int8 activations with an INT8 layer:
//   y[t][o] = (sum_k q[t][k] * W[o][k]) * scale[t] * fp16(mu16[o] / 127) + bias[o]
// The sum is exact in int32 (in_features is bounded so that it cannot
// overflow), the scaling is fp32 and y is rounded once.  The weight's scale
// is the one PackedInt8Linear.materialize uses (pollux.py:545-554).
//
// The weights are the M operand (128 output features a tile, one TMEM lane
// each) and the tokens the N operand, so one token costs 16 columns of a tile
// and not 128 rows, and a warp's 32 lanes store 32 neighbouring outputs.
//
// Three kernels, chosen by make_plan from an estimate of bytes and latency:
//   one or two tokens (four, where the layer is small): dp4a over the weight
//     rows, bound by their bytes
//     ([1,1920] x [50688,1920] 15.0-16.1 us: 0.93-0.99 of the measured HBM rate);
//   a few to a few hundred: tiles of 128 x n, the k split over a cluster where
//     tiles are few; bound by a launch's chain of latencies (5.4 us for [32,1920]
//     x [7680,1920], 2.3 of them bytes) and by the fill of shared memory;
//   many: pairs of SMs on 256 x n tiles, bound by L2: at 2.6-2.7 PTOP/s the pairs
//     fetch 10-11 TB/s through it, what it gave in every run ([4096,1920] x
//     [7680,1920] bf16 46.8 us, [1024,1920] x [50688,1920] fp32 88.7).
#include "h24_tile.cuh"

namespace h24 {
namespace {

// Rows of a byte matrix at any pitch and alignment, copied to rows of `pitch`
// bytes (a multiple of 16), zeros past their end: what TMA can read.  Where a
// layer or its input is not 16-byte aligned, the copy and the tiles over it
// (2 more bytes of traffic a byte) take [4096,1919] x [7680,1919] from 1,106 us
// with tiles filled by hand to 57, and [20,1921] x [7680,1921] from 61 to 14.
struct RepackArgs {
  const int8_t *src;
  int64_t stride;
  int8_t *dst;
  int64_t rows;
};
constexpr int kRepackThreads = 256;
__global__ void __launch_bounds__(kRepackThreads) repack_rows_kernel(const RepackArgs a0, const RepackArgs a1, int cols,
                                                                     int chunks) {
  pdl_enter();
  const int64_t total0 = a0.rows * chunks, total = total0 + a1.rows * chunks;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kRepackThreads) + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * kRepackThreads) {
    const RepackArgs &a = i < total0 ? a0 : a1;
    const int64_t at = i < total0 ? i : i - total0;
    const int64_t r = at <= 0xFFFFFFFFll ? static_cast<uint32_t>(at) / static_cast<uint32_t>(chunks) : at / chunks;
    const int c = static_cast<int>(at - r * chunks) * 16;
    const int8_t *hi = a.src + (a.rows - 1) * a.stride + cols;
    reinterpret_cast<uint4 *>(a.dst)[at] = load16_any(a.src + r * a.stride + c, cols - c, a.src, hi);
  }
}

constexpr int kM = 128;        // output features per tile
constexpr int kKB = 128;       // k per stage: one 128-byte swizzle row
constexpr int kABytes = kM * kKB;
constexpr int kMaxStages = 12;
constexpr int kHeadBytes = 1024;  // barriers, TMEM address, abort flag; the stages start on 1 KB

struct LinArgs {
  const int8_t *q;
  const float *scale;
  const int8_t *w;
  const uint16_t *mu16;
  const float *bias;
  void *y;
  int *err;
  int64_t q_stride;
  int tokens, out, in;
  int n;          // tokens per tile, a multiple of 16, at most 256
  int tok_tiles;  // token tiles
  int split;      // CTAs of a cluster that share a tile's k
  int stages;
  int tmem_cols;
  bool y_vec;     // y is 16-byte aligned
};

struct LinHead {
  uint64_t full[kMaxStages], empty[kMaxStages], done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(LinHead) <= kHeadBytes, "head");

// Instruction descriptor: kind::i8, D = s32, A = B = s8, both K-major.
__host__ __device__ constexpr uint32_t i8_idesc(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// A whole converged warp executes these; one elected lane issues.
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// The layer's reconstruction scale of one output row.
__device__ __forceinline__ float weight_scale(const uint16_t *mu16, int64_t o) {
  return __half2float(__float2half_rn(__fdiv_rn(__half2float(__ushort_as_half(__ldg(mu16 + o))), 127.0f)));
}

// One output: every path rounds the same way.
__device__ __forceinline__ float finish(int acc, float scale, float ws, float b) {
  return fmaf(__fmul_rn(__int2float_rn(acc), scale), ws, b);
}
__device__ __forceinline__ void put(float *y, float v) { *y = v; }
__device__ __forceinline__ void put(__half *y, float v) { *y = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16 *y, float v) { *y = __float2bfloat16_rn(v); }

// Four neighbouring outputs in one store.
__device__ __forceinline__ void put4(float *y, const float (&v)[4]) {
  *reinterpret_cast<float4 *>(y) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename Half>
__device__ __forceinline__ void put4(Half *y, const float (&v)[4]) {
  alignas(8) Half h[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) put(h + j, v[j]);
  *reinterpret_cast<uint2 *>(y) = *reinterpret_cast<const uint2 *>(h);
}

// 32 columns of this warp's lanes to the outputs of `left` (at least 1) tokens
// at `col` (of the first feature of the warp; the same for all lanes), lane
// l's feature at col + l.  Lane j holds token j's scale, loaded before: a load
// inside each column's test put its latency between every two stores (11.5 us
// a 256 x 256 tile).
template <typename Out>
__device__ __forceinline__ void store32(const int (&r)[32], float scales, int left, float ws, float b, Out *col,
                                        int64_t pitch, uint32_t lane, bool live) {
  if (left >= 32) {
#pragma unroll
    for (int j = 0; j < 32; ++j, col += pitch) {
      const float v = finish(r[j], __shfl_sync(0xffffffffu, scales, j), ws, b);
      if (live) put(col + lane, v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j, col += pitch) {
      const float v = finish(r[j], __shfl_sync(0xffffffffu, scales, j), ws, b);
      if (live && j < left) put(col + lane, v);
    }
  }
}

// A CTA's share of the sum of a cluster's partial tiles: every split-th token,
// a token a warp and step, four features a lane; the remote loads of two steps
// are in flight together (their latency, not their bytes, is what this costs).
template <typename Out>
__device__ __forceinline__ void reduce_tile(const LinArgs &a, const uint8_t *part, int rank, int o0, int t0, int warp,
                                            int lane) {
  constexpr int kWarps = 6, kSteps = 2;
  const int64_t o = static_cast<int64_t>(o0) + 4 * lane;
  float ws[4], b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    ws[j] = o + j < a.out ? weight_scale(a.mu16, o + j) : 0.f;
    b[j] = o + j < a.out && a.bias ? __ldg(a.bias + o + j) : 0.f;
  }
  const bool whole = a.y_vec && a.out % 4 == 0 && o + 4 <= a.out;
  const uint32_t mine = su32(part) + static_cast<uint32_t>(lane) * 16;
  const int n_live = min(a.n, a.tokens - t0);
  for (int c0 = rank + warp * a.split; c0 < n_live; c0 += kWarps * kSteps * a.split) {
    int4 v[kSteps][8];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int c = min(c0 + u * kWarps * a.split, n_live - 1);
#pragma unroll
      for (int p = 0; p < 8; ++p) {
        if (p >= a.split) break;
        uint32_t addr;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(mine + c * kM * 4), "r"(p));
        asm volatile("ld.shared::cluster.v4.s32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[u][p].x), "=r"(v[u][p].y), "=r"(v[u][p].z), "=r"(v[u][p].w)
                     : "r"(addr)
                     : "memory");
      }
    }
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
      const int c = c0 + u * kWarps * a.split;
      if (c >= n_live) break;
      int4 acc = v[u][0];
#pragma unroll
      for (int p = 1; p < 8; ++p) {
        if (p >= a.split) break;
        acc.x += v[u][p].x;
        acc.y += v[u][p].y;
        acc.z += v[u][p].z;
        acc.w += v[u][p].w;
      }
      const float sc = __ldg(a.scale + t0 + c);
      const float f[4] = {finish(acc.x, sc, ws[0], b[0]), finish(acc.y, sc, ws[1], b[1]),
                          finish(acc.z, sc, ws[2], b[2]), finish(acc.w, sc, ws[3], b[3])};
      Out *y = static_cast<Out *>(a.y) + (static_cast<int64_t>(t0) + c) * a.out + o;
      if (whole) {
        put4(y, f);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (o + j < a.out) put(y + j, f[j]);
      }
    }
  }
}

constexpr int kSplitThreads = 192;  // warp 0 loads, warp 1 issues MMAs, warps 2-5 read TMEM

// One CTA per 128 x n tile and k slice.  The `split` CTAs of a cluster take a
// slice of the tile's k each; their int32 partial tiles meet in distributed
// shared memory, where CTA r finishes every split-th part of the tokens (the
// sum is an integer, so the order does not matter).
template <typename Out>
__global__ void __launch_bounds__(kSplitThreads) int8_linear_split_kernel(const __grid_constant__ CUtensorMap wmap,
                                                                          const __grid_constant__ CUtensorMap qmap,
                                                                          const __grid_constant__ LinArgs a) {
  extern __shared__ uint8_t lin_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(lin_raw) + 1023) & ~uintptr_t(1023));
  LinHead &H = *reinterpret_cast<LinHead *>(smem);
  uint8_t *stages = smem + kHeadBytes;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int rank = static_cast<int>(blockIdx.x) % a.split, tile = static_cast<int>(blockIdx.x) / a.split;
  const int o0 = tile / a.tok_tiles * kM, t0 = tile % a.tok_tiles * a.n;
  const int kblocks = (a.in + kKB - 1) / kKB;
  const int kb0 = static_cast<int>(static_cast<int64_t>(kblocks) * rank / a.split);
  const int nkb = static_cast<int>(static_cast<int64_t>(kblocks) * (rank + 1) / a.split) - kb0;
  const int stage_bytes = kABytes + a.n * kKB;
  volatile int *abort = &H.abort;

  if (t == 0) {
    for (int s = 0; s < a.stages; ++s) {
      bar_init(&H.full[s], 1);
      bar_init(&H.empty[s], 1);
    }
    bar_init(&H.done, 1);
    H.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (a.in > 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(&wmap) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
    }
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(su32(&H.tmem)),
                 "r"(a.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = H.tmem;
  pdl_enter();

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      int issued = 0;
      for (; issued < nkb; ++issued) {
        if (!bar_wait(&H.empty[s], ph ^ 1, abort, a.err)) break;
        uint8_t *st = stages + static_cast<size_t>(s) * stage_bytes;
        bar_expect(&H.full[s], stage_bytes);
        tma_load(&wmap, st, &H.full[s], (kb0 + issued) * kKB, o0);
        tma_load(&qmap, st + kABytes, &H.full[s], (kb0 + issued) * kKB, t0);
        if (++s == a.stages) s = 0, ph ^= 1;
      }
      if (*abort)  // let the copies in flight land before the CTA leaves
        for (int i = issued > a.stages ? issued - a.stages : 0; i < issued; ++i)
          bar_wait(&H.full[i % a.stages], (i / a.stages) & 1, abort, a.err, false);
    }
  } else if (warp == 1) {
    int s = 0;
    uint32_t ph = 0;
    const uint32_t idesc = i8_idesc(kM, a.n);
    for (int i = 0; i < nkb; ++i) {
      if (!__all_sync(0xffffffffu, bar_wait(&H.full[s], ph, abort, a.err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t st = su32(stages) + static_cast<uint32_t>(s * stage_bytes);
      const uint64_t ad = tile_desc(st), bd = tile_desc(st + kABytes);
#pragma unroll
      for (int k = 0; k < kKB / 32; ++k) mma_i8(tmem, ad + 2 * k, bd + 2 * k, idesc, i > 0 || k > 0);
      mma_commit(&H.empty[s]);
      if (++s == a.stages) s = 0, ph ^= 1;
    }
    mma_commit(&H.done);
  } else {
    // The warp's number from lane 0: the compiler then keeps what follows from
    // it, the column addresses above all, in uniform registers.
    const int quarter = __shfl_sync(0xffffffffu, warp, 0) & 3, row = quarter * 32 + lane;  // TMEM lanes
    const int64_t o = static_cast<int64_t>(o0) + row;
    const bool live = o < a.out;
    const float ws = live ? weight_scale(a.mu16, o) : 0.f, b = live && a.bias ? __ldg(a.bias + o) : 0.f;
    const int n_live = min(a.n, a.tokens - t0);
    const float *scale = a.scale + t0;
    float sc = __ldg(scale + min(lane, n_live - 1));  // before the wait
    bar_wait(&H.done, 0, abort, a.err, false);
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t ta = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    if (a.split == 1) {
      // (Columns past n, up to the 32 of a chunk, are allocated and not stored.)
      Out *col = static_cast<Out *>(a.y) + static_cast<int64_t>(t0) * a.out + o0 + quarter * 32;
      int r[32];
      for (int c = 0; c < n_live; c += 32, col += 32 * static_cast<int64_t>(a.out)) {
        __syncwarp();
        tmem_ask32(ta + c, r);
        const float next = c + 32 < n_live ? __ldg(scale + min(c + 32 + lane, n_live - 1)) : 0.f;
        tmem_wait32(r);
        if (nkb == 0) {  // in_features 0: an empty sum
#pragma unroll
          for (int j = 0; j < 32; ++j) r[j] = 0;
        }
        store32(r, sc, n_live - c, ws, b, col, a.out, lane, live && !*abort);
        sc = next;
      }
    } else {
      // The partial tile as [token][feature] over the stages (the MMAs and
      // copies that used them are complete).
      int *part = reinterpret_cast<int *>(stages);
      int r[16];
      for (int c = 0; c < n_live; c += 16) {
        __syncwarp();
        tmem_ld16(ta + c, r);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kM + row] = r[j];
      }
    }
  }
  __syncwarp();
  if (a.split > 1) {
    cluster_sync_all();
    if (!*abort) reduce_tile<Out>(a, stages, rank, o0, t0, warp, lane);
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its tile
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

// ---------------------------------------------------------------------------
// Few tokens: no tiles
// ---------------------------------------------------------------------------
constexpr int kVecThreads = 256;

// 1 to T tokens.  A warp owns R weight rows; lane l reads 16 bytes of each row
// at 512 i + 16 l and multiplies them with the tokens' bytes from shared
// memory (dp4a).  Bound by the weights' bytes; what a tile of MMAs would add
// is latency: the ring's first fill, the wait for the last MMA, the read of
// TMEM.
template <int T, int R, bool kAhead, bool kAligned, typename Out>
__global__ void __launch_bounds__(kVecThreads) int8_linear_vec_kernel(const LinArgs a) {
  constexpr int kVecChunk = 8192;  // k per pass: the tokens' rows of a pass lie in shared memory
  constexpr int U = 4;             // 16-byte loads of each row in flight
  __shared__ __align__(16) uint8_t xs[T][kVecChunk];
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int kRows = kVecThreads / 32 * R;  // of a block
  const int8_t *wend = a.w + static_cast<int64_t>(a.out) * a.in;
  // Towards L2 while the kernel before this one ends (L2 holds whatever that
  // one may still write, so the loads after it see it).
  if (kAhead) {
    const int64_t o0 = (static_cast<int64_t>(blockIdx.x) * (kVecThreads / 32) + warp) * R;
    for (int r = 0; r < R && o0 + r < a.out; ++r)
      for (int k = lane * 128; k < a.in; k += 32 * 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(a.w + (o0 + r) * a.in + k));
  }
  pdl_enter();
  bool placed = false;  // the tokens are in shared memory, all of them
  for (int64_t group = blockIdx.x; group * kRows < a.out; group += gridDim.x) {
    const int64_t o0 = (group * (kVecThreads / 32) + warp) * R;
    const int live = static_cast<int>(min(static_cast<int64_t>(R), a.out - o0));  // rows of this warp, maybe none
    // The blocks around these rows lie inside the matrix.
    const bool inner = live == R && o0 * a.in >= 16 && (o0 + R) * a.in + 32 <= static_cast<int64_t>(a.out) * a.in;
    // Lane k * R + r finishes row r, token k; what it needs is asked for first.
    const int fr = lane % R, fk = lane / R;
    const bool finishes = fr < live && fk < T && fk < a.tokens;
    const float sc = finishes ? __ldg(a.scale + fk) : 0.f, ws = finishes ? weight_scale(a.mu16, o0 + fr) : 0.f;
    const float b = finishes && a.bias ? __ldg(a.bias + o0 + fr) : 0.f;
    uint4 w[R][U], next[kAligned ? 1 : R][kAligned ? 1 : U];
    // Vectors v0 + 32 u + lane of the rows, of the kn bytes from k0.  `settle`
    // makes them from their two blocks where the rows are off the boundary.
    auto ask = [&](int k0, int kn, int v0) {
      const int vecs = (kn + 15) / 16;
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = v0 + 32 * u + lane;
          const int8_t *p = a.w + (o0 + r) * a.in + k0 + 16 * v;
          if constexpr (kAligned) {
            w[r][u] = v < vecs && r < live ? __ldcs(reinterpret_cast<const uint4 *>(p)) : make_uint4(0, 0, 0, 0);
          } else if (inner) {
            p -= 16 * max(v - (vecs - 1), 0);
            const uint4 *block = reinterpret_cast<const uint4 *>(p - offset16(p));
            w[r][u] = __ldg(block);
            next[r][u] = __ldg(block + 1);
          } else {
            w[r][u] = v < vecs && r < live ? load16_any(p, kn - 16 * v, a.w, wend) : make_uint4(0, 0, 0, 0);
          }
        }
    };
    auto settle = [&](int k0, int kn, int v0) {
      if constexpr (!kAligned) {
        if (inner) {
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int u = 0; u < U; ++u)
              w[r][u] = join16(w[r][u], next[r][u], offset16(a.w + (o0 + r) * a.in + k0),
                               kn - 16 * (v0 + 32 * u + lane));
        }
      }
    };
    int acc[R][T] = {};
    for (int k0 = 0; k0 < a.in; k0 += kVecChunk) {
      const int kn = min(kVecChunk, a.in - k0), vecs = (kn + 15) / 16;
      ask(k0, kn, 0);  // on their way while the tokens are placed
      if (!placed) {
        if (k0 || group != blockIdx.x) __syncthreads();
        const int8_t *qend = a.q + (a.tokens - 1) * a.q_stride + a.in;
        for (int i = t; i < T * vecs; i += kVecThreads) {
          const int tok = i / vecs, v = i - tok * vecs;
          uint4 x = make_uint4(0, 0, 0, 0);
          if (tok < a.tokens) {
            const int8_t *p = a.q + tok * a.q_stride + k0 + 16 * v;
            x = kAligned ? __ldg(reinterpret_cast<const uint4 *>(p)) : load16_any(p, kn - 16 * v, a.q, qend);
          }
          *reinterpret_cast<uint4 *>(&xs[tok][16 * v]) = x;
        }
        __syncthreads();
        placed = a.in <= kVecChunk;
      }
      for (int v0 = 0; v0 < vecs; v0 += 32 * U) {
        if (v0) ask(k0, kn, v0);
        settle(k0, kn, v0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int v = v0 + 32 * u + lane;
          if (v >= vecs) break;
#pragma unroll
          for (int k = 0; k < T; ++k) {
            const int4 x = *reinterpret_cast<const int4 *>(&xs[k][16 * v]);
#pragma unroll
            for (int r = 0; r < R; ++r) {
              acc[r][k] = __dp4a(static_cast<int>(w[r][u].x), x.x, acc[r][k]);
              acc[r][k] = __dp4a(static_cast<int>(w[r][u].y), x.y, acc[r][k]);
              acc[r][k] = __dp4a(static_cast<int>(w[r][u].z), x.z, acc[r][k]);
              acc[r][k] = __dp4a(static_cast<int>(w[r][u].w), x.w, acc[r][k]);
            }
          }
        }
      }
    }
    int mine = 0;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int k = 0; k < T; ++k) {
        const int sum = __reduce_add_sync(0xffffffffu, acc[r][k]);
        if (lane == k * R + r) mine = sum;
      }
    if (finishes)
      put(static_cast<Out *>(a.y) + fk * static_cast<int64_t>(a.out) + o0 + fr, finish(mine, sc, ws, b));
  }
}

template <int T, int R, bool kAhead, bool kAligned, typename Out>
int launch_vec(const LinArgs &a, cudaStream_t s) {
  const int64_t per_block = static_cast<int64_t>(kVecThreads / 32) * R;
  const int64_t groups = (a.out + per_block - 1) / per_block;
  // Off the boundary placing the tokens costs as much as eight rows: the blocks
  // of one wave place them once each.  ([1,1919] x [50688,1919]: 39 us, 49 with a
  // block for each eight rows.)
  constexpr auto kernel = int8_linear_vec_kernel<T, R, kAhead, kAligned, Out>;
  const int grid = kAligned ? static_cast<int>(groups) : wave_grid(groups, blocks_per_sm_once<kernel>(kVecThreads));
  H24_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kVecThreads), s, a));
  count_launches(1);
  return H24_OK;
}

template <int T, typename Out>
int launch_vec_rows(const LinArgs &a, bool aligned, cudaStream_t s) {
  // Off the boundary two blocks are held for each vector: one row a warp.
  if (!aligned)
    return a.out >= 148 * 8 * 8 ? launch_vec<T, 1, true, false, Out>(a, s) : launch_vec<T, 1, false, false, Out>(a, s);
  // Rows a warp, so that the warps of the layer fill the GPU; the L2 requests
  // ahead of the previous kernel's end only where the grid is many waves.
  // One token, us, 1 / 2 / 4 rows with and (without) the requests:
  // 50688 x 1920: 16.0 (17.6) / 15.0 (18.0) / 17.4 (18.1);
  // 7680 x 1920: 4.7 (4.3) / 3.8 (3.8) / 3.7 (3.5); 1920 x 7680: 5.7 (4.5) / 5.6 (5.9) / 6.4 (6.0).
  const int R = a.out >= 148 * 8 * 8 ? 2 : a.out >= 148 * 8 * 4 ? 4 : 1;
  if (R == 4) return launch_vec<T, 4, false, true, Out>(a, s);
  if (R == 2) return launch_vec<T, 2, true, true, Out>(a, s);
  return launch_vec<T, 1, false, true, Out>(a, s);
}

// ---------------------------------------------------------------------------
// Pairs: many tokens
// ---------------------------------------------------------------------------
constexpr int kPairM = 256;      // output features of a pair's tile, 128 a CTA
constexpr int kPairThreads = 320;  // warp 0 loads, warp 1 issues MMAs, warps 2-9 read TMEM
constexpr int kEpiWarps = 8;

struct PairHead {
  uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2], drain;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(PairHead) <= kHeadBytes, "head");

__device__ __forceinline__ void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Persistent pairs of CTAs, one pair per two SMs.  A tile is 256 features x n
// tokens: each CTA brings its 128 weight rows and half of the tokens, and one
// MMA (M = 256, cta_group::2) multiplies both, so a byte of shared memory is
// read for twice the products of a CTA on its own.  The accumulators of two
// tiles alternate in TMEM: the MMAs of one run while eight warps of each CTA
// scale and store the other.
template <typename Out>
__global__ void __launch_bounds__(kPairThreads, 1) int8_linear_pair_kernel(const __grid_constant__ CUtensorMap wmap,
                                                                           const __grid_constant__ CUtensorMap qmap,
                                                                           const __grid_constant__ LinArgs a) {
  extern __shared__ uint8_t lin_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(lin_raw) + 1023) & ~uintptr_t(1023));
  PairHead &H = *reinterpret_cast<PairHead *>(smem);
  uint8_t *stages = smem + kHeadBytes;
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int rank = static_cast<int>(blockIdx.x) & 1;
  const int kblocks = (a.in + kKB - 1) / kKB;
  const int half = a.n / 2, stage_bytes = kABytes + half * kKB;
  const int tiles = (a.out + kPairM - 1) / kPairM * a.tok_tiles;
  const int first = static_cast<int>(blockIdx.x) >> 1, step = static_cast<int>(gridDim.x) >> 1;
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
    bar_init(&H.drain, 1);
    H.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&wmap) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&qmap) : "memory");
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

  if (warp == 0) {
    if (lane == 0) {
      int s = 0;
      uint32_t ph = 0;
      for (int tile = first; tile < tiles; tile += step) {
        const int o = tile / a.tok_tiles * kPairM + rank * kM, tok = tile % a.tok_tiles * a.n + rank * half;
        for (int i = 0; i < kblocks; ++i) {
          if (!bar_wait(&H.empty[s], ph ^ 1, abort, a.err)) goto loaded;
          uint8_t *st = stages + static_cast<size_t>(s) * stage_bytes;
          // The first CTA's barrier counts the bytes of both; its phase cannot
          // end before its own arrival here.
          const uint32_t bar = cluster_addr(&H.full[s], 0);
          if (rank == 0) bar_expect(&H.full[s], 2 * stage_bytes);
          tma_load_pair(&wmap, st, bar, i * kKB, o);
          tma_load_pair(&qmap, st + kABytes, bar, i * kKB, tok);
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
      const uint32_t idesc = i8_idesc(kPairM, a.n);
      bool ok = true;
      for (int tile = first; ok && tile < tiles; tile += step) {
        ok = __all_sync(0xffffffffu, bar_wait(&H.acc_empty[acc], acc_ph ^ 1, abort, a.err));
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (int i = 0; i < kblocks; ++i) {
          ok = __all_sync(0xffffffffu, bar_wait(&H.full[s], ph, abort, a.err));
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t st = su32(stages) + static_cast<uint32_t>(s * stage_bytes);
          const uint64_t ad = tile_desc(st), bd = tile_desc(st + kABytes);
#pragma unroll
          for (int k = 0; k < kKB / 32; ++k)
            mma_i8_pair(tmem + acc * 256, ad + 2 * k, bd + 2 * k, idesc, i > 0 || k > 0);
          mma_commit_pair(&H.empty[s]);
          if (++s == a.stages) s = 0, ph ^= 1;
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
    const int mid = (half + 31) / 32 * 32;
    const int c0 = part ? mid : 0, c1 = part ? a.n : mid;
    const uint32_t ta = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    int acc = 0;
    uint32_t ph = 0;
    for (int tile = first; tile < tiles; tile += step) {
      const int64_t o0 = static_cast<int64_t>(tile / a.tok_tiles) * kPairM + rank * kM + quarter * 32, o = o0 + lane;
      const int t0 = tile % a.tok_tiles * a.n, end = min(c1, a.tokens - t0);
      const bool live = o < a.out;
      const float ws = live ? weight_scale(a.mu16, o) : 0.f, b = live && a.bias ? __ldg(a.bias + o) : 0.f;
      const float *scale = a.scale + t0;
      float s0 = c0 < end ? __ldg(scale + min(c0 + lane, end - 1)) : 0.f, s1;
      if (!__all_sync(0xffffffffu, bar_wait(&H.acc_full[acc], ph, abort, a.err))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      Out *col = static_cast<Out *>(a.y) + (static_cast<int64_t>(t0) + c0) * a.out + o0;
      const uint32_t d = ta + acc * 256;
      int r0[32], r1[32];
      if (c0 < end) tmem_ask32(d + c0, r0);
      for (int c = c0; c < end; c += 64) {  // a chunk of 32 is stored while the next one is loaded
        tmem_wait32(r0);
        if (c + 32 < end) {
          s1 = __ldg(scale + min(c + 32 + lane, end - 1));
          tmem_ask32(d + c + 32, r1);
        }
        store32(r0, s0, end - c, ws, b, col, a.out, lane, live);
        col += 32 * static_cast<int64_t>(a.out);
        if (c + 32 >= end) break;
        tmem_wait32(r1);
        if (c + 64 < end) {
          s0 = __ldg(scale + min(c + 64 + lane, end - 1));
          tmem_ask32(d + c + 64, r0);
        }
        store32(r1, s1, end - c - 32, ws, b, col, a.out, lane, live);
        col += 32 * static_cast<int64_t>(a.out);
      }
      __syncwarp();
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                         cluster_addr(&H.acc_empty[acc], 0))
                     : "memory");
      if (++acc == 2) acc = 0, ph ^= 1;
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
// Which kernel, and how it cuts the work
// ---------------------------------------------------------------------------
enum Kind { kVec, kSplit, kPair };
struct Plan {
  Kind kind;
  int n;      // tokens a tile
  int split;  // CTAs that share a tile's k
};

// Estimated microseconds of the two tiled kernels.  Both are bound by what
// their CTAs fetch through L2 (a tile's operands for each k block) or by HBM;
// measured on a B200: about 0.14 TB/s into an SM that has its pair of SMs for
// itself and 0.18 into a pair, 8 to 10 TB/s in all; 3.3 us for a launch's first
// loads, last MMAs and stores, 0.9 more for a cluster and its reduction, 4.5
// for the pairs.  (Measured against it, us: [333,7680] x [1920,7680], n 176,
// split 4: 13.5, estimated 12.9; [32,1920] x [7680,1920], n 16, split 1: 5.6,
// 5.9; [4096,1920] x [7680,1920], pairs, n 256: 47.1, 42.8.)
double split_us(int64_t tokens, int64_t out, int64_t kblocks, int n, int split, double hbm_us) {
  const double tiles = static_cast<double>((out + kM - 1) / kM * ((tokens + n - 1) / n)), ctas = tiles * split;
  // Clusters that a B200 holds at once, a CTA an SM.
  const double room = split == 8 ? 15 : split == 4 ? 36 : split == 2 ? 74 : 1e9;
  if (split > 1 && tiles > room) return 1e9;
  const double bytes = ctas * static_cast<double>((kblocks + split - 1) / split) * (kABytes + n * kKB);
  double rate = split == 1 && ctas <= 74 ? 0.14e6 * ctas : 0.18e6 * (ctas < 148 ? ctas / 2 : 74);
  if (split == 1 && ctas > 74) rate = 8e6;
  rate = rate > 8e6 ? 8e6 : rate;
  const double us = bytes / rate;
  // Beyond two CTAs an SM each waits for its own first loads and last stores
  // where the pairs go on loading.
  return 3.3 + (split > 1 ? 0.9 : 0.0) + (ctas > 296 ? 3.0 : 0.0) + (us > hbm_us ? us : hbm_us);
}
double pair_us(int64_t tokens, int64_t out, int64_t kblocks, int n, double hbm_us) {
  const double tiles = static_cast<double>((out + kPairM - 1) / kPairM * ((tokens + n - 1) / n));
  const double rounds = static_cast<double>(static_cast<int64_t>((tiles + kPairs - 1) / kPairs));
  const double us = rounds * static_cast<double>(kblocks) * (2 * kABytes + n * kKB) / 0.18e6;
  return 4.5 + (us > hbm_us ? us : hbm_us);
}

Plan make_plan(int64_t tokens, int64_t out, int64_t in, int out_size) {
  // (Whether rows lie on 16 bytes has no say here, although the copy that the
  // tiles then need costs two more bytes a byte: [3,3473] x [19944,3473] takes
  // 48 us through it, [3,1919] x [50688,1919] 68, and one token on such rows 37.
  // The limits below were measured on aligned rows.)
  // Up to four tokens without tiles; three and four only where the weights are
  // few (dp4a's work grows with the tokens): [4,1920] x [7680,1920] 4.8 us
  // against 5.5 in tiles, x [50688,1920] 22 against 18.
  if (tokens <= 2 || (tokens <= 4 && out * in <= (int64_t(24) << 20))) return {kVec, 0, 1};
  const int64_t kblocks = (in + kKB - 1) / kKB;
  const double hbm_us = static_cast<double>(out * in + tokens * in + tokens * out * out_size) / 6.3e6;
  Plan best{kSplit, 16, 1};
  double best_us = 1e30;
  for (int64_t t = (tokens + 255) / 256, last = t + 3; t <= last; ++t) {
    const int n = static_cast<int>(((tokens + t - 1) / t + 15) / 16 * 16);
    for (int split = 1; split <= 8 && (split == 1 || split * 2 <= kblocks); split *= 2) {
      const double us = split_us(tokens, out, kblocks, n, split, hbm_us);
      if (us < best_us) best_us = us, best = {kSplit, n, split};
    }
  }
  for (int n = 32; n <= 256 && in > 0; n += 32) {  // (an empty sum has no MMA to fill a pair's accumulators)
    if (n > 32 && tokens <= n - 32) break;
    const double us = pair_us(tokens, out, kblocks, n, hbm_us);
    if (us < best_us) best_us = us, best = {kPair, n, 1};
  }
  return best;
}

// Map of a byte matrix [rows][cols], row pitch `stride`, in boxes of 128
// columns x box_rows with the 128-byte swizzle.
bool make_map(CUtensorMap *map, const void *base, int64_t rows, int64_t cols, int64_t stride, int box_rows) {
  const EncodeTiled fn = encode_tiled();
  if (!fn) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  const cuuint32_t box[2] = {kKB, static_cast<cuuint32_t>(box_rows)}, es[2] = {1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kSmemPerSm = 228 * 1024, kSmemMax = 227 * 1024;

// Shared memory of a split-kernel CTA with `stages` stages.
int split_smem(int n, int stages) { return 1024 + kHeadBytes + stages * (kABytes + n * kKB); }

template <typename Out>
int launch_split(const CUtensorMap &wmap, const CUtensorMap &qmap, const LinArgs &a, int smem, cudaStream_t s) {
  constexpr auto kernel = int8_linear_split_kernel<Out>;
  H24_CUDA_TRY(allow_smem<kernel>(kSmemMax));
  const int64_t tiles = (static_cast<int64_t>(a.out) + kM - 1) / kM * a.tok_tiles;
  if (tiles * a.split > INT32_MAX) return fail(H24_ERR_INVALID, "int8_linear: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.split));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(a.split);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = a.split > 1 ? 2 : 1;
  H24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, wmap, qmap, a));
  count_launches(1);
  return H24_OK;
}

template <typename Out>
int launch_pair(const CUtensorMap &wmap, const CUtensorMap &qmap, const LinArgs &a, cudaStream_t s) {
  constexpr auto kernel = int8_linear_pair_kernel<Out>;
  H24_CUDA_TRY(allow_smem<kernel>(kSmemMax));
  const int64_t tiles = (static_cast<int64_t>(a.out) + kPairM - 1) / kPairM * a.tok_tiles;
  if (tiles > INT32_MAX) return fail(H24_ERR_INVALID, "int8_linear: too many tiles");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < kPairs ? tiles : kPairs)));
  cfg.blockDim = dim3(kPairThreads);
  // All of the SM's shared memory: the pair takes all TMEM columns, so nothing
  // that waits for columns may be resident beside it.
  cfg.dynamicSmemBytes = kSmemMax;
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
  H24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, wmap, qmap, a));
  count_launches(1);
  return H24_OK;
}

template <typename Out>
int launch_typed(const Plan &plan, bool aligned, const CUtensorMap &wmap, const CUtensorMap &qmap, const LinArgs &a,
                 int smem, cudaStream_t s) {
  if (plan.kind == kVec) {
    if (a.tokens == 1) return launch_vec_rows<1, Out>(a, aligned, s);
    if (a.tokens == 2) return launch_vec_rows<2, Out>(a, aligned, s);
    return launch_vec_rows<4, Out>(a, aligned, s);
  }
  if (plan.kind == kPair) return launch_pair<Out>(wmap, qmap, a, s);
  return launch_split<Out>(wmap, qmap, a, smem, s);
}

}  // namespace

void int8_linear_plan(int64_t tokens, int64_t out, int64_t in, int out_dtype, int32_t plan[3]) {
  const Plan p = make_plan(tokens, out, in, out_dtype == H24_DTYPE_F32 ? 4 : 2);
  plan[0] = p.kind;
  plan[1] = p.n;
  plan[2] = p.split;
}

int launch_int8_linear(const Tables *T, const int8_t *q, const float *scale, int64_t tokens, int64_t q_stride,
                       const int8_t *w, const uint16_t *mu16, int64_t out, int64_t in, const float *bias,
                       int out_dtype, void *y, cudaStream_t s) {
  LinArgs a{};
  a.q = q;
  a.scale = scale;
  a.w = w;
  a.mu16 = mu16;
  a.bias = bias;
  a.y = y;
  a.err = T->err;
  a.q_stride = q_stride;
  a.tokens = static_cast<int>(tokens);
  a.out = static_cast<int>(out);
  a.in = static_cast<int>(in);
  a.y_vec = aligned16(y);
  const bool w_aligned = in % 16 == 0 && aligned16(w);
  const bool q_aligned = in % 16 == 0 && q_stride % 16 == 0 && q_stride >= in && aligned16(q);
  const Plan plan = make_plan(tokens, out, in, out_dtype == H24_DTYPE_F32 ? 4 : 2);
  int8_t *copy = nullptr;
  int64_t w_stride = in;
  if (plan.kind != kVec && in > 0 && !(w_aligned && q_aligned)) {
    const int64_t pitch = (in + 15) / 16 * 16, w_rows = w_aligned ? 0 : out, q_rows = q_aligned ? 0 : tokens;
    H24_CUDA_TRY(cudaMallocFromPoolAsync(reinterpret_cast<void **>(&copy), static_cast<size_t>((w_rows + q_rows) * pitch),
                                         T->pool, s));
    const RepackArgs rw{w, in, copy, w_rows}, rq{q, q_stride, copy + w_rows * pitch, q_rows};
    const int chunks = static_cast<int>(pitch / 16);
    const int64_t blocks = ((w_rows + q_rows) * chunks + kRepackThreads - 1) / kRepackThreads;
    const cudaError_t e = launch_pdl(repack_rows_kernel, dim3(wave_grid(blocks, 8)), dim3(kRepackThreads), s, rw, rq,
                                     static_cast<int>(in), chunks);
    if (e != cudaSuccess) {
      cudaFreeAsync(copy, s);
      return cuda_fail(e, "int8_linear: repack launch");
    }
    count_launches(1);
    if (w_rows) w = rw.dst, w_stride = pitch;
    if (q_rows) q = rq.dst, q_stride = pitch;
  }
  a.n = plan.n;
  a.split = plan.split;
  CUtensorMap wmap{}, qmap{};
  int smem = 0;
  if (plan.kind != kVec) {
    a.tok_tiles = static_cast<int>((tokens + a.n - 1) / a.n);
    const int rows = plan.kind == kPair ? a.n / 2 : a.n;  // tokens a CTA loads
    const int stage = kABytes + rows * kKB, kblocks = static_cast<int>((in + kKB - 1) / kKB);
    if (plan.kind == kPair) {
      a.stages = (kSmemMax - 1024 - kHeadBytes) / stage;
    } else {
      a.tmem_cols = 32;
      while (a.tmem_cols < a.n) a.tmem_cols *= 2;
      // As many stages as fit beside the CTAs that share an SM, and no more
      // than a CTA's k blocks.
      const int64_t ctas = (out + kM - 1) / kM * a.tok_tiles * a.split;
      const int per_sm = ctas <= 148 || a.n > 128 ? 1 : ctas <= 296 || a.n > 64 ? 2 : 3;
      const int per = (kblocks + a.split - 1) / a.split;
      a.stages = (kSmemMax / per_sm - 2 * 1024 - kHeadBytes) / stage;
      a.stages = a.stages > per && per > 0 ? per : a.stages;
    }
    a.stages = a.stages > kMaxStages ? kMaxStages : a.stages;
    // A CTA holds no smaller share of an SM's shared memory than of its TMEM,
    // so that every CTA that is resident, of whatever calls, finds its columns:
    // the CTAs of a cluster wait for one another and must not wait for TMEM too.
    smem = split_smem(a.n, a.stages);
    const int part = a.split > 1 ? 1024 + kHeadBytes + a.n * kM * 4 : 0;  // the int32 tile over the stages
    const int share = static_cast<int>(static_cast<int64_t>(kSmemPerSm) * a.tmem_cols / 512);
    smem = smem < part ? part : smem;
    smem = smem < share ? share : smem;
    // (An empty sum loads nothing and needs no maps.)
    if (in > 0 && (!make_map(&wmap, w, out, w_stride, w_stride, kM) ||
                   !make_map(&qmap, q, tokens, w_stride, q_stride, rows))) {
      if (copy) cudaFreeAsync(copy, s);
      return fail(H24_ERR_CUDA, "int8_linear: cuTensorMapEncodeTiled failed");
    }
  }
  int rc;
  switch (out_dtype) {
    case H24_DTYPE_F32: rc = launch_typed<float>(plan, w_aligned && q_aligned, wmap, qmap, a, smem, s); break;
    case H24_DTYPE_F16: rc = launch_typed<__half>(plan, w_aligned && q_aligned, wmap, qmap, a, smem, s); break;
    default: rc = launch_typed<__nv_bfloat16>(plan, w_aligned && q_aligned, wmap, qmap, a, smem, s); break;
  }
  if (copy) {
    const cudaError_t e = cudaFreeAsync(copy, s);
    if (rc == H24_OK && e != cudaSuccess) rc = cuda_fail(e, "cudaFreeAsync");
  }
  return rc;
}

}  // namespace h24
