// h24_int8_linear.cu -- product of int8 activations with an INT8 layer:
//   y[t][o] = (sum_k q[t][k] * W[o][k]) * scale[t] * fp16(mu16[o] / 127) + bias[o]
// The sum is exact in int32 (in_features is bounded so that it cannot
// overflow), the scaling is fp32 and y is rounded once.  The weight's scale
// is the one PackedInt8Linear.materialize uses (pollux.py:545-554).
//
// The weights are the M operand (128 output features a tile, one TMEM lane
// each) and the tokens the N operand, so one token costs 16 columns of a tile
// and not 128 rows, and a warp's 32 lanes store 32 neighbouring outputs.
#include <cuda.h>  // CUtensorMap and its enums; the entry point is looked up at run time

#include "h24_internal.cuh"

namespace h24 {
namespace {

constexpr int kM = 128;        // output features per tile
constexpr int kKB = 128;       // k per stage: one 128-byte swizzle row
constexpr int kABytes = kM * kKB;
constexpr int kMaxStages = 12;
constexpr int kHeadBytes = 1024;  // barriers, TMEM address, abort flag; the stages start on 1 KB
constexpr unsigned long long kWaitNs = 2000000000ull;  // bounded waits: 2 s

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
};

struct LinHead {
  uint64_t full[kMaxStages], empty[kMaxStages], done;
  uint32_t tmem;
  int abort;
};
static_assert(sizeof(LinHead) <= kHeadBytes, "head");

__device__ __forceinline__ uint32_t su32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void bar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(count));
}

__device__ __forceinline__ bool bar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(su32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Waits for a phase for at most kWaitNs; false on a timeout (abort flag and
// device error word raised) or, where `heed`, when another role gave up.
__device__ __noinline__ bool bar_wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort, int *err, bool heed) {
  const unsigned long long t0 = now_ns();
  for (;;) {
    if (bar_try(bar, parity)) return true;
    if (heed && *abort) return false;
    if (now_ns() - t0 > kWaitNs) {
      *abort = 1;
      atomicExch(err, H24_ERR_TIMEOUT);
      return false;
    }
  }
}
__device__ __forceinline__ bool bar_wait(uint64_t *bar, uint32_t parity, volatile int *abort, int *err,
                                         bool heed = true) {
  return bar_try(bar, parity) || bar_wait_slow(bar, parity, abort, err, heed);
}

__device__ __forceinline__ void bar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}

// A box of the map at (k, row) into shared memory.  k is a multiple of 128;
// what lies outside the matrix arrives as zeros.
__device__ __forceinline__ void tma_load(const CUtensorMap *map, void *dst, uint64_t *bar, int k, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::
          "r"(su32(dst)),
      "l"(map), "r"(k), "r"(row), "r"(su32(bar))
      : "memory");
}

// Shared-memory descriptor of a K-major tile of 128-byte rows with the
// 128-byte swizzle: 8-row groups 1,024 bytes apart, version 1.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr >> 4) & 0x3FFFu) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(2) << 61);
}

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
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(su32(bar))
      : "memory");
}

// 16 TMEM columns of this warp's 32 lanes.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, int (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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

// 16 bytes at `p`, any alignment, from the 4-byte words around it; words not
// wholly inside [lo, hi) are read by the byte, and bytes from p + valid on
// come back as zeros.
__device__ __forceinline__ uint4 load16_any(const int8_t *p, int valid, const int8_t *lo, const int8_t *hi) {
  const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 3u);
  const int8_t *a = p - sh;
  uint32_t w[5];
#pragma unroll
  for (int i = 0; i < 5; ++i) {
    const int8_t *x = a + 4 * i;
    w[i] = 0;
    if (i == 4 && sh == 0) break;
    if (x >= lo && x + 4 <= hi) {
      w[i] = __ldg(reinterpret_cast<const uint32_t *>(x));
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (x + j >= lo && x + j < hi)
          w[i] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(x + j))) << (8 * j);
    }
  }
  uint32_t r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = __funnelshift_r(w[i], w[i + 1], 8 * sh);
    const int left = valid - 4 * i;
    if (left < 4) r[i] &= left <= 0 ? 0u : (0xFFFFFFFFu >> (8 * (4 - left)));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

// Rows [row0, row0 + rows) x k [k0, k0 + 128) of a byte matrix into a swizzled
// tile, by the 128 threads of the filling warps; outside it zeros.
__device__ __forceinline__ void fill_tile(uint8_t *tile, int rows, const int8_t *base, int64_t stride, int row0,
                                          int nrows, int k0, int in, int t) {
  const int8_t *hi = base + static_cast<int64_t>(nrows - 1) * stride + in;
  for (int i = t; i < rows * 8; i += 128) {
    const int r = i >> 3, c = i & 7, k = k0 + 16 * c;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row0 + r < nrows && k < in)
      v = load16_any(base + static_cast<int64_t>(row0 + r) * stride + k, in - k, base, hi);
    *reinterpret_cast<uint4 *>(tile + r * 128 + ((c ^ (r & 7)) << 4)) = v;
  }
}

constexpr int kSplitThreads = 192;  // warp 0 loads, warp 1 issues MMAs, warps 2-5 read TMEM

// One CTA per 128 x n tile and k slice.  The `split` CTAs of a cluster take a
// slice of the tile's k each; their int32 partial tiles meet in distributed
// shared memory, where CTA r finishes every split-th part of the tokens (the
// sum is an integer, so the order does not matter).  kTma: operands arrive by
// TMA (16-byte aligned rows); otherwise warps 2-5 place them by hand.
template <bool kTma, typename Out>
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
      bar_init(&H.full[s], kTma ? 1 : 128);
      bar_init(&H.empty[s], 1);
    }
    bar_init(&H.done, 1);
    H.abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    if (kTma) {
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
    if (kTma && lane == 0) {
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
    const int ft = t - 64;
    if (!kTma) {
      int s = 0;
      uint32_t ph = 0;
      for (int i = 0; i < nkb; ++i) {
        if (!bar_wait(&H.empty[s], ph ^ 1, abort, a.err)) break;
        uint8_t *st = stages + static_cast<size_t>(s) * stage_bytes;
        fill_tile(st, kM, a.w, a.in, o0, a.out, (kb0 + i) * kKB, a.in, ft);
        fill_tile(st + kABytes, a.n, a.q, a.q_stride, t0, a.tokens, (kb0 + i) * kKB, a.in, ft);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        bar_arrive(&H.full[s]);
        if (++s == a.stages) s = 0, ph ^= 1;
      }
    }
    // TMEM lane quarter of this warp, and its output feature.
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const int64_t o = static_cast<int64_t>(o0) + row;
    const bool live = o < a.out;
    const float ws = live ? weight_scale(a.mu16, o) : 0.f, b = live && a.bias ? __ldg(a.bias + o) : 0.f;
    Out *y = static_cast<Out *>(a.y) + static_cast<int64_t>(t0) * a.out + o;
    const int n_live = min(a.n, a.tokens - t0);
    bar_wait(&H.done, 0, abort, a.err, false);
    __syncwarp();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t ta = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    int r[16];
    if (a.split == 1) {
      for (int c = 0; c < n_live; c += 16) {
        __syncwarp();
        tmem_ld16(ta + c, r);
        if (nkb == 0) {  // in_features 0: an empty sum
#pragma unroll
          for (int j = 0; j < 16; ++j) r[j] = 0;
        }
        if (live && !*abort) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < n_live)
              put(y + static_cast<int64_t>(c + j) * a.out, finish(r[j], __ldg(a.scale + t0 + c + j), ws, b));
        }
      }
    } else {
      // The partial tile as [token][feature] over the stages (the MMAs and
      // copies that used them are complete).
      int *part = reinterpret_cast<int *>(stages);
      for (int c = 0; c < n_live; c += 16) {
        tmem_ld16(ta + c, r);
#pragma unroll
        for (int j = 0; j < 16; ++j) part[(c + j) * kM + row] = r[j];
      }
    }
  }
  __syncwarp();
  if (a.split > 1) {
    cluster_sync_all();
    if (warp >= 2 && !*abort) {
      const int row = (warp & 3) * 32 + lane;
      const int64_t o = static_cast<int64_t>(o0) + row;
      if (o < a.out) {
        const float ws = weight_scale(a.mu16, o), b = a.bias ? __ldg(a.bias + o) : 0.f;
        Out *y = static_cast<Out *>(a.y) + static_cast<int64_t>(t0) * a.out + o;
        const uint32_t mine = su32(stages) + static_cast<uint32_t>(row) * 4;
        const int n_live = min(a.n, a.tokens - t0);
        for (int c = rank; c < n_live; c += a.split) {
          int acc = 0;
          for (int p = 0; p < a.split; ++p) {
            uint32_t addr;
            int v;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(mine + c * kM * 4), "r"(p));
            asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
            acc += v;
          }
          put(y + static_cast<int64_t>(c) * a.out, finish(acc, __ldg(a.scale + t0 + c), ws, b));
        }
      }
    }
    __syncwarp();
    cluster_sync_all();  // no CTA leaves while another reads its tile
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_cols) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &got) != cudaSuccess ||
        got != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
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

template <bool kTma, typename Out>
int launch_split(const CUtensorMap &wmap, const CUtensorMap &qmap, const LinArgs &a, int smem, cudaStream_t s) {
  constexpr auto kernel = int8_linear_split_kernel<kTma, Out>;
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
int launch_typed(bool tma, const CUtensorMap &wmap, const CUtensorMap &qmap, const LinArgs &a, int smem,
                 cudaStream_t s) {
  return tma ? launch_split<true, Out>(wmap, qmap, a, smem, s) : launch_split<false, Out>(wmap, qmap, a, smem, s);
}

}  // namespace

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
  const int64_t otiles = (out + kM - 1) / kM;
  a.tok_tiles = static_cast<int>((tokens + 255) / 256);
  a.n = static_cast<int>(((tokens + a.tok_tiles - 1) / a.tok_tiles + 15) / 16 * 16);
  const int kblocks = static_cast<int>((in + kKB - 1) / kKB);
  a.split = 1;
  while (a.split < 8 && a.split * 2 <= kblocks && otiles * a.tok_tiles * a.split * 2 <= 148 * 2) a.split *= 2;
  a.tmem_cols = 32;
  while (a.tmem_cols < a.n) a.tmem_cols *= 2;
  const int per = (kblocks + a.split - 1) / a.split;  // stages a CTA can use
  a.stages = (kSmemMax / (a.n <= 32 ? 3 : a.n <= 128 ? 2 : 1) - 2 * 1024 - kHeadBytes) / (kABytes + a.n * kKB);
  a.stages = a.stages > kMaxStages ? kMaxStages : a.stages;
  a.stages = a.stages > per && per > 0 ? per : a.stages;
  // A CTA holds no smaller share of an SM's shared memory than of its TMEM, so
  // that every CTA that is resident, of whatever calls, finds its columns: the
  // CTAs of a cluster wait for one another and must not wait for TMEM too.
  int smem = split_smem(a.n, a.stages);
  const int part = a.split > 1 ? 1024 + kHeadBytes + a.n * kM * 4 : 0;  // the int32 tile over the stages
  const int share = static_cast<int>(static_cast<int64_t>(kSmemPerSm) * a.tmem_cols / 512);
  smem = smem < part ? part : smem;
  smem = smem < share ? share : smem;
  const bool tma = in > 0 && in % 16 == 0 && q_stride % 16 == 0 && q_stride >= in && aligned16(q) && aligned16(w);
  CUtensorMap wmap{}, qmap{};
  if (tma && (!make_map(&wmap, w, out, in, in, kM) || !make_map(&qmap, q, tokens, in, q_stride, a.n)))
    return fail(H24_ERR_CUDA, "int8_linear: cuTensorMapEncodeTiled failed");
  switch (out_dtype) {
    case H24_DTYPE_F32: return launch_typed<float>(tma, wmap, qmap, a, smem, s);
    case H24_DTYPE_F16: return launch_typed<__half>(tma, wmap, qmap, a, smem, s);
    default: return launch_typed<__nv_bfloat16>(tma, wmap, qmap, a, smem, s);
  }
}

}  // namespace h24
