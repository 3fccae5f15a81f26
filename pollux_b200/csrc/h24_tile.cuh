// h24_tile.cuh -- what the tcgen05 kernels over TMA-filled tiles share: bounded
// barrier waits, tile loads, commits, TMEM reads, tensor maps and loads of 16
// bytes from any alignment.
#pragma once

#include <cuda.h>  // CUtensorMap and its enums; the entry point is looked up at run time

#include "h24_internal.cuh"

namespace h24 {

constexpr unsigned long long kWaitNs = 2000000000ull;  // bounded waits: 2 s
constexpr int kPairs = 74;  // pairs of CTAs that a B200's 148 SMs hold

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
static __device__ __noinline__ bool bar_wait_slow(uint64_t *bar, uint32_t parity, volatile int *abort, int *err, bool heed) {
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

__device__ __forceinline__ void bar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(bar)), "r"(bytes) : "memory");
}

// A box of the map at (k, row) into shared memory.  k lies on 16 bytes; what
// lies outside the matrix arrives as zeros.
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

__device__ __forceinline__ void mma_commit(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(su32(bar))
      : "memory");
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// The 16 bytes at `a` (16-byte aligned); those outside [lo, hi) are not read
// and come back as zeros.
__device__ __forceinline__ uint4 load16_within(const int8_t *a, const int8_t *lo, const int8_t *hi) {
  if (a >= lo && a + 16 <= hi) return __ldg(reinterpret_cast<const uint4 *>(a));
  uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll  // the sixteen loads in flight together
  for (int j = 0; j < 16; ++j)
    if (a + j >= lo && a + j < hi) w[j / 4] |= static_cast<uint32_t>(static_cast<uint8_t>(__ldg(a + j))) << (8 * (j & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 16 bytes at offset `off` (0-15) of two aligned blocks; bytes from `valid` on
// come back as zeros.
__device__ __forceinline__ uint4 join16(uint4 x, uint4 y, uint32_t off, int valid) {
  const uint32_t v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
  uint32_t h[6], w[5], r[4];  // words off / 8 * 2 on, then off / 4 on
#pragma unroll
  for (int i = 0; i < 6; ++i) h[i] = (off & 8) ? v[i + 2] : v[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) w[i] = (off & 4) ? h[i + 1] : h[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = __funnelshift_r(w[i], w[i + 1], 8 * (off & 3));
    const int left = valid - 4 * i;
    if (left < 4) r[i] &= left <= 0 ? 0u : (0xFFFFFFFFu >> (8 * (4 - left)));
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}

__device__ __forceinline__ uint32_t offset16(const int8_t *p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u);
}

// 16 bytes at `p`, any alignment, from the two aligned blocks around it (a
// warp's neighbours share them in L1); bytes from p + valid on come back as zeros.
__device__ __forceinline__ uint4 load16_any(const int8_t *p, int valid, const int8_t *lo, const int8_t *hi) {
  const uint32_t off = offset16(p);
  return join16(load16_within(p - off, lo, hi), off ? load16_within(p - off + 16, lo, hi) : make_uint4(0, 0, 0, 0), off,
                valid);
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

#define H24_O8(b) "=r"(r[b]), "=r"(r[b + 1]), "=r"(r[b + 2]), "=r"(r[b + 3]), "=r"(r[b + 4]), "=r"(r[b + 5]), \
                  "=r"(r[b + 6]), "=r"(r[b + 7])
#define H24_I8(b) "+r"(r[b]), "+r"(r[b + 1]), "+r"(r[b + 2]), "+r"(r[b + 3]), "+r"(r[b + 4]), "+r"(r[b + 5]), \
                  "+r"(r[b + 6]), "+r"(r[b + 7])
// Starts the load of 32 TMEM columns; r holds them after tmem_wait32(r).
__device__ __forceinline__ void tmem_ask32(uint32_t taddr, int (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : H24_O8(0), H24_O8(8), H24_O8(16), H24_O8(24)
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait32(int (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : H24_I8(0), H24_I8(8), H24_I8(16), H24_I8(24) : : "memory");
}
#undef H24_I8
#undef H24_O8

__device__ __forceinline__ uint32_t cluster_addr(const void *p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(su32(p)), "r"(rank));
  return r;
}
// As tma_load, for a CTA of a pair: the bytes count on a barrier of the pair.
__device__ __forceinline__ void tma_load_pair(const CUtensorMap *map, void *dst, uint32_t bar, int k, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3}], [%4];" ::"r"(su32(dst)),
      "l"(map), "r"(k), "r"(row), "r"(bar)
      : "memory");
}

// An arrival on the barrier at this offset in both CTAs.
__device__ __forceinline__ void mma_commit_pair(uint64_t *bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::
          "r"(su32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiled encode_tiled() {
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

}  // namespace h24
