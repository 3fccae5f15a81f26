// h24_sample.cu -- one token a row under temperature, top-k, top-p and min-p.
//
//   m = max_i l_i,  z_i = (l_i - m) * fp32(1 / T)  (0 where l_i = m)
//   w_i = rint(exp(z_i) * 2^40)                       a 64-bit integer
//   order: z descending, ties by index ascending
//   1. the first k of the order           (T <= 0: k = 1, T = 1)
//   2. of these, those whose mass before them is < max(1, ceil(p * M_k)), M_k = the mass of step 1
//   3. of these, w_i >= ceil(min_p * 2^40)
//   token = the first index, ascending, at which the running mass of what is
//   left exceeds min(floor(u * M), M - 1);  logprob = z_token - log(sum_i w_i / 2^40)
//
// Weights are fixed-point integers so that every sum is exact: the token does
// not depend on how a row is split over threads and blocks.  2^-40 of the
// largest probability is the smallest weight kept; with at most 2^22 tokens a
// row's mass stays below 2^62.
//
// A row is held by a cluster of 1 to 8 CTAs, a slice each in shared memory, or,
// where there are rows enough for the SMs, read by one CTA from L2 in each pass.
// A cut is found from a histogram of |z| in steps of 1/72 (beyond |z| = 28.4 a
// weight rounds to 0), which the CTAs add through distributed shared memory, a
// share of the steps each.
//   top-k: only each thread's largest logit is counted.  The k-th largest of
//     those bounds the k-th token, so the tokens of the steps up to its own (k
//     and a few more) are listed in the pass that adds the weights; the first
//     CTA ranks the list and makes all three cuts and the choice.
//   top-p alone: the steps get masses in the pass that adds the weights, which
//     gives the step in which the cut falls.  A second pass adds what lies
//     before that step and lists its tokens; the first CTA finds the last one
//     kept, and the warp in whose part the target falls walks it.
//   neither, or a min-p that leaves less than p: the walk alone.
// What bounds it, measured on a B200: one row, the chain of a dozen barriers
// and exchanges ([1,50688] fp32, k = 50, p = 0.9: 10.9 us; no cut: 7.3); many
// rows, instruction issue and the second and third read from L2 ([512,50688]
// fp32: no cut 51 us, k = 50 43-58, p = 0.9 122-127, for 15.9 us of HBM traffic;
// fp16 and bf16, p = 0.9: 134; rows off 16 bytes, which every pass reads by the
// element: [512,50257] fp32 73, 65 and 143).  For
// a cut at p, a list bounded by the threads' maxima as for k was tried: half of
// the rows' cuts lie behind 700 tokens, and 2,200 cost what the steps cost.
//
// "z descending, index ascending" is one 64-bit key: |z|'s bits above the
// index (z <= 0, so |z| ascending is z descending, and the bits of
// non-negative floats ascend with them).  A selection is then a cut on that
// key, found by histograms of its digits.
#include "h24_internal.cuh"

namespace h24 {
namespace {

using u64 = unsigned long long;

constexpr float kOne = 1099511627776.0f;  // 2^40
constexpr float kLargest = 3.402823466e38f;

struct SampleArgs {
  const void *logits;
  int64_t rows, vocab, stride;
  const float *u;
  const float *temperature;
  const int32_t *top_k;
  const float *top_p;
  const float *min_p;
  float temperature1, top_p1, min_p1;
  int32_t top_k1;
  int64_t *tokens;
  float *logprobs;
  bool sorted;  // rows in the order of costly_first()
};

// |z| of a logit; m is finite and inv_t within fp32's normal range.  l = m
// gives 0, -inf gives inf, NaN gives NaN (which no comparison lets pass), and
// +inf, which counts as the largest number, gives -inf: see near().
__device__ __forceinline__ float dist(float l, float m, float inv_t) { return __fmul_rn(__fsub_rn(m, l), inv_t); }
__device__ __forceinline__ float near(float d) { return fmaxf(d, 0.f); }  // of a d that has passed a comparison

// A weight from f = exp(-d) * 2^40.  Below 2^32 (|z| above 5.5, nearly every
// token) one conversion; from there the float is an integer, its mantissa
// shifted.  (A 64-bit conversion, or integer steps for both ranges, cost more
// issue slots.)
__device__ __forceinline__ float scaled(float d) { return expf(-d) * kOne; }
__device__ __forceinline__ u64 to_weight(float f) {
  u64 w = __float2uint_rn(f);
  if (f >= 4294967040.0f) {
    const uint32_t bits = __float_as_uint(fminf(f, kOne));
    w = static_cast<u64>((bits & 0x7FFFFFu) | 0x800000u) << ((bits >> 23) - 150);
  }
  return w;
}
__device__ __forceinline__ u64 weight(float d) { return to_weight(scaled(d)); }

constexpr int kIndexBits = 22;
__device__ __forceinline__ u64 order_key(float d, int64_t i) {
  return (static_cast<u64>(__float_as_uint(d)) << kIndexBits) | static_cast<u64>(i);
}
__device__ __forceinline__ float key_dist(u64 key) { return __uint_as_float(static_cast<uint32_t>(key >> kIndexBits)); }
__device__ __forceinline__ uint32_t key_index(u64 key) { return static_cast<uint32_t>(key) & ((1u << kIndexBits) - 1); }

// What step 2 and 3 ask for, in the arithmetic the header states.
__device__ __forceinline__ u64 mass_limit(float p, u64 mk) {
  const double x = ceil(static_cast<double>(p) * static_cast<double>(mk));
  return x > 1.0 ? static_cast<u64>(x) : 1ull;
}
__device__ __forceinline__ u64 weight_floor(float min_p) {
  const double x = ceil(fmin(fmax(static_cast<double>(min_p), 0.0), 1.0) * static_cast<double>(kOne));
  return x > 1.0 ? static_cast<u64>(x) : 1ull;  // weight 0 is never chosen
}
__device__ __forceinline__ u64 draw_target(float u, u64 mass) {
  const double x = floor((u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(mass));
  return x >= static_cast<double>(mass - 1) ? mass - 1 : static_cast<u64>(x);
}

// ---------------------------------------------------------------------------
// distributed shared memory of the cluster
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t su32(const void *p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t peer(const void *p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(su32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint4 peer_ld4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
__device__ __forceinline__ void peer_st(uint32_t addr, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void peer_add64(uint32_t addr, u64 v) {
  asm volatile("red.shared::cluster.add.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t peer_add(uint32_t addr, uint32_t v) {
  uint32_t r;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(r) : "r"(addr), "r"(v) : "memory");
  return r;
}

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;
// Steps of |z|: 2,046 up to 28.45, where exp(-|z|) * 2^40 is below 1/2.
constexpr float kBinsPerNat = 71.9f, kFar = 28.45f;
constexpr int kList = 1024;
constexpr int kFew = 128;  // lists up to this long are ranked by counting
constexpr int kMaxCluster = 8;
constexpr int kQueue = 6;  // tokens a lane keeps until a warp works on them together

struct Cut {  // where a cut falls: the step, what is before it and in it
  u64 bin, count_before, mass_before, count, mass;
};

struct SampleShared {
  uint32_t count[kBins], lo[kBins], hi[kBins];
  u64 list[kList];
  u64 few[2][kFew];
  uint2 queue[kWarps][kQueue][32];
  u64 slot[kMaxCluster];  // one value of each CTA
  u64 slice_count[kMaxCluster], slice_mass[kMaxCluster];
  u64 total[kMaxCluster], first[kMaxCluster], kept[kMaxCluster];
  Cut cut;
  u64 scan_m[kWarps];
  uint32_t step_c[kWarps], warp_first[kWarps];
  u64 warp_total[kWarps], warp_kept[kWarps];
  u64 red[kWarps];
  u64 pick;
  uint32_t list_n, local_n, base;
};

static_assert(kList * 8 <= kBins * 4, "a CTA's own list lies over one word of the steps");

__device__ __forceinline__ void cluster_sync(int c) {
  if (c == 1) {
    __syncthreads();
  } else {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <typename T>
__device__ __forceinline__ T warp_scan(T v, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  return v;
}
__device__ u64 sum_block(u64 v, u64 *red) {
  v = warp_sum(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 r = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) r += red[w];
  __syncthreads();
  return r;
}

// The elements of one 16-byte vector of a slice.
template <int DT>
struct Vec {
  static constexpr int kN = DT == H24_DTYPE_F32 ? 4 : 8;
  float v[kN];
  __device__ __forceinline__ explicit Vec(uint4 raw) {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (DT == H24_DTYPE_F32) {
        v[i] = __uint_as_float(w[i]);
      } else if (DT == H24_DTYPE_F16) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
};

// The step of a |z| below kFar: the nearest one (an addition, no conversion).
__device__ __forceinline__ int bin_of(float d) {
  return static_cast<int>(__float_as_uint(fmaf(d, kBinsPerNat, 8388608.0f)) - 0x4B000000u);
}

// Sorts the first n (a power of two) keys of the list, ascending.
__device__ __noinline__ void sort_list(u64 *list, int n) {
  for (int k = 2; k <= n; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
        const u64 x = list[a], y = list[b];
        if ((x > y) == ((a & k) == 0)) list[a] = y, list[b] = x;
      }
      __syncthreads();
    }
}

// The row that a CTA of its own takes, when rows with different settings are
// more than fit at once: those with a cut at p alone first (three passes), then
// those with a cut at k, then the rest, so that no long row starts last.
__device__ int64_t costly_first(const SampleArgs &a) {
  auto kind = [&](int64_t r) {
    const float t = a.temperature ? a.temperature[r] : a.temperature1, p = a.top_p ? a.top_p[r] : a.top_p1;
    const int64_t k = t > 0.f ? (a.top_k ? a.top_k[r] : a.top_k1) : 1;
    return k == 1 ? 2 : k > 0 && k < a.vocab ? 1 : p < 1.f ? 0 : 2;
  };
  __shared__ int64_t row;
  const int64_t want = blockIdx.x;
  int64_t before = 0;  // rows of the kinds, and of the rows, before
  for (int c = 0; c < 3; ++c)
    for (int64_t r0 = 0; r0 < a.rows; r0 += kThreads) {
      const int64_t r = r0 + threadIdx.x;
      const bool is = r < a.rows && kind(r) == c;
      const int here = __syncthreads_count(is);
      if (want < before + here) {
        // The (want - before)-th of these: counted by warps, then by lanes.
        __shared__ int warps[kWarps];
        const uint32_t votes = __ballot_sync(0xffffffffu, is);
        if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = __popc(votes);
        __syncthreads();
        int64_t at = before;
        for (int w = 0; w < static_cast<int>(threadIdx.x >> 5); ++w) at += warps[w];
        if (is && at + __popc(votes & ((1u << (threadIdx.x & 31)) - 1)) == want) row = r;
        __syncthreads();
        return row;
      }
      before += here;
    }
  return want;  // not reached: every row is of a kind
}

struct Always {  // a condition that the compiler knows
  constexpr operator bool() const { return true; }
};

struct RowSettings {
  int64_t k;
  float inv_t, p, u;
  u64 least;
};

template <int DT, bool kHeld>
__global__ void __launch_bounds__(kThreads, kHeld ? 1 : 2) sample_cluster_kernel(const SampleArgs a, int nc, int slice) {
  using V = Vec<DT>;
  constexpr int kVN = V::kN, kSize = DT == H24_DTYPE_F32 ? 4 : 2;
  extern __shared__ __align__(16) uint8_t sample_raw[];
  SampleShared &S = *reinterpret_cast<SampleShared *>(sample_raw);
  uint4 *data = reinterpret_cast<uint4 *>(sample_raw + (sizeof(SampleShared) + 15) / 16 * 16);
  const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
  const int rank = static_cast<int>(blockIdx.x) % nc;
  const int begin = rank * slice;
  const int n = static_cast<int>(max(int64_t(0), min(static_cast<int64_t>(slice), a.vocab - begin)));
  const int nvec = (n + kVN - 1) / kVN;
  // A warp's part of the slice, in the order of the indices.
  const int v0 = static_cast<int>(static_cast<int64_t>(nvec) * warp / kWarps);
  const int v1 = static_cast<int>(static_cast<int64_t>(nvec) * (warp + 1) / kWarps);

  auto clear_steps = [&]() {
    for (int i = t; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4 *>(S.count)[i] = make_uint4(0, 0, 0, 0);
  };
  if (t == 0) S.list_n = 0, S.local_n = 0;
  clear_steps();
  __syncwarp();
  if (nc > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_enter();
  const int64_t r = a.sorted ? costly_first(a) : blockIdx.x / nc;
  RowSettings R;
  {
    float temp = a.temperature ? a.temperature[r] : a.temperature1;
    R.k = a.top_k ? a.top_k[r] : a.top_k1;
    R.p = a.top_p ? a.top_p[r] : a.top_p1;
    if (R.p < 0.f) R.p = 0.f;  // the first token alone
    R.least = weight_floor(a.min_p ? a.min_p[r] : a.min_p1);
    R.u = a.u[r];
    if (!(temp > 0.f)) temp = 1.f, R.k = 1;
    if (R.k <= 0 || R.k > a.vocab) R.k = a.vocab;
    R.inv_t = fminf(fmaxf(__fdiv_rn(1.0f, temp), 1.17549435e-38f), kLargest);
  }

  // ---- the slice into shared memory (kHeld; else it is read again in each
  // pass, from L2); each thread's and the row's largest logit ----
  const uint8_t *src = static_cast<const uint8_t *>(a.logits) + (r * a.stride + begin) * kSize;
  float mine_max = -INFINITY;
  const int nfull = aligned16(src) ? n / kVN : 0;  // vectors that can be loaded whole
  // Vector i by the element, -inf past the slice's end.
  auto pieces = [&](int i) -> uint4 {
    alignas(16) uint8_t raw[16];
#pragma unroll
    for (int j = 0; j < kVN; ++j) {
      const int e = i * kVN + j;
      if (DT == H24_DTYPE_F32)
        reinterpret_cast<float *>(raw)[j] = e < n ? reinterpret_cast<const float *>(src)[e] : -INFINITY;
      else
        reinterpret_cast<uint16_t *>(raw)[j] = e < n ? reinterpret_cast<const uint16_t *>(src)[e]
                                                    : static_cast<uint16_t>(DT == H24_DTYPE_F16 ? 0xFC00 : 0xFF80);
    }
    return *reinterpret_cast<const uint4 *>(raw);
  };
  auto raw_at = [&](int i) -> uint4 {
    if (kHeld) return data[i];
    return i < nfull ? __ldcg(reinterpret_cast<const uint4 *>(src) + i) : pieces(i);
  };
  auto at = [&](int i) -> V { return V(raw_at(i)); };
  // Every vector of this warp's part, a lane each: f(vector, its number, live);
  // the lanes stay together, past the end with live false.  What is not held
  // is loaded kAhead vectors at a time.
  auto each_vector = [&](auto f) {
    int i0 = v0;
    if constexpr (!kHeld) {
      constexpr int kAhead = 16 / kVN;
      const int whole = min(v1, nfull);
      for (; i0 + 32 * kAhead <= whole; i0 += 32 * kAhead) {
        uint4 raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = __ldcg(reinterpret_cast<const uint4 *>(src) + i0 + 32 * u + lane);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) f(V(raw[u]), i0 + 32 * u + lane, Always{});
      }
    }
    for (; i0 < v1; i0 += 32) {
      const int i = i0 + lane;
      f(V(raw_at(min(i, v1 - 1))), i, i < v1);
    }
  };
  if (kHeld) {
#pragma unroll 4
    for (int i = t; i < nfull; i += kThreads) {
      const uint4 raw = __ldcs(reinterpret_cast<const uint4 *>(src) + i);
      data[i] = raw;
      const V v(raw);
#pragma unroll
      for (int j = 0; j < kVN; ++j) mine_max = fmaxf(mine_max, v.v[j]);
    }
    for (int i = nfull + t; i < nvec; i += kThreads) {
      const uint4 raw = pieces(i);
      data[i] = raw;
      const V v(raw);
#pragma unroll
      for (int j = 0; j < kVN; ++j) mine_max = fmaxf(mine_max, v.v[j]);
    }
  } else {
    each_vector([&](const V &v, int, auto live) {
#pragma unroll
      for (int j = 0; j < kVN; ++j)
        if (live) mine_max = fmaxf(mine_max, v.v[j]);
    });
  }
  float mx = mine_max;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) S.red[warp] = __float_as_uint(mx);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, __uint_as_float(static_cast<uint32_t>(S.red[w])));
  if (nc > 1) {
    // Every CTA of the cluster has started: its shared memory may be written.
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (t < nc) peer_st(peer(&S.slot[rank], t), __float_as_uint(mx));
    cluster_sync(nc);
    for (int c = 0; c < nc; ++c) mx = fmaxf(mx, __uint_as_float(static_cast<uint32_t>(S.slot[c])));
  }
  const float m = fminf(mx, kLargest);
  if (m == -INFINITY) {  // nothing to choose from (the same for the whole cluster)
    if (rank == 0 && t == 0) {
      a.tokens[r] = -1;
      if (a.logprobs) a.logprobs[r] = -INFINITY;
    }
    return;
  }

  const bool greedy = R.k == 1, cut_k = !greedy && R.k < a.vocab;
  bool cut_p = !greedy && R.p < 1.f;
  auto count_step = [&](int b, u64 w, bool counts, bool masses) {
    if (counts) atomicAdd(&S.count[b], 1u);
    if (masses) {
      const uint32_t wl = static_cast<uint32_t>(w), old = atomicAdd(&S.lo[b], wl);
      const uint32_t wh = static_cast<uint32_t>(w >> 32) + (old + wl < old ? 1u : 0u);
      if (wh) atomicAdd(&S.hi[b], wh);
    }
  };

  // This CTA's share of the steps, added over the cluster: four steps for each
  // group of nc lanes, one CTA's counts a lane, with the count and mass before
  // them (of the whole row).
  const int share = kBins / nc, my_bin = rank * share + t / nc * 4;
  uint32_t bc[4];
  uint32_t pre_c = 0;
  u64 bm[4], pre_m = 0;
  auto gather_bins = [&](bool masses) {
    const int x = t & (nc - 1);
    const uint4 c4 = peer_ld4(peer(&S.count[my_bin], x));
    bc[0] = c4.x, bc[1] = c4.y, bc[2] = c4.z, bc[3] = c4.w;
#pragma unroll
    for (int j = 0; j < 4; ++j) bm[j] = 0;
    if (masses) {
      const uint4 l4 = peer_ld4(peer(&S.lo[my_bin], x)), h4 = peer_ld4(peer(&S.hi[my_bin], x));
      bm[0] = l4.x | static_cast<u64>(h4.x) << 32;
      bm[1] = l4.y | static_cast<u64>(h4.y) << 32;
      bm[2] = l4.z | static_cast<u64>(h4.z) << 32;
      bm[3] = l4.w | static_cast<u64>(h4.w) << 32;
    }
    for (int o = 1; o < nc; o <<= 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bc[j] += __shfl_xor_sync(0xffffffffu, bc[j], o);
        if (masses) bm[j] += __shfl_xor_sync(0xffffffffu, bm[j], o);
      }
    }
    const uint32_t c = bc[0] + bc[1] + bc[2] + bc[3];
    const u64 q = bm[0] + bm[1] + bm[2] + bm[3];
    const uint32_t ic = warp_scan(x == 0 ? c : 0u, lane);
    const u64 im = masses ? warp_scan(x == 0 ? q : u64(0), lane) : 0;
    if (lane == 31) S.step_c[warp] = ic, S.scan_m[warp] = im;
    __syncthreads();
    pre_c = ic - c;
    pre_m = im - q;
    // Warps before this one, and all of them.
    const uint32_t wc = lane < kWarps ? S.step_c[lane] : 0u;
    pre_c += __reduce_add_sync(0xffffffffu, lane < warp ? wc : 0u);
    const uint32_t all_c = __reduce_add_sync(0xffffffffu, wc);
    u64 all_m = 0;
    if (masses) {
      const u64 wm = lane < kWarps ? S.scan_m[lane] : 0;
      pre_m += warp_sum(lane < warp ? wm : 0);
      all_m = warp_sum(wm);
    }
    if (t < nc) {
      peer_st(peer(&S.slice_count[rank], t), all_c);
      peer_st(peer(&S.slice_mass[rank], t), all_m);
    }
    cluster_sync(nc);
    for (int y = 0; y < rank; ++y) pre_c += S.slice_count[y], pre_m += S.slice_mass[y];
  };
  auto counted = [&]() -> u64 {
    u64 c = 0;
    for (int y = 0; y < nc; ++y) c += S.slice_count[y];
    return c;
  };
  // The step at which the running count (or mass) reaches `want`, told to all.
  auto find = [&](bool by_mass, u64 want) -> Cut {
    if ((t & (nc - 1)) == 0) {
      u64 c = pre_c, q = pre_m;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const u64 before = by_mass ? q : c, in = by_mass ? bm[j] : bc[j];
        if (before < want && want <= before + in) {
          for (int x = 0; x < nc; ++x) {
            const uint32_t to = peer(&S.cut, x);
            peer_st(to, static_cast<u64>(my_bin + j));
            peer_st(to + 8, c);
            peer_st(to + 16, q);
            peer_st(to + 24, bc[j]);
            peer_st(to + 32, bm[j]);
          }
        }
        c += bc[j];
        q += bm[j];
      }
    }
    cluster_sync(nc);
    return S.cut;
  };
  // Sends this CTA's own list (S.local_n keys) to the first CTA's, as many as
  // fit; returns the number in the cluster.  The cluster is in step after it.
  u64 *own = nc == 1 ? S.list : reinterpret_cast<u64 *>(S.lo);  // over the steps' masses, read by then
  auto ship = [&]() -> u64 {
    __syncthreads();
    const uint32_t here = S.local_n;
    if (nc == 1) return here;
    if (t < nc) peer_st(peer(&S.slot[rank], t), here);
    if (t == 0 && here) S.base = peer_add(peer(&S.list_n, 0), here);
    __syncthreads();
    const uint32_t to = peer(&S.list[0], 0), base = S.base;
    for (uint32_t i = t; i < min(here, static_cast<uint32_t>(kList)); i += kThreads)
      if (base + i < kList) peer_st(to + (base + i) * 8, own[i]);
    cluster_sync(nc);
    u64 all = 0;
    for (int c = 0; c < nc; ++c) all += S.slot[c];
    return all;
  };
  auto list_key = [&](u64 key) {
    const uint32_t place = atomicAdd(&S.local_n, 1u);
    if (place < kList) own[place] = key;
  };
  // Of the tokens of steps up to `last`: keys that satisfy `wanted` go to the
  // own list, and of those that satisfy `sure` before it, what min-p leaves is
  // added up a warp.  Each lane keeps what lies within the bound until one has
  // no room for four more: a token in a hundred would otherwise hold up its
  // warp each time, and a vote on every token costs more than its weight.
  auto collect = [&](int last, auto sure, auto wanted) {
    const float bound = fminf(static_cast<float>(last + 1) / kBinsPerNat, kFar);  // a step ends half a step before
    uint2 *mine = &S.queue[warp][0][lane];
    u64 sum = 0;
    int have = 0;
    auto flush = [&]() {
      const int rounds = __reduce_max_sync(0xffffffffu, have);
      for (int q = 0; q < rounds; ++q) {
        if (q >= have) continue;
        const uint2 e = mine[q * 32];
        const float d = __uint_as_float(e.y);
        if (bin_of(d) > last) continue;
        const u64 w = weight(d), key = order_key(d, e.x);
        if (sure(d, key))
          sum += w >= R.least ? w : 0;
        else if (w && wanted(d, key))
          list_key(key);
      }
      have = 0;
      __syncwarp();
    };
    each_vector([&](const V &v, int i, auto live) {
#pragma unroll
      for (int g = 0; g < kVN; g += 4) {
#pragma unroll
        for (int j = g; j < g + 4; ++j) {
          const float d = dist(v.v[j], m, R.inv_t);
          if (d < bound && live) {
            mine[have * 32] = make_uint2(begin + i * kVN + j, __float_as_uint(near(d)));
            ++have;
          }
        }
        if (__any_sync(0xffffffffu, have > kQueue - 4)) flush();
      }
    });
    flush();
    sum = warp_sum(sum);
    if (lane == 0) S.warp_kept[warp] = sum;
  };

  const auto none = [](float, u64) { return false; };

  // The k-th largest of the threads' largest logits is at most the k-th
  // largest logit: the steps of those alone give one at or beyond that in which
  // the cut at k falls.
  int k_last = -1;
  if (cut_k) {
    const float d = near(dist(fminf(mine_max, kLargest), m, R.inv_t));
    if (d < kFar && weight(d)) atomicAdd(&S.count[bin_of(d)], 1u);
    cluster_sync(nc);
    gather_bins(false);
    if (counted() >= static_cast<u64>(R.k)) k_last = static_cast<int>(find(false, static_cast<u64>(R.k)).bin);
  }

  // ---- one pass: total mass, and what the settings ask for beside it ----
  // f(|z|s, weights) of every vector of this warp's part; `few` where all of
  // its weights are below 2^32, one conversion each, else `each` for each.
  // (With a bound of 2^29, which lets four add up in 32 bits, half of the
  // warps had a lane above it.)
  auto pass = [&](auto few, auto each) -> u64 {
    u64 sum = 0;
    each_vector([&](const V &v, int i, auto live) {
      float d[kVN], f[kVN], top = 0.f;
#pragma unroll
      for (int j = 0; j < kVN; ++j) {
        d[j] = live ? dist(v.v[j], m, R.inv_t) : INFINITY;
        f[j] = scaled(d[j]);
        top = fmaxf(top, f[j]);
      }
      if (top < 4294967040.0f) {
        uint32_t w[kVN];
#pragma unroll
        for (int j = 0; j < kVN; ++j) {
          w[j] = __float2uint_rn(f[j]);
          sum += w[j];
        }
        few(i, v.v, d, w);
      } else {
#pragma unroll
        for (int j = 0; j < kVN; ++j) {
          const u64 w = to_weight(f[j]);
          sum += w;
          each(i, j, v.v[j], d[j], w);
        }
      }
    });
    return warp_sum(sum);
  };
  // `each` for a vector of small weights too.
  auto same = [&](auto each) {
    return [each](int i, const float(&l)[kVN], const float(&d)[kVN], const uint32_t(&w)[kVN]) {
#pragma unroll
      for (int j = 0; j < kVN; ++j) each(i, j, l[j], d[j], w[j]);
    };
  };
  // The masses of the steps that the cut at p may fall in.  Tokens beyond |z| =
  // ln(1.25 V / ((1 - p) L)) hold less than (1 - p) of a mass of at least L, so
  // the cut falls before them.  L: the threads' largest logits of this CTA
  // (CTAs may differ in what they leave out; the cut falls before all of it).
  auto pass_steps = [&]() -> u64 {
    float far = kFar;
    if (!kHeld) {  // (a slice that is held has too few tokens for this to pay)
      float some = mine_max > -INFINITY ? expf(-near(dist(fminf(mine_max, kLargest), m, R.inv_t))) : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) some += __shfl_xor_sync(0xffffffffu, some, o);
      if (lane == 0) S.warp_first[warp] = __float_as_uint(some);
      __syncthreads();
      some = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) some += __uint_as_float(S.warp_first[w]);
      far = logf(1.25f * static_cast<float>(a.vocab) / ((1.0f - R.p) * fmaxf(some, 1.0f))) + 0.01f;
      if (far > 26.f) far = kFar;  // beyond, the weights' rounding counts
    }
    // Small weights have no high word but a carry: the sums of a vector are
    // asked for together and looked at after.
    return pass(
        [&](int, const float(&)[kVN], const float(&d)[kVN], const uint32_t(&w)[kVN]) {
          uint32_t old[kVN];
          bool carry = false;
#pragma unroll
          for (int j = 0; j < kVN; ++j) old[j] = d[j] < far ? atomicAdd(&S.lo[bin_of(d[j])], w[j]) : 0u;
#pragma unroll
          for (int j = 0; j < kVN; ++j) carry |= d[j] < far && old[j] + w[j] < old[j];
          if (carry) {
#pragma unroll
            for (int j = 0; j < kVN; ++j)
              if (d[j] < far && old[j] + w[j] < old[j]) atomicAdd(&S.hi[bin_of(d[j])], 1u);
          }
        },
        [&](int, int, float, float d, u64 w) {
          if (d < far) count_step(bin_of(near(d)), w, false, true);
        });
  };
  // What min-p leaves may lie before the cut at p as a whole, and then p cuts
  // nothing of it: its mass is looked at first.
  const bool steps_of_all = cut_p && !cut_k;
  const bool floor_counts = !greedy && !cut_k && R.least > 1;
  if (a.logprobs || !cut_k) {
    u64 sum = 0, kept = 0;
    uint32_t first = 0xFFFFFFFFu;
    if (k_last >= 0) {
      const float bound = fminf(static_cast<float>(k_last + 1) / kBinsPerNat, kFar);
      auto each = [&](int i, int j, float, float d, u64 w) {
        if (d < bound && w && bin_of(near(d)) <= k_last) list_key(order_key(near(d), begin + i * kVN + j));
      };
      sum = pass(
          [&](int i, const float(&l)[kVN], const float(&d)[kVN], const uint32_t(&w)[kVN]) {
            float least = d[0];
#pragma unroll
            for (int j = 1; j < kVN; ++j) least = fminf(least, d[j]);
            if (least < bound) {  // rare: one test a vector
#pragma unroll
              for (int j = 0; j < kVN; ++j) each(i, j, l[j], d[j], w[j]);
            }
          },
          each);
    } else if (greedy) {
      auto each = [&](int i, int j, float l, float, u64) {
        if (l >= m && i < v1) first = min(first, static_cast<uint32_t>(begin + i * kVN + j));
      };
      sum = pass(same(each), each);
      first = __reduce_min_sync(0xffffffffu, first);
    } else if (floor_counts) {
      auto each = [&](int, int, float, float, u64 w) { kept += w >= R.least ? w : 0; };
      sum = pass(same(each), each);
    } else if (steps_of_all) {
      sum = pass_steps();
    } else {
      sum = pass([](int, const float(&)[kVN], const float(&)[kVN], const uint32_t(&)[kVN]) {},
                 [](int, int, float, float, u64) {});
    }
    kept = floor_counts ? warp_sum(kept) : sum;
    if (lane == 0) {
      S.warp_total[warp] = sum;
      S.warp_kept[warp] = kept;
      if (greedy) S.warp_first[warp] = first;
    }
  } else {
    if (lane == 0) S.warp_total[warp] = 0;
    if (k_last >= 0) collect(k_last, none, [](float, u64) { return true; });
  }
  __syncthreads();
  if (warp == 0) {
    const u64 tot = warp_sum(lane < kWarps ? S.warp_total[lane] : 0);
    const u64 kep = floor_counts ? warp_sum(lane < kWarps ? S.warp_kept[lane] : 0) : tot;
    const uint32_t fir = greedy ? __reduce_min_sync(0xffffffffu, lane < kWarps ? S.warp_first[lane] : 0xFFFFFFFFu) : 0;
    if (lane < nc) {
      peer_st(peer(&S.total[rank], lane), tot);
      peer_st(peer(&S.kept[rank], lane), kep);
      if (greedy) peer_st(peer(&S.first[rank], lane), fir);
    }
  }
  u64 listed = 0;
  if (k_last >= 0)
    listed = ship();
  else
    cluster_sync(nc);
  u64 total = 0;
  for (int c = 0; c < nc; ++c) total += S.total[c];
  if (steps_of_all && floor_counts) {
    u64 kept = 0;
    for (int c = 0; c < nc; ++c) kept += S.kept[c];
    if (kept <= mass_limit(R.p, total)) {
      cut_p = false;
    } else {
      pass_steps();
      cluster_sync(nc);
    }
  }
  auto answer = [&](uint32_t index, float d) {
    a.tokens[r] = index;
    if (a.logprobs)
      a.logprobs[r] = -d - logf(static_cast<float>(static_cast<double>(total) / static_cast<double>(kOne)));
  };
  if (greedy) {
    if (rank == 0 && t == 0) {
      u64 first = ~0ull;
      for (int c = 0; c < nc; ++c) first = min(first, S.first[c]);
      answer(static_cast<uint32_t>(first), 0.f);
    }
    return;
  }

  auto sort_by_key = [&](int len) {
    int pow2 = 2;
    while (pow2 < len) pow2 <<= 1;
    for (int i = len + t; i < pow2; i += kThreads) S.list[i] = ~0ull;
    __syncthreads();
    sort_list(S.list, pow2);
  };
  // Exclusive running sum over the list of the values of entries 2t and 2t + 1.
  auto list_scan = [&](u64 x0, u64 x1, u64 &b0, u64 &b1, u64 &all) {
    const u64 inc = warp_scan(x0 + x1, lane);
    if (lane == 31) S.red[warp] = inc;
    __syncthreads();
    b0 = inc - x0 - x1;
    all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) b0 += S.red[w];
      all += S.red[w];
    }
    b1 = b0 + x0;
    __syncthreads();
  };
  // For lists of at most kFew keys: four threads an entry (entry t / 4) count
  // the keys before it and add their weights, `total_w` those of all.
  constexpr int kPer = kThreads / kFew;
  auto rank_few = [&](int len, u64 key, u64 *before_w, u64 *total_w) -> int {
    int before = 0;
    u64 w = 0, all = 0;
    for (int i = t % kPer; i < len; i += kPer) {
      const bool less = S.list[i] < key;
      const u64 wi = S.few[0][i];
      before += less;
      w += less ? wi : 0;
      all += wi;
    }
#pragma unroll
    for (int o = 1; o < kPer; o <<= 1) {
      before += __shfl_xor_sync(0xffffffffu, before, o);
      w += __shfl_xor_sync(0xffffffffu, w, o);
      all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    *before_w = w;
    *total_w = all;
    return before;
  };
  // First CTA: all three cuts and the choice, from the list (which holds at
  // least every token that step 1 keeps).
  auto finish_list = [&](int len, u64 keep_n, bool by_p) {
    if (len <= kFew) {
      for (int i = t; i < len; i += kThreads) S.few[0][i] = weight(key_dist(S.list[i]));
      __syncthreads();
      const int e = t / kPer;
      const u64 key = e < len ? S.list[e] : ~0ull;
      u64 before, all, w = e < len ? S.few[0][e] : 0;
      const int place = rank_few(len, key, &before, &all);
      if (static_cast<u64>(place) >= keep_n) w = 0;
      if (by_p) {
        // The mass of the first keep_n.
        if (static_cast<u64>(place) == min(keep_n, static_cast<u64>(len)) - 1 && t % kPer == 0 && e < len)
          S.pick = before + S.few[0][e];
        __syncthreads();
        if (before >= mass_limit(R.p, S.pick)) w = 0;
      }
      if (w < R.least) w = 0;
      if (t % kPer == 0 && e < len) S.few[1][e] = w;
      __syncthreads();
      // The running mass in the order of the indices.
      u64 run = 0, mass = 0;
      const uint32_t index = key_index(key);
      for (int i = t % kPer; i < len; i += kPer) {
        const u64 wi = S.few[1][i];
        mass += wi;
        run += key_index(S.list[i]) < index ? wi : 0;
      }
#pragma unroll
      for (int o = 1; o < kPer; o <<= 1) {
        run += __shfl_xor_sync(0xffffffffu, run, o);
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
      }
      const u64 target = draw_target(R.u, mass);
      if (t % kPer == 0 && w && run <= target && target < run + w) answer(index, key_dist(key));
      return;
    }
    sort_by_key(len);
    const int i0 = 2 * t, i1 = 2 * t + 1;
    const u64 k0 = i0 < len ? S.list[i0] : ~0ull, k1 = i1 < len ? S.list[i1] : ~0ull;
    u64 w0 = i0 < len && static_cast<u64>(i0) < keep_n ? weight(key_dist(k0)) : 0;
    u64 w1 = i1 < len && static_cast<u64>(i1) < keep_n ? weight(key_dist(k1)) : 0;
    u64 b0, b1, all;
    list_scan(w0, w1, b0, b1, all);
    if (by_p) {
      const u64 limit = mass_limit(R.p, all);
      if (b0 >= limit) w0 = 0;
      if (b1 >= limit) w1 = 0;
    }
    if (w0 < R.least) w0 = 0;
    if (w1 < R.least) w1 = 0;
    const u64 target = draw_target(R.u, sum_block(w0 + w1, S.red));
    // What is kept, by index: index above |z|'s bits.
    auto flip = [](u64 key) { return (static_cast<u64>(key_index(key)) << 32) | (key >> kIndexBits); };
    int pow2 = 2;
    while (pow2 < len) pow2 <<= 1;
    if (i0 < pow2) S.list[i0] = w0 ? flip(k0) : ~0ull;
    if (i1 < pow2) S.list[i1] = w1 ? flip(k1) : ~0ull;
    __syncthreads();
    sort_list(S.list, pow2);
    const u64 f0 = i0 < pow2 ? S.list[i0] : ~0ull, f1 = i1 < pow2 ? S.list[i1] : ~0ull;
    w0 = f0 != ~0ull ? weight(__uint_as_float(static_cast<uint32_t>(f0))) : 0;
    w1 = f1 != ~0ull ? weight(__uint_as_float(static_cast<uint32_t>(f1))) : 0;
    list_scan(w0, w1, b0, b1, all);
    if (w0 && b0 <= target && target < b0 + w0)
      answer(static_cast<uint32_t>(f0 >> 32), __uint_as_float(static_cast<uint32_t>(f0)));
    if (w1 && b1 <= target && target < b1 + w1)
      answer(static_cast<uint32_t>(f1 >> 32), __uint_as_float(static_cast<uint32_t>(f1)));
  };
  // The key of the last token a cut keeps, when it falls into step c.bin: the
  // first at which the count (mass) reaches `want`; `mass` gets what is kept in
  // all, S.warp_kept what min-p leaves of it in each warp's part.  Steps with
  // more tokens than the list are divided 2^11-fold by key until they fit.
  auto settle = [&](Cut c, bool by_mass, u64 want, u64 limit_key, bool masses, u64 *mass) -> u64 {
    const int bin = static_cast<int>(c.bin);
    u64 lo = order_key(fmaxf(static_cast<float>(bin - 2), 0.f) / kBinsPerNat, 0);
    u64 width = order_key(static_cast<float>(bin + 2) / kBinsPerNat, 0) - lo;
    auto in_reach = [&](float d, u64 key) {
      return bin_of(d) == bin && key <= limit_key && key >= lo && key - lo < width;
    };
    int len;
    for (;;) {
      if (t == 0) S.list_n = 0, S.local_n = 0;
      cluster_sync(nc);
      collect(
          bin,
          [&](float d, u64 key) {
            const int b = bin_of(d);
            return b < bin || (b == bin && key < lo);
          },
          in_reach);
      const u64 found = ship();
      len = static_cast<int>(found);
      if (found <= kList) break;
      int shift = 0;
      while ((width >> shift) > static_cast<u64>(kBins - 1)) ++shift;
      cluster_sync(nc);
      clear_steps();
      __syncthreads();
      for (int i = v0 + lane; i < v1; i += 32) {
        const V v = at(i);
#pragma unroll
        for (int j = 0; j < kVN; ++j) {
          float d = dist(v.v[j], m, R.inv_t);
          if (!(d < kFar)) continue;
          d = near(d);
          const u64 key = order_key(d, begin + i * kVN + j);
          if (!in_reach(d, key)) continue;
          const u64 w = weight(d);
          if (w) count_step(static_cast<int>((key - lo) >> shift), w, !by_mass, masses);
        }
      }
      const u64 cb = c.count_before, mb = c.mass_before;
      cluster_sync(nc);
      gather_bins(masses);
      c = find(by_mass, want - (by_mass ? mb : cb));
      c.count_before += cb;
      c.mass_before += mb;
      lo += c.bin << shift;
      width = u64(1) << shift;
    }
    if (rank == 0) {
      const u64 left = want - (by_mass ? c.mass_before : c.count_before);  // at least 1
      auto tell = [&](u64 key, u64 through) {
        for (int x = 0; x < nc; ++x) {
          peer_st(peer(&S.pick, x), key);
          peer_st(peer(&S.cut.mass, x), c.mass_before + through);
        }
      };
      // A kept token of the list joins the sum of the warp that holds it.
      auto keep = [&](u64 key, u64 w) {
        if (w < R.least) return;
        const int index = static_cast<int>(key_index(key)), cta = index / slice;
        const int its = static_cast<int>(min(static_cast<int64_t>(slice), a.vocab - static_cast<int64_t>(cta) * slice));
        const int vecs = (its + kVN - 1) / kVN, vec = (index - cta * slice) / kVN;
        int w16 = static_cast<int>(static_cast<int64_t>(vec) * kWarps / vecs);
        while (static_cast<int>(static_cast<int64_t>(vecs) * (w16 + 1) / kWarps) <= vec) ++w16;
        peer_add64(peer(&S.warp_kept[w16], cta), w);
      };
      if (len <= kFew) {
        for (int i = t; i < len; i += kThreads) S.few[0][i] = weight(key_dist(S.list[i]));
        __syncthreads();
        const int e = t / kPer;
        const u64 key = e < len ? S.list[e] : ~0ull, w = e < len ? S.few[0][e] : 0;
        u64 before, all;
        const int place = rank_few(len, key, &before, &all);
        if (t % kPer == 0 && e < len &&
            (by_mass ? before < left && left <= before + w : static_cast<u64>(place + 1) == left))
          tell(key, before + w);
        if (t % kPer == 0 && e < len && (by_mass ? before < left : static_cast<u64>(place) < left)) keep(key, w);
      } else {
        sort_by_key(len);
        const u64 k0 = 2 * t < len ? S.list[2 * t] : ~0ull, k1 = 2 * t + 1 < len ? S.list[2 * t + 1] : ~0ull;
        const u64 w0 = 2 * t < len ? weight(key_dist(k0)) : 0, w1 = 2 * t + 1 < len ? weight(key_dist(k1)) : 0;
        u64 b0, b1, all;
        list_scan(w0, w1, b0, b1, all);
        if (by_mass ? (w0 && b0 < left && left <= b0 + w0) : static_cast<u64>(2 * t + 1) == left) tell(k0, b0 + w0);
        if (by_mass ? (w1 && b1 < left && left <= b1 + w1) : static_cast<u64>(2 * t + 2) == left) tell(k1, b1 + w1);
        if (w0 && (by_mass ? b0 < left : static_cast<u64>(2 * t) < left)) keep(k0, w0);
        if (w1 && (by_mass ? b1 < left : static_cast<u64>(2 * t + 1) < left)) keep(k1, w1);
      }
    }
    cluster_sync(nc);
    *mass = S.cut.mass;
    return S.pick;
  };

  u64 cut = ~0ull;
  if (cut_k) {
    if (k_last >= 0 && listed <= kList) {
      if (rank == 0) finish_list(static_cast<int>(listed), static_cast<u64>(R.k), cut_p);
      return;
    }
    // Too many, or k above the number of threads: the steps of all tokens.
    cluster_sync(nc);
    clear_steps();
    if (t == 0) S.list_n = 0, S.local_n = 0;
    __syncthreads();
    u64 all = 0;
    for (int i = v0 + lane; i < v1; i += 32) {
      const V v = at(i);
#pragma unroll
      for (int j = 0; j < kVN; ++j) {
        const float d = dist(v.v[j], m, R.inv_t);
        const u64 w = weight(d);
        all += w;
        if (w) count_step(bin_of(near(d)), w, true, cut_p);
      }
    }
    all = sum_block(all, S.red);
    if (t < nc) peer_st(peer(&S.total[rank], t), all);
    cluster_sync(nc);
    total = 0;
    for (int c = 0; c < nc; ++c) total += S.total[c];
  }
  if (cut_k || cut_p) {
    gather_bins(cut_p);
    u64 mk = total;
    const uint32_t c0 = pre_c;
    const u64 m0 = pre_m;
    uint32_t bc0[4];
    u64 bm0[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) bc0[j] = bc[j], bm0[j] = bm[j];
    if (cut_k && static_cast<u64>(R.k) < counted()) {
      const Cut c = find(false, static_cast<u64>(R.k));
      cut = settle(c, false, static_cast<u64>(R.k), ~0ull, cut_p, &mk);
    }
    if (cut_p) {
      const u64 limit = mass_limit(R.p, mk);
      pre_c = c0;
      pre_m = m0;
#pragma unroll
      for (int j = 0; j < 4; ++j) bc[j] = bc0[j], bm[j] = bm0[j];
      cluster_sync(nc);  // S.cut has been read by all
      const Cut c = find(true, limit);
      u64 unused;
      cut = settle(c, true, limit, cut, true, &unused);
    }
  }

  // ---- what is kept, in place: its mass a warp, and the walk ----
  auto kept = [&](float l, int index, float *dd) -> u64 {
    const float d = dist(l, m, R.inv_t);
    const u64 w = weight(d);  // 0 of a NaN
    *dd = near(d);
    return w >= R.least && order_key(near(d), index) <= cut ? w : 0;
  };
  float d;
  if (cut_k || cut_p) {
    // (k may have had nothing to cut, and then there was no pass for it.)
    if (cut == ~0ull) {
      u64 mine = 0;
      for (int i = v0 + lane; i < v1; i += 32) {
        const V v = at(i);
#pragma unroll
        for (int j = 0; j < kVN; ++j) mine += kept(v.v[j], begin + i * kVN + j, &d);
      }
      mine = warp_sum(mine);
      if (lane == 0) S.warp_kept[warp] = mine;
      __syncthreads();
    }
    if (t < nc) {
      u64 all = 0;
      for (int w = 0; w < kWarps; ++w) all += S.warp_kept[w];
      peer_st(peer(&S.kept[rank], t), all);
    }
    cluster_sync(nc);
  }
  u64 base = 0, mass = 0;  // what is kept before this CTA, and in all
  for (int c = 0; c < nc; ++c) {
    if (c < rank) base += S.kept[c];
    mass += S.kept[c];
  }
  const u64 target = draw_target(R.u, mass);
  if (target < base || target >= base + S.kept[rank]) return;  // (the same for the whole CTA)
  // The warp's part in which the target falls, walked by all warps, a vector a
  // thread and round.  (By its own warp, 25 reads from L2 one after the other
  // took as long as the pass before.)
  int part = 0;
  for (; part < kWarps - 1; ++part) {
    if (target < base + S.warp_kept[part]) break;
    base += S.warp_kept[part];
  }
  const int p1 = static_cast<int>(static_cast<int64_t>(nvec) * (part + 1) / kWarps);
  for (int p0 = static_cast<int>(static_cast<int64_t>(nvec) * part / kWarps); p0 < p1; p0 += kThreads) {
    const int i = p0 + t;
    u64 own = 0;
    if (i < p1) {
      const V v = at(i);
#pragma unroll
      for (int j = 0; j < kVN; ++j) own += kept(v.v[j], begin + i * kVN + j, &d);
    }
    const u64 through = warp_scan(own, lane);
    __syncthreads();  // S.red
    if (lane == 31) S.red[warp] = through;
    __syncthreads();
    u64 here = base + through - own;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const u64 all = S.red[w];
      if (w < warp) here += all;
      base += all;
    }
    if (own && here <= target && target < here + own) {
      const V v = at(i);
#pragma unroll
      for (int j = 0; j < kVN; ++j) {
        const u64 w = kept(v.v[j], begin + i * kVN + j, &d);
        if (w && here <= target && target < here + w) answer(begin + i * kVN + j, d);
        here += w;
      }
    }
    if (base > target) break;
  }
}

constexpr int kSampleSmemMax = 226 * 1024;  // (and a little static)

// Shared memory of a CTA whose slice holds `slice` logits of `size` bytes.
size_t sample_smem(int64_t slice, int size) {
  return (sizeof(SampleShared) + 15) / 16 * 16 + static_cast<size_t>(slice * size + 15) / 16 * 16;
}

template <int DT, bool kHeld>
int launch_cluster(const SampleArgs &a, int nc, int64_t slice, size_t smem, cudaStream_t s) {
  constexpr auto kernel = sample_cluster_kernel<DT, kHeld>;
  H24_CUDA_TRY(allow_smem<kernel>(kSampleSmemMax));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(a.rows * nc));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(nc);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = nc > 1 ? 2 : 1;
  H24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, nc, static_cast<int>(slice)));
  count_launches(1);
  return H24_OK;
}

template <int DT>
int launch_sample_typed(const SampleArgs &a, cudaStream_t s) {
  const int size = DT == H24_DTYPE_F32 ? 4 : 2;
  if (a.rows > INT32_MAX / kMaxCluster) return fail(H24_ERR_INVALID, "sample_tokens: too many rows");
  // Clusters where the rows' CTAs are no more than the SMs, with slices of at least
  // 1,024 logits.  (What fits at once is less: 15 clusters of eight and 36 of four,
  // so 16 to 18 rows, and 37, take a second wave: [15,50688] fp32, p = 0.9: 21 us,
  // [16,50688] 39, [19,50688] 23.)  Rows enough for the SMs by
  // themselves, or too long for a cluster, run a CTA a row that reads it from
  // L2 in each pass ([512,50688] fp32, p = 0.9: 127 us, in clusters of four 275;
  // [64,50688] bf16, p = 0.95: 60 us, in clusters of two 36; [1,50688] fp32,
  // k = 50: 15.6 us, in a cluster of eight 10.9).  A slice of fp32 logits fits up
  // to 42,700 of them: [74,50688] fp32, p = 0.9, in clusters of two 30 us, [75,50688]
  // by a CTA a row 46, [147,50688] 52; [64,131072] 75; one row of 600,001 254.
  int nc = kMaxCluster;
  while (nc > 1 && (a.rows * nc > 148 || a.vocab < 1024 * nc)) nc /= 2;
  const int64_t slice = ((a.vocab + nc - 1) / nc + 15) / 16 * 16;
  if (a.rows >= 148 || sample_smem(slice, size) > kSampleSmemMax) {
    SampleArgs b = a;
    // Two CTAs an SM are there at once.  (Up to 8,192 rows: every CTA counts the settings of all.)
    b.sorted = a.rows > 296 && a.rows <= 8192 && (a.top_k || a.top_p || a.temperature);
    return launch_cluster<DT, false>(b, 1, a.vocab, sample_smem(0, size), s);
  }
  return launch_cluster<DT, true>(a, nc, slice, sample_smem(slice, size), s);
}

}  // namespace

int launch_sample(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const float *u,
                  const float *temperature, float temperature1, const int32_t *top_k, int32_t top_k1,
                  const float *top_p, float top_p1, const float *min_p, float min_p1, int64_t *tokens,
                  float *logprobs, cudaStream_t s) {
  const SampleArgs a{logits, rows, vocab, stride, u, temperature, top_k, top_p, min_p, temperature1, top_p1, min_p1,
                     top_k1, tokens, logprobs, false};
  switch (dtype) {
    case H24_DTYPE_F32: return launch_sample_typed<H24_DTYPE_F32>(a, s);
    case H24_DTYPE_F16: return launch_sample_typed<H24_DTYPE_F16>(a, s);
    default: return launch_sample_typed<H24_DTYPE_BF16>(a, s);
  }
}

}  // namespace h24
