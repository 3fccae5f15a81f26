// h24_int8_rows.cu -- activations in 8 bits: residual addition, RMS norm and
// quantisation of each row to int8 with one fp32 scale, and the way back.
//
//   s_c    = x_c + r_c                                  fp32 (residual_out = s rounded to x's type)
//   v_c    = s_c * g_c,  m = max_c |v_c|                fp32
//   i      = 1 / sqrt(mean_c(s_c^2) + eps)              fp32
//   mu     = max(m * i, fp32(1e-8)),  scale = mu / 127  fp32
//   q_c    = rint(v_c * (i * 127 / mu))                 within [-127, 127]
// Quantisation alone takes v = x and i = 1.  A NaN in a row (or an infinite
// element under the norm) makes its scale NaN and every q 0, as the row
// quantiser of the weights does.  The norm is taken of the unrounded sum.  Where
// the sum of squares passes fp32's range (an element above 1.8e19), it is taken
// again of s * 2^-80: see wide_factor.
//
// Bound by HBM where there are rows: 7 bytes an element in bf16 (x, r, r', q).
// On a B200, a call among others: [4096,1920] bf16 10.1 us (5.5 TB/s, 0.83 of
// the measured copy rate), [4096,7680] 37.1 (5.9, 0.91; fp16 44.0), [4096,1920]
// fp32 15.8 (6.5, 0.99); one row 2.1 us, a launch's latency.  Rows off 16 bytes
// are read and written by the element, which costs a sector each time:
// [4096,1919] bf16 38.9 us, [2028,841] 11.3.  Rows of 16,385 to 65,536 elements
// of 16 bits do not fit the registers (see the kernel): [512,32768] bf16 92 us
// for 117 MB, [512,65536] 182 for 235.  The way back: 4.9 us for [4096,1920] to
// bf16, its int8 rows still in L2.
#include "h24_internal.cuh"

namespace h24 {
namespace {

constexpr float kRowEps = 1e-8f;  // smallest mu, as for the weights (pack.py:124-136)
constexpr float kSmall = 8.271806125530277e-25f;  // 2^-80
constexpr int kDeqThreads = 256;

template <int DT>
struct Elem;
template <>
struct Elem<H24_DTYPE_F32> {
  using T = float;
  static constexpr int kVec = 4;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<H24_DTYPE_F16> {
  using T = __half;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<H24_DTYPE_BF16> {
  using T = __nv_bfloat16;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float up(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 down(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ float nan_max(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct RowArgs {
  const void *x;
  const void *residual;
  const void *gain;
  int64_t rows, cols, x_stride, residual_stride;
  float eps;
  bool gain_f32;
  int8_t *q;
  float *scale;
  void *residual_out;
};

// rint(v * k), |v * k| below 2^22, in the low byte: adding 1.5 * 2^23 leaves the
// integer, rounded to nearest even, in the low bits of the sum.  One fused
// multiply-add an element, where a rounding and a conversion instruction each
// run at an eighth of its rate.
__device__ __forceinline__ uint32_t quant_act(float v, float k) {
  return __float_as_uint(fmaf(v, k, 12582912.0f));
}

// The value of one row's partial (sum of squares, largest magnitude) over a
// block of `warps` warps.
__device__ __forceinline__ void reduce_row(float &ss, float &m, float (*red)[32], int warps) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    ss += __shfl_xor_sync(0xffffffffu, ss, o);
    m = nan_max(m, __shfl_xor_sync(0xffffffffu, m, o));
  }
  if (warps == 1) return;
  const int t = threadIdx.x;
  if ((t & 31) == 0) red[0][t >> 5] = ss, red[1][t >> 5] = m;
  __syncthreads();
  ss = 0.f;
  m = 0.f;
  for (int w = 0; w < warps; ++w) ss += red[0][w], m = nan_max(m, red[1][w]);
}

// mu / 127 and the factor that takes v to q, from a row's sums.  |v * factor|
// is at most 127 (1 + 2^-21), which rounds to 127: q needs no clamp.  A row
// whose mu is not finite has every q 0: `dead`.  A sum of squares that is not
// finite makes mu NaN (ss - ss; it is 0 of any other).
template <bool kNorm>
__device__ __forceinline__ float row_factor(const RowArgs &a, float ss, float m, float *scale, bool *dead) {
  const float inv = kNorm ? 1.0f / sqrtf(ss / static_cast<float>(a.cols) + a.eps) : 1.0f;
  float mu = kNorm ? fmaf(m, inv, ss - ss) : m;
  mu = mu != mu ? mu : fmaxf(mu, kRowEps);
  *scale = mu / 127.0f;
  *dead = !(mu <= 3.402823466e38f);
  return inv * (127.0f / mu);
}

// The same for a finite row whose squares pass fp32's range, from big, the sum of
// (s * 2^-80)^2.  That cannot overflow, and what underflows in it is below a
// rounding of such a sum.  inv is i * 2^80, since i itself may be too small a
// number; q takes v to 127 v / m, without i, unless mu is at its floor.
__device__ __forceinline__ float wide_factor(const RowArgs &a, float big, float m, float *scale) {
  const float inv = 1.0f / sqrtf(big / static_cast<float>(a.cols) + a.eps * kSmall * kSmall);
  const float mu = fmaxf(m * kSmall * inv, kRowEps);
  *scale = mu / 127.0f;
  return mu > kRowEps ? 127.0f / m : inv * (127.0f / kRowEps) * kSmall;
}
__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// The elements of a 16-byte group as fp32.
template <int DT>
__device__ __forceinline__ void widen(uint4 raw, float (&v)[Elem<DT>::kVec]) {
  using E = Elem<DT>;
  alignas(16) typename E::T x[E::kVec];
  *reinterpret_cast<uint4 *>(x) = raw;
#pragma unroll
  for (int j = 0; j < E::kVec; ++j) v[j] = E::up(x[j]);
}

// The block's finite rows among those that rows_int8_kernel gave a NaN scale,
// read again by the element.  Where the sum was written over x or the residual,
// it stands for them, in 16 bits rounded.
template <int DT>
__device__ __noinline__ void wide_rows(const RowArgs &a, float (*red)[32]) {
  using E = Elem<DT>;
  using T = typename E::T;
  const bool over = a.residual_out && (a.residual_out == a.x || a.residual_out == a.residual);
  auto sum_at = [&](int64_t r, int64_t c) {
    if (over) return E::up(static_cast<const T *>(a.residual_out)[r * a.cols + c]);
    const float s = E::up(static_cast<const T *>(a.x)[r * a.x_stride + c]);
    return a.residual ? s + E::up(static_cast<const T *>(a.residual)[r * a.residual_stride + c]) : s;
  };
  auto gain = [&](int64_t c) {
    return a.gain_f32 ? static_cast<const float *>(a.gain)[c] : E::up(static_cast<const T *>(a.gain)[c]);
  };
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const float marked = a.scale[r];
    if (marked == marked) continue;
    float big = 0.f, m = 0.f;
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x) {
      const float s = sum_at(r, c);
      big = fmaf(s * kSmall, s * kSmall, big);
      m = nan_max(m, fabsf(s * gain(c)));
    }
    __syncthreads();  // all have read the mark, and what red held
    reduce_row(big, m, red, blockDim.x >> 5);
    if (!finite(big) || !finite(m)) continue;  // (the same for the whole block)
    float scale;
    const float k = wide_factor(a, big, m, &scale);
    for (int64_t c = threadIdx.x; c < a.cols; c += blockDim.x)
      a.q[r * a.cols + c] = static_cast<int8_t>(quant_act(sum_at(r, c) * gain(c), k));
    if (threadIdx.x == 0) a.scale[r] = scale;
  }
}

// Thread t of a block holds the 16-byte groups t, t + blockDim.x, ... (at most
// NV) of its row in registers, so the row is read once.  (For NV = 8 the 1,024
// threads' registers are too few, and part of the row goes through local memory:
// ptxas reports 1.6 KB of spill stores a thread in bf16, 0.6 in fp32.)  A block
// walks rows r, r + gridDim.x, ..., and asks for the next row before it reduces
// the present one.  Rows that are not 16-byte
// aligned, or end inside a group, are read and written by the element in the
// same groups: a row's result does not depend on where it lies.
template <int DT, bool kAligned, int NV, bool kNorm>
__global__ void __launch_bounds__(NV < 8 ? 512 : 1024) rows_int8_kernel(const __grid_constant__ RowArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VEC = E::kVec;
  __shared__ float red[2][2][32];
  pdl_enter();
  const int t = threadIdx.x, nt = blockDim.x;
  const int cols = static_cast<int>(a.cols);
  const bool has_res = kNorm && a.residual != nullptr;
  uint4 raw[NV], raw_res[NV];
  auto ask = [&](int64_t r) {
    if (!kAligned || r >= a.rows) return;
    const uint4 *x = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.x) + r * a.x_stride);
    const uint4 *res = reinterpret_cast<const uint4 *>(static_cast<const T *>(a.residual) + r * a.residual_stride);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if ((t + i * nt) * VEC < cols) {
        raw[i] = x[t + i * nt];
        if (has_res) raw_res[i] = res[t + i * nt];
      }
  };
  ask(blockIdx.x);
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    float v[NV][VEC];
    float ss = 0.f, m = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (t + i * nt) * VEC;
      if (at >= cols) continue;
      if (kAligned) {
        widen<DT>(raw[i], v[i]);
        if (has_res) {
          float s[VEC];
          widen<DT>(raw_res[i], s);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] += s[j];
        }
      } else {
        const T *x = static_cast<const T *>(a.x) + r * a.x_stride + at;
        const T *res = static_cast<const T *>(a.residual) + r * a.residual_stride + at;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          v[i][j] = at + j < cols ? E::up(x[j]) : 0.f;
          if (has_res && at + j < cols) v[i][j] += E::up(res[j]);
        }
      }
    }
    ask(r + gridDim.x);
    T *sum_out = static_cast<T *>(a.residual_out) + r * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (t + i * nt) * VEC;
      if (at >= cols) continue;
      if (kNorm && a.residual_out) {
        alignas(16) T o[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) o[j] = E::down(v[i][j]);
        if (kAligned) {
          *reinterpret_cast<uint4 *>(sum_out + at) = *reinterpret_cast<const uint4 *>(o);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (at + j < cols) sum_out[at + j] = o[j];
        }
      }
      if (kNorm) {
        float g[VEC];
        if (DT != H24_DTYPE_F32 && a.gain_f32) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            g[j] = kAligned || at + j < cols ? __ldg(static_cast<const float *>(a.gain) + at + j) : 0.f;
        } else if (kAligned) {
          widen<DT>(__ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(a.gain) + at)), g);
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) g[j] = at + j < cols ? E::up(static_cast<const T *>(a.gain)[at + j]) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ss = fmaf(v[i][j], v[i][j], ss);
          v[i][j] *= g[j];
        }
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) m = nan_max(m, fabsf(v[i][j]));
    }
    reduce_row(ss, m, red[turn], nt >> 5);
    float scale;
    bool dead;
    const float k = row_factor<kNorm>(a, ss, m, &scale, &dead);
    int8_t *q = a.q + r * a.cols;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (t + i * nt) * VEC;
      if (at >= cols) continue;
      if (kAligned) {
        uint32_t w[VEC / 4];
#pragma unroll
        for (int j = 0; j < VEC; j += 4)
          w[j / 4] = dead ? 0u
                          : __byte_perm(__byte_perm(quant_act(v[i][j], k), quant_act(v[i][j + 1], k), 0x0040),
                                        __byte_perm(quant_act(v[i][j + 2], k), quant_act(v[i][j + 3], k), 0x0040),
                                        0x5410);
        if constexpr (VEC == 8)
          *reinterpret_cast<uint2 *>(q + at) = make_uint2(w[0], w[1]);
        else
          *reinterpret_cast<uint32_t *>(q + at) = w[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at + j < cols) q[at + j] = dead ? int8_t(0) : static_cast<int8_t>(quant_act(v[i][j], k));
      }
    }
    if (t == 0) a.scale[r] = scale;
  }
  // Rows that look like NaN are looked at here, outside the loop: a test and a
  // second sum inside it took [4096,7680] bf16 from 36.6 us to 44 and more (this:
  // 37.1).  The squares of fp16 cannot overflow.
  if (kNorm && DT != H24_DTYPE_F16) {
    bool marked = false;
    __syncthreads();
    for (int64_t r = blockIdx.x + static_cast<int64_t>(t) * gridDim.x; r < a.rows;
         r += static_cast<int64_t>(nt) * gridDim.x)
      marked |= a.scale[r] != a.scale[r];
    if (__syncthreads_or(marked)) wide_rows<DT>(a, red[0]);
  }
}

constexpr int kLongThreads = 512;

// Rows too long for the registers of a block: two passes over the row.
template <int DT, bool kNorm>
__global__ void __launch_bounds__(kLongThreads) rows_int8_long_kernel(const RowArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float red[2][32];
  pdl_enter();
  const int t = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + r * a.residual_stride : nullptr;
  auto gain = [&](int64_t c) {
    return a.gain_f32 ? static_cast<const float *>(a.gain)[c] : E::up(static_cast<const T *>(a.gain)[c]);
  };
  float ss = 0.f, m = 0.f;
  for (int64_t c = t; c < a.cols; c += kLongThreads) {
    float s = E::up(x[c]);
    if (kNorm) {
      if (res) s += E::up(res[c]);
      ss = fmaf(s, s, ss);
      m = nan_max(m, fabsf(s * gain(c)));
    } else {
      m = nan_max(m, fabsf(s));
    }
  }
  reduce_row(ss, m, red, kLongThreads / 32);
  float scale;
  bool dead;
  float k = row_factor<kNorm>(a, ss, m, &scale, &dead);
  if (kNorm && !finite(ss) && finite(m)) {  // (the same for the whole block)
    float big = 0.f, unused = 0.f;
    for (int64_t c = t; c < a.cols; c += kLongThreads) {
      const float s = (E::up(x[c]) + (res ? E::up(res[c]) : 0.f)) * kSmall;
      big = fmaf(s, s, big);
    }
    __syncthreads();  // red has been read
    reduce_row(big, unused, red, kLongThreads / 32);
    if (finite(big)) {
      k = wide_factor(a, big, m, &scale);
      dead = false;
    }
  }
  for (int64_t c = t; c < a.cols; c += kLongThreads) {
    float s = E::up(x[c]);
    if (kNorm) {
      if (res) s += E::up(res[c]);
      if (a.residual_out) static_cast<T *>(a.residual_out)[r * a.cols + c] = E::down(s);
      s *= gain(c);
    }
    a.q[r * a.cols + c] = dead ? int8_t(0) : static_cast<int8_t>(quant_act(s, k));
  }
  if (t == 0) a.scale[r] = scale;
}

constexpr int kDeqUnroll = 4;

// Groups of 16 output bytes of the flat array, kDeqUnroll in flight a thread
// (a warp's store covers whole sectors: two groups a thread side by side wrote
// half sectors and ran at 4.5 TB/s).  kInRow: cols is a multiple of a group, so
// its elements share a row.
template <int DT, bool kInRow>
__global__ void __launch_bounds__(kDeqThreads) rows_dequant_kernel(const int8_t *__restrict__ q,
                                                                   const float *__restrict__ scale, int64_t total,
                                                                   int64_t cols, typename Elem<DT>::T *out) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VEC = E::kVec;
  pdl_enter();
  const int64_t nvec = total / VEC, step = static_cast<int64_t>(gridDim.x) * kDeqThreads * kDeqUnroll;
  const bool narrow = total <= 0xFFFFFFFFll;
  for (int64_t i0 = blockIdx.x * static_cast<int64_t>(kDeqThreads) * kDeqUnroll + threadIdx.x; i0 < nvec; i0 += step) {
    uint32_t raw[kDeqUnroll][VEC / 4];
    float s[kDeqUnroll];
    int64_t row[kDeqUnroll];
#pragma unroll
    for (int u = 0; u < kDeqUnroll; ++u) {
      const int64_t i = i0 + u * kDeqThreads;
      if (i >= nvec) continue;
      if constexpr (VEC == 8) {
        const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(q) + i);
        raw[u][0] = w.x;
        raw[u][1] = w.y;
      } else {
        raw[u][0] = __ldcs(reinterpret_cast<const uint32_t *>(q) + i);
      }
      row[u] = narrow ? static_cast<uint32_t>(i * VEC) / static_cast<uint32_t>(cols) : i * VEC / cols;
      s[u] = __ldg(scale + row[u]);
    }
#pragma unroll
    for (int u = 0; u < kDeqUnroll; ++u) {
      const int64_t i = i0 + u * kDeqThreads;
      if (i >= nvec) continue;
      int64_t left = (row[u] + 1) * cols - i * VEC;  // elements of the row from here
      alignas(16) T o[VEC];
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (!kInRow && left-- == 0) {
          s[u] = __ldg(scale + ++row[u]);
          left = cols - 1;
        }
        const int8_t b = static_cast<int8_t>(raw[u][j / 4] >> (8 * (j % 4)));
        o[j] = E::down(static_cast<float>(b) * s[u]);
      }
      __stcs(reinterpret_cast<uint4 *>(out) + i, *reinterpret_cast<const uint4 *>(o));
    }
  }
  if (blockIdx.x == 0 && threadIdx.x < total % VEC) {
    const int64_t i = nvec * VEC + threadIdx.x;
    out[i] = E::down(static_cast<float>(q[i]) * scale[i / cols]);
  }
}

template <int DT, bool kAligned, int NV, bool kNorm>
int launch_rows_kernel(const RowArgs &a, int threads, cudaStream_t s) {
  constexpr auto kernel = rows_int8_kernel<DT, kAligned, NV, kNorm>;
  H24_CUDA_TRY(launch_pdl(kernel, dim3(wave_grid(a.rows, blocks_per_sm_once<kernel>(threads))), dim3(threads), s, a));
  count_launches(1);
  return H24_OK;
}

template <int DT, bool kNorm, int NV>
int launch_rows_nv(const RowArgs &a, bool aligned, int threads, cudaStream_t s) {
  return aligned ? launch_rows_kernel<DT, true, NV, kNorm>(a, threads, s)
                 : launch_rows_kernel<DT, false, NV, kNorm>(a, threads, s);
}

template <int DT, bool kNorm>
int launch_rows(const RowArgs &a, cudaStream_t s) {
  constexpr int kVec = Elem<DT>::kVec;
  const bool aligned = a.cols % kVec == 0 && a.x_stride % kVec == 0 && a.residual_stride % kVec == 0 &&
                       aligned16(a.x) && aligned16(a.residual) && aligned16(a.residual_out) && aligned16(a.gain) &&
                       (reinterpret_cast<uintptr_t>(a.q) & 7) == 0;
  const int64_t nvec = (a.cols + kVec - 1) / kVec;
  // Two groups a thread, more where a row needs over 512 threads.  One group
  // runs [1,1920] bf16 in 1.82 us instead of 2.08 but [4096,1920] in 13.3
  // instead of 10.5.  The number of rows has no say, so that a row's sum is
  // the same in every batch.
  for (int nv = 2; nv <= 8; nv *= 2) {
    const int64_t threads = nvec == 0 ? 32 : ((nvec + nv - 1) / nv + 31) / 32 * 32;
    if (threads > (nv < 8 ? 512 : 1024)) continue;
    switch (nv) {
      case 2: return launch_rows_nv<DT, kNorm, 2>(a, aligned, static_cast<int>(threads), s);
      case 4: return launch_rows_nv<DT, kNorm, 4>(a, aligned, static_cast<int>(threads), s);
      default: return launch_rows_nv<DT, kNorm, 8>(a, aligned, static_cast<int>(threads), s);
    }
  }
  H24_CUDA_TRY(launch_pdl(rows_int8_long_kernel<DT, kNorm>, dim3(static_cast<unsigned>(a.rows)), dim3(kLongThreads), s, a));
  count_launches(1);
  return H24_OK;
}

template <int DT>
int launch_dequant_rows(const int8_t *q, const float *scale, int64_t total, int64_t cols, void *out, cudaStream_t s) {
  constexpr int kPerBlock = Elem<DT>::kVec * kDeqThreads * kDeqUnroll;
  const int grid = wave_grid((total + kPerBlock - 1) / kPerBlock, 8);
  const auto kernel = cols % Elem<DT>::kVec == 0 ? rows_dequant_kernel<DT, true> : rows_dequant_kernel<DT, false>;
  H24_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kDeqThreads), s, q, scale, total, cols,
                          static_cast<typename Elem<DT>::T *>(out)));
  count_launches(1);
  return H24_OK;
}

}  // namespace

int launch_rows_int8(const void *x, const void *residual, const void *gain, int gain_dtype, int64_t rows,
                     int64_t cols, int64_t x_stride, int64_t residual_stride, int dtype, float eps, int8_t *q,
                     float *scale, void *residual_out, cudaStream_t s) {
  const RowArgs a{x, residual, gain, rows, cols, x_stride, residual_stride, eps,
                  gain_dtype == H24_DTYPE_F32, q, scale, residual_out};
  const bool norm = gain != nullptr && cols > 0;  // (rows without elements: the scale of zeros)
  switch (dtype) {
    case H24_DTYPE_F32: return norm ? launch_rows<H24_DTYPE_F32, true>(a, s) : launch_rows<H24_DTYPE_F32, false>(a, s);
    case H24_DTYPE_F16: return norm ? launch_rows<H24_DTYPE_F16, true>(a, s) : launch_rows<H24_DTYPE_F16, false>(a, s);
    default: return norm ? launch_rows<H24_DTYPE_BF16, true>(a, s) : launch_rows<H24_DTYPE_BF16, false>(a, s);
  }
}

int launch_rows_dequant(const int8_t *q, const float *scale, int64_t rows, int64_t cols, int dtype, void *out,
                        cudaStream_t s) {
  const int64_t total = rows * cols;
  switch (dtype) {
    case H24_DTYPE_F32: return launch_dequant_rows<H24_DTYPE_F32>(q, scale, total, cols, out, s);
    case H24_DTYPE_F16: return launch_dequant_rows<H24_DTYPE_F16>(q, scale, total, cols, out, s);
    default: return launch_dequant_rows<H24_DTYPE_BF16>(q, scale, total, cols, out, s);
  }
}

}  // namespace h24
