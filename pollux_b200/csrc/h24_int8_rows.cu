// h24_int8_rows.cu -- activations in 8 bits: residual addition, RMS norm and
// quantisation of each row to int8 with one fp32 scale, and the way back.
//
//   s_c    = x_c + r_c                                  fp32 (residual_out = s rounded to x's type)
//   v_c    = s_c * g_c,  m = max_c |v_c|                fp32
//   i      = 1 / sqrt(mean_c(s_c^2) + eps)              fp32
//   mu     = max(m * i, fp32(1e-8)),  scale = mu / 127  fp32
//   q_c    = clamp(rint(v_c * (i * 127 / mu)), -128, 127)
// Quantisation alone takes v = x and i = 1.  A NaN in a row (or an infinite
// element under the norm) makes its scale NaN and every q 0, as the row
// quantiser of the weights does.  The norm is taken of the unrounded sum.
#include "h24_internal.cuh"

namespace h24 {
namespace {

constexpr float kRowEps = 1e-8f;  // smallest mu, as for the weights (pack.py:124-136)
constexpr int kRowThreads = 256;

template <int DT>
struct Elem;
template <>
struct Elem<H24_DTYPE_F32> {
  using T = float;
  static __device__ __forceinline__ float up(float v) { return v; }
  static __device__ __forceinline__ float down(float v) { return v; }
};
template <>
struct Elem<H24_DTYPE_F16> {
  using T = __half;
  static __device__ __forceinline__ float up(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half down(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<H24_DTYPE_BF16> {
  using T = __nv_bfloat16;
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

// rint(v * k) as int8; NaN gives 0.
__device__ __forceinline__ int8_t quant_act(float v, float k) {
  const float t = v * k;
  return t != t ? int8_t(0) : static_cast<int8_t>(static_cast<int>(fminf(fmaxf(rintf(t), -128.0f), 127.0f)));
}

// One block per row, two passes over it.
template <int DT, bool kNorm>
__global__ void __launch_bounds__(kRowThreads) rows_int8_kernel(const RowArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float red[2][kRowThreads / 32];
  pdl_enter();
  const int t = threadIdx.x;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
    const T *res = a.residual ? static_cast<const T *>(a.residual) + r * a.residual_stride : nullptr;
    auto gain = [&](int64_t c) {
      return a.gain_f32 ? static_cast<const float *>(a.gain)[c] : E::up(static_cast<const T *>(a.gain)[c]);
    };
    float ss = 0.f, m = 0.f;
    for (int64_t c = t; c < a.cols; c += kRowThreads) {
      float s = E::up(x[c]);
      if (kNorm) {
        if (res) s += E::up(res[c]);
        ss = fmaf(s, s, ss);
        m = nan_max(m, fabsf(s * gain(c)));
      } else {
        m = nan_max(m, fabsf(s));
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ss += __shfl_xor_sync(0xffffffffu, ss, o);
      m = nan_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    }
    if ((t & 31) == 0) red[0][t >> 5] = ss, red[1][t >> 5] = m;
    __syncthreads();
    ss = 0.f, m = 0.f;
    for (int w = 0; w < kRowThreads / 32; ++w) ss += red[0][w], m = nan_max(m, red[1][w]);
    __syncthreads();
    const float inv = kNorm ? 1.0f / sqrtf(ss / static_cast<float>(a.cols) + a.eps) : 1.0f;
    float mu = m * inv;
    mu = mu != mu ? mu : fmaxf(mu, kRowEps);
    const float k = inv * (127.0f / mu);
    for (int64_t c = t; c < a.cols; c += kRowThreads) {
      float s = E::up(x[c]);
      if (kNorm) {
        if (res) s += E::up(res[c]);
        if (a.residual_out) static_cast<T *>(a.residual_out)[r * a.cols + c] = E::down(s);
        s *= gain(c);
      }
      a.q[r * a.cols + c] = quant_act(s, k);
    }
    if (t == 0) a.scale[r] = mu / 127.0f;
  }
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads) rows_dequant_kernel(const int8_t *__restrict__ q,
                                                                   const float *__restrict__ scale, int64_t rows,
                                                                   int64_t cols, void *out) {
  using E = Elem<DT>;
  pdl_enter();
  const int64_t total = rows * cols, stride = static_cast<int64_t>(gridDim.x) * kRowThreads;
  for (int64_t i = blockIdx.x * static_cast<int64_t>(kRowThreads) + threadIdx.x; i < total; i += stride)
    static_cast<typename E::T *>(out)[i] = E::down(static_cast<float>(q[i]) * scale[i / cols]);
}

template <int DT, bool kNorm>
int launch_rows(const RowArgs &a, cudaStream_t s) {
  const int grid = wave_grid(a.rows, blocks_per_sm(rows_int8_kernel<DT, kNorm>, kRowThreads, 0));
  H24_CUDA_TRY(launch_pdl(rows_int8_kernel<DT, kNorm>, dim3(grid), dim3(kRowThreads), s, a));
  count_launches(1);
  return H24_OK;
}

}  // namespace

int launch_rows_int8(const void *x, const void *residual, const void *gain, int gain_dtype, int64_t rows,
                     int64_t cols, int64_t x_stride, int64_t residual_stride, int dtype, float eps, int8_t *q,
                     float *scale, void *residual_out, cudaStream_t s) {
  const RowArgs a{x, residual, gain, rows, cols, x_stride, residual_stride, eps,
                  gain_dtype == H24_DTYPE_F32, q, scale, residual_out};
  const bool norm = gain != nullptr;
  switch (dtype) {
    case H24_DTYPE_F32: return norm ? launch_rows<H24_DTYPE_F32, true>(a, s) : launch_rows<H24_DTYPE_F32, false>(a, s);
    case H24_DTYPE_F16: return norm ? launch_rows<H24_DTYPE_F16, true>(a, s) : launch_rows<H24_DTYPE_F16, false>(a, s);
    default: return norm ? launch_rows<H24_DTYPE_BF16, true>(a, s) : launch_rows<H24_DTYPE_BF16, false>(a, s);
  }
}

int launch_rows_dequant(const int8_t *q, const float *scale, int64_t rows, int64_t cols, int dtype, void *out,
                        cudaStream_t s) {
  const int grid = wave_grid((rows * cols + kRowThreads - 1) / kRowThreads, 8);
  const auto kernel = dtype == H24_DTYPE_F32   ? rows_dequant_kernel<H24_DTYPE_F32>
                      : dtype == H24_DTYPE_F16 ? rows_dequant_kernel<H24_DTYPE_F16>
                                               : rows_dequant_kernel<H24_DTYPE_BF16>;
  H24_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kRowThreads), s, q, scale, rows, cols, out));
  count_launches(1);
  return H24_OK;
}

}  // namespace h24
