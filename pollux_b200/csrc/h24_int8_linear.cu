// h24_int8_linear.cu -- product of int8 activations with an INT8 layer:
//   y[t][o] = (sum_k q[t][k] * W[o][k]) * scale[t] * fp16(mu16[o] / 127) + bias[o]
// The sum is exact in int32 (in_features is bounded so that it cannot
// overflow), the scaling is fp32 and y is rounded once.  The weight's scale
// is the one PackedInt8Linear.materialize uses (pollux.py:545-554).
#include "h24_internal.cuh"

namespace h24 {
namespace {

constexpr int kTile = 64, kKStep = 64;  // 64 tokens x 64 outputs, 64 k a step
constexpr int kThreads = 256;

struct LinArgs {
  const int8_t *q;
  const float *scale;
  const int8_t *w;
  const uint16_t *mu16;
  const float *bias;
  void *y;
  int64_t tokens, q_stride, out, in;
  int out_dtype;
};

// The layer's reconstruction scale of one output row.
__device__ __forceinline__ float weight_scale(const uint16_t *mu16, int64_t o) {
  return __half2float(__float2half_rn(__fdiv_rn(__half2float(__ushort_as_half(__ldg(mu16 + o))), 127.0f)));
}

__device__ __forceinline__ void store_y(void *y, int dtype, int64_t i, float v) {
  if (dtype == H24_DTYPE_F32)
    static_cast<float *>(y)[i] = v;
  else if (dtype == H24_DTYPE_F16)
    static_cast<__half *>(y)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16 *>(y)[i] = __float2bfloat16_rn(v);
}

// A block owns 64 x 64 outputs, a thread 4 x 4 of them; both operands pass
// through shared memory as bytes and are multiplied four at a time.
__global__ void __launch_bounds__(kThreads) int8_linear_simple_kernel(const LinArgs a) {
  __shared__ int8_t sq[kTile][kKStep + 4], sw[kTile][kKStep + 4];
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
  const int64_t o0 = static_cast<int64_t>(blockIdx.x) * kTile, t0 = static_cast<int64_t>(blockIdx.y) * kTile;
  int acc[4][4] = {};
  for (int64_t k0 = 0; k0 < a.in; k0 += kKStep) {
    for (int i = t; i < kTile * kKStep; i += kThreads) {
      const int r = i / kKStep, c = i % kKStep;
      const bool k_in = k0 + c < a.in;
      sq[r][c] = k_in && t0 + r < a.tokens ? a.q[(t0 + r) * a.q_stride + k0 + c] : int8_t(0);
      sw[r][c] = k_in && o0 + r < a.out ? a.w[(o0 + r) * a.in + k0 + c] : int8_t(0);
    }
    __syncthreads();
    for (int c = 0; c < kKStep; c += 4)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[i][j] = __dp4a(*reinterpret_cast<const int *>(&sq[ty + 16 * i][c]),
                             *reinterpret_cast<const int *>(&sw[tx + 16 * j][c]), acc[i][j]);
    __syncthreads();
  }
  for (int j = 0; j < 4; ++j) {
    const int64_t o = o0 + tx + 16 * j;
    if (o >= a.out) continue;
    const float ws = weight_scale(a.mu16, o), b = a.bias ? a.bias[o] : 0.f;
    for (int i = 0; i < 4; ++i) {
      const int64_t tok = t0 + ty + 16 * i;
      if (tok < a.tokens)
        store_y(a.y, a.out_dtype, tok * a.out + o, static_cast<float>(acc[i][j]) * a.scale[tok] * ws + b);
    }
  }
}

}  // namespace

int launch_int8_linear(const Tables *, const int8_t *q, const float *scale, int64_t tokens, int64_t q_stride,
                       const int8_t *w, const uint16_t *mu16, int64_t out, int64_t in, const float *bias,
                       int out_dtype, void *y, cudaStream_t s) {
  const LinArgs a{q, scale, w, mu16, bias, y, tokens, q_stride, out, in, out_dtype};
  for (int64_t t0 = 0; t0 < tokens; t0 += 65535LL * kTile) {
    LinArgs b = a;
    b.tokens = tokens - t0 < 65535LL * kTile ? tokens - t0 : 65535LL * kTile;
    b.q = q + t0 * q_stride;
    b.scale = scale + t0;
    b.y = static_cast<uint8_t *>(y) + t0 * out * (out_dtype == H24_DTYPE_F32 ? 4 : 2);
    int8_linear_simple_kernel<<<dim3(static_cast<unsigned>((out + kTile - 1) / kTile),
                                     static_cast<unsigned>((b.tokens + kTile - 1) / kTile)),
                                kThreads, 0, s>>>(b);
    H24_CUDA_TRY(cudaGetLastError());
    count_launches(1);
  }
  return H24_OK;
}

}  // namespace h24
