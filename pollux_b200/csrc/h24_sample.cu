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
// "z descending, index ascending" is one 64-bit key: |z|'s bits above the
// index (z <= 0, so |z| ascending is z descending, and the bits of
// non-negative floats ascend with them).  A selection is then a cut on that
// key, found by histograms of its digits.
#include "h24_internal.cuh"

namespace h24 {
namespace {

constexpr float kOne = 1099511627776.0f;  // 2^40
constexpr int kSampleThreads = 1024;

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
};

template <int DT>
__device__ __forceinline__ float logit_at(const void *row, int64_t i) {
  float v;
  if (DT == H24_DTYPE_F32)
    v = __ldg(static_cast<const float *>(row) + i);
  else if (DT == H24_DTYPE_F16)
    v = __half2float(static_cast<const __half *>(row)[i]);
  else
    v = __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[i]);
  return v == v ? v : -INFINITY;  // NaN: never chosen
}

// |z| of a logit.
__device__ __forceinline__ float dist(float l, float m, float inv_t) {
  return l == m ? 0.f : fabsf(__fmul_rn(__fsub_rn(l, m), inv_t));
}

__device__ __forceinline__ unsigned long long weight(float d) {
  return static_cast<unsigned long long>(__float2ll_rn(expf(-d) * kOne));
}

__device__ __forceinline__ unsigned long long order_key(float d, int64_t i) {
  return (static_cast<unsigned long long>(__float_as_uint(d)) << 32) | static_cast<unsigned long long>(i);
}

// What step 2 and 3 ask for, in the arithmetic the header states.
__device__ __forceinline__ unsigned long long mass_limit(float p, unsigned long long mk) {
  const double x = ceil(static_cast<double>(p) * static_cast<double>(mk));
  return x > 1.0 ? static_cast<unsigned long long>(x) : 1ull;
}
__device__ __forceinline__ unsigned long long weight_floor(float min_p) {
  const double x = ceil(fmin(fmax(static_cast<double>(min_p), 0.0), 1.0) * static_cast<double>(kOne));
  return x > 1.0 ? static_cast<unsigned long long>(x) : 1ull;  // weight 0 is never chosen
}
__device__ __forceinline__ unsigned long long draw_target(float u, unsigned long long mass) {
  const double x = floor((u > 0.f ? static_cast<double>(u) : 0.0) * static_cast<double>(mass));
  return x >= static_cast<double>(mass - 1) ? mass - 1 : static_cast<unsigned long long>(x);
}

__device__ unsigned long long block_sum(unsigned long long v, unsigned long long *red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long r = 0;
  for (int w = 0; w < kSampleThreads / 32; ++w) r += red[w];
  __syncthreads();
  return r;
}

// A block per row; every step reads the row again.
template <int DT>
__global__ void __launch_bounds__(kSampleThreads) sample_rows_kernel(const SampleArgs a) {
  __shared__ unsigned long long hist[256], red[32], sh_digit, sh_left;
  __shared__ float redf[32];
  const int t = threadIdx.x;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const uint8_t *row = static_cast<const uint8_t *>(a.logits) + r * a.stride * (DT == H24_DTYPE_F32 ? 4 : 2);
    float temp = a.temperature ? a.temperature[r] : a.temperature1;
    int64_t k = a.top_k ? a.top_k[r] : a.top_k1;
    const float p = a.top_p ? a.top_p[r] : a.top_p1;
    const float min_p = a.min_p ? a.min_p[r] : a.min_p1;
    if (!(temp > 0.f)) temp = 1.f, k = 1;
    const float inv_t = __fdiv_rn(1.0f, temp);
    float m = -INFINITY;
    for (int64_t i = t; i < a.vocab; i += kSampleThreads) m = fmaxf(m, logit_at<DT>(row, i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((t & 31) == 0) redf[t >> 5] = m;
    __syncthreads();
    for (int w = 0; w < kSampleThreads / 32; ++w) m = fmaxf(m, redf[w]);
    __syncthreads();
    if (m == -INFINITY) {  // nothing to choose from
      if (t == 0) {
        a.tokens[r] = -1;
        if (a.logprobs) a.logprobs[r] = -INFINITY;
      }
      continue;
    }
    unsigned long long sum = 0;
    for (int64_t i = t; i < a.vocab; i += kSampleThreads) sum += weight(dist(logit_at<DT>(row, i), m, inv_t));
    const unsigned long long total = block_sum(sum, red);

    // The key of the last element kept: the first at which the count (by_mass
    // false) or the mass of the order up to and with it reaches `want`, among
    // keys <= cut.
    unsigned long long cut = ~0ull;
    auto select = [&](bool by_mass, unsigned long long want) {
      unsigned long long prefix = 0, left = want;
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = t; i < 256; i += kSampleThreads) hist[i] = 0;
        __syncthreads();
        for (int64_t i = t; i < a.vocab; i += kSampleThreads) {
          const float d = dist(logit_at<DT>(row, i), m, inv_t);
          const unsigned long long key = order_key(d, i);
          if (key <= cut && (shift == 56 || (key >> (shift + 8)) == prefix))
            atomicAdd(&hist[(key >> shift) & 255], by_mass ? weight(d) : 1ull);
        }
        __syncthreads();
        if (t == 0) {
          int b = 0;
          unsigned long long l = left;
          while (b < 255 && hist[b] < l) l -= hist[b++];
          sh_digit = b;
          sh_left = l;
        }
        __syncthreads();
        prefix = (prefix << 8) | sh_digit;
        left = sh_left;
        __syncthreads();
      }
      cut = prefix;
    };
    unsigned long long mk = total;
    if (k > 0 && k < a.vocab) {
      select(false, static_cast<unsigned long long>(k));
      sum = 0;
      for (int64_t i = t; i < a.vocab; i += kSampleThreads) {
        const float d = dist(logit_at<DT>(row, i), m, inv_t);
        if (order_key(d, i) <= cut) sum += weight(d);
      }
      mk = block_sum(sum, red);
    }
    if (p < 1.f) select(true, mass_limit(p, mk));
    const unsigned long long least = weight_floor(min_p);
    auto kept = [&](int64_t i) -> unsigned long long {
      const float d = dist(logit_at<DT>(row, i), m, inv_t);
      const unsigned long long w = weight(d);
      return order_key(d, i) <= cut && w >= least ? w : 0ull;
    };
    sum = 0;
    for (int64_t i = t; i < a.vocab; i += kSampleThreads) sum += kept(i);
    const unsigned long long target = draw_target(a.u[r], block_sum(sum, red));
    // The running mass, a block's width of indices at a time.
    unsigned long long base = 0;
    for (int64_t i0 = 0; i0 < a.vocab; i0 += kSampleThreads) {
      const int64_t i = i0 + t;
      const unsigned long long w = i < a.vocab ? kept(i) : 0ull;
      unsigned long long run = w;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long up = __shfl_up_sync(0xffffffffu, run, o);
        if ((t & 31) >= o) run += up;
      }
      if ((t & 31) == 31) red[t >> 5] = run;
      __syncthreads();
      unsigned long long before = base, all = base;
      for (int j = 0; j < kSampleThreads / 32; ++j) {
        if (j < (t >> 5)) before += red[j];
        all += red[j];
      }
      run += before;
      if (w && run > target && run - w <= target) {
        a.tokens[r] = i;
        if (a.logprobs)
          a.logprobs[r] = -dist(logit_at<DT>(row, i), m, inv_t) -
                          logf(static_cast<float>(static_cast<double>(total) / static_cast<double>(kOne)));
      }
      base = all;
      __syncthreads();
      if (base > target) break;
    }
    __syncthreads();
  }
}

}  // namespace

int launch_sample(const void *logits, int dtype, int64_t rows, int64_t vocab, int64_t stride, const float *u,
                  const float *temperature, float temperature1, const int32_t *top_k, int32_t top_k1,
                  const float *top_p, float top_p1, const float *min_p, float min_p1, int64_t *tokens,
                  float *logprobs, cudaStream_t s) {
  const SampleArgs a{logits, rows, vocab, stride, u, temperature, top_k, top_p, min_p, temperature1, top_p1, min_p1,
                     top_k1, tokens, logprobs};
  const int grid = wave_grid(rows, 2);
  switch (dtype) {
    case H24_DTYPE_F32: sample_rows_kernel<H24_DTYPE_F32><<<grid, kSampleThreads, 0, s>>>(a); break;
    case H24_DTYPE_F16: sample_rows_kernel<H24_DTYPE_F16><<<grid, kSampleThreads, 0, s>>>(a); break;
    default: sample_rows_kernel<H24_DTYPE_BF16><<<grid, kSampleThreads, 0, s>>>(a); break;
  }
  H24_CUDA_TRY(cudaGetLastError());
  count_launches(1);
  return H24_OK;
}

}  // namespace h24
