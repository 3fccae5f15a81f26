// h24_norm.cu -- RMS and layer norm of a residual stream, and their gradients.
//
//   s_c = x_c + r_c, rounded to x's type (what is handed on)
//   m   = mean(s) under the layer norm, 0 under the RMS norm
//   i   = 1 / sqrt(mean((s - m)^2) + eps),  n_c = (s_c - m) i
//   y_c = n_c w_c + b_c
// and back, with v_c = dy_c w_c:
//   ds_c = i (v_c - [layer] mean(v) - n_c mean(v n)) + dsummed_c
//   dw_c = sum over rows of dy_c n_c,  db_c = sum over rows of dy_c
// The norm is taken of the rounded sum, so that the gradients, which are taken
// of it too (the unrounded one is nowhere in memory), are those of what was
// computed.  Sums and statistics are fp32; deviations are squared, not squares
// subtracted.  Where the squares of a row of finite numbers pass fp32's range,
// its statistics are those of s * 2^-80, and i is stored negative to say so.
//
// A thread holds 8 or 16 columns of a row, so a row is read once; rows of up to
// 512 columns take a warp or a part of one, of up to 16,384 a block.  In the backward pass a thread
// keeps its columns for all of its rows and adds dw and db up in registers; the
// blocks' sums meet in a second kernel, in a fixed order.
//
// Bound by HBM where there are rows: forward and backward move 8 bytes an element
// each in bf16 (x, r, y, s; s, dy, dsummed, dx).  On a B200 [16384,1920] bf16
// with the RMS norm takes 40 us forward (6.4 TB/s, 0.97 of the measured copy rate)
// and 43 + 6 back (5.8); [8192,7680] with the layer norm 90 (5.6) and 95 + 6 (5.3).
// Rows off 16 bytes cost more instructions: [8838,6946] bf16 211 us forward and
// 165 + 6 back, where [8838,6944] takes 88 and 108 + 6 (read and written by the
// element, as up to 1,023 rows and those of more than 16,384 columns are, 740 us
// for both).
#include "h24_tile.cuh"

#include <type_traits>

namespace h24 {
namespace {

constexpr float kSmall = 8.271806125530277e-25f;  // 2^-80
constexpr int kHold = 16;                         // columns a thread holds
constexpr int kWarpCols = 32 * kHold;              // of a row that lanes of a warp hold
constexpr int kBlockCols = 1024 * kHold;
constexpr int kNarrowThreads = 256, kWarpRows = kNarrowThreads / 32;  // of a block with such rows
constexpr int kLongThreads = 512;
constexpr int kSumCols = 32;                      // of a block of the last sum

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

struct NormArgs {
  const void *x, *residual, *gain, *bias;
  int64_t rows, cols, x_stride, residual_stride;
  float eps;
  bool gain_f32;
  void *y, *summed;
  float *inv, *mean;  // of each row; mean: layer norm only
};

struct BackArgs {
  const void *s, *dy, *dsummed, *gain;
  int64_t rows, cols, s_stride, dy_stride, dsummed_stride;
  bool gain_f32;
  const float *inv, *mean;
  void *dx;
  float *dgain, *dbias;  // sums of each block, `cols` apart; either may be null
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) <= 3.402823466e38f; }

// Two columns at a time: one instruction for both, where the kernels were bound by
// their instructions ([16384,1920] bf16 42 and 49 us one by one, 40 and 43 in
// pairs; [8192,7680] with the layer norm 93 and 105, 90 and 95).
__device__ __forceinline__ float2 as_pair(uint64_t v) { return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32))); }
__device__ __forceinline__ uint64_t bits(float2 v) {
  return static_cast<uint64_t>(__float_as_uint(v.x)) | static_cast<uint64_t>(__float_as_uint(v.y)) << 32;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return as_pair(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
  return as_pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
  return as_pair(r);
}

// Two neighbouring elements, as words of memory.
template <int DT>
struct Pair;
template <>
struct Pair<H24_DTYPE_F32> {
  using W = uint64_t;
  static __device__ __forceinline__ float2 up(W w) { return as_pair(w); }
  static __device__ __forceinline__ W down(float2 v) { return bits(v); }
};
template <>
struct Pair<H24_DTYPE_F16> {
  using W = uint32_t;
  static __device__ __forceinline__ float2 up(W w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
  static __device__ __forceinline__ W down(float2 v) {
    const __half2 h = __float22half2_rn(v);
    return *reinterpret_cast<const W *>(&h);
  }
};
template <>
struct Pair<H24_DTYPE_BF16> {
  using W = uint32_t;
  static __device__ __forceinline__ float2 up(W w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ W down(float2 v) {
    const __nv_bfloat162 h = __float22bfloat162_rn(v);
    return *reinterpret_cast<const W *>(&h);
  }
};

// Thread t of a row's threads holds the columns of the vectors t, t + nt, ..., in pairs.
template <int DT, int HOLD = kHold>
struct Held {
  using W = typename Pair<DT>::W;
  static constexpr int VEC = Elem<DT>::kVec, NV = HOLD / VEC;
  uint4 raw[NV];

  template <bool kAligned>
  __device__ __forceinline__ void load(const void *base, int64_t offset, int t, int nt, int cols) {
    using T = typename Elem<DT>::T;
    const T *p = static_cast<const T *>(base) + offset;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = (t + i * nt) * VEC;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (kAligned) {
        if (at < cols) raw[i] = __ldg(reinterpret_cast<const uint4 *>(p + at));
      } else {
        T *e = reinterpret_cast<T *>(&raw[i]);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (at + j < cols) e[j] = p[at + j];
      }
    }
  }
  // The same columns of a row in shared memory.
  __device__ __forceinline__ void take(const uint8_t *row, int t, int nt, int cols) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      raw[i] = (t + i * nt) * VEC < cols ? *reinterpret_cast<const uint4 *>(row + (t + i * nt) * 16)
                                         : make_uint4(0, 0, 0, 0);
  }
  // The same of a row that lies `off` bytes into its place there.
  __device__ __forceinline__ void take_off(const uint8_t *row, uint32_t off, int t, int nt, int cols) {
    const uint4 *p = reinterpret_cast<const uint4 *>(row);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int at = t + i * nt, left = cols - at * VEC;
      raw[i] = make_uint4(0, 0, 0, 0);
      if (left >= VEC)
        raw[i] = join16(p[at], p[at + 1], off, 16);
      else if (left > 0)
        raw[i] = join16(p[at], p[at + 1], off, left * (16 / VEC));
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ float2 get(int k) const { return Pair<DT>::up(reinterpret_cast<const W *>(raw)[k]); }
};

// The held columns of a row to memory.
template <int DT, bool kAligned, int P>
__device__ __forceinline__ void store_held(void *base, int64_t offset, const float2 (&v)[P], int t, int nt, int cols) {
  using T = typename Elem<DT>::T;
  using W = typename Pair<DT>::W;
  constexpr int VEC = Elem<DT>::kVec;
  T *p = static_cast<T *>(base) + offset;
#pragma unroll
  for (int i = 0; i < 2 * P / VEC; ++i) {
    const int at = (t + i * nt) * VEC;
    alignas(16) W o[VEC / 2];
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) o[j] = Pair<DT>::down(v[i * VEC / 2 + j]);
    if (kAligned) {
      if (at < cols) *reinterpret_cast<uint4 *>(p + at) = *reinterpret_cast<const uint4 *>(o);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (at + j < cols) p[at + j] = reinterpret_cast<const T *>(o)[j];
    }
  }
}

// The same to a row anywhere: a lane puts the end of its neighbour's vector and
// the start of its own into one block of 16 bytes; what is left at the ends of a
// warp and of the row goes by the element.  For whole warps.
template <int DT, int P>
__device__ __forceinline__ void store_off(void *base, int64_t offset, const float2 (&v)[P], int t, int nt, int cols) {
  using T = typename Elem<DT>::T;
  using W = typename Pair<DT>::W;
  constexpr int VEC = Elem<DT>::kVec, SIZE = 16 / VEC;
  T *p = static_cast<T *>(base) + offset;
  const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15u);  // the same for all
  const int over = static_cast<int>(off) / SIZE, first = VEC - over;  // a vector's elements in the next block, in its own
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 2 * P / VEC; ++i) {
    const int at = t + i * nt, left = cols - at * VEC;
    alignas(16) W o[VEC / 2];
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) o[j] = Pair<DT>::down(v[i * VEC / 2 + j]);
    const uint4 mine = *reinterpret_cast<const uint4 *>(o);
    T *to = p + at * VEC;
    uint4 before;
    before.x = __shfl_up_sync(0xffffffffu, mine.x, 1);
    before.y = __shfl_up_sync(0xffffffffu, mine.y, 1);
    before.z = __shfl_up_sync(0xffffffffu, mine.z, 1);
    before.w = __shfl_up_sync(0xffffffffu, mine.w, 1);
    const bool whole = left >= first && (lane > 0 || over == 0);
    if (whole) *reinterpret_cast<uint4 *>(to - over) = over ? join16(before, mine, 16 - off, 16) : mine;
    const T *e = reinterpret_cast<const T *>(&mine);
    const bool tail = lane == 31 || left - VEC < first;  // the next block has no lane that writes it whole
#pragma unroll
    for (int j = 0; j < VEC; ++j)
      if (j < left && (j < first ? !whole : tail)) to[j] = e[j];
  }
}

// The held columns of a parameter vector as fp32 (0 past the end).
template <int DT, bool kAligned, int P>
__device__ __forceinline__ void load_param(const void *param, bool f32, float2 (&v)[P], int t, int nt, int cols) {
  constexpr int VEC = Elem<DT>::kVec;
  if (!f32 || DT == H24_DTYPE_F32) {
    Held<DT, 2 * P> h;
    h.template load<kAligned>(param, 0, t, nt, cols);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = h.get(k);
    return;
  }
  const float *p = static_cast<const float *>(param);
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const int at = (t + 2 * k / VEC * nt) * VEC + 2 * k % VEC;
    v[k] = make_float2(at < cols ? __ldg(p + at) : 0.f, at + 1 < cols ? __ldg(p + at + 1) : 0.f);
  }
}

// The mean off the held columns; past the row's end they stay 0.
template <int DT, int P>
__device__ __forceinline__ void center(float2 (&v)[P], float mean, int t, int nt, int cols) {
  constexpr int VEC = Elem<DT>::kVec;
#pragma unroll
  for (int i = 0; i < 2 * P / VEC; ++i) {
    const int left = cols - (t + i * nt) * VEC;  // columns of the vector that are there
    const float2 m = both(left > 0 ? -mean : 0.f);
#pragma unroll
    for (int j = 0; j < VEC / 2; ++j) {
      float2 &x = v[i * VEC / 2 + j];
      x = add2(x, m);
      if (left < VEC) {  // (rows that end inside a vector)
        if (2 * j >= left) x.x = 0.f;
        if (2 * j + 1 >= left) x.y = 0.f;
      }
    }
  }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Over each `lanes` neighbouring lanes, a power of two.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
#pragma unroll
  for (int o = 16; o; o >>= 1)
    if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sums over a row's threads: a warp, or the block (`red` is not used again
// before a barrier that all of its threads pass).  Each warp adds up the warps'
// sums across its lanes: one after the other they cost 30 reads of shared memory.
template <bool kWarp>
__device__ __forceinline__ float row_sum(float v, float *red) {
  v = warp_sum(v);
  if (kWarp) return v;
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_sum(lane < (blockDim.x >> 5) ? red[lane] : 0.f);
}
// Two sums over the block behind one barrier.
__device__ __forceinline__ void row_sums(float &v, float &w, float (*red)[32]) {
  v = warp_sum(v);
  w = warp_sum(w);
  const int lane = threadIdx.x & 31;
  if (lane == 0) red[0][threadIdx.x >> 5] = v, red[1][threadIdx.x >> 5] = w;
  __syncthreads();
  const bool live = lane < (blockDim.x >> 5);
  v = warp_sum(live ? red[0][lane] : 0.f);
  w = warp_sum(live ? red[1][lane] : 0.f);
}

// The finite rows among those whose statistics passed fp32's range, again and
// by the element, from s * 2^-80.  The block had `per_block` neighbours at a time.
template <int DT, bool kLayer, bool kWarp>
__device__ __noinline__ void wide_rows(const NormArgs &a, int per_block, float (*red)[32]) {
  using E = Elem<DT>;
  using T = typename E::T;
  const int t = kWarp ? threadIdx.x & 31 : threadIdx.x, nt = kWarp ? 32 : blockDim.x;
  auto param = [&](const void *p, int64_t c) {
    return a.gain_f32 ? static_cast<const float *>(p)[c] : E::up(static_cast<const T *>(p)[c]);
  };
  auto again = [&](int64_t r) {
    const float marked = a.inv[r];
    if (marked > 0.f && finite(marked)) return;
    const T *s = a.summed ? static_cast<const T *>(a.summed) + r * a.cols : static_cast<const T *>(a.x) + r * a.x_stride;
    float sum = 0.f, bad = 0.f;
    for (int64_t c = t; c < a.cols; c += nt) {
      const float v = E::up(s[c]);
      sum = fmaf(v, kSmall, sum);
      bad += finite(v) ? 0.f : 1.f;
    }
    sum = row_sum<kWarp>(sum, red[0]);
    bad = row_sum<kWarp>(bad, red[1]);
    if (bad == 0.f) {  // (the same for all threads of the row)
      const float mean = kLayer ? sum / static_cast<float>(a.cols) : 0.f;
      float ss = 0.f;
      for (int64_t c = t; c < a.cols; c += nt) {
        const float v = fmaf(E::up(s[c]), kSmall, -mean);
        ss = fmaf(v, v, ss);
      }
      ss = row_sum<kWarp>(ss, red[2]);
      const double var = static_cast<double>(ss) / static_cast<double>(a.cols);
      const float inv = static_cast<float>(1.0 / sqrt(var + static_cast<double>(a.eps) * kSmall * kSmall));
      for (int64_t c = t; c < a.cols; c += nt) {
        const float n = fmaf(E::up(s[c]), kSmall, -mean) * inv;
        static_cast<T *>(a.y)[r * a.cols + c] = E::down(fmaf(n, param(a.gain, c), a.bias ? param(a.bias, c) : 0.f));
      }
      if (!kWarp) __syncthreads();  // all have read the mark
      __syncwarp();
      if (t == 0) {
        a.inv[r] = -inv;
        if (kLayer) a.mean[r] = mean;
      }
    }
    if (!kWarp) __syncthreads();
  };
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * per_block; r0 < a.rows; r0 += static_cast<int64_t>(gridDim.x) * per_block)
    for (int i = kWarp ? threadIdx.x >> 5 : 0; i < per_block && r0 + i < a.rows; i += kWarp ? kWarpRows : 1) again(r0 + i);
}

// Rows off 16 bytes that do not come through the ring (ring_of_any_rows), by the element.
template <int DT, bool kLayer, int kMax, int HOLD>
__global__ void __launch_bounds__(kMax) norm_kernel(const __grid_constant__ NormArgs a) {
  __shared__ float red[2][3][32];
  pdl_enter();
  const int t = threadIdx.x, nt = blockDim.x;
  const int cols = static_cast<int>(a.cols);
  const int64_t first = blockIdx.x, step = gridDim.x;
  const float n_cols = static_cast<float>(cols);
  Held<DT, HOLD> x, res;
  auto ask = [&](int64_t r) {
    if (r >= a.rows) return;
    x.template load<false>(a.x, r * a.x_stride, t, nt, cols);
    if (a.residual) res.template load<false>(a.residual, r * a.residual_stride, t, nt, cols);
  };
  ask(first);
  int turn = 0;
  for (int64_t r = first; r < a.rows; r += step, turn ^= 1) {
    constexpr int P = HOLD / 2;
    float2 v[P];
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = x.get(k);
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = Pair<DT>::up(Pair<DT>::down(add2(v[k], res.get(k))));
    }
    ask(r + step);
    if (a.summed) store_held<DT, false>(a.summed, r * a.cols, v, t, nt, cols);
    float mean = 0.f;
    float2 sum = both(0.f), ss = both(0.f);
    if (kLayer) {
#pragma unroll
      for (int k = 0; k < P; ++k) sum = add2(sum, v[k]);
      mean = row_sum<false>(sum.x + sum.y, red[turn][0]) / n_cols;
      center<DT>(v, mean, t, nt, cols);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) ss = fma2(v[k], v[k], ss);
    const float var = row_sum<false>(ss.x + ss.y, red[turn][1]) / n_cols;
    const float inv = 1.0f / sqrtf(var + a.eps);
    float2 w[P];
    load_param<DT, false>(a.gain, a.gain_f32, w, t, nt, cols);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = mul2(v[k], both(inv));
    if (kLayer && a.bias) {
      float2 b[P];
      load_param<DT, false>(a.bias, a.gain_f32, b, t, nt, cols);
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = fma2(v[k], w[k], b[k]);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = mul2(v[k], w[k]);
    }
    store_held<DT, false>(a.y, r * a.cols, v, t, nt, cols);
    if (t == 0) {
      a.inv[r] = inv;
      if (kLayer) a.mean[r] = mean;
    }
  }
  // Rows that passed fp32's range are looked for here, outside the loop.  (The
  // squares of fp16 cannot.)
  if (DT != H24_DTYPE_F16) {
    bool marked = false;
    __syncthreads();
    for (int64_t r = first + t * step; r < a.rows; r += nt * step) marked |= !(a.inv[r] > 0.f && finite(a.inv[r]));
    if (__syncthreads_or(marked)) wide_rows<DT, kLayer, false>(a, 1, red[0]);
  }
}

// Rows of up to 512 columns: `lanes` lanes have a row and a warp 32 / lanes of
// them, so that no lane is left without columns ([1048576,64] bf16 55 us forward,
// 214 with a warp a row; both directions of a training step 150 and 628).  A lane
// holds 8, of rows of more than 256 columns 16.  The parameters stay in registers.
template <int DT, bool kAligned, bool kLayer, int HOLD>
__global__ void __launch_bounds__(kNarrowThreads) norm_narrow_kernel(const __grid_constant__ NormArgs a, int lanes) {
  __shared__ float red[3][32];
  pdl_enter();
  constexpr int P = HOLD / 2;
  const int t = threadIdx.x & (lanes - 1), cols = static_cast<int>(a.cols), per_block = kNarrowThreads / lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  const int mine = threadIdx.x / lanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block + mine;
  const int ahead = mine - (threadIdx.x & ~31) / lanes;  // of the warp's first row
  const float n_cols = static_cast<float>(cols);
  float2 w[P], b[P] = {};
  load_param<DT, kAligned>(a.gain, a.gain_f32, w, t, lanes, cols);
  if (kLayer && a.bias) load_param<DT, kAligned>(a.bias, a.gain_f32, b, t, lanes, cols);
  Held<DT, HOLD> x, res;
  auto ask = [&](int64_t r) {
    if (r >= a.rows) return;
    x.template load<kAligned>(a.x, r * a.x_stride, t, lanes, cols);
    if (a.residual) res.template load<kAligned>(a.residual, r * a.residual_stride, t, lanes, cols);
  };
  x.clear();
  res.clear();
  ask(first);
  for (int64_t r = first; r - ahead < a.rows; r += step) {  // (as often for the whole warp)
    float2 v[P];
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = x.get(k);
    if (a.residual) {
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = Pair<DT>::up(Pair<DT>::down(add2(v[k], res.get(k))));
    }
    ask(r + step);
    const bool live = r < a.rows;
    if (a.summed && live) store_held<DT, kAligned>(a.summed, r * a.cols, v, t, lanes, cols);
    float mean = 0.f;
    float2 sum = both(0.f), ss = both(0.f);
    if (kLayer) {
#pragma unroll
      for (int k = 0; k < P; ++k) sum = add2(sum, v[k]);
      mean = lanes_sum(sum.x + sum.y, lanes) / n_cols;
      center<DT>(v, mean, t, lanes, cols);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) ss = fma2(v[k], v[k], ss);
    const float var = lanes_sum(ss.x + ss.y, lanes) / n_cols;
    const float inv = 1.0f / sqrtf(var + a.eps);
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = mul2(v[k], both(inv));
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = kLayer && a.bias ? fma2(v[k], w[k], b[k]) : mul2(v[k], w[k]);
    if (!live) continue;
    store_held<DT, kAligned>(a.y, r * a.cols, v, t, lanes, cols);
    if (t == 0) {
      a.inv[r] = inv;
      if (kLayer) a.mean[r] = mean;
    }
  }
  if (DT != H24_DTYPE_F16) {  // as above
    bool marked = false;
    __syncthreads();
    for (int64_t r = first + t * step; r < a.rows; r += lanes * step) marked |= !(a.inv[r] > 0.f && finite(a.inv[r]));
    if (__syncthreads_or(marked)) wide_rows<DT, kLayer, true>(a, per_block, red);
  }
}

// ---------------------------------------------------------------------------
// Rows through a ring in shared memory
// ---------------------------------------------------------------------------
// Rows of 513 to 16,384 columns on 16 bytes: one thread keeps the next rows on
// their way (bulk copies into a ring of stages, each with a row of every input),
// so that the loads of a block do not wait for its sums.  A thread holds 8
// columns where a block then has at most 512 threads, else 16 (30 warps of 8
// columns spend more on a row's sums than on the row: [8192,7680] bf16 with the
// layer norm 104 and 117 us, 93 and 105 with 15 warps of 16).  Two rows at a
// time behind one barrier cost more registers than they save waits: 130 and 146.
// Before the ring, rows asked for one ahead in registers: 129 and 153, and
// [16384,1920] with the RMS norm 42 and 60, 42 and 49 with it.
constexpr int kFew = 8, kFewCols = 512 * kFew, kMaxRing = 8;
constexpr int kRingHead = 128;  // barriers
constexpr int kRingSmem = 220 * 1024;  // of an SM, for the rings of its blocks

struct Ring {
  uint8_t *rows;    // stage s, input i: rows + (s * inputs + i) * pitch
  uint64_t *full;
  int stages, inputs, pitch;
  uint32_t bytes;   // of a row
};

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(su32(dst)),
               "l"(src), "r"(bytes), "r"(su32(bar))
               : "memory");
}

struct RingInput {
  const uint8_t *base;
  int64_t stride;  // bytes
};
// Rows off 16 bytes (kOff) are copied with what stands around them in their first
// and last 16 bytes, the first row and the last one, around which nothing of the
// tensor may stand, not at all: the threads read these themselves.
__device__ __forceinline__ bool row_at_edge(int64_t r, int64_t rows) { return r == 0 || r + 1 == rows; }

// Row r of every input on its way to stage s, by one thread.
template <bool kOff, int N>
__device__ __forceinline__ void ring_ask(const Ring &g, const RingInput (&in)[N], int s, int64_t r, int64_t rows) {
  uint32_t total = g.inputs * g.bytes, size[N], off[N];
  if (kOff) {
    total = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      off[i] = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in[i].base + r * in[i].stride) & 15u);
      size[i] = (off[i] + g.bytes + 15u) & ~15u;
      if (i < g.inputs && !row_at_edge(r, rows)) total += size[i];
    }
  }
  bar_expect(&g.full[s], total);
  if (kOff && row_at_edge(r, rows)) return;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < g.inputs)
      bulk_load(g.rows + (s * g.inputs + i) * g.pitch, in[i].base + r * in[i].stride - (kOff ? off[i] : 0u),
                kOff ? size[i] : g.bytes, &g.full[s]);
}

// The columns of input i of the row that stage s holds.
template <bool kOff, int DT, int HOLD>
__device__ __forceinline__ void ring_take(Held<DT, HOLD> &h, const Ring &g, const RingInput &in, int s, int i, int64_t r,
                                          int64_t rows, int t, int nt, int cols) {
  const uint8_t *row = g.rows + (s * g.inputs + i) * g.pitch;
  if (!kOff)
    h.take(row, t, nt, cols);
  else if (row_at_edge(r, rows))
    h.template load<false>(in.base, r * in.stride / (16 / Elem<DT>::kVec), t, nt, cols);
  else
    h.take_off(row, static_cast<uint32_t>(reinterpret_cast<uintptr_t>(in.base + r * in.stride) & 15u), t, nt, cols);
}

// Bytes between a stage's rows.
__host__ __device__ __forceinline__ int ring_pitch(int64_t bytes, bool off) {
  return static_cast<int>((bytes + (off ? 48 : 0) + 127) / 128 * 128);
}

template <bool kOff, int N>
__device__ __forceinline__ Ring ring_start(uint8_t *smem, int stages, int inputs, int64_t cols, int size,
                                           const RingInput (&in)[N], int64_t rows) {
  Ring g;
  g.full = reinterpret_cast<uint64_t *>(smem);
  g.rows = smem + kRingHead;
  g.stages = stages;
  g.inputs = inputs;
  g.bytes = static_cast<uint32_t>(cols * size);
  g.pitch = ring_pitch(g.bytes, kOff);
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) bar_init(&g.full[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  pdl_enter();
  if (threadIdx.x == 0) {
    asm volatile("fence.proxy.async;" ::: "memory");  // the rows were written by ordinary stores
    for (int s = 0; s < stages && blockIdx.x + static_cast<int64_t>(s) * gridDim.x < rows; ++s)
      ring_ask<kOff>(g, in, s, blockIdx.x + static_cast<int64_t>(s) * gridDim.x, rows);
  }
  return g;
}

template <int DT, bool kLayer, int HOLD, int kMax, bool kOff>
__global__ void __launch_bounds__(kMax, 1024 / kMax) norm_ring_kernel(const __grid_constant__ NormArgs a, int stages, int *err) {
  extern __shared__ __align__(128) uint8_t norm_smem[];
  __shared__ float red[2][3][32];
  __shared__ int abort;
  constexpr int VEC = Elem<DT>::kVec, SIZE = 16 / VEC;
  const int t = threadIdx.x, nt = blockDim.x;
  const int cols = static_cast<int>(a.cols);
  const int64_t step = gridDim.x;
  const float n_cols = static_cast<float>(cols);
  if (t == 0) abort = 0;
  const RingInput in[2] = {{static_cast<const uint8_t *>(a.x), a.x_stride * SIZE},
                           {static_cast<const uint8_t *>(a.residual), a.residual_stride * SIZE}};
  const Ring g = ring_start<kOff>(norm_smem, stages, a.residual ? 2 : 1, a.cols, SIZE, in, a.rows);
  constexpr int P = HOLD / 2;
  float2 w[P], b[P] = {};
  load_param<DT, !kOff>(a.gain, a.gain_f32, w, t, nt, cols);
  if (kLayer && a.bias) load_param<DT, !kOff>(a.bias, a.gain_f32, b, t, nt, cols);
  int turn = 0, s = 0;
  uint32_t ph = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += step, turn ^= 1) {
    if (!bar_wait(&g.full[s], ph, &abort, err, false)) break;
    Held<DT, HOLD> x, res;
    ring_take<kOff>(x, g, in[0], s, 0, r, a.rows, t, nt, cols);
    float2 v[P];
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = x.get(k);
    if (a.residual) {
      ring_take<kOff>(res, g, in[1], s, 1, r, a.rows, t, nt, cols);
#pragma unroll
      for (int k = 0; k < P; ++k) v[k] = Pair<DT>::up(Pair<DT>::down(add2(v[k], res.get(k))));
      if constexpr (kOff) store_off<DT>(a.summed, r * a.cols, v, t, nt, cols);
      else store_held<DT, true>(a.summed, r * a.cols, v, t, nt, cols);
    }
    float mean = 0.f;
    float2 sum = both(0.f), ss = both(0.f);
    if (kLayer) {
#pragma unroll
      for (int k = 0; k < P; ++k) sum = add2(sum, v[k]);
      mean = row_sum<false>(sum.x + sum.y, red[turn][0]) / n_cols;
      center<DT>(v, mean, t, nt, cols);
    }
#pragma unroll
    for (int k = 0; k < P; ++k) ss = fma2(v[k], v[k], ss);
    const float var = row_sum<false>(ss.x + ss.y, red[turn][1]) / n_cols;
    // All threads have taken their columns: the stage is free.
    if (t == 0 && r + stages * step < a.rows) ring_ask<kOff>(g, in, s, r + stages * step, a.rows);
    if (++s == stages) s = 0, ph ^= 1;
    const float inv = 1.0f / sqrtf(var + a.eps);
#pragma unroll
    for (int k = 0; k < P; ++k) {
      v[k] = mul2(v[k], both(inv));
      v[k] = kLayer ? fma2(v[k], w[k], b[k]) : mul2(v[k], w[k]);
    }
    if constexpr (kOff) store_off<DT>(a.y, r * a.cols, v, t, nt, cols);
    else store_held<DT, true>(a.y, r * a.cols, v, t, nt, cols);
    if (t == 0) {
      a.inv[r] = inv;
      if (kLayer) a.mean[r] = mean;
    }
  }
  if (DT != H24_DTYPE_F16) {
    bool marked = false;
    __syncthreads();
    for (int64_t r = blockIdx.x + t * step; r < a.rows; r += nt * step) marked |= !(a.inv[r] > 0.f && finite(a.inv[r]));
    if (__syncthreads_or(marked)) wide_rows<DT, kLayer, false>(a, 1, red[0]);
  }
}

// Rows too long for the registers of a block: three passes over the row.
template <int DT, bool kLayer>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const __grid_constant__ NormArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float red[3][32];
  pdl_enter();
  const int t = threadIdx.x;
  const int64_t r = blockIdx.x;
  const T *x = static_cast<const T *>(a.x) + r * a.x_stride;
  const T *res = a.residual ? static_cast<const T *>(a.residual) + r * a.residual_stride : nullptr;
  T *out = a.summed ? static_cast<T *>(a.summed) + r * a.cols : nullptr;
  auto param = [&](const void *p, int64_t c) {
    return a.gain_f32 ? static_cast<const float *>(p)[c] : E::up(static_cast<const T *>(p)[c]);
  };
  // (Each thread reads back only what it wrote itself.)
  auto at = [&](int64_t c) { return E::up(res ? E::down(E::up(x[c]) + E::up(res[c])) : x[c]); };
  float sum = 0.f, ss = 0.f, mean = 0.f;
  if (kLayer) {
    for (int64_t c = t; c < a.cols; c += kLongThreads) sum += at(c);
    mean = row_sum<false>(sum, red[0]) / static_cast<float>(a.cols);
  }
  for (int64_t c = t; c < a.cols; c += kLongThreads) {
    const float s = at(c);
    if (out) out[c] = E::down(s);
    ss = fmaf(s - mean, s - mean, ss);
  }
  ss = row_sum<false>(ss, red[1]);
  const float inv = 1.0f / sqrtf(ss / static_cast<float>(a.cols) + a.eps);
  for (int64_t c = t; c < a.cols; c += kLongThreads)
    static_cast<T *>(a.y)[r * a.cols + c] =
        E::down((at(c) - mean) * inv * param(a.gain, c) + (kLayer && a.bias ? param(a.bias, c) : 0.f));
  if (t == 0) {
    a.inv[r] = inv;
    if (kLayer) a.mean[r] = mean;
  }
  if (DT != H24_DTYPE_F16) {
    const bool marked = !(inv > 0.f && finite(inv));  // (the same for the whole block)
    __syncthreads();
    if (marked) wide_rows<DT, kLayer, false>(a, 1, red);
  }
}

// ---------------------------------------------------------------------------
// Back
// ---------------------------------------------------------------------------

// A row's factors: n = fmaf(s, k, -shift) * inv.
struct RowScale {
  float inv, k, shift;
};
template <bool kLayer>
__device__ __forceinline__ RowScale row_scale(const BackArgs &a, int64_t r) {
  const float i = __ldg(a.inv + r);
  return {fabsf(i), i < 0.f ? kSmall : 1.f, kLayer ? __ldg(a.mean + r) : 0.f};
}

// A row's n and v = w dy (v holds w before), what it adds to dw and db, and the
// thread's part of the sums of v n and v.
template <int DT, bool kLayer, int HOLD, int P>
__device__ __forceinline__ void back_sums(const Held<DT, HOLD> &s, const Held<DT, HOLD> &dy, const RowScale &sc,
                                          float2 (&n)[P], float2 (&v)[P], float2 (&dw)[P], float2 (&db)[P], float &c1,
                                          float &c2) {
  const float2 k2 = both(sc.k), shift = both(-sc.shift), inv = both(sc.inv), direct = both(sc.k * sc.inv);
  float2 a1 = both(0.f), a2 = both(0.f);
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const float2 g = dy.get(k);
    n[k] = kLayer ? mul2(fma2(s.get(k), k2, shift), inv) : mul2(s.get(k), direct);
    dw[k] = fma2(g, n[k], dw[k]);
    if (kLayer) db[k] = add2(db[k], g);
    v[k] = mul2(v[k], g);  // (0 past the row's end)
    a1 = fma2(v[k], n[k], a1);
    if (kLayer) a2 = add2(a2, v[k]);
  }
  c1 = a1.x + a1.y;
  c2 = a2.x + a2.y;
}
// dx from them, in v.
template <int DT, int HOLD, int P>
__device__ __forceinline__ void back_row(const float2 (&n)[P], float2 (&v)[P], const Held<DT, HOLD> &ds, bool has_ds,
                                         const RowScale &sc, float c1, float c2) {
  const float2 m1 = both(-c1), m2 = both(-c2), scale = both(sc.inv * sc.k);
#pragma unroll
  for (int k = 0; k < P; ++k) {
    const float2 d = add2(fma2(n[k], m1, v[k]), m2);
    v[k] = has_ds ? fma2(d, scale, ds.get(k)) : mul2(d, scale);
  }
}

template <int DT, bool kLayer, int kMax, int HOLD>
__global__ void __launch_bounds__(kMax) norm_back_kernel(const __grid_constant__ BackArgs a) {
  __shared__ float red[2][2][32];
  pdl_enter();
  const int t = threadIdx.x, nt = blockDim.x;
  const int cols = static_cast<int>(a.cols);
  const int64_t first = blockIdx.x, step = gridDim.x;
  const float one_over = 1.0f / static_cast<float>(cols);
  constexpr int VEC = Elem<DT>::kVec, P = HOLD / 2;
  float2 dw[P] = {}, db[P] = {};
  int turn = 0;
  for (int64_t r = first; r < a.rows; r += step, turn ^= 1) {
    Held<DT, HOLD> s, dy, ds;
    s.template load<false>(a.s, r * a.s_stride, t, nt, cols);
    dy.template load<false>(a.dy, r * a.dy_stride, t, nt, cols);
    if (a.dsummed) ds.template load<false>(a.dsummed, r * a.dsummed_stride, t, nt, cols);
    const RowScale sc = row_scale<kLayer>(a, r);
    float2 n[P], v[P];
    load_param<DT, false>(a.gain, a.gain_f32, v, t, nt, cols);
    float c1, c2;
    back_sums<DT, kLayer>(s, dy, sc, n, v, dw, db, c1, c2);
    if (a.dx) {
      if (kLayer) row_sums(c1, c2, red[turn]);
      else c1 = row_sum<false>(c1, red[turn][0]);
      back_row<DT>(n, v, ds, a.dsummed != nullptr, sc, c1 * one_over, c2 * one_over);
      store_held<DT, false>(a.dx, r * a.cols, v, t, nt, cols);
    }
  }
  // The sums of this block.
  auto put = [&](float *out, const float2 (&sum)[P]) {
    if (!out) return;
    float *o = out + static_cast<int64_t>(blockIdx.x) * a.cols;
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int at = (t + 2 * k / VEC * nt) * VEC + 2 * k % VEC;
      if (at < cols) o[at] = sum[k].x;
      if (at + 1 < cols) o[at + 1] = sum[k].y;
    }
  };
  put(a.dgain, dw);
  if (kLayer) put(a.dbias, db);
}

// Rows of up to 512 columns, as in the forward pass; each lane adds dw and db up
// over its rows, and the block over its lanes with the same columns.
template <int DT, bool kAligned, bool kLayer, int HOLD>
__global__ void __launch_bounds__(kNarrowThreads) norm_back_narrow_kernel(const __grid_constant__ BackArgs a, int lanes) {
  __shared__ __align__(8) float held[kNarrowThreads * HOLD];
  pdl_enter();
  constexpr int VEC = Elem<DT>::kVec, P = HOLD / 2;
  const int t = threadIdx.x & (lanes - 1), cols = static_cast<int>(a.cols), per_block = kNarrowThreads / lanes;
  const int64_t step = static_cast<int64_t>(gridDim.x) * per_block;
  const int mine = threadIdx.x / lanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * per_block + mine;
  const int ahead = mine - (threadIdx.x & ~31) / lanes;
  const float one_over = 1.0f / static_cast<float>(cols);
  float2 w[P], dw[P] = {}, db[P] = {};
  load_param<DT, kAligned>(a.gain, a.gain_f32, w, t, lanes, cols);
  Held<DT, HOLD> s, dy, ds;
  RowScale sc;
  auto ask = [&](int64_t r) {
    s.clear();
    dy.clear();
    ds.clear();
    sc = {0.f, 1.f, 0.f};
    if (r >= a.rows) return;
    s.template load<kAligned>(a.s, r * a.s_stride, t, lanes, cols);
    dy.template load<kAligned>(a.dy, r * a.dy_stride, t, lanes, cols);
    if (a.dsummed) ds.template load<kAligned>(a.dsummed, r * a.dsummed_stride, t, lanes, cols);
    sc = row_scale<kLayer>(a, r);
  };
  ask(first);
  for (int64_t r = first; r - ahead < a.rows; r += step) {
    float2 n[P], v[P];
    float c1, c2;
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = w[k];
    back_sums<DT, kLayer>(s, dy, sc, n, v, dw, db, c1, c2);
    const Held<DT, HOLD> own = ds;
    const RowScale scale = sc;
    ask(r + step);
    if (a.dx) {
      c1 = lanes_sum(c1, lanes);
      if (kLayer) c2 = lanes_sum(c2, lanes);
      back_row<DT>(n, v, own, a.dsummed != nullptr, scale, c1 * one_over, c2 * one_over);
      if (r < a.rows) store_held<DT, kAligned>(a.dx, r * a.cols, v, t, lanes, cols);
    }
  }
  // The sums of this block: of a warp's rows across its lanes, then of the warps.
  const int row_cols = lanes * HOLD;
  auto put = [&](float *out, const float2 (&sum)[P]) {
    if (!out) return;
    float *o = out + static_cast<int64_t>(blockIdx.x) * a.cols;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < P; ++k) {
      float2 v = sum[k];
#pragma unroll
      for (int o = 16; o; o >>= 1)
        if (o >= lanes) {
          v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
          v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
        }
      if ((threadIdx.x & 31) < lanes)
        *reinterpret_cast<float2 *>(held + (threadIdx.x >> 5) * row_cols + (t + 2 * k / VEC * lanes) * VEC + 2 * k % VEC) = v;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += kNarrowThreads) {
      float total = 0.f;
#pragma unroll
      for (int g = 0; g < kWarpRows; ++g) total += held[g * row_cols + c];
      o[c] = total;
    }
  };
  put(a.dgain, dw);
  if (kLayer) put(a.dbias, db);
}

template <int DT, bool kLayer, int HOLD, int kMax, bool kOff>
__global__ void __launch_bounds__(kMax) norm_back_ring_kernel(const __grid_constant__ BackArgs a, int stages, int *err) {
  extern __shared__ __align__(128) uint8_t norm_smem[];
  __shared__ float red[2][2][32];
  __shared__ int abort;
  constexpr int VEC = Elem<DT>::kVec, SIZE = 16 / VEC;
  const int t = threadIdx.x, nt = blockDim.x;
  const int cols = static_cast<int>(a.cols);
  const int64_t step = gridDim.x;
  const float one_over = 1.0f / static_cast<float>(cols);
  if (t == 0) abort = 0;
  const RingInput in[3] = {{static_cast<const uint8_t *>(a.s), a.s_stride * SIZE},
                           {static_cast<const uint8_t *>(a.dy), a.dy_stride * SIZE},
                           {static_cast<const uint8_t *>(a.dsummed), a.dsummed_stride * SIZE}};
  const Ring g = ring_start<kOff>(norm_smem, stages, a.dsummed ? 3 : 2, a.cols, SIZE, in, a.rows);
  constexpr int P = HOLD / 2;
  float2 w[P], dw[P] = {}, db[P] = {};
  load_param<DT, !kOff>(a.gain, a.gain_f32, w, t, nt, cols);
  int turn = 0, st = 0;
  uint32_t ph = 0;
  RowScale next = {};
  if (blockIdx.x < a.rows) next = row_scale<kLayer>(a, blockIdx.x);
  for (int64_t r = blockIdx.x; r < a.rows; r += step, turn ^= 1) {
    const RowScale sc = next;
    if (r + step < a.rows) next = row_scale<kLayer>(a, r + step);
    if (!bar_wait(&g.full[st], ph, &abort, err, false)) break;
    Held<DT, HOLD> s, dy, ds;
    ring_take<kOff>(s, g, in[0], st, 0, r, a.rows, t, nt, cols);
    ring_take<kOff>(dy, g, in[1], st, 1, r, a.rows, t, nt, cols);
    if (a.dsummed) ring_take<kOff>(ds, g, in[2], st, 2, r, a.rows, t, nt, cols);
    float2 n[P], v[P];
#pragma unroll
    for (int k = 0; k < P; ++k) v[k] = w[k];
    float c1, c2;
    back_sums<DT, kLayer>(s, dy, sc, n, v, dw, db, c1, c2);
    // (The sums' barrier also says that the stage is free.)
    if (kLayer) row_sums(c1, c2, red[turn]);
    else c1 = row_sum<false>(c1, red[turn][0]);
    if (t == 0 && r + stages * step < a.rows) ring_ask<kOff>(g, in, st, r + stages * step, a.rows);
    if (++st == stages) st = 0, ph ^= 1;
    if (a.dx) {
      back_row<DT>(n, v, ds, a.dsummed != nullptr, sc, c1 * one_over, c2 * one_over);
      if constexpr (kOff) store_off<DT>(a.dx, r * a.cols, v, t, nt, cols);
      else store_held<DT, true>(a.dx, r * a.cols, v, t, nt, cols);
    }
  }
  auto put = [&](float *out, const float2 (&sum)[P]) {
    if (!out) return;
    float *o = out + static_cast<int64_t>(blockIdx.x) * a.cols;
#pragma unroll
    for (int k = 0; k < P; k += 2) {
      const int at = (t + 2 * k / VEC * nt) * VEC + 2 * k % VEC;
      const float f[4] = {sum[k].x, sum[k].y, sum[k + 1].x, sum[k + 1].y};
      if (kOff) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (at + i < cols) o[at + i] = f[i];
      } else if (at < cols) {
        *reinterpret_cast<float4 *>(o + at) = make_float4(f[0], f[1], f[2], f[3]);
      }
    }
  };
  put(a.dgain, dw);
  if (kLayer) put(a.dbias, db);
}

// dx of rows too long for the registers of a block.
template <int DT, bool kLayer>
__global__ void __launch_bounds__(kLongThreads) norm_back_long_kernel(const __grid_constant__ BackArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ float red[2][32];
  pdl_enter();
  const int64_t r = blockIdx.x;
  const T *s = static_cast<const T *>(a.s) + r * a.s_stride, *dy = static_cast<const T *>(a.dy) + r * a.dy_stride;
  const T *ds = a.dsummed ? static_cast<const T *>(a.dsummed) + r * a.dsummed_stride : nullptr;
  const RowScale sc = row_scale<kLayer>(a, r);
  const float one_over = 1.0f / static_cast<float>(a.cols);
  auto gain = [&](int64_t c) {
    return a.gain_f32 ? static_cast<const float *>(a.gain)[c] : E::up(static_cast<const T *>(a.gain)[c]);
  };
  float c1 = 0.f, c2 = 0.f;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float v = E::up(dy[c]) * gain(c);
    c1 = fmaf(v, fmaf(E::up(s[c]), sc.k, -sc.shift) * sc.inv, c1);
    if (kLayer) c2 += v;
  }
  row_sums(c1, c2, red);
  c1 *= one_over, c2 *= one_over;
  for (int64_t c = threadIdx.x; c < a.cols; c += kLongThreads) {
    const float n = fmaf(E::up(s[c]), sc.k, -sc.shift) * sc.inv;
    float d = (fmaf(-n, c1, E::up(dy[c]) * gain(c)) - c2) * sc.inv * sc.k;
    if (ds) d += E::up(ds[c]);
    static_cast<T *>(a.dx)[r * a.cols + c] = E::down(d);
  }
}

// Sums of dw and db of such rows: a thread a column, blockIdx.y a part of the rows.
template <int DT, bool kLayer>
__global__ void __launch_bounds__(256) norm_back_columns_kernel(const __grid_constant__ BackArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  pdl_enter();
  const int64_t c = blockIdx.x * static_cast<int64_t>(256) + threadIdx.x;
  if (c >= a.cols) return;
  float dw = 0.f, db = 0.f;
  for (int64_t r = blockIdx.y; r < a.rows; r += gridDim.y) {
    const RowScale sc = row_scale<kLayer>(a, r);
    const float g = E::up(static_cast<const T *>(a.dy)[r * a.dy_stride + c]);
    dw = fmaf(g, fmaf(E::up(static_cast<const T *>(a.s)[r * a.s_stride + c]), sc.k, -sc.shift) * sc.inv, dw);
    db += g;
  }
  if (a.dgain) a.dgain[blockIdx.y * a.cols + c] = dw;
  if (a.dbias) a.dbias[blockIdx.y * a.cols + c] = db;
}

// The blocks' sums, in the blocks' order: blockIdx.y 0 is dw, 1 db.
template <typename Out, int kSumGroups>
__global__ void __launch_bounds__(kSumCols * kSumGroups) norm_sums_kernel(const float *dgain, const float *dbias,
                                                                          int parts, int64_t cols, Out *gain_out,
                                                                          Out *bias_out) {
  __shared__ float red[kSumGroups][kSumCols + 1];
  pdl_enter();
  const float *in = blockIdx.y ? dbias : dgain;
  Out *out = blockIdx.y ? bias_out : gain_out;
  const int x = threadIdx.x % kSumCols, g = threadIdx.x / kSumCols;
  const int64_t c = blockIdx.x * static_cast<int64_t>(kSumCols) + x;
  float sum = 0.f;
  if (in && c < cols) {
#pragma unroll 8
    for (int p = g; p < parts; p += kSumGroups) sum += __ldcs(in + p * cols + c);
  }
  red[g][x] = sum;
  __syncthreads();
  // Each warp adds up some of the columns, a group a lane.
  const int lane = threadIdx.x & 31;
  for (int w = threadIdx.x >> 5; w < kSumCols; w += kSumGroups) {
    const float total = warp_sum(lane < kSumGroups ? red[lane][w] : 0.f);
    const int64_t cw = blockIdx.x * static_cast<int64_t>(kSumCols) + w;
    if (lane == 0 && in && cw < cols) {
      if constexpr (sizeof(Out) == 4)
        out[cw] = total;
      else
        out[cw] = Out(total);
    }
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
// Columns of a thread and threads of a block.  They go by the columns alone, and
// whether a row comes through the ring or not, its sums have the same order: a
// row's result does not depend on where it lies.
int row_threads(int64_t cols) {
  const int hold = cols <= kFewCols ? kFew : kHold;
  return static_cast<int>(((cols + hold - 1) / hold + 31) / 32 * 32);
}
// Lanes of a row of up to kWarpCols columns.
int narrow_lanes(int64_t cols) {
  const int hold = cols > 32 * kFew ? kHold : kFew;
  int lanes = 1;
  while (lanes * hold < cols) lanes *= 2;
  return lanes;
}
template <auto kernel>
int narrow_grid(int64_t rows, int64_t cols) {
  const int per_block = kNarrowThreads / narrow_lanes(cols);
  return wave_grid((rows + per_block - 1) / per_block, blocks_per_sm_once<kernel>(kNarrowThreads));
}
template <auto kernel>
int launch_norm_narrow(const NormArgs &a, cudaStream_t s) {
  H24_CUDA_TRY(launch_pdl(kernel, dim3(narrow_grid<kernel>(a.rows, a.cols)), dim3(kNarrowThreads), s, a, narrow_lanes(a.cols)));
  count_launches(1);
  return H24_OK;
}
template <auto kernel>
int launch_norm_rows(const NormArgs &a, int threads, cudaStream_t s) {
  H24_CUDA_TRY(launch_pdl(kernel, dim3(wave_grid(a.rows, blocks_per_sm_once<kernel>(threads))), dim3(threads), s, a));
  count_launches(1);
  return H24_OK;
}

// Whether rows off 16 bytes come through the ring: where a block has several rows,
// so that the first and the last of all, which it reads itself, are few among
// them.  (Inputs whose rows lie over one another, a row stride below their
// length, do not: what stands around such a row may be outside the tensor.)
bool ring_of_any_rows(int64_t rows, int64_t cols) { return rows >= 1024 && cols > kWarpCols; }

// Stages of a ring and blocks an SM: about 200 KB of rows on their way, in
// blocks of what the registers of an SM hold, and fewer of them where a block's
// ring would have less than two stages.  Of the longest rows one SM holds one stage
// alone (fp32 with three inputs from some 9,300 columns on, with two from some
// 14,000): the next row is then asked for once this one's sums are there.
struct RingPlan {
  int threads, stages, smem, grid;
};
template <auto kernel>
int ring_plan(int64_t rows, int64_t cols, int size, int inputs, bool off, RingPlan *p) {
  H24_CUDA_TRY(allow_smem<kernel>(kRingSmem));
  p->threads = row_threads(cols);
  const int one = ring_pitch(cols * size, off) * inputs;
  int per_sm = blocks_per_sm_once<kernel>(p->threads);
  while (per_sm > 1 && kRingSmem / per_sm < kRingHead + 2 * one) --per_sm;
  p->stages = (kRingSmem / per_sm - kRingHead - 1024) / one;
  p->stages = p->stages < 1 ? 1 : p->stages > kMaxRing ? kMaxRing : p->stages;
  p->smem = kRingHead + p->stages * one;
  p->grid = wave_grid(rows, per_sm);
  return H24_OK;
}
template <typename K, typename Args>
int launch_ring(K kernel, const Args &a, const RingPlan &p, int *err, cudaStream_t s) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(p.grid);
  cfg.blockDim = dim3(p.threads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  H24_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, a, p.stages, err));
  count_launches(1);
  return H24_OK;
}
template <auto kernel, int DT, bool kOff>
int run_norm_ring(const Tables *T, const NormArgs &a, cudaStream_t s) {
  RingPlan p;
  const int rc = ring_plan<kernel>(a.rows, a.cols, 16 / Elem<DT>::kVec, a.residual ? 2 : 1, kOff, &p);
  return rc != H24_OK ? rc : launch_ring(kernel, a, p, T->err, s);
}

template <int DT, bool kLayer>
int launch_norm_typed(const Tables *T, const NormArgs &a, cudaStream_t s) {
  constexpr int kVec = Elem<DT>::kVec;
  if (a.cols > kBlockCols) {
    H24_CUDA_TRY(launch_pdl(norm_long_kernel<DT, kLayer>, dim3(static_cast<unsigned>(a.rows)), dim3(kLongThreads), s, a));
    count_launches(1);
    return H24_OK;
  }
  const bool aligned = a.cols % kVec == 0 && a.x_stride % kVec == 0 && a.residual_stride % kVec == 0 && aligned16(a.x) &&
                       aligned16(a.residual) && aligned16(a.summed) && aligned16(a.y) && aligned16(a.gain) && aligned16(a.bias);
  if (a.cols <= 32 * kFew)
    return aligned ? launch_norm_narrow<norm_narrow_kernel<DT, true, kLayer, kFew>>(a, s)
                   : launch_norm_narrow<norm_narrow_kernel<DT, false, kLayer, kFew>>(a, s);
  if (a.cols <= kWarpCols)
    return aligned ? launch_norm_narrow<norm_narrow_kernel<DT, true, kLayer, kHold>>(a, s)
                   : launch_norm_narrow<norm_narrow_kernel<DT, false, kLayer, kHold>>(a, s);
  const int threads = row_threads(a.cols);
  const bool off = !aligned && ring_of_any_rows(a.rows, a.cols) && a.x_stride >= a.cols && (!a.residual || a.residual_stride >= a.cols);
  if (a.cols <= kFewCols)
    return aligned ? run_norm_ring<norm_ring_kernel<DT, kLayer, kFew, 512, false>, DT, false>(T, a, s)
           : off   ? run_norm_ring<norm_ring_kernel<DT, kLayer, kFew, 512, true>, DT, true>(T, a, s)
                   : launch_norm_rows<norm_kernel<DT, kLayer, 512, kFew>>(a, threads, s);
  if (threads <= 512)
    return aligned ? run_norm_ring<norm_ring_kernel<DT, kLayer, kHold, 512, false>, DT, false>(T, a, s)
           : off   ? run_norm_ring<norm_ring_kernel<DT, kLayer, kHold, 512, true>, DT, true>(T, a, s)
                   : launch_norm_rows<norm_kernel<DT, kLayer, 512, kHold>>(a, threads, s);
  return aligned ? run_norm_ring<norm_ring_kernel<DT, kLayer, kHold, 1024, false>, DT, false>(T, a, s)
         : off   ? run_norm_ring<norm_ring_kernel<DT, kLayer, kHold, 1024, true>, DT, true>(T, a, s)
                 : launch_norm_rows<norm_kernel<DT, kLayer, 1024, kHold>>(a, threads, s);
}

// The backward kernel of rows that a block holds: its grid (one wave; asked for
// first, since each block has its sums), or its launch.
template <auto kernel>
int back_rows(const BackArgs &a, int grid, int threads, int *ask, cudaStream_t s) {
  if (ask) {
    *ask = wave_grid(a.rows, blocks_per_sm_once<kernel>(threads));
    return H24_OK;
  }
  H24_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(threads), s, a));
  count_launches(1);
  return H24_OK;
}
template <auto kernel>
int back_narrow(const BackArgs &a, int grid, int *ask, cudaStream_t s) {
  if (ask) {
    *ask = narrow_grid<kernel>(a.rows, a.cols);
    return H24_OK;
  }
  H24_CUDA_TRY(launch_pdl(kernel, dim3(grid), dim3(kNarrowThreads), s, a, narrow_lanes(a.cols)));
  count_launches(1);
  return H24_OK;
}
template <auto kernel, int DT, bool kOff>
int back_ring(const Tables *T, const BackArgs &a, int *ask, cudaStream_t s) {
  RingPlan p;
  const int rc = ring_plan<kernel>(a.rows, a.cols, 16 / Elem<DT>::kVec, a.dsummed ? 3 : 2, kOff, &p);
  if (rc == H24_OK && ask) *ask = p.grid;
  return rc != H24_OK || ask ? rc : launch_ring(kernel, a, p, T->err, s);
}
template <int DT, bool kLayer>
int back_width(const Tables *T, const BackArgs &a, bool aligned, int grid, int *ask, cudaStream_t s) {
  if (a.cols <= 32 * kFew)
    return aligned ? back_narrow<norm_back_narrow_kernel<DT, true, kLayer, kFew>>(a, grid, ask, s)
                   : back_narrow<norm_back_narrow_kernel<DT, false, kLayer, kFew>>(a, grid, ask, s);
  if (a.cols <= kWarpCols)
    return aligned ? back_narrow<norm_back_narrow_kernel<DT, true, kLayer, kHold>>(a, grid, ask, s)
                   : back_narrow<norm_back_narrow_kernel<DT, false, kLayer, kHold>>(a, grid, ask, s);
  const int threads = row_threads(a.cols);
  const bool off = !aligned && ring_of_any_rows(a.rows, a.cols) && a.s_stride >= a.cols && a.dy_stride >= a.cols &&
                   (!a.dsummed || a.dsummed_stride >= a.cols);
  if (a.cols <= kFewCols)
    return aligned ? back_ring<norm_back_ring_kernel<DT, kLayer, kFew, 512, false>, DT, false>(T, a, ask, s)
           : off   ? back_ring<norm_back_ring_kernel<DT, kLayer, kFew, 512, true>, DT, true>(T, a, ask, s)
                   : back_rows<norm_back_kernel<DT, kLayer, 512, kFew>>(a, grid, threads, ask, s);
  if (threads <= 512)
    return aligned ? back_ring<norm_back_ring_kernel<DT, kLayer, kHold, 512, false>, DT, false>(T, a, ask, s)
           : off   ? back_ring<norm_back_ring_kernel<DT, kLayer, kHold, 512, true>, DT, true>(T, a, ask, s)
                   : back_rows<norm_back_kernel<DT, kLayer, 512, kHold>>(a, grid, threads, ask, s);
  return aligned ? back_ring<norm_back_ring_kernel<DT, kLayer, kHold, 1024, false>, DT, false>(T, a, ask, s)
         : off   ? back_ring<norm_back_ring_kernel<DT, kLayer, kHold, 1024, true>, DT, true>(T, a, ask, s)
                 : back_rows<norm_back_kernel<DT, kLayer, 1024, kHold>>(a, grid, threads, ask, s);
}

template <int DT, bool kLayer>
int launch_back_typed(const Tables *T, BackArgs a, void *dgain, void *dbias, cudaStream_t s) {
  constexpr int kVec = Elem<DT>::kVec;
  const bool sums = dgain || dbias;
  const bool is_long = a.cols > kBlockCols;
  const bool aligned = a.cols % kVec == 0 && a.s_stride % kVec == 0 && a.dy_stride % kVec == 0 &&
                       a.dsummed_stride % kVec == 0 && aligned16(a.s) && aligned16(a.dy) && aligned16(a.dsummed) &&
                       aligned16(a.dx) && aligned16(a.gain);
  const int64_t col_blocks = (a.cols + 255) / 256;
  auto rows = [&](int grid, int *ask) {
    return back_width<DT, kLayer>(T, a, aligned, grid, ask, s);
  };
  int grid = static_cast<int>(wave_grid(a.rows, 8) / col_blocks + 1);
  if (!is_long) {
    const int rc = rows(0, &grid);
    if (rc != H24_OK) return rc;
  }
  float *parts = nullptr;
  if (sums) {
    const size_t one = static_cast<size_t>(grid) * static_cast<size_t>(a.cols);
    H24_CUDA_TRY(cudaMallocFromPoolAsync(reinterpret_cast<void **>(&parts), one * 8, T->pool, s));
    a.dgain = dgain ? parts : nullptr;
    a.dbias = dbias ? parts + one : nullptr;
  }
  auto run = [&]() -> int {
    if (is_long) {
      if (a.dx) {
        H24_CUDA_TRY(launch_pdl(norm_back_long_kernel<DT, kLayer>, dim3(static_cast<unsigned>(a.rows)),
                                dim3(kLongThreads), s, a));
        count_launches(1);
      }
      if (sums) {
        H24_CUDA_TRY(launch_pdl(norm_back_columns_kernel<DT, kLayer>,
                                dim3(static_cast<unsigned>(col_blocks), static_cast<unsigned>(grid)), dim3(256), s, a));
        count_launches(1);
      }
    } else {
      const int rc = rows(grid, nullptr);
      if (rc != H24_OK) return rc;
    }
    if (sums) {
      // 32 groups of rows a block where that leaves the GPU in one wave, 8 where
      // the columns alone fill it ([8192,7680], dw and db: 6.4 us, 9.4 with 32).
      // Blocks of 16 columns took 8 us instead of 6 for [16384,1920].
      using P = typename Elem<DT>::T;
      const int64_t blocks = (a.cols + kSumCols - 1) / kSumCols * (dbias ? 2 : 1);
      auto sum = [&](auto out_type, auto groups) -> int {
        using Out = decltype(out_type);
        constexpr int G = decltype(groups)::value;
        H24_CUDA_TRY(launch_pdl(norm_sums_kernel<Out, G>,
                                dim3(static_cast<unsigned>((a.cols + kSumCols - 1) / kSumCols), dbias ? 2 : 1),
                                dim3(kSumCols * G), s, static_cast<const float *>(a.dgain),
                                static_cast<const float *>(a.dbias), grid, a.cols, static_cast<Out *>(dgain),
                                static_cast<Out *>(dbias)));
        return H24_OK;
      };
      constexpr std::integral_constant<int, 32> many;
      constexpr std::integral_constant<int, 8> few;
      const bool f32 = a.gain_f32 || DT == H24_DTYPE_F32;
      const int rc = blocks <= 296 ? f32 ? sum(float(), many) : sum(P(), many) : f32 ? sum(float(), few) : sum(P(), few);
      if (rc != H24_OK) return rc;
      count_launches(1);
    }
    return H24_OK;
  };
  int rc = run();
  if (parts) {
    const cudaError_t e = cudaFreeAsync(parts, s);
    if (rc == H24_OK && e != cudaSuccess) rc = cuda_fail(e, "cudaFreeAsync");
  }
  return rc;
}

}  // namespace

int launch_add_norm(const Tables *T, const AddNormArgs &c, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                    const void *bias, float eps, void *y, void *summed, float *stats, cudaStream_t s) {
  const NormArgs a{x, residual, c.gain, bias, c.rows, c.cols, x_stride, residual ? residual_stride : 0, eps,
                   c.param_dtype == H24_DTYPE_F32, y, summed, stats, stats + c.rows};
  switch (c.dtype) {
    case H24_DTYPE_F32: return c.layer ? launch_norm_typed<H24_DTYPE_F32, true>(T, a, s) : launch_norm_typed<H24_DTYPE_F32, false>(T, a, s);
    case H24_DTYPE_F16: return c.layer ? launch_norm_typed<H24_DTYPE_F16, true>(T, a, s) : launch_norm_typed<H24_DTYPE_F16, false>(T, a, s);
    default: return c.layer ? launch_norm_typed<H24_DTYPE_BF16, true>(T, a, s) : launch_norm_typed<H24_DTYPE_BF16, false>(T, a, s);
  }
}

int launch_add_norm_backward(const Tables *T, const AddNormArgs &c, const void *summed, int64_t summed_stride,
                             const float *stats, const void *dy, int64_t dy_stride, const void *dsummed,
                             int64_t dsummed_stride, void *dx, void *dgain, void *dbias, cudaStream_t s) {
  const BackArgs a{summed, dy, dsummed, c.gain, c.rows, c.cols, summed_stride, dy_stride, dsummed ? dsummed_stride : 0,
                   c.param_dtype == H24_DTYPE_F32, stats, stats + c.rows, dx, nullptr, nullptr};
  switch (c.dtype) {
    case H24_DTYPE_F32: return c.layer ? launch_back_typed<H24_DTYPE_F32, true>(T, a, dgain, dbias, s) : launch_back_typed<H24_DTYPE_F32, false>(T, a, dgain, dbias, s);
    case H24_DTYPE_F16: return c.layer ? launch_back_typed<H24_DTYPE_F16, true>(T, a, dgain, dbias, s) : launch_back_typed<H24_DTYPE_F16, false>(T, a, dgain, dbias, s);
    default: return c.layer ? launch_back_typed<H24_DTYPE_BF16, true>(T, a, dgain, dbias, s) : launch_back_typed<H24_DTYPE_BF16, false>(T, a, dgain, dbias, s);
  }
}

}  // namespace h24
