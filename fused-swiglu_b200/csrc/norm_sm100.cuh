// Layer norm and RMS norm of the rows of a matrix, forward and backward.
//
//   z = (x - mean) rstd      y = z w + b      rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   a = dy w                 dx = rstd (a - mean(a) - z mean(a z)) (+ res)      dw = sum_rows dy z      db = sum_rows dy
//
// RMS norm is the same with 0 in the place of mean and without the term mean(a).  Rows are read as bf16 or fp32; all
// sums, statistics and products are fp32, and each output is rounded once.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

namespace fsw {

struct NormForwardParams {
  const void* x;
  const void* weight;  // NULL: ones
  const void* bias;    // NULL: zeros
  void* y;
  float* mean;  // layer norm only
  float* rstd;
  long long ldx, ldy;
  int M, d;
  int w_f32;  // weight and bias are fp32, not bf16
  float eps;
};

struct NormBackwardParams {
  const void* dout;
  const void* x;
  const void* weight;    // NULL: ones
  const void* residual;  // NULL, or added to dx
  const float* mean;     // layer norm only
  const float* rstd;
  void* dx;
  float* partial;  // [splits][2][d]: sums of dy z and of dy over a split's rows
  long long ld_dout, ldx, ld_res, ld_dx;
  int M, d, splits;
  int w_f32;
};

struct NormReduceParams {
  const float* partial;
  void* dweight;  // NULL: not wanted
  void* dbias;    // NULL: not wanted
  int d, splits;
  int out_f32;
};

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of a vector of bf16 or fp32 values; `none` where there is no vector.
__device__ __forceinline__ float load_vector(const void* p, long long i, int f32, float none) {
  if (p == nullptr) return none;
  return f32 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

constexpr int kNormThreads = 256;

// Sums of two values over the block, in a fixed order, known to every thread.
__device__ __forceinline__ float2 block_sum2(float2 v, float2* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  __syncthreads();  // the previous sums have been read
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  float2 s = make_float2(0.0f, 0.0f);
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    s.x += shared[w].x;
    s.y += shared[w].y;
  }
  return s;
}

// Any width, alignment and pitch: one block a row, which is read once for each of mean, variance and result.
template <typename T, bool kLayer>
__global__ void __launch_bounds__(kNormThreads) norm_forward_any_kernel(const NormForwardParams p) {
  __shared__ float2 shared[kNormThreads / 32];
  for (int row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    T* y = static_cast<T*>(p.y) + row * p.ldy;
    float mean = 0.0f;
    if (kLayer) {
      float s = 0.0f;
      for (int i = threadIdx.x; i < p.d; i += kNormThreads) s += to_float<T>(x[i]);
      mean = block_sum2(make_float2(s, 0.0f), shared).x / static_cast<float>(p.d);
    }
    float ss = 0.0f;
    for (int i = threadIdx.x; i < p.d; i += kNormThreads) {
      const float c = to_float<T>(x[i]) - mean;
      ss = fmaf(c, c, ss);
    }
    const float rstd = rsqrtf(block_sum2(make_float2(ss, 0.0f), shared).x / static_cast<float>(p.d) + p.eps);
    for (int i = threadIdx.x; i < p.d; i += kNormThreads) {
      const float z = (to_float<T>(x[i]) - mean) * rstd;
      y[i] = from_float<T>(fmaf(z, load_vector(p.weight, i, p.w_f32, 1.0f), load_vector(p.bias, i, p.w_f32, 0.0f)));
    }
    if (threadIdx.x == 0) {
      if (kLayer) p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

// dx for any width, alignment and pitch: one block a row, read once for the two means and once for the result.
template <typename T, bool kLayer>
__global__ void __launch_bounds__(kNormThreads) norm_backward_any_kernel(const NormBackwardParams p) {
  __shared__ float2 shared[kNormThreads / 32];
  for (int row = blockIdx.x; row < p.M; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.ldx;
    const T* dy = static_cast<const T*>(p.dout) + row * p.ld_dout;
    const T* res = p.residual == nullptr ? nullptr : static_cast<const T*>(p.residual) + row * p.ld_res;
    T* dx = static_cast<T*>(p.dx) + row * p.ld_dx;
    const float mean = kLayer ? p.mean[row] : 0.0f, rstd = p.rstd[row];
    float2 s = make_float2(0.0f, 0.0f);
    for (int i = threadIdx.x; i < p.d; i += kNormThreads) {
      const float a = to_float<T>(dy[i]) * load_vector(p.weight, i, p.w_f32, 1.0f);
      const float z = (to_float<T>(x[i]) - mean) * rstd;
      s.x += a;
      s.y = fmaf(a, z, s.y);
    }
    s = block_sum2(s, shared);
    const float c1 = kLayer ? s.x / static_cast<float>(p.d) : 0.0f, c2 = s.y / static_cast<float>(p.d);
    for (int i = threadIdx.x; i < p.d; i += kNormThreads) {
      const float a = to_float<T>(dy[i]) * load_vector(p.weight, i, p.w_f32, 1.0f);
      const float z = (to_float<T>(x[i]) - mean) * rstd;
      float v = (a - c1 - z * c2) * rstd;
      if (res != nullptr) v += to_float<T>(res[i]);
      dx[i] = from_float<T>(v);
    }
  }
}

// Sums over rows for any width, alignment and pitch: a block takes 256 columns of one split of the rows.
template <typename T, bool kLayer>
__global__ void __launch_bounds__(kNormThreads) norm_backward_columns_any_kernel(const NormBackwardParams p) {
  const long long tiles = (p.d + kNormThreads - 1) / kNormThreads;
  for (long long t = blockIdx.x; t < tiles * p.splits; t += gridDim.x) {
    const int split = static_cast<int>(t / tiles);
    const int i = static_cast<int>(t % tiles) * kNormThreads + threadIdx.x;
    if (i >= p.d) continue;
    const int r0 = static_cast<int>(static_cast<long long>(p.M) * split / p.splits);
    const int r1 = static_cast<int>(static_cast<long long>(p.M) * (split + 1) / p.splits);
    float dw = 0.0f, db = 0.0f;
    for (int r = r0; r < r1; ++r) {
      const float dy = to_float<T>(static_cast<const T*>(p.dout)[r * p.ld_dout + i]);
      const float x = to_float<T>(static_cast<const T*>(p.x)[r * p.ldx + i]);
      dw = fmaf(dy, (x - (kLayer ? p.mean[r] : 0.0f)) * p.rstd[r], dw);
      db += dy;
    }
    float* out = p.partial + 2ll * split * p.d;
    out[i] = dw;
    out[p.d + i] = db;
  }
}

// Joins the splits' sums, in the order of the splits.
__global__ void __launch_bounds__(kNormThreads) norm_reduce_kernel(const NormReduceParams p) {
  const long long i = static_cast<long long>(blockIdx.x) * kNormThreads + threadIdx.x;
  if (i >= p.d) return;
  float dw = 0.0f, db = 0.0f;
  for (int s = 0; s < p.splits; ++s) {
    dw += p.partial[2ll * s * p.d + i];
    db += p.partial[2ll * s * p.d + p.d + i];
  }
  if (p.dweight != nullptr) {
    if (p.out_f32) static_cast<float*>(p.dweight)[i] = dw;
    else static_cast<__nv_bfloat16*>(p.dweight)[i] = __float2bfloat16_rn(dw);
  }
  if (p.dbias != nullptr) {
    if (p.out_f32) static_cast<float*>(p.dbias)[i] = db;
    else static_cast<__nv_bfloat16*>(p.dbias)[i] = __float2bfloat16_rn(db);
  }
}

}  // namespace fsw
