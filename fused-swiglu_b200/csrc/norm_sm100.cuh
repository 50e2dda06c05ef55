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

#include "vector_io_sm100.cuh"

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

// ---- rows held in registers ----
//
// blockDim.x threads (a multiple of 32) hold one row, N vectors of V values each, and blockDim.y such groups of a block
// take rows of their own; a group's next row is on its way while the present one is reduced.  A row is read once.

// Sum over a group, in a fixed order, known to its threads.  A group has two sets of slots and takes them in turn: who
// writes one again has passed the barrier of the other, which all reached after they had read the first.
__device__ __forceinline__ float2 group_sum(float2 v, float2* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  const int warps = blockDim.x >> 5;
  if (warps == 1) return v;
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
  float2 s = slots[0];
  for (int w = 1; w < warps; ++w) {
    s.x += slots[w].x;
    s.y += slots[w].y;
  }
  return s;
}

constexpr int kNormGroups = 8;       // most groups of a block
constexpr int kNormRowThreads = 512;  // most threads of a block

template <typename T, int V, int N>
__device__ __forceinline__ void load_row(RawVector<T, V> (&raw)[N], const T* row, int d) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
    if (c < d) raw[j].load(row + c);
  }
}

// A weight or bias vector's values of this thread, and `none` where there are none.
template <int V, int N>
__device__ __forceinline__ void load_columns(float (&v)[N * V], const void* p, int f32, int d, float none) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) v[j * V + i] = none;
    if (p != nullptr && c < d) {
      if (f32) {
        RawVector<float, V> r;
        r.load(static_cast<const float*>(p) + c);
        r.get(v + j * V);
      } else {
        RawVector<__nv_bfloat16, V> r;
        r.load(static_cast<const __nv_bfloat16*>(p) + c);
        r.get(v + j * V);
      }
    }
  }
}

template <typename T, bool kLayer, int V, int N>
__global__ void __launch_bounds__(kNormRowThreads) norm_forward_rows_kernel(const NormForwardParams p) {
  __shared__ float2 slots[kNormGroups][2][kNormRowThreads / 32];
  float w[N * V], b[N * V];
  load_columns<V, N>(w, p.weight, p.w_f32, p.d, 1.0f);
  if (kLayer) load_columns<V, N>(b, p.bias, p.w_f32, p.d, 0.0f);
  const float inv_d = 1.0f / static_cast<float>(p.d);
  const int stride = gridDim.x * blockDim.y;
  int row = blockIdx.x * blockDim.y + threadIdx.y, turn = 0;
  RawVector<T, V> raw[N];
  if (row < p.M) load_row<T, V, N>(raw, static_cast<const T*>(p.x) + row * p.ldx, p.d);
  for (; row < p.M; row += stride) {
    float x[N * V];
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) x[j * V + i] = 0.0f;
      if ((j * blockDim.x + threadIdx.x) * V < p.d) raw[j].get(x + j * V);
    }
    if (row < p.M - stride) load_row<T, V, N>(raw, static_cast<const T*>(p.x) + (row + stride) * p.ldx, p.d);
    float mean = 0.0f;
    if (kLayer) {
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < N * V; ++i) s += x[i];
      mean = group_sum(make_float2(s, 0.0f), slots[threadIdx.y][turn]).x * inv_d;
      turn ^= 1;
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if ((j * blockDim.x + threadIdx.x) * V < p.d) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[j * V + i] -= mean;
          ss = fmaf(x[j * V + i], x[j * V + i], ss);
        }
      }
    }
    const float rstd = rsqrtf(fmaf(group_sum(make_float2(ss, 0.0f), slots[threadIdx.y][turn]).x, inv_d, p.eps));
    turn ^= 1;
    T* y = static_cast<T*>(p.y) + row * p.ldy;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c < p.d) {
        float out[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float z = x[j * V + i] * rstd;
          out[i] = kLayer ? fmaf(z, w[j * V + i], b[j * V + i]) : z * w[j * V + i];
        }
        store_vector<V, T>(y + c, out);
      }
    }
    if (threadIdx.x == 0) {
      if (kLayer) p.mean[row] = mean;
      p.rstd[row] = rstd;
    }
  }
}

// dx, and the block's part of the sums over rows: a thread keeps them for its columns over all its rows, the groups of a
// block are joined in shared memory, and the blocks by norm_reduce_kernel.
template <typename T, bool kLayer, int V, int N>
__global__ void __launch_bounds__(kNormRowThreads) norm_backward_rows_kernel(const NormBackwardParams p) {
  __shared__ float2 slots[kNormGroups][2][kNormRowThreads / 32];
  extern __shared__ float joined[];  // [2][columns of a group], more than one group only
  float w[N * V], dw[N * V], db[kLayer ? N * V : 1];
  load_columns<V, N>(w, p.weight, p.w_f32, p.d, 1.0f);
#pragma unroll
  for (int i = 0; i < N * V; ++i) dw[i] = 0.0f;
  if (kLayer) {
#pragma unroll
    for (int i = 0; i < N * V; ++i) db[i] = 0.0f;
  }
  const float inv_d = 1.0f / static_cast<float>(p.d);
  const int stride = gridDim.x * blockDim.y;
  int row = blockIdx.x * blockDim.y + threadIdx.y, turn = 0;
  RawVector<T, V> raw_x[N], raw_dy[N], raw_res[N];
  float next_mean = 0.0f, next_rstd = 0.0f;
  auto fetch = [&](int r) {
    load_row<T, V, N>(raw_x, static_cast<const T*>(p.x) + r * p.ldx, p.d);
    load_row<T, V, N>(raw_dy, static_cast<const T*>(p.dout) + r * p.ld_dout, p.d);
    if (p.residual != nullptr) load_row<T, V, N>(raw_res, static_cast<const T*>(p.residual) + r * p.ld_res, p.d);
    if (kLayer) next_mean = p.mean[r];
    next_rstd = p.rstd[r];
  };
  if (row < p.M) fetch(row);
  for (; row < p.M; row += stride) {
    float z[N * V], a[N * V];
    const float mean = next_mean, rstd = next_rstd;
    RawVector<T, V> res[N];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) z[j * V + i] = a[j * V + i] = 0.0f;
      if ((j * blockDim.x + threadIdx.x) * V < p.d) {
        raw_x[j].get(z + j * V);
        raw_dy[j].get(a + j * V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = j * V + i;
          z[k] = (z[k] - mean) * rstd;
          dw[k] = fmaf(a[k], z[k], dw[k]);
          if (kLayer) db[k] += a[k];
          a[k] *= w[k];
          s.x += a[k];
          s.y = fmaf(a[k], z[k], s.y);
        }
      }
      res[j] = raw_res[j];
    }
    if (row < p.M - stride) fetch(row + stride);
    s = group_sum(s, slots[threadIdx.y][turn]);
    turn ^= 1;
    const float c1 = kLayer ? s.x * inv_d : 0.0f, c2 = s.y * inv_d;
    T* dx = static_cast<T*>(p.dx) + row * p.ld_dx;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * V;
      if (c < p.d) {
        float out[V], add[V];
        if (p.residual != nullptr) res[j].get(add);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = j * V + i;
          const float t = fmaf(-z[k], c2, kLayer ? a[k] - c1 : a[k]);
          out[i] = p.residual != nullptr ? fmaf(t, rstd, add[i]) : t * rstd;
        }
        store_vector<V, T>(dx + c, out);
      }
    }
  }
  if (p.partial == nullptr) return;
  float* part = p.partial + 2ll * blockIdx.x * p.d;
  const int columns = blockDim.x * N * V;
  for (int g = 0; g < static_cast<int>(blockDim.y); ++g) {
    if (static_cast<int>(threadIdx.y) == g) {
      const bool last = g + 1 == static_cast<int>(blockDim.y);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int c = (j * blockDim.x + threadIdx.x) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int k = j * V + i;
          if (g > 0) {
            dw[k] += joined[c + i];
            if (kLayer) db[k] += joined[columns + c + i];
          }
          if (!last) {
            joined[c + i] = dw[k];
            if (kLayer) joined[columns + c + i] = db[k];
          }
        }
        if (last && c < p.d) {
          store_vector<V, float>(part + c, dw + j * V);
          if (kLayer) store_vector<V, float>(part + p.d + c, db + j * V);
        }
      }
    }
    if (blockDim.y > 1) __syncthreads();
  }
}

// Joins the splits' sums: 32 columns a block, whose 32 rows of threads take every 32nd split.  The order is fixed.
constexpr int kNormReduceRows = 32;
template <bool kBias>
__global__ void __launch_bounds__(32 * kNormReduceRows) norm_reduce_kernel(const NormReduceParams p) {
  __shared__ float shared[kBias ? 2 : 1][kNormReduceRows][33];
  const int i = blockIdx.x * 32 + threadIdx.x;
  float dw = 0.0f, db = 0.0f;
  if (i < p.d) {
    for (int s = threadIdx.y; s < p.splits; s += kNormReduceRows) {
      dw += p.partial[2ll * s * p.d + i];
      if (kBias) db += p.partial[2ll * s * p.d + p.d + i];
    }
  }
  shared[0][threadIdx.y][threadIdx.x] = dw;
  if (kBias) shared[kBias ? 1 : 0][threadIdx.y][threadIdx.x] = db;
  __syncthreads();
  if (threadIdx.y >= (kBias ? 2 : 1)) return;
  float sum = 0.0f;
#pragma unroll
  for (int r = 0; r < kNormReduceRows; ++r) sum += shared[threadIdx.y][r][threadIdx.x];
  void* out = threadIdx.y == 0 ? p.dweight : p.dbias;
  if (out == nullptr || i >= p.d) return;
  if (p.out_f32) static_cast<float*>(out)[i] = sum;
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(sum);
}

}  // namespace fsw
