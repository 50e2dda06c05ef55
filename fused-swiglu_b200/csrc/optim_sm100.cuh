// One AdamW step over many tensors, and the 2-norm over many gradients with the factor that clips it.
//
//   g' = s g     m <- b1 m + (1 - b1) g'     v <- b2 v + (1 - b2) g'^2
//   p <- p (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
//
// in fp32 from the parameter's fp32 copy where there is one.  m and v are rounded after each product and sum (no fused
// multiply-add), so that they do not depend on how a compiler contracts them: the 8-bit moments below are discontinuous
// in them.
//
// 8-bit moments.  A tensor's moments are cut into blocks of 256 elements.  A block's scale is a power of two: the values
// of m are float8_e4m3fn times the scale, the largest below 2^8 of it, those of v float8_e5m2, the largest below 2^15 of
// it.  A power of two, because then a value that a step leaves alone is on the new grid whatever the block's new
// largest value is.  Rounding is stochastic: at b2 = 0.999 a step changes v by a thousandth of its distance from g'^2,
// against half a unit of an eighth, and to the nearest it would stand still; at random it is right on average.  v above
// zero never becomes zero, since the next division by its root would then be by eps alone.  Moments that are not finite
// make their block's scale NaN.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx_sm100.cuh"

namespace fsw {

constexpr int kAdamThreads = 256;
constexpr int kAdamGroup = 8;                              // elements of a thread at a time
constexpr int kAdamBlock = 256;                            // elements that share a scale: one warp's groups
constexpr int kAdamChunk = kAdamThreads * kAdamGroup * 2;  // elements of a thread block at a time

struct AdamTensor {
  void* param;
  const void* grad;
  void* exp_avg;
  void* exp_avg_sq;
  float* master;
  float* exp_avg_scale;
  float* exp_avg_sq_scale;
  long long numel;
};

struct AdamOptions {
  double log_beta1, log_beta2;  // for bias corrections of a step count on the device
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, weight_decay;
  float step_size, inv_sqrt_correction2;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t) where lr and t are the host's
  const float* lr_device;
  const long long* step_device;
  const float* grad_scale;
  uint32_t seed_lo, seed_hi, step_lo;
  int grad_dtype_f32;
};

template <int kCapacity>
struct AdamTable {
  AdamTensor tensors[kCapacity];
  uint32_t first_chunk[kCapacity + 1];  // of this launch's chunks; the last entry is their number
  long long first_block[kCapacity];     // of the call's blocks of 256: what the random bits are counted by
  int count;
  AdamOptions opt;
};

// 32 bits of a position, for the roundings of one group of eight elements: two rounds of xor-shift and multiplication.
__device__ __forceinline__ uint32_t mix32(uint32_t x) {
  x = (x ^ (x >> 16)) * 0xDDC24D79u;
  x = (x ^ (x >> 15)) * 0x77D0AC3Du;
  return x ^ (x >> 16);
}

// Element i of the group takes hash * odd_multiplier(i): the upper 16 bits round v, the lower 16 m.
__device__ __forceinline__ constexpr uint32_t odd_multiplier(int i) {
  constexpr uint32_t k[kAdamGroup] = {0x5ECD29B7u, 0xDB623B29u, 0x69758763u, 0x7D45CE1Du,
                                      0x74A1B41Du, 0x75BBB081u, 0x5AD24435u, 0x73B07CC5u};
  return k[i];
}

struct AdamRates {
  float step_size, inv_sqrt_correction2, decay, scale;
  uint32_t key;
  bool skip;
};

// What the step uses of its options, from the device's learning rate and step count where it has them.
__device__ __forceinline__ AdamRates adam_rates(const AdamOptions& o) {
  AdamRates r;
  const float lr = o.lr_device != nullptr ? *o.lr_device : o.lr;
  r.step_size = o.step_size;
  r.inv_sqrt_correction2 = o.inv_sqrt_correction2;
  uint32_t step = o.step_lo;
  if (o.step_device != nullptr) {
    // 1 - b^t as -expm1(t log b): exact to a few units in fp32 where b^t is close to one
    const long long t = *o.step_device;
    step = static_cast<uint32_t>(t);
    r.step_size = lr / -expm1f(static_cast<float>(static_cast<double>(t) * o.log_beta1));
    r.inv_sqrt_correction2 = rsqrtf(-expm1f(static_cast<float>(static_cast<double>(t) * o.log_beta2)));
  } else if (o.lr_device != nullptr) {
    r.step_size = o.step_size * lr;  // the host left 1 / (1 - b1^t)
  }
  r.decay = 1.0f - lr * o.weight_decay;
  r.scale = o.grad_scale != nullptr ? *o.grad_scale : 1.0f;
  r.skip = !isfinite(r.scale);
  r.key = mix32(o.seed_lo ^ mix32(step ^ o.seed_hi));
  return r;
}

// m, v and p of one element.
__device__ __forceinline__ void adam_element(const AdamOptions& o, const AdamRates& r, float g, float& m, float& v, float& p) {
  g = __fmul_rn(g, r.scale);
  m = __fadd_rn(__fmul_rn(o.beta1, m), __fmul_rn(o.one_minus_beta1, g));
  v = __fadd_rn(__fmul_rn(o.beta2, v), __fmul_rn(o.one_minus_beta2, __fmul_rn(g, g)));
  const float root = sqrtf(v) * r.inv_sqrt_correction2 + o.eps;
  p = p * r.decay - __fdividef(r.step_size * m, root);
}

// ---- 8-bit floats with a block's scale ----

__device__ __forceinline__ float decode_e4m3(uint32_t code, float scale) {
  // the exponent of the 8-bit type moved to where fp32 has it, subnormal values too
  const uint32_t bits = ((code & 0x7fu) << 20) | ((code & 0x80u) << 24);
  return __uint_as_float(bits) * 0x1p120f * scale;
}

__device__ __forceinline__ float decode_e5m2(uint32_t code, float scale) {
  return __uint_as_float(code << 21) * 0x1p112f * scale;
}

// The scale of a block whose largest magnitude has the fp32 bits `peak`, and its inverse; the largest value comes
// below 2^(top + 1).  The lower bound on the exponent keeps both normal.
__device__ __forceinline__ float2 block_scale(uint32_t peak, uint32_t top) {
  const uint32_t field = max(peak >> 23, top + 1);
  if (field >= 255u) return make_float2(__uint_as_float(0x7fc00000u), 0.0f);
  return make_float2(__uint_as_float((field - top) << 23), __uint_as_float((254u + top - field) << 23));
}

__device__ __forceinline__ uint32_t encode_e4m3(float m, float inverse, uint32_t random16) {
  const float t = fabsf(m) * inverse * 0x1p-120f;
  const uint32_t code = (__float_as_uint(t) + (random16 << 4)) >> 20;
  return (code & 0x7fu) | (__float_as_uint(m) >> 31 << 7);
}

__device__ __forceinline__ uint32_t encode_e5m2(float v, float inverse, uint32_t random16) {
  const float t = v * inverse * 0x1p-112f;
  const uint32_t code = (__float_as_uint(t) + (random16 << 5)) >> 21;
  return max(code, v > 0.0f ? 1u : 0u);
}

// The tensor that holds a chunk: the last whose first chunk is not behind it.
template <int kCapacity>
__device__ __forceinline__ int find_tensor(const uint32_t (&first)[kCapacity], int count, uint32_t chunk) {
  int lo = 0, hi = count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// P: type of the parameters.  A warp takes one block of 256 elements at a time, each thread eight neighbours.
template <typename P, bool kEight, int kCapacity>
__global__ void __launch_bounds__(kAdamThreads) adamw_kernel(const __grid_constant__ AdamTable<kCapacity> t) {
  const AdamOptions& o = t.opt;
  const AdamRates r = adam_rates(o);
  if (r.skip) return;
  const uint32_t chunks = t.first_chunk[t.count];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t.first_chunk, t.count, chunk);
    const AdamTensor& a = t.tensors[k];
    const long long base = static_cast<long long>(chunk - t.first_chunk[k]) * kAdamChunk;
    for (int part = 0; part < 2; ++part) {
      const long long at = base + (part * kAdamThreads + threadIdx.x) * kAdamGroup;
      const long long block = at / kAdamBlock;
      float m[kAdamGroup], v[kAdamGroup];
      uint32_t peak_m = 0, peak_v = 0;
      float sm = 0.0f, sv = 0.0f;
      if (kEight && at < a.numel) {
        sm = a.exp_avg_scale[block];
        sv = a.exp_avg_sq_scale[block];
      }
#pragma unroll
      for (int i = 0; i < kAdamGroup; ++i) {
        m[i] = v[i] = 0.0f;
        const long long e = at + i;
        if (e < a.numel) {
          if (kEight) {
            m[i] = decode_e4m3(static_cast<const uint8_t*>(a.exp_avg)[e], sm);
            v[i] = decode_e5m2(static_cast<const uint8_t*>(a.exp_avg_sq)[e], sv);
          } else {
            m[i] = static_cast<const float*>(a.exp_avg)[e];
            v[i] = static_cast<const float*>(a.exp_avg_sq)[e];
          }
          const float g = o.grad_dtype_f32 ? static_cast<const float*>(a.grad)[e]
                                           : __bfloat162float(static_cast<const __nv_bfloat16*>(a.grad)[e]);
          float p = a.master != nullptr ? a.master[e] : static_cast<float>(static_cast<const P*>(a.param)[e]);
          adam_element(o, r, g, m[i], v[i], p);
          if (a.master != nullptr) a.master[e] = p;
          static_cast<P*>(a.param)[e] = static_cast<P>(p);
          if (!kEight) {
            static_cast<float*>(a.exp_avg)[e] = m[i];
            static_cast<float*>(a.exp_avg_sq)[e] = v[i];
          }
          peak_m = max(peak_m, __float_as_uint(m[i]) & 0x7fffffffu);
          peak_v = max(peak_v, __float_as_uint(v[i]) & 0x7fffffffu);
        }
      }
      if (kEight) {
        peak_m = __reduce_max_sync(0xffffffffu, peak_m);
        peak_v = __reduce_max_sync(0xffffffffu, peak_v);
        if (at >= a.numel) continue;
        const float2 cm = block_scale(peak_m, 7), cv = block_scale(peak_v, 14);
        const unsigned long long group = (t.first_block[k] + block) * (kAdamBlock / kAdamGroup) + (threadIdx.x & 31);
        const uint32_t h = mix32(static_cast<uint32_t>(group) ^ (static_cast<uint32_t>(group >> 32) * odd_multiplier(0)) ^ r.key);
        if ((threadIdx.x & 31) == 0) {
          a.exp_avg_scale[block] = cm.x;
          a.exp_avg_sq_scale[block] = cv.x;
        }
#pragma unroll
        for (int i = 0; i < kAdamGroup; ++i) {
          if (at + i >= a.numel) break;
          const uint32_t bits = h * odd_multiplier(i);
          static_cast<uint8_t*>(a.exp_avg)[at + i] = static_cast<uint8_t>(encode_e4m3(m[i], cm.y, bits & 0xffffu));
          static_cast<uint8_t*>(a.exp_avg_sq)[at + i] = static_cast<uint8_t>(encode_e5m2(v[i], cv.y, bits >> 16));
        }
      }
    }
  }
}

// ---- 2-norm over many gradients ----

constexpr int kGradNormSlots = 1184;  // partial sums of squares, one a thread block: eight for each of 148 SMs

struct GradTensor {
  const void* grad;
  long long numel;
  int f32;
};

template <int kCapacity>
struct GradTable {
  GradTensor tensors[kCapacity];
  uint32_t first_chunk[kCapacity + 1];
  int count;
  int accumulate;  // a later launch of the same call adds to the slots
  double* slots;
};

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) s += shared[w];
  return s;
}

// Squares are summed in fp32 over a thread's elements of one chunk, and in fp64 from there on.
template <int kCapacity>
__global__ void __launch_bounds__(kAdamThreads) grad_norm_kernel(const __grid_constant__ GradTable<kCapacity> t) {
  __shared__ double shared[kAdamThreads / 32];
  double sum = 0.0;
  const uint32_t chunks = t.first_chunk[t.count];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t.first_chunk, t.count, chunk);
    const GradTensor& a = t.tensors[k];
    const long long base = static_cast<long long>(chunk - t.first_chunk[k]) * kAdamChunk;
    float s = 0.0f;
    for (int i = threadIdx.x; i < kAdamChunk; i += kAdamThreads) {
      if (base + i < a.numel) {
        const float g = a.f32 ? static_cast<const float*>(a.grad)[base + i]
                              : __bfloat162float(static_cast<const __nv_bfloat16*>(a.grad)[base + i]);
        s = fmaf(g, g, s);
      }
    }
    sum += static_cast<double>(s);
  }
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) t.slots[blockIdx.x] = t.accumulate ? t.slots[blockIdx.x] + sum : sum;
}

// out[0] = the norm, out[1] = min(1, max_norm / (norm + 1e-6)); NaN where the norm is not finite.
__global__ void __launch_bounds__(kAdamThreads) grad_norm_finish_kernel(const double* slots, int count, float max_norm,
                                                                       float* out) {
  __shared__ double shared[kAdamThreads / 32];
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += kAdamThreads) sum += slots[i];
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) {
    const double norm = sqrt(sum);
    out[0] = static_cast<float>(norm);
    out[1] = isfinite(out[0]) ? static_cast<float>(fmin(1.0, static_cast<double>(max_norm) / (norm + 1e-6)))
                              : __uint_as_float(0x7fc00000u);
  }
}

}  // namespace fsw
