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
#include <cuda_fp16.h>
#include <cstdint>
#include <type_traits>

#include "ptx_sm100.cuh"
#include "vector_io_sm100.cuh"

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
  long long numel;  // negative (its complement) where some pointer is not aligned to eight of its elements
};

struct AdamOptions {
  double log_beta1, log_beta2;  // for bias corrections of a step count on the device
  float lr, beta1, one_minus_beta1, beta2, one_minus_beta2, eps, weight_decay;
  float step_size, inv_sqrt_correction2;  // lr / (1 - b1^t), 1 / sqrt(1 - b2^t) where lr and t are the host's
  const float* lr_device;
  const long long* step_device;
  const float* grad_scale;
  uint32_t seed_lo, seed_hi, step_lo;
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

// m, v and p of one element from b1 m, b2 v and the gradient.  The root and the quotient are the fast ones, off by a few
// units of fp32: p alone depends on them.
__device__ __forceinline__ void adam_element(const AdamOptions& o, const AdamRates& r, float g, float old_m, float old_v,
                                             float& m, float& v, float& p) {
  g = __fmul_rn(g, r.scale);
  m = __fadd_rn(old_m, __fmul_rn(o.one_minus_beta1, g));
  v = __fadd_rn(old_v, __fmul_rn(o.one_minus_beta2, __fmul_rn(g, g)));
  float root, quotient;
  asm("sqrt.approx.f32 %0, %1;" : "=f"(root) : "f"(v));
  root = fmaf(root, r.inv_sqrt_correction2, o.eps);
  asm("div.approx.ftz.f32 %0, %1, %2;" : "=f"(quotient) : "f"(r.step_size * m), "f"(root));
  p = fmaf(p, r.decay, -quotient);
}

// ---- 8-bit floats with a block's scale ----

// Values of eight codes, without the scale.
__device__ __forceinline__ void decode_e4m3x8(uint2 q, float (&v)[kAdamGroup]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? q.x : q.y;
    const uint16_t pair = static_cast<uint16_t>((i & 1) ? w >> 16 : w);
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(pair));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&halves));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// An e5m2 is the upper byte of a half.
__device__ __forceinline__ void decode_e5m2x8(uint2 q, float (&v)[kAdamGroup]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t halves = __byte_perm(i < 2 ? q.x : q.y, 0u, (i & 1) ? 0x3424 : 0x1404);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&halves));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// The scale of a block whose largest magnitude has the fp32 bits `peak`, and its inverse; the largest value comes
// below 2^(top + 1).  The lower bound on the exponent keeps both normal.
__device__ __forceinline__ float2 block_scale(uint32_t peak, uint32_t top) {
  const uint32_t field = max(peak >> 23, top + 1);
  if (field >= 255u) return make_float2(__uint_as_float(0x7fc00000u), 0.0f);
  return make_float2(__uint_as_float((field - top) << 23), __uint_as_float((254u + top - field) << 23));
}

// A value brought to where the exponents of the 8-bit type, its subnormal ones too, are those of fp32; then the bits that
// the type keeps are the upper ones, and random bits added below them round up as often as the rest is large.
__device__ __forceinline__ uint32_t encode_e4m3(float m, float inverse, uint32_t bits) {
  const float t = m * inverse * 0x1p-120f;
  const uint32_t x = (__float_as_uint(t) + ((bits & 0xffffu) << 4)) >> 20;  // sign in bit 11, code in bits 0 to 6
  return (x & 0x7fu) | ((x >> 4) & 0x80u);
}

__device__ __forceinline__ uint32_t encode_e5m2(float v, float inverse, uint32_t bits) {
  const float t = v * inverse * 0x1p-112f;
  const uint32_t code = (__float_as_uint(t) + ((bits >> 16) << 5)) >> 21;
  return max(code, min(__float_as_uint(v), 1u));
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

// Eight elements of one thread; `whole`: all of them exist and are reached by wide accesses.  A group at a tensor's end
// or of an unaligned tensor goes element by element.
template <typename T>
__device__ __forceinline__ void load_group(const T* p, bool whole, int n, float (&v)[kAdamGroup]) {
  if (whole) {
    load8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) v[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store_group(T* p, bool whole, int n, const float (&v)[kAdamGroup]) {
  if (whole) {
    store8(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) {
      if (i < n) p[i] = static_cast<T>(v[i]);
    }
  }
}

__device__ __forceinline__ uint2 load_codes(const uint8_t* p, bool whole, int n) {
  if (whole) return load_bytes8(p);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < kAdamGroup; ++i) {
    if (i < n) w[i >> 2] |= static_cast<uint32_t>(p[i]) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

__device__ __forceinline__ void store_codes(uint8_t* p, bool whole, int n, uint2 v) {
  if (whole) {
    store_bytes8(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kAdamGroup; ++i) {
    if (i < n) p[i] = static_cast<uint8_t>((i < 4 ? v.x : v.y) >> (8 * (i & 3)));
  }
}

// Where a warp is in a launch's tensors: at one block of 256 elements, this thread at its eight.
template <int kCapacity>
struct AdamCursor {
  const AdamTable<kCapacity>& t;
  uint32_t chunk;
  int part = 0, k = 0, n = 0;  // n: elements of this thread that exist
  long long at = 0;
  bool whole = false;

  // To the first block from (chunk, part) on that has elements; false behind the last.  The same for all lanes of a warp.
  __device__ __forceinline__ bool seek() {
    const uint32_t chunks = t.first_chunk[t.count];
    for (; chunk < chunks; chunk += gridDim.x, part = 0) {
      if (part == 0) k = find_tensor(t.first_chunk, t.count, chunk);
      const long long numel = t.tensors[k].numel >= 0 ? t.tensors[k].numel : ~t.tensors[k].numel;
      at = static_cast<long long>(chunk - t.first_chunk[k]) * kAdamChunk + (part * kAdamThreads + threadIdx.x) * kAdamGroup;
      if (part < kAdamChunk / (kAdamThreads * kAdamGroup) && numel > at / kAdamBlock * kAdamBlock) {
        const long long left = numel - at;
        n = left <= 0 ? 0 : left < kAdamGroup ? static_cast<int>(left) : kAdamGroup;
        whole = t.tensors[k].numel >= 0 && n == kAdamGroup;
        return true;
      }
    }
    return false;
  }
};

// Eight values as they lie in memory.
template <typename T>
struct RawGroup;
template <>
struct RawGroup<float> {
  float v[kAdamGroup];
  __device__ __forceinline__ void load(const float* p, bool whole, int n) { load_group(p, whole, n, v); }
  __device__ __forceinline__ void get(float (&out)[kAdamGroup]) const {
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) out[i] = v[i];
  }
};
template <>
struct RawGroup<__nv_bfloat16> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p, bool whole, int n) {
    if (whole) {
      asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                   : "l"(p));
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = 2 * i < n ? __bfloat16_as_ushort(p[2 * i]) : 0, hi = 2 * i + 1 < n ? __bfloat16_as_ushort(p[2 * i + 1]) : 0;
        w[i] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void get(float (&out)[kAdamGroup]) const { unpack_bf16x8(w, out); }
};

// P, G: types of parameters and gradients; kEight: 8-bit moments, else fp32 ones.  A warp takes one block of 256 elements at a
// time, each thread eight neighbours, so that a block's largest magnitudes are one reduction over the warp.  With 8-bit
// moments there is as much to compute as to move: the next block's values are on their way meanwhile.
template <typename P, typename G, bool kEight, bool kMaster, int kCapacity>
__global__ void __launch_bounds__(kAdamThreads, kEight ? 3 : 4) adamw_kernel(const __grid_constant__ AdamTable<kCapacity> t) {
  using Weight = typename std::conditional<kMaster, float, P>::type;
  const AdamOptions& o = t.opt;
  const AdamRates r = adam_rates(o);
  if (r.skip) return;
  AdamCursor<kCapacity> c{t, blockIdx.x};
  RawGroup<Weight> raw_p;
  RawGroup<G> raw_g;
  RawGroup<float> raw_m, raw_v;
  uint2 codes_m = make_uint2(0u, 0u), codes_v = codes_m;
  float scale_m = 0.0f, scale_v = 0.0f;
  auto fetch = [&]() {
    const AdamTensor& a = t.tensors[c.k];
    if (kEight) {
      codes_m = load_codes(static_cast<const uint8_t*>(a.exp_avg) + c.at, c.whole, c.n);
      codes_v = load_codes(static_cast<const uint8_t*>(a.exp_avg_sq) + c.at, c.whole, c.n);
      if (c.n > 0) {
        scale_m = a.exp_avg_scale[c.at / kAdamBlock];
        scale_v = a.exp_avg_sq_scale[c.at / kAdamBlock];
      }
    } else {
      raw_m.load(static_cast<const float*>(a.exp_avg) + c.at, c.whole, c.n);
      raw_v.load(static_cast<const float*>(a.exp_avg_sq) + c.at, c.whole, c.n);
    }
    raw_g.load(static_cast<const G*>(a.grad) + c.at, c.whole, c.n);
    raw_p.load(kMaster ? reinterpret_cast<const Weight*>(a.master) + c.at : static_cast<const Weight*>(a.param) + c.at, c.whole, c.n);
  };
  bool more = c.seek();
  if (kEight && more) fetch();
  while (more) {
    if (!kEight) fetch();
    const AdamTensor& a = t.tensors[c.k];
    const long long at = c.at, block = at / kAdamBlock;
    const unsigned long long group = (t.first_block[c.k] + block) * (kAdamBlock / kAdamGroup) + (threadIdx.x & 31);
    const int n = c.n;
    const bool whole = c.whole;
    float m[kAdamGroup], v[kAdamGroup], p[kAdamGroup], g[kAdamGroup];
    if (kEight) {
      decode_e4m3x8(codes_m, m);
      decode_e5m2x8(codes_v, v);
    } else {
      raw_m.get(m);
      raw_v.get(v);
    }
    raw_g.get(g);
    raw_p.get(p);
    // the scale is a power of two: b times the scale, and that times the code, rounds as b times the value does
    const float b1 = kEight ? o.beta1 * scale_m : o.beta1, b2 = kEight ? o.beta2 * scale_v : o.beta2;
    ++c.part;
    more = c.seek();
    if (kEight && more) fetch();
    uint32_t peak_m = 0, peak_v = 0;
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) {
      adam_element(o, r, g[i], __fmul_rn(b1, m[i]), __fmul_rn(b2, v[i]), m[i], v[i], p[i]);
      if (kEight) {
        peak_m = max(peak_m, __float_as_uint(m[i]) & 0x7fffffffu);
        peak_v = max(peak_v, __float_as_uint(v[i]) & 0x7fffffffu);
      }
    }
    if (kMaster) store_group(a.master + at, whole, n, p);
    store_group(static_cast<P*>(a.param) + at, whole, n, p);
    if (kEight) {
      peak_m = __reduce_max_sync(0xffffffffu, peak_m);
      peak_v = __reduce_max_sync(0xffffffffu, peak_v);
      const float2 cm = block_scale(peak_m, 7), cv = block_scale(peak_v, 14);
      const uint32_t h = mix32(static_cast<uint32_t>(group) ^ (static_cast<uint32_t>(group >> 32) * odd_multiplier(0)) ^ r.key);
      if ((threadIdx.x & 31) == 0) {
        a.exp_avg_scale[block] = cm.x;
        a.exp_avg_sq_scale[block] = cv.x;
      }
      uint2 qm = make_uint2(0u, 0u), qv = qm;
#pragma unroll
      for (int i = 0; i < kAdamGroup; ++i) {
        const uint32_t bits = h * odd_multiplier(i);
        (i < 4 ? qm.x : qm.y) |= encode_e4m3(m[i], cm.y, bits) << (8 * (i & 3));
        (i < 4 ? qv.x : qv.y) |= (encode_e5m2(v[i], cv.y, bits) & 0xffu) << (8 * (i & 3));
      }
      store_codes(static_cast<uint8_t*>(a.exp_avg) + at, whole, n, qm);
      store_codes(static_cast<uint8_t*>(a.exp_avg_sq) + at, whole, n, qv);
    } else {
      store_group(static_cast<float*>(a.exp_avg) + at, whole, n, m);
      store_group(static_cast<float*>(a.exp_avg_sq) + at, whole, n, v);
    }
  }
}

// ---- 2-norm over many gradients ----

constexpr int kGradNormSlots = 1184;  // partial sums of squares, one a thread block: eight for each of 148 SMs

struct GradTensor {
  const void* grad;
  long long numel;
  int f32;
  int vector;  // aligned to eight elements
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
  let_next_start();
  const uint32_t chunks = t.first_chunk[t.count];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t.first_chunk, t.count, chunk);
    const GradTensor& a = t.tensors[k];
    const long long at = static_cast<long long>(chunk - t.first_chunk[k]) * kAdamChunk + threadIdx.x * kAdamGroup;
    float g[2][kAdamGroup];
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const long long e = at + part * kAdamThreads * kAdamGroup;
      const long long left = a.numel - e;
      const int n = left <= 0 ? 0 : left < kAdamGroup ? static_cast<int>(left) : kAdamGroup;
      const bool whole = a.vector && n == kAdamGroup;
      if (a.f32) load_group(static_cast<const float*>(a.grad) + e, whole, n, g[part]);
      else load_group(static_cast<const __nv_bfloat16*>(a.grad) + e, whole, n, g[part]);
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) s = fmaf(g[0][i], g[0][i], s);
#pragma unroll
    for (int i = 0; i < kAdamGroup; ++i) s = fmaf(g[1][i], g[1][i], s);
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
  wait_for_previous();
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
