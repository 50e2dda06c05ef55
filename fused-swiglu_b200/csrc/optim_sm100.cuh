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
constexpr int kAdamPart = kAdamThreads * kAdamGroup;       // elements of a thread block at a time

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
  int parts;  // of kAdamPart elements in a chunk
  uint32_t* status;  // of the bounded waits
  unsigned long long wait_limit_ns;
  int withhold;  // test aid: the first part's copies are left out
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

// ---- 8-bit floats with a block's scale ----

// Values of eight codes, without the scale.
__device__ __forceinline__ void decode_e4m3x8(uint2 q, Pair (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = i < 2 ? q.x : q.y;
    const uint16_t pair = static_cast<uint16_t>((i & 1) ? w >> 16 : w);
    uint32_t halves;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(halves) : "h"(pair));
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&halves));
    v[i] = make_pair(f.x, f.y);
  }
}

// An e5m2 is the upper byte of a half.
__device__ __forceinline__ void decode_e5m2x8(uint2 q, Pair (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t halves = __byte_perm(i < 2 ? q.x : q.y, 0u, (i & 1) ? 0x3424 : 0x1404);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&halves));
    v[i] = make_pair(f.x, f.y);
  }
}

// How a block whose largest magnitude has the fp32 bits `peak` is encoded: its scale, the power of two that brings its values
// to where the exponents of the 8-bit type, its subnormal ones too, are those of fp32, and what they have to come down by
// first, so that this power is a normal number: 2^-100 where the largest is above 2^14 or so, 2^-114 from 2^114 on (m alone), which
// the smaller values next to it have room for.  `top`: the type's exponent that the largest value gets; `low`: the difference
// of the types' biases.
struct BlockScale {
  float scale, factor, down;
};
__device__ __forceinline__ BlockScale block_scale(uint32_t peak, int top, int low) {
  const int field = max(static_cast<int>(peak >> 23), top + 1);  // keeps the scale normal
  BlockScale b;
  b.scale = field < 255 ? __uint_as_float(static_cast<uint32_t>(field - top) << 23) : __uint_as_float(0x7fc00000u);
  const int exponent = 254 + top - low - field;
  const int by = exponent >= 1 ? 0 : exponent >= -99 ? 100 : 114;
  b.down = __uint_as_float(static_cast<uint32_t>(127 - by) << 23);
  b.factor = __uint_as_float(static_cast<uint32_t>(exponent + by) << 23);
  return b;
}

// The bits that the 8-bit type keeps are the upper ones of t; random bits added below them round up as often as the rest is
// large.  The code comes in the uppermost byte.
__device__ __forceinline__ uint32_t encode_e4m3(float t, uint32_t bits) {
  const uint32_t x = __float_as_uint(t) + ((bits & 0xffffu) << 4);  // sign in bit 31, code in bits 20 to 26
  return (x << 4) | (x & 0x80000000u);
}
__device__ __forceinline__ uint32_t encode_e5m2(float t, float v, uint32_t bits) {
  const uint32_t x = (__float_as_uint(t) + ((bits >> 16) << 5)) << 3;  // code in bits 21 to 27
  return max(x, v > 0.0f ? 1u << 24 : 0u);
}
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
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

// Eight values as they lie in memory.
template <typename T>
struct RawGroup;
template <>
struct RawGroup<float> {
  float v[kAdamGroup];
  __device__ __forceinline__ void load(const float* p, bool whole, int n) { load_group(p, whole, n, v); }
  __device__ __forceinline__ void read(const float* p) {  // shared memory
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
  __device__ __forceinline__ void get(Pair (&out)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = make_pair(v[2 * i], v[2 * i + 1]);
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
  __device__ __forceinline__ void read(const __nv_bfloat16* p) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
  }
  __device__ __forceinline__ void get(Pair (&out)[4]) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = unpack_bf16x2(w[i]);
  }
};

template <typename T>
__device__ __forceinline__ void store_pairs(T* p, bool whole, int n, const Pair (&v)[4]) {
  float f[kAdamGroup];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 t = split(v[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
  store_group(p, whole, n, f);
}

// The moments of one element, each product and sum rounded on its own.
__device__ __forceinline__ void adam_moments(const AdamOptions& o, const AdamRates& r, float b1, float b2, float g, float& m, float& v) {
  g = __fmul_rn(g, r.scale);
  m = __fadd_rn(__fmul_rn(b1, m), __fmul_rn(o.one_minus_beta1, g));
  v = __fadd_rn(__fmul_rn(b2, v), __fmul_rn(o.one_minus_beta2, __fmul_rn(g, g)));
}

// Fast roots and quotients, off by a unit or two of fp32: p alone depends on them.  Under the root a second moment below the
// smallest normal number counts as that.
__device__ __forceinline__ float adam_root(float v) {
  float root;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(root) : "f"(v), "f"(0x1p-126f));
  asm("sqrt.approx.ftz.f32 %0, %0;" : "+f"(root));
  return root;
}
__device__ __forceinline__ float adam_inverse_root(float root) {
  float inverse;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(root));
  return inverse;
}

// fp32 moments.  P, G: types of parameters and gradients.  A thread has eight neighbours at a time; three blocks an SM
// keep enough on its way, and more of them are slower (3 x 45 M weights: three 595 us, four 599, five 645).  Bound by memory: bf16 weights and gradients with
// fp32 copies, 28 bytes an element, 3 x 45 M weights in 559 us, 6.8 TB/s; 224 tensors of 65 k in 64 us, 6.4 TB/s.
template <typename P, typename G, bool kMaster, int kCapacity>
__global__ void __launch_bounds__(kAdamThreads, 3) adamw32_kernel(const __grid_constant__ AdamTable<kCapacity> t) {
  using Weight = typename std::conditional<kMaster, float, P>::type;
  const AdamOptions& o = t.opt;
  grid_launch_dependents();
  grid_dependency_wait();
  const AdamRates r = adam_rates(o);
  const uint32_t chunks = t.first_chunk[t.count];
  const int chunk_size = t.parts * kAdamPart;
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t.first_chunk, t.count, chunk);
    const AdamTensor& a = t.tensors[k];
    const bool vector = a.numel >= 0;
    const long long base = static_cast<long long>(chunk - t.first_chunk[k]) * chunk_size;
    const int size = static_cast<int>(min((vector ? a.numel : ~a.numel) - base, static_cast<long long>(chunk_size)));
#pragma unroll 1
    for (int e = threadIdx.x * kAdamGroup; e < size; e += kAdamPart) {
      const int n = min(size - e, kAdamGroup);
      const bool whole = vector && n == kAdamGroup;
      const long long at = base + e;
      float m[kAdamGroup], v[kAdamGroup], g[kAdamGroup], p[kAdamGroup];
      load_group(static_cast<const float*>(a.exp_avg) + at, whole, n, m);
      load_group(static_cast<const float*>(a.exp_avg_sq) + at, whole, n, v);
      load_group(static_cast<const G*>(a.grad) + at, whole, n, g);
      load_group((kMaster ? reinterpret_cast<const Weight*>(a.master) : static_cast<const Weight*>(a.param)) + at, whole, n, p);
      if (r.skip) return;  // only here, where this is not waited for before the loads
#pragma unroll
      for (int i = 0; i < kAdamGroup; ++i) {
        adam_moments(o, r, o.beta1, o.beta2, g[i], m[i], v[i]);
        p[i] = fmaf(-r.step_size * m[i], adam_inverse_root(fmaf(adam_root(v[i]), r.inv_sqrt_correction2, o.eps)), p[i] * r.decay);
      }
      if (kMaster) store_group(a.master + at, whole, n, p);
      store_group(static_cast<P*>(a.param) + at, whole, n, p);
      store_group(static_cast<float*>(a.exp_avg) + at, whole, n, m);
      store_group(static_cast<float*>(a.exp_avg_sq) + at, whole, n, v);
    }
  }
}

// ---- 8-bit moments ----
//
// There is nearly as much to compute as to move, and a warp that waits for its loads does not compute: a part's values come
// by bulk copies into a ring of shared memory, asked for by a warp of their own while the eight others work on earlier
// parts.  A part at a tensor's end, or of a tensor whose pointers are not aligned, is loaded by its threads.
// 3 x 45 M bf16 weights with fp32 copies, 16 bytes an element: 351 to 367 us, 5.9 to 6.2 TB/s, 59 instructions an element on 68 % of the issue
// slots; with each warp loading its own values 467 us.  Places and blocks an SM: three of two 356 us, two of three 360, four of
// two 368, three of three 386.

constexpr int kAdam8Places = 3;
constexpr int kAdam8RingThreads = kAdamThreads + 32;
constexpr int kAdam8Blocks = 2;  // of an SM

struct Adam8Part {  // of one place: what it holds
  long long base;   // first element
  int k, size;      // tensor, elements
};

template <typename Weight, typename G>
struct Adam8Place {
  __align__(128) Weight p[kAdamPart];
  __align__(16) G g[kAdamPart];
  __align__(16) uint8_t m[kAdamPart], v[kAdamPart];
  __align__(16) float scale_m[kAdamPart / kAdamBlock], scale_v[kAdamPart / kAdamBlock];
};

template <typename Weight, typename G>
struct Adam8Shared {
  Adam8Place<Weight, G> place[kAdam8Places];
  Adam8Part part[kAdam8Places];
  unsigned long long full[kAdam8Places], empty[kAdam8Places];
  uint32_t abort_flag;
};

__device__ __forceinline__ void bulk_copy(void* dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// The part of a launch: copied where it is whole and aligned.
template <bool kRing, int kCapacity>
__device__ __forceinline__ Adam8Part adam8_part(const AdamTable<kCapacity>& t, uint32_t part) {
  const int k = find_tensor(t.first_chunk, t.count, part);
  const long long numel = t.tensors[k].numel, base = static_cast<long long>(part - t.first_chunk[k]) * kAdamPart;
  const int size = static_cast<int>(min((numel >= 0 ? numel : ~numel) - base, static_cast<long long>(kAdamPart)));
  return Adam8Part{base, kRing && numel >= 0 && size == kAdamPart ? k : ~k, size};
}

// One thread asks for this block's parts, a ring ahead of those that work on them.  Behind the last, or where a wait gave up,
// it sees to it that no copy is on its way any more.
template <typename Weight, typename G, bool kMaster, int kCapacity>
__device__ __forceinline__ void adam8_ask(const AdamTable<kCapacity>& t, Adam8Shared<Weight, G>& sh, const Watchdog& wd) {
  const uint32_t parts = t.first_chunk[t.count];
  int i = 0;
  for (uint32_t part = blockIdx.x; part < parts; part += gridDim.x, ++i) {
    const int at = i % kAdam8Places;
    const uint32_t full = smem_u32(&sh.full[at]);
    if (i >= kAdam8Places && !wd.wait(smem_u32(&sh.empty[at]), (i / kAdam8Places - 1) & 1, kSiteAdamRing)) break;
    const Adam8Part here = adam8_part<true>(t, part);
    sh.part[at] = here;
    if (here.k < 0) {
      mbar_arrive(full);
      continue;
    }
    if (t.withhold && part == 0) {
      mbar_arrive_expect_tx(full, 16);
      continue;
    }
    const AdamTensor& a = t.tensors[here.k];
    const long long base = here.base, block = base / kAdamBlock;
    Adam8Place<Weight, G>& place = sh.place[at];
    mbar_arrive_expect_tx(full, sizeof(place.p) + sizeof(place.g) + sizeof(place.m) + sizeof(place.v) + sizeof(place.scale_m) +
                                    sizeof(place.scale_v));
    bulk_copy(place.p, (kMaster ? reinterpret_cast<const Weight*>(a.master) : static_cast<const Weight*>(a.param)) + base,
              sizeof(place.p), full);
    bulk_copy(place.g, static_cast<const G*>(a.grad) + base, sizeof(place.g), full);
    bulk_copy(place.m, static_cast<const uint8_t*>(a.exp_avg) + base, sizeof(place.m), full);
    bulk_copy(place.v, static_cast<const uint8_t*>(a.exp_avg_sq) + base, sizeof(place.v), full);
    bulk_copy(place.scale_m, a.exp_avg_scale + block, sizeof(place.scale_m), full);
    bulk_copy(place.scale_v, a.exp_avg_sq_scale + block, sizeof(place.scale_v), full);
  }
  const unsigned long long t0 = global_timer_ns();
  for (int j = max(0, i - kAdam8Places); j < i; ++j) {
    while (!mbar_try_wait(smem_u32(&sh.full[j % kAdam8Places]), (j / kAdam8Places) & 1) &&
           !(wd.aborted() && global_timer_ns() - t0 > kDrainLimitNs)) {
      if (global_timer_ns() - t0 > wd.limit_ns) wd.give_up(kSiteAdamRing);
    }
  }
}

// Eight elements of a thread.
struct AdamGroup {
  Pair m[4], v[4], p[4], g[4];
};

// m, v and p from b1 and b2 times m and v, and the gradient, two at a time where that may be (pairs' products and sums may
// come fused, which the moments' must not).
__device__ __forceinline__ void adam_step(const AdamOptions& o, const AdamRates& r, float b1, float b2, AdamGroup& a) {
  const Pair inv = both(r.inv_sqrt_correction2), eps = both(o.eps), rate = both(-r.step_size), decay = both(r.decay);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 g = split(a.g[i]);
    float2 m = split(a.m[i]), v = split(a.v[i]);
    adam_moments(o, r, b1, b2, g.x, m.x, v.x);
    adam_moments(o, r, b1, b2, g.y, m.y, v.y);
    a.m[i] = make_pair(m.x, m.y);
    a.v[i] = make_pair(v.x, v.y);
    const float2 root = split(fma2(make_pair(adam_root(v.x), adam_root(v.y)), inv, eps));
    a.p[i] = fma2(a.m[i] * rate, make_pair(adam_inverse_root(root.x), adam_inverse_root(root.y)), a.p[i] * decay);
  }
}

// P, G: types of parameters and gradients.  A warp takes one block of 256 elements of a part, each thread eight neighbours, so
// that a block's largest magnitudes are one reduction over the warp.
template <typename P, typename G, bool kMaster, bool kRing, int kCapacity>
__global__ void __launch_bounds__(kRing ? kAdam8RingThreads : kAdamThreads, kRing ? kAdam8Blocks : 4) adamw8_kernel(const __grid_constant__ AdamTable<kCapacity> t) {
  using Weight = typename std::conditional<kMaster, float, P>::type;
  extern __shared__ __align__(128) unsigned char memory[];
  Adam8Shared<Weight, G>& sh = *reinterpret_cast<Adam8Shared<Weight, G>*>(memory);
  const AdamOptions& o = t.opt;
  const Watchdog wd{&sh.abort_flag, t.status, t.wait_limit_ns};
  if (kRing) {
    if (threadIdx.x == 0) {
      for (int i = 0; i < kAdam8Places; ++i) {
        mbar_init(smem_u32(&sh.full[i]), 1);
        mbar_init(smem_u32(&sh.empty[i]), kAdamThreads / 32);
      }
      sh.abort_flag = 0;
      fence_mbar_init();
    }
    __syncthreads();
  }
  grid_launch_dependents();
  grid_dependency_wait();
  const AdamRates r = adam_rates(o);
  if (kRing && r.skip) return;
  if (kRing && threadIdx.x >= kAdamThreads) {
    if (threadIdx.x == kAdamThreads) adam8_ask<Weight, G, kMaster>(t, sh, wd);
    return;
  }
  const uint32_t parts = t.first_chunk[t.count];
  const int e = threadIdx.x * kAdamGroup, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int at = 0;
  uint32_t phase = 0;
  for (uint32_t part = blockIdx.x; part < parts; part += gridDim.x) {
    // a warp that gives up leaves what it has not read as it was
    if (kRing && !__all_sync(0xffffffffu, wd.wait(smem_u32(&sh.full[at]), phase, kSiteAdamRing))) return;
    const Adam8Part here = kRing ? sh.part[at] : adam8_part<false>(t, part);
    const bool copied = kRing && here.k >= 0;
    const int k = copied ? here.k : ~here.k;
    const AdamTensor& a = t.tensors[k];
    const int n = min(max(here.size - e, 0), kAdamGroup);
    const bool some = warp * kAdamBlock < here.size;  // of the warp's block
    const long long first = here.base + e, block = here.base / kAdamBlock + warp;
    uint2 codes_m, codes_v;
    float scale_m = 0.0f, scale_v = 0.0f;
    RawGroup<Weight> raw_p;
    RawGroup<G> raw_g;
    bool whole = true;
    if (copied) {
      const Adam8Place<Weight, G>& place = sh.place[at];
      raw_p.read(place.p + e);
      raw_g.read(place.g + e);
      codes_m = *reinterpret_cast<const uint2*>(place.m + e);
      codes_v = *reinterpret_cast<const uint2*>(place.v + e);
      scale_m = place.scale_m[warp];
      scale_v = place.scale_v[warp];
    } else {
      whole = a.numel >= 0 && n == kAdamGroup;
      raw_p.load((kMaster ? reinterpret_cast<const Weight*>(a.master) : static_cast<const Weight*>(a.param)) + first, whole, n);
      raw_g.load(static_cast<const G*>(a.grad) + first, whole, n);
      codes_m = load_codes(static_cast<const uint8_t*>(a.exp_avg) + first, whole, n);
      codes_v = load_codes(static_cast<const uint8_t*>(a.exp_avg_sq) + first, whole, n);
      if (some) {
        scale_m = a.exp_avg_scale[block];
        scale_v = a.exp_avg_sq_scale[block];
      }
    }
    if (kRing) {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sh.empty[at]));
      if (++at == kAdam8Places) {
        at = 0;
        phase ^= 1;
      }
    }
    if (!some) continue;
    if (!kRing && r.skip) return;  // only here, where this is not waited for before the loads
    AdamGroup q;
    decode_e4m3x8(codes_m, q.m);
    decode_e5m2x8(codes_v, q.v);
    raw_g.get(q.g);
    raw_p.get(q.p);
    // the scale is a power of two: b times the scale, and that times the code, rounds as b times the value does
    adam_step(o, r, o.beta1 * scale_m, o.beta2 * scale_v, q);
    uint32_t peak_m = 0, peak_v = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 m = split(q.m[i]), v = split(q.v[i]);
      peak_m = max(peak_m, max(__float_as_uint(m.x) & 0x7fffffffu, __float_as_uint(m.y) & 0x7fffffffu));
      peak_v = max(peak_v, max(__float_as_uint(v.x), __float_as_uint(v.y)));
    }
    const BlockScale bm = block_scale(__reduce_max_sync(0xffffffffu, peak_m), 7, 120);
    const BlockScale bv = block_scale(__reduce_max_sync(0xffffffffu, peak_v), 14, 112);
    if (kMaster) store_pairs(a.master + first, whole, n, q.p);
    store_pairs(static_cast<P*>(a.param) + first, whole, n, q.p);
    if (lane == 0) {
      a.exp_avg_scale[block] = bm.scale;
      a.exp_avg_sq_scale[block] = bv.scale;
    }
    const unsigned long long group = (t.first_block[k] + block) * (kAdamBlock / kAdamGroup) + lane;
    const uint32_t h = mix32(static_cast<uint32_t>(group) ^ (static_cast<uint32_t>(group >> 32) * odd_multiplier(0)) ^ r.key);
    const Pair fm = both(bm.factor), fv = both(bv.factor);
    if (fminf(bm.down, bv.down) < 1.0f) {
      const Pair down_m = both(bm.down), down_v = both(bv.down);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        q.m[i] = q.m[i] * down_m;
        q.v[i] = q.v[i] * down_v;
      }
    }
    uint32_t cm[kAdamGroup], cv[kAdamGroup];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 tm = split(q.m[i] * fm), tv = split(q.v[i] * fv), v = split(q.v[i]);
      const uint32_t b0 = h * odd_multiplier(2 * i), b1 = h * odd_multiplier(2 * i + 1);
      cm[2 * i] = encode_e4m3(tm.x, b0);
      cm[2 * i + 1] = encode_e4m3(tm.y, b1);
      cv[2 * i] = encode_e5m2(tv.x, v.x, b0);
      cv[2 * i + 1] = encode_e5m2(tv.y, v.y, b1);
    }
    store_codes(static_cast<uint8_t*>(a.exp_avg) + first, whole, n,
                make_uint2(upper_bytes(cm[0], cm[1], cm[2], cm[3]), upper_bytes(cm[4], cm[5], cm[6], cm[7])));
    store_codes(static_cast<uint8_t*>(a.exp_avg_sq) + first, whole, n,
                make_uint2(upper_bytes(cv[0], cv[1], cv[2], cv[3]), upper_bytes(cv[4], cv[5], cv[6], cv[7])));
  }
}

// ---- 2-norm over many gradients ----

constexpr int kGradChunk = 4 * kAdamPart;  // elements of a thread block at a time
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

// Squares of this thread's elements of kParts parts of a chunk from part `first` on, all loaded before the first is used: in
// fp32 over two parts, sixteen elements, in fp64 from there on.  (3 x 45 M fp32 gradients 80 us, 6.8 TB/s, bound by memory; 224 of
// 65 k bf16, from the L2 cache, 10.5 to 11.5 us, most of it the two launches' and each block's search for its tensors.)
template <int kParts, bool kScaled, typename T>
__device__ __forceinline__ double sum_squares(const T* p, bool vector, int size, int first, float& least) {
  RawGroup<T> raw[kParts];
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    const int e = (first + i) * kAdamPart + threadIdx.x * kAdamGroup, n = min(max(size - e, 0), kAdamGroup);
    raw[i].load(p + e, vector && n == kAdamGroup, n);
  }
  double sum = 0.0;
#pragma unroll
  for (int i = 0; i < kParts; i += 2) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      Pair v[4];
      raw[i + j].get(v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 f = split(v[k]);
        if (kScaled) f = make_float2(f.x * 0x1p100f, f.y * 0x1p100f);
        s = fmaf(f.x, f.x, s);
        s = fmaf(f.y, f.y, s);
      }
    }
    if ((first + i) * kAdamPart + static_cast<int>(threadIdx.x) * kAdamGroup < size) least = fminf(least, s);
    sum += static_cast<double>(s);
  }
  return sum;
}

// The same for sums that may have lost squares below fp32's normal numbers: below kLeastSum all of sixteen values are below
// 2^-45, and 2^100 times them have squares within the normal numbers, down to the smallest values that there are.  Read a
// second time: what every gradient passes keeps its loads together (with the choice in place, 3 x 45 M fp32 gradients took
// 84 us in the place of 80, bf16 48 for 42.5; gradients of nothing but zeros, which all come here, take 95).
constexpr float kLeastSum = 0x1p-90f;
template <typename T>
__device__ __forceinline__ double sum_squares_again(const T* p, bool vector, int size) {
  double sum = 0.0;
#pragma unroll 1
  for (int first = 0; first < kGradChunk / kAdamPart; first += 2) {
    float least = kLeastSum;
    const double s = sum_squares<2, false>(p, vector, size, first, least);
    sum += least < kLeastSum ? sum_squares<2, true>(p, vector, size, first, least) * 0x1p-200 : s;
  }
  return sum;
}

// The squares of every gridDim.x-th chunk, over the block.
template <int kCapacity>
__device__ __forceinline__ double sum_chunks(const GradTable<kCapacity>& t, double* shared) {
  double sum = 0.0;
  const uint32_t chunks = t.first_chunk[t.count];
  for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int k = find_tensor(t.first_chunk, t.count, chunk);
    const GradTensor& a = t.tensors[k];
    const long long base = static_cast<long long>(chunk - t.first_chunk[k]) * kGradChunk;
    const int size = static_cast<int>(min(a.numel - base, static_cast<long long>(kGradChunk)));
    float least = kLeastSum;
    double s;
    if (a.f32) {
      const float* const g = static_cast<const float*>(a.grad) + base;
      s = sum_squares<2, false>(g, a.vector, size, 0, least);
      s += sum_squares<2, false>(g, a.vector, size, 2, least);
      if (least < kLeastSum) s = sum_squares_again(g, a.vector, size);
    } else {
      const __nv_bfloat16* const g = static_cast<const __nv_bfloat16*>(a.grad) + base;
      s = sum_squares<4, false>(g, a.vector, size, 0, least);
      if (least < kLeastSum) s = sum_squares_again(g, a.vector, size);
    }
    sum += s;
  }
  return block_sum(sum, shared);
}

// out[0] = the norm, out[1] = min(1, max_norm / (norm + 1e-6)); NaN where the norm is not finite.
__device__ __forceinline__ void write_norm(double sum, float max_norm, float* out) {
  const double norm = sqrt(sum);
  out[0] = static_cast<float>(norm);
  out[1] = isfinite(out[0]) ? static_cast<float>(fmin(1.0, static_cast<double>(max_norm) / (norm + 1e-6)))
                            : __uint_as_float(0x7fc00000u);
}

template <int kCapacity>
__global__ void __launch_bounds__(kAdamThreads) grad_norm_kernel(const __grid_constant__ GradTable<kCapacity> t) {
  __shared__ double shared[kAdamThreads / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const double sum = sum_chunks(t, shared);
  if (threadIdx.x == 0) t.slots[blockIdx.x] = t.accumulate ? t.slots[blockIdx.x] + sum : sum;
}

__global__ void __launch_bounds__(kAdamThreads) grad_norm_finish_kernel(const double* slots, int count, float max_norm,
                                                                       float* out) {
  __shared__ double shared[kAdamThreads / 32];
  double sum = 0.0;
  grid_launch_dependents();
  grid_dependency_wait();
  for (int i = threadIdx.x; i < count; i += kAdamThreads) sum += slots[i];
  sum = block_sum(sum, shared);
  if (threadIdx.x == 0) write_norm(sum, max_norm, out);
}

// Few chunks: the blocks are one cluster, which joins their sums in the memory of its first, in place of a second launch.
template <int kCapacity>
__global__ void __launch_bounds__(kAdamThreads) grad_norm_few_kernel(const __grid_constant__ GradTable<kCapacity> t, float max_norm,
                                                                    float* out) {
  __shared__ double shared[kAdamThreads / 32], joined[kFewBlocks];
  cluster_arrive();
  grid_launch_dependents();
  grid_dependency_wait();
  const double sum = sum_chunks(t, shared);
  cluster_wait();  // all blocks have started: their memory can be written
  if (threadIdx.x == 0) store_cluster(map_to_cta(smem_u32(&joined[blockIdx.x]), 0), sum);
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (blockIdx.x > 0 || threadIdx.x > 0) return;
  double total = 0.0;
  for (int r = 0; r < kFewBlocks; ++r) total += joined[r];
  write_norm(total, max_norm, out);
}

}  // namespace fsw
