// Eight neighbouring values at a time, as fp32: 32 bytes of fp32 (the widest access of sm_100), 16 of bf16, 8 of bytes.
// Addresses are aligned to these sizes.  Streaming: what is read once does not stay in L1.
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx_sm100.cuh"

namespace fsw {

__device__ __forceinline__ void unpack_bf16x8(const uint32_t (&w)[4], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p));
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  uint32_t w[4];
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
               : "l"(p));
  unpack_bf16x8(w, v);
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
               "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(p), "r"(pack_bf16x2(v[0], v[1])), "r"(pack_bf16x2(v[2], v[3])),
               "r"(pack_bf16x2(v[4], v[5])), "r"(pack_bf16x2(v[6], v[7]))
               : "memory");
}

__device__ __forceinline__ uint2 load_bytes8(const void* p) {
  uint2 v;
  asm volatile("ld.global.L1::no_allocate.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

__device__ __forceinline__ void store_bytes8(void* p, uint2 v) {
  asm volatile("st.global.v2.b32 [%0], {%1, %2};" ::"l"(p), "r"(v.x), "r"(v.y) : "memory");
}

// V neighbouring values of a row as they lie in memory, V = 8 (aligned as above) or 1.
template <typename T, int V>
struct RawVector;
template <>
struct RawVector<float, 8> {
  float v[8];
  __device__ __forceinline__ void load(const float* p) { load8(p, v); }
  __device__ __forceinline__ void get(float* out) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = v[i];
  }
};
template <>
struct RawVector<__nv_bfloat16, 8> {
  uint32_t w[4];
  __device__ __forceinline__ void load(const __nv_bfloat16* p) {
    asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                 : "l"(p));
  }
  __device__ __forceinline__ void get(float* out) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      out[2 * i] = __uint_as_float(w[i] << 16);
      out[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};
template <>
struct RawVector<float, 1> {
  float v;
  __device__ __forceinline__ void load(const float* p) { v = *p; }
  __device__ __forceinline__ void get(float* out) const { out[0] = v; }
};
template <>
struct RawVector<__nv_bfloat16, 1> {
  __nv_bfloat16 v;
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { v = *p; }
  __device__ __forceinline__ void get(float* out) const { out[0] = __bfloat162float(v); }
};

template <int V, typename T>
__device__ __forceinline__ void store_vector(T* p, const float* v) {
  if constexpr (V == 8) {
    float t[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = v[i];
    store8(p, t);
  } else {
    *p = static_cast<T>(v[0]);
  }
}

}  // namespace fsw
