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

template <typename T>
constexpr int kPerVector = 16 / static_cast<int>(sizeof(T));  // values of 16 bytes

// Two fp32 values in one register pair: sm_100 adds, multiplies and fuses two at a time, each rounded as on its own.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair make_pair(float lo, float hi) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(lo), "f"(hi));
  return p;
}
__device__ __forceinline__ Pair both(float x) { return make_pair(x, x); }
__device__ __forceinline__ float2 split(Pair p) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
  return f;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ float sum(Pair p) {
  const float2 f = split(p);
  return f.x + f.y;
}

// The values of 16 bytes, and back.
__device__ __forceinline__ void unpack16(uint4 w, Pair (&v)[2]) {
  v[0] = make_pair(__uint_as_float(w.x), __uint_as_float(w.y));
  v[1] = make_pair(__uint_as_float(w.z), __uint_as_float(w.w));
}
__device__ __forceinline__ Pair unpack_bf16x2(uint32_t w) {
  return make_pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ void unpack16(uint4 w, Pair (&v)[4]) {
  v[0] = unpack_bf16x2(w.x);
  v[1] = unpack_bf16x2(w.y);
  v[2] = unpack_bf16x2(w.z);
  v[3] = unpack_bf16x2(w.w);
}

__device__ __forceinline__ uint4 read16(uint32_t src_smem) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(src_smem));
  return w;
}
__device__ __forceinline__ void clear16(uint32_t dst_smem) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(dst_smem), "r"(0) : "memory");
}

__device__ __forceinline__ void store16(void* p, const Pair (&v)[2]) {
  const float2 a = split(v[0]), b = split(v[1]);
  *static_cast<float4*>(p) = make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ uint32_t pack_pair(Pair p) {
  const float2 f = split(p);
  return pack_bf16x2(f.x, f.y);
}
__device__ __forceinline__ void store16(void* p, const Pair (&v)[4]) {
  *static_cast<uint4*>(p) = make_uint4(pack_pair(v[0]), pack_pair(v[1]), pack_pair(v[2]), pack_pair(v[3]));
}

}  // namespace fsw
