// Layer norm and RMS norm of the rows of a matrix, forward and backward.
//
//   z = (x - mean) rstd      y = z w + b      rstd = 1 / sqrt(mean((x - mean)^2) + eps)
//   a = dy w                 dx = rstd (a - mean(a) - z mean(a z)) (+ res)      dw = sum_rows dy z      db = sum_rows dy
//
// RMS norm is the same with 0 in the place of mean and without the term mean(a).  Rows are read as bf16 or fp32; all
// sums, statistics and products are fp32, and each output is rounded once.  z is the difference first, then the product: of values
// close to the mean the difference is exact, where x rstd - mean rstd keeps the rounding of mean rstd (2e-5 at a mean of 1000
// deviations).
//
// Memory bound: forward reads and writes a row once, backward reads two or three and writes one, at 8 to 15 operations an
// element.  The variance is that of the centred values, from a second sum over the row as it lies on the SM.  Four forms:
//   short   rows of at most 32 vectors of 16 bytes: a part of a warp a row (200000 x 128 bf16, layer norm: forward 21 to 23 us,
//           against 63 of the wide form; backward 51 against 109)
//   wide    rows of whole 16-byte vectors up to 16384 columns (backward: 12288 bf16, 9216 fp32): rings of shared memory filled by
//           bulk copies
//   odd     other rows up to 8192 columns: the same rings, by the 16-byte granules that a row touches, element by element
//   any     what is longer: a row is read again for each pass over it
#pragma once

#include <cuda_bf16.h>
#include <cstdint>

#include "ptx_sm100.cuh"
#include "row_granules.h"
#include "vector_io_sm100.cuh"

namespace fsw {

__device__ __forceinline__ void store_shared(uint32_t at, float v) {
  asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void store_shared(uint32_t at, __nv_bfloat16 v) {
  asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(__bfloat16_as_ushort(v)) : "memory");
}

// Of the kernels that wait for rows on their way (below).
struct RingParams {
  uint32_t* status;  // where a wait that gave up is recorded
  unsigned long long wait_limit_ns;
  int places;
  int withhold;  // test aid: the first row of all is never copied
  int edge;      // rows that start anywhere: edge_rows
};

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
  long long y_step;  // bytes from a group's row to its next
  RingParams ring;
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
  int cluster;    // the grid is one cluster, which joins the splits itself and writes these:
  int grad_f32;
  void* dweight;  // NULL: not wanted
  void* dbias;    // NULL: not wanted
  long long dx_step;  // bytes from a group's row to its next
  RingParams ring;
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
  grid_launch_dependents();
  grid_dependency_wait();
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
  grid_launch_dependents();
  grid_dependency_wait();
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
  grid_launch_dependents();
  grid_dependency_wait();
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

// ---- a group of threads a row ----
//
// blockDim.x threads (a multiple of 32) take one row at a time, and blockDim.y such groups of a block rows of their own.

__device__ __forceinline__ void group_barrier() {
  asm volatile("bar.sync %0, %1;" ::"r"(threadIdx.y + 1), "r"(blockDim.x) : "memory");
}

// Two sums over a group, in a fixed order, known to its threads; kPair: of both parts, else of y alone.  `span`: the group's
// warps, rounded up to a power of two.  A group has two sets of slots and takes them in turn: who writes one again has
// passed the barrier of the other, which all reached after they had read the first.
template <bool kPair>
__device__ __forceinline__ float2 group_sums(float2 v, float2* slots, int span) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (kPair) v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  if (span == 1) return v;
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) slots[threadIdx.x >> 5] = v;
  group_barrier();
  const int at = lane & (span - 1);
  v = at < warps ? slots[at] : make_float2(0.0f, 0.0f);
  for (int o = span >> 1; o > 0; o >>= 1) {
    if (kPair) v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
    v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
  }
  return v;
}

__device__ __forceinline__ int round_up_pow2(int v) { return v <= 1 ? 1 : 1 << (32 - __clz(v - 1)); }

// ---- rows through shared memory ----
//
// A group's rows to come are on their way into its ring of S places: one thread asks for a row's arrays by bulk copies, S - 1
// rows ahead, and all wait for their bytes on the place's barrier.  The bytes on the way cost neither registers, which the sums
// over rows need, nor instructions of the threads that compute.  A place is free again once the group has met in the next
// row's reduction.

constexpr int kWideGroups = 24;       // most groups of a block, those of one warp
constexpr int kWideMultiGroups = 8;   // most groups of more than one warp: each has a barrier of its own
constexpr int kWidePlaces = 4;         // most places of a ring

struct WideShared {
  __align__(16) unsigned long long full[kWideGroups][kWidePlaces];
  float2 slots[kWideMultiGroups][2][32];  // of each warp of a group, in turn
  uint32_t abort_flag;
};

// Bytes from the start of its 16-byte granule to an address.
__device__ __forceinline__ uint32_t behind(const void* p) { return static_cast<uint32_t>(reinterpret_cast<uint64_t>(p)) & 15u; }

// A group's ring: `places` places of kArrays rows of `row_bytes`.  The present row's place and its barrier's phase advance
// row by row.
template <int kArrays>
struct RowRing {
  uint32_t data, bars, place_bytes, array_bytes, row_bytes;
  int places, at;
  uint32_t phase;
  Watchdog wd;

  __device__ __forceinline__ RowRing(WideShared& sh, unsigned char* ring, uint32_t slot_bytes, uint32_t bytes, const RingParams& p)
      : array_bytes(slot_bytes), row_bytes(bytes), places(p.places), at(0), phase(0),
        wd{&sh.abort_flag, p.status, p.wait_limit_ns} {
    place_bytes = kArrays * slot_bytes;
    data = smem_u32(ring) + threadIdx.y * places * place_bytes;
    bars = smem_u32(&sh.full[threadIdx.y][0]);
    if (threadIdx.x == 0) {
      for (int s = 0; s < places; ++s) mbar_init(bars + 8 * s, 1);
    }
    if (threadIdx.x + threadIdx.y == 0) sh.abort_flag = 0;
  }
  // Where the present row lies.
  __device__ __forceinline__ uint32_t here() const { return data + at * place_bytes; }
  // The place that the row before the present one had, and the row `places - 1` ahead gets.
  __device__ __forceinline__ int before() const { return at == 0 ? places - 1 : at - 1; }
  __device__ __forceinline__ void advance() {
    if (++at == places) {
      at = 0;
      phase ^= 1;
    }
  }
  // One thread of the group: ask for a row into a place; whether it did.
  __device__ __forceinline__ bool ask(int place, const void* const (&src)[kArrays], int arrays, bool withhold) const {
    if (wd.aborted()) return false;
    const uint32_t bar = bars + 8 * place;
    mbar_arrive_expect_tx(bar, row_bytes * arrays);
    if (withhold) return true;
#pragma unroll
    for (int i = 0; i < kArrays; ++i) {
      if (i < arrays) bulk_row(data + place * place_bytes + i * array_bytes, src[i], row_bytes, bar);
    }
    return true;
  }
  // The same for rows that start anywhere: whole granules of 16 bytes, so that a row lies in its place as far behind a granule's
  // start as in memory.  What the granules hold beyond the row belongs to its neighbours.
  template <typename T>
  __device__ __forceinline__ bool ask_granules(int place, const T* const (&src)[kArrays], int arrays) const {
    if (wd.aborted()) return false;
    const uint32_t bar = bars + 8 * place;
    uint32_t size[kArrays], bytes = 0;
#pragma unroll
    for (int i = 0; i < kArrays; ++i) {
      size[i] = i < arrays ? (behind(src[i]) + row_bytes + 15u) & ~15u : 0u;
      bytes += size[i];
    }
    mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
    for (int i = 0; i < kArrays; ++i) {
      if (i < arrays) bulk_row(data + place * place_bytes + i * array_bytes, reinterpret_cast<const char*>(src[i]) - behind(src[i]), size[i], bar);
    }
    return true;
  }
  // The first rows of all and the last (edge_rows) have no neighbours on one side: the elements of their granules there, fewer
  // than 16 bytes, are copied one by one.
  template <typename T>
  __device__ __noinline__ bool ask_edge(int place, const T* x, const T* dy, const T* res, int arrays, int d, bool first, bool last,
                                        bool withhold) const {
    if (wd.aborted()) return false;
    const uint32_t bar = bars + 8 * place;
    const T* const src[3] = {x, dy, res};
    uint32_t bytes = withhold ? 16 : 0;
    for (int turn = 0; turn < 2; ++turn) {  // what a barrier is to expect it is told before the copies begin
      if (turn == 1) mbar_arrive_expect_tx(bar, bytes);
      for (int i = 0; i < arrays; ++i) {
        const uint64_t begin = reinterpret_cast<uint64_t>(src[i]), end = begin + static_cast<uint64_t>(d) * sizeof(T);
        const RowGranules g(begin, end, first, last);
        const uint32_t here = data + place * place_bytes + i * array_bytes, size = g.bytes();
        if (turn == 1) {
          if (size > 0 && !withhold) bulk_row(here + static_cast<uint32_t>(g.lo - g.granule), reinterpret_cast<const void*>(g.lo), size, bar);
          continue;
        }
        if (!withhold) bytes += size;
        for (uint64_t q = begin; first && q < g.lo && q < end; q += sizeof(T)) {
          store_shared(here + static_cast<uint32_t>(q - g.granule), *reinterpret_cast<const T*>(q));
        }
        for (uint64_t q = g.hi < begin ? begin : g.hi; last && q < end; q += sizeof(T)) {
          store_shared(here + static_cast<uint32_t>(q - g.granule), *reinterpret_cast<const T*>(q));
        }
      }
    }
    fence_proxy_async();  // the place's next row may come over these elements by a bulk copy, which this thread asks for
    return true;
  }
  __device__ __forceinline__ void wait() const { wd.wait(bars + 8 * at, phase, kSiteRowRing); }
  // After a wait that gave up: the last of the `asked` rows may still be on their way.
  __device__ __noinline__ void drain(int asked) const {
    const unsigned long long t0 = global_timer_ns();
    for (int n = max(0, asked - places); n < asked; ++n) {
      while (!mbar_try_wait(bars + 8 * (n % places), (n / places) & 1) && global_timer_ns() - t0 < kDrainLimitNs) {
      }
    }
  }
  static __device__ __forceinline__ void bulk_row(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
  }
};

// Vectors may be what the kernel before this one is still writing while these blocks come up (an optimiser's step in front of a
// norm): they are read by ordinary loads, behind grid_dependency_wait, not by way of the non-coherent path, which asks for
// data that nobody writes while the kernel lives.  The pointer is made known behind the wait, so that a load of it, which the
// compiler may otherwise move and issue early, stays there.
__device__ __forceinline__ const void* behind_wait(const void* p) {
  const void* q;
  asm volatile("mov.b64 %0, %1;" : "=l"(q) : "l"(p) : "memory");
  return q;
}
__device__ __forceinline__ float4 load_columns(const float4* p) {
  float4 f;
  asm("ld.global.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w) : "l"(p));
  return f;
}
__device__ __forceinline__ uint32_t load_columns(const uint32_t* p) {
  uint32_t w;
  asm("ld.global.b32 %0, [%1];" : "=r"(w) : "l"(p));
  return w;
}

// What a thread keeps of a weight or bias vector: bf16 values as they are, and few fp32 ones; many fp32 ones come from the L1
// cache row by row.  A missing vector is bf16 ones or zeros.  `init` is called behind grid_dependency_wait.
template <typename W, int N, int P, bool kKeep = true>
struct Columns;
template <int N, int P>
struct Columns<float, N, P, true> {
  Pair w[N][P / 2];
  __device__ __forceinline__ void init(const void* given, uint32_t, int d) {
    const void* const p = behind_wait(given);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * P;
#pragma unroll
      for (int i = 0; i < P / 4; ++i) {
        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (c < d) f = load_columns(reinterpret_cast<const float4*>(static_cast<const float*>(p) + c) + i);
        w[j][2 * i] = make_pair(f.x, f.y);
        w[j][2 * i + 1] = make_pair(f.z, f.w);
      }
    }
  }
  __device__ __forceinline__ void get(int j, bool, Pair (&v)[P / 2]) const {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) v[i] = w[j][i];
  }
};
template <int N, int P, bool kKeep>
struct Columns<__nv_bfloat16, N, P, kKeep> {
  uint32_t w[N][P / 2];
  __device__ __forceinline__ void init(const void* given, uint32_t none, int d) {
    const void* const p = behind_wait(given);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = (j * blockDim.x + threadIdx.x) * P;
      const uint32_t* q = reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(p) + c);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) w[j][i] = p != nullptr && c < d ? load_columns(q + i) : none;
    }
  }
  __device__ __forceinline__ void get(int j, bool, Pair (&v)[P / 2]) const {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) v[i] = unpack_bf16x2(w[j][i]);
  }
};
template <int N, int P>
struct Columns<float, N, P, false> {
  const float* q;
  __device__ __forceinline__ void init(const void* given, uint32_t, int) {
    q = static_cast<const float*>(behind_wait(given)) + threadIdx.x * P;
  }
  __device__ __forceinline__ void get(int j, bool valid, Pair (&v)[P / 2]) const {
#pragma unroll
    for (int i = 0; i < P / 4; ++i) {
      float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (valid) f = load_columns(reinterpret_cast<const float4*>(q + j * blockDim.x * P) + i);
      v[2 * i] = make_pair(f.x, f.y);
      v[2 * i + 1] = make_pair(f.z, f.w);
    }
  }
};

// Sums over rows are fp32 within a block, whose threads hold them in registers; the blocks' sums, up to 296 of them, are joined
// with what each addition drops kept beside the sum (Knuth's two-sum), and rounded once: in fp32 most of a gradient's error came
// from there (1000 x 1003: 1.3e-7 against 6e-8).  Two-sums, because conversions to fp64 cost more than their additions: 8 x 4096 in a
// graph 5.9 us, 6.6 with every part converted, 5.6 in fp32; the reducing kernel takes 0.1 to 0.3 us longer than in fp32.
struct JoinedSum {
  float sum, rest;
  __device__ __forceinline__ void add(float v) {
    const float t = sum + v, taken = t - sum;
    rest += (sum - (t - taken)) + (v - taken);
    sum = t;
  }
  __device__ __forceinline__ double value() const {
    return isfinite(sum) ? static_cast<double>(sum) + static_cast<double>(rest) : static_cast<double>(sum);
  }
};
__device__ __forceinline__ void store_gradient(void* out, int i, bool f32, double v) {
  if (f32) static_cast<float*>(out)[i] = static_cast<float>(v);
  else static_cast<__nv_bfloat16*>(out)[i] = __double2bfloat16(v);
}

// The end of a backward kernel whose grid is one cluster: behind the cluster's barrier every block knows what the others wrote,
// and takes its share of the columns.  In the order of the blocks; by way of L2, where the sums are.
template <bool kLayer>
__device__ __forceinline__ void join_in_cluster(const NormBackwardParams& p) {
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  const int threads = blockDim.x * blockDim.y, thread = threadIdx.y * blockDim.x + threadIdx.x;
  for (int i = blockIdx.x * threads + thread; i < (kLayer ? 2 * p.d : p.d); i += gridDim.x * threads) {
    const int which = i >= p.d, c = i - which * p.d;
    void* const out = which ? p.dbias : p.dweight;
    if (out == nullptr) continue;
    float part[kFewBlocks];  // all on their way at once
    JoinedSum sum = {0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < kFewBlocks; ++s) part[s] = s < p.splits ? __ldcg(p.partial + (2ll * s + which) * p.d + c) : 0.0f;
#pragma unroll
    for (int s = 0; s < kFewBlocks; ++s) sum.add(part[s]);
    store_gradient(out, c, p.grad_f32, sum.value());
  }
}

// Most threads of a block by the columns that a thread holds: what registers allow.  A scheduler holds a quarter of the
// warps, so that 12 of them have 168 registers each, and 16 have 128.
constexpr int wide_forward_threads(int) { return 512; }
constexpr int wide_backward_threads(int columns, bool again) { return columns <= 16 && again ? 640 : columns <= 24 ? 512 : 384; }

// T: type of the rows, W: type of weight and bias.  Places of the ring behind a row's end stay zero.
// Bound by memory: RMS norm of 32414 x 5120 bf16 103 us, 6.4 TB/s; layer norm 114 us, 5.8 TB/s, its two reductions a row one after
// the other; layer norm of 4096 x 4096, 28 rows an SM, 14.6 us, 4.6 TB/s, a third of it the first rows' way in.
template <typename T, typename W, bool kLayer, int N>
__global__ void __launch_bounds__(wide_forward_threads(N * kPerVector<T>)) norm_forward_wide_kernel(const NormForwardParams p) {
  constexpr int P = kPerVector<T>;
  __shared__ WideShared shared;
  extern __shared__ __align__(128) unsigned char ring_memory[];  // [groups][places][N * blockDim.x][16 bytes]
  const int stride = gridDim.x * blockDim.y, row = blockIdx.x * blockDim.y + threadIdx.y;
  const int rows = row < p.M ? (p.M - 1 - row) / stride + 1 : 0;  // of this group
  const uint32_t jump = blockDim.x * 16;                          // bytes from a thread's vector to its next
  RowRing<1> ring(shared, ring_memory, N * jump, p.d * static_cast<uint32_t>(sizeof(T)), p.ring);
  bool valid[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    valid[j] = static_cast<int>(j * blockDim.x + threadIdx.x) * P < p.d;
    if (!valid[j]) {
      for (int k = 0; k < ring.places; ++k) clear16(ring.here() + threadIdx.x * 16 + (k * N + j) * jump);
    }
  }
  fence_mbar_init();
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  int asked = 0;  // of the group's first thread
  auto ask = [&](int place, int n) {
    const void* const src[1] = {static_cast<const T*>(p.x) + (row + n * stride) * p.ldx};
    asked += ring.ask(place, src, 1, p.ring.withhold && row + n == 0);
  };
  const int ahead = ring.places - 1;
  if (threadIdx.x == 0) {
    for (int n = 0; n < ahead && n < rows; ++n) ask(n, n);
  }
  Columns<W, N, P, (N * P <= 16)> weight, bias;
  weight.init(p.weight, 0x3f803f80u, p.d);
  if (kLayer) bias.init(p.bias, 0u, p.d);
  const int span = round_up_pow2(blockDim.x >> 5);
  float2* const slots = shared.slots[span > 1 ? threadIdx.y : 0][0];
  const float inv_d = 1.0f / static_cast<float>(p.d);
  char* out = static_cast<char*>(p.y) + row * p.ldy * static_cast<long long>(sizeof(T)) + threadIdx.x * 16;
  int turn = 0;
  for (int n = 0; n < rows; ++n) {
    ring.wait();
    const uint32_t here = ring.here() + threadIdx.x * 16;
    Pair x[N][P / 2];
#pragma unroll
    for (int j = 0; j < N; ++j) unpack16(read16(here + j * jump), x[j]);
    float mean = 0.0f;
    if (kLayer) {
      Pair s = both(0.0f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
#pragma unroll
        for (int i = 0; i < P / 2; ++i) s = s + x[j][i];
      }
      mean = group_sums<false>(make_float2(0.0f, sum(s)), slots + 32 * turn, span).y * inv_d;
      turn ^= 1;
    }
    const Pair away = both(-mean);
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pair q = both(0.0f);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        if (kLayer) x[j][i] = x[j][i] + away;
        q = fma2(x[j][i], x[j][i], q);
      }
      if (!kLayer || valid[j]) ss += sum(q);
    }
    const float rstd = rsqrtf(fmaf(group_sums<false>(make_float2(0.0f, ss), slots + 32 * turn, span).y, inv_d, p.eps));
    turn ^= 1;
    // the group has read this row, and the one before it long ago: its place takes another
    if (threadIdx.x == 0 && n + ahead < rows) ask(ring.before(), n + ahead);
    const Pair by = both(rstd);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pair w[P / 2], b[P / 2];
      weight.get(j, valid[j], w);
      if (kLayer) bias.get(j, valid[j], b);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        const Pair f = w[i] * by;
        x[j][i] = kLayer ? fma2(x[j][i], f, b[i]) : x[j][i] * f;
      }
      if (valid[j]) store16(out + j * jump, x[j]);
    }
    out += p.y_step;
    ring.advance();
    if (threadIdx.x == 0) {
      if (kLayer) p.mean[row + n * stride] = mean;
      p.rstd[row + n * stride] = rstd;
    }
  }
  if (ring.wd.aborted() && threadIdx.x == 0) ring.drain(asked);
}

// dx, and the block's part of the sums over rows: a thread keeps them for its columns over all its rows, the groups of a
// block are joined in the ring's memory at the end, and the blocks by norm_reduce_kernel.
// Bound by memory: RMS norm with a residual, 32414 x 5120 bf16, 200 to 217 us, 6.1 to 6.6 TB/s; layer norm, whose second sum takes as many
// registers again, 16384 x 4096 87 us, 6.2 TB/s, and 32414 x 5120 207 to 217 us, 6.1 to 6.4 TB/s.  kAgain: a row's z and a are not kept over its reduction but computed
// again from shared memory, which frees their registers.
template <typename T, typename W, bool kLayer, int N, bool kAgain>
__global__ void __launch_bounds__(wide_backward_threads(N * kPerVector<T>, kAgain)) norm_backward_wide_kernel(const NormBackwardParams p) {
  constexpr int P = kPerVector<T>;
  constexpr long long kSize = sizeof(T);
  __shared__ WideShared shared;
  extern __shared__ __align__(128) unsigned char ring_memory[];  // [groups][places][x, dy, res][N * blockDim.x][16 bytes]
  const int stride = gridDim.x * blockDim.y, row = blockIdx.x * blockDim.y + threadIdx.y;
  const int rows = row < p.M ? (p.M - 1 - row) / stride + 1 : 0;  // of this group
  const uint32_t jump = blockDim.x * 16;                          // bytes from a thread's vector to its next
  const bool residual = p.residual != nullptr;
  RowRing<3> ring(shared, ring_memory, N * jump, p.d * static_cast<uint32_t>(kSize), p.ring);
  bool valid[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    valid[j] = static_cast<int>(j * blockDim.x + threadIdx.x) * P < p.d;
    if (!valid[j]) {
      for (int k = 0; k < 3 * ring.places; ++k) clear16(ring.here() + threadIdx.x * 16 + (k * N + j) * jump);
    }
  }
  fence_mbar_init();
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  int asked = 0;  // of the group's first thread
  auto ask = [&](int place, int n) {
    const long long r = row + n * stride;
    const void* const src[3] = {static_cast<const T*>(p.x) + r * p.ldx, static_cast<const T*>(p.dout) + r * p.ld_dout,
                                static_cast<const T*>(p.residual) + (residual ? r * p.ld_res : 0)};
    asked += ring.ask(place, src, residual ? 3 : 2, p.ring.withhold && row + n == 0);
  };
  const int ahead = ring.places - 1;
  if (threadIdx.x == 0) {
    for (int n = 0; n < ahead && n < rows; ++n) ask(n, n);
  }
  float next_mean = 0.0f, next_rstd = 0.0f;
  if (rows > 0) {
    if (kLayer) next_mean = p.mean[row];
    next_rstd = p.rstd[row];
  }
  Columns<W, N, P, (N * P <= 8)> weight;
  weight.init(p.weight, 0x3f803f80u, p.d);
  Pair dw[N][P / 2], db[kLayer ? N : 1][P / 2];
#pragma unroll
  for (int j = 0; j < N; ++j) {
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      dw[j][i] = both(0.0f);
      if (kLayer) db[j][i] = both(0.0f);
    }
  }
  const int span = round_up_pow2(blockDim.x >> 5);
  float2* const slots = shared.slots[span > 1 ? threadIdx.y : 0][0];
  const float inv_d = 1.0f / static_cast<float>(p.d);
  char* out = static_cast<char*>(p.dx) + row * p.ld_dx * kSize + threadIdx.x * 16;
  for (int n = 0; n < rows; ++n) {
    const float rstd = next_rstd;
    const Pair by = both(rstd), away = both(-next_mean);
    if (n + 1 < rows) {
      if (kLayer) next_mean = p.mean[row + (n + 1) * stride];
      next_rstd = p.rstd[row + (n + 1) * stride];
    }
    ring.wait();
    const uint32_t here = ring.here() + threadIdx.x * 16;
    Pair z[kAgain ? 1 : N][P / 2], a[kAgain ? 1 : N][P / 2];
    Pair s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      constexpr int kOne = kAgain ? 0 : 1;
      Pair(&zj)[P / 2] = z[j * kOne];
      Pair(&aj)[P / 2] = a[j * kOne];
      Pair w[P / 2];
      unpack16(read16(here + j * jump), zj);
      unpack16(read16(here + (N + j) * jump), aj);
      weight.get(j, valid[j], w);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        zj[i] = (kLayer ? zj[i] + away : zj[i]) * by;
        dw[j][i] = fma2(aj[i], zj[i], dw[j][i]);
        if (kLayer) {
          db[j][i] = db[j][i] + aj[i];
          s1 = fma2(aj[i], w[i], s1);
        }
        aj[i] = aj[i] * w[i];
        s2 = fma2(aj[i], zj[i], s2);
      }
    }
    const float2 s = group_sums<kLayer>(make_float2(kLayer ? sum(s1) : 0.0f, sum(s2)), slots + 32 * (n & 1), span);
    // all have read the row before this one to its end: its place takes another
    if (threadIdx.x == 0 && n + ahead < rows) ask(ring.before(), n + ahead);
    // dx = a rstd - c1 rstd - z c2 rstd (+ res)
    const Pair k1 = both(-s.x * inv_d * rstd), k2 = both(-s.y * inv_d * rstd * (kAgain ? rstd : 1.0f));
#pragma unroll
    for (int j = 0; j < N; ++j) {
      Pair add[P / 2], zj[P / 2], aj[P / 2];
      if (kAgain) {
        Pair w[P / 2];
        unpack16(read16(here + j * jump), zj);
        unpack16(read16(here + (N + j) * jump), aj);
        weight.get(j, valid[j], w);
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
          zj[i] = zj[i] + away;  // times rstd in k2
          aj[i] = aj[i] * w[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
          zj[i] = z[kAgain ? 0 : j][i];
          aj[i] = a[kAgain ? 0 : j][i];
        }
      }
      if (residual) unpack16(read16(here + (2 * N + j) * jump), add);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        const Pair t = fma2(zj[i], k2, kLayer ? fma2(aj[i], by, k1) : aj[i] * by);
        zj[i] = residual ? t + add[i] : t;
      }
      if (valid[j]) store16(out + j * jump, zj);
    }
    out += p.dx_step;
    ring.advance();
  }
  if (ring.wd.aborted() && threadIdx.x == 0) ring.drain(asked);
  if (p.partial == nullptr) return;
  // [group][2][columns]: the groups' sums side by side, joined in the order of the groups
  const int columns = blockDim.x * N * P, group_floats = 2 * columns;
  const int threads = blockDim.x * blockDim.y, thread = threadIdx.y * blockDim.x + threadIdx.x;
  float* joined = reinterpret_cast<float*>(ring_memory);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = (j * blockDim.x + threadIdx.x) * P;
#pragma unroll
    for (int i = 0; i < P / 2; i += 2) {
      float* at = joined + threadIdx.y * group_floats + c + 2 * i;
      const Pair pair_w[2] = {dw[j][i], dw[j][i + 1]};
      store16(at, pair_w);
      if (kLayer) {
        const Pair pair_b[2] = {db[kLayer ? j : 0][i], db[kLayer ? j : 0][i + 1]};
        store16(at + columns, pair_b);
      }
    }
  }
  __syncthreads();
  float* part = p.partial + 2ll * blockIdx.x * p.d;
  const bool counted = static_cast<int>(blockIdx.x) < p.splits;  // a cluster may have blocks without rows
  for (int i = thread * 4; i < (kLayer ? 2 * columns : columns); i += threads * 4) {
    const int which = i >= columns, c = i - which * columns;
    if (c >= p.d || !counted) continue;
    float4 total = *reinterpret_cast<const float4*>(joined + i);
    for (int g = 1; g < static_cast<int>(blockDim.y); ++g) {
      const float4 q = *reinterpret_cast<const float4*>(joined + g * group_floats + i);
      total.x += q.x;
      total.y += q.y;
      total.z += q.z;
      total.w += q.w;
    }
    *reinterpret_cast<float4*>(part + which * p.d + c) = total;
  }
  if (p.cluster) join_in_cluster<kLayer>(p);
}

// ---- rows that start anywhere ----
//
// The same rings for rows that are not whole granules of 16 bytes, or not all on granules' starts.  A thread takes every
// blockDim.x-th column, element by element, so that neighbours still read and write next to one another.  Bound by the
// instructions on single elements: layer norm of 16000 x 4097 bf16, forward 154 us, backward 273 us (1.7 and 1.9 TB/s; row by row from
// memory, without a ring, 258 and 366); 16000 x 1003 fp32, backward 50 us, 5.2 TB/s.

constexpr int kOddThreads = 512;  // most threads of a block

// Elements of two bytes go through shared memory on their way out: stored one by one they took most of the time.
template <typename T>
constexpr bool kStaged = sizeof(T) == 2;

// Bytes of a place for one array: the granules that a row of a group's `columns` touches.
__host__ __device__ constexpr uint32_t odd_array_bytes(int columns, int size) {
  return static_cast<uint32_t>(columns) * size + 16u;  // columns are a multiple of 32
}

// A group's row from its staging memory, where it lies as far behind a granule's start as its target: whole granules by wide
// stores, the elements before and behind them one by one.
template <typename T>
__device__ __forceinline__ void store_staged(T* target, const unsigned char* staging, int d, int span) {
  if (span > 1) group_barrier();
  else __syncwarp();
  const int size = sizeof(T);
  const int begin = static_cast<int>(reinterpret_cast<uint64_t>(target) & 15u), end = begin + d * size;
  const int lo = min((begin + 15) & ~15, end), hi = max(end & ~15, lo);
  char* const granule = reinterpret_cast<char*>(target) - begin;
  for (int v = lo + static_cast<int>(threadIdx.x) * 16; v < hi; v += blockDim.x * 16) {
    *reinterpret_cast<uint4*>(granule + v) = *reinterpret_cast<const uint4*>(staging + v);
  }
  const int head = (lo - begin) / size, tail = (end - hi) / size;  // below 16 bytes each
  for (int i = threadIdx.x; i < head + tail; i += blockDim.x) {
    const int at = i < head ? begin + i * size : hi + (i - head) * size;
    *reinterpret_cast<T*>(granule + at) = *reinterpret_cast<const T*>(staging + at);
  }
}

template <typename T, bool kLayer, int N>
__global__ void __launch_bounds__(kOddThreads, 2) norm_forward_odd_kernel(const NormForwardParams p) {
  __shared__ WideShared shared;
  extern __shared__ __align__(128) unsigned char ring_memory[];  // [groups][places][granules]; [groups][granules]: rows to store
  const int stride = gridDim.x * blockDim.y, row = blockIdx.x * blockDim.y + threadIdx.y;
  const int rows = row < p.M ? (p.M - 1 - row) / stride + 1 : 0;  // of this group
  const uint32_t array = odd_array_bytes(blockDim.x * N, sizeof(T));
  RowRing<1> ring(shared, ring_memory, array, p.d * static_cast<uint32_t>(sizeof(T)), p.ring);
  fence_mbar_init();
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  auto source = [&](int n) { return static_cast<const T*>(p.x) + (row + n * stride) * p.ldx; };
  int asked = 0;  // of the group's first thread
  auto ask = [&](int place, int n) {
    const T* const src[1] = {source(n)};
    const int r = row + n * stride;
    const bool first = r < p.ring.edge, last = r >= p.M - p.ring.edge;
    if (!first && !last) asked += ring.ask_granules(place, src, 1);
    else asked += ring.ask_edge(place, src[0], src[0], src[0], 1, p.d, first, last, p.ring.withhold && r == 0);
  };
  const int ahead = ring.places - 1;
  if (threadIdx.x == 0) {
    for (int n = 0; n < ahead && n < rows; ++n) ask(n, n);
  }
  float w[N], b[kLayer ? N : 1];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = j * blockDim.x + threadIdx.x;
    w[j] = c < p.d ? load_vector(p.weight, c, p.w_f32, 1.0f) : 0.0f;
    if (kLayer) b[j] = c < p.d ? load_vector(p.bias, c, p.w_f32, 0.0f) : 0.0f;
  }
  const int span = round_up_pow2(blockDim.x >> 5);
  float2* const slots = shared.slots[span > 1 ? threadIdx.y : 0][0];
  unsigned char* const mine = ring_memory + threadIdx.y * ring.places * array;  // the group's ring
  unsigned char* const staging = ring_memory + (blockDim.y * ring.places + threadIdx.y) * array;
  const float inv_d = 1.0f / static_cast<float>(p.d);
  int turn = 0;
  for (int n = 0; n < rows; ++n) {
    ring.wait();
    const T* const here = reinterpret_cast<const T*>(mine + ring.at * array + behind(source(n)));
    float x[N], s = 0.0f, ss = 0.0f, mean = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      const float v = to_float<T>(here[c]);  // behind the row's end whatever the place holds
      x[j] = c < p.d ? v : 0.0f;
      s += x[j];
    }
    if (kLayer) {
      mean = group_sums<false>(make_float2(0.0f, s), slots + 32 * turn, span).y * inv_d;
      turn ^= 1;
    }
#pragma unroll
    for (int j = 0; j < N; ++j) {
      x[j] = static_cast<int>(j * blockDim.x + threadIdx.x) < p.d ? x[j] - mean : 0.0f;
      ss = fmaf(x[j], x[j], ss);
    }
    const float rstd = rsqrtf(fmaf(group_sums<false>(make_float2(0.0f, ss), slots + 32 * turn, span).y, inv_d, p.eps));
    turn ^= 1;
    // the group has read this row, and the one before it long ago: its place takes another
    if (threadIdx.x == 0 && n + ahead < rows) ask(ring.before(), n + ahead);
    T* const y = static_cast<T*>(p.y) + (row + n * stride) * p.ldy;
    T* const stage = kStaged<T> ? reinterpret_cast<T*>(staging + behind(y)) : y;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      if (!kStaged<T> && c >= p.d) continue;
      stage[c] = from_float<T>(kLayer ? fmaf(x[j] * rstd, w[j], b[kLayer ? j : 0]) : x[j] * rstd * w[j]);
    }
    if (kStaged<T>) store_staged(y, staging, p.d, span);
    if (threadIdx.x == 0) {
      if (kLayer) p.mean[row + n * stride] = mean;
      p.rstd[row + n * stride] = rstd;
    }
    ring.advance();
  }
  if (ring.wd.aborted() && threadIdx.x == 0) ring.drain(asked);
}

template <typename T, bool kLayer, int N>
__global__ void __launch_bounds__(kOddThreads) norm_backward_odd_kernel(const NormBackwardParams p) {
  __shared__ WideShared shared;
  extern __shared__ __align__(128) unsigned char ring_memory[];  // [groups][places][x, dy, res][granules]; [groups][granules]: rows
                                                                  // to store; at the end [groups][2][columns] fp32
  const int stride = gridDim.x * blockDim.y, row = blockIdx.x * blockDim.y + threadIdx.y;
  const int rows = row < p.M ? (p.M - 1 - row) / stride + 1 : 0;  // of this group
  const bool residual = p.residual != nullptr;
  const uint32_t array = odd_array_bytes(blockDim.x * N, sizeof(T));
  RowRing<3> ring(shared, ring_memory, array, p.d * static_cast<uint32_t>(sizeof(T)), p.ring);
  fence_mbar_init();
  __syncthreads();
  grid_launch_dependents();
  grid_dependency_wait();
  auto x_of = [&](int n) { return static_cast<const T*>(p.x) + (row + n * stride) * p.ldx; };
  auto dy_of = [&](int n) { return static_cast<const T*>(p.dout) + (row + n * stride) * p.ld_dout; };
  auto res_of = [&](int n) { return static_cast<const T*>(p.residual) + (residual ? (row + n * stride) * p.ld_res : 0); };
  int asked = 0;  // of the group's first thread
  auto ask = [&](int place, int n) {
    const T* const src[3] = {x_of(n), dy_of(n), res_of(n)};
    const int r = row + n * stride;
    const int arrays = residual ? 3 : 2;
    const bool first = r < p.ring.edge, last = r >= p.M - p.ring.edge;
    if (!first && !last) asked += ring.ask_granules(place, src, arrays);
    else asked += ring.ask_edge(place, src[0], src[1], src[2], arrays, p.d, first, last, p.ring.withhold && r == 0);
  };
  const int ahead = ring.places - 1;
  if (threadIdx.x == 0) {
    for (int n = 0; n < ahead && n < rows; ++n) ask(n, n);
  }
  float next_mean = 0.0f, next_rstd = 0.0f;
  if (rows > 0) {
    if (kLayer) next_mean = p.mean[row];
    next_rstd = p.rstd[row];
  }
  float w[N], dw[N], db[kLayer ? N : 1];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int c = j * blockDim.x + threadIdx.x;
    w[j] = c < p.d ? load_vector(p.weight, c, p.w_f32, 1.0f) : 0.0f;
    dw[j] = 0.0f;
    if (kLayer) db[j] = 0.0f;
  }
  const int span = round_up_pow2(blockDim.x >> 5);
  float2* const slots = shared.slots[span > 1 ? threadIdx.y : 0][0];
  unsigned char* const mine = ring_memory + threadIdx.y * ring.places * 3 * array;  // the group's ring
  unsigned char* const staging = ring_memory + (blockDim.y * ring.places * 3 + threadIdx.y) * array;
  const float inv_d = 1.0f / static_cast<float>(p.d);
  for (int n = 0; n < rows; ++n) {
    const float mean = next_mean, rstd = next_rstd;
    if (n + 1 < rows) {
      if (kLayer) next_mean = p.mean[row + (n + 1) * stride];
      next_rstd = p.rstd[row + (n + 1) * stride];
    }
    ring.wait();
    const unsigned char* const here = mine + ring.at * 3 * array;
    const T* const x = reinterpret_cast<const T*>(here + behind(x_of(n)));
    const T* const dy = reinterpret_cast<const T*>(here + array + behind(dy_of(n)));
    const T* const res = reinterpret_cast<const T*>(here + 2 * array + behind(res_of(n)));
    float z[N], a[N];
    float2 s = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      // behind the row's end whatever the place holds: there both are zero
      const float xv = to_float<T>(x[c]), dyv = to_float<T>(dy[c]);
      z[j] = c < p.d ? (xv - mean) * rstd : 0.0f;
      a[j] = c < p.d ? dyv : 0.0f;
      dw[j] = fmaf(a[j], z[j], dw[j]);
      if (kLayer) db[j] += a[j];
      a[j] *= w[j];
      s.x += a[j];
      s.y = fmaf(a[j], z[j], s.y);
    }
    s = group_sums<kLayer>(s, slots + 32 * (n & 1), span);
    // all have read the row before this one to its end: its place takes another
    if (threadIdx.x == 0 && n + ahead < rows) ask(ring.before(), n + ahead);
    const float c1 = kLayer ? s.x * inv_d : 0.0f, c2 = s.y * inv_d;
    T* const dx = static_cast<T*>(p.dx) + (row + n * stride) * p.ld_dx;
    T* const stage = kStaged<T> ? reinterpret_cast<T*>(staging + behind(dx)) : dx;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      if (!kStaged<T> && c >= p.d) continue;
      const float add = residual ? to_float<T>(res[c]) : 0.0f;
      stage[c] = from_float<T>(fmaf(fmaf(-z[j], c2, a[j] - c1), rstd, add));
    }
    if (kStaged<T>) store_staged(dx, staging, p.d, span);
    ring.advance();
  }
  if (ring.wd.aborted() && threadIdx.x == 0) ring.drain(asked);
  if (p.partial == nullptr) return;
  const int columns = blockDim.x * N, group_floats = 2 * columns;
  const int threads = blockDim.x * blockDim.y, thread = threadIdx.y * blockDim.x + threadIdx.x;
  float* part = p.partial + 2ll * blockIdx.x * p.d;
  const bool counted = static_cast<int>(blockIdx.x) < p.splits;  // a cluster may have blocks without rows
  if (blockDim.y == 1) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      if (c >= p.d || !counted) continue;
      part[c] = dw[j];
      if (kLayer) part[p.d + c] = db[kLayer ? j : 0];
    }
  } else {
    // [group][2][columns]: the groups' sums side by side, joined in the order of the groups
    float* joined = reinterpret_cast<float*>(ring_memory);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int c = j * blockDim.x + threadIdx.x;
      joined[threadIdx.y * group_floats + c] = dw[j];
      if (kLayer) joined[threadIdx.y * group_floats + columns + c] = db[kLayer ? j : 0];
    }
    __syncthreads();
    for (int i = thread; i < (kLayer ? 2 * columns : columns); i += threads) {
      const int which = i >= columns, c = i - which * columns;
      if (c >= p.d || !counted) continue;
      float total = 0.0f;
      for (int g = 0; g < static_cast<int>(blockDim.y); ++g) total += joined[g * group_floats + i];
      part[which * p.d + c] = total;
    }
  }
  if (p.cluster) join_in_cluster<kLayer>(p);
}

// ---- short rows ----
//
// Rows of at most 32 vectors: a part of a warp, blockDim.x = 8, 16 or 32 lanes, takes a row, one vector a lane, and several rows
// at a time, since one row's loads would not keep the memory busy.  Nothing but shuffles joins the lanes.

constexpr int kShortThreads = 256;

__device__ __forceinline__ float part_sum(float v) {
  for (int o = blockDim.x >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  uint4 w;
  asm volatile("ld.global.L1::no_allocate.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p));
  return w;
}

template <typename T, typename W, bool kLayer>
__global__ void __launch_bounds__(kShortThreads) norm_forward_short_kernel(const NormForwardParams p) {
  constexpr int P = kPerVector<T>, R = 4;
  const int c = threadIdx.x * P;
  const bool valid = c < p.d;
  grid_launch_dependents();
  grid_dependency_wait();
  Columns<W, 1, P> weight, bias;
  weight.init(p.weight, 0x3f803f80u, p.d);
  if (kLayer) bias.init(p.bias, 0u, p.d);
  const float inv_d = 1.0f / static_cast<float>(p.d);
  const int stride = gridDim.x * blockDim.y;
  // all lanes of a warp go round as often: `first` is the row of the block's first part
  for (int first = blockIdx.x * blockDim.y; first < p.M; first += R * stride) {
    uint4 raw[R];
    int row[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      row[k] = first + k * stride + threadIdx.y;
      raw[k] = make_uint4(0u, 0u, 0u, 0u);
      if (valid && row[k] < p.M) raw[k] = load16(static_cast<const T*>(p.x) + row[k] * p.ldx + c);
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      Pair x[P / 2];
      unpack16(raw[k], x);
      float mean = 0.0f;
      if (kLayer) {
        Pair s = x[0];
#pragma unroll
        for (int i = 1; i < P / 2; ++i) s = s + x[i];
        mean = part_sum(sum(s)) * inv_d;
      }
      const Pair away = both(-mean);
      Pair q = both(0.0f);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        if (kLayer) x[i] = x[i] + away;
        q = fma2(x[i], x[i], q);
      }
      const float rstd = rsqrtf(fmaf(part_sum(!kLayer || valid ? sum(q) : 0.0f), inv_d, p.eps));
      if (row[k] >= p.M) continue;
      const Pair by = both(rstd);
      Pair w[P / 2], b[P / 2];
      weight.get(0, valid, w);
      if (kLayer) bias.get(0, valid, b);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        const Pair f = w[i] * by;
        x[i] = kLayer ? fma2(x[i], f, b[i]) : x[i] * f;
      }
      if (valid) store16(static_cast<T*>(p.y) + row[k] * p.ldy + c, x);
      if (threadIdx.x == 0) {
        if (kLayer) p.mean[row[k]] = mean;
        p.rstd[row[k]] = rstd;
      }
    }
  }
}

template <typename T, typename W, bool kLayer>
__global__ void __launch_bounds__(kShortThreads) norm_backward_short_kernel(const NormBackwardParams p) {
  constexpr int P = kPerVector<T>, R = 2;
  __shared__ float joined[2][kShortThreads * P];  // [parts][columns]
  const int c = threadIdx.x * P;
  const bool valid = c < p.d, residual = p.residual != nullptr;
  grid_launch_dependents();
  grid_dependency_wait();
  Columns<W, 1, P> weight;
  weight.init(p.weight, 0x3f803f80u, p.d);
  Pair dw[P / 2], db[P / 2];
#pragma unroll
  for (int i = 0; i < P / 2; ++i) dw[i] = db[i] = both(0.0f);
  const float inv_d = 1.0f / static_cast<float>(p.d);
  const int stride = gridDim.x * blockDim.y;
  for (int first = blockIdx.x * blockDim.y; first < p.M; first += R * stride) {
    uint4 raw_x[R], raw_dy[R], raw_res[R];
    float mean[R], rstd[R];
    int row[R];
#pragma unroll
    for (int k = 0; k < R; ++k) {
      row[k] = first + k * stride + threadIdx.y;
      raw_x[k] = raw_dy[k] = raw_res[k] = make_uint4(0u, 0u, 0u, 0u);
      mean[k] = rstd[k] = 0.0f;
      if (row[k] < p.M) {
        if (kLayer) mean[k] = p.mean[row[k]];
        rstd[k] = p.rstd[row[k]];
        if (valid) {
          raw_x[k] = load16(static_cast<const T*>(p.x) + row[k] * p.ldx + c);
          raw_dy[k] = load16(static_cast<const T*>(p.dout) + row[k] * p.ld_dout + c);
          if (residual) raw_res[k] = load16(static_cast<const T*>(p.residual) + row[k] * p.ld_res + c);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < R; ++k) {
      Pair z[P / 2], a[P / 2], w[P / 2], add[P / 2];
      unpack16(raw_x[k], z);
      unpack16(raw_dy[k], a);
      unpack16(raw_res[k], add);
      weight.get(0, valid, w);
      const Pair by = both(rstd[k]), away = both(-mean[k]);
      Pair s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        z[i] = (kLayer ? z[i] + away : z[i]) * by;
        dw[i] = fma2(a[i], z[i], dw[i]);
        if (kLayer) db[i] = db[i] + a[i];
        a[i] = a[i] * w[i];
        if (kLayer) s1 = s1 + a[i];
        s2 = fma2(a[i], z[i], s2);
      }
      const float c1 = kLayer ? part_sum(sum(s1)) * inv_d : 0.0f, c2 = part_sum(sum(s2)) * inv_d;
      const Pair k1 = both(-c1 * rstd[k]), k2 = both(-c2 * rstd[k]);
#pragma unroll
      for (int i = 0; i < P / 2; ++i) {
        const Pair t = fma2(z[i], k2, kLayer ? fma2(a[i], by, k1) : a[i] * by);
        z[i] = residual ? t + add[i] : t;
      }
      if (valid && row[k] < p.M) store16(static_cast<T*>(p.dx) + row[k] * p.ld_dx + c, z);
    }
  }
  if (p.partial == nullptr) return;
  const int columns = blockDim.x * P, thread = threadIdx.y * blockDim.x + threadIdx.x;
#pragma unroll
  for (int i = 0; i < P / 2; i += 2) {
    const Pair pair_w[2] = {dw[i], dw[i + 1]}, pair_b[2] = {db[i], db[i + 1]};
    store16(&joined[0][thread * P + 2 * i], pair_w);
    if (kLayer) store16(&joined[1][thread * P + 2 * i], pair_b);
  }
  __syncthreads();
  float* part = p.partial + 2ll * blockIdx.x * p.d;
  const bool counted = static_cast<int>(blockIdx.x) < p.splits;  // a cluster may have blocks without rows
  for (int i = thread; i < (kLayer ? 2 * columns : columns); i += kShortThreads) {
    const int which = i >= columns, column = i - which * columns;
    if (column >= p.d || !counted) continue;
    float total = 0.0f;
    for (int g = 0; g < static_cast<int>(blockDim.y); ++g) total += joined[which][g * columns + column];
    part[which * p.d + column] = total;
  }
  if (p.cluster) join_in_cluster<kLayer>(p);
}

// Joins the splits' sums: 32 columns a block, whose 32 rows of threads take every 32nd split, five at a time on their way, and
// whose first rows join theirs.  The order is fixed.  Its blocks come up while the backward kernel ends (148 splits of 4096
// columns: 2 us of the pass's 29).
constexpr int kNormReduceRows = 32;
template <bool kBias>
__global__ void __launch_bounds__(32 * kNormReduceRows) norm_reduce_kernel(const NormReduceParams p) {
  constexpr int kAtOnce = 5;
  __shared__ double shared[kBias ? 2 : 1][kNormReduceRows][33];
  const int i = blockIdx.x * 32 + threadIdx.x;
  JoinedSum dw = {0.0f, 0.0f}, db = {0.0f, 0.0f};
  grid_launch_dependents();
  grid_dependency_wait();
  for (int s = threadIdx.y; s < p.splits; s += kAtOnce * kNormReduceRows) {
    float part[kBias ? 2 : 1][kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      const int at = s + k * kNormReduceRows;
      const bool some = at < p.splits && i < p.d;
      part[0][k] = some ? p.partial[2ll * at * p.d + i] : 0.0f;
      if (kBias) part[kBias ? 1 : 0][k] = some ? p.partial[2ll * at * p.d + p.d + i] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; ++k) {
      dw.add(part[0][k]);
      if (kBias) db.add(part[kBias ? 1 : 0][k]);
    }
  }
  shared[0][threadIdx.y][threadIdx.x] = dw.value();
  if (kBias) shared[kBias ? 1 : 0][threadIdx.y][threadIdx.x] = db.value();
  __syncthreads();
  if (threadIdx.y >= (kBias ? 2 : 1)) return;
  double sum[4] = {};  // side by side: they do not wait for one another
#pragma unroll
  for (int r = 0; r < kNormReduceRows; ++r) sum[r & 3] += shared[threadIdx.y][r][threadIdx.x];
  void* out = threadIdx.y == 0 ? p.dweight : p.dbias;
  if (out == nullptr || i >= p.d) return;
  store_gradient(out, i, p.out_f32, (sum[0] + sum[1]) + (sum[2] + sum[3]));
}

}  // namespace fsw
