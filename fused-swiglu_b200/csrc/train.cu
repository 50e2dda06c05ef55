// C ABI of the training operators around the MLP (declared in include/fswiglu.h): norms with their gradients, AdamW over
// many tensors, the clipped gradient norm.  Argument checks and launches; no allocation of device memory, no throw.
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdint>
#include <memory>
#include <new>
#include <type_traits>

#include "../../include/fswiglu.h"
#include "host_state.h"
#include "norm_sm100.cuh"
#include "optim_sm100.cuh"

namespace {

using namespace fsw;

bool known_type(int t) { return t == FSWIGLU_OUT_BF16 || t == FSWIGLU_OUT_F32; }
bool aligned(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
size_t type_bytes(int t) { return t == FSWIGLU_OUT_F32 ? 4u : 2u; }

// A launch that may start while the stream's previous kernel ends: its blocks come up, and wait (grid_dependency_wait) before
// they touch memory.  Clusters of `cluster` blocks, where that is not 1.
template <typename... Params, typename... Args>
int launch_clusters(unsigned cluster, void (*kernel)(Params...), int64_t grid, dim3 block, size_t shared, cudaStream_t s,
                    const Args&... args) {
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(grid));
  config.blockDim = block;
  config.dynamicSmemBytes = shared;
  config.stream = s;
  config.attrs = attributes;
  config.numAttrs = cluster == 1 ? 1 : 2;
  const cudaError_t e = cudaLaunchKernelEx(&config, kernel, static_cast<const std::decay_t<Params>&>(args)...);
  count_launch();
  return e == cudaSuccess ? FSWIGLU_OK : FSWIGLU_ERR_CUDA;
}

template <typename... Params, typename... Args>
int launch(void (*kernel)(Params...), int64_t grid, dim3 block, size_t shared, cudaStream_t s, const Args&... args) {
  return launch_clusters(1, kernel, grid, block, shared, s, args...);
}

// ---- norms ----

constexpr int64_t kMaxNormWidth = 1 << 24;                // a row's length is exact in fp32
constexpr int64_t kMaxNormRows = 0x7fffffff - (1 << 20);  // a row behind the last one is still an int
constexpr int kMaxNormSplits = 296;         // two thread blocks for each of 148 SMs

int check_rows(const void* p, int64_t M, int64_t d, int64_t ld, int type) {
  if (p == nullptr) return FSWIGLU_ERR_BAD_ARG;
  if (ld < d && M > 1) return FSWIGLU_ERR_SHAPE;
  return aligned(p, type_bytes(type)) ? FSWIGLU_OK : FSWIGLU_ERR_ALIGNMENT;
}

int check_norm(int64_t M, int64_t d, int x_dtype, int w_dtype) {
  if (M < 0 || d <= 0 || !known_type(x_dtype) || !known_type(w_dtype)) return FSWIGLU_ERR_BAD_ARG;
  if (M > kMaxNormRows || d > kMaxNormWidth) return FSWIGLU_ERR_SHAPE;
  return FSWIGLU_OK;
}

int norm_splits(int64_t M) { return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(M, kMaxNormSplits))); }

constexpr size_t kRingBytes = 216 * 1024;  // of the 227 KB of a block

// How the wide kernels lay a row out: each thread holds `columns` of it.
struct WidePlan {
  int columns, group, groups, places;
  bool again;           // backward: a row's values are computed a second time where they are used
  size_t place, extra;  // bytes of shared memory: of the block's places of one row each, and beside the ring
  size_t ring() const { return places * place + extra; }
  int threads() const { return group * groups; }
};

// The plan for rows of d values of `size` bytes, `arrays` of them on their way, in blocks of at most `most_threads`;
// columns == 0 where a row does not fit.
WidePlan wide_plan(int64_t d, int64_t M, size_t size, int columns, int most_threads, int arrays, int most_places, int sms) {
  WidePlan w = {};
  const int64_t group = (d + 32 * columns - 1) / (32 * columns) * 32;
  if (group > most_threads) return w;
  // no more groups than leave every SM a block
  const int64_t spread = std::max<int64_t>(1, (M + sms - 1) / sms);
  int64_t groups = std::min<int64_t>({most_threads / group, group > 32 ? kWideMultiGroups : kWideGroups, spread});
  for (; groups >= 1; --groups) {
    const size_t place = static_cast<size_t>(arrays) * static_cast<size_t>(group * groups * columns) * size;
    const size_t places = std::min<size_t>(static_cast<size_t>(most_places), kRingBytes / place);
    // two places keep one row of each group on its way: enough where that is 64 KB
    if (places < 2 || (places == 2 && most_places > 2 && groups > 1 && place < 64 * 1024)) continue;
    w = WidePlan{columns, static_cast<int>(group), static_cast<int>(groups), static_cast<int>(places), false, place, 0};
    break;
  }
  return w;
}

// The same for rows that start anywhere: values of a thread, threads of a group, and the plan.
int odd_values(int d) { return d <= 128 ? 4 : d <= 8 * kOddThreads ? 8 : 16; }
int odd_group(int d) { return (d + 32 * odd_values(d) - 1) / (32 * odd_values(d)) * 32; }
WidePlan odd_plan(int d, int64_t M, size_t size, int most_threads, int arrays, int most_places, int sms) {
  WidePlan w = {};
  const int64_t group = odd_group(d);
  if (group > kOddThreads) return w;
  const int64_t spread = std::max<int64_t>(1, (M + sms - 1) / sms);
  int64_t groups = std::min<int64_t>({most_threads / group, group > 32 ? kWideMultiGroups : kWideGroups, spread});
  for (; groups >= 1; --groups) {
    const size_t array = odd_array_bytes(static_cast<int>(group) * odd_values(d), static_cast<int>(size)), place = static_cast<size_t>(arrays * groups) * array;
    const size_t staging = size == 2 ? static_cast<size_t>(groups) * array : 0;  // and a row of each group that is stored
    const size_t places = std::min<size_t>(static_cast<size_t>(most_places), (kRingBytes - staging) / place);
    if (places < 2 || (places == 2 && most_places > 2 && groups > 1 && place < 64 * 1024)) continue;
    // the groups' sums over rows are joined in the ring's memory
    const size_t joined = arrays == 3 && groups > 1 ? static_cast<size_t>(groups * group * odd_values(d)) * 2 * sizeof(float) : 0;
    if (joined > kRingBytes) continue;
    w = WidePlan{odd_values(d), static_cast<int>(group), static_cast<int>(groups), static_cast<int>(places), false, place,
                 std::max(places * place + staging, joined) - places * place};
    break;
  }
  return w;
}

// Lets a kernel have a whole ring of shared memory; once for each device.
template <typename Kernel>
int opt_in(Kernel k, std::atomic<uint64_t>* done, const Device& dev) {
  const uint64_t bit = 1ull << dev.index;
  if (done->load(std::memory_order_relaxed) & bit) return FSWIGLU_OK;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kRingBytes)) != cudaSuccess)
    return FSWIGLU_ERR_CUDA;
  done->fetch_or(bit, std::memory_order_relaxed);
  return FSWIGLU_OK;
}

// Forward kernels have several blocks on an SM.  The places of their rings are the fewest that keep 56 KB of rows on their way
// to it: fewer wait, and more are slower, since reads far ahead of the writes take the memory's pages from them (RMS norm of
// 32414 x 5120 bf16: two places 138 us, three 106, four 123; of 16000 x 4096 fp32: 82, 94).  Sets the plan's places, and returns the
// SM's blocks; the last answer is kept with what it was for.
template <typename Kernel>
int64_t fill_sm(Kernel k, std::atomic<uint64_t>* known, WidePlan& w) {
  constexpr size_t kOnItsWay = 56 * 1024;
  const uint64_t key = static_cast<uint64_t>(w.threads()) << 48 | static_cast<uint64_t>(w.place + w.extra) << 16 |
                       static_cast<uint64_t>(w.places) << 12;
  const uint64_t seen = known->load(std::memory_order_relaxed);
  int blocks = 0;
  if ((seen & ~0xfffull) == key && (seen & 0xffu) != 0) {
    w.places = static_cast<int>(seen >> 8 & 0xfu);
    return static_cast<int64_t>(seen & 0xffu);
  }
  const int most = w.places;
  for (w.places = 2;; ++w.places) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&blocks, k, w.threads(), w.ring()) != cudaSuccess || blocks < 1) blocks = 1;
    if (w.places >= most || (w.places - 1) * w.place * blocks >= kOnItsWay) break;
  }
  known->store(key | static_cast<uint64_t>(w.places) << 8 | static_cast<uint64_t>(blocks), std::memory_order_relaxed);
  return blocks;
}

// Wide kernels take weights of the rows' type or fp32 ones (bf16 rows), and stand-ins for missing ones in bf16.
template <typename T, typename W, bool kLayer, int kColumns>
int launch_norm_forward_wide(NormForwardParams& p, WidePlan w, const Device& dev, cudaStream_t s) {
  constexpr auto kernel = norm_forward_wide_kernel<T, W, kLayer, kColumns / kPerVector<T>>;
  static std::atomic<uint64_t> done{0}, known{0};
  if (int rc = opt_in(kernel, &done, dev)) return rc;
  const int64_t blocks = (static_cast<int64_t>(p.M) + w.groups - 1) / w.groups;
  const int64_t resident = dev.sms * fill_sm(kernel, &known, w);
  const int grid = static_cast<int>(std::min(blocks, resident));
  p.y_step = static_cast<long long>(grid) * w.groups * p.ldy * static_cast<long long>(sizeof(T));
  p.ring.places = w.places;
  p.ring.withhold = take_withhold();
  return launch(kernel, grid, dim3(w.group, w.groups), w.ring(), s, p);
}

// Forward: 32 columns a thread, since a row's reductions cost every warp the same; 16 where a warp holds a whole row with
// them, where fp32 weights are kept in registers, and for fp32 rows, whose places would take twice the shared memory.
WidePlan forward_plan(const NormForwardParams& p, size_t size, int sms) {
  const bool few = p.d <= 512 || ((p.w_f32 || size == 4) && p.d <= 16 * wide_forward_threads(16));
  const int columns = few ? 16 : 32, group = (p.d + 32 * columns - 1) / (32 * columns) * 32;
  if (group > wide_forward_threads(columns)) return WidePlan{};
  return wide_plan(p.d, p.M, size, columns, std::max(256, group), 1, kWidePlaces, sms);
}

template <typename T, typename W, bool kLayer>
int launch_norm_forward_wide(NormForwardParams& p, const WidePlan& w, const Device& dev, cudaStream_t s) {
  if (w.columns == 16) return launch_norm_forward_wide<T, W, kLayer, 16>(p, w, dev, s);
  return launch_norm_forward_wide<T, W, kLayer, 32>(p, w, dev, s);
}

template <typename T, bool kLayer, int N>
int launch_norm_forward_odd(NormForwardParams& p, WidePlan w, const Device& dev, cudaStream_t s) {
  constexpr auto kernel = norm_forward_odd_kernel<T, kLayer, N>;
  static std::atomic<uint64_t> done{0}, known{0};
  if (int rc = opt_in(kernel, &done, dev)) return rc;
  const int64_t blocks = (static_cast<int64_t>(p.M) + w.groups - 1) / w.groups;
  const int64_t resident = dev.sms * fill_sm(kernel, &known, w);
  p.ring.places = w.places;
  p.ring.edge = edge_rows(p.d * static_cast<int>(sizeof(T)));
  p.ring.withhold = take_withhold();
  return launch(kernel, std::min(blocks, resident), dim3(w.group, w.groups), w.ring(), s, p);
}

// Lanes that take a short row.
int short_lanes(int d, int per_vector) { return d <= 8 * per_vector ? 8 : d <= 16 * per_vector ? 16 : 32; }

template <typename T, typename W, bool kLayer>
int launch_norm_forward_short(const NormForwardParams& p, const Device& dev, cudaStream_t s) {
  const int lanes = short_lanes(p.d, kPerVector<T>), parts = kShortThreads / lanes;
  const int64_t blocks = (static_cast<int64_t>(p.M) + parts - 1) / parts;
  return launch(norm_forward_short_kernel<T, W, kLayer>, std::min<int64_t>(blocks, static_cast<int64_t>(dev.sms) * 8),
                dim3(lanes, parts), 0, s, p);
}

template <typename T, bool kLayer>
int launch_norm_forward(NormForwardParams& p, bool wide, const Device& dev, cudaStream_t s) {
  if (wide) {
    if (p.d <= 32 * kPerVector<T>) {
      if (p.w_f32) return launch_norm_forward_short<T, float, kLayer>(p, dev, s);
      return launch_norm_forward_short<T, __nv_bfloat16, kLayer>(p, dev, s);
    }
    const WidePlan w = forward_plan(p, sizeof(T), dev.sms);
    if (w.columns > 0) {
      if (p.w_f32) return launch_norm_forward_wide<T, float, kLayer>(p, w, dev, s);
      return launch_norm_forward_wide<T, __nv_bfloat16, kLayer>(p, w, dev, s);
    }
  } else {
    const WidePlan w = odd_plan(p.d, p.M, sizeof(T), std::max(256, odd_group(p.d)), 1, kWidePlaces, dev.sms);
    if (w.columns > 0) {
      if (w.columns == 4) return launch_norm_forward_odd<T, kLayer, 4>(p, w, dev, s);
      if (w.columns == 8) return launch_norm_forward_odd<T, kLayer, 8>(p, w, dev, s);
      return launch_norm_forward_odd<T, kLayer, 16>(p, w, dev, s);
    }
  }
  return launch(norm_forward_any_kernel<T, kLayer>, std::min<int64_t>(p.M, static_cast<int64_t>(dev.sms) * 8),
                dim3(kNormThreads), 0, s, p);
}

// Little work: one cluster, whose blocks join their sums over rows themselves, takes the place of a grid over all SMs and a
// second launch.  Layer norm, bf16, a call / in a graph, us, with two launches in brackets: 64 x 128 6.7 / 3.3 (9.2 / 3.9), 128 x 256
// 6.9 / 3.7 (9.5 / 4.3), 32 x 1024 7.0 / 4.1 (9.5 / 5.1), 32 x 1003 6.9 / 5.7 (9.6 / 5.7).  Of rows of 4096 columns and more a call
// gains but a graph loses: 8 x 4096 7.0 / 5.9 (9.6 / 4.9), 4 x 8192 7.9 / 7.8 (9.3 / 7.4).  More values, and graphs lose as much as
// calls gain: 512 x 128 6.6 / 4.6 (8.5 / 3.8), 64 x 1003 7.0 / 6.6 (8.4 / 4.6), 8 x 8192 7.9 / 7.5 (8.5 / 6.7).
constexpr int64_t kFewValues = 1 << 15;
bool few_values(const NormBackwardParams& p) { return p.partial != nullptr && static_cast<int64_t>(p.M) * p.d <= kFewValues; }
int backward_splits(const NormBackwardParams& p, int64_t blocks, int64_t most) {
  return static_cast<int>(std::min<int64_t>({blocks, p.cluster ? kFewBlocks : most, kMaxNormSplits}));
}
template <typename Kernel>
int launch_backward(Kernel kernel, dim3 block, size_t shared, cudaStream_t s, const NormBackwardParams& p) {
  if (p.cluster) return launch_clusters(kFewBlocks, kernel, kFewBlocks, block, shared, s, p);
  return launch(kernel, p.splits, block, shared, s, p);
}

template <typename T, bool kLayer, int N>
int launch_norm_backward_odd(NormBackwardParams& p, const WidePlan& w, const Device& dev, cudaStream_t s) {
  constexpr auto kernel = norm_backward_odd_kernel<T, kLayer, N>;
  static std::atomic<uint64_t> done{0};
  if (int rc = opt_in(kernel, &done, dev)) return rc;
  const int64_t blocks = (static_cast<int64_t>(p.M) + w.groups - 1) / w.groups;
  p.splits = backward_splits(p, blocks, dev.sms);
  p.ring.places = w.places;
  p.ring.edge = edge_rows(p.d * static_cast<int>(sizeof(T)));
  p.ring.withhold = take_withhold();
  return launch_backward(kernel, dim3(w.group, w.groups), w.ring(), s, p);
}

template <typename T, typename W, bool kLayer, int kColumns, bool kAgain>
int launch_norm_backward_wide(NormBackwardParams& p, const WidePlan& w, const Device& dev, cudaStream_t s) {
  constexpr auto kernel = norm_backward_wide_kernel<T, W, kLayer, kColumns / kPerVector<T>, kAgain>;
  static std::atomic<uint64_t> done{0};
  if (int rc = opt_in(kernel, &done, dev)) return rc;
  const int64_t blocks = (static_cast<int64_t>(p.M) + w.groups - 1) / w.groups;
  p.splits = backward_splits(p, blocks, dev.sms);
  const int grid = p.cluster ? kFewBlocks : p.splits;
  p.dx_step = static_cast<long long>(grid) * w.groups * p.ld_dx * static_cast<long long>(sizeof(T));
  p.ring.places = w.places;
  p.ring.withhold = take_withhold();
  return launch_backward(kernel, dim3(w.group, w.groups), w.ring(), s, p);
}

// Backward: one block an SM, its registers full of the sums over rows.  Of the columns a thread may hold, those that keep most
// warps busy.  Layer norm's threads of more than 16 columns compute a row's values twice, for want of registers; those of 16
// do where that makes room for a second group (32414 x 5120 bf16: two groups 207 us; 24 columns a thread 237).
WidePlan backward_plan(const NormBackwardParams& p, bool layer, size_t size, int sms) {
  WidePlan best = {};
  for (int columns = 16; columns <= 32; columns += 8) {
    const bool again = layer && columns > 16;
    WidePlan w = wide_plan(p.d, p.M, size, columns, wide_backward_threads(columns, again), 3, kWidePlaces, sms);
    if (layer && columns == 16 && w.groups == 1) {
      const WidePlan two = wide_plan(p.d, p.M, size, columns, wide_backward_threads(columns, true), 3, kWidePlaces, sms);
      if (two.groups == 2) {
        w = two;
        w.again = true;
      }
    }
    if (w.threads() > best.threads()) best = w;
  }
  return best;
}

template <typename T, typename W, bool kLayer>
int launch_norm_backward_wide(NormBackwardParams& p, const WidePlan& w, const Device& dev, cudaStream_t s) {
  switch (w.columns) {
    case 16:
      if constexpr (kLayer) {
        if (w.again) return launch_norm_backward_wide<T, W, kLayer, 16, true>(p, w, dev, s);
      }
      return launch_norm_backward_wide<T, W, kLayer, 16, false>(p, w, dev, s);
    case 24: return launch_norm_backward_wide<T, W, kLayer, 24, kLayer>(p, w, dev, s);
    default: return launch_norm_backward_wide<T, W, kLayer, 32, kLayer>(p, w, dev, s);
  }
}

template <typename T, typename W, bool kLayer>
int launch_norm_backward_short(NormBackwardParams& p, const Device& dev, cudaStream_t s) {
  const int lanes = short_lanes(p.d, kPerVector<T>), parts = kShortThreads / lanes;
  const int64_t blocks = (static_cast<int64_t>(p.M) + parts - 1) / parts;
  p.cluster = few_values(p);
  p.splits = backward_splits(p, blocks, static_cast<int64_t>(dev.sms) * 2);
  return launch_backward(norm_backward_short_kernel<T, W, kLayer>, dim3(lanes, parts), 0, s, p);
}

template <typename T, bool kLayer>
int launch_norm_backward(NormBackwardParams& p, bool wide, const Device& dev, cudaStream_t s) {
  if (wide) {
    if (p.d <= 32 * kPerVector<T>) {
      if (p.w_f32) return launch_norm_backward_short<T, float, kLayer>(p, dev, s);
      return launch_norm_backward_short<T, __nv_bfloat16, kLayer>(p, dev, s);
    }
    const bool few = few_values(p);
    const WidePlan w = backward_plan(p, kLayer, sizeof(T), few ? kFewBlocks : dev.sms);
    if (w.columns > 0) {
      p.cluster = few;
      if (p.w_f32) return launch_norm_backward_wide<T, float, kLayer>(p, w, dev, s);
      return launch_norm_backward_wide<T, __nv_bfloat16, kLayer>(p, w, dev, s);
    }
  } else {
    const bool few = few_values(p);
    const WidePlan w = odd_plan(p.d, p.M, sizeof(T), kOddThreads, 3, kWidePlaces, few ? kFewBlocks : dev.sms);
    if (w.columns > 0) {
      p.cluster = few;
      if (w.columns == 4) return launch_norm_backward_odd<T, kLayer, 4>(p, w, dev, s);
      if (w.columns == 8) return launch_norm_backward_odd<T, kLayer, 8>(p, w, dev, s);
      return launch_norm_backward_odd<T, kLayer, 16>(p, w, dev, s);
    }
  }
  if (int rc = launch(norm_backward_any_kernel<T, kLayer>, std::min<int64_t>(p.M, static_cast<int64_t>(dev.sms) * 8),
                      dim3(kNormThreads), 0, s, p))
    return rc;
  if (p.partial == nullptr) return FSWIGLU_OK;
  const int64_t tiles = (p.d + kNormThreads - 1) / kNormThreads * static_cast<int64_t>(p.splits);
  return launch(norm_backward_columns_any_kernel<T, kLayer>, std::min<int64_t>(tiles, static_cast<int64_t>(dev.sms) * 32),
                dim3(kNormThreads), 0, s, p);
}

// Whether a matrix's rows all start on 16 bytes.
bool wide_rows(const void* p, int64_t ld, int64_t M, int type) {
  return aligned(p, 16) && (M == 1 || ld * static_cast<int64_t>(type_bytes(type)) % 16 == 0);
}

int norm_forward(bool layer, const void* x, int64_t ldx, const void* weight, const void* bias, void* y, int64_t ldy,
                 float* mean, float* rstd, int64_t M, int64_t d, int x_dtype, int w_dtype, float eps, void* stream) {
  if (int rc = check_norm(M, d, x_dtype, w_dtype)) return rc;
  if (!(eps >= 0.0f)) return FSWIGLU_ERR_BAD_ARG;
  if (M == 0) return FSWIGLU_OK;
  if (int rc = check_rows(x, M, d, ldx, x_dtype)) return rc;
  if (int rc = check_rows(y, M, d, ldy, x_dtype)) return rc;
  if (rstd == nullptr || (layer && mean == nullptr)) return FSWIGLU_ERR_BAD_ARG;
  if (!aligned(weight, type_bytes(w_dtype)) || !aligned(bias, type_bytes(w_dtype)) || !aligned(mean, 4) || !aligned(rstd, 4))
    return FSWIGLU_ERR_ALIGNMENT;
  Device dev;
  if (int rc = current_device(&dev)) return rc;
  NormForwardParams p = {};
  p.x = x;
  p.weight = weight;
  p.bias = bias;
  p.y = y;
  p.mean = mean;
  p.rstd = rstd;
  p.ldx = ldx;
  p.ldy = ldy;
  p.M = static_cast<int>(M);
  p.d = static_cast<int>(d);
  p.ring = RingParams{dev.status, dev.wait_limit_ns, 0, 0, 1};
  p.w_f32 = w_dtype == FSWIGLU_OUT_F32 && (weight != nullptr || bias != nullptr);
  p.eps = eps;
  // fp32 vectors are read where they are: one without the other goes the odd way
  const bool wide = !(layer && p.w_f32 && (weight == nullptr || bias == nullptr)) &&
                    d * type_bytes(x_dtype) % 16 == 0 && wide_rows(x, ldx, M, x_dtype) && wide_rows(y, ldy, M, x_dtype) &&
                    aligned(weight, 16) && aligned(bias, 16);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  using BF = __nv_bfloat16;
  if (x_dtype == FSWIGLU_OUT_F32)
    return layer ? launch_norm_forward<float, true>(p, wide, dev, s) : launch_norm_forward<float, false>(p, wide, dev, s);
  return layer ? launch_norm_forward<BF, true>(p, wide, dev, s) : launch_norm_forward<BF, false>(p, wide, dev, s);
}

int norm_backward(bool layer, const void* dout, int64_t ld_dout, const void* x, int64_t ldx, const float* mean,
                  const float* rstd, const void* weight, const void* residual, int64_t ld_res, void* dx, int64_t ld_dx,
                  void* dweight, void* dbias, int64_t M, int64_t d, int x_dtype, int w_dtype, int grad_dtype,
                  void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = check_norm(M, d, x_dtype, w_dtype)) return rc;
  if (!known_type(grad_dtype)) return FSWIGLU_ERR_BAD_ARG;
  if (!aligned(weight, type_bytes(w_dtype)) || !aligned(dweight, type_bytes(grad_dtype)) ||
      !aligned(dbias, type_bytes(grad_dtype)) || !aligned(mean, 4) || !aligned(rstd, 4))
    return FSWIGLU_ERR_ALIGNMENT;
  const bool columns = dweight != nullptr || dbias != nullptr;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  NormBackwardParams p = {};
  if (M > 0) {
    if (int rc = check_rows(dout, M, d, ld_dout, x_dtype)) return rc;
    if (int rc = check_rows(x, M, d, ldx, x_dtype)) return rc;
    if (int rc = check_rows(dx, M, d, ld_dx, x_dtype)) return rc;
    if (residual != nullptr) {
      if (int rc = check_rows(residual, M, d, ld_res, x_dtype)) return rc;
    }
    if (rstd == nullptr || (layer && mean == nullptr)) return FSWIGLU_ERR_BAD_ARG;
    if (columns && (workspace == nullptr || workspace_bytes < fswiglu_norm_backward_workspace_bytes(M, d) || !aligned(workspace, 256)))
      return FSWIGLU_ERR_WORKSPACE;
  }
  Device dev;
  if (int rc = current_device(&dev)) return rc;
  if (M > 0) {
    p.dout = dout;
    p.x = x;
    p.weight = weight;
    p.residual = residual;
    p.mean = mean;
    p.rstd = rstd;
    p.dx = dx;
    p.partial = columns ? static_cast<float*>(workspace) : nullptr;
    p.ld_dout = ld_dout;
    p.ldx = ldx;
    p.ld_res = ld_res;
    p.ld_dx = ld_dx;
    p.grad_f32 = grad_dtype == FSWIGLU_OUT_F32;
    p.dweight = dweight;
    p.dbias = dbias;
    p.M = static_cast<int>(M);
    p.d = static_cast<int>(d);
    p.splits = norm_splits(M);
    p.ring = RingParams{dev.status, dev.wait_limit_ns, 0, 0, 1};
    p.w_f32 = w_dtype == FSWIGLU_OUT_F32 && weight != nullptr;
    const bool wide = d * type_bytes(x_dtype) % 16 == 0 && wide_rows(dout, ld_dout, M, x_dtype) && wide_rows(x, ldx, M, x_dtype) &&
                      wide_rows(dx, ld_dx, M, x_dtype) && wide_rows(residual, residual == nullptr ? 0 : ld_res, M, x_dtype) &&
                      aligned(weight, 16);
    using BF = __nv_bfloat16;
    int rc;
    if (x_dtype == FSWIGLU_OUT_F32)
      rc = layer ? launch_norm_backward<float, true>(p, wide, dev, s) : launch_norm_backward<float, false>(p, wide, dev, s);
    else
      rc = layer ? launch_norm_backward<BF, true>(p, wide, dev, s) : launch_norm_backward<BF, false>(p, wide, dev, s);
    if (rc) return rc;
  }
  if (!columns || p.cluster) return FSWIGLU_OK;
  NormReduceParams q = {};  // no rows: no splits, the gradients are zero
  q.partial = p.partial;
  q.dweight = dweight;
  q.dbias = dbias;
  q.d = static_cast<int>(d);
  q.splits = p.splits;
  q.out_f32 = grad_dtype == FSWIGLU_OUT_F32;
  const dim3 block(32, kNormReduceRows);
  return dbias != nullptr ? launch(norm_reduce_kernel<true>, (d + 31) / 32, block, 0, s, q)
                          : launch(norm_reduce_kernel<false>, (d + 31) / 32, block, 0, s, q);
}

// ---- many tensors ----

constexpr int kSmallTable = 48;   // kernel parameters below 4 KB: what every launch copies
constexpr int kLargeTable = 400;  // below the 32764 bytes that a launch takes

struct Range {
  uintptr_t begin, end;
};

// Whether no two of the call's written ranges of one kind overlap.  Ranges in ascending order, as an allocator hands
// them out, need no copy; others are sorted.
template <typename Get>
int disjoint(int64_t count, Get get) {
  bool ascending = true;
  uintptr_t last = 0;
  for (int64_t i = 0; i < count && ascending; ++i) {
    const Range r = get(i);
    if (r.begin == r.end) continue;
    ascending = r.begin >= last;
    last = r.end;
  }
  if (ascending) return FSWIGLU_OK;
  std::unique_ptr<Range[]> all(new (std::nothrow) Range[count]);
  if (all == nullptr) return FSWIGLU_ERR_BAD_ARG;
  int64_t n = 0;
  for (int64_t i = 0; i < count; ++i) {
    const Range r = get(i);
    if (r.begin != r.end) all[n++] = r;
  }
  std::sort(all.get(), all.get() + n, [](const Range& a, const Range& b) { return a.begin < b.begin; });
  for (int64_t i = 1; i < n; ++i) {
    if (all[i].begin < all[i - 1].end) return FSWIGLU_ERR_BAD_ARG;
  }
  return FSWIGLU_OK;
}

Range range_of(const void* p, int64_t bytes) {
  const uintptr_t b = reinterpret_cast<uintptr_t>(p);
  return Range{b, b + static_cast<uintptr_t>(p == nullptr ? 0 : bytes)};
}

uint32_t chunks_of(int64_t numel, int64_t chunk) { return static_cast<uint32_t>((numel + chunk - 1) / chunk); }

constexpr int64_t kMaxNumel = 1ll << 34;  // chunks of a full table are counted in 32 bits

struct AdamKind {
  bool param_f32, grad_f32, eight, master;
};

template <typename P, typename G, bool kMaster, int kCapacity>
int launch_adamw(AdamTable<kCapacity>& t, const AdamKind& k, const Device& dev, cudaStream_t s) {
  const int64_t chunks = t.first_chunk[t.count];
  if (k.eight) {
    // a ring pays where each block has several parts
    const int64_t resident = static_cast<int64_t>(dev.sms) * kAdam8Blocks;
    if (chunks >= 4 * resident) {
      constexpr auto kernel = adamw8_kernel<P, G, kMaster, true, kCapacity>;
      static_assert(sizeof(Adam8Shared<typename std::conditional<kMaster, float, P>::type, G>) <= kRingBytes / kAdam8Blocks,
                    "the blocks of an SM share its memory");
      static std::atomic<uint64_t> done{0};
      if (int rc = opt_in(kernel, &done, dev)) return rc;
      t.withhold = take_withhold();
      // all of the SM's memory for its two blocks: a third one, of a launch that starts early, would leave other SMs one
      return launch(kernel, resident, dim3(kAdam8RingThreads), kRingBytes / kAdam8Blocks, s, t);
    }
    return launch(adamw8_kernel<P, G, kMaster, false, kCapacity>, chunks, dim3(kAdamThreads), 0, s, t);
  }
  // a block for each chunk: SMs that are done take the next (3 x 45 M weights: 559 us; 16 blocks an SM that stay: 584)
  return launch(adamw32_kernel<P, G, kMaster, kCapacity>, std::min<int64_t>(chunks, 1 << 30), dim3(kAdamThreads), 0, s, t);
}

template <int kCapacity>
int launch_adamw(AdamTable<kCapacity>& t, const AdamKind& k, const Device& dev, cudaStream_t s) {
  using BF = __nv_bfloat16;
  if (k.param_f32) return k.grad_f32 ? launch_adamw<float, float, false>(t, k, dev, s) : launch_adamw<float, BF, false>(t, k, dev, s);
  if (k.master) return k.grad_f32 ? launch_adamw<BF, float, true>(t, k, dev, s) : launch_adamw<BF, BF, true>(t, k, dev, s);
  return k.grad_f32 ? launch_adamw<BF, float, false>(t, k, dev, s) : launch_adamw<BF, BF, false>(t, k, dev, s);
}

// Whether every pointer of a tensor takes the wide accesses of eight elements, and bulk copies.
bool wide(const fswiglu_adamw_tensor& a, const AdamKind& k) {
  const size_t p = k.param_f32 ? 32 : 16, g = k.grad_f32 ? 32 : 16, m = k.eight ? 16 : 32;
  return aligned(a.param, p) && aligned(a.grad, g) && aligned(a.exp_avg, m) && aligned(a.exp_avg_sq, m) && aligned(a.master, 32) &&
         aligned(a.exp_avg_scale, 16) && aligned(a.exp_avg_sq_scale, 16);
}

template <int kCapacity>
int adamw_launches(const fswiglu_adamw_tensor* tensors, int64_t count, const AdamOptions& o, AdamKind kind, int parts,
                   const Device& dev, cudaStream_t s) {
  AdamTable<kCapacity> t;
  t.opt = o;
  t.count = 0;
  t.parts = parts;
  t.status = dev.status;
  t.wait_limit_ns = dev.wait_limit_ns;
  t.withhold = 0;
  t.first_chunk[0] = 0;
  long long blocks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const fswiglu_adamw_tensor& a = tensors[i];
    if (a.numel > 0) {
      // one launch's tensors all have a master or none has
      if (t.count > 0 && (a.master != nullptr) != kind.master) {
        if (int rc = launch_adamw<kCapacity>(t, kind, dev, s)) return rc;
        t.count = 0;
      }
      kind.master = a.master != nullptr;
      const long long n = a.numel;
      t.tensors[t.count] = AdamTensor{a.param,  a.grad, a.exp_avg, a.exp_avg_sq, a.master, a.exp_avg_scale,
                                      a.exp_avg_sq_scale, wide(a, kind) ? n : ~n};
      t.first_block[t.count] = blocks;
      t.first_chunk[t.count + 1] = t.first_chunk[t.count] + chunks_of(a.numel, static_cast<int64_t>(t.parts) * kAdamPart);
      blocks += (a.numel + kAdamBlock - 1) / kAdamBlock;
      ++t.count;
    }
    if (t.count == 0 || (t.count < kCapacity && i + 1 < count)) continue;
    if (int rc = launch_adamw<kCapacity>(t, kind, dev, s)) return rc;
    t.count = 0;
  }
  return FSWIGLU_OK;
}

template <int kCapacity>
void add_grad(GradTable<kCapacity>& t, const fswiglu_grad_tensor& a) {
  if (a.numel == 0) return;
  const bool f32 = a.dtype == FSWIGLU_OUT_F32;
  t.tensors[t.count] = GradTensor{a.grad, static_cast<long long>(a.numel), f32, aligned(a.grad, f32 ? 32 : 16)};
  t.first_chunk[t.count + 1] = t.first_chunk[t.count] + chunks_of(a.numel, kGradChunk);
  ++t.count;
}

template <int kCapacity>
int grad_norm_launches(const fswiglu_grad_tensor* tensors, int64_t count, double* slots, int* used, int sms, cudaStream_t s) {
  GradTable<kCapacity> t;
  t.slots = slots;
  t.count = 0;
  t.first_chunk[0] = 0;
  t.accumulate = 0;
  for (int64_t i = 0; i < count; ++i) {
    add_grad(t, tensors[i]);
    if (t.count == 0 || (t.count < kCapacity && i + 1 < count)) continue;
    // every launch of a call has the same thread blocks: a later one adds to the slots of the first
    const int grid = std::min(kGradNormSlots, sms * 8);
    if (int rc = launch(grad_norm_kernel<kCapacity>, grid, dim3(kAdamThreads), 0, s, t)) return rc;
    *used = grid;
    t.accumulate = 1;
    t.count = 0;
  }
  return FSWIGLU_OK;
}

// Up to this many chunks a launch of one cluster takes the place of one over all SMs and another that joins: 16 chunks of one
// tensor 5.0 us a call (6.6 with two launches) and 2.7 to 3.4 us in a graph (3.2 to 3.5); 24 chunks 5.0 (6.5) and 3.0 to 3.9 (3.3 to
// 3.6); 48 chunks 6.8 (6.5) and 6.2 (3.6) in fp32.
constexpr int64_t kFewChunks = 24;
static_assert(kFewChunks <= kSmallTable, "a tensor has a chunk at least");

int grad_norm_few(const fswiglu_grad_tensor* tensors, int64_t count, float max_norm, float* out, cudaStream_t s) {
  GradTable<kSmallTable> t;
  t.slots = nullptr;
  t.count = 0;
  t.first_chunk[0] = 0;
  t.accumulate = 0;
  for (int64_t i = 0; i < count; ++i) add_grad(t, tensors[i]);
  return launch_clusters(kFewBlocks, grad_norm_few_kernel<kSmallTable>, kFewBlocks, dim3(kAdamThreads), 0, s, t, max_norm, out);
}

}  // namespace

extern "C" {

int fswiglu_layer_norm_forward(const void* x, int64_t ldx, const void* weight, const void* bias, void* y, int64_t ldy,
                               float* mean, float* rstd, int64_t M, int64_t d, int x_dtype, int w_dtype, float eps,
                               void* stream) {
  return norm_forward(true, x, ldx, weight, bias, y, ldy, mean, rstd, M, d, x_dtype, w_dtype, eps, stream);
}

int fswiglu_rms_norm_forward(const void* x, int64_t ldx, const void* weight, void* y, int64_t ldy, float* rstd, int64_t M,
                             int64_t d, int x_dtype, int w_dtype, float eps, void* stream) {
  return norm_forward(false, x, ldx, weight, nullptr, y, ldy, nullptr, rstd, M, d, x_dtype, w_dtype, eps, stream);
}

size_t fswiglu_norm_backward_workspace_bytes(int64_t M, int64_t d) {
  if (M <= 0 || d <= 0 || d > kMaxNormWidth) return 0;
  return (static_cast<size_t>(norm_splits(M)) * 2u * static_cast<size_t>(d) * 4u + 255u) / 256u * 256u;
}

int fswiglu_layer_norm_backward(const void* dout, int64_t ld_dout, const void* x, int64_t ldx, const float* mean,
                                const float* rstd, const void* weight, const void* residual, int64_t ld_res, void* dx,
                                int64_t ld_dx, void* dweight, void* dbias, int64_t M, int64_t d, int x_dtype, int w_dtype,
                                int grad_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  return norm_backward(true, dout, ld_dout, x, ldx, mean, rstd, weight, residual, ld_res, dx, ld_dx, dweight, dbias, M, d,
                       x_dtype, w_dtype, grad_dtype, workspace, workspace_bytes, stream);
}

int fswiglu_rms_norm_backward(const void* dout, int64_t ld_dout, const void* x, int64_t ldx, const float* rstd,
                              const void* weight, const void* residual, int64_t ld_res, void* dx, int64_t ld_dx,
                              void* dweight, int64_t M, int64_t d, int x_dtype, int w_dtype, int grad_dtype,
                              void* workspace, size_t workspace_bytes, void* stream) {
  return norm_backward(false, dout, ld_dout, x, ldx, nullptr, rstd, weight, residual, ld_res, dx, ld_dx, dweight, nullptr,
                       M, d, x_dtype, w_dtype, grad_dtype, workspace, workspace_bytes, stream);
}

int fswiglu_adamw_step(const fswiglu_adamw_tensor* tensors, int64_t count, int param_dtype, int grad_dtype, int state_bits,
                       const fswiglu_adamw_options* options, void* stream) {
  if (count < 0 || (count > 0 && tensors == nullptr) || options == nullptr) return FSWIGLU_ERR_BAD_ARG;
  if (!known_type(param_dtype) || !known_type(grad_dtype) || (state_bits != 8 && state_bits != 32)) return FSWIGLU_ERR_BAD_ARG;
  const fswiglu_adamw_options& in = *options;
  if (!(in.beta1 >= 0.0 && in.beta1 < 1.0 && in.beta2 >= 0.0 && in.beta2 < 1.0 && in.eps >= 0.0 && in.weight_decay >= 0.0) ||
      !std::isfinite(in.eps) || !std::isfinite(in.weight_decay))
    return FSWIGLU_ERR_BAD_ARG;
  if (in.lr_device == nullptr && !(in.lr >= 0.0 && std::isfinite(in.lr))) return FSWIGLU_ERR_BAD_ARG;
  if (in.step_device == nullptr && in.step < 1) return FSWIGLU_ERR_BAD_ARG;
  if (!aligned(in.lr_device, 4) || !aligned(in.step_device, 8) || !aligned(in.grad_scale, 4)) return FSWIGLU_ERR_ALIGNMENT;
  const size_t pb = type_bytes(param_dtype), gb = type_bytes(grad_dtype), sb = state_bits == 8 ? 1u : 4u;
  bool any = false;
  for (int64_t i = 0; i < count; ++i) {
    const fswiglu_adamw_tensor& a = tensors[i];
    if (a.numel < 0) return FSWIGLU_ERR_BAD_ARG;
    if (a.numel == 0) continue;
    if (a.numel > kMaxNumel) return FSWIGLU_ERR_SHAPE;
    any = true;
    if (a.param == nullptr || a.grad == nullptr || a.exp_avg == nullptr || a.exp_avg_sq == nullptr) return FSWIGLU_ERR_BAD_ARG;
    if (state_bits == 8 && (a.exp_avg_scale == nullptr || a.exp_avg_sq_scale == nullptr)) return FSWIGLU_ERR_BAD_ARG;
    if (param_dtype == FSWIGLU_OUT_F32 && a.master != nullptr) return FSWIGLU_ERR_BAD_ARG;
    if (!aligned(a.param, pb) || !aligned(a.grad, gb) || !aligned(a.exp_avg, sb) || !aligned(a.exp_avg_sq, sb) ||
        !aligned(a.master, 4) || !aligned(a.exp_avg_scale, 4) || !aligned(a.exp_avg_sq_scale, 4))
      return FSWIGLU_ERR_ALIGNMENT;
  }
  if (!any) return FSWIGLU_OK;
  int rc;
  if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].param, tensors[i].numel * static_cast<int64_t>(pb)); })))
    return rc;
  if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].exp_avg, tensors[i].numel * static_cast<int64_t>(sb)); })))
    return rc;
  if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].exp_avg_sq, tensors[i].numel * static_cast<int64_t>(sb)); })))
    return rc;
  if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].master, tensors[i].numel * 4); }))) return rc;
  if (state_bits == 8) {
    auto scales = [&](int64_t i) { return (tensors[i].numel + kAdamBlock - 1) / kAdamBlock * 4; };
    if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].exp_avg_scale, scales(i)); }))) return rc;
    if ((rc = disjoint(count, [&](int64_t i) { return range_of(tensors[i].exp_avg_sq_scale, scales(i)); }))) return rc;
  }
  Device dev;
  if ((rc = current_device(&dev))) return rc;
  AdamOptions o = {};
  o.log_beta1 = std::log(in.beta1);
  o.log_beta2 = std::log(in.beta2);
  o.lr = static_cast<float>(in.lr);
  o.beta1 = static_cast<float>(in.beta1);
  o.one_minus_beta1 = static_cast<float>(1.0 - in.beta1);
  o.beta2 = static_cast<float>(in.beta2);
  o.one_minus_beta2 = static_cast<float>(1.0 - in.beta2);
  o.eps = static_cast<float>(in.eps);
  o.weight_decay = static_cast<float>(in.weight_decay);
  if (in.step_device == nullptr) {
    const double t = static_cast<double>(in.step);
    const double lr = in.lr_device == nullptr ? in.lr : 1.0;
    o.step_size = static_cast<float>(lr / (1.0 - std::pow(in.beta1, t)));
    o.inv_sqrt_correction2 = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(in.beta2, t)));
  }
  o.lr_device = in.lr_device;
  o.step_device = reinterpret_cast<const long long*>(in.step_device);
  o.grad_scale = in.grad_scale;
  o.seed_lo = static_cast<uint32_t>(in.seed);
  o.seed_hi = static_cast<uint32_t>(in.seed >> 32);
  o.step_lo = static_cast<uint32_t>(in.step);
  const AdamKind kind = {param_dtype == FSWIGLU_OUT_F32, grad_dtype == FSWIGLU_OUT_F32, state_bits == 8, false};
  // with fp32 moments two parts to a chunk where each SM has chunks enough
  int64_t total = 0;
  for (int64_t i = 0; i < count; ++i) total += tensors[i].numel;
  const int parts = state_bits == 32 && total / (2 * kAdamPart) >= 8 * dev.sms ? 2 : 1;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return count <= kSmallTable ? adamw_launches<kSmallTable>(tensors, count, o, kind, parts, dev, s)
                              : adamw_launches<kLargeTable>(tensors, count, o, kind, parts, dev, s);
}

size_t fswiglu_grad_norm_workspace_bytes(void) { return kGradNormSlots * sizeof(double); }

int fswiglu_grad_norm_clip(const fswiglu_grad_tensor* tensors, int64_t count, float max_norm, float* out, void* workspace,
                           size_t workspace_bytes, void* stream) {
  if (count < 0 || (count > 0 && tensors == nullptr) || out == nullptr || !(max_norm >= 0.0f)) return FSWIGLU_ERR_BAD_ARG;
  if (workspace == nullptr || workspace_bytes < fswiglu_grad_norm_workspace_bytes() || !aligned(workspace, 256))
    return FSWIGLU_ERR_WORKSPACE;
  if (!aligned(out, 4)) return FSWIGLU_ERR_ALIGNMENT;
  int64_t chunks = 0;
  for (int64_t i = 0; i < count; ++i) {
    const fswiglu_grad_tensor& a = tensors[i];
    if (a.numel < 0 || !known_type(a.dtype)) return FSWIGLU_ERR_BAD_ARG;
    if (a.numel == 0) continue;
    if (a.numel > kMaxNumel) return FSWIGLU_ERR_SHAPE;
    if (a.grad == nullptr) return FSWIGLU_ERR_BAD_ARG;
    if (!aligned(a.grad, type_bytes(a.dtype))) return FSWIGLU_ERR_ALIGNMENT;
    chunks += chunks_of(a.numel, kGradChunk);
  }
  Device dev;
  if (int rc = current_device(&dev)) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (chunks <= kFewChunks) return grad_norm_few(tensors, count, max_norm, out, s);
  double* slots = static_cast<double*>(workspace);
  int used = 0;
  const int rc = count <= kSmallTable ? grad_norm_launches<kSmallTable>(tensors, count, slots, &used, dev.sms, s)
                                      : grad_norm_launches<kLargeTable>(tensors, count, slots, &used, dev.sms, s);
  if (rc) return rc;
  return launch(grad_norm_finish_kernel, 1, dim3(kAdamThreads), 0, s, static_cast<const double*>(slots), used, max_norm, out);
}

}  // extern "C"
