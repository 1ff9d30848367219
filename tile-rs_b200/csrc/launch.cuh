// What the launch functions of every operator share: messages, scratch, facts about kernels that are asked once, launches in clusters or as
// programmatic dependents, tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <tuple>
#include <utility>

#include "../../include/tile_sm100.h"
#include "scratch.hpp"

namespace tsm100 {
namespace ops {

inline int32_t op_fail(std::string* err, int32_t code, const std::string& msg) {
  if (err) *err = msg;
  return code;
}

inline int32_t cuda_ok(std::string* err, cudaError_t e, const char* what) {
  if (e == cudaSuccess) return TSM100_OK;
  const int32_t code = (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) ? TSM100_ERR_NO_DEVICE
                                                                                      : TSM100_ERR_LAUNCH;
  return op_fail(err, code, std::string(what) + " failed: " + cudaGetErrorString(e));
}

// What an operator's launch function answers, without a message, when the pool cannot give it the scratch it would like
// and a form without scratch exists: the dispatch then takes that one.
constexpr int32_t kNoScratch = -1;
inline int32_t take_scratch(std::string* err, void** ws, size_t bytes, cudaStream_t s) {
  const cudaError_t e = scratch::take(ws, bytes, s);
  if (e == cudaErrorMemoryAllocation || e == cudaErrorNotSupported) {
    (void)cudaGetLastError();
    return kNoScratch;
  }
  return cuda_ok(err, e, "scratch from the library's memory pool");
}

inline size_t dtype_size(int32_t dtype) { return dtype == TSM100_F32 ? 4 : 2; }
inline bool dtype_valid(int32_t dtype) { return dtype == TSM100_F32 || dtype == TSM100_F16 || dtype == TSM100_BF16; }
inline bool dtype_16bit(int32_t dtype) { return dtype == TSM100_F16 || dtype == TSM100_BF16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---------------------------------------------------------------------------
// per-(kernel, device) facts: asked of the CUDA runtime once, then remembered
// ---------------------------------------------------------------------------
// cudaFuncSetAttribute and the occupancy queries cost a few microseconds each, which is as long as
// a small launch itself; their answers depend on the kernel and the device only.
struct KernelFacts {
  std::mutex mu;
  std::map<std::tuple<const void*, int, int>, int> value;  // (kernel, device, what) -> answer
};
// Hidden, so that the library and every kernel module built from these headers have one each: a module's kernels lie at addresses that another may have after it is
// unloaded, and what a module is first to construct is destroyed with it.
__attribute__((visibility("hidden"))) inline KernelFacts& kernel_facts() {
  static KernelFacts f;
  return f;
}
enum { kFactSmemSet = 1, kFactNonPortableSet = 2, kFactBlocksPerSm = 3, kFactClusters = 4 };

// `compute` returns (ok, answer); an answer is remembered only when ok.
template <typename F>
inline bool kernel_fact(const void* kern, int what, int* answer, F compute) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) dev = -1;
  KernelFacts& f = kernel_facts();
  const auto key = std::make_tuple(kern, dev, what);
  {
    std::lock_guard<std::mutex> lock(f.mu);
    auto it = f.value.find(key);
    if (it != f.value.end()) {
      *answer = it->second;
      return true;
    }
  }
  if (!compute(answer)) return false;
  std::lock_guard<std::mutex> lock(f.mu);
  f.value[key] = *answer;
  return true;
}

// cudaFuncAttributeMaxDynamicSharedMemorySize, set once per kernel and device.
template <typename K>
inline cudaError_t set_dyn_smem_once(K kern, int bytes) {
  cudaError_t e = cudaSuccess;
  int unused = 0;
  kernel_fact(reinterpret_cast<const void*>(kern), kFactSmemSet, &unused, [&](int* out) {
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    *out = bytes;
    return e == cudaSuccess;
  });
  return e;
}
template <typename K>
inline cudaError_t allow_wide_clusters_once(K kern) {
  cudaError_t e = cudaSuccess;
  int unused = 0;
  kernel_fact(reinterpret_cast<const void*>(kern), kFactNonPortableSet, &unused, [&](int* out) {
    e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kern), cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    *out = 1;
    return e == cudaSuccess;
  });
  return e;
}
// Launches a kernel in clusters of `cluster` CTAs where that is not 0; chained: as a programmatic dependent of the one before it in
// the stream (the rules that such kernels keep are in ptx.cuh).  What that saves is the time between two kernels of a chain of calls:
// the end of one grid, the launch of the next and its set-up run side by side.  bf16 MLP of 16 tokens, 4096 x 16384: 84.1 us, 78.1
// chained and with the weights' first tiles fetched meanwhile; one token of one sequence of 32768, with rotation and appends: 38.1 / 36.3, of
// 1000 18.8 / 14.1; 16 x 4096 x 4096 in a row of calls 8.9 / 8.4 (all as graph replays).
template <typename... P, typename... A>
inline cudaError_t launch_kernel(bool chained, void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, unsigned cluster, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if (cluster) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = cluster;
    attr[n].val.clusterDim.y = 1;
    attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (chained) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<A>(args)...);
}
template <typename... P, typename... A>
inline cudaError_t launch_chained(void (*kern)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s, unsigned cluster, A&&... args) {
  return launch_kernel(true, kern, grid, threads, smem, s, cluster, std::forward<A>(args)...);
}
// How many clusters of `cluster` CTAs of a kernel the GPU holds at once, asked once per kernel and device; `fallback` if it cannot tell.
template <typename K>
inline int resident_clusters(K kern, unsigned threads, size_t smem, unsigned cluster, unsigned grid, int fallback) {
  int answer = fallback;
  kernel_fact(reinterpret_cast<const void*>(kern), kFactClusters, &answer, [&](int* out) {
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      return false;
    }
    *out = n;
    return true;
  });
  return answer;
}
// Resident CTAs per SM of a kernel launched with `threads` threads and no dynamic shared memory (at least 1).
template <typename K>
inline int blocks_per_sm(K kern, int threads) {
  int per_sm = 1;
  kernel_fact(reinterpret_cast<const void*>(kern), kFactBlocksPerSm + (threads << 8), &per_sm, [&](int* out) {
    int n = 1;
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, 0) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      return false;
    }
    *out = n;
    return true;
  });
  return per_sm < 1 ? 1 : per_sm;
}

// ---------------------------------------------------------------------------
// tensor maps
// ---------------------------------------------------------------------------
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline int32_t encode_fn(std::string* err, EncodeTiledFn* out) {
  static EncodeTiledFn cached = nullptr;
  if (!cached) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult qres;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &qres);
    if (e != cudaSuccess || qres != cudaDriverEntryPointSuccess || !fn)
      return op_fail(err, TSM100_ERR_NO_DEVICE, "cuTensorMapEncodeTiled is not available from the CUDA driver");
    cached = reinterpret_cast<EncodeTiledFn>(fn);
  }
  *out = cached;
  return TSM100_OK;
}

// A map is a pure function of its arguments, and a repeated launch (same pointers, same shape) asks for the same
// ones again: each thread keeps the last few it encoded.
struct TmapKey {
  const void* base;
  uint64_t dim[4], stride[3];  // stride: bytes; dimension 0 is contiguous
  uint32_t box[4];
  int32_t dtype, rank;
};
struct TmapSlot {
  TmapKey key;
  CUtensorMap map;
  bool used = false;
};

// `key` all zeros beyond its rank.  128-byte swizzle (64-byte where a row of the box has 64 bytes), out-of-range elements read as zero.
inline int32_t make_tmap(std::string* err, CUtensorMap* out, const TmapKey& key, uint32_t elem_bytes) {
  constexpr int kSlots = 16;
  static thread_local TmapSlot cache[kSlots];
  static thread_local int next = 0;
  for (int i = 0; i < kSlots; ++i)
    if (cache[i].used && std::memcmp(&cache[i].key, &key, sizeof key) == 0) {
      *out = cache[i].map;
      return TSM100_OK;
    }
  EncodeTiledFn fn;
  int32_t st = encode_fn(err, &fn);
  if (st != TSM100_OK) return st;
  cuuint64_t dims[4], strides[3];
  cuuint32_t box[4], estr[4] = {1, 1, 1, 1};
  for (int i = 0; i < key.rank; ++i) dims[i] = key.dim[i], box[i] = key.box[i];
  for (int i = 0; i + 1 < key.rank; ++i) {
    strides[i] = key.stride[i];
    if (strides[i] & 15u) return op_fail(err, TSM100_ERR_INVALID, "tensor map needs a 16-byte aligned base and 16-byte-multiple strides");
  }
  if (!aligned16(key.base)) return op_fail(err, TSM100_ERR_INVALID, "tensor map needs a 16-byte aligned base and 16-byte-multiple strides");
  CUresult r = fn(out, static_cast<CUtensorMapDataType>(key.dtype), static_cast<cuuint32_t>(key.rank), const_cast<void*>(key.base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, box[0] * elem_bytes == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    char buf[96];
    snprintf(buf, sizeof buf, "cuTensorMapEncodeTiled failed: CUresult %d", static_cast<int>(r));
    return op_fail(err, TSM100_ERR_LAUNCH, buf);
  }
  TmapSlot& slot = cache[next];
  next = (next + 1) % kSlots;
  slot.key = key;
  slot.map = *out;
  slot.used = true;
  return TSM100_OK;
}
// dims (x contiguous, y, z), strides in elements of `elem_bytes`, box (box_x, box_y, 1).
inline int32_t make_tmap_3d(std::string* err, CUtensorMap* out, const void* base, uint64_t dim_x, uint64_t dim_y,
                            uint64_t dim_z, uint64_t stride_y, uint64_t stride_z, uint32_t box_x, uint32_t box_y,
                            CUtensorMapDataType dtype, uint32_t elem_bytes) {
  TmapKey key;
  std::memset(&key, 0, sizeof key);
  key.base = base;
  key.dim[0] = dim_x, key.dim[1] = dim_y, key.dim[2] = dim_z;
  key.stride[0] = stride_y * elem_bytes, key.stride[1] = stride_z * elem_bytes;
  key.box[0] = box_x, key.box[1] = box_y, key.box[2] = 1;
  key.dtype = static_cast<int32_t>(dtype), key.rank = 3;
  return make_tmap(err, out, key, elem_bytes);
}

// 16-bit elements (bf16 or f16).
inline int32_t make_tmap_16bit_3d(std::string* err, CUtensorMap* out, const void* base, uint64_t dim_x,
                                  uint64_t dim_y, uint64_t dim_z, uint64_t stride_y, uint64_t stride_z,
                                  uint32_t box_x, uint32_t box_y, bool is_bf16) {
  return make_tmap_3d(err, out, base, dim_x, dim_y, dim_z, stride_y, stride_z, box_x, box_y,
                      is_bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2);
}

inline int32_t sm_count(std::string* err, int* sms) {
  static int cached[64] = {0};
  int dev = 0;
  int32_t st = cuda_ok(err, cudaGetDevice(&dev), "cudaGetDevice");
  if (st != TSM100_OK) return st;
  if (dev < 64 && cached[dev]) {
    *sms = cached[dev];
    return TSM100_OK;
  }
  int n = 0;
  st = cuda_ok(err, cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev), "cudaDeviceGetAttribute");
  if (st != TSM100_OK) return st;
  if (dev < 64) cached[dev] = n;
  *sms = n;
  return TSM100_OK;
}

}  // namespace ops
}  // namespace tsm100
