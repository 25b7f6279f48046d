// host.cuh -- host-side helpers of the C ABI entry points: streams, alignment checks,
// shared-memory opt-in, launches with programmatic stream serialization (PDL) and TMA
// tensor maps.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>
#include <utility>

#include "common.cuh"

namespace spark {

inline int g_pdl = 1;

inline cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// cudaFuncSetAttribute is per (function, device).  Remember which pairs are done so
// that launches during stream capture make no further attribute calls.
struct SmemDone {
  const void* fn;
  int dev;
  size_t bytes;
};
inline SmemDone g_smem_done[512];
inline int g_smem_count = 0;
inline std::mutex g_smem_mu;

inline int set_smem(const void* kernel, size_t smem) {
  if (smem <= 48 * 1024) return kOk;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return kErrLaunch;
  std::lock_guard<std::mutex> lock(g_smem_mu);
  for (int i = 0; i < g_smem_count; i++)
    if (g_smem_done[i].fn == kernel && g_smem_done[i].dev == dev && g_smem_done[i].bytes >= smem) return kOk;
  // always request the maximum (what the kernel's static part leaves of it) so one call
  // serves every later size
  cudaFuncAttributes fa;
  if (cudaFuncGetAttributes(&fa, kernel) != cudaSuccess) return kErrLaunch;
  const int max_bytes = 227 * 1024 - (int)fa.sharedSizeBytes;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, max_bytes) != cudaSuccess)
    return kErrLaunch;
  for (int i = 0; i < g_smem_count; i++)
    if (g_smem_done[i].fn == kernel && g_smem_done[i].dev == dev) {
      g_smem_done[i].bytes = max_bytes;
      return kOk;
    }
  if (g_smem_count < 512) g_smem_done[g_smem_count++] = {kernel, dev, (size_t)max_bytes};
  return kOk;
}

template <typename... KArgs, typename... Args>
int launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
  if (set_smem(reinterpret_cast<const void*>(kernel), smem) != kOk) return kErrLaunch;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = g_pdl;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
  return e == cudaSuccess ? kOk : kErrLaunch;
}

inline int num_sms() {
  static int cached[64] = {0};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return kNumSMs;
  if (!cached[dev]) {
    int v = 0;
    cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev);
    cached[dev] = v > 0 ? v : kNumSMs;
  }
  return cached[dev];
}

// cuTensorMapEncodeTiled from the driver, through the runtime's entry-point query (no
// link against libcuda)
inline PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// 3-D tensor map of 2-byte elements with the 128-byte swizzle (pitches in bytes)
inline bool encode_map3(CUtensorMap* m, CUtensorMapDataType dt, const void* base, const uint64_t (&dim)[3],
                        const uint64_t (&pitch)[2], const uint32_t (&boxes)[3]) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[3] = {dim[0], dim[1], dim[2]};
  cuuint64_t strides[2] = {pitch[0], pitch[1]};
  cuuint32_t box[3] = {boxes[0], boxes[1], boxes[2]};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(m, dt, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) ==
         CUDA_SUCCESS;
}

// 2-D tensor map: `inner` elements per row (row pitch `pitch` bytes), `outer` rows
inline bool encode_map(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t outer,
                       uint64_t pitch, uint32_t box_inner, uint32_t box_outer, CUtensorMapSwizzle sw) {
  auto fn = tensor_map_encoder();
  if (!fn) return false;
  cuuint64_t dims[2] = {inner, outer};
  cuuint64_t strides[1] = {pitch};
  cuuint32_t box[2] = {box_inner, box_outer};
  cuuint32_t estr[2] = {1, 1};
  return fn(m, dt, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace spark
