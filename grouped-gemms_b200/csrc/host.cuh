// Host-side helpers shared by the C ABI's translation units (capi.cu defines
// them): error messages, per-device state and tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "../../include/mxgg.h"

namespace mxgg {

// Records the calling thread's message (mxgg_last_error) and returns `code`.
int fail(int code, const char* fmt, ...);

#define MXGG_CUDA_TRY(expr)                                                                   \
  do {                                                                                        \
    cudaError_t e_ = (expr);                                                                  \
    if (e_ != cudaSuccess) return fail(MXGG_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(e_)); \
  } while (0)

struct DeviceState {
  bool init = false;
  int device = 0;
  int num_sms = 0;
  uint32_t* status = nullptr;   // device address of the status word bounded waits raise
};

// State of the current device (checked to be sm_100 on first use).
int get_device_state(DeviceState** out);

// Limit of every bounded device-side wait, in ns.
unsigned long long wait_limit_ns();

int make_tmap_2d(CUtensorMap* map, const void* base, CUtensorMapDataType dt, int esize, uint64_t rows, uint64_t cols,
                 uint64_t row_stride_elems, uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swz);
int make_tmap_3d(CUtensorMap* map, const void* base, CUtensorMapDataType dt, int esize, uint64_t mats, uint64_t rows,
                 uint64_t cols, uint64_t row_stride_elems, uint64_t mat_stride_elems, uint32_t box_cols,
                 uint32_t box_rows, uint32_t box_mats, CUtensorMapSwizzle swz);

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Allows `kernel` `bytes` of dynamic shared memory (and clusters of more than 8
// CTAs), on the first call for a device.  `bytes` is the most that any launch of
// it takes, never one call's own size: the limit belongs to the function, and a
// call that lowered it between another thread's setting and launch would make
// that launch fail.  Two first calls at once both set the same.
constexpr int kMaxDevices = 64;
template <auto kernel>
int allow_smem(const DeviceState& st, int bytes, bool large_cluster = false) {
  static std::atomic<bool> done[kMaxDevices] = {};
  if (done[st.device].load(std::memory_order_acquire)) return MXGG_OK;
  MXGG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  if (large_cluster) MXGG_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  done[st.device].store(true, std::memory_order_release);
  return MXGG_OK;
}

// Launch with a cluster along x and/or programmatic stream serialisation: the
// kernel may then start while the stream's previous kernel drains, and must
// execute griddepcontrol.wait before it reads what that one wrote.
template <typename... KArgs, typename... Args>
cudaError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, int cluster, bool pdl,
                   cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (cluster > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = (unsigned)cluster;
    at[n].val.clusterDim.y = 1;
    at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace mxgg
