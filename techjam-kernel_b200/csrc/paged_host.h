// paged_host.h — host-side pieces shared by the paged-cache kernels: argument
// checks, device selection and the launch helper.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <mutex>

#include "b200_paged.h"
#include "error_word.cuh"

namespace b200paged {

using b200attn::count_launch;
using b200attn::resolve_error_word;
using b200attn::set_error;

constexpr int kMaxDevices = 64;

inline int64_t elem_bytes(int32_t dtype) { return dtype == B200_ATTN_DTYPE_FP32 ? 4 : 2; }

inline bool known_dtype(int32_t dtype) {
  return dtype == B200_ATTN_DTYPE_BF16 || dtype == B200_ATTN_DTYPE_FP16 ||
         dtype == B200_ATTN_DTYPE_FP32;
}

// A base and the strides of its dimensions with extent > 1 on 16-byte
// boundaries (rows are read and written 16 bytes at a time).
inline bool vectors_aligned(const void* base, const int64_t* stride, const int64_t* extent, int n,
                            int64_t eb) {
  if (reinterpret_cast<uintptr_t>(base) & 15u) return false;
  for (int d = 0; d < n; ++d)
    if (extent[d] > 1 && (stride[d] < 0 || (stride[d] * eb) % 16 != 0)) return false;
  return true;
}

// Makes the device of `ptr` current for the call; the caller's is restored.
struct DeviceScope {
  int prev = -1;
  int device = 0;
  int32_t enter(const void* ptr, const char* what) {
    cudaPointerAttributes attr;
    if (cudaPointerGetAttributes(&attr, ptr) != cudaSuccess || attr.device < 0 ||
        attr.device >= kMaxDevices ||
        (attr.type != cudaMemoryTypeDevice && attr.type != cudaMemoryTypeManaged)) {
      cudaGetLastError();
      set_error(what);
      return B200_ATTN_ERR_DEVICE;
    }
    device = attr.device;
    int cur = -1;
    if (cudaGetDevice(&cur) != cudaSuccess || cur != device) {
      if (cudaSetDevice(device) != cudaSuccess) {
        cudaGetLastError();
        set_error("cudaSetDevice failed");
        return B200_ATTN_ERR_DEVICE;
      }
      prev = cur;
    }
    return B200_ATTN_OK;
  }
  ~DeviceScope() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// SMs of a device, queried once.
inline int sm_count(int device) {
  static std::once_flag once[kMaxDevices];
  static int sms[kMaxDevices];
  std::call_once(once[device], [device] {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n < 1) {
      cudaGetLastError();
      n = 148;
    }
    sms[device] = n;
  });
  return sms[device];
}

// Launch with programmatic stream serialization: the kernel's set-up overlaps
// the tail of the kernel before it; every kernel of these files waits for that
// kernel (griddepcontrol.wait) before it touches memory.
template <class... P, class... A>
int32_t launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
               A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, P(args)...);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) {
    set_error(cudaGetErrorString(e));
    return B200_ATTN_ERR_LAUNCH;
  }
  count_launch();
  return B200_ATTN_OK;
}

}  // namespace b200paged
