// Host-side argument checks shared by the library's launchers.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>

namespace geoattn {

constexpr size_t kAlign = 256;
inline size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

// Every data pointer handed to a kernel must be memory of the current device (or managed memory): the kernels run
// on the current device, which would dereference a host pointer or another device's memory. Checked on the host
// before any launch.
inline bool dev_ptr(const void* p) {
  if (!p) return false;
  cudaPointerAttributes a;
  if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
    cudaGetLastError();  // clear the sticky-free error of an unregistered host pointer
    return false;
  }
  if (a.type == cudaMemoryTypeManaged) return true;
  int cur = -1;
  return a.type == cudaMemoryTypeDevice && cudaGetDevice(&cur) == cudaSuccess && a.device == cur;
}

}  // namespace geoattn
