// Shared by the mixture-of-experts operators (route.cu, columns.cu,
// expert_product.cu, gradient_clip.cu): argument errors, the device-side error
// word and launch helpers.
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <string>

#include "model.h"

namespace ponni_b200 {
namespace ops {

constexpr int kMaxExperts = 1024;
constexpr int kMaxTopK = 8;

// Records `msg` as the calling thread's operator error and returns `s`.
ponni_b200_status fail(ponni_b200_status s, const std::string& msg);
ponni_b200_status fail_cuda(cudaError_t e, const char* what);
// Status of the launches just made.
ponni_b200_status launched(const char* what);

// Device address of the current device's operator error word (zero: no error), a
// static device variable.
int* error_word(int device);

int num_sms(int device);
int num_devices();  // asked once; 0 without a driver

// Lets `kernel` use up to `bytes` of dynamic shared memory on `device`; `done` is
// the kernel's own mask of the devices on which this has been said.
cudaError_t allow_smem(const void* kernel, int bytes, int device, std::atomic<uint64_t>& done);

// Runs `body` (returning a status) with `device` current and no exception
// leaving the C entry.
template <class F>
ponni_b200_status entry(int device, F&& body) noexcept {
  try {
    const int n = num_devices();
    if (n == 0) return fail(PONNI_B200_ERR_CUDA, "no CUDA device");
    if (device < 0 || device >= n)
      return fail(PONNI_B200_ERR_INVALID_ARGUMENT, "device " + std::to_string(device) + " does not exist");
    DeviceGuard guard(device);
    return body();
  } catch (const std::exception& e) {
    try {
      return fail(PONNI_B200_ERR_CUDA, e.what());
    } catch (...) {
      return PONNI_B200_ERR_CUDA;
    }
  } catch (...) {
    return PONNI_B200_ERR_CUDA;
  }
}

inline bool is_real_type(int dtype) {
  return dtype == PONNI_B200_F32 || dtype == PONNI_B200_F16 || dtype == PONNI_B200_BF16;
}
// Every pointer a multiple of `bytes` (a misaligned one would fault in the kernels).
template <class... P>
bool aligned_to(int bytes, P... p) {
  uintptr_t all = 0;
  ((all |= reinterpret_cast<uintptr_t>(p)), ...);
  return all % bytes == 0;
}

inline int element_bytes(int dtype) { return dtype == PONNI_B200_F64 ? 8 : dtype == PONNI_B200_F32 ? 4 : 2; }

// Launch with programmatic stream serialisation: the kernel may start while its
// predecessor on the stream drains; it calls griddepcontrol.wait before it
// reads what that one wrote.
template <class... P, class... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

#ifdef __CUDACC__
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;\n" ::: "memory"); }
__device__ __forceinline__ void let_successor_start() { asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory"); }
#endif

}  // namespace ops
}  // namespace ponni_b200
