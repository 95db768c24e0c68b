// Errors and per-device state of the mixture-of-experts operators.
#include "operators.h"

#include <mutex>

namespace ponni_b200 {
namespace ops {
namespace {

thread_local std::string g_error;

constexpr int kMaxDevices = 64;
struct PerDevice {
  int* error = nullptr;
  int sms = 0;
};
PerDevice g_device[kMaxDevices];
std::mutex g_mutex;

}  // namespace

ponni_b200_status fail(ponni_b200_status s, const std::string& msg) {
  g_error = msg;
  return s;
}

ponni_b200_status fail_cuda(cudaError_t e, const char* what) {
  cudaGetLastError();  // reported here, not again by the caller's next look at the runtime's error
  return fail(PONNI_B200_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

ponni_b200_status launched(const char* what) {
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? PONNI_B200_OK : fail_cuda(e, what);
}

// A static device variable: the first call on a device allocates nothing.
static __device__ int g_error_word;

int* error_word(int device) {
  if (device < 0 || device >= kMaxDevices) return nullptr;
  std::lock_guard<std::mutex> lock(g_mutex);
  if (!g_device[device].error) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_error_word) != cudaSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    g_device[device].error = static_cast<int*>(p);
  }
  return g_device[device].error;
}

int num_sms(int device) {
  if (device < 0 || device >= kMaxDevices) return 148;
  std::lock_guard<std::mutex> lock(g_mutex);
  if (!g_device[device].sms) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    g_device[device].sms = n;
  }
  return g_device[device].sms;
}

int num_devices() {
  static const int n = [] {
    int c = 0;
    if (cudaGetDeviceCount(&c) != cudaSuccess) {
      cudaGetLastError();
      c = 0;
    }
    return c;
  }();
  return n;
}

cudaError_t allow_smem(const void* kernel, int bytes, int device, std::atomic<uint64_t>& done) {
  const uint64_t bit = device >= 0 && device < kMaxDevices ? 1ull << device : 0;
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

}  // namespace ops
}  // namespace ponni_b200

using namespace ponni_b200;

extern "C" {

const char* ponni_b200_operator_error(void) { return ops::g_error.c_str(); }

ponni_b200_status ponni_b200_operator_check(int device, void* stream) {
  return ops::entry(device, [&]() -> ponni_b200_status {
    int* word = ops::error_word(device);
    if (!word) return ops::fail(PONNI_B200_ERR_CUDA, "no operator error word on this device");
    int seen = 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = cudaMemcpyAsync(&seen, word, sizeof seen, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return ops::fail_cuda(e, "operator check");
    if (!seen) return PONNI_B200_OK;
    const int zero = 0;
    e = cudaMemcpyAsync(word, &zero, sizeof zero, cudaMemcpyHostToDevice, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    if (e != cudaSuccess) return ops::fail_cuda(e, "operator check");
    if (seen & 1)
      return ops::fail(PONNI_B200_ERR_DEVICE, "expert_product: a bounded wait gave up; the outputs are not valid");
    return ops::fail(PONNI_B200_ERR_INVALID_ARGUMENT,
                     "group offsets are not ascending from 0 to at most the number of rows");
  });
}

}  // extern "C"
