// Per-device state of the quantised linear layer: the tensor-map encoder, the error word of the bounded
// waits, the SM count and the kernels' shared-memory attributes. Made once per device, never changed.
#include <mutex>

#include "dense.hpp"

namespace imd {
namespace {

__device__ unsigned int g_error_word = 0;

constexpr int kMaxDevices = 64;
std::mutex g_lock;
DeviceInfo g_info[kMaxDevices];
bool g_ready[kMaxDevices];

bool make(int device, DeviceInfo* info) {
  void* fn = nullptr;
  void* word = nullptr;
  cudaDriverEntryPointQueryResult q;
  if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
      q != cudaDriverEntryPointSuccess || fn == nullptr || cudaGetSymbolAddress(&word, g_error_word) != cudaSuccess ||
      cudaDeviceGetAttribute(&info->sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
      !norm_setup() || !stream_setup() || !dense8_setup() || !dense4_setup())
    return false;
  info->encode_tiled = fn;
  info->error_word = static_cast<unsigned int*>(word);
  return true;
}

}  // namespace

const DeviceInfo* device_info() {
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= kMaxDevices) {
    cudaGetLastError();
    return nullptr;
  }
  std::lock_guard<std::mutex> hold(g_lock);
  if (!g_ready[device]) {
    if (!make(device, &g_info[device])) {
      cudaGetLastError();
      return nullptr;
    }
    g_ready[device] = true;
  }
  return &g_info[device];
}

}  // namespace imd

extern "C" imd_status_t imd_linear_device_error(unsigned int* word) {
  if (word == nullptr) return IMD_STATUS_INVALID_VALUE;
  const imd::DeviceInfo* dev = imd::device_info();
  unsigned int v = 0, zero = 0;
  if (dev == nullptr || cudaDeviceSynchronize() != cudaSuccess ||
      cudaMemcpy(&v, dev->error_word, sizeof v, cudaMemcpyDeviceToHost) != cudaSuccess ||
      cudaMemcpy(dev->error_word, &zero, sizeof zero, cudaMemcpyHostToDevice) != cudaSuccess) {
    cudaGetLastError();
    return IMD_STATUS_CUDA_ERROR;
  }
  *word = v;
  return IMD_STATUS_SUCCESS;
}
