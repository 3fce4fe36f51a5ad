// Per-device state of the quantised linear layer: the tensor-map encoder, the error word of the bounded
// waits, the SM count and the kernels' shared-memory attributes. Made once per device, never changed.
#include <mutex>

#include "cuda/sm100.cuh"
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
      !norm_setup() || !stream_setup() || !dense8_setup() || !dense4_setup() ||
      !dense4_clusters(info->sms, info->clusters))
    return false;
  info->encode_tiled = fn;
  info->error_word = static_cast<unsigned int*>(word);
  return true;
}

}  // namespace

bool encode_rows_128(const DeviceInfo& dev, CUtensorMap* map, const void* base, int64_t row_bytes, int64_t rows,
                     int64_t stride_bytes, int box_rows) {
  const int64_t pitch = rows > 1 ? stride_bytes : (row_bytes + 15) / 16 * 16;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows), 1};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(pitch), static_cast<cuuint64_t>(pitch) * rows};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t elem[3] = {1, 1, 1};
  const EncodeTiled fn = reinterpret_cast<EncodeTiled>(dev.encode_tiled);
  // rows that straddle the 128-byte lines cost more with larger fetches (e4m3 1999 x 5003 x 4176: 63 against 58 us)
  const CUtensorMapL2promotion fetch = pitch % 128 == 0 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_NONE;
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, fetch,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

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
