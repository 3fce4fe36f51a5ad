// The tensor-core kernels' share of a device: what is looked up or set once per device.
#pragma once
#include <cuda.h>

#include "linear.hpp"

namespace imd {

struct DeviceInfo {
  void* encode_tiled = nullptr;  // cuTensorMapEncodeTiled
  unsigned int* error_word = nullptr;
  int sms = 0;
};
// Of the current device; made on first use, nullptr where that fails (asked again at the next call).
const DeviceInfo* device_info();

// Rows that TMA can bring: 16-byte units, not overlapping, few enough for 32-bit coordinates of whole tiles.
constexpr int64_t kMostRowsTma = INT64_C(1) << 30;
inline bool rows_for_tma(const void* p, int64_t rows, int64_t stride_bytes, int64_t row_bytes) {
  return rows <= kMostRowsTma && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         (rows == 1 || (stride_bytes % 16 == 0 && stride_bytes >= row_bytes));
}
// Tensor map of such rows as bytes, boxes of box_rows x 128 bytes with the 128-byte swizzle; what lies outside is zero.
bool encode_rows_128(const DeviceInfo& dev, CUtensorMap* map, const void* base, int64_t row_bytes, int64_t rows,
                     int64_t stride_bytes, int box_rows);

bool norm_setup();  // kernel attributes on the current device
// The same; whether these kernels take this call; the call.
bool dense8_setup();
bool dense8_takes(const LinearArgs& a);
imd_status_t dense8_launch(const LinearArgs& a, cudaStream_t stream);
bool stream_setup();
bool stream_takes(const LinearArgs& a);
imd_status_t stream_launch(const LinearArgs& a, cudaStream_t stream);
bool dense4_setup();
bool dense4_takes(const LinearArgs& a);
imd_status_t dense4_launch(const LinearArgs& a, cudaStream_t stream);

}  // namespace imd
