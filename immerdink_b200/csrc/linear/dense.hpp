// The tensor-core kernels' share of a device: what is looked up or set once per device.
#pragma once
#include <cuda.h>

#include "choice.hpp"

namespace imd {

struct DeviceInfo {
  void* encode_tiled = nullptr;  // cuTensorMapEncodeTiled
  unsigned int* error_word = nullptr;
  int sms = 0;
  int clusters[4] = {};          // of 1, 2, 4 and 8 CTAs that fit at once, one CTA on an SM
};
// Of the current device; made on first use, nullptr where that fails (asked again at the next call).
const DeviceInfo* device_info();

// Tensor map of such rows as bytes, boxes of box_rows x 128 bytes with the 128-byte swizzle; what lies outside is zero.
bool encode_rows_128(const DeviceInfo& dev, CUtensorMap* map, const void* base, int64_t row_bytes, int64_t rows,
                     int64_t stride_bytes, int box_rows);

bool norm_setup();  // kernel attributes on the current device
// The same, and a call that the rules of choice.hpp give to these kernels.
bool dense8_setup();
imd_status_t dense8_launch(const LinearArgs& a, cudaStream_t stream);
bool stream_setup();
imd_status_t stream_launch(const LinearArgs& a, cudaStream_t stream);
bool dense4_setup();
bool dense4_clusters(int sms, int* clusters);  // DeviceInfo's
imd_status_t dense4_launch(const LinearArgs& a, cudaStream_t stream);

}  // namespace imd
