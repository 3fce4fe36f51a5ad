// The tensor-core kernels' share of a device: what is looked up or set once per device.
#pragma once
#include "linear.hpp"

namespace imd {

struct DeviceInfo {
  void* encode_tiled = nullptr;  // cuTensorMapEncodeTiled
  unsigned int* error_word = nullptr;
  int sms = 0;
};
// Of the current device; made on first use, nullptr where that fails (asked again at the next call).
const DeviceInfo* device_info();

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
