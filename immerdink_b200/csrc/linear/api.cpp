// C ABI of libimmerdink_linear.so: argument checks in the order the header documents; a failing call
// touches nothing and no exception leaves a function.
#include <cmath>
#include <cstdint>

#include "dense.hpp"
#include "linear.hpp"

namespace {

using i128 = __int128;

constexpr int64_t kMaxExtent = INT64_C(1) << 31;  // rows, n, k, dim stay below this
constexpr int64_t kMaxI8Depth = 131071;           // k * 128^2 < 2^31
constexpr double kMostEps = 0x1p127;              // mean + eps stays in the range of 32 bits

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
bool is_float(int32_t t) { return t == IMD_TYPE_F32 || t == IMD_TYPE_BF16 || t == IMD_TYPE_F16; }
bool is_8bit(int32_t t) { return t == IMD_TYPE_I8 || t == IMD_TYPE_E4M3; }
int size_of(int32_t t) { return t == IMD_TYPE_F32 ? 4 : is_float(t) ? 2 : 1; }

// The bytes of a row-major matrix: rows of `width`, `pitch` apart (0: one row), inside [lo, hi); empty for a null pointer or
// an empty matrix.
struct Bytes {
  i128 lo = 0, hi = 0, width = 0, pitch = 0;
};
Bytes bytes_of(const void* p, int64_t rows, int64_t cols, int64_t stride, int size) {
  Bytes r;
  if (p == nullptr || rows == 0 || cols == 0) return r;
  r.width = static_cast<i128>(cols) * size;
  r.pitch = rows == 1 ? 0 : static_cast<i128>(stride) * size;
  r.lo = static_cast<i128>(reinterpret_cast<uintptr_t>(p));
  r.hi = r.lo + (rows - 1) * r.pitch + r.width;
  return r;
}
// Whether two matrices may share a byte. Rows at the same distance, as columns of one buffer have, interleave without doing
// so where one's rows begin behind the other's and end before its next; other distances are not looked into.
bool overlap(const Bytes& x, const Bytes& y) {
  if (x.lo >= x.hi || y.lo >= y.hi || x.lo >= y.hi || y.lo >= x.hi) return false;
  const i128 pitch = x.pitch != 0 ? x.pitch : y.pitch;
  if (pitch == 0 || (y.pitch != 0 && y.pitch != pitch)) return true;
  i128 behind = (y.lo - x.lo) % pitch;
  if (behind < 0) behind += pitch;
  return behind < x.width || behind + y.width > pitch;
}
bool extent_ok(int64_t e) { return e >= 0 && e < kMaxExtent; }
bool in_stride_ok(int64_t s) { return s >= 0 && s < (INT64_C(1) << 40); }
bool out_stride_ok(int64_t s, int64_t rows, int64_t cols) {
  return in_stride_ok(s) && (rows <= 1 || s >= cols);
}

}  // namespace

extern "C" {

imd_status_t imd_norm_quantize(int64_t rows, int64_t dim, int32_t x_type, const void* x,
                               int64_t x_stride, const void* residual, int64_t residual_stride,
                               int32_t weight_type, const void* weight, double eps,
                               void* residual_out, int64_t residual_out_stride, int32_t q_type,
                               void* q, int64_t q_stride, float* scale, cudaStream_t stream) {
  if (!extent_ok(rows) || !extent_ok(dim) || dim == 0 || !is_float(x_type) || !is_8bit(q_type) ||
      !is_float(weight_type) || !(eps >= 0.0 && eps <= kMostEps))
    return IMD_STATUS_INVALID_VALUE;
  if (weight_type != x_type && weight_type != IMD_TYPE_F32) return IMD_STATUS_NOT_SUPPORTED;
  if (rows == 0) return IMD_STATUS_SUCCESS;
  if (rows == 1) x_stride = residual_stride = residual_out_stride = q_stride = dim;  // a single row has no distance
  if (x == nullptr || weight == nullptr || q == nullptr || scale == nullptr ||
      (residual_out != nullptr && residual == nullptr) || !in_stride_ok(x_stride) ||
      (residual != nullptr && !in_stride_ok(residual_stride)) ||
      (residual_out != nullptr && !out_stride_ok(residual_out_stride, rows, dim)) ||
      !out_stride_ok(q_stride, rows, dim))
    return IMD_STATUS_INVALID_VALUE;
  const int sx = size_of(x_type), sw = size_of(weight_type);
  const Bytes ix = bytes_of(x, rows, dim, x_stride, sx),
                 ir = bytes_of(residual, rows, dim, residual_stride, sx),
                 iw = bytes_of(weight, 1, dim, 0, sw),
                 ih = bytes_of(residual_out, rows, dim, residual_out_stride, sx),
                 iq = bytes_of(q, rows, dim, q_stride, 1), is = bytes_of(scale, 1, rows, 0, 4);
  // in place only when every element is written by the thread that read it
  const bool same_x = residual_out == x && residual_out_stride == x_stride,
             same_r = residual_out == residual && residual_out_stride == residual_stride;
  if ((!same_x && overlap(ih, ix)) || (!same_r && overlap(ih, ir)) || overlap(ih, iw) ||
      overlap(iq, ix) || overlap(iq, ir) || overlap(iq, iw) || overlap(iq, ih) || overlap(is, ix) ||
      overlap(is, ir) || overlap(is, iw) || overlap(is, ih) || overlap(is, iq))
    return IMD_STATUS_ALIASING;
  if (!aligned(x, sx) || !aligned(residual, sx) || !aligned(weight, sw) ||
      !aligned(residual_out, sx) || !aligned(scale, 4))
    return IMD_STATUS_MISALIGNED;
  imd::NormArgs a{};
  a.rows = rows, a.dim = dim;
  a.x = x, a.residual = residual, a.weight = weight, a.residual_out = residual_out, a.q = q;
  a.scale = scale;
  a.x_stride = x_stride, a.residual_stride = residual_stride;
  a.residual_out_stride = residual_out_stride, a.q_stride = q_stride;
  a.eps = static_cast<float>(eps), a.eps_root = static_cast<float>(std::sqrt(eps));
  a.x_type = x_type, a.weight_type = weight_type, a.q_type = q_type;
  return imd::norm_quantize_launch(a, stream);
}

imd_status_t imd_scaled_linear(int64_t rows, int64_t n, int64_t k, int32_t type, const void* x,
                               int64_t x_stride, const void* w, int64_t w_stride,
                               const float* x_scale, const float* w_scale, int32_t out_type,
                               void* out, int64_t out_stride, cudaStream_t stream) {
  if (!extent_ok(rows) || !extent_ok(n) || !extent_ok(k) || !is_8bit(type) || !is_float(out_type))
    return IMD_STATUS_INVALID_VALUE;
  if (type == IMD_TYPE_I8 && k > kMaxI8Depth) return IMD_STATUS_NOT_SUPPORTED;
  if (rows == 0 || n == 0) return IMD_STATUS_SUCCESS;
  if (rows == 1) x_stride = k, out_stride = n;
  if (n == 1) w_stride = k;
  if ((k > 0 && (x == nullptr || w == nullptr)) || x_scale == nullptr || w_scale == nullptr ||
      out == nullptr || !in_stride_ok(x_stride) || !in_stride_ok(w_stride) ||
      !out_stride_ok(out_stride, rows, n))
    return IMD_STATUS_INVALID_VALUE;
  const int so = size_of(out_type);
  const Bytes io = bytes_of(out, rows, n, out_stride, so);
  if (overlap(io, bytes_of(x, rows, k, x_stride, 1)) || overlap(io, bytes_of(w, n, k, w_stride, 1)) ||
      overlap(io, bytes_of(x_scale, 1, rows, 0, 4)) || overlap(io, bytes_of(w_scale, 1, n, 0, 4)))
    return IMD_STATUS_ALIASING;
  if (!aligned(x_scale, 4) || !aligned(w_scale, 4) || !aligned(out, so)) return IMD_STATUS_MISALIGNED;
  imd::LinearArgs a{};
  a.rows = rows, a.n = n, a.k = k;
  a.x = x, a.w = w, a.x_stride = x_stride, a.w_stride = w_stride;
  a.x_scale = x_scale, a.w_scale8 = w_scale;
  a.out = out, a.out_stride = out_stride;
  a.kind = type == IMD_TYPE_I8 ? imd::WeightKind::kI8 : imd::WeightKind::kE4M3;
  a.x_type = type, a.out_type = out_type;
  return imd::dense8_takes(a) ? imd::dense8_launch(a, stream) : imd::linear_small_launch(a, stream);
}

imd_status_t imd_linear_w4(int64_t rows, int64_t n, int64_t k, int32_t group, int32_t x_type,
                           const void* x, int64_t x_stride, const void* w, int64_t w_stride,
                           int32_t scale_type, const void* w_scale, int64_t scale_stride,
                           const void* zeros, int64_t zeros_stride, int32_t out_type, void* out,
                           int64_t out_stride, cudaStream_t stream) {
  if (!extent_ok(rows) || !extent_ok(n) || !extent_ok(k) || !is_float(x_type) ||
      !is_float(scale_type) || !is_float(out_type) || group <= 0)
    return IMD_STATUS_INVALID_VALUE;
  if ((group != 32 && group != 64 && group != 128) || x_type == IMD_TYPE_F32 ||
      (out_type != IMD_TYPE_F32 && out_type != x_type))
    return IMD_STATUS_NOT_SUPPORTED;
  if (rows == 0 || n == 0) return IMD_STATUS_SUCCESS;
  const int64_t groups = (k + group - 1) / group, half = (k + 1) / 2;
  if (rows == 1) x_stride = k, out_stride = n;
  if (n == 1) w_stride = half, scale_stride = zeros_stride = groups;
  if ((k > 0 && (x == nullptr || w == nullptr || w_scale == nullptr)) || out == nullptr ||
      !in_stride_ok(x_stride) || !in_stride_ok(w_stride) || !in_stride_ok(scale_stride) ||
      (zeros != nullptr && !in_stride_ok(zeros_stride)) || !out_stride_ok(out_stride, rows, n))
    return IMD_STATUS_INVALID_VALUE;
  const int sx = size_of(x_type), ss = size_of(scale_type), so = size_of(out_type);
  const Bytes io = bytes_of(out, rows, n, out_stride, so);
  if (overlap(io, bytes_of(x, rows, k, x_stride, sx)) || overlap(io, bytes_of(w, n, half, w_stride, 1)) ||
      overlap(io, bytes_of(w_scale, n, groups, scale_stride, ss)) ||
      overlap(io, bytes_of(zeros, n, groups, zeros_stride, 1)))
    return IMD_STATUS_ALIASING;
  if (!aligned(x, sx) || !aligned(w_scale, ss) || !aligned(out, so)) return IMD_STATUS_MISALIGNED;
  imd::LinearArgs a{};
  a.rows = rows, a.n = n, a.k = k;
  a.x = x, a.w = w, a.x_stride = x_stride, a.w_stride = w_stride;
  a.scale4 = w_scale, a.scale_stride = scale_stride;
  a.zeros = static_cast<const uint8_t*>(zeros), a.zeros_stride = zeros_stride;
  a.out = out, a.out_stride = out_stride;
  a.kind = imd::WeightKind::kU4;
  a.x_type = x_type, a.scale_type = scale_type, a.out_type = out_type, a.group = group;
  const imd::DeviceInfo* dev = imd::device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  if (imd::stream_takes(a, dev->clusters)) return imd::stream_launch(a, stream);
  return imd::dense4_takes(a) ? imd::dense4_launch(a, stream) : imd::linear_small_launch(a, stream);
}

}  // extern "C"
