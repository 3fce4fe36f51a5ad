// Which kernel takes a product: the rules on sizes, types and alignment, apart from the kernels so that a host
// program can ask them (tests/linear_choice_shim.cpp).
#pragma once
#include <cstdint>

#include "linear.hpp"

namespace imd {

// Rows that TMA can bring: 16-byte units, not overlapping. Its coordinates are 32-bit: few enough rows for whole tiles, and
// rows short enough for whole blocks of k (which start at most 256 bytes behind a row's end) counted in bytes.
constexpr int64_t kMostRowsTma = INT64_C(1) << 30, kMostBytesTma = (INT64_C(1) << 31) - 512;
inline bool rows_for_tma(const void* p, int64_t rows, int64_t stride_bytes, int64_t row_bytes) {
  return rows <= kMostRowsTma && row_bytes <= kMostBytesTma && reinterpret_cast<uintptr_t>(p) % 16 == 0 &&
         (rows == 1 || (stride_bytes % 16 == 0 && stride_bytes >= row_bytes));
}
inline bool x4_for_tma(const LinearArgs& a) { return rows_for_tma(a.x, a.rows, 2 * a.x_stride, 2 * a.k); }
inline bool w4_for_tma(const LinearArgs& a) { return rows_for_tma(a.w, a.n, a.w_stride, (a.k + 1) / 2); }
inline bool both8_for_tma(const LinearArgs& a) {
  return rows_for_tma(a.x, a.rows, a.x_stride, a.k) && rows_for_tma(a.w, a.n, a.w_stride, a.k);
}

// 8 bits: the tensor-core kernels take rows of any alignment; with little work those are quicker in the small kernel (int8,
// 1000 x 300 x 777: 12 against 28 us; 100 x 5000 x 4001: 74 against 54 us, 2000 x 5000 x 4001: 958 against 299 us).
constexpr int64_t kLeastWork8 = INT64_C(1) << 30, kMostRowsAny8 = 65535 * 256;  // (a grid's third extent)
inline bool dense8_takes(const LinearArgs& a) {
  if (a.kind == WeightKind::kU4 || a.k == 0) return false;
  return (a.rows > 16 && a.rows <= kMostRowsAny8 && a.n <= kMostRowsTma && a.rows * a.n >= kLeastWork8 / a.k) ||
         both8_for_tma(a);
}

// CTAs that share a tile of a tensor-core kernel by splitting K: a cluster of 1, 2, 4 or 8, as many as fit the GPU at once
// with at least two steps of K each. A cluster lies in one part of the GPU, so 8 x 15 or 4 x 33 CTAs fit 148 SMs, not 8 x 18
// or 4 x 37, and what does not fit costs a second round (4 bits, 40 x 2048 x 2048: clusters of 8 18.8, of 4 11.4 us; 40 x 4736 x
// 8192: of 4 46.8, of 2 40.0; 8 bits 1 x 4736 x 8192: of 8 17.2, of 4 12.1). clusters[i]: how many of 2^i CTAs fit with one
// CTA on an SM.
inline int split_of(int64_t tiles, int64_t steps, const int* clusters, int ctas_per_sm) {
  int i = 0;
  while (i < 3 && tiles <= static_cast<int64_t>(clusters[i + 1]) * ctas_per_sm && steps >= INT64_C(4) << i) ++i;
  return 1 << i;
}

// 4 bits, streamed: up to 16 rows of x in one pass over the weights. 17 to 32 take two passes where the tensor-core kernel,
// whose time hardly depends on the rows, is slower: with groups of 32, whose sums bound it, and where its tiles leave much of
// their last round idle; little is enough from kStreamTallN rows of w on, where a streamed tile has 32 of them. (And with rows of x
// that only loads bring there, such as a repeated one.)
// (us, two passes / tensor cores, zero points: 24 x 8192 x 28672 g32 163 / 219; idle more than a third, 24 x 2048 x 2048 g128
// 9.1 / 10.9, 24 x 4736 x 2816 g64 14 / 20; idle 14 %, 17 x 4096 x 4096 g128 16.8 / 16.1, 32 rows 20.8 / 16.4, 24 x 8192 x 8192 57
// / 40, g64 50 / 44; many rows of w, idle a quarter, 24 x 28672 x 8192 g128 123 / 139; not idle, 24 x 18944 x 3584 g128 42 / 35.)
// Over 18 shapes from 512 x 1024 to 128256 x 4096, 17 to 32 rows, all groups, the choice is 1.1 % slower than the better of the two
// on average, two passes throughout 4.7 %, the tensor cores throughout 21 %; most at 32 x 512 x 16384 g128 (33 / 24).
// The kernel walks k in 32 bits, up to eight pieces of 256 and a step past a row's end.
constexpr int64_t kStreamPassRows = 16, kStreamMostRows = 32, kStreamMostK = (INT64_C(1) << 31) - 4096;
constexpr int64_t kStreamTallN = 64 * 148;  // two tiles of 32 rows of w for each of 148 SMs
inline bool two_passes(const LinearArgs& a, const int* clusters) {
  if (a.group == 32 || !x4_for_tma(a)) return true;
  const int64_t tiles = (a.n + 127) / 128, unit = a.group > 64 ? a.group : 64;
  const int64_t ctas = tiles * split_of(tiles, (a.k + unit - 1) / unit, clusters, 1);
  const int64_t slots = (ctas + clusters[0] - 1) / clusters[0] * clusters[0];
  return 100 * slots >= ctas * (a.n >= kStreamTallN ? 102 : a.group == 64 ? 136 : 150);
}
inline bool stream_takes(const LinearArgs& a, const int* clusters) {
  return a.kind == WeightKind::kU4 && a.k > 0 && a.k <= kStreamMostK &&
         (a.rows <= kStreamPassRows || (a.rows <= kStreamMostRows && two_passes(a, clusters))) &&
         reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.rows == 1 || a.x_stride % 8 == 0) && w4_for_tma(a);
}

// 4 bits on the tensor cores. Rows of any alignment with little work are quicker in the small kernel (1802 x 83 x 150 9.6
// against 20 us, 50 x 1000 x 1001 7.9 against 11.9), with more here (100 x 4000 x 1001 26 against 18 us, 1000 x 4000 x 1001 218
// against 99).
constexpr int64_t kLeastWork4 = INT64_C(1) << 28;
inline bool dense4_takes(const LinearArgs& a) {
  return a.kind == WeightKind::kU4 && a.k > 0 && a.rows > 16 && a.rows <= kMostRowsTma && a.n <= kMostRowsTma &&
         (x4_for_tma(a) || a.rows * a.n >= kLeastWork4 / a.k);
}

}  // namespace imd
