// Conversions and vector access shared by the kernels of the quantised linear layer.
#pragma once
#include <cstdint>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "linear.hpp"

namespace imd {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements of T moved as one access (16 bytes or a single element).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T v[V];
};

// The value of a scale stored as `type`, element i.
__device__ __forceinline__ float load_scale(const void* p, int32_t type, int64_t i) {
  if (type == IMD_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == IMD_TYPE_F16) return to_float(static_cast<const __half*>(p)[i]);
  return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_out(void* out, int32_t type, int64_t i, float v) {
  if (type == IMD_TYPE_F32) static_cast<float*>(out)[i] = v;
  else if (type == IMD_TYPE_F16) static_cast<__half*>(out)[i] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
}

// The addresses [lo, hi) of a matrix: what a load may touch.
struct Span {
  uintptr_t lo, hi;
};
__device__ __forceinline__ Span span_of(const void* p, int64_t rows, int64_t stride_bytes, int64_t row_bytes) {
  const uintptr_t lo = reinterpret_cast<uintptr_t>(p);
  return {lo, lo + static_cast<uintptr_t>((rows - 1) * stride_bytes + row_bytes)};
}

// `BYTES` bytes at row + at, zeros from `end` (the row's length in bytes) on, for rows of any alignment. INSIDE: the
// piece lies inside the row with at least 3 bytes before and 4 behind it, and is read as the aligned words around it,
// shifted into place, without a branch (so that many such loads are in flight together). Otherwise the same where
// those words lie inside the matrix, and single bytes elsewhere.
template <int BYTES, bool INSIDE>
__device__ __forceinline__ void load_bytes(const uint8_t* row, int64_t at, int64_t end, const Span& span, uint32_t* v) {
  const uint8_t* p = row + at;
  const uintptr_t first = reinterpret_cast<uintptr_t>(p) & ~static_cast<uintptr_t>(3);
  if (INSIDE || (at + BYTES <= end && first >= span.lo && first + BYTES + 4 <= span.hi)) {
    const uint32_t shift = 8 * (reinterpret_cast<uintptr_t>(p) & 3);
    const uint32_t* q = reinterpret_cast<const uint32_t*>(first);
    uint32_t word[BYTES / 4 + 1];
#pragma unroll
    for (int i = 0; i <= BYTES / 4; ++i) word[i] = q[i];
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) v[i] = __funnelshift_r(word[i], word[i + 1], shift);
    return;
  }
#pragma unroll
  for (int i = 0; i < BYTES / 4; ++i) {
    uint32_t word = 0;
#pragma unroll
    for (int b = 0; b < 4; ++b)
      if (at + 4 * i + b < end) word |= static_cast<uint32_t>(p[4 * i + b]) << (8 * b);
    v[i] = word;
  }
}

// 128 bytes of each of ROWS rows of any alignment, by one warp, into shared memory in the layout of a TMA box with the
// 128-byte swizzle (row r of the box at r * 128, its 16-byte pieces exchanged by r mod 8). A lane loads two
// neighbouring aligned words of each row and shifts them into place; all loads are issued before the first store.
// Row i is box row r0 + i * step and starts at base + (row0 + r0 + i * step) * stride; bytes from `end` of a row on and
// rows from `rows` on are zero. Where a word might lie outside the matrix single bytes are loaded.
template <int ROWS>
__device__ __forceinline__ void bring_rows(const uint8_t* base, int64_t stride, int64_t rows, int64_t row0, int r0, int step,
                                           int box_rows, int64_t at, int64_t end, const Span& span, uint32_t dst) {
  const int lane = threadIdx.x & 31;
  const int64_t valid = end - at - 4 * lane;  // bytes of this lane's word inside the row
  const uint32_t keep = valid >= 4 ? ~0u : valid <= 0 ? 0u : (1u << (8 * valid)) - 1u;
  const int64_t first = min(row0 + r0, rows - 1), last = min(row0 + r0 + (ROWS - 1) * step, rows - 1);
  const uintptr_t from = reinterpret_cast<uintptr_t>(base + first * stride + at);
  uint32_t v[ROWS];
  if ((from & ~static_cast<uintptr_t>(3)) >= span.lo &&
      reinterpret_cast<uintptr_t>(base + last * stride + at) + 128 + 4 <= span.hi) {  // the same for the whole warp
    uint32_t low[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t row = min(row0 + r0 + i * step, rows - 1);
      const uint32_t* a = reinterpret_cast<const uint32_t*>(reinterpret_cast<uintptr_t>(base + row * stride + at) &
                                                            ~static_cast<uintptr_t>(3)) + lane;
      low[i] = a[0];
      v[i] = a[1];
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int64_t row = min(row0 + r0 + i * step, rows - 1);
      v[i] = __funnelshift_r(low[i], v[i], 8 * (reinterpret_cast<uintptr_t>(base + row * stride + at) & 3));
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < ROWS; ++i) {
      const int64_t row = min(row0 + r0 + i * step, rows - 1);
      uint32_t w = 0;
      for (int b = 0; b < 4; ++b)
        if (b < valid) w |= static_cast<uint32_t>(base[row * stride + at + 4 * lane + b]) << (8 * b);
#pragma unroll
      for (int j = 0; j < ROWS; ++j)
        if (j == i) v[j] = w;
    }
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = r0 + i * step;
    if (r < box_rows)
      asm volatile("st.shared.u32 [%0], %1;" ::"r"(dst + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + 4 * (lane & 3)),
                   "r"(row0 + r < rows ? v[i] & keep : 0u)
                   : "memory");
  }
}

// 4-bit weights as exact 16-bit floats: a nibble or'ed into the mantissa of 128 (bf16) or 1024 (f16).
template <typename X>
__host__ __device__ constexpr uint32_t nibble_magic();
template <>
__host__ __device__ constexpr uint32_t nibble_magic<__half>() { return 0x64006400u; }
template <>
__host__ __device__ constexpr uint32_t nibble_magic<__nv_bfloat16>() { return 0x43004300u; }

__device__ __forceinline__ uint32_t sub_pair(uint32_t a, uint32_t b, __half) {
  __half2 r = __hsub2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t sub_pair(uint32_t a, uint32_t b, __nv_bfloat16) {
  __nv_bfloat162 r = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&a), *reinterpret_cast<__nv_bfloat162*>(&b));
  return *reinterpret_cast<uint32_t*>(&r);
}
// The two constants of the unpacking, in registers: the compiler would materialise them again at each use.
template <typename X>
struct Nibbles {
  uint32_t mask, magic;
  __device__ __forceinline__ Nibbles() {
    asm volatile("mov.u32 %0, 0x000F000F;" : "=r"(mask));
    asm volatile("mov.u32 %0, %1;" : "=r"(magic) : "n"(nibble_magic<X>()));
  }
  // The pairs (w_i - z, w_i+4 - z), i = 0..3, of the eight nibbles of a word; zero = magic | z | z << 16.
  // (word & mask) | magic is one lop3 when written as one; from C++ the compiler makes two of it.
  __device__ __forceinline__ void pairs(uint32_t word, uint32_t zero, uint32_t* pair) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t v;
      asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(v) : "r"(word >> (4 * i)), "r"(mask), "r"(magic));
      pair[i] = sub_pair(v, zero, X());
    }
  }
};

}  // namespace imd
