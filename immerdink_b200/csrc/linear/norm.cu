// RMS norm with the residual's addition and an 8-bit output with one scale per row.
//
//   h = x + r;  y_j = h_j * rsqrt(mean h^2 + eps) * w_j;  a = max_j |y_j|;  scale = a / Q;
//   q_j = round(y_j * (Q / a))                                       Q = 127 (int8), 448 (e4m3)
//
// The row's factor r = rsqrt(..) cancels in y_j / a. So it is split into a power of two p and m in [1, 2): the codes follow from
// g_j = h_j p w_j, whatever r was rounded to, and the scale is max |g_j| m / Q. Q / max |g| is held in two parts, so that g_j
// times it is rounded once: a value in the middle of two codes goes to the even one where h_j w_j is exact in 32 bits (with
// one part and with r in the products such values went to either side).
//
// Bound by HBM with a residual that is written back, 2 + 2 + 2 + 1 bytes per element of 16 bits (8191 x 8192: 79 us, 6.0
// TB/s, 0.91 of the measured copy rate; f32 139 us, 0.95). Without a residual the bytes are 3 and 5, and instructions and the
// two reductions' barriers bound it: 61 us (int8 codes 63, f32 78), 0.67 instructions a cycle and scheduler, 0.5 (f32 0.65) of the copy rate.
// A row is read once: its values stay in registers (`E` vectors per thread) through both row
// reductions, the sum of squares and the largest |y|. Short rows take one warp each, longer rows
// one CTA; rows beyond the register capacity are read three times (twice from L2).
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "dense.hpp"
#include "cuda/sm100.cuh"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kWarpRows = 4;     // rows (= warps) of a CTA in the warp-per-row form
constexpr int kMaxSlots = 8;     // rows in flight per CTA in the ring form
constexpr int kRingBytes = 200 * 1024;  // of one SM, shared by its CTAs
constexpr float kTiny = 0x1p-90f, kHuge = 0x1p+120f;

// Row reductions. WARP: the row belongs to one warp. Otherwise to the CTA: each warp leaves its
// partial in shared memory, one barrier, and every warp folds the partials in the same order.
// Consecutive reductions of a row use different slots, so one barrier each is enough.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* slot) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  if (WARP) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  v = lane < warps ? slot[lane] : 0.0f;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}
// Largest magnitude as a bit pattern: |y| orders like its bits, and a NaN is above an infinity.
template <bool WARP>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* slot) {
  v = __reduce_max_sync(~0u, v);
  if (WARP) return v;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  if (lane == 0) slot[warp] = v;
  __syncthreads();
  return __reduce_max_sync(~0u, lane < warps ? slot[lane] : 0u);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// 16 bytes of a row as four words, or one element (V = 1); their values; and the reverse.
template <typename T, int V>
struct Piece {
  static constexpr int kWords = V == 1 ? 1 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0;
  }
  __device__ __forceinline__ void load(const void* p, int64_t i) {
    const T* at = static_cast<const T*>(p) + i;
    if constexpr (V > 1) {
      const uint4 t = *reinterpret_cast<const uint4*>(at);
      w[0] = t.x, w[1] = t.y, w[2] = t.z, w[3] = t.w;
    } else if constexpr (sizeof(T) == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(at);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(at);
    }
  }
  // The first n elements (at most V), one by one; zeros behind them.
  __device__ __forceinline__ void load_part(const void* p, int64_t i, int n) {
    clear();
    const T* at = static_cast<const T*>(p) + i;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      if (v >= n) continue;
      if constexpr (sizeof(T) == 4) w[v] = reinterpret_cast<const uint32_t*>(at)[v];
      else w[v / 2] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[v]) << (16 * (v & 1));
    }
  }
  __device__ __forceinline__ float value(int v) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[v]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      return __uint_as_float(v % 2 != 0 ? w[v / 2] & 0xFFFF0000u : w[v / 2] << 16);
    } else {
      const __half2 h = *reinterpret_cast<const __half2*>(&w[v / 2]);
      return v % 2 != 0 ? __high2float(h) : __low2float(h);
    }
  }
  __device__ __forceinline__ static void store(void* p, int64_t i, const float* f) {
    T* at = static_cast<T*>(p) + i;
    if constexpr (V == 1) {
      *at = from_float<T>(f[0]);
    } else {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (sizeof(T) == 4) {
          o[j] = __float_as_uint(f[j]);
        } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
          o[j] = *reinterpret_cast<const uint32_t*>(&b);
        } else {
          const __half2 b = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
          o[j] = *reinterpret_cast<const uint32_t*>(&b);
        }
      }
      *reinterpret_cast<uint4*>(at) = make_uint4(o[0], o[1], o[2], o[3]);
    }
  }
};

// V codes of the scaled values y as bytes of words. int8: adding 1.5 * 2^23 rounds to the nearest even integer and
// leaves it, in two's complement, in the low bits; `keep` clears the codes of a row that has no finite scale.
template <int V>
__device__ __forceinline__ void codes(const float* y, bool e4m3, uint32_t keep, uint32_t* o) {
  if constexpr (V == 1) {
    o[0] = e4m3 ? static_cast<uint32_t>(__nv_cvt_float_to_fp8(y[0], __NV_SATFINITE, __NV_E4M3))
                : __float_as_uint(y[0] + 12582912.0f) & keep;
  } else {
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float* f = y + 4 * j;
      if (e4m3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE, __NV_E4M3);
        o[j] = lo | (hi << 16);
      } else {
        uint32_t b[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) b[c] = __float_as_uint(f[c] + 12582912.0f);
        o[j] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410) & keep;
      }
    }
  }
}
template <int V>
__device__ __forceinline__ void store_codes(void* p, int64_t i, const float* y, bool e4m3, uint32_t keep) {
  uint8_t* at = static_cast<uint8_t*>(p) + i;
  uint32_t o[V < 4 ? 1 : V / 4];
  codes<V>(y, e4m3, keep, o);
  if constexpr (V == 8) *reinterpret_cast<uint2*>(at) = make_uint2(o[0], o[1]);
  else if constexpr (V == 4) *reinterpret_cast<uint32_t*>(at) = o[0];
  else *at = static_cast<uint8_t>(o[0]);
}

// `bytes` bytes of words to an address of any alignment that is the same for the whole warp modulo 4: as many
// aligned words as there are, halves and bytes around them.
template <int WORDS>
__device__ __forceinline__ void store_bytes(uint8_t* at, const uint32_t* o, int bytes) {
  if (bytes < 4 * WORDS) {
#pragma unroll
    for (int i = 0; i < 4 * WORDS; ++i)
      if (i < bytes) at[i] = static_cast<uint8_t>(o[i / 4] >> (8 * (i & 3)));
    return;
  }
  const int head = static_cast<int>(-reinterpret_cast<uintptr_t>(at) & 3);  // bytes before the first aligned word
  if (head == 0) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) reinterpret_cast<uint32_t*>(at)[i] = o[i];
    return;
  }
  if (head & 1) *at = static_cast<uint8_t>(o[0]);
  if (head & 2) *reinterpret_cast<uint16_t*>(at + (head & 1)) = static_cast<uint16_t>(o[0] >> (8 * (head & 1)));
#pragma unroll
  for (int i = 0; i + 1 < WORDS; ++i) *reinterpret_cast<uint32_t*>(at + head + 4 * i) = __funnelshift_r(o[i], o[i + 1], 8 * head);
  const uint32_t tail = o[WORDS - 1] >> (8 * head);  // 4 - head bytes
  uint8_t* end = at + 4 * WORDS - (4 - head);
  if (head == 3) {
    *end = static_cast<uint8_t>(tail);
  } else {
    *reinterpret_cast<uint16_t*>(end) = static_cast<uint16_t>(tail);
    if (head == 1) end[2] = static_cast<uint8_t>(tail >> 16);
  }
}
template <int V>
__device__ __forceinline__ void store_codes_any(uint8_t* at, const float* y, int n, bool e4m3, uint32_t keep) {
  uint32_t o[V / 4];
  codes<V>(y, e4m3, keep, o);
  if (n > 0) store_bytes<V / 4>(at, o, n);
}
template <typename T, int V>
__device__ __forceinline__ void store_any(T* at, const float* f, int n) {
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if constexpr (sizeof(T) == 4) {
      o[j] = __float_as_uint(f[j]);
    } else {
      Pack<T, 2> h{{from_float<T>(f[2 * j]), from_float<T>(f[2 * j + 1])}};
      o[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  if (n > 0) store_bytes<4>(reinterpret_cast<uint8_t*>(at), o, n < V ? n * static_cast<int>(sizeof(T)) : 16);
}

// r as p * m, p a power of two and m in [1, 2). An r below the normal range, an infinity and a NaN are p.
struct Factor {
  float p, m;
};
__device__ __forceinline__ Factor split(float r) {
  const uint32_t bits = __float_as_uint(r), e = bits & 0x7F800000u;
  if (e == 0 || e == 0x7F800000u) return {r, 1.0f};
  return {__uint_as_float(e), __uint_as_float((bits & 0x007FFFFFu) | 0x3F800000u)};
}

// What turns a row's g into codes: q = round(g * pre * (inv + low)). `top`: the bits of the largest |g|; most = max |g| m,
// Q times the scale.
struct RowScale {
  float pre, inv, low, most;
  uint32_t keep;  // all ones, or zero for a row without a finite scale
};
__device__ __forceinline__ RowScale row_scale(uint32_t top, float m, bool e4m3) {
  const float q_max = e4m3 ? 448.0f : 127.0f;
  RowScale s{1.0f, 0.0f, 0.0f, __uint_as_float(top) * m, ~0u};
  if (!(s.most < __uint_as_float(0x7F800000u))) {
    s.inv = s.most = __uint_as_float(0x7FC00000u);  // a NaN or an infinity in the row
    s.keep = 0;
  } else if (top != 0) {
    float a = __uint_as_float(top), inverse;
    if (a < 0x1p-100f) s.pre = 0x1p+100f, a *= 0x1p+100f;  // Q / a would leave the range
    asm("rcp.approx.f32 %0, %1;" : "=f"(inverse) : "f"(a));  // within an ulp; the second part makes up for that too
    s.inv = inverse * q_max;
    s.low = fmaf(-s.inv, a, q_max) * inverse;
  }
  return s;
}
// most / Q: the product with the rounded 1 / Q, corrected by its remainder.
__device__ __forceinline__ float scale_of(float most, bool e4m3) {
  const float q_max = e4m3 ? 448.0f : 127.0f, inverse = e4m3 ? 1.0f / 448.0f : 1.0f / 127.0f, s = most * inverse;
  return fmaf(fmaf(-s, q_max, most), inverse, s);
}
__device__ __forceinline__ float code_value(float g, const RowScale& s) { return fmaf(g, s.inv, g * s.low); }

struct Shared {
  float sums[2][32];
  uint32_t tops[2][32];
};
__device__ __forceinline__ bool in_range(float ss, float eps) { return ss < kHuge && (ss >= kTiny || eps >= kTiny); }

// Rows whose squares leave the 32-bit range are summed again after the exact scaling by the power of two
// 2^-e (in two factors) that brings the largest entry to [1, 2).
struct Down {
  float f1, f2;
  int e;
};
__device__ __forceinline__ Down scale_down(uint32_t top) {
  const int e = ilogbf(__uint_as_float(top)), half = -e / 2;
  return {ldexpf(1.0f, half), ldexpf(1.0f, -e - half), e};
}
// 1 / sqrt(mean + eps 2^-2e) for such a row; `top` is its largest magnitude (0: factor 0, so zeros stay zeros).
__device__ __forceinline__ float root_down(float mean, float eps_root, uint32_t top, int e) {
  if (top == 0) return 0.0f;
  if (top >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  const float t = ldexpf(eps_root, -e);
  return t > 0x1p+60f ? 1.0f / t : 1.0f / sqrtf(mean + t * t);
}

// Rows of any length, by repeated passes over memory, element by element. residual_out is written in the last
// pass, by the thread that reads the same element, so it may be x or residual.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_quantize_long(const __grid_constant__ NormArgs p) {
  __shared__ Shared s;
  const bool e4m3 = p.q_type == IMD_TYPE_E4M3;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* res = p.residual == nullptr ? nullptr : static_cast<const T*>(p.residual) + row * p.residual_stride;
    auto sum = [&](int64_t j) { return to_float(x[j]) + (res != nullptr ? to_float(res[j]) : 0.0f); };
    auto weight = [&](int64_t j) {
      return p.weight_type == p.x_type ? to_float(static_cast<const T*>(p.weight)[j]) : static_cast<const float*>(p.weight)[j];
    };
    Down d{1.0f, 1.0f, 0};
    float ss = 0.0f;
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
      const float h = sum(j);
      ss = fmaf(h, h, ss);
    }
    ss = row_sum<false>(ss, s.sums[0]);
    float r = 1.0f / sqrtf(ss / static_cast<float>(p.dim) + p.eps);
    if (!in_range(ss, p.eps)) {  // uniform over the row
      uint32_t top = 0;
      for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) top = max(top, magnitude(sum(j)));
      top = row_max<false>(top, s.tops[0]);
      if (top != 0 && top < 0x7F800000u) d = scale_down(top);
      ss = 0.0f;
      for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
        const float h = sum(j) * d.f1 * d.f2;
        ss = fmaf(h, h, ss);
      }
      ss = row_sum<false>(ss, s.sums[1]);
      r = root_down(ss / static_cast<float>(p.dim), p.eps_root, top, d.e);
    }
    const Factor f = split(r);
    uint32_t top = 0;
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) top = max(top, magnitude(sum(j) * d.f1 * d.f2 * f.p * weight(j)));
    const RowScale q = row_scale(row_max<false>(top, s.tops[1]), f.m, e4m3);
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
      const float h = sum(j);
      if (p.residual_out != nullptr) static_cast<T*>(p.residual_out)[row * p.residual_out_stride + j] = from_float<T>(h);
      const float y = code_value(h * d.f1 * d.f2 * f.p * weight(j) * q.pre, q);
      store_codes<1>(static_cast<uint8_t*>(p.q) + row * p.q_stride, j, &y, e4m3, q.keep);
    }
    if (threadIdx.x == 0) p.scale[row] = scale_of(q.most, e4m3);
  }
}

// From the 32-bit sums h of a row to its outputs; E vectors of V elements per thread. `loaded` is called once,
// after the first reduction: every thread of the row has then taken its h from wherever the row was. ANY: rows, weight
// and outputs of any alignment, the last vector of a row may be short (its h are zeros).
template <typename T, int V, int E, bool WARP, bool ANY, typename Loaded>
__device__ __forceinline__ void finish_row(const NormArgs& p, int64_t row, int threads, int t, float (*h)[V], Shared& s,
                                           Loaded loaded) {
  const int dim = static_cast<int>(p.dim);
  const bool e4m3 = p.q_type == IMD_TYPE_E4M3, same = p.weight_type == p.x_type;
  Piece<T, V> w[E];
  if (p.residual_out != nullptr) {
    T* out = static_cast<T*>(p.residual_out) + row * p.residual_out_stride;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      if constexpr (ANY) store_any<T, V>(out + j, h[i], dim - j);
      else if (j < dim) Piece<T, V>::store(out, j, h[i]);
    }
  }
  if (same) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      w[i].clear();
      if (ANY && (j + V > dim || reinterpret_cast<uintptr_t>(p.weight) % 16 != 0)) w[i].load_part(p.weight, j, dim - j);
      else if (j < dim) w[i].load(p.weight, j);
    }
  }
  float r;
  for (uint32_t top = ~0u, e = 0;;) {  // a second time only for rows that leave the range
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) ss = fmaf(h[i][v], h[i][v], ss);
    ss = row_sum<WARP>(ss, s.sums[top == ~0u ? 0 : 1]);
    if (top == ~0u) loaded();
    const float mean = ss / static_cast<float>(dim);
    if (top != ~0u) {
      r = root_down(mean, p.eps_root, top, static_cast<int>(e));
      break;
    }
    if (in_range(ss, p.eps)) {
      r = 1.0f / sqrtf(mean + p.eps);
      break;
    }
    top = 0;
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) top = max(top, magnitude(h[i][v]));
    top = row_max<WARP>(top, s.tops[0]);
    if (top != 0 && top < 0x7F800000u) {
      const Down d = scale_down(top);
      e = static_cast<uint32_t>(d.e);
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] = h[i][v] * d.f1 * d.f2;
    }
  }
  const Factor f = split(r);
  uint32_t top = 0;
  if (same) {
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] = h[i][v] * f.p * w[i].value(v);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
#pragma unroll
      for (int v = 0; v < V; ++v)
        if (j + v < dim) h[i][v] = h[i][v] * f.p * static_cast<const float*>(p.weight)[j + v];
    }
  }
#pragma unroll
  for (int i = 0; i < E; ++i)
#pragma unroll
    for (int v = 0; v < V; ++v) top = max(top, magnitude(h[i][v]));
  const RowScale c = row_scale(row_max<WARP>(top, s.tops[1]), f.m, e4m3);
  if (c.pre != 1.0f) {  // rare, the same for the row
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] *= c.pre;
  }
#pragma unroll
  for (int i = 0; i < E; ++i) {
    const int j = (i * threads + t) * V;
    if (j < dim) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] = code_value(h[i][v], c);
      if constexpr (ANY) store_codes_any<V>(static_cast<uint8_t*>(p.q) + row * p.q_stride + j, h[i], dim - j, e4m3, c.keep);
      else store_codes<V>(static_cast<uint8_t*>(p.q) + row * p.q_stride, j, h[i], e4m3, c.keep);
    }
  }
  if (t == 0) p.scale[row] = scale_of(c.most, e4m3);
}

// Rows in registers, one per warp or per CTA.
// Up to 64 registers allow 1024 threads (f32 64 x 14128 with the residual: 6.6 us, by repeated passes 12.8; 4000 x 16384: 147
// against 352).
template <int V, int E>
constexpr int kMostThreads = V * E <= 16 ? 1024 : 512;
template <typename T, int V, int E, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : kMostThreads<V, E>)
k_norm_quantize(const __grid_constant__ NormArgs p) {
  __shared__ Shared s;
  const int threads = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t first = WARP ? blockIdx.x * static_cast<int64_t>(kWarpRows) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? kWarpRows : 1);
  const int dim = static_cast<int>(p.dim);
  for (int64_t row = first; row < p.rows; row += step) {
    // every load of the row is issued before its first store: residual_out may be x or residual
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    Piece<T, V> in[E], res[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      in[i].clear();
      if (j < dim) in[i].load(x, j);
    }
    if (p.residual != nullptr) {
      const T* r = static_cast<const T*>(p.residual) + row * p.residual_stride;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int j = (i * threads + t) * V;
        res[i].clear();
        if (j < dim) res[i].load(r, j);
      }
    }
    float h[E][V];
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] = in[i].value(v);
    if (p.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] += res[i].value(v);
    }
    finish_row<T, V, E, WARP, false>(p, row, threads, t, h, s, [] {});
  }
}

// Many rows: a persistent CTA whose rows arrive by bulk copies in a ring of shared memory, so that the bytes
// in flight do not depend on registers and the next rows arrive while this one is reduced and stored. A slot
// is refilled right after the row's first reduction, whose barrier says that every thread has read it. (8191 x 8192 bf16
// with the residual 78 us, rows loaded to registers 108.)
template <typename T, int V, int E>
__global__ void __launch_bounds__(512, 2) k_norm_quantize_ring(const __grid_constant__ NormArgs p, int slots) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ Shared s;
  __shared__ uint64_t bars[kMaxSlots];
  __shared__ int gave_up;
  const int threads = blockDim.x, t = threadIdx.x, dim = static_cast<int>(p.dim);
  const uint32_t row_bytes = static_cast<uint32_t>(dim) * sizeof(T);
  const uint32_t slot_bytes = row_bytes * (p.residual != nullptr ? 2 : 1);
  volatile int* abort = &gave_up;
  auto fetch = [&](int64_t row, int slot) {
    const uint32_t bar = smem_u32(&bars[slot]), dst = smem_u32(ring) + slot * slot_bytes;
    mbar_expect_tx(bar, slot_bytes);
    bulk_load(dst, static_cast<const T*>(p.x) + row * p.x_stride, row_bytes, bar);
    if (p.residual != nullptr)
      bulk_load(dst + row_bytes, static_cast<const T*>(p.residual) + row * p.residual_stride, row_bytes, bar);
  };
  if (t == 0) {
    gave_up = 0;
    for (int i = 0; i < slots; ++i) mbar_init(smem_u32(&bars[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    for (int i = 0; i < slots; ++i) {
      const int64_t row = blockIdx.x + static_cast<int64_t>(i) * gridDim.x;
      if (row < p.rows) fetch(row, i);
    }
  }
  __syncthreads();
  int slot = 0;
  uint32_t phase = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    mbar_wait(smem_u32(&bars[slot]), phase, abort);
    const T* x = reinterpret_cast<const T*>(ring + slot * slot_bytes);
    float h[E][V];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      Piece<T, V> in;
      in.clear();
      if (j < dim) in.load(x, j);
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] = in.value(v);
    }
    if (p.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int j = (i * threads + t) * V;
        Piece<T, V> res;
        res.clear();
        if (j < dim) res.load(x + dim, j);
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] += res.value(v);
      }
    }
    finish_row<T, V, E, false, false>(p, row, threads, t, h, s, [&] {
      const int64_t next = row + static_cast<int64_t>(slots) * gridDim.x;
      if (t == 0 && next < p.rows && !*abort) {  // after a wait that gave up every barrier is passed, but nothing is fetched
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        fetch(next, slot);
      }
    });
    if (++slot == slots) {
      slot = 0;
      phase ^= 1u;
    }
  }
  if (t == 0 && *abort) {
    let_land_any(slots, [&](int i) { return smem_u32(&bars[i]); });
    atomicOr(p.error_word, 1u);
  }
}

// Rows of any alignment and length: the same ring, filled by 4-byte asynchronous copies of the aligned words that hold a
// row; a thread shifts its vector out of them (4096 x 5001 bf16 70 us, element by element 155). `area` bytes of a slot hold a row's words.
template <typename T, int V, int E>
__global__ void __launch_bounds__(512, 2) k_norm_quantize_any(const __grid_constant__ NormArgs p, int slots, int area) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ Shared s;
  const int threads = blockDim.x, t = threadIdx.x, dim = static_cast<int>(p.dim);
  const int slot_bytes = area * (p.residual != nullptr ? 2 : 1), row_bytes = dim * static_cast<int>(sizeof(T));
  const Span span_x = span_of(p.x, p.rows, p.x_stride * static_cast<int64_t>(sizeof(T)), row_bytes);
  const Span span_r = span_of(p.residual, p.rows, p.residual_stride * static_cast<int64_t>(sizeof(T)), row_bytes);
  auto bring = [&](const T* from, const Span& span, uint8_t* to) {
    const uintptr_t first = reinterpret_cast<uintptr_t>(from) & ~static_cast<uintptr_t>(3);
    const int words = static_cast<int>((reinterpret_cast<uintptr_t>(from) + row_bytes - first + 3) / 4);
    for (int i = t; i < words; i += threads) {
      const uintptr_t a = first + 4 * static_cast<uintptr_t>(i);
      if (a >= span.lo && a + 4 <= span.hi) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(to) + 4 * i), "l"(a) : "memory");
      } else {  // a word that reaches beyond the matrix, at its two ends
#pragma unroll
        for (int b = 0; b < 4; b += 2)
          if (a + b >= span.lo && a + b + 2 <= span.hi)
            *reinterpret_cast<uint16_t*>(to + 4 * i + b) = *reinterpret_cast<const uint16_t*>(a + b);
      }
    }
  };
  auto fetch = [&](int64_t row, int slot) {
    if (row < p.rows) {
      bring(static_cast<const T*>(p.x) + row * p.x_stride, span_x, ring + slot * slot_bytes);
      if (p.residual != nullptr)
        bring(static_cast<const T*>(p.residual) + row * p.residual_stride, span_r, ring + slot * slot_bytes + area);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto take = [&](const T* from, const uint8_t* words, int j) {  // the vector at element j
    Piece<T, V> v;
    const uint4 a = *reinterpret_cast<const uint4*>(words + j * sizeof(T));
    v.w[0] = a.x, v.w[1] = a.y, v.w[2] = a.z, v.w[3] = a.w;
    if (sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(from) & 2) != 0) {
      const uint32_t next = *reinterpret_cast<const uint32_t*>(words + j * sizeof(T) + 16);
      v.w[0] = __funnelshift_r(a.x, a.y, 16), v.w[1] = __funnelshift_r(a.y, a.z, 16);
      v.w[2] = __funnelshift_r(a.z, a.w, 16), v.w[3] = __funnelshift_r(a.w, next, 16);
    }
    return v;
  };
  for (int i = 0; i + 1 < slots; ++i) fetch(blockIdx.x + static_cast<int64_t>(i) * gridDim.x, i);
  int slot = 0;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    if (slots == 2) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (slots == 3) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else asm volatile("cp.async.wait_group 2;" ::: "memory");
    __syncthreads();  // this row is here, and the slot of the row before it has been read by every thread
    fetch(row + static_cast<int64_t>(slots - 1) * gridDim.x, slot == 0 ? slots - 1 : slot - 1);
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* r = static_cast<const T*>(p.residual) + row * p.residual_stride;
    const uint8_t* words = ring + slot * slot_bytes;
    float h[E][V];
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      Piece<T, V> in;
      in.clear();
      if (j < dim) in = take(x, words, j);
#pragma unroll
      for (int v = 0; v < V; ++v) h[i][v] = j + v < dim ? in.value(v) : 0.0f;
    }
    if (p.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int j = (i * threads + t) * V;
        Piece<T, V> in;
        in.clear();
        if (j < dim) in = take(r, words + area, j);
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] += j + v < dim ? in.value(v) : 0.0f;
      }
    }
    finish_row<T, V, E, false, true>(p, row, threads, t, h, s, [] {});
    if (++slot == slots) slot = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

unsigned int grid_of(int64_t ctas) { return static_cast<unsigned int>(ctas < (1 << 30) ? ctas : (1 << 30)); }

// Fewest vectors per thread that hold the row: a warp for rows of up to 32 * 4 vectors, else a CTA of
// up to 1024 threads with 1, 2 or 4 (16 when the vectors are single elements) vectors each.
template <typename T, int V>
bool launch_registers(const NormArgs& a, cudaStream_t stream) {
  const int64_t vecs = (a.dim + V - 1) / V;
  if (vecs <= 128) {
    const unsigned int grid = grid_of((a.rows + kWarpRows - 1) / kWarpRows);
    if (vecs <= 32) k_norm_quantize<T, V, 1, true><<<grid, 32 * kWarpRows, 0, stream>>>(a);
    else k_norm_quantize<T, V, 4, true><<<grid, 32 * kWarpRows, 0, stream>>>(a);
    return true;
  }
  constexpr int kMost = V == 1 ? 16 : 4;
  if (vecs > kMostThreads<V, kMost> * kMost) return false;
  // with rows to fill the GPU, few threads with many loads in flight each; else as many threads as help
  const int64_t least = a.rows >= 512 ? 2 : 1;
  int64_t per_thread = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : kMost;
  if (per_thread < least) per_thread = least;
  const int threads = static_cast<int>(((vecs + per_thread - 1) / per_thread + 31) / 32 * 32);
  const unsigned int grid = grid_of(a.rows);
  if (per_thread == 1) k_norm_quantize<T, V, 1, false><<<grid, threads, 0, stream>>>(a);
  else if (per_thread == 2) k_norm_quantize<T, V, 2, false><<<grid, threads, 0, stream>>>(a);
  else k_norm_quantize<T, V, kMost, false><<<grid, threads, 0, stream>>>(a);
  return true;
}

// The ring form: rows enough for every CTA slot of the GPU to take several.
template <typename T, int V, int E>
bool launch_ring(const NormArgs& a, const DeviceInfo& dev, int least_per_sm, cudaStream_t stream) {
  const int64_t vecs = a.dim / V;
  const int threads = static_cast<int>(((vecs + E - 1) / E + 31) / 32 * 32);
  if (threads > 512) return false;
  const int64_t slot_bytes = a.dim * static_cast<int64_t>(sizeof(T)) * (a.residual != nullptr ? 2 : 1);
  int64_t per_sm = 1024 / threads;
  if (per_sm > kRingBytes / (2 * slot_bytes)) per_sm = kRingBytes / (2 * slot_bytes);
  if (per_sm < least_per_sm) return false;
  int64_t slots = kRingBytes / per_sm / slot_bytes;
  if (slots > kMaxSlots) slots = kMaxSlots;
  const int64_t ctas = static_cast<int64_t>(dev.sms) * per_sm;
  if (a.rows < 3 * ctas) return false;
  k_norm_quantize_ring<T, V, E><<<static_cast<unsigned int>(ctas), threads, slots * slot_bytes, stream>>>(a, static_cast<int>(slots));
  return true;
}

template <typename T, int V, int E>
bool launch_any(const NormArgs& a, const DeviceInfo& dev, cudaStream_t stream) {
  const int64_t vecs = (a.dim + V - 1) / V;
  const int threads = static_cast<int>(((vecs + E - 1) / E + 31) / 32 * 32);
  if (threads > 512) return false;
  const int64_t area = (a.dim * static_cast<int64_t>(sizeof(T)) + 15) / 16 * 16 + 32;  // a word more, vectors read whole
  const int64_t slot_bytes = area * (a.residual != nullptr ? 2 : 1);
  int64_t per_sm = 1024 / threads;
  if (per_sm > kRingBytes / (2 * slot_bytes)) per_sm = kRingBytes / (2 * slot_bytes);
  if (per_sm < 1) return false;
  int64_t slots = kRingBytes / per_sm / slot_bytes;
  if (slots > 4) slots = 4;
  const int64_t ctas = static_cast<int64_t>(dev.sms) * per_sm;
  k_norm_quantize_any<T, V, E><<<static_cast<unsigned int>(a.rows < ctas ? a.rows : ctas), threads, slots * slot_bytes, stream>>>(
      a, static_cast<int>(slots), static_cast<int>(area));
  return true;
}

template <typename T>
imd_status_t launch(NormArgs a, cudaStream_t stream) {
  const DeviceInfo* dev = device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  a.error_word = dev->error_word;
  constexpr int V = 16 / sizeof(T);
  auto wide = [](const void* p, int64_t stride, int size, int64_t rows) {
    const uintptr_t unit = static_cast<uintptr_t>(V) * size;
    return reinterpret_cast<uintptr_t>(p) % unit == 0 && (rows <= 1 || stride % V == 0);
  };
  const int sw = a.weight_type == IMD_TYPE_F32 ? 4 : 2;
  const bool vec = a.dim % V == 0 && wide(a.x, a.x_stride, sizeof(T), a.rows) &&
                   wide(a.residual, a.residual_stride, sizeof(T), a.rows) &&
                   wide(a.residual_out, a.residual_out_stride, sizeof(T), a.rows) &&
                   wide(a.q, a.q_stride, 1, a.rows) && reinterpret_cast<uintptr_t>(a.weight) % (V * sw) == 0;
  if (vec && a.dim / V > 64 &&
      (launch_ring<T, V, 4>(a, *dev, 4, stream) || launch_ring<T, V, 2>(a, *dev, 2, stream) || launch_ring<T, V, 4>(a, *dev, 1, stream)))
    return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
  // (f32 rows of 8193 to 16384 elements with a residual: two slots fill the ring, registers are quicker, 76 against 91 us at
  // 1000 x 12001; without it 42 against 63)
  if (!vec && a.dim >= 256 &&
      (launch_any<T, V, 2>(a, *dev, stream) || launch_any<T, V, 4>(a, *dev, stream) ||
       (a.residual == nullptr && launch_any<T, V, 32 / V>(a, *dev, stream))))
    return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
  if (!(vec ? launch_registers<T, V>(a, stream) : launch_registers<T, 1>(a, stream)))
    k_norm_quantize_long<T><<<grid_of(a.rows), 1024, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace

bool norm_setup() {
  auto smem = [](auto* f) {
    return cudaFuncSetAttribute(reinterpret_cast<const void*>(f), cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes) ==
           cudaSuccess;
  };
  return smem(k_norm_quantize_ring<float, 4, 2>) && smem(k_norm_quantize_ring<float, 4, 4>) &&
         smem(k_norm_quantize_ring<__half, 8, 2>) && smem(k_norm_quantize_ring<__half, 8, 4>) &&
         smem(k_norm_quantize_ring<__nv_bfloat16, 8, 2>) && smem(k_norm_quantize_ring<__nv_bfloat16, 8, 4>) &&
         smem(k_norm_quantize_any<float, 4, 2>) && smem(k_norm_quantize_any<float, 4, 4>) && smem(k_norm_quantize_any<float, 4, 8>) &&
         smem(k_norm_quantize_any<__half, 8, 2>) && smem(k_norm_quantize_any<__half, 8, 4>) &&
         smem(k_norm_quantize_any<__nv_bfloat16, 8, 2>) && smem(k_norm_quantize_any<__nv_bfloat16, 8, 4>);
}

imd_status_t norm_quantize_launch(const NormArgs& a, cudaStream_t stream) {
  if (a.x_type == IMD_TYPE_F32) return launch<float>(a, stream);
  if (a.x_type == IMD_TYPE_F16) return launch<__half>(a, stream);
  return launch<__nv_bfloat16>(a, stream);
}

}  // namespace imd
