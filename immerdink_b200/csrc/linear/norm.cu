// RMS norm with the residual's addition and an 8-bit output with one scale per row.
//
//   h = x + r;  y_j = h_j * rsqrt(mean h^2 + eps) * w_j;  a = max_j |y_j|;  scale = a / Q;
//   q_j = round(y_j * (Q / a))                                       Q = 127 (int8), 448 (e4m3)
//
// Bound by HBM: 2 + 2 + 2 + 1 bytes per element for 16-bit x with a residual that is written back.
// A row is read once: its values stay in registers (`E` vectors per thread) through both row
// reductions, the sum of squares and the largest |y|. Short rows take one warp each, longer rows
// one CTA; rows beyond the register capacity are read three times (twice from L2).
#include <cmath>
#include <cstdint>

#include "types.cuh"

namespace imd {
namespace {

constexpr int kWarpRows = 4;     // rows (= warps) of a CTA in the warp-per-row form
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

template <typename T, int V>
__device__ __forceinline__ void load(const void* p, int64_t i, float* f) {
  const Pack<T, V> t = *reinterpret_cast<const Pack<T, V>*>(static_cast<const T*>(p) + i);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = to_float(t.v[j]);
}
template <int V>
__device__ __forceinline__ void store_codes(void* p, int64_t i, const float* y, bool e4m3) {
  Pack<uint8_t, V> t;
#pragma unroll
  for (int j = 0; j < V; ++j)
    t.v[j] = e4m3 ? static_cast<uint8_t>(__nv_cvt_float_to_fp8(y[j], __NV_SATFINITE, __NV_E4M3))
                  : static_cast<uint8_t>(y[j] != y[j] ? 0 : __float2int_rn(y[j]));
  *reinterpret_cast<Pack<uint8_t, V>*>(static_cast<uint8_t*>(p) + i) = t;
}

// What turns a row's y into codes: q = round(y * pre * inv), scale as stored.
struct RowScale {
  float pre, inv, scale;
};
__device__ __forceinline__ RowScale row_scale(uint32_t top, float q_max) {
  RowScale s{1.0f, 0.0f, 0.0f};
  if (top >= 0x7F800000u) {
    s.inv = s.scale = __uint_as_float(0x7FC00000u);  // a NaN or an infinity in the row
  } else if (top != 0) {
    const float a = __uint_as_float(top);
    s.scale = a / q_max;
    if (a < 0x1p-100f) s.pre = 0x1p+100f;  // Q / a would leave the range
    s.inv = q_max / (a * s.pre);
  }
  return s;
}

// 1 / sqrt(mean h^2 + eps) of a row whose squares left the 32-bit range: the row is scaled by the
// power of two 2^-e that brings its largest entry to [1, 2), and the factor for the scaled values
// is returned (0 rows: factor 0). `scale_down` receives 2^-e in two factors.
struct Rescaled {
  float f1, f2, r;
};
__device__ __forceinline__ void power_of_two(uint32_t top, Rescaled* s, int* e) {
  *e = top == 0 ? 0 : ilogbf(__uint_as_float(top));
  const int a = -*e / 2;
  s->f1 = ldexpf(1.0f, a);
  s->f2 = ldexpf(1.0f, -*e - a);
}

template <typename T, int V, int E, bool WARP>
__global__ void __launch_bounds__(WARP ? 32 * kWarpRows : 1024)
k_norm_quantize(const __grid_constant__ NormArgs p) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  const int threads = WARP ? 32 : blockDim.x;
  const int t = WARP ? (threadIdx.x & 31) : threadIdx.x;
  const int64_t first = WARP ? blockIdx.x * static_cast<int64_t>(kWarpRows) + (threadIdx.x >> 5) : blockIdx.x;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (WARP ? kWarpRows : 1);
  const int dim = static_cast<int>(p.dim);
  const bool e4m3 = p.q_type == IMD_TYPE_E4M3;
  for (int64_t row = first; row < p.rows; row += step) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    float h[E][V];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      if (j < dim) {
        load<T, V>(x, j, h[i]);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] = 0.0f;
      }
    }
    if (p.residual != nullptr) {
      const T* r = static_cast<const T*>(p.residual) + row * p.residual_stride;
#pragma unroll
      for (int i = 0; i < E; ++i) {
        const int j = (i * threads + t) * V;
        if (j < dim) {
          float f[V];
          load<T, V>(r, j, f);
#pragma unroll
          for (int v = 0; v < V; ++v) h[i][v] += f[v];
          if (p.residual_out != nullptr) {
            Pack<T, V> o;
#pragma unroll
            for (int v = 0; v < V; ++v) o.v[v] = from_float<T>(h[i][v]);
            *reinterpret_cast<Pack<T, V>*>(static_cast<T*>(p.residual_out) + row * p.residual_out_stride + j) = o;
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
#pragma unroll
      for (int v = 0; v < V; ++v) ss = fmaf(h[i][v], h[i][v], ss);
    ss = row_sum<WARP>(ss, sums[0]);
    float r = 1.0f / sqrtf(ss / static_cast<float>(dim) + p.eps);
    if (!(ss < kHuge) || (ss < kTiny && p.eps < kTiny)) {  // uniform over the row
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) top = max(top, magnitude(h[i][v]));
      top = row_max<WARP>(top, tops[0]);
      r = 0.0f;
      if (top >= 0x7F800000u) {
        r = __uint_as_float(0x7FC00000u);
      } else if (top != 0) {
        Rescaled s;
        int e;
        power_of_two(top, &s, &e);
        ss = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            h[i][v] = h[i][v] * s.f1 * s.f2;
            ss = fmaf(h[i][v], h[i][v], ss);
          }
        ss = row_sum<WARP>(ss, sums[1]);
        r = static_cast<float>(1.0 / sqrt(static_cast<double>(ss) / dim + p.eps64 * exp2(-2.0 * e)));
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      if (j < dim) {
        float w[V];
        if (p.weight_type == p.x_type) {
          load<T, V>(p.weight, j, w);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) w[v] = static_cast<const float*>(p.weight)[j + v];
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
          h[i][v] = h[i][v] * r * w[v];
          top = max(top, magnitude(h[i][v]));
        }
      }
    }
    const RowScale s = row_scale(row_max<WARP>(top, tops[1]), e4m3 ? 448.0f : 127.0f);
#pragma unroll
    for (int i = 0; i < E; ++i) {
      const int j = (i * threads + t) * V;
      if (j < dim) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[i][v] = h[i][v] * s.pre * s.inv;
        store_codes<V>(static_cast<uint8_t*>(p.q) + row * p.q_stride, j, h[i], e4m3);
      }
    }
    if (t == 0) p.scale[row] = s.scale;
  }
}

// Rows of any length: the row is read once per reduction and once for the codes; residual_out is
// written in the last pass, by the thread that reads the same elements, so it may be x or residual.
template <typename T>
__global__ void __launch_bounds__(1024) k_norm_quantize_long(const __grid_constant__ NormArgs p) {
  __shared__ float sums[2][32];
  __shared__ uint32_t tops[2][32];
  const bool e4m3 = p.q_type == IMD_TYPE_E4M3;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const T* res = p.residual == nullptr ? nullptr : static_cast<const T*>(p.residual) + row * p.residual_stride;
    auto sum = [&](int64_t j) { return to_float(x[j]) + (res != nullptr ? to_float(res[j]) : 0.0f); };
    auto weight = [&](int64_t j) {
      return p.weight_type == p.x_type ? to_float(static_cast<const T*>(p.weight)[j])
                                       : static_cast<const float*>(p.weight)[j];
    };
    float ss = 0.0f;
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
      const float h = sum(j);
      ss = fmaf(h, h, ss);
    }
    ss = row_sum<false>(ss, sums[0]);
    Rescaled f{1.0f, 1.0f, 1.0f / sqrtf(ss / static_cast<float>(p.dim) + p.eps)};
    if (!(ss < kHuge) || (ss < kTiny && p.eps < kTiny)) {
      uint32_t top = 0;
      for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) top = max(top, magnitude(sum(j)));
      top = row_max<false>(top, tops[0]);
      f.r = 0.0f;
      if (top >= 0x7F800000u) {
        f.r = __uint_as_float(0x7FC00000u);
      } else if (top != 0) {
        int e;
        power_of_two(top, &f, &e);
        ss = 0.0f;
        for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
          const float h = sum(j) * f.f1 * f.f2;
          ss = fmaf(h, h, ss);
        }
        ss = row_sum<false>(ss, sums[1]);
        f.r = static_cast<float>(1.0 / sqrt(static_cast<double>(ss) / p.dim + p.eps64 * exp2(-2.0 * e)));
      }
    }
    uint32_t top = 0;
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x)
      top = max(top, magnitude(sum(j) * f.f1 * f.f2 * f.r * weight(j)));
    const RowScale s = row_scale(row_max<false>(top, tops[1]), e4m3 ? 448.0f : 127.0f);
    for (int64_t j = threadIdx.x; j < p.dim; j += blockDim.x) {
      const float h = sum(j);
      if (p.residual_out != nullptr)
        static_cast<T*>(p.residual_out)[row * p.residual_out_stride + j] = from_float<T>(h);
      const float y = h * f.f1 * f.f2 * f.r * weight(j) * s.pre * s.inv;
      store_codes<1>(static_cast<uint8_t*>(p.q) + row * p.q_stride, j, &y, e4m3);
    }
    if (threadIdx.x == 0) p.scale[row] = s.scale;
  }
}

unsigned int grid_of(int64_t ctas) { return static_cast<unsigned int>(ctas < (1 << 30) ? ctas : (1 << 30)); }

// Fewest vectors per thread that hold the row: a warp for rows of up to 32 * 4 vectors, else a CTA of
// up to 1024 threads with 1, 2, 4 (16 when the vectors are single elements) vectors each.
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
  const int64_t per_thread = vecs <= 1024 ? 1 : vecs <= 2048 ? 2 : kMost;
  if (vecs > 1024 * kMost) return false;
  const int threads = static_cast<int>(((vecs + per_thread - 1) / per_thread + 31) / 32 * 32);
  const unsigned int grid = grid_of(a.rows);
  if (per_thread == 1) k_norm_quantize<T, V, 1, false><<<grid, threads, 0, stream>>>(a);
  else if (per_thread == 2) k_norm_quantize<T, V, 2, false><<<grid, threads, 0, stream>>>(a);
  else k_norm_quantize<T, V, kMost, false><<<grid, threads, 0, stream>>>(a);
  return true;
}

template <typename T>
imd_status_t launch(const NormArgs& a, cudaStream_t stream) {
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
  if (!(vec ? launch_registers<T, V>(a, stream) : launch_registers<T, 1>(a, stream)))
    k_norm_quantize_long<T><<<grid_of(a.rows), 1024, 0, stream>>>(a);
  return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace

imd_status_t norm_quantize_launch(const NormArgs& a, cudaStream_t stream) {
  if (a.x_type == IMD_TYPE_F32) return launch<float>(a, stream);
  if (a.x_type == IMD_TYPE_F16) return launch<__half>(a, stream);
  return launch<__nv_bfloat16>(a, stream);
}

}  // namespace imd
