// Products of operands whose rows start anywhere, with few rows of x or little work (choice.hpp): more of it is quicker on
// the tensor-core kernels (dense8.cu, dense4.cu), which then bring the rows as words too.
//
//   8 bits:  out[t, n] = xs[t] ws[n] sum_k x[t, k] w[n, k]
//   4 bits:  out[t, n] = sum_g ws[n, g] sum_{k in g} x[t, k] (w[n, k] - z[n, g])
//
// A CTA owns 16 rows of w (one mma.sync row tile) and up to 8 NT rows of x; its eight warps take the
// K chunks in turn and their partial sums are folded in a fixed order at the end. The order of k
// inside a chunk is free as long as both operands use the same one: a lane takes the consecutive k of
// its quarter of the chunk, and whatever four (16-bit) or eight (8-bit) of them a tensor instruction
// wants are already in its registers.
//
// 4-bit weights become exact 16-bit floats: a nibble or'ed into the mantissa of 128 (bf16) or 1024
// (f16) is 128 + w or 1024 + w, and subtracting 128 + z or 1024 + z is exact. A shift by 4 i and one
// lop3 give the nibbles i and i + 4 of a word as a pair, so the pairs of x are formed in that order
// too. A quad of lanes covers one group, so a group's sum is one accumulator, scaled in 32 bits.
// Bound by the loads of single words (5 x 5001 x 4091, g64: 16.8 us for 11 MB; int8 1000 x 300 x 777 12 us).
// e4m3 values are exact in f16 and their products are summed in 32-bit floats by the f16 instruction.
#include <cstdint>

#include "mma.cuh"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kWarps = 8;
constexpr int kRowsPerTile = 16;

// Folds the warps' partial tiles in the order of the warps and hands each output to `write`.
template <int NT, typename Acc, typename Write>
__device__ __forceinline__ void fold(Acc (*acc)[4], const LinearArgs& p, int64_t n0, int64_t t0, Write write) {
  __shared__ Acc part[kWarps][8 * NT][kRowsPerTile + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      part[warp][8 * j + 2 * (lane & 3) + (i & 1)][(lane >> 2) + 8 * (i >> 1)] = acc[j][i];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * NT * kRowsPerTile; i += 32 * kWarps) {
    const int c = i / kRowsPerTile, r = i % kRowsPerTile;
    Acc v = part[0][c][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) v += part[w][c][r];
    if (t0 + c < p.rows && n0 + r < p.n) write(t0 + c, n0 + r, v);
  }
}

template <typename X, int GROUP, int NT>
__global__ void __launch_bounds__(32 * kWarps) k_small_w4(const __grid_constant__ LinearArgs p) {
  constexpr int kBytes = GROUP / 8;       // weights of one lane and row in one group
  constexpr int kWords = kBytes / 4;
  constexpr uint32_t kMagic = nibble_magic<X>();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kRowsPerTile), t0 = blockIdx.y * static_cast<int64_t>(8 * NT);
  const int64_t row[2] = {min(n0 + (lane >> 2), p.n - 1), min(n0 + (lane >> 2) + 8, p.n - 1)};
  const uint8_t* w[2] = {static_cast<const uint8_t*>(p.w) + row[0] * p.w_stride,
                         static_cast<const uint8_t*>(p.w) + row[1] * p.w_stride};
  const int64_t w_end = (p.k + 1) / 2;
  const Span span_w = span_of(p.w, p.n, p.w_stride, w_end), span_x = span_of(p.x, p.rows, 2 * p.x_stride, 2 * p.k);
  const int64_t groups = (p.k + GROUP - 1) / GROUP;
  const uint8_t* x_row[NT];  // columns behind the last row of x repeat it and are not stored
#pragma unroll
  for (int j = 0; j < NT; ++j)
    x_row[j] = static_cast<const uint8_t*>(p.x) + 2 * min(t0 + 8 * j + (lane >> 2), p.rows - 1) * p.x_stride;
  const Nibbles<X> nibbles;
  float acc[NT][4] = {};
  auto group_of = [&](int64_t g, auto inside) {
    constexpr bool kInside = decltype(inside)::value;
    const int64_t k0 = g * GROUP + (lane & 3) * (GROUP / 4);
    uint32_t q[2][kWords], zero[2];
    float scale[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load_bytes<kBytes, kInside>(w[h], k0 / 2, w_end, span_w, q[h]);
      scale[h] = load_scale(p.scale4, p.scale_type, row[h] * p.scale_stride + g);
      const uint32_t z = p.zeros == nullptr ? 8u : p.zeros[row[h] * p.zeros_stride + g] & 15u;
      zero[h] = kMagic | z | (z << 16);
    }
    uint32_t x[NT][kWords][4];  // eight consecutive values of x for each word of weights
#pragma unroll
    for (int j = 0; j < NT; ++j)
      load_bytes<16 * kWords, kInside>(x_row[j], 2 * k0, 2 * p.k, span_x, &x[j][0][0]);
    float sum[NT][4] = {};
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      uint32_t a[2][4];  // [row][pair]: pairs (0, 4), (1, 5), (2, 6), (3, 7) of the word
#pragma unroll
      for (int h = 0; h < 2; ++h) nibbles.pairs(q[h][i], zero[h], a[h]);
      const uint32_t a01[4] = {a[0][0], a[1][0], a[0][1], a[1][1]}, a23[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const uint32_t* v = x[j][i];
        mma_pair(sum[j], a01, __byte_perm(v[0], v[2], 0x5410), __byte_perm(v[0], v[2], 0x7632), X());
        mma_pair(sum[j], a23, __byte_perm(v[1], v[3], 0x5410), __byte_perm(v[1], v[3], 0x7632), X());
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = fmaf(scale[i >> 1], sum[j][i], acc[j][i]);
  };
#pragma unroll 1
  for (int64_t g = warp; g < groups; g += kWarps) {
    if (g > 0 && (g + 1) * (GROUP / 2) + 4 <= w_end && (g + 1) * GROUP + 2 <= p.k) group_of(g, std::true_type());
    else group_of(g, std::false_type());
  }
  fold<NT, float>(acc, p, n0, t0, [&](int64_t t, int64_t n, float v) { store_out(p.out, p.out_type, t * p.out_stride + n, v); });
}

template <bool I8, int NT>
__global__ void __launch_bounds__(32 * kWarps) k_small_8(const __grid_constant__ LinearArgs p) {
  using Acc = typename std::conditional<I8, int, float>::type;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t n0 = blockIdx.x * static_cast<int64_t>(kRowsPerTile), t0 = blockIdx.y * static_cast<int64_t>(8 * NT);
  const uint8_t* w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
    w[h] = static_cast<const uint8_t*>(p.w) + min(n0 + (lane >> 2) + 8 * h, p.n - 1) * p.w_stride;
  const Span span_w = span_of(p.w, p.n, p.w_stride, p.k), span_x = span_of(p.x, p.rows, p.x_stride, p.k);
  Acc acc[NT][4] = {};
  const uint8_t* x_row[NT];  // columns behind the last row of x repeat it and are not stored
#pragma unroll
  for (int j = 0; j < NT; ++j)
    x_row[j] = static_cast<const uint8_t*>(p.x) + min(t0 + 8 * j + (lane >> 2), p.rows - 1) * p.x_stride;
  auto chunk = [&](int64_t c, auto inside) {
    constexpr bool kInside = decltype(inside)::value;
    const int64_t k0 = c * 64 + (lane & 3) * 16;
    uint32_t q[2][4], x[NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) load_bytes<16, kInside>(w[h], k0, p.k, span_w, q[h]);
#pragma unroll
    for (int j = 0; j < NT; ++j) load_bytes<16, kInside>(x_row[j], k0, p.k, span_x, x[j]);
    if constexpr (I8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t a[4] = {q[0][2 * i], q[1][2 * i], q[0][2 * i + 1], q[1][2 * i + 1]};
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_s8(acc[j], a, x[j][2 * i], x[j][2 * i + 1]);
      }
    } else {
      uint32_t wide[2][4][2], wx[NT][4][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) widen_e4m3(q[h], wide[h]);
#pragma unroll
      for (int j = 0; j < NT; ++j) widen_e4m3(x[j], wx[j]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a[4] = {wide[0][i][0], wide[1][i][0], wide[0][i][1], wide[1][i][1]};
#pragma unroll
        for (int j = 0; j < NT; ++j) mma_f16(acc[j], a, wx[j][i][0], wx[j][i][1]);
      }
    }
  };
#pragma unroll 1
  for (int64_t c = warp; c * 64 < p.k; c += kWarps) {
    if (c > 0 && (c + 1) * 64 + 4 <= p.k) chunk(c, std::true_type());
    else chunk(c, std::false_type());
  }
  fold<NT, Acc>(acc, p, n0, t0, [&](int64_t t, int64_t n, Acc v) {
    store_out(p.out, p.out_type, t * p.out_stride + n, static_cast<float>(v) * p.x_scale[t] * p.w_scale8[n]);
  });
}

template <int NT>
void launch(const LinearArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr int threads = 32 * kWarps;
  if (a.kind == WeightKind::kI8) {
    k_small_8<true, NT><<<grid, threads, 0, stream>>>(a);
  } else if (a.kind == WeightKind::kE4M3) {
    k_small_8<false, NT><<<grid, threads, 0, stream>>>(a);
  } else if (a.x_type == IMD_TYPE_F16) {
    if (a.group == 128) k_small_w4<__half, 128, NT><<<grid, threads, 0, stream>>>(a);
    else if (a.group == 64) k_small_w4<__half, 64, NT><<<grid, threads, 0, stream>>>(a);
    else k_small_w4<__half, 32, NT><<<grid, threads, 0, stream>>>(a);
  } else {
    if (a.group == 128) k_small_w4<__nv_bfloat16, 128, NT><<<grid, threads, 0, stream>>>(a);
    else if (a.group == 64) k_small_w4<__nv_bfloat16, 64, NT><<<grid, threads, 0, stream>>>(a);
    else k_small_w4<__nv_bfloat16, 32, NT><<<grid, threads, 0, stream>>>(a);
  }
}

}  // namespace

imd_status_t linear_small_launch(const LinearArgs& a, cudaStream_t stream) {
  const int x_size = a.kind == WeightKind::kU4 ? 2 : 1;
  const int nt = a.rows <= 8 ? 1 : a.rows <= 16 ? 2 : 4;
  const int64_t tiles = (a.rows + 8 * nt - 1) / (8 * nt);
  LinearArgs part = a;
  for (int64_t t = 0; t < tiles; t += 65535) {  // the grid's second extent
    const int64_t t0 = t * 8 * nt, count = tiles - t < 65535 ? tiles - t : 65535;
    part.rows = a.rows - t0;
    part.x = static_cast<const uint8_t*>(a.x) + t0 * a.x_stride * x_size;
    if (a.x_scale != nullptr) part.x_scale = a.x_scale + t0;
    part.out = static_cast<uint8_t*>(a.out) + t0 * a.out_stride * (a.out_type == IMD_TYPE_F32 ? 4 : 2);
    const dim3 grid(static_cast<unsigned int>((a.n + kRowsPerTile - 1) / kRowsPerTile), static_cast<unsigned int>(count));
    if (nt == 1) launch<1>(part, grid, stream);
    else if (nt == 2) launch<2>(part, grid, stream);
    else launch<4>(part, grid, stream);
  }
  return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace imd
