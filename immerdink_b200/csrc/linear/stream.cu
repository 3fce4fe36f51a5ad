// 4-bit products with up to 16 rows of x whose weights lie in 16-byte units: the weights are streamed once.
//
//   out[t, n] = sum_g ws[n, g] sum_{k in g} x[t, k] (w[n, k] - z[n, g])
//
// Bound by HBM (n k / 2 bytes) and, next to it, by the issue of the unpacking. A persistent CTA walks tiles of
// 16 MT rows of w. One warp brings their next kStageBytes bytes per row by bulk copies, a row per lane, into a
// ring in shared memory, so that the bytes in flight depend on neither registers nor occupancy; eight warps each
// multiply their own kPieceBytes of every row by mma.sync (16 rows of w by 8 rows of x) and fold their sums
// in a fixed order at the end of a tile while the ring keeps filling.
//
// The order of k inside an instruction is free as long as both operands use the same one: a lane takes
// consecutive k of its quarter of a group with one load, and the words that an instruction wants are in its
// registers. See small.cu for how nibbles become exact 16-bit floats in pairs.
#include <cstdint>
#include <type_traits>

#include "cuda/sm100.cuh"
#include "dense.hpp"
#include "mma.cuh"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kWarps = 8;                  // multiplying warps; one more loads
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kPieceBytes = 128;           // of a row, per warp and stage
constexpr int kStageBytes = kPieceBytes * kWarps;
constexpr int kMaxStages = 8;
// Two CTAs share an SM; with 9 to 16 rows of x their registers allow one.
template <int NT>
constexpr int kSmemPerCta = (NT == 1 ? 110 : 220) * 1024;
template <int MT, int NT>
constexpr int kRingBytes = kSmemPerCta<NT> - 4 * 2 * kWarps * 8 * NT * (16 * MT + 1) - 1024;  // beside the partial sums

struct Params {
  LinearArgs a;
  int32_t stages, steps;  // ring depth; stages of a row
  int64_t tiles;
  unsigned int* error_word;
};

struct Ring {
  uint64_t full[kMaxStages], empty[kMaxStages];
  int gave_up;
};

__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(addr));
}
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&v)[2]) {
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(addr));
}
__device__ __forceinline__ void lds(uint32_t addr, uint32_t (&v)[1]) {
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(addr));
}

// The per-warp work: GROUP k are one quad's share of a load, kPerStep groups make a step of 128 k.
template <typename X, int GROUP, int MT, int NT>
struct Piece {
  static constexpr int kPerStep = 128 / GROUP, kWords = GROUP / 32, kXWords = kPerStep * kWords;
  // Row pitch in the ring: 16, 8 or 4 bytes per lane, without bank conflicts.
  static constexpr int kPitch = kStageBytes + (GROUP == 128 ? 64 : GROUP == 64 ? 32 : 16);
  uint32_t x[2][NT][kXWords][4];  // pairs of x in the order of the nibbles: (0, 4), (1, 5), (2, 6), (3, 7)
  float scale[2][2 * MT];
  uint32_t zero[2][2 * MT];
};

// What a warp needs beside the ring's bytes: this lane's rows of x, and its rows' scales and zero points.
template <typename X, int GROUP, int MT, int NT>
struct Source {
  using P = Piece<X, GROUP, MT, NT>;
  const uint16_t* x[NT];
  const uint8_t *scale[2 * MT], *zero[2 * MT];
  int k, groups, scale_type;
  bool row[NT], zeros;

  __device__ __forceinline__ void set_x(const LinearArgs& p, int lane) {
    k = static_cast<int>(p.k);
    groups = (k + GROUP - 1) / GROUP;
    scale_type = p.scale_type;
    zeros = p.zeros != nullptr;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int t = 8 * j + (lane >> 2);
      row[j] = t < p.rows;
      x[j] = static_cast<const uint16_t*>(p.x) + t * p.x_stride;
    }
  }
  __device__ __forceinline__ void set_tile(const LinearArgs& p, int64_t n0, int lane) {
    const int size = scale_type == IMD_TYPE_F32 ? 4 : 2;
#pragma unroll
    for (int h = 0; h < 2 * MT; ++h) {
      const int64_t n = min(n0 + (lane >> 2) + 8 * h, p.n - 1);
      scale[h] = static_cast<const uint8_t*>(p.scale4) + n * p.scale_stride * size;
      zero[h] = p.zeros + n * p.zeros_stride;
    }
  }
  // Loads of a piece that starts at k0, issued before the wait for the ring.
  __device__ __forceinline__ void fetch(int k0, int lane, P& q) const {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < P::kXWords; ++i) {
          const int at = k0 + 128 * s + GROUP * (i / P::kWords) + (lane & 3) * (GROUP / 4) + 8 * (i % P::kWords);
          uint4 v = make_uint4(0, 0, 0, 0);
          if (row[j] && at < k) v = __ldg(reinterpret_cast<const uint4*>(x[j] + at));
          q.x[s][j][i][0] = v.x, q.x[s][j][i][1] = v.y, q.x[s][j][i][2] = v.z, q.x[s][j][i][3] = v.w;
        }
    // the quad's lanes share a step's groups: lane l holds group l mod kPerStep
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int g = (k0 + 128 * s) / GROUP + (lane & (P::kPerStep - 1));
      const bool inside = g < groups;
      if (scale_type == IMD_TYPE_F32) {
#pragma unroll
        for (int h = 0; h < 2 * MT; ++h) q.scale[s][h] = inside ? __ldg(reinterpret_cast<const float*>(scale[h]) + g) : 0.0f;
      } else {
#pragma unroll
        for (int h = 0; h < 2 * MT; ++h) {
          const uint32_t v = inside ? __ldg(reinterpret_cast<const uint16_t*>(scale[h]) + g) : 0u;
          q.scale[s][h] = __uint_as_float(v);  // as a value: settle()
        }
      }
      if (zeros) {
#pragma unroll
        for (int h = 0; h < 2 * MT; ++h) q.zero[s][h] = inside ? __ldg(zero[h] + g) : 0u;
      } else {
#pragma unroll
        for (int h = 0; h < 2 * MT; ++h) q.zero[s][h] = 8u;
      }
    }
  }
  // The loads' results in the form the products take.
  __device__ __forceinline__ void settle(P& q) const {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < P::kXWords; ++i) {
          uint32_t* v = q.x[s][j][i];
          const uint32_t a = v[0], b = v[1], c = v[2], d = v[3];
          v[0] = __byte_perm(a, c, 0x5410), v[1] = __byte_perm(a, c, 0x7632);
          v[2] = __byte_perm(b, d, 0x5410), v[3] = __byte_perm(b, d, 0x7632);
        }
#pragma unroll
      for (int h = 0; h < 2 * MT; ++h) {
        const uint32_t bits = __float_as_uint(q.scale[s][h]);
        if (scale_type == IMD_TYPE_BF16) q.scale[s][h] = __uint_as_float(bits << 16);
        else if (scale_type == IMD_TYPE_F16) q.scale[s][h] = __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        q.zero[s][h] = nibble_magic<X>() | ((q.zero[s][h] & 15u) * 0x10001u);
      }
    }
  }
};

template <typename X, int GROUP, int MT, int NT>
__device__ __forceinline__ void multiply(const Piece<X, GROUP, MT, NT>& q, uint32_t from, int lane, float (&acc)[MT][NT][4]) {
  using P = Piece<X, GROUP, MT, NT>;
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int g = 0; g < P::kPerStep; ++g)
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint32_t w[2][P::kWords], z[2];
        float c[2], sum[NT][4] = {};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          lds(from + (16 * m + 8 * h + (lane >> 2)) * P::kPitch + 64 * s + (GROUP / 2) * g + (lane & 3) * (GROUP / 8), w[h]);
          z[h] = P::kPerStep == 1 ? q.zero[s][2 * m + h] : __shfl_sync(~0u, q.zero[s][2 * m + h], (lane & ~3) + g);
          c[h] = P::kPerStep == 1 ? q.scale[s][2 * m + h] : __shfl_sync(~0u, q.scale[s][2 * m + h], (lane & ~3) + g);
        }
#pragma unroll
        for (int i = 0; i < P::kWords; ++i) {
          uint32_t a[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h) nibble_pairs<X>(w[h][i], z[h], a[h]);
          const uint32_t a01[4] = {a[0][0], a[1][0], a[0][1], a[1][1]}, a23[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            const uint32_t* v = q.x[s][j][g * P::kWords + i];
            mma_pair(sum[j], a01, v[0], v[1], X());
            mma_pair(sum[j], a23, v[2], v[3], X());
          }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[m][j][i] = fmaf(c[i >> 1], sum[j][i], acc[m][j][i]);
      }
}

template <typename X, int GROUP, int MT, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 2 : 1) k_stream(const __grid_constant__ Params p) {
  constexpr int kRows = 16 * MT, kCols = 8 * NT, kPitch = Piece<X, GROUP, MT, NT>::kPitch;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ Ring ring;
  __shared__ float part[2][kWarps][kCols][kRows + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &ring.gave_up;
  auto full = [&](int s) { return smem_u32(&ring.full[s]); };
  auto empty = [&](int s) { return smem_u32(&ring.empty[s]); };
  const uint32_t base = smem_u32(smem);
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), kWarps);
    }
    ring.gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  const int64_t row_bytes = p.a.k / 2;
  int stage = 0;
  uint32_t phase = 0;
  if (warp == kWarps) {
    bool okay = true;
    uint32_t issued = 0;
    for (int64_t tile = blockIdx.x; tile < p.tiles && okay; tile += gridDim.x) {
      const int64_t n0 = tile * kRows;
      const int rows = static_cast<int>(min(static_cast<int64_t>(kRows), p.a.n - n0));
      const uint8_t* row = static_cast<const uint8_t*>(p.a.w) + (n0 + lane) * p.a.w_stride;
      for (int step = 0; step < p.steps; ++step) {
        const int64_t at = static_cast<int64_t>(step) * kStageBytes;
        const uint32_t bytes = static_cast<uint32_t>(min(static_cast<int64_t>(kStageBytes), row_bytes - at));
        if (!mbar_wait(empty(stage), phase ^ 1u, abort)) {  // the same for every lane but for its timing
          okay = false;
        }
        okay = __all_sync(~0u, okay);
        if (!okay) break;
        if (lane == 0) mbar_expect_tx(full(stage), bytes * rows);
        __syncwarp();
        if (lane < rows) bulk_load(base + stage * (kRows * kPitch) + lane * kPitch, row + at, bytes, full(stage));
        issued |= 1u << stage;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
    if (!okay && lane == 0) {
      // copies still in flight get a bounded time to land before their memory is given back
      for (int s = 0; s < p.stages; ++s)
        if (issued & (1u << s))
          for (uint32_t it = 0; it < (1u << 20); ++it)
            if (mbar_try_wait(full(s), 0) || mbar_try_wait(full(s), 1)) break;
      atomicOr(p.error_word, 1u);
    }
  } else {
    int turn = 0;
    Source<X, GROUP, MT, NT> source;
    source.set_x(p.a, lane);
    for (int64_t tile = blockIdx.x; tile < p.tiles; tile += gridDim.x) {
      const int64_t n0 = tile * kRows;
      source.set_tile(p.a, n0, lane);
      float acc[MT][NT][4] = {};
      for (int step = 0; step < p.steps; ++step) {
        const int k0 = (step * kStageBytes + warp * kPieceBytes) * 2;
        Piece<X, GROUP, MT, NT> piece;
        const bool any = k0 < source.k;  // uniform in the warp
        if (any) source.fetch(k0, lane, piece);
        mbar_wait(full(stage), phase, abort);  // after a wait that gave up the values are of no use, but every barrier is passed
        __syncwarp();
        if (any) {
          source.settle(piece);
          multiply(piece, base + stage * (kRows * kPitch) + warp * kPieceBytes, lane, acc);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty(stage));
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            part[turn][warp][8 * j + 2 * (lane & 3) + (i & 1)][16 * m + (lane >> 2) + 8 * (i >> 1)] = acc[m][j][i];
      asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory");
      const int cols = static_cast<int>(p.a.rows);
      for (int i = threadIdx.x; i < cols * kRows; i += 32 * kWarps) {
        const int c = i / kRows, r = i % kRows;
        float v = part[turn][0][c][r];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) v += part[turn][w][c][r];
        if (n0 + r < p.a.n) store_out(p.a.out, p.a.out_type, c * p.a.out_stride + n0 + r, v);
      }
      turn ^= 1;  // the next tile's partial sums go where nobody reads any more
    }
  }
}

template <typename X, int GROUP, int MT, int NT>
bool launch(Params p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kStage = 16 * MT * Piece<X, GROUP, MT, NT>::kPitch;
  p.tiles = (p.a.n + 16 * MT - 1) / (16 * MT);
  p.stages = kRingBytes<MT, NT> / kStage;
  if (p.stages > kMaxStages) p.stages = kMaxStages;
  const int64_t most = static_cast<int64_t>(dev.sms) * (NT == 1 ? 2 : 1);
  const int64_t ctas = p.tiles < most ? p.tiles : most;
  k_stream<X, GROUP, MT, NT><<<static_cast<unsigned int>(ctas), kThreads, p.stages * kStage, stream>>>(p);
  return true;
}
template <typename X, int GROUP, int MT, int NT>
bool set_attribute() {
  return cudaFuncSetAttribute(reinterpret_cast<const void*>(k_stream<X, GROUP, MT, NT>),
                              cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes<MT, NT>) == cudaSuccess;
}

// f<X, GROUP, MT, NT>() of a call's types and sizes.
template <typename X_, int GROUP_, int MT_, int NT_>
struct Choice {
  using X = X_;
  static constexpr int GROUP = GROUP_, MT = MT_, NT = NT_;
};
template <typename X, int GROUP, typename F>
bool choose_tile(bool tall, bool two, F f) {
  if (tall) return two ? f(Choice<X, GROUP, 2, 2>()) : f(Choice<X, GROUP, 2, 1>());
  return two ? f(Choice<X, GROUP, 1, 2>()) : f(Choice<X, GROUP, 1, 1>());
}
template <typename X, typename F>
bool choose_group(int group, bool tall, bool two, F f) {
  if (group == 128) return choose_tile<X, 128>(tall, two, f);
  return group == 64 ? choose_tile<X, 64>(tall, two, f) : choose_tile<X, 32>(tall, two, f);
}

}  // namespace

bool stream_setup() {
  bool ok = true;
  auto set = [](auto c) {
    using C = decltype(c);
    return set_attribute<typename C::X, C::GROUP, C::MT, C::NT>();
  };
  for (int group : {32, 64, 128})
    for (bool tall : {false, true})
      for (bool two : {false, true})
        ok = ok && choose_group<__half>(group, tall, two, set) && choose_group<__nv_bfloat16>(group, tall, two, set);
  return ok;
}

bool stream_takes(const LinearArgs& a) {
  auto rows_ok = [](const void* p, int64_t rows, int64_t stride_bytes) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || stride_bytes % 16 == 0);
  };
  return a.kind == WeightKind::kU4 && a.rows <= 16 && a.k > 0 && a.k % 32 == 0 && rows_ok(a.x, a.rows, a.x_stride * 2) &&
         rows_ok(a.w, a.n, a.w_stride);
}

imd_status_t stream_launch(const LinearArgs& a, cudaStream_t stream) {
  const DeviceInfo* dev = device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  Params p{};
  p.a = a;
  p.error_word = dev->error_word;
  p.steps = static_cast<int32_t>((a.k / 2 + kStageBytes - 1) / kStageBytes);
  // 32 rows per tile share the loads of x; 16 where there would be too few tiles to occupy the SMs
  const bool tall = a.n >= static_cast<int64_t>(32) * 2 * dev->sms;
  auto go = [&](auto c) {
    using C = decltype(c);
    return launch<typename C::X, C::GROUP, C::MT, C::NT>(p, *dev, stream);
  };
  const bool ok = a.x_type == IMD_TYPE_F16 ? choose_group<__half>(a.group, tall, a.rows > 8, go)
                                           : choose_group<__nv_bfloat16>(a.group, tall, a.rows > 8, go);
  return cudaGetLastError() == cudaSuccess && ok ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace imd
