// 4-bit products with up to 16 rows of x in one pass over the weights; 17 to 32 rows in two where that is quicker (choice.hpp).
//
//   out[t, n] = sum_g ws[n, g] sum_{k in g} x[t, k] (w[n, k] - z[n, g])
//
// Bound by the issue and latency of the unpacking (18.7 instructions for 8 weights and lane, 11 of them the unpacking itself)
// at 16 warps per SM, well before HBM (n k / 2 bytes): 1 row x 28672 x 8192 34 us with groups of 128 (3.6 TB/s, 0.54 of the
// measured copy rate), 44 us with groups of 64 and zero points; 16 rows 61 and 67 us.
//
// A persistent CTA walks tiles of 16 MT rows of w; its eight warps take 256 k of every row (a piece) in turn. A warp has its
// own ring of pieces that arrive by TMA, one instruction each, so the bytes in flight depend on neither registers nor
// occupancy and a warp waits for nobody within a tile; at the end of a tile the warps' sums are folded in a fixed order. x,
// scales and zero points of the next piece are loaded to registers under the products of this one.
//
// Products are mma.sync of 16 rows of w by 8 rows of x. The order of k inside an instruction is free as long as
// both operands use the same one: a lane takes consecutive k of its quarter of a group with one load, and the words
// that an instruction wants are in its registers. See small.cu for how nibbles become exact 16-bit floats in
// pairs. Columns behind the last row of x repeat it and are not stored.
#include <cstdint>
#include <type_traits>

#include "cuda/sm100.cuh"
#include "dense.hpp"
#include "mma.cuh"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kPieceK = 256;               // k of a piece: 128 bytes of a row, one swizzle row
constexpr int kMaxSlots = 8;
// Two CTAs share an SM; with 9 to 16 rows of x their registers allow one.
template <int NT>
constexpr int kSmemPerCta = (NT == 1 ? 110 : 220) * 1024;
template <int MT, int NT>
constexpr int kRingBytes = kSmemPerCta<NT> - 4 * 2 * kWarps * 8 * NT * (16 * MT + 1) - 2048;  // beside the partial sums

struct Params {
  LinearArgs a;
  int32_t slots;   // pieces in flight per warp
  int32_t pieces;  // of a row
  int64_t tiles;
  unsigned int* error_word;
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

// What a call's types fix: GROUP k are one quad's share of a load, kPerStep groups make a step of 128 k, two steps
// a piece. LEAN: scales in x's type; ZEROS: zero points may be given (with
// LEAN: are given).
template <typename X_, int GROUP_, int MT_, int NT_, bool LEAN_, bool ZEROS_>
struct Choice {
  using X = X_;
  static constexpr int GROUP = GROUP_, MT = MT_, NT = NT_;
  static constexpr bool LEAN = LEAN_, ZEROS = ZEROS_;
  static constexpr int kPerStep = 128 / GROUP, kWords = GROUP / 32, kXWords = kPerStep * kWords;
};

// What a step needs beside the ring's bytes, as loaded.
template <typename C>
struct Raw {
  uint4 x[C::NT][C::kXWords];
  uint32_t scale[2 * C::MT], zero[2 * C::MT];  // lane l of a quad: group l mod kPerStep of the step
};
// The same as the products take it: pairs of x in the order of the nibbles, (0, 4), (1, 5), (2, 6), (3, 7).
template <typename C>
struct Ready {
  uint32_t x[C::NT][C::kXWords][4];
  float scale[2 * C::MT];
  uint32_t zero[2 * C::MT];
};

// This lane's rows of x and, per tile, of the scales and zero points.
template <typename C>
struct Source {
  const uint16_t* x[C::NT];
  const uint8_t *scale[2 * C::MT], *zero[2 * C::MT];
  int k, groups, scale_type;

  __device__ __forceinline__ Source(const LinearArgs& p, int lane) {
    k = static_cast<int>(p.k);
    groups = (k + C::GROUP - 1) / C::GROUP;
    scale_type = p.scale_type;
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
      x[j] = static_cast<const uint16_t*>(p.x) + min(static_cast<int64_t>(8 * j + (lane >> 2)), p.rows - 1) * p.x_stride +
             (lane & 3) * (C::GROUP / 4);
  }
  // The pointers are those of this lane's group of a step.
  __device__ __forceinline__ void set_tile(const LinearArgs& p, int64_t n0, int lane) {
    const int size = !C::LEAN && scale_type == IMD_TYPE_F32 ? 4 : 2, g = lane & (C::kPerStep - 1);
#pragma unroll
    for (int h = 0; h < 2 * C::MT; ++h) {
      const int64_t n = min(n0 + (lane >> 2) + 8 * h, p.n - 1);
      scale[h] = static_cast<const uint8_t*>(p.scale4) + (n * p.scale_stride + g) * size;
      if (C::ZEROS) zero[h] = p.zeros == nullptr ? nullptr : p.zeros + n * p.zeros_stride + g;
    }
  }
  template <bool TAIL>
  __device__ __forceinline__ void fetch_step(int k0, int lane, Raw<C>& q) const {
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int i = 0; i < C::kXWords; ++i) {
        const int place = C::GROUP * (i / C::kWords) + 8 * (i % C::kWords), at = k0 + (lane & 3) * (C::GROUP / 4) + place;
        if (!TAIL || at + 8 <= k) {
          q.x[j][i] = __ldg(reinterpret_cast<const uint4*>(x[j] + k0 + place));
        } else {
          uint32_t v[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[c] = 0;
            if (at + 2 * c < k) v[c] = x[j][k0 + place + 2 * c];
            if (at + 2 * c + 1 < k) v[c] |= static_cast<uint32_t>(x[j][k0 + place + 2 * c + 1]) << 16;
          }
          q.x[j][i] = make_uint4(v[0], v[1], v[2], v[3]);
        }
      }
    const int g = k0 / C::GROUP;
    const bool inside = !TAIL || g + (lane & (C::kPerStep - 1)) < groups;
#pragma unroll
    for (int h = 0; h < 2 * C::MT; ++h) {
      q.scale[h] = q.zero[h] = 0;
      if (!inside) continue;
      if (!C::LEAN && scale_type == IMD_TYPE_F32) q.scale[h] = __ldg(reinterpret_cast<const uint32_t*>(scale[h]) + g);
      else q.scale[h] = __ldg(reinterpret_cast<const uint16_t*>(scale[h]) + g);
      if (C::ZEROS) q.zero[h] = zero[h] == nullptr ? 8u : __ldg(zero[h] + g);
    }
  }
  __device__ __forceinline__ void fetch(int k0, int lane, Raw<C>& q) const {
    if (k0 + 128 <= k) fetch_step<false>(k0, lane, q);
    else fetch_step<true>(k0, lane, q);
  }
  __device__ __forceinline__ void settle(const Raw<C>& q, Ready<C>& r) const {
#pragma unroll
    for (int j = 0; j < C::NT; ++j)
#pragma unroll
      for (int i = 0; i < C::kXWords; ++i) {
        const uint4 v = q.x[j][i];
        r.x[j][i][0] = __byte_perm(v.x, v.z, 0x5410), r.x[j][i][1] = __byte_perm(v.x, v.z, 0x7632);
        r.x[j][i][2] = __byte_perm(v.y, v.w, 0x5410), r.x[j][i][3] = __byte_perm(v.y, v.w, 0x7632);
      }
#pragma unroll
    for (int h = 0; h < 2 * C::MT; ++h) {
      const uint32_t bits = q.scale[h];
      const float half = __half2float(__ushort_as_half(static_cast<unsigned short>(bits))), bf = __uint_as_float(bits << 16);
      if (C::LEAN) r.scale[h] = std::is_same<typename C::X, __half>::value ? half : bf;
      else r.scale[h] = scale_type == IMD_TYPE_F16 ? half : scale_type == IMD_TYPE_BF16 ? bf : __uint_as_float(bits);
      r.zero[h] = nibble_magic<typename C::X>() | (C::ZEROS ? (q.zero[h] & 15u) * 0x10001u : 0x80008u);
    }
  }
};

// One step of a tile: `row` is this lane's first row in the slot, `half` the step's 64 bytes of it.
template <typename C>
__device__ __forceinline__ void multiply(const Ready<C>& q, const Nibbles<typename C::X>& nibbles, uint32_t row, int half, int lane, float (&acc)[C::MT][C::NT][4]) {
  using X = typename C::X;
#pragma unroll
  for (int g = 0; g < C::kPerStep; ++g) {
    // bytes of this lane's quarter of the group; TMA exchanged the 16-byte pieces of a row by its number mod 8
    const int at = 64 * half + (C::GROUP / 2) * g + (lane & 3) * (C::GROUP / 8);
    const uint32_t from = row + ((((at >> 4) ^ (lane >> 2)) << 4) | (at & 15));
#pragma unroll
    for (int m = 0; m < C::MT; ++m) {
      uint32_t w[2][C::kWords], z[2];
      float c[2], sum[C::NT][4] = {};
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        lds(from + (16 * m + 8 * h) * 128, w[h]);
        z[h] = C::kPerStep == 1 || !C::ZEROS ? q.zero[2 * m + h] : __shfl_sync(~0u, q.zero[2 * m + h], (lane & ~3) + g);
        c[h] = C::kPerStep == 1 ? q.scale[2 * m + h] : __shfl_sync(~0u, q.scale[2 * m + h], (lane & ~3) + g);
      }
#pragma unroll
      for (int i = 0; i < C::kWords; ++i) {
        uint32_t a[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) nibbles.pairs(w[h][i], z[h], a[h]);
        const uint32_t a01[4] = {a[0][0], a[1][0], a[0][1], a[1][1]}, a23[4] = {a[0][2], a[1][2], a[0][3], a[1][3]};
#pragma unroll
        for (int j = 0; j < C::NT; ++j) {
          const uint32_t* v = q.x[j][g * C::kWords + i];
          mma_pair(sum[j], a01, v[0], v[1], X());
          mma_pair(sum[j], a23, v[2], v[3], X());
        }
      }
#pragma unroll
      for (int j = 0; j < C::NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[m][j][i] = fmaf(c[i >> 1], sum[j][i], acc[m][j][i]);
    }
  }
}

template <typename C>
__global__ void __launch_bounds__(kThreads, C::NT == 1 ? 2 : 1)
k_stream(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ Params p) {
  constexpr int MT = C::MT, NT = C::NT, kRows = 16 * MT, kCols = 8 * NT, kSlotBytes = kRows * 128;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ uint64_t bars[kWarps][kMaxSlots];
  __shared__ int gave_up;
  __shared__ float part[2][kWarps][kCols][kRows + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort = &gave_up;
  const uint32_t ring = ((smem_u32(smem) + 1023u) & ~1023u) + warp * p.slots * kSlotBytes;
  auto bar = [&](int s) { return smem_u32(&bars[warp][s]); };
  if (lane == 0) {
    for (int s = 0; s < p.slots; ++s) mbar_init(bar(s), 1);
    if (warp == 0) gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // the warp's pieces: warp, warp + 8, ... of each tile of the CTA
  const int mine = (p.pieces - warp + kWarps - 1) / kWarps, tiles = static_cast<int>(p.tiles);
  const uint64_t policy = l2_policy(2);  // weights pass through once
  int load_row = mine > 0 ? static_cast<int>(blockIdx.x) * kRows : tiles * kRows, load_step = 0;
  auto load = [&](int slot) {  // the next piece of the walk into `slot`, by one lane
    if (load_row >= tiles * kRows) return;
    if (lane == 0) {
      mbar_expect_tx(bar(slot), kSlotBytes);
      tma_load_3d(ring + slot * kSlotBytes, &map_w, bar(slot), (load_step * kWarps + warp) * (kPieceK / 2), load_row, 0, policy);
    }
    if (++load_step == mine) load_step = 0, load_row += gridDim.x * kRows;
  };
  for (int s = 0; s < p.slots; ++s) load(s);

  Source<C> source(p.a, lane);
  const Nibbles<typename C::X> nibbles;
  Raw<C> raw;
  const int k_first = warp * kPieceK;
  if (mine > 0 && blockIdx.x < p.tiles) {
    source.set_tile(p.a, static_cast<int64_t>(blockIdx.x) * kRows, lane);
    source.fetch(k_first, lane, raw);
  }
  int slot = 0, turn = 0;
  uint32_t phase = 0;
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t n0 = static_cast<int64_t>(tile) * kRows;
    float acc[MT][NT][4] = {};
    int k0 = k_first;
#pragma unroll 1
    for (int left = mine; left > 0; --left) {
      const uint32_t row = ring + slot * kSlotBytes + (lane >> 2) * 128;
      Ready<C> ready;
      source.settle(raw, ready);
      source.fetch(k0 + 128, lane, raw);
      // after a wait that gave up the values are of no use and nothing more is loaded, but every barrier is passed
      if (!mbar_wait(bar(slot), phase, abort)) load_row = tiles * kRows;
      __syncwarp();
      multiply<C>(ready, nibbles, row, 0, lane, acc);
      source.settle(raw, ready);
      k0 += kWarps * kPieceK;
      if (left > 1) {
        source.fetch(k0, lane, raw);
      } else if (tile + static_cast<int>(gridDim.x) < tiles) {
        source.set_tile(p.a, n0 + static_cast<int64_t>(gridDim.x) * kRows, lane);
        source.fetch(k_first, lane, raw);
      }
      multiply<C>(ready, nibbles, row, 1, lane, acc);
      __syncwarp();
      load(slot);
      if (++slot == p.slots) {
        slot = 0;
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
    __syncthreads();
    const int cols = static_cast<int>(p.a.rows);
    for (int i = threadIdx.x; i < cols * kRows; i += kThreads) {
      const int c = i / kRows, r = i % kRows;
      float v = part[turn][0][c][r];
#pragma unroll
      for (int w = 1; w < kWarps; ++w) v += part[turn][w][c][r];
      if (n0 + r < p.a.n) store_out(p.a.out, p.a.out_type, c * p.a.out_stride + n0 + r, v);
    }
    turn ^= 1;  // the next tile's partial sums go where nobody reads any more
  }
  if (*abort && lane == 0) {
    let_land_any(p.slots, bar);
    atomicOr(p.error_word, 1u);
  }
}

template <typename C>
bool launch(Params p, const DeviceInfo& dev, cudaStream_t stream) {
  constexpr int kSlot = 16 * C::MT * 128;
  p.tiles = (p.a.n + 16 * C::MT - 1) / (16 * C::MT);
  p.slots = (kRingBytes<C::MT, C::NT> - 1024) / (kWarps * kSlot);
  if (p.slots > kMaxSlots) p.slots = kMaxSlots;
  CUtensorMap map;
  if (!encode_rows_128(dev, &map, p.a.w, (p.a.k + 1) / 2, p.a.n, p.a.w_stride, 16 * C::MT)) return false;
  const int64_t most = static_cast<int64_t>(dev.sms) * (C::NT == 1 ? 2 : 1);
  const int64_t ctas = p.tiles < most ? p.tiles : most;
  k_stream<C><<<static_cast<unsigned int>(ctas), kThreads, p.slots * kWarps * kSlot + 1024, stream>>>(map, p);
  return true;
}

// f(Choice) of a call.
struct Call {
  bool f16, lean, zeros, tall, two;
  int group;
};
template <typename X, int GROUP, int MT, int NT, typename F>
bool choose_scales(const Call& c, F f) {
  if (!c.lean) return f(Choice<X, GROUP, MT, NT, false, true>());
  return c.zeros ? f(Choice<X, GROUP, MT, NT, true, true>()) : f(Choice<X, GROUP, MT, NT, true, false>());
}
template <typename X, int GROUP, typename F>
bool choose_tile(const Call& c, F f) {
  if (c.tall) return c.two ? choose_scales<X, GROUP, 2, 2>(c, f) : choose_scales<X, GROUP, 2, 1>(c, f);
  return c.two ? choose_scales<X, GROUP, 1, 2>(c, f) : choose_scales<X, GROUP, 1, 1>(c, f);
}
template <typename X, typename F>
bool choose_group(const Call& c, F f) {
  if (c.group == 128) return choose_tile<X, 128>(c, f);
  return c.group == 64 ? choose_tile<X, 64>(c, f) : choose_tile<X, 32>(c, f);
}
template <typename F>
bool choose(const Call& c, F f) {
  return c.f16 ? choose_group<__half>(c, f) : choose_group<__nv_bfloat16>(c, f);
}

}  // namespace

bool stream_setup() {
  bool ok = true;
  for (int i = 0; i < 32; ++i)
    for (int group : {32, 64, 128}) {
      const Call c{(i & 1) != 0, (i & 2) != 0, (i & 4) != 0, (i & 8) != 0, (i & 16) != 0, group};
      ok = ok && choose(c, [](auto choice) {
             using C = decltype(choice);
             return cudaFuncSetAttribute(reinterpret_cast<const void*>(k_stream<C>), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         kRingBytes<C::MT, C::NT>) == cudaSuccess;
           });
    }
  return ok;
}

imd_status_t stream_launch(const LinearArgs& all, cudaStream_t stream) {
  const DeviceInfo* dev = device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  const int64_t passes = (all.rows + kStreamPassRows - 1) / kStreamPassRows, share = (all.rows + passes - 1) / passes;
  for (int64_t t0 = 0; t0 < all.rows; t0 += share) {
    LinearArgs a = all;
    a.rows = all.rows - t0 < share ? all.rows - t0 : share;
    a.x = static_cast<const uint8_t*>(all.x) + 2 * t0 * all.x_stride;
    a.out = static_cast<uint8_t*>(all.out) + t0 * all.out_stride * (all.out_type == IMD_TYPE_F32 ? 4 : 2);
    Params p{};
    p.a = a;
    p.error_word = dev->error_word;
    p.pieces = static_cast<int32_t>((a.k + kPieceK - 1) / kPieceK);
    // 32 rows per tile share the loads of x; 16 where there would be too few tiles to occupy the SMs
    const bool tall = a.n >= kStreamTallN;
    const Call c{a.x_type == IMD_TYPE_F16, a.scale_type == a.x_type, a.zeros != nullptr, tall, a.rows > 8, a.group};
    if (!choose(c, [&](auto choice) { return launch<decltype(choice)>(p, *dev, stream); })) {
      cudaGetLastError();
      return IMD_STATUS_CUDA_ERROR;
    }
  }
  return cudaGetLastError() == cudaSuccess ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace imd
