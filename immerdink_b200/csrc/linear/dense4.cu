// 4-bit weights with many rows of x on the tensor cores:
//
//   out[t, n] = sum_g ws[n, g] sum_{k in g} x[t, k] (w[n, k] - z[n, g])
//
// The weights are the M side (128 rows per CTA), up to 256 rows of x the N side. w - z is a small integer
// and exact in x's 16-bit type, so the inner sum is an ordinary tcgen05.mma.kind::f16 with 32-bit
// accumulators; the scale would not be exact there. So a group's sum is one accumulator of its own (two
// in tensor memory, used in turn) and is added to registers as scale * sum while the next group is
// multiplied: no weight is ever rounded, for one multiply-add per output and group. A row of w is one
// lane of tensor memory, so its scale is one register.
//
// Warpgroups (512 threads, 128 registers each at launch, shared out again by setmaxnreg):
//   0     warp 0 brings x by TMA (64 k = 128 bytes of a row, 128-byte swizzle), warp 1 issues the MMAs, warp 2
//         brings the packed weights by TMA, 256 k (128 bytes of a row) at a time into two slots of their own
//         (rows that TMA cannot bring: x by warpgroups 2 and 3, each row's weights by the thread that unpacks it)
//   1     thread r turns row r of the weights' next 64 k into 16-bit floats in the swizzled layout
//   2, 3  halves of the rows of x: out += scale * accumulator, then the stores
// Bound by what the roles' own loops take at one to three warps per scheduler. A block of 64 k takes, at 33 and at 256 rows of x,
// 1050 and 1150 cycles with groups of 128 (the MMAs of 256 rows need 512; a second unpacking warpgroup changes nothing), 1190 and
// 1630 with groups of 64, 1920 and 2870 with two groups of 32, whose sums bound it at 950 to 1450 cycles a group. 28672 x 8192, g128: 141
// us at 33 rows, 154 at 256; 2048 x 8192 x 8192 304 us (0.55 of the measured bf16 rate), with groups of 64 433, of 32 762. Hence few and wide instructions a group: multiply-adds in pairs (316 against 304
// us), eight scales in one load. A cluster of up to 8 CTAs splits K (whole groups) where the row tiles
// alone would not fill the GPU; the parts are added through distributed shared memory in rank order.
// Every wait is bounded, as in the 8-bit kernels.
#include <cstdint>
#include <type_traits>

#include "cuda/sm100.cuh"
#include "dense.hpp"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kThreads = 512;
constexpr int kRegsLaunch = 128;                                   // 65536 / kThreads
// (56, 56, 200: no role spills; less for warpgroup 0 did)
constexpr int kRegsIssue = 56, kRegsUnpack = 56, kRegsSum = 200;  // per thread of warpgroup 0, 1, 2 and 3
static_assert(kRegsIssue + kRegsUnpack + 2 * kRegsSum <= 4 * kRegsLaunch, "register shares above the launch's total");
constexpr int kTileM = 128, kTileN = 256;
constexpr int kBlockK = 64;                                        // k of one pipeline stage: 128 bytes a row
constexpr int kBytesM = kTileM * 128;
constexpr int kMaxStages = 8;
constexpr int kCtrlBytes = 256;
constexpr int kSmem = 227 * 1024;
constexpr int kChunkBlocks = 4;                                    // 64-k blocks of one packed chunk
constexpr int kChunkBytes = kTileM * 128;

struct Params {
  LinearArgs a;
  int32_t units;                  // K in steps of max(group, 64)
  int32_t tiles_t, cols, stages;  // row tiles of x; rows of x per tile, padded to 16
  int32_t acc_cols;               // tensor-memory columns of one accumulator, a power of two
  int32_t wide;                   // rows of w are 16-byte aligned: they come by TMA
  int32_t scale_quad;             // 16-bit scales whose rows are whole 16-byte units
  int32_t out_wide;               // four neighbours of the output are aligned
  unsigned int* error_word;
};

template <typename X>
__device__ __forceinline__ void mma16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
      : "memory");
}
__device__ __forceinline__ void add_cluster(uint32_t addr, float (&v)[4]) {
  float u[4];
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(u[0]), "=f"(u[1]), "=f"(u[2]), "=f"(u[3])
               : "r"(addr)
               : "memory");
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] += u[i];
}
__device__ __forceinline__ void store4(float* to, const float (&v)[4]) {
  *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store4(__nv_bfloat16* to, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(to) = make_uint2(reinterpret_cast<const uint32_t&>(a), reinterpret_cast<const uint32_t&>(b));
}
__device__ __forceinline__ void store4(__half* to, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(to) = make_uint2(reinterpret_cast<const uint32_t&>(a), reinterpret_cast<const uint32_t&>(b));
}

// The tile's sums, in shared memory as 128 rows of w per row of x (in every CTA of the cluster), to the output: part r
// adds and stores rows r, r + parts, ... of x, in the order of the ranks; a warp stores a row of x at a time, a lane four
// neighbours of it. Rolled: the code of a tile's end runs once, from a cold instruction cache (each thread's 128 sums
// stored from registers, unrolled: 15 against 7 us at 128 x 128 x 128).
template <typename Out>
__device__ __forceinline__ void finish_tile(const Params& p, uint32_t sums, int64_t t0, int64_t n0, int part, int parts, int warp) {
  const int q = 4 * (threadIdx.x & 31), step = 8 * parts;
  const int last = static_cast<int>(min(static_cast<int64_t>(p.cols), p.a.rows - t0));
  const int valid = static_cast<int>(min(static_cast<int64_t>(4), p.a.n - n0 - q));
  if (valid <= 0) return;
  Out* out = static_cast<Out*>(p.a.out) + t0 * p.a.out_stride + n0 + q;
#pragma unroll 1
  for (int c = part + parts * warp; c < last; c += 4 * step) {
    float v[4][4] = {};
#pragma unroll 1
    for (int r = 0; r < parts; ++r) {
      const uint32_t base = map_to_cta(sums + q * 4, r);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (c + j * step < last) add_cluster(base + (c + j * step) * kTileM * 4, v[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j * step < last) {
        Out* to = out + static_cast<int64_t>(c + j * step) * p.a.out_stride;
        if (p.out_wide && valid == 4) {
          store4(to, v[j]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < valid) to[i] = Out(v[j][i]);
        }
      }
  }
}

// Scales of a row from group i on, as bits: eight 16-bit ones in a 16-byte load (quad) or up to four, one per word. Lanes hold
// different rows, so a load costs 32 lookups whatever its width: one load per group and warp took 270 cycles of the load unit
// a group (33 rows x 28672 x 8192, g64: 190 against 164 us). Predicated, so that no branch's end waits for the loads.
__device__ __forceinline__ void load_scales(const void* scales, bool quad, bool wide, int64_t i, int left, uint32_t (&v)[4]) {
  const uint8_t* at = static_cast<const uint8_t*>(scales) + (i << (wide ? 2 : 1));
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = 0;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %5, 0;\n\t@p ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3])
      : "l"(at), "r"(quad && left > 0 ? 1u : 0u));
#pragma unroll
  for (int j = 0; j < 4; ++j)
    asm volatile(
        "{\n\t.reg .pred a, b;\n\tsetp.ne.u32 a, %2, 0;\n\tsetp.ne.u32 b, %3, 0;\n\t@a ld.global.nc.u32 %0, [%1];\n\t"
        "@b ld.global.nc.u16 %0, [%1];\n\t}"
        : "+r"(v[j])
        : "l"(at + (j << (wide ? 2 : 1))), "r"(!quad && wide && j < left ? 1u : 0u), "r"(!quad && !wide && j < left ? 1u : 0u));
}
__device__ __forceinline__ float scale_value(int32_t type, uint32_t bits) {
  if (type == IMD_TYPE_F32) return __uint_as_float(bits);
  return type == IMD_TYPE_BF16 ? __uint_as_float(bits << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
}

template <typename X, int GROUP, bool ANY>
__global__ void __launch_bounds__(kThreads, 1)
k_dense4(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
         const __grid_constant__ Params p) {
  constexpr int kUnit = GROUP > kBlockK ? GROUP : kBlockK;       // k of one step of the split
  constexpr int kBlocks = kUnit / kBlockK, kGroups = kUnit / GROUP;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const int stage_bytes = kBytesM + p.cols * 128;
  const uint32_t packed = tiles + p.stages * stage_bytes;         // two chunks of packed weights
  uint8_t* ctrl = smem_raw + (packed - raw) + 2 * kChunkBytes;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 216);
  volatile int* abort = reinterpret_cast<volatile int*>(ctrl + 224);
  const uint32_t bar0 = smem_u32(ctrl);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto tfull = [&](int a) { return bar0 + 8u * (2 * kMaxStages + a); };
  auto tempty = [&](int a) { return bar0 + 8u * (2 * kMaxStages + 2 + a); };
  auto wfull = [&](int c) { return bar0 + 8u * (2 * kMaxStages + 4 + c); };
  auto wempty = [&](int c) { return bar0 + 8u * (2 * kMaxStages + 6 + c); };
  const uint32_t drain = bar0 + 8u * (2 * kMaxStages + 8);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, wg = warp >> 2;
  const int parts = gridDim.y, part = blockIdx.y;
  const int u0 = static_cast<int>(static_cast<int64_t>(p.units) * part / parts);
  const int u1 = static_cast<int>(static_cast<int64_t>(p.units) * (part + 1) / parts);
  const int64_t t0 = static_cast<int64_t>(blockIdx.x % p.tiles_t) * kTileN;
  const int64_t n0 = static_cast<int64_t>(blockIdx.x / p.tiles_t) * kTileM;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), (ANY ? 8 : 1) + 4);  // who brings x, and the four unpacking warps
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull(a), 1);
      mbar_init(tempty(a), 8);
      mbar_init(wfull(a), 1);
      mbar_init(wempty(a), 4);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * p.acc_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (wg == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsIssue));
    if (!ANY && warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      const uint64_t policy = l2_policy(1);  // x is read by every row tile of the weights
      for (int kb = u0 * kBlocks; kb < u1 * kBlocks; ++kb) {
        if (!mbar_wait(empty(stage), phase ^ 1u, abort)) break;
        mbar_expect_tx(full(stage), p.cols * 128);
        tma_load_3d(tiles + stage * stage_bytes + kBytesM, &map_x, full(stage), kb * 2 * kBlockK, static_cast<int>(t0), 0, policy);
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      let_land(issued, p.stages, full);
    } else if (warp == 1 && lane == 0) {
      constexpr uint32_t kType = std::is_same<X, __nv_bfloat16>::value ? 1u : 0u;
      const uint32_t idesc = (1u << 4) | (kType << 7) | (kType << 10) | (static_cast<uint32_t>(p.cols >> 3) << 17) |
                             (static_cast<uint32_t>(kTileM >> 4) << 24);
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool okay = true;
#pragma unroll 1
      for (int kb = u0 * kBlocks; kb < u1 * kBlocks && okay; ++kb) {
        if (!mbar_wait(full(stage), phase, abort)) break;
        tc_fence_after();
        const uint32_t a = tiles + stage * stage_bytes, b = a + kBytesM;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // 16 k = 32 bytes an instruction
          const int at = (kb % kBlocks) * kBlockK + 16 * i;  // place in the unit
          if (at % GROUP == 0) {
            if (!mbar_wait(tempty(acc), acc_phase ^ 1u, abort)) {
              okay = false;
              break;
            }
            tc_fence_after();
          }
          mma16<X>(tmem_base + acc * p.acc_cols, smem_desc(a + 32 * i), smem_desc(b + 32 * i), idesc, at % GROUP != 0);
          if ((at + 16) % GROUP == 0) {
            tc_commit(tfull(acc));
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
          }
        }
        if (okay) tc_commit(empty(stage));
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(drain);
      for (uint32_t it = 0; it < kSpinLimit; ++it)
        if (mbar_try_wait(drain, 0)) break;
    } else if (warp == 2 && lane == 0 && p.wide) {
      const uint64_t policy = l2_policy(0);
      const int chunks = ((u1 - u0) * kBlocks + kChunkBlocks - 1) / kChunkBlocks;
      int c = 0;
      for (; c < chunks; ++c) {
        const int slot = c & 1;
        if (!mbar_wait(wempty(slot), ((c >> 1) & 1) ^ 1u, abort)) break;
        mbar_expect_tx(wfull(slot), kChunkBytes);
        tma_load_3d(packed + slot * kChunkBytes, &map_w, wfull(slot), (u0 * kBlocks + c * kChunkBlocks) * (kBlockK / 2),
                    static_cast<int>(n0), 0, policy);
      }
      let_land(c, 2, wfull);
    }
    __syncwarp();
  } else if (wg == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsUnpack));
    const Nibbles<X> nibbles;
    const int r = threadIdx.x & 127;
    const int64_t row = min(n0 + r, p.a.n - 1);
    const uint8_t* w = static_cast<const uint8_t*>(p.a.w) + row * p.a.w_stride;
    const uint8_t* zeros = p.a.zeros == nullptr ? nullptr : p.a.zeros + row * p.a.zeros_stride;
    const int64_t end = (p.a.k + 1) / 2;
    const int groups = static_cast<int>((p.a.k + GROUP - 1) / GROUP);
    const Span span = span_of(p.a.w, p.a.n, p.a.w_stride, end);
    // a chunk's zero points (four bits each) and, for rows of any alignment, a block's weights are loaded one
    // step ahead
    constexpr int kZeros = kChunkBlocks * kBlockK / GROUP;
    uint32_t zero_next[kZeros];
    auto fetch_zeros = [&](int kb) {
      const int g0 = kb * kBlockK / GROUP;
#pragma unroll
      for (int i = 0; i < kZeros; ++i) zero_next[i] = zeros == nullptr ? 8u : g0 + i < groups ? zeros[g0 + i] : 0u;
    };
    const int kb0 = u0 * kBlocks, kb1 = u1 * kBlocks;
    const uint32_t own = packed + r * 128;  // this row in the packed chunks
    // rows of any alignment: each thread brings its own row's chunk to the place where TMA would put it
    auto fetch_row = [&](int kb, int slot) {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) {
        uint32_t q[4];
        load_bytes<16, false>(w, static_cast<int64_t>(kb) * (kBlockK / 2) + 16 * i, end, span, q);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(own + slot * kChunkBytes + ((i ^ (r & 7)) << 4)),
                     "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3])
                     : "memory");
      }
    };
    int stage = 0;
    uint32_t phase = 0, zero_bits = 0;
    fetch_zeros(kb0);
    if (!p.wide) fetch_row(kb0, 0);
    // Rolled, as are the other roles' loops: one warp of each scheduler runs this code, so what does not fit the
    // smallest instruction cache is fetched again at every turn.
#pragma unroll 1
    for (int kb = kb0; kb < kb1; ++kb) {
      const int b = (kb - kb0) % kChunkBlocks, c = (kb - kb0) / kChunkBlocks;
      if (b == 0) {
        zero_bits = 0;
#pragma unroll
        for (int i = 0; i < kZeros; ++i) zero_bits |= (zero_next[i] & 15u) << (4 * i);
        if (kb + kChunkBlocks < kb1) {
          fetch_zeros(kb + kChunkBlocks);
          if (!p.wide) fetch_row(kb + kChunkBlocks, (c + 1) & 1);
        }
        if (p.wide && !mbar_wait(wfull(c & 1), (c >> 1) & 1, abort)) break;
      }
      const uint32_t from = own + (c & 1) * kChunkBytes, dst = tiles + stage * stage_bytes + r * 128;
      uint32_t q[8];
#pragma unroll
      for (int i = 0; i < 8; i += 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(q[i]), "=r"(q[i + 1]), "=r"(q[i + 2]), "=r"(q[i + 3])
                     : "r"(from + (((2 * b + i / 4) ^ (r & 7)) << 4)));
      uint32_t zero[2];  // of the first and the second 32 k
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t v = (zero_bits >> (4 * ((b * kBlockK + 32 * h) / GROUP))) & 15u;
        zero[h] = nibble_magic<X>() | v | (v << 16);
      }
      if (!mbar_wait(empty(stage), phase ^ 1u, abort)) break;
#pragma unroll
      for (int i = 0; i < 8; ++i) {  // 16 bytes = 8 weights; the swizzle exchanges the pieces of a row by its number mod 8
        uint32_t o[4];
        nibbles.pairs(q[i], zero[i >> 2], o);
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst + ((i ^ (r & 7)) << 4)),
                     "r"(__byte_perm(o[0], o[1], 0x5410)), "r"(__byte_perm(o[2], o[3], 0x5410)),
                     "r"(__byte_perm(o[0], o[1], 0x7632)), "r"(__byte_perm(o[2], o[3], 0x7632))
                     : "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads through the async proxy
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(full(stage));
        if (p.wide && (b == kChunkBlocks - 1 || kb + 1 == kb1)) mbar_arrive(wempty(c & 1));
      }
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSum));
    const int quarter = warp & 3, row = quarter * 32 + lane;
    const int64_t n = n0 + row, nc = min(n, p.a.n - 1);
    const int half = (p.cols + 63) / 64 * 32;                     // columns of warpgroup 2
    const int c0 = wg == 2 ? 0 : half, width = wg == 2 ? half : max(p.cols - half, 0);
    const int groups = static_cast<int>((p.a.k + GROUP - 1) / GROUP);
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + c0;
    uint64_t sum[64];  // pairs
#pragma unroll
    for (int j = 0; j < 64; ++j) sum[j] = 0;
    int acc = 0;
    uint32_t acc_phase = 0;
    const int g1 = u1 * kGroups;
    // four or eight groups' scales are loaded as many groups ahead. The loop over the groups stays rolled: the roles' hot
    // loops share a small instruction cache (unrolled by four it was slower by 6 % at 2048 x 8192 x 8192)
    const int g0 = u0 * kGroups;
    const bool scale_wide = p.a.scale_type == IMD_TYPE_F32, quad = p.scale_quad && g0 % 8 == 0;
    const int ahead = quad ? 8 : 4;
    uint32_t scale[4], next[4];
    auto fetch_scales = [&](int g) { load_scales(p.a.scale4, quad, scale_wide, nc * p.a.scale_stride + g, groups - g, next); };
    fetch_scales(g0);
    // ANY: rows of x that TMA cannot bring. These warps bring them, as far ahead as the ring allows: a stage is free
    // once the group that used it is complete.
    const int blocks = (u1 - u0) * kBlocks;
    const Span span = span_of(p.a.x, p.a.rows, 2 * p.a.x_stride, 2 * p.a.k);
    int brought = 0, stage = 0;
    uint32_t phase = 0;
    auto bring = [&](int limit) {
#pragma unroll 1
      for (; brought < min(limit, blocks); ++brought) {
        if (!mbar_wait(empty(stage), phase ^ 1u, abort)) break;
        const int64_t at = static_cast<int64_t>(u0 * kBlocks + brought) * 2 * kBlockK;
#pragma unroll 1
        for (int r = warp - 8; r < p.cols; r += 64)
          bring_rows<8>(static_cast<const uint8_t*>(p.a.x), 2 * p.a.x_stride, p.a.rows, t0, r, 8, p.cols, at, 2 * p.a.k, span,
                        tiles + stage * stage_bytes + kBytesM);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(full(stage));
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
    };
    if (ANY) bring(p.stages);
#pragma unroll 1
    for (int g = g0; g < g1; ++g) {
      const int i = (g - g0) & (ahead - 1);
      if (i == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) scale[j] = next[j];
        fetch_scales(g + ahead);
      }
      const int word = quad ? i >> 1 : i;
      uint32_t bits = word == 0 ? scale[0] : word == 1 ? scale[1] : word == 2 ? scale[2] : scale[3];
      if (quad) bits = i & 1 ? bits >> 16 : bits & 0xFFFFu;
      const float s = scale_value(p.a.scale_type, bits);
      if (!mbar_wait(tfull(acc), acc_phase, abort)) break;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < 128; c += 32) {
        if (c < width) {  // uniform
          uint32_t v[32];
          tmem_load_32(taddr + acc * p.acc_cols + c, v);
#pragma unroll
          for (int j = 0; j < 32; j += 2)
            asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%1, %2};\n\tmov.b64 b, {%3, %3};\n\tfma.rn.f32x2 %0, a, b, %0;\n\t}"
                : "+l"(sum[(c + j) / 2])
                : "r"(v[j]), "r"(v[j + 1]), "r"(__float_as_uint(s)));
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty(acc));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
      if (ANY) bring((g + 1 - g0) / kGroups * kBlocks + p.stages);
    }
    __syncwarp();
    // the ring is free: the last group's accumulator was complete, so every operand had been read
#pragma unroll
    for (int j = 0; j < 128; ++j)
      if (j < width)
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(tiles + ((c0 + j) * kTileM + row) * 4),
                     "r"(static_cast<uint32_t>(sum[j / 2] >> (32 * (j & 1))))
                     : "memory");
    __syncwarp();
  }

  if (parts > 1) cluster_sync_all();
  if (wg >= 2) {
    if (parts == 1) asm volatile("bar.sync 1, 256;" ::: "memory");
    if (p.a.out_type == IMD_TYPE_F32)
      finish_tile<float>(p, tiles, t0, n0, part, parts, warp - 8);
    else if (p.a.out_type == IMD_TYPE_F16)
      finish_tile<__half>(p, tiles, t0, n0, part, parts, warp - 8);
    else
      finish_tile<__nv_bfloat16>(p, tiles, t0, n0, part, parts, warp - 8);
    __syncwarp();
  }
  if (parts > 1) cluster_sync_all();  // the peers have read this CTA's sums
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicOr(p.error_word, 1u);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * p.acc_cols) : "memory");
  }
}

using Kernel = void (*)(const CUtensorMap, const CUtensorMap, const Params);
template <typename X>
Kernel kernel_of(int group, bool any) {
  if (any) return group == 128 ? k_dense4<X, 128, true> : group == 64 ? k_dense4<X, 64, true> : k_dense4<X, 32, true>;
  return group == 128 ? k_dense4<X, 128, false> : group == 64 ? k_dense4<X, 64, false> : k_dense4<X, 32, false>;
}

}  // namespace

// The shares above are drawn from the registers of the launch, so a kernel compiled for fewer is refused.
bool dense4_setup() {
  for (int group : {32, 64, 128})
    for (Kernel k : {kernel_of<__half>(group, false), kernel_of<__nv_bfloat16>(group, false), kernel_of<__half>(group, true),
                     kernel_of<__nv_bfloat16>(group, true)}) {
      cudaFuncAttributes attr;
      const void* f = reinterpret_cast<const void*>(k);
      if (cudaFuncGetAttributes(&attr, f) != cudaSuccess || attr.numRegs < kRegsLaunch ||
          cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess)
        return false;
    }
  return true;
}

bool dense4_clusters(int sms, int* clusters) {  // any kernel whose shared memory leaves room for one CTA
  for (int i = 0; i < 4; ++i) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned int>(sms), 1u << i);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmem;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim = {1, 1u << i, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters[i], kernel_of<__half>(128, false), &cfg) != cudaSuccess) return false;
  }
  return true;
}

imd_status_t dense4_launch(const LinearArgs& a, cudaStream_t stream) {
  const DeviceInfo* dev = device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  Params p{};
  p.a = a;
  const int unit = a.group > kBlockK ? a.group : kBlockK;
  p.units = static_cast<int32_t>((a.k + unit - 1) / unit);
  p.tiles_t = static_cast<int32_t>((a.rows + kTileN - 1) / kTileN);
  p.cols = a.rows < kTileN ? static_cast<int32_t>((a.rows + 15) / 16 * 16) : kTileN;
  p.acc_cols = 32;
  while (p.acc_cols < p.cols) p.acc_cols *= 2;
  p.wide = w4_for_tma(a);
  const int64_t groups = (a.k + a.group - 1) / a.group;
  p.scale_quad = a.scale_type != IMD_TYPE_F32 && groups % 8 == 0 && reinterpret_cast<uintptr_t>(a.scale4) % 16 == 0 &&
                 (a.n == 1 || a.scale_stride % 8 == 0);
  const int size = a.out_type == IMD_TYPE_F32 ? 4 : 2;
  p.out_wide = reinterpret_cast<uintptr_t>(a.out) % (4 * size) == 0 && (a.rows == 1 || a.out_stride % 4 == 0);
  p.error_word = dev->error_word;
  const int stage_bytes = kBytesM + p.cols * 128;
  p.stages = (kSmem - 1024 - kCtrlBytes - 2 * kChunkBytes) / stage_bytes;
  if (p.stages > kMaxStages) p.stages = kMaxStages;

  // the swizzle goes by bytes, so x is described as bytes too
  const bool any = !x4_for_tma(a);
  CUtensorMap map_x{}, map_w{};
  if ((!any && !encode_rows_128(*dev, &map_x, a.x, 2 * a.k, a.rows, 2 * a.x_stride, p.cols)) ||
      (p.wide && !encode_rows_128(*dev, &map_w, a.w, (a.k + 1) / 2, a.n, a.w_stride, kTileM)))
    return IMD_STATUS_CUDA_ERROR;

  const int64_t tiles = (a.n + kTileM - 1) / kTileM * p.tiles_t;
  if (tiles >= (INT64_C(1) << 31)) return IMD_STATUS_NOT_SUPPORTED;
  const int parts = split_of(tiles, p.units, dev->clusters, 1);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned int>(tiles), static_cast<unsigned int>(parts));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.stages) * stage_bytes + 2 * kChunkBytes + 1024 + kCtrlBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {1, static_cast<unsigned int>(parts), 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const Kernel k = a.x_type == IMD_TYPE_F16 ? kernel_of<__half>(a.group, any) : kernel_of<__nv_bfloat16>(a.group, any);
  const bool ok = cudaLaunchKernelEx(&cfg, k, map_x, map_w, p) == cudaSuccess;
  return cudaGetLastError() == cudaSuccess && ok ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace imd
