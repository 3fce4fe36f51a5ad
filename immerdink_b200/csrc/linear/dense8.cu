// 8-bit products with many rows on the tensor cores:
//
//   out[t, n] = xs[t] ws[n] sum_k x[t, k] w[n, k]         int8: exact int32 sums; e4m3: 32-bit float sums
//
// Bound by the tensor pipe once both operands have a few hundred rows (int8 8192^3 335 to 350 us in a short run of calls, 3100 to 3300
// T/s; 400 us, 2750 T/s, in a long one, under the power cap), by the weights' bytes below (e4m3 48 x 28672 x 8192 42 us, 5.7
// TB/s, 0.87 of the measured copy rate; 1 row 41 us). Between, 129 to 256 rows leave one CTA on an SM, whose tiles may fill their
// rounds badly: 256 x 28672 x 8192 has 224 of them on 148 SMs, two rounds for the work of 1.5 (62 us for 37).
// Two kernels share the pipeline of the contraction's GEMM (TMA into a ring of 128-byte K blocks with the
// 128-byte swizzle, one thread issuing tcgen05.mma, accumulators in tensor memory):
//
//   k_dense8_pair   CTA pairs, 256 rows of x by BN rows of w per tile, persistent, two accumulators so that
//                   the epilogue of a tile runs under the main loop of the next
//   k_dense8_swap   up to 256 rows of x: the weights are the M side (128 of their rows per CTA, whatever
//                   the rows of x), all rows of x the N side, so no tensor work is spent on padding and the
//                   weights pass through once. A cluster of up to 8 CTAs splits K where the row tiles alone
//                   would not fill the GPU; the parts are added through distributed shared memory in the
//                   order of the ranks, so results do not depend on timing and no workspace is needed.
//
// Every wait is bounded: one that gives up sets the device error word, the roles drain and the CTA ends.
#include <cstdint>
#include <type_traits>

#include "cuda/sm100.cuh"
#include "dense.hpp"
#include "types.cuh"

namespace imd {
namespace {

constexpr int kThreads = 320;       // warp 0 TMA, warp 1 MMA, warps 2-9 epilogue
constexpr int kTileM = 128;         // rows of one CTA's accumulator
constexpr int kTileK = 128;         // bytes of K per pipeline stage = one swizzle row
constexpr int kMmaK = 32;
constexpr int kBytesM = kTileM * kTileK;
constexpr int kCtrlBytes = 256;     // barriers, tensor-memory address, abort flag

struct Params {
  int32_t rows, n, k_blocks;
  int32_t tiles_m, tiles_n, band_rows;  // pair kernel
  int32_t cols, stages, tmem_cols;      // swap kernel: rows of x padded to 16, ring depth
  const float *x_scale, *w_scale;
  void* out;
  int64_t out_stride;
  int32_t out_type, out_wide;           // out_wide: 16-byte stores are aligned
  unsigned int* error_word;
  const uint8_t *x, *w;                 // rows of any alignment: where they are
  int64_t x_stride, w_stride, k;
};

// Instruction descriptor: D s32 (2) with A = B = s8 (1), or D f32 (1) with A = B = e4m3 (0); both K-major.
template <bool I8>
__host__ __device__ constexpr uint32_t instr_desc(int m, int n) {
  return ((I8 ? 2u : 1u) << 4) | ((I8 ? 1u : 0u) << 7) | ((I8 ? 1u : 0u) << 10) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}
template <bool I8, bool PAIR>
__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  const uint32_t acc = add ? 1u : 0u;
#define IMD_MMA8(GROUP, KIND)                                                              \
  asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"                           \
               "tcgen05.mma.cta_group::" GROUP ".kind::" KIND " [%0], %1, %2, %3, p;\n\t}" \
               ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)                              \
               : "memory")
  if constexpr (PAIR && I8) IMD_MMA8("2", "i8");
  else if constexpr (PAIR) IMD_MMA8("2", "f8f6f4");
  else if constexpr (I8) IMD_MMA8("1", "i8");
  else IMD_MMA8("1", "f8f6f4");
#undef IMD_MMA8
}

template <bool I8>
__device__ __forceinline__ float acc_value(uint32_t v) {
  return I8 ? static_cast<float>(static_cast<int32_t>(v)) : __uint_as_float(v);
}

// 32 columns of a warp's 32 rows (lane = row) to output rows, by way of shared memory: 64 bytes of each row at a time
// (pitch 80 bytes: no bank conflicts), so that a store covers neighbours. WIDE: 16-byte units, 64 bytes of 8 rows a
// store instead of 16 bytes of 32. Otherwise rows that start anywhere and the columns of the last tile, an element per
// lane. `at` is the element of lane 0's row; `rows` and `cols` how many of the block exist.
template <bool I8, typename T, bool WIDE>
__device__ __forceinline__ void store_block(const Params& p, int64_t at, int rows, int cols, const uint32_t* v, float xs,
                                            const float* ws, uint8_t* turn, int lane) {
  constexpr int kCols = 64 / sizeof(T), V = 16 / sizeof(T);
#pragma unroll
  for (int h = 0; h < 32; h += kCols) {
#pragma unroll
    for (int c = 0; c < kCols; c += V) {
      Pack<T, V> o;
#pragma unroll
      for (int j = 0; j < V; ++j) o.v[j] = from_float<T>(acc_value<I8>(v[h + c + j]) * xs * ws[h + c + j]);
      *reinterpret_cast<uint4*>(turn + lane * 80 + c * sizeof(T)) = *reinterpret_cast<const uint4*>(&o);
    }
    __syncwarp();
    if (WIDE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 8 * i + (lane >> 2);
        if (r < rows)
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + at + r * p.out_stride + h + (lane & 3) * V) =
              *reinterpret_cast<const uint4*>(turn + r * 80 + (lane & 3) * 16);
      }
    } else {
      constexpr int kRowsAtOnce = 32 / kCols;  // of a store
      const int c = lane % kCols, r0 = lane / kCols, last = h + c < cols ? rows : 0;
      T* out = static_cast<T*>(p.out) + at + r0 * p.out_stride + h + c;
      const T* from = reinterpret_cast<const T*>(turn + r0 * 80) + c;
#pragma unroll
      for (int r = 0; r < 32; r += kRowsAtOnce, out += kRowsAtOnce * p.out_stride)
        if (r0 + r < last) *out = from[r * (80 / sizeof(T))];
    }
    __syncwarp();
  }
}
template <bool I8, typename T>
__device__ __forceinline__ void store_block(const Params& p, int64_t at, int rows, int cols, const uint32_t* v, float xs,
                                            const float* ws, uint8_t* turn, int lane) {
  if (p.out_wide && cols >= 32) store_block<I8, T, true>(p, at, rows, cols, v, xs, ws, turn, lane);
  else store_block<I8, T, false>(p, at, rows, cols, v, xs, ws, turn, lane);
}

// ---- many rows: CTA pairs ------------------------------------------------------------------------------
// Signals as in the contraction's pair kernel: full[s] in the leader, armed with the bytes of both CTAs;
// empty[s] and tfull[a] by commits that reach both CTAs; tempty[a] in the leader, the sixteen epilogue
// warps of both.
constexpr int kTurnBytes = 32 * 80;  // a warp's block on its way to stores along the rows
template <int BN>
constexpr int kPairStageBytes = kBytesM + BN / 2 * kTileK;
template <int BN>
constexpr int kPairStages = BN == 256 ? 6 : 8;
template <int BN>
constexpr int kPairSmem = kPairStages<BN> * kPairStageBytes<BN> + 1024 + kCtrlBytes + 8 * kTurnBytes + 2 * BN * 4;

__device__ __forceinline__ void pair_tile(const Params& p, int w, int* tm, int* tn) {
  const int band = p.band_rows * p.tiles_n;
  const int first = (w / band) * p.band_rows;
  const int rows = min(p.tiles_m - first, p.band_rows);
  const int r = w % band;
  *tm = first + r % rows;
  *tn = r / rows;
}

template <bool I8, int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
k_dense8_pair(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
              const __grid_constant__ Params p) {
  constexpr int kStages = kPairStages<BN>, kStageBytes = kPairStageBytes<BN>;
  constexpr uint32_t kDesc = instr_desc<I8>(256, BN);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  uint8_t* ctrl = smem_raw + (tiles - raw) + kStages * kStageBytes;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 200);
  volatile int* abort = reinterpret_cast<volatile int*>(ctrl + 208);
  const uint32_t bar0 = smem_u32(ctrl);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kStages + s); };
  auto tfull = [&](int a) { return bar0 + 8u * (2 * kStages + a); };
  auto tempty = [&](int a) { return bar0 + 8u * (2 * kStages + 2 + a); };
  const uint32_t drain = bar0 + 8u * (2 * kStages + 4);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(tfull(a), 1);
      mbar_init(tempty(a), 16);
    }
    mbar_init(drain, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(2 * BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  const int total = p.tiles_m * p.tiles_n;
  const int first = blockIdx.x >> 1, step = gridDim.x >> 1;
  const uint32_t peer_abort = map_to_cta(smem_u32(const_cast<int*>(abort)), rank ^ 1u);
  auto tell_peer = [&]() { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(peer_abort), "r"(1u) : "memory"); };
  bool gave_up = false;  // of an epilogue warp

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      bool okay = true;
      const uint64_t policy = l2_policy(0);
      for (int w = first; w < total && okay; w += step) {
        int tm, tn;
        pair_tile(p, w, &tm, &tn);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(empty(stage), phase ^ 1u, abort)) {
            okay = false;
            tell_peer();
            break;
          }
          const uint32_t leader_full = map_to_cta(full(stage), 0);
          if (leader) mbar_expect_tx(full(stage), 2 * kStageBytes);
          const uint32_t dst = tiles + stage * kStageBytes;
          tma_load_3d_pair(dst, &map_x, leader_full, kb * kTileK, tm * 256 + static_cast<int>(rank) * 128, 0, policy);
          tma_load_3d_pair(dst + kBytesM, &map_w, leader_full, kb * kTileK,
                           tn * BN + static_cast<int>(rank) * (BN / 2), 0, policy);
          ++issued;
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      let_land_pair(leader, !okay, issued, kStages, full);  // then the pair's last cluster barrier
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool okay = true;
      for (int w = first; w < total && okay; w += step) {
        if (!mbar_wait(tempty(acc), acc_phase ^ 1u, abort)) {
          tell_peer();
          break;
        }
        tc_fence_after();
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(full(stage), phase, abort)) {
            okay = false;
            tell_peer();
            break;
          }
          tc_fence_after();
          const uint32_t a = tiles + stage * kStageBytes, b = a + kBytesM;
#pragma unroll
          for (int i = 0; i < kTileK / kMmaK; ++i)
            mma8<I8, true>(tmem_base + acc * BN, smem_desc(a + i * kMmaK), smem_desc(b + i * kMmaK), kDesc, (kb | i) != 0);
          tc_commit_pair(empty(stage));
          if (++stage == kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!okay) break;
        tc_commit_pair(tfull(acc));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      tc_commit_pair(drain, 1);
      for (uint32_t it = 0; it < kSpinLimit; ++it)
        if (mbar_try_wait(drain, 0)) break;
    }
  } else {
    // two warps per quarter of the tensor memory's lanes take the columns by turns of 32
    const int quarter = warp & 3, first_col = warp < 6 ? 0 : 32, id = static_cast<int>(threadIdx.x) - 64;
    uint8_t* turn = ctrl + kCtrlBytes + (warp - 2) * kTurnBytes;
    float* scales = reinterpret_cast<float*>(ctrl + kCtrlBytes + 8 * kTurnBytes);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int w = first; w < total; w += step) {
      int tm, tn;
      pair_tile(p, w, &tm, &tn);
      // the columns' scales to shared memory, in the half that the tile before last used
      float* ws = scales + acc * BN;
      if (id < BN) ws[id] = tn * BN + id < p.n ? p.w_scale[tn * BN + id] : 0.0f;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      if (!mbar_wait(tfull(acc), acc_phase, abort)) {
        if (lane == 0) tell_peer();
        // the other warps of the CTA give up at their own wait: every one of them passes the barrier above
        gave_up = true;
      }
      __syncwarp();
      tc_fence_after();
      const int row = tm * 256 + static_cast<int>(rank) * 128 + quarter * 32 + lane;
      const float xs = row < p.rows ? p.x_scale[row] : 0.0f;
      const uint32_t taddr = tmem_base + acc * BN + (static_cast<uint32_t>(quarter * 32) << 16);
#pragma unroll 1
      for (int cc = first_col; cc < BN && !gave_up; cc += 64) {
        const int col = tn * BN + cc;
        if (col >= p.n) break;  // the same for the whole warp
        uint32_t v[32];
        tmem_load_32(taddr + cc, v);
        const int64_t at = static_cast<int64_t>(row - lane) * p.out_stride + col;
        const int rows = p.rows - (row - lane), cols = p.n - col;
        if (p.out_type == IMD_TYPE_F32) store_block<I8, float>(p, at, rows, cols, v, xs, ws + cc, turn, lane);
        else if (p.out_type == IMD_TYPE_F16) store_block<I8, __half>(p, at, rows, cols, v, xs, ws + cc, turn, lane);
        else store_block<I8, __nv_bfloat16>(p, at, rows, cols, v, xs, ws + cc, turn, lane);
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(map_to_cta(tempty(acc), 0));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  tc_fence_before();
  cluster_sync_all();  // no CTA leaves while its peer may still signal it or write its tensor memory
  if (threadIdx.x == 0 && *abort) atomicOr(p.error_word, 1u);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2 * BN) : "memory");
  }
}

// ---- up to 256 rows: weights on the M side ---------------------------------------------------------------
constexpr int kSwapMaxStages = 12;
// Two CTAs of an SM take turns (one stores while the other loads) as long as their rings stay deep enough (up to kSwapColsHalf
// rows of x) and their registers allow it (checked below); bringing rows of any alignment takes more than half of them.
template <bool ANY>
constexpr int kSwapCtas = ANY ? 1 : 2;

__device__ __forceinline__ uint32_t load_cluster(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

// Accumulators to outputs. Warps 2-9: two per quarter of the tensor memory's lanes (= rows of w), which take the
// columns (= rows of x) by turns of 32. A warp's stores are 32 neighbours of one output row.
template <bool I8, typename T>
__device__ __forceinline__ void swap_epilogue(const Params& p, uint32_t tmem_base, uint32_t tiles, const float* x_scale, int n0,
                                              int part, int parts) {
  const int warp = threadIdx.x >> 5, quarter = warp & 3, turn = warp < 6 ? 0 : 1;
  const int row = quarter * 32 + static_cast<int>(threadIdx.x & 31);
  const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
  const bool inside = n0 + row < p.n;
  const float ws = inside ? p.w_scale[n0 + row] : 0.0f;
  T* out = static_cast<T*>(p.out) + n0 + row;
  if (parts == 1) {
    if (warp >= 2) {
#pragma unroll 1
      for (int c = 32 * turn; c < p.cols; c += 64) {
        uint32_t v[32];
        tmem_load_32(taddr + c, v);
        if (inside) {
          T* o = out + c * p.out_stride;
#pragma unroll
          for (int j = 0; j < 32; ++j, o += p.out_stride)
            if (c + j < p.rows) *o = from_float<T>(acc_value<I8>(v[j]) * x_scale[c + j] * ws);
        }
        __syncwarp();
      }
    }
    return;
  }
  // every column's partial sums fit the ring's memory: 512 bytes a column, and a stage has 128 of them and 16 KB
  if (warp >= 2) {
    for (int c = 32 * turn; c < p.cols; c += 64) {
      uint32_t v[32];
      tmem_load_32(taddr + c, v);
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (c + j < p.cols)
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(tiles + ((c + j) * kTileM + row) * 4), "r"(v[j]) : "memory");
    }
  }
  __syncwarp();
  cluster_sync_all();
  // part r adds columns r, r + parts, ..., eight at a time so that the remote loads overlap
  if (warp >= 2 && inside) {
    const int step = 2 * parts;
    for (int c = part + parts * turn; c < p.rows; c += 8 * step) {
      uint32_t v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0;  // also 0.0f
      for (int r = 0; r < parts; ++r) {
        const uint32_t base = map_to_cta(tiles + row * 4, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int cj = c + j * step;
          const uint32_t u = cj < p.rows ? load_cluster(base + cj * kTileM * 4) : 0u;
          v[j] = I8 ? v[j] + u : __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(u));
        }
      }
      T* o = out + c * p.out_stride;
#pragma unroll
      for (int j = 0; j < 8; ++j, o += step * p.out_stride)
        if (c + j * step < p.rows) *o = from_float<T>(acc_value<I8>(v[j]) * x_scale[c + j * step] * ws);
    }
  }
  __syncwarp();
  cluster_sync_all();  // the peers have read this CTA's columns
}

// ANY: rows that TMA cannot bring. The epilogue's warps, idle until the sums are complete, bring the operands'
// next 128 bytes per row instead, row by row.
template <bool I8, bool ANY>
__global__ void __launch_bounds__(kThreads)
k_dense8_swap(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x,
              const __grid_constant__ Params call) {
  Params p = call;
  if (ANY) {  // a tile of the rows of x per z
    const int64_t t0 = static_cast<int64_t>(blockIdx.z) * p.cols;
    p.x += t0 * p.x_stride;
    p.x_scale += t0;
    p.out = static_cast<uint8_t*>(p.out) + t0 * p.out_stride * (p.out_type == IMD_TYPE_F32 ? 4 : 2);
    p.rows = min(p.cols, static_cast<int32_t>(p.rows - t0));
  }
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t tiles = (raw + 1023u) & ~1023u;
  const int stage_bytes = kBytesM + p.cols * kTileK;  // a multiple of 2048
  uint8_t* ctrl = smem_raw + (tiles - raw) + p.stages * stage_bytes;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(ctrl + 216);
  volatile int* abort = reinterpret_cast<volatile int*>(ctrl + 224);
  const uint32_t bar0 = smem_u32(ctrl);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kSwapMaxStages + s); };
  const uint32_t done = bar0 + 8u * (2 * kSwapMaxStages);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = gridDim.y, part = blockIdx.y;  // the cluster spans y: its rank is the part of K
  const int kb0 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * part / parts);
  const int kb1 = static_cast<int>(static_cast<int64_t>(p.k_blocks) * (part + 1) / parts);
  const int n0 = blockIdx.x * kTileM;
  __shared__ float x_scale[256];
  for (int i = threadIdx.x; i < p.cols; i += kThreads) x_scale[i] = i < p.rows ? p.x_scale[i] : 0.0f;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full(s), ANY ? 8 : 1);
      mbar_init(empty(s), 1);
    }
    mbar_init(done, 1);
    *abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                 "r"(p.tmem_cols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;

  if (ANY && warp >= 2) {
    const Span span_w = span_of(p.w, p.n, p.w_stride, p.k), span_x = span_of(p.x, p.rows, p.x_stride, p.k);
    int stage = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait(empty(stage), phase ^ 1u, abort)) break;
      const uint32_t dst = tiles + stage * stage_bytes;
      const int64_t at = static_cast<int64_t>(kb) * kTileK;
      bring_rows<16>(p.w, p.w_stride, p.n, n0, warp - 2, 8, kTileM, at, p.k, span_w, dst);
      for (int r = 0; r < p.cols; r += 128)
        bring_rows<16>(p.x, p.x_stride, p.rows, 0, r + warp - 2, 8, p.cols, at, p.k, span_x, dst + kBytesM);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the tensor core reads through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(full(stage));
      if (++stage == p.stages) {
        stage = 0;
        phase ^= 1u;
      }
    }
    __syncwarp();
  } else if (!ANY && warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0;
      const uint64_t policy_w = l2_policy(2), policy_x = l2_policy(1);  // weights stream through, x stays
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty(stage), phase ^ 1u, abort)) break;
        mbar_expect_tx(full(stage), stage_bytes);
        const uint32_t dst = tiles + stage * stage_bytes;
        tma_load_3d(dst, &map_w, full(stage), kb * kTileK, n0, 0, policy_w);
        tma_load_3d(dst + kBytesM, &map_x, full(stage), kb * kTileK, 0, 0, policy_x);
        ++issued;
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      let_land(issued, p.stages, full);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = instr_desc<I8>(kTileM, p.cols);
      int stage = 0;
      uint32_t phase = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full(stage), phase, abort)) break;
        tc_fence_after();
        const uint32_t a = tiles + stage * stage_bytes, b = a + kBytesM;
#pragma unroll
        for (int i = 0; i < kTileK / kMmaK; ++i)
          mma8<I8, false>(tmem_base, smem_desc(a + i * kMmaK), smem_desc(b + i * kMmaK), idesc, kb != kb0 || i != 0);
        tc_commit(empty(stage));
        if (++stage == p.stages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      tc_commit(done);  // arrives once every instruction issued above has retired
    }
  }
  // every thread waits for the accumulator; the ring's memory is free for the fold after that
  __syncwarp();
  mbar_wait(done, 0, abort);
  tc_fence_after();
  __syncthreads();

  if (p.out_type == IMD_TYPE_F32) swap_epilogue<I8, float>(p, tmem_base, tiles, x_scale, n0, part, parts);
  else if (p.out_type == IMD_TYPE_F16) swap_epilogue<I8, __half>(p, tmem_base, tiles, x_scale, n0, part, parts);
  else swap_epilogue<I8, __nv_bfloat16>(p, tmem_base, tiles, x_scale, n0, part, parts);
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && *abort) atomicOr(p.error_word, 1u);
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(p.tmem_cols) : "memory");
  }
}

constexpr int kSwapSmem = 200 * 1024, kSwapSmemHalf = 110 * 1024, kSwapColsHalf = 128;

template <bool I8, int BN>
bool launch_pair(const LinearArgs& a, const DeviceInfo& dev, Params p, cudaStream_t stream) {
  CUtensorMap mx, mw;
  if (!encode_rows_128(dev, &mx, a.x, a.k, a.rows, a.x_stride, 128) ||
      !encode_rows_128(dev, &mw, a.w, a.k, a.n, a.w_stride, BN / 2))
    return false;
  p.tiles_m = static_cast<int32_t>((a.rows + 255) / 256);
  p.tiles_n = static_cast<int32_t>((a.n + BN - 1) / BN);
  // rows of x walked together: about 32 MB of the 126 MB L2, as in the contraction's GEMM
  const int64_t band = (INT64_C(32) << 20) / (256 * a.k);
  p.band_rows = static_cast<int32_t>(band < 4 ? 4 : band);
  if (p.band_rows > p.tiles_m) p.band_rows = p.tiles_m;
  const int64_t total = static_cast<int64_t>(p.tiles_m) * p.tiles_n;
  if (total >= (INT64_C(1) << 31)) return false;
  const int64_t pairs = total < dev.sms / 2 ? total : dev.sms / 2;
  k_dense8_pair<I8, BN><<<static_cast<unsigned int>(2 * pairs), kThreads, kPairSmem<BN>, stream>>>(mx, mw, p);
  return true;
}

template <bool I8, bool ANY>
bool launch_swap(const LinearArgs& a, const DeviceInfo& dev, Params p, cudaStream_t stream) {
  CUtensorMap mx{}, mw{};
  // rows of x per tile: all of them, or (any alignment) even shares of at most 256
  const int64_t tiles_t = (a.rows + 255) / 256;
  p.cols = static_cast<int32_t>(((a.rows + tiles_t - 1) / tiles_t + 15) / 16 * 16);
  p.tmem_cols = 32;
  while (p.tmem_cols < p.cols) p.tmem_cols *= 2;
  if (!ANY && (!encode_rows_128(dev, &mx, a.x, a.k, a.rows, a.x_stride, p.cols) ||
               !encode_rows_128(dev, &mw, a.w, a.k, a.n, a.w_stride, kTileM)))
    return false;
  p.x = static_cast<const uint8_t*>(a.x), p.w = static_cast<const uint8_t*>(a.w);
  p.x_stride = a.x_stride, p.w_stride = a.w_stride, p.k = a.k;
  const int64_t tiles = (a.n + kTileM - 1) / kTileM, tiles_z = (a.rows + p.cols - 1) / p.cols;
  if (tiles_z > 65535) return false;
  const bool two = kSwapCtas<ANY> == 2 && p.cols <= kSwapColsHalf;
  const int parts = split_of(tiles * tiles_z, p.k_blocks, dev.clusters, two ? 2 : 1);
  const int stage_bytes = kBytesM + p.cols * kTileK;
  p.stages = ((two ? kSwapSmemHalf : kSwapSmem) - 1024 - kCtrlBytes) / stage_bytes;
  if (p.stages > kSwapMaxStages) p.stages = kSwapMaxStages;
  if (static_cast<int64_t>(p.stages) * stage_bytes < static_cast<int64_t>(p.cols) * kTileM * 4) return false;  // (the fold)
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned int>(tiles), static_cast<unsigned int>(parts), static_cast<unsigned int>(tiles_z));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(p.stages) * stage_bytes + 1024 + kCtrlBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {1, static_cast<unsigned int>(parts), 1};
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, k_dense8_swap<I8, ANY>, mw, mx, p) == cudaSuccess;
}

template <bool I8>
bool set_attributes() {
  auto smem = [](const void* f, int bytes) {
    return cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) == cudaSuccess;
  };
  cudaFuncAttributes attr;
  return cudaFuncGetAttributes(&attr, k_dense8_swap<I8, false>) == cudaSuccess &&
         kSwapCtas<false> * kThreads * ((attr.numRegs + 7) / 8 * 8) <= 65536 &&
         smem(reinterpret_cast<const void*>(k_dense8_pair<I8, 256>), kPairSmem<256>) &&
         smem(reinterpret_cast<const void*>(k_dense8_pair<I8, 128>), kPairSmem<128>) &&
         smem(reinterpret_cast<const void*>(k_dense8_swap<I8, false>), kSwapSmem) &&
         smem(reinterpret_cast<const void*>(k_dense8_swap<I8, true>), kSwapSmem);
}

template <bool I8>
bool launch(const LinearArgs& a, const DeviceInfo& dev, const Params& p, cudaStream_t stream) {
  if (!both8_for_tma(a)) return launch_swap<I8, true>(a, dev, p, stream);
  if (a.rows <= 256) return launch_swap<I8, false>(a, dev, p, stream);
  // whole waves of tiles on the CTA pairs: 128 columns where their last wave is fuller by more than the
  // narrower tile costs
  const int64_t tiles_m = (a.rows + 255) / 256, pairs = dev.sms / 2;
  auto waves = [&](int64_t bn) { return (tiles_m * ((a.n + bn - 1) / bn) + pairs - 1) / pairs * bn; };
  if (waves(128) * 125 < waves(256) * 100) return launch_pair<I8, 128>(a, dev, p, stream);
  return launch_pair<I8, 256>(a, dev, p, stream);
}

}  // namespace

bool dense8_setup() { return set_attributes<true>() && set_attributes<false>(); }

imd_status_t dense8_launch(const LinearArgs& a, cudaStream_t stream) {
  const DeviceInfo* dev = device_info();
  if (dev == nullptr) return IMD_STATUS_CUDA_ERROR;
  Params p{};
  p.rows = static_cast<int32_t>(a.rows), p.n = static_cast<int32_t>(a.n);
  p.k_blocks = static_cast<int32_t>((a.k + kTileK - 1) / kTileK);
  p.x_scale = a.x_scale, p.w_scale = a.w_scale8;
  p.out = a.out, p.out_stride = a.out_stride, p.out_type = a.out_type;
  const int unit = a.out_type == IMD_TYPE_F32 ? 4 : 8;
  p.out_wide = reinterpret_cast<uintptr_t>(a.out) % 16 == 0 && a.out_stride % unit == 0;
  p.error_word = dev->error_word;
  const bool ok = a.kind == WeightKind::kI8 ? launch<true>(a, *dev, p, stream) : launch<false>(a, *dev, p, stream);
  return cudaGetLastError() == cudaSuccess && ok ? IMD_STATUS_SUCCESS : IMD_STATUS_CUDA_ERROR;
}

}  // namespace imd
