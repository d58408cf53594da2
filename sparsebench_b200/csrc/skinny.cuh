// Products of a few rows with a streamed weight matrix: a decoding step of the gated layer (gated.cu) and of the
// projection with adapters (lora.cu).
//
// With few rows the weights are all that moves, so they take the 128-row side of the tensor-core tile: M = 128 weight
// columns, N = the rows (16 to 128, in steps of 16), K = 64 per stage. A weight tile [64 k x 128 columns] is the MN-major
// operand it is in memory, the rows are the K-major one. One thread block per 128 columns would leave most SMs without
// work, so K is split over the thread blocks of a cluster: each leaves its sums in its shared memory and the blocks add
// them up over distributed shared memory in rank order, each for its share of the rows. No atomics, no workspace.
//
// Two blocks fit an SM, so that one's start and end hide behind the other's stream. The kernels of a chain are launched
// with programmatic dependence: a kernel's weights are on their way before the rows it waits for are written.
//
// Bound by the weights' way from memory; with little of it, by the latency of start, first loads and join (about 5 us).
// Measured as replayed graphs: gated layer, D = 4096, F = 14336, E = 8: one token (two experts, 0.70 GB) 119 us, 5.9 TB/s;
// 16 tokens 413 us, 6.8 TB/s. D = 1024, F = 4096, E = 64: one token (50 MB) 16.5 us, 16 tokens 111 us (5.8 TB/s).
// Projection with adapters, 4096 x 4096: one token 12 us; 4096 x 14336, 64 tokens with 32 adapters: 31 us (4.5 TB/s).
//
// Waits are bounded as in tile_gemm.cuh; a block that gave up still takes part in the cluster's barriers.
#pragma once

#include <algorithm>

#include "bsr_gemm.cuh"

namespace sb {

constexpr int kSkinnyThreads = 192;   // warp 0 TMA, warp 1 MMA, warps 2-5 rows and epilogue
constexpr int kSkinnyWorkers = 128;   // threads of warps 2-5
constexpr int kSkinnyCols = 128;
constexpr int kSkinnyStep = 64;
constexpr int kSkinnyWBytes = kSkinnyCols * kSkinnyStep * 2;
constexpr int kSkinnyMaxRows = 128;

__device__ __forceinline__ void named_barrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}

__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

struct alignas(64) SkinnyMaps {
  CUtensorMap w[2];  // weights, boxes of 64 x 64
  CUtensorMap x;     // rows, boxes of 64 k x the padded row count (policies that do not gather)
};

struct SkinnyShape {
  int32_t splits;      // thread blocks of a cluster
  int32_t steps;       // K steps per split
  int32_t total_steps;
  int32_t stages;
  int32_t rows_pad;    // rows of the operand in shared memory, a multiple of 16
};

constexpr int kSkinnyHeadBytes = 512 + 2 * 4 * kSkinnyMaxRows;  // barriers and words, ids, list of rows

inline int skinny_smem_bytes(const SkinnyShape& s) {
  return 1024 + kSkinnyHeadBytes + s.stages * (kSkinnyWBytes + s.rows_pad * 128);
}

// A policy Op has
//   Params (with SkinnyShape shape)
//   Item: what the block works on; bool begin(p, item, block_item, ids, list): false = nothing to do (uniform over the
//         block and its cluster); item.rows is the number of rows
//   static constexpr bool kGather; gather_row(p, item, list, row) -> source of an operand row
//   load_w(maps, p, item, k_step, dst, bar): both 64-column slabs
//   Extra: registers that the workers fill while the weights stream; extra(p, item, rank, worker, Extra&)
//   finish(p, item, list, rank, worker, red, extra): the block's share of the rows, red.sum(row, column) = 8 columns
struct SkinnySums {
  uint32_t local;  // shared-memory address of red[row][128] in this block
  int32_t splits;
  // Sums over the cluster of columns c .. c + 7 of a row, in rank order.
  __device__ __forceinline__ void sum(int32_t row, int32_t c, float (&v)[8]) const {
    const uint32_t at = local + static_cast<uint32_t>(row * kSkinnyCols + c) * 4u;
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = 0.0f;
    for (int32_t r = 0; r < splits; ++r) {
      const uint32_t remote = ptx::map_to_cta(at, static_cast<uint32_t>(r));
      const float4 a = ld_cluster_f4(remote);
      const float4 b = ld_cluster_f4(remote + 16u);
      v[0] += a.x; v[1] += a.y; v[2] += a.z; v[3] += a.w;
      v[4] += b.x; v[5] += b.y; v[6] += b.z; v[7] += b.w;
    }
  }
};

template <class Op>
__global__ void __launch_bounds__(kSkinnyThreads, 2)
skinny_kernel(const __grid_constant__ SkinnyMaps maps, const __grid_constant__ typename Op::Params p, int32_t* dev_status) {
  extern __shared__ uint8_t smem_raw[];
  const SkinnyShape& sh = p.shape;
  const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
  const uint32_t x_bytes = static_cast<uint32_t>(sh.rows_pad) * 128u;
  const uint32_t w_base = smem_base;
  const uint32_t x_base = w_base + static_cast<uint32_t>(sh.stages) * kSkinnyWBytes;
  const uint32_t head = x_base + static_cast<uint32_t>(sh.stages) * x_bytes;
  const uint32_t full_bar = head;               // [stages], at most 16
  const uint32_t empty_bar = head + 128;        // [stages]
  const uint32_t acc_bar = head + 256;
  const uint32_t tmem_slot = head + 264;
  const uint32_t abort_slot = head + 268;
  volatile uint32_t* tmem_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (tmem_slot - smem_base));
  volatile uint32_t* abort_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (abort_slot - smem_base));
  int32_t* ids = reinterpret_cast<int32_t*>(smem_aligned + (head + 512 - smem_base));
  int32_t* list = ids + kSkinnyMaxRows;

  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int32_t rank = static_cast<int32_t>(blockIdx.x) % sh.splits;
  const int32_t block_item = static_cast<int32_t>(blockIdx.x) / sh.splits;

  ptx::grid_launch_dependents();
  typename Op::Item item;
  if (!Op::begin(p, item, block_item, ids, list)) {
    ptx::grid_dependency_wait();
    return;
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < sh.stages; ++s) {
      ptx::mbar_init(full_bar + 8 * s, Op::kGather ? 1 + kSkinnyWorkers : 1);
      ptx::mbar_init(empty_bar + 8 * s, 1);
    }
    ptx::mbar_init(acc_bar, 1);
    *abort_word = 0u;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, kSkinnyMaxRows);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_word;
  const int32_t first = rank * sh.steps;
  const int32_t steps = max(0, min(sh.steps, sh.total_steps - first));
  auto give_up = [&](int bit) {
    *abort_word = 1u;
    if (dev_status != nullptr) atomicOr(dev_status, bit);
  };

  typename Op::Extra extra;
  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      for (int32_t ks = 0; ks < steps; ++ks) {
        if (!ptx::mbar_wait_bounded(empty_bar + 8 * stage, phase ^ 1u, abort_word)) {
          give_up(SB_DEV_TIMEOUT_PRODUCER);
          break;
        }
        const uint32_t bar = full_bar + 8 * stage;
        ptx::mbar_arrive_expect_tx(bar, kSkinnyWBytes + (Op::kGather ? 0u : x_bytes));
        Op::load_w(maps, p, item, first + ks, w_base + stage * kSkinnyWBytes, bar);
        if (!Op::kGather) ptx::tma_load_2d(x_base + stage * x_bytes, &maps.x, (first + ks) * kSkinnyStep, 0, bar);
        if (++stage == static_cast<uint32_t>(sh.stages)) { stage = 0; phase ^= 1u; }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && steps > 0) {
      const int n = (item.rows + 15) & ~15;
      const uint32_t idesc = ptx::make_idesc_bf16(kSkinnyCols, n, false) | (1u << 15);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int32_t ks = 0; ks < steps; ++ks) {
        if (!ptx::mbar_wait_bounded(full_bar + 8 * stage, phase, abort_word)) {
          give_up(SB_DEV_TIMEOUT_MMA);
          ok = false;
          break;
        }
        if (Op::kGather) ptx::fence_proxy_async_shared();
        ptx::tcgen05_fence_after_sync();
#pragma unroll
        for (int kk = 0; kk < 4; ++kk)
          ptx::umma_bf16(tmem_base, ptx::make_smem_desc(w_base + stage * kSkinnyWBytes + kk * 2048, kSkinnyWBytes / 2, 1024),
                         ptx::make_smem_desc(x_base + stage * x_bytes + kk * 32, 16, 1024), idesc, (ks | kk) != 0);
        ptx::umma_commit(empty_bar + 8 * stage);
        if (++stage == static_cast<uint32_t>(sh.stages)) { stage = 0; phase ^= 1u; }
      }
      if (ok) ptx::umma_commit(acc_bar);
    }
    __syncwarp();
  } else {
    const int worker = static_cast<int>(threadIdx.x) - 64;
    ptx::grid_dependency_wait();
    if constexpr (Op::kGather) {
      // Eight lanes share a row's 128 bytes of the K step; 128 threads move 16 rows at a time.
      const int row0 = worker >> 3;
      const uint32_t chunk = static_cast<uint32_t>(worker & 7);
      const int passes = (((item.rows + 15) & ~15) + 15) / 16;
      const __nv_bfloat16* src[kSkinnyMaxRows / 16];
      bool real[kSkinnyMaxRows / 16];
#pragma unroll
      for (int j = 0; j < kSkinnyMaxRows / 16; ++j) {
        const int row = row0 + 16 * j;
        real[j] = row < item.rows;
        src[j] = Op::gather_row(p, item, list, real[j] ? row : 0) + chunk * 8;
      }
      const uint32_t dst0 = x_base + static_cast<uint32_t>(row0) * 128u + ((chunk ^ static_cast<uint32_t>(row0 & 7)) << 4);
      uint32_t stage = 0, phase = 0;
      for (int32_t ks = 0; ks < steps; ++ks) {
        if (!ptx::mbar_wait_bounded(empty_bar + 8 * stage, phase ^ 1u, abort_word)) {
          give_up(SB_DEV_TIMEOUT_PRODUCER);
          break;
        }
#pragma unroll
        for (int j = 0; j < kSkinnyMaxRows / 16; ++j)
          if (j < passes)
            ptx::cp_async_16_zfill(dst0 + stage * x_bytes + j * 2048, src[j] + static_cast<int64_t>(first + ks) * kSkinnyStep, real[j]);
        ptx::cp_async_mbar_arrive_noinc(full_bar + 8 * stage);
        if (++stage == static_cast<uint32_t>(sh.stages)) { stage = 0; phase ^= 1u; }
      }
      ptx::cp_async_wait_all();
    }
    Op::extra(p, item, rank, worker, extra);
    // The sums of this split: TMEM lane = column, TMEM column = row -> red[row][column], over the ring (all of it read).
    const int quarter = warp & 3;
    const int col = quarter * 32 + lane;
    float* red = reinterpret_cast<float*>(smem_aligned);
    bool got = true;
    if (steps > 0) {
      got = ptx::mbar_wait_bounded(acc_bar, 0, abort_word);
      if (!got) give_up(SB_DEV_TIMEOUT_EPILOGUE);
      got = __all_sync(0xffffffffu, got);
      ptx::tcgen05_fence_after_sync();
    }
    named_barrier(1, kSkinnyWorkers);  // no worker's copies or reads of the ring are left
#pragma unroll 1
    for (int r0 = 0; got && r0 < item.rows; r0 += 8) {
      uint32_t v[8];
      if (steps > 0) {
        ptx::tmem_ld_32x32b_x8(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + r0, v);
        ptx::tmem_ld_wait();
      } else {
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] = 0u;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q)
        if (r0 + q < item.rows) red[(r0 + q) * kSkinnyCols + col] = __uint_as_float(v[q]);
    }
  }
  if (*abort_word != 0u) {
    // Gave up mid-stream: leave copies still in flight time to land before the shared memory is handed back.
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  __syncwarp();
  ptx::tcgen05_fence_before_sync();
  if (sh.splits > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, kSkinnyMaxRows);
  }
  if (warp >= 2 && *abort_word == 0u) {
    const SkinnySums sums{smem_base, sh.splits};
    Op::finish(p, item, list, rank, static_cast<int>(threadIdx.x) - 64, sums, extra);
  }
  if (sh.splits > 1) ptx::cluster_sync_all();  // nobody's shared memory is read any more
}

// ---- host side ---------------------------------------------------------------------------------------------------

// Splits of K so that about two blocks per SM have work, each at least four steps (64 KB of weights) of it.
inline SkinnyShape skinny_shape(int64_t items, int32_t total_steps, int32_t rows, int sm_count) {
  SkinnyShape s{};
  s.total_steps = total_steps;
  s.rows_pad = (rows + 15) & ~15;
  s.splits = 1;
  while (s.splits < 8 && items * s.splits < 3 * static_cast<int64_t>(sm_count) / 2 && total_steps >= 8 * s.splits) s.splits *= 2;
  s.steps = (total_steps + s.splits - 1) / s.splits;
  // Two blocks per SM: at most 113 KB each.
  s.stages = std::min(8, (113 * 1024 - 1024 - kSkinnyHeadBytes - 1024) / (kSkinnyWBytes + s.rows_pad * 128));
  return s;
}

template <class Op>
int launch_skinny(const SkinnyMaps& maps, const typename Op::Params& p, int64_t items, bool dependent, int32_t* dev_status,
                  cudaStream_t stream, const char* what) {
  int device = 0;
  if (current_device_info(&device) == nullptr) return SB_ERR_CUDA;
  static std::atomic<bool> done[kMaxDevices] = {};
  if (!done[device].load(std::memory_order_acquire)) {
    const cudaError_t err = cudaFuncSetAttribute(skinny_kernel<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, 113 * 1024);
    if (err != cudaSuccess) return fail(SB_ERR_CUDA, "%s: shared memory opt-in: %s", what, cudaGetErrorString(err));
    done[device].store(true, std::memory_order_release);
  }
  if (items <= 0) return SB_OK;
  if (items * p.shape.splits > INT32_MAX) return fail(SB_ERR_INVALID_ARGUMENT, "%s: problem too large", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items * p.shape.splits));
  cfg.blockDim = dim3(kSkinnyThreads);
  cfg.dynamicSmemBytes = static_cast<size_t>(skinny_smem_bytes(p.shape));
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
  attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(p.shape.splits);
  attr[cfg.numAttrs].val.clusterDim.y = 1;
  attr[cfg.numAttrs].val.clusterDim.z = 1;
  ++cfg.numAttrs;
  if (dependent) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs].val.programmaticStreamSerializationAllowed = 1;
    ++cfg.numAttrs;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, skinny_kernel<Op>, maps, p, dev_status);
  if (err != cudaSuccess) return fail(SB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  return SB_OK;
}

}  // namespace sb
