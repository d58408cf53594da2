// A persistent tcgen05 matmul kernel whose tiles, operand loads and epilogue come from a policy class; the matmuls
// of the gated expert layer and of its backward pass (gated.cu) and of the projection with adapters (lora.cu) are
// policies of it.
//
// One output tile = 128 rows x 256 columns, accumulated in fp32 in TMEM (two accumulators, so the epilogue of one
// tile runs while the tensor cores fill the other). K steps of 64. Warp roles, with nothing but mbarriers between
// them: warp 0 TMA producer, warp 1 MMA issuer, 8 or 16 epilogue warps, 4 warps for rows of A (policies that have them).
//
// A stage of the shared-memory ring holds A (16 KB) and B (32 KB) with the 128-byte swizzle, each in one of two forms:
//   K-major   rows of the M (N) dimension, 64 K elements = 128 bytes per row
//   MN-major  slabs of 64 K rows x 64 M (N) elements, 8 KB per slab
// so weights and their gradients are consumed and written as they lie in memory and nothing is transposed. (Which rows of x
// and of the output's gradient belong together is the policies' business: gated.cu copies them into layout order.)
//
// Every wait is bounded; on expiry the role sets a bit in *dev_status, raises the block's abort flag and all roles
// drain to the common exit, where TMEM is released.
#pragma once

#include "bsr_gemm.cuh"

namespace sb {

constexpr int kTileRows = 128;
constexpr int kTileCols = 256;
constexpr int kTileStep = 64;

struct alignas(64) TileMaps {
  CUtensorMap m[8];
};

struct TileSmem {
  static constexpr int kABytes = kTileRows * kTileStep * 2;
  static constexpr int kBBytes = kTileCols * kTileStep * 2;
  static constexpr int kSlabBytes = kTileStep * 128;
  static constexpr int kStagingBytes = 32 * 128;  // one staging tile of an epilogue warp: 32 rows x 128 bytes
  static constexpr int kBarrierBytes = 256;
};

// What an epilogue warp works with.
struct EpilogueWarp {
  int quarter;       // rows quarter * 32 .. + 31 of the tile (TMEM lanes this warp may read)
  int part;          // which of the kEpilogueWarps / 4 parts of the tile's columns is this warp's
  int lane;
  uint32_t staging;  // this warp's staging tile in shared memory, 4 KB (policies that have one)
  uint32_t taddr;    // TMEM address of (lane quarter, column 0) of the finished accumulator
};

// 128 bytes of this lane's row (64 bf16 columns as pairs, or 32 fp32 columns) -> a staging tile of the warp -> one TMA
// store of 32 rows.
__device__ __forceinline__ void store_rows_128b(EpilogueWarp& w, const CUtensorMap* map, const uint32_t (&packed)[32],
                                                int32_t col, int32_t row) {
  if (w.lane == 0) ptx::bulk_wait_read();  // the last store has read it
  __syncwarp();
  const uint32_t swz = static_cast<uint32_t>(w.lane & 7);
  const uint32_t dst = w.staging + static_cast<uint32_t>(w.lane) * 128u;
#pragma unroll
  for (uint32_t c = 0; c < 8; ++c)
    ptx::st_shared_v4(dst + ((c ^ swz) << 4), packed[4 * c], packed[4 * c + 1], packed[4 * c + 2], packed[4 * c + 3]);
  ptx::fence_proxy_async_shared();
  __syncwarp();
  if (w.lane == 0) {
    ptx::tma_store_2d(map, w.staging, col, row);
    ptx::bulk_commit();
  }
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 pair = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&pair);
}

// 64 accumulator columns as they are, rounded to bf16.
__device__ __forceinline__ void load_packed_x64(uint32_t taddr, uint32_t (&packed)[32]) {
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    uint32_t v[32];
    ptx::tmem_ld_32x32b_x32(taddr + part * 32, v);
    ptx::tmem_ld_wait();
#pragma unroll
    for (int h = 0; h < 16; ++h)
      packed[part * 16 + h] = pack_bf16(__uint_as_float(v[2 * h]), __uint_as_float(v[2 * h + 1]));
  }
}

// A policy Op has
//   Params, Tile (with int32_t k_steps: 0 = nothing to multiply; bool live: the epilogue has something to do)
//   static constexpr bool kAMnMajor, kBMnMajor, kAhead, kVariable, kExtension
//   total_tiles(p), tile(p, index), load(maps, p, tile, ks, a, b, bar)
//   prefetch(p, tile, w) -> Early: global loads that can start before the accumulator is ready; then
//   epilogue(maps, p, tile, w, early). With kAhead: ahead(p, next tile, w) between the two.
//   static constexpr int kStages (of the ring), kEpilogueWarps, kStaging (staging tiles of each: 1, or 0 where it stores from registers)
//   With kExtension: Tile has base_steps; four warps fill the stages of the K steps behind them. A from registers:
//   Rows rows(p, tile, row0) once per tile, extension_chunk(p, tile, rows, j, row, ks, chunk) = the 16 bytes of chunk
//   `chunk` of row `row` = row0 + 16 j. B (MN-major) eight K rows at a time: extension_row(p, tile, ks, i) says where
//   piece i comes from, ahead of time, extension_load(maps, p, tile, i, row, b, bar) issues its loads.
//   With kVariable: columns(p, tile) <= 256 (a multiple of 16) accumulator columns in use, tx_bytes(p, tile, ks) per stage
template <class Op>
struct TileConfig {
  static constexpr int kExtensionWarps = Op::kExtension ? 4 : 0;
  static constexpr int kFirstExtensionWarp = 2 + Op::kEpilogueWarps;
  static constexpr int kThreads = 32 * (kFirstExtensionWarp + kExtensionWarps);
  static constexpr int kSmemBytes = 1024 + Op::kStages * (TileSmem::kABytes + TileSmem::kBBytes) +
                                    Op::kEpilogueWarps * Op::kStaging * TileSmem::kStagingBytes + TileSmem::kBarrierBytes;
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

template <class Op>
__global__ void __launch_bounds__(TileConfig<Op>::kThreads, 1)
tile_gemm_kernel(const __grid_constant__ TileMaps maps, const __grid_constant__ typename Op::Params p, int32_t* dev_status) {
  using Cfg = TileConfig<Op>;
  using S = TileSmem;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
  const uint32_t a_base = smem_base;
  const uint32_t b_base = a_base + Op::kStages * S::kABytes;
  const uint32_t staging_base = b_base + Op::kStages * S::kBBytes;
  const uint32_t full_bar = staging_base + Op::kEpilogueWarps * Op::kStaging * S::kStagingBytes;  // [kStages]
  const uint32_t empty_bar = full_bar + 8 * Op::kStages;                          // [kStages]
  const uint32_t acc_full_bar = empty_bar + 8 * Op::kStages;                      // [2]
  const uint32_t acc_empty_bar = acc_full_bar + 16;                               // [2]
  const uint32_t tmem_slot = acc_empty_bar + 16;
  const uint32_t abort_slot = tmem_slot + 4;
  const uint32_t go_bar = abort_slot + 4;             // [kStages] extension: the stage is free for the warps' A rows
  const uint32_t ready_bar = go_bar + 8 * Op::kStages;  // [kStages] extension: they are written
  uint8_t* smem_aligned = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
  volatile uint32_t* tmem_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (tmem_slot - smem_base));
  volatile uint32_t* abort_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (abort_slot - smem_base));

  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31);

  if (threadIdx.x == 0) {
    for (int s = 0; s < Op::kStages; ++s) {
      ptx::mbar_init(full_bar + 8 * s, 1);
      ptx::mbar_init(empty_bar + 8 * s, 1);
      if (Op::kExtension) {
        ptx::mbar_init(go_bar + 8 * s, 1);
        ptx::mbar_init(ready_bar + 8 * s, Cfg::kExtensionWarps);
      }
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(acc_full_bar + 8 * a, 1);
      ptx::mbar_init(acc_empty_bar + 8 * a, 32 * Op::kEpilogueWarps);
    }
    *abort_word = 0u;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 2 * kTileCols);
    ptx::tmem_relinquish();
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_word;
  // Launched with programmatic dependence: everything up to here may overlap the end of the kernel before.
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  ptx::fence_proxy_async_global();  // what earlier kernels stored is read by TMA

  const int32_t total = Op::total_tiles(p);
  const int32_t step = static_cast<int32_t>(gridDim.x);
  auto give_up = [&](int bit) {
    *abort_word = 1u;
    if (dev_status != nullptr) atomicOr(dev_status, bit);
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      int32_t index = blockIdx.x;
      typename Op::Tile next{};
      if (index < total) next = Op::tile(p, index);
      for (; ok && index < total; index += step) {
        const typename Op::Tile tile = next;
        if (index + step < total) next = Op::tile(p, index + step);
        for (int32_t ks = 0; ks < tile.k_steps; ++ks) {
          if (!ptx::mbar_wait_bounded(empty_bar + 8 * stage, phase ^ 1u, abort_word)) {
            give_up(SB_DEV_TIMEOUT_PRODUCER);
            ok = false;
            break;
          }
          const uint32_t bar = full_bar + 8 * stage;
          bool extension = false;
          if constexpr (Op::kExtension) extension = ks >= tile.base_steps;
          if (extension) {
            ptx::mbar_arrive(go_bar + 8 * stage);  // the extension warps fill this stage
          } else {
            if constexpr (Op::kVariable) ptx::mbar_arrive_expect_tx(bar, Op::tx_bytes(p, tile, ks));
            else ptx::mbar_arrive_expect_tx(bar, S::kBBytes + S::kABytes);
            Op::load(maps, p, tile, ks, a_base + stage * S::kABytes, b_base + stage * S::kBBytes, bar);
          }
          if (++stage == Op::kStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (lane == 0) {
      uint32_t idesc = ptx::make_idesc_bf16(kTileRows, kTileCols, Op::kBMnMajor) | (Op::kAMnMajor ? 1u << 15 : 0u);
      uint32_t stage = 0, phase = 0, acc = 0, acc_phase = 0, ready_phases = 0;
      bool ok = true;
      int32_t index = blockIdx.x;
      typename Op::Tile next{};
      if (index < total) next = Op::tile(p, index);
      for (; ok && index < total; index += step) {
        const int32_t k_steps = next.k_steps;
        int32_t base_steps = k_steps;
        if constexpr (Op::kExtension) base_steps = next.base_steps;
        if constexpr (Op::kVariable)
          idesc = ptx::make_idesc_bf16(kTileRows, Op::columns(p, next), Op::kBMnMajor) | (Op::kAMnMajor ? 1u << 15 : 0u);
        if (index + step < total) next = Op::tile(p, index + step);
        if (k_steps == 0) continue;
        if (!ptx::mbar_wait_bounded(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_word)) {
          give_up(SB_DEV_TIMEOUT_MMA);
          break;
        }
        ptx::tcgen05_fence_after_sync();
        const uint32_t d_tmem = tmem_base + acc * kTileCols;
        for (int32_t ks = 0; ks < k_steps; ++ks) {
          if (!ptx::mbar_wait_bounded(full_bar + 8 * stage, phase, abort_word)) {
            give_up(SB_DEV_TIMEOUT_MMA);
            ok = false;
            break;
          }
          if (Op::kExtension && ks >= base_steps) {
            if (!ptx::mbar_wait_bounded(ready_bar + 8 * stage, (ready_phases >> stage) & 1u, abort_word)) {
              give_up(SB_DEV_TIMEOUT_MMA);
              ok = false;
              break;
            }
            ready_phases ^= 1u << stage;
          }
          ptx::tcgen05_fence_after_sync();
          const uint32_t a_addr = a_base + stage * S::kABytes;
          const uint32_t b_addr = b_base + stage * S::kBBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint64_t desc_a = Op::kAMnMajor ? ptx::make_smem_desc(a_addr + kk * 2048, S::kSlabBytes, 1024)
                                                  : ptx::make_smem_desc(a_addr + kk * 32, 16, 1024);
            const uint64_t desc_b = Op::kBMnMajor ? ptx::make_smem_desc(b_addr + kk * 2048, S::kSlabBytes, 1024)
                                                  : ptx::make_smem_desc(b_addr + kk * 32, 16, 1024);
            ptx::umma_bf16(d_tmem, desc_a, desc_b, idesc, (ks | kk) != 0);
          }
          ptx::umma_commit(empty_bar + 8 * stage);
          if (++stage == Op::kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        ptx::umma_commit(acc_full_bar + 8 * acc);
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else if (warp < Cfg::kFirstExtensionWarp) {
    // ---------------------------------------------------------------- epilogue
    EpilogueWarp w;
    w.quarter = warp & 3;
    w.part = (warp - 2) >> 2;
    w.lane = lane;
    w.staging = staging_base + static_cast<uint32_t>(warp - 2) * (Op::kStaging * S::kStagingBytes);
    uint32_t acc = 0, acc_phase = 0;
    typename Op::Tile next{};
    if (static_cast<int32_t>(blockIdx.x) < total) next = Op::tile(p, blockIdx.x);
    for (int32_t index = blockIdx.x; index < total; index += step) {
      const typename Op::Tile tile = next;
      typename Op::Early early{};
      if (tile.live) early = Op::prefetch(p, tile, w);
      if (index + step < total) {
        next = Op::tile(p, index + step);
        if constexpr (Op::kAhead) Op::ahead(p, next, w);
      }
      if (!tile.live) continue;
      if (tile.k_steps > 0) {
        if (!ptx::mbar_wait_bounded(acc_full_bar + 8 * acc, acc_phase, abort_word)) {
          give_up(SB_DEV_TIMEOUT_EPILOGUE);
          break;
        }
        ptx::tcgen05_fence_after_sync();
      }
      w.taddr = tmem_base + (static_cast<uint32_t>(w.quarter * 32) << 16) + acc * kTileCols;
      Op::epilogue(maps, p, tile, w, early);
      if (tile.k_steps > 0) {
        ptx::tcgen05_fence_before_sync();
        ptx::mbar_arrive(acc_empty_bar + 8 * acc);
        acc ^= 1u;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
    if (lane == 0) ptx::bulk_wait_all();
  } else {
    // ---------------------------------------------------------------- extension rows of A
    if constexpr (Op::kExtension) {
      // Eight lanes share a row's 128 bytes of the K step; rows j * 16 + warp * 4 + lane / 8. The producer says when a stage is free
      // (its own wait on empty_bar passed), so that these warps need not follow the ring through the base steps.
      const int row0 = (warp - Cfg::kFirstExtensionWarp) * 4 + (lane >> 3);
      const int chunk = lane & 7;
      const uint32_t dst_off = static_cast<uint32_t>(row0) * 128u + (static_cast<uint32_t>(chunk ^ (row0 & 7)) << 4);
      uint32_t stage = 0, go_phases = 0;
      bool ok = true;
      for (int32_t index = blockIdx.x; ok && index < total; index += step) {
        const typename Op::Tile tile = Op::tile(p, index);
        stage = (stage + static_cast<uint32_t>(tile.base_steps)) % Op::kStages;
        if (tile.base_steps >= tile.k_steps) continue;
        const typename Op::Rows rows = Op::rows(p, tile, row0);
        for (int32_t ks = tile.base_steps; ks < tile.k_steps; ++ks) {
          uint4 chunks[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) chunks[j] = Op::extension_chunk(p, tile, rows, j, row0 + j * 16, ks, chunk);
          const bool loads = warp == Cfg::kFirstExtensionWarp && lane < 8;
          const int32_t b_row = loads ? Op::extension_row(p, tile, ks, lane) : 0;
          if (!ptx::mbar_wait_bounded(go_bar + 8 * stage, (go_phases >> stage) & 1u, abort_word)) {
            give_up(SB_DEV_TIMEOUT_PRODUCER);
            ok = false;
            break;
          }
          go_phases ^= 1u << stage;
          if (warp == Cfg::kFirstExtensionWarp) {
            if (lane == 0) ptx::mbar_arrive_expect_tx(full_bar + 8 * stage, Op::tx_bytes(p, tile, ks));
            __syncwarp();
            if (loads) Op::extension_load(maps, p, tile, lane, b_row, b_base + stage * S::kBBytes, full_bar + 8 * stage);
          }
          const uint32_t dst = a_base + stage * S::kABytes + dst_off;
#pragma unroll
          for (int j = 0; j < 8; ++j) ptx::st_shared_v4(dst + j * 2048, chunks[j].x, chunks[j].y, chunks[j].z, chunks[j].w);
          ptx::fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) ptx::mbar_arrive(ready_bar + 8 * stage);
          if (++stage == Op::kStages) stage = 0;
        }
      }
    }
  }

  if (*abort_word != 0u) {
    // Gave up mid-pipeline: leave copies still in flight time to land before the shared memory is handed back.
    for (int i = 0; i < 64; ++i) __nanosleep(1000);
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, 2 * kTileCols);
  }
}

// ---- host side ---------------------------------------------------------------------------------------------------

// A row-major [rows, cols] map of 2-byte (bf16) or 4-byte (fp32) elements whose boxes are 128 bytes wide, with the
// 128-byte swizzle.
int encode_2d_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint32_t box_rows, uint32_t box_cols,
                  uint32_t element_bytes, const char* what);

template <class Op>
int launch_tile_gemm(const TileMaps& maps, const typename Op::Params& p, int64_t tiles, int32_t* dev_status,
                     cudaStream_t stream, const char* what) {
  int device = 0;
  const DeviceInfo* info = current_device_info(&device);
  if (info == nullptr) return SB_ERR_CUDA;
  static std::atomic<bool> done[kMaxDevices] = {};
  if (!done[device].load(std::memory_order_acquire)) {
    const cudaError_t err = cudaFuncSetAttribute(tile_gemm_kernel<Op>, cudaFuncAttributeMaxDynamicSharedMemorySize, TileConfig<Op>::kSmemBytes);
    if (err != cudaSuccess) return fail(SB_ERR_CUDA, "%s: shared memory opt-in: %s", what, cudaGetErrorString(err));
    done[device].store(true, std::memory_order_release);
  }
  if (tiles <= 0) return SB_OK;
  if (tiles > INT32_MAX - info->sm_count) return fail(SB_ERR_INVALID_ARGUMENT, "%s: problem too large", what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles < info->sm_count ? tiles : info->sm_count));
  cfg.blockDim = dim3(TileConfig<Op>::kThreads);
  cfg.dynamicSmemBytes = TileConfig<Op>::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, tile_gemm_kernel<Op>, maps, p, dev_status);
  if (err != cudaSuccess) return fail(SB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  return SB_OK;
}

}  // namespace sb
