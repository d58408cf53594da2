// A projection with the low-rank adapters of many requests at once:
//
//   y[t] = x[t] W + scale[a] * sum_j (x[t] . A[a, j]) B[a, j],   a = adapter_idx[t]   (outside [0, L): no second term)
//
// The products run on tiles of 128 consecutive tokens. A tile's distinct adapters are its slots, in order of first
// appearance (a batch is its requests' tokens one after another, so a tile has few). Per call:
//
//   shrink   the slots of every tile; V = x A[a]^T: the rows of all slots' A side by side are the columns of one product,
//            of which each token keeps its own slot's; split over D within a cluster, joined there with the scale
//   expand   y = [x | V in its slot's columns, zeros elsewhere] [W ; B of the slots]: the second term is a few more K
//            steps of the projection itself, so y is written once and never read back
//
// Up to 64 tokens (a decoding step) the weights are streamed by the kernel of skinny.cuh and the second term is plain
// fp32 arithmetic on each token's own rows of A and B (lora_rows_kernel, SkinnyLora).
//
// In the products V is rounded to bf16 for y in bf16; for y in fp32 it travels as three bf16 (V, what rounding took from it,
// and what that left, against the same rows of B): the 24 bits of an fp32.
//
// There a zero of V meets B of other requests' adapters: an infinity or NaN in one adapter would reach its neighbours'
// rows. So an adapter whose B is not finite stays out of the product (shrink finds it, reading B beside its own loads and
// on its way into L2) and its own rows get their term from the epilogue, number by number.

#include <algorithm>
#include <initializer_list>

#include "skinny.cuh"
#include "tile_gemm.cuh"

namespace sb {
namespace {

// Up to here a batch is a decoding step.
constexpr int64_t kSmallTokens = 64;
static_assert(kSmallTokens <= kSkinnyMaxRows, "rows of the skinny kernel");

constexpr int kMaxSlots = kTileRows;
// Per tile: the slot count, the adapter of each slot, the slot of each row (-1: none).
constexpr int kSlotAdapter = 1, kRowSlot = kSlotAdapter + kMaxSlots;
constexpr int kTableInts = kRowSlot + kTileRows;
constexpr int kMaxSplits = 8;  // thread blocks of a cluster; also the bytes per adapter that say whether its B is finite

// Every block of the shrink kernel looks through its part of the adapter's B and sets its byte.
__device__ __forceinline__ bool adapter_finite(const uint8_t* not_finite, int32_t adapter, int32_t splits) {
  const unsigned long long f = __ldg(reinterpret_cast<const unsigned long long*>(not_finite) + adapter);
  return (splits < kMaxSplits ? f & ((1ull << (8 * splits)) - 1ull) : f) == 0ull;
}

// ---- shrink -------------------------------------------------------------------------------------------------------
// A cluster per tile of 128 tokens, each block a part of D. Per group of slots (as many as fit 128 columns) one product:
// x tile (K-major) times the slots' rows of A (K-major, 8 to 128 rows by TMA per slot and step). Row i of the tile takes
// the columns of its slot from TMEM into shared memory; after the last group the blocks of the cluster add their parts up
// over distributed shared memory, in rank order, each for its share of the rows.
//
// Latency sets the time: 11 us at T = 4096, D = 1024, rank 8 (most of it start, slots and join), 40 us cold and about half of
// that behind a warm L2 at T = 8191, D = 4096, rank 64, where the tiles with most slots finish last.
//
// Meanwhile twelve more warps look for infinities and NaN in B: of those of the tile's adapters that the tile before
// does not have (they are being looked through there, or further up). For a batch of whole requests that is once per
// request; in any order it is at most what expand reads of B anyway. Tiles that share an adapter write the same answer.
constexpr int kScanThreads = 384;
constexpr int kShrinkThreads = 192 + kScanThreads;  // warp 0 TMA, warp 1 MMA, warps 2-5 workers (a row of the tile each), scan
constexpr int kShrinkCols = 128;
constexpr int kShrinkStageBytes = (kTileRows + kShrinkCols) * 128;

struct ShrinkMaps {
  CUtensorMap x, a;
};
struct ShrinkParams {
  const void* adapter_idx;
  const uint4* b;
  const float* scale;
  int32_t* tables;
  uint8_t* not_finite;
  __nv_bfloat16* v;  // [T, rank * parts]: the values, with parts = 3 then what rounding took from them, twice
  int32_t idx_is_i64, num_tokens, num_adapters, rank, parts, splits, steps, total_steps, stages;
  int32_t b_vecs;  // 16-byte pieces of an adapter's B
};
constexpr int kShrinkHeadBytes = 512 + 4 * (5 * kTileRows + 8);  // barriers, ids, slots, first rows, seen, new slots, counts

inline int shrink_smem_bytes(int stages, int rank) { return 1024 + kShrinkHeadBytes + stages * kShrinkStageBytes + kTileRows * rank * 4; }

__device__ __forceinline__ int32_t adapter_of(const ShrinkParams& p, int32_t token) {
  if (token < 0 || token >= p.num_tokens) return -1;
  const int64_t a = p.idx_is_i64 ? __ldg(static_cast<const long long*>(p.adapter_idx) + token)
                                 : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.adapter_idx) + token));
  return a >= 0 && a < p.num_adapters ? static_cast<int32_t>(a) : -1;
}

__global__ void __launch_bounds__(kShrinkThreads, 1)
lora_shrink_kernel(const __grid_constant__ ShrinkMaps maps, const __grid_constant__ ShrinkParams p, int32_t* dev_status) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (ptx::smem_addr(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_aligned = smem_raw + (smem_base - ptx::smem_addr(smem_raw));
  const uint32_t red_base = smem_base + static_cast<uint32_t>(p.stages) * kShrinkStageBytes;  // red[rank][128] fp32
  const uint32_t head = red_base + static_cast<uint32_t>(kTileRows * p.rank) * 4u;
  const uint32_t full_bar = head;             // [stages], at most 8
  const uint32_t empty_bar = head + 64;       // [stages]
  const uint32_t acc_full_bar = head + 128;   // [2]
  const uint32_t acc_empty_bar = head + 144;  // [2]
  const uint32_t tmem_slot = head + 160;
  const uint32_t abort_slot = head + 164;
  volatile uint32_t* tmem_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (tmem_slot - smem_base));
  volatile uint32_t* abort_word = reinterpret_cast<volatile uint32_t*>(smem_aligned + (abort_slot - smem_base));
  int32_t* id = reinterpret_cast<int32_t*>(smem_aligned + (head + 512 - smem_base));
  int32_t* slot_adapter = id + kTileRows;
  int32_t* work = slot_adapter + kTileRows;  // slot of the first row of an adapter; then: slot of each row
  int32_t* seen = work + kTileRows;          // the slot's adapter is in the tile before, too
  int32_t* fresh_slot = seen + kTileRows;    // the slots whose adapter is not
  int32_t* count = fresh_slot + kTileRows;   // [4] per worker warp
  float* red = reinterpret_cast<float*>(smem_aligned + (red_base - smem_base));

  const int warp = static_cast<int>(threadIdx.x >> 5);
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int row = static_cast<int>(threadIdx.x) - 64;  // of the workers
  const bool worker = row >= 0 && row < kTileRows;
  const int32_t rank = static_cast<int32_t>(blockIdx.x) % p.splits;
  const int32_t tile = static_cast<int32_t>(blockIdx.x) / p.splits;
  const int32_t first_token = tile * kTileRows;

  ptx::grid_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      ptx::mbar_init(full_bar + 8 * s, 1);
      ptx::mbar_init(empty_bar + 8 * s, 1);
    }
    for (int a = 0; a < 2; ++a) {
      ptx::mbar_init(acc_full_bar + 8 * a, 1);
      ptx::mbar_init(acc_empty_bar + 8 * a, kTileRows);
    }
    *abort_word = 0u;
    ptx::fence_barrier_init();
  }
  if (warp == 1) {
    ptx::tmem_alloc(tmem_slot, 2 * kShrinkCols);
    ptx::tmem_relinquish();
  }
  int32_t mine = -1;
  if (worker) {
    mine = adapter_of(p, first_token + row);
    id[row] = mine;
    seen[row] = 0;
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem_base = *tmem_word;
  // Slots. first never lies behind the row: its own id matches.
  int first = row;
  if (mine >= 0) {
    for (int j = 0; j < row; j += 4) {
      const int4 four = *reinterpret_cast<const int4*>(id + j);
      if (four.x == mine) { first = j; break; }
      if (four.y == mine) { first = j + 1; break; }
      if (four.z == mine) { first = j + 2; break; }
      if (four.w == mine) { first = j + 3; break; }
    }
  }
  const bool leads = mine >= 0 && first == row;
  const unsigned leaders = __ballot_sync(0xffffffffu, leads);
  if (worker && lane == 0) count[warp - 2] = __popc(leaders);
  __syncthreads();
  const int32_t slots = count[0] + count[1] + count[2] + count[3];
  if (leads) {
    int32_t slot = __popc(leaders & ((1u << lane) - 1u));
    for (int w = 0; w < warp - 2; ++w) slot += count[w];
    slot_adapter[slot] = mine;
    work[row] = slot;
  }
  __syncthreads();
  const int32_t my_slot = mine >= 0 ? work[first] : -1;
  if (worker && rank == 0) {
    int32_t* table = p.tables + static_cast<int64_t>(tile) * kTableInts;
    if (row == 0) table[0] = slots;
    if (row < slots) table[kSlotAdapter + row] = slot_adapter[row];
    table[kRowSlot + row] = my_slot;
  }
  const int32_t group_slots = kShrinkCols / p.rank;
  const int32_t groups = (slots + group_slots - 1) / group_slots;
  const int32_t k0 = rank * p.steps;
  const int32_t steps = max(0, min(p.steps, p.total_steps - k0));
  auto give_up = [&](int bit) {
    *abort_word = 1u;
    if (dev_status != nullptr) atomicOr(dev_status, bit);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int32_t g = 0; ok && g < groups; ++g) {
        const int32_t n = min(group_slots, slots - g * group_slots);
        for (int32_t ks = 0; ks < steps; ++ks) {
          if (!ptx::mbar_wait_bounded(empty_bar + 8 * stage, phase ^ 1u, abort_word)) {
            give_up(SB_DEV_TIMEOUT_PRODUCER);
            ok = false;
            break;
          }
          const uint32_t bar = full_bar + 8 * stage;
          const uint32_t a = smem_base + stage * kShrinkStageBytes;
          const int32_t k = (k0 + ks) * kTileStep;
          ptx::mbar_arrive_expect_tx(bar, kTileRows * 128u + static_cast<uint32_t>(n * p.rank) * 128u);
          ptx::tma_load_2d(a, &maps.x, k, first_token, bar);
          for (int32_t s = 0; s < n; ++s)
            ptx::tma_load_2d(a + (kTileRows + s * p.rank) * 128u, &maps.a, k, slot_adapter[g * group_slots + s] * p.rank, bar);
          if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && steps > 0) {
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int32_t g = 0; ok && g < groups; ++g) {
        const uint32_t acc = static_cast<uint32_t>(g) & 1u;
        const uint32_t acc_phase = (static_cast<uint32_t>(g) >> 1) & 1u;
        if (!ptx::mbar_wait_bounded(acc_empty_bar + 8 * acc, acc_phase ^ 1u, abort_word)) {
          give_up(SB_DEV_TIMEOUT_MMA);
          break;
        }
        ptx::tcgen05_fence_after_sync();
        const int n = (min(group_slots, slots - g * group_slots) * p.rank + 15) & ~15;
        const uint32_t idesc = ptx::make_idesc_bf16(kTileRows, n, false);
        for (int32_t ks = 0; ks < steps; ++ks) {
          if (!ptx::mbar_wait_bounded(full_bar + 8 * stage, phase, abort_word)) {
            give_up(SB_DEV_TIMEOUT_MMA);
            ok = false;
            break;
          }
          ptx::tcgen05_fence_after_sync();
          const uint32_t a = smem_base + stage * kShrinkStageBytes;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            ptx::umma_bf16(tmem_base + acc * kShrinkCols, ptx::make_smem_desc(a + kk * 32, 16, 1024),
                           ptx::make_smem_desc(a + kTileRows * 128 + kk * 32, 16, 1024), idesc, (ks | kk) != 0);
          ptx::umma_commit(empty_bar + 8 * stage);
          if (++stage == static_cast<uint32_t>(p.stages)) { stage = 0; phase ^= 1u; }
        }
        if (ok) ptx::umma_commit(acc_full_bar + 8 * acc);
      }
    }
    __syncwarp();
  } else if (!worker) {
    // ---- B of the adapters that are new in this tile
    const int i = static_cast<int>(threadIdx.x) - 192;
    if (i < kTileRows && first_token > 0) {
      const int32_t before = adapter_of(p, first_token - kTileRows + i);
      if (before >= 0)
        for (int32_t s = 0; s < slots; ++s)
          if (slot_adapter[s] == before) seen[s] = 1;
    }
    named_barrier(2, kScanThreads);
    // The slots that are new, in slot order, and the flag of each: both in `seen`, whose entry of a slot in front has been
    // read by everybody before it is written again.
    int32_t fresh = 0, nth = -1;
    for (int32_t s = 0; s < slots; ++s) {
      if (s == i && seen[s] == 0) nth = fresh;
      fresh += seen[s] == 0 ? 1 : 0;
    }
    named_barrier(2, kScanThreads);
    if (nth >= 0) fresh_slot[nth] = i;
    if (i < kTileRows) seen[i] = 0;
    named_barrier(2, kScanThreads);
    // The warps are shared out over the new slots: several to one slot where there are few, one after another where many.
    constexpr int kScanWarps = kScanThreads / 32;
    const int32_t per_part = (p.b_vecs + p.splits - 1) / p.splits;
    const int32_t end = min(p.b_vecs, (rank + 1) * per_part);
    const int32_t team = max(1, kScanWarps / max(1, fresh));  // warps of a slot
    const int32_t teams = kScanWarps / team;
    const int32_t me = (i >> 5) % team, threads = team * 32;
    for (int32_t f = (i >> 5) / team; f < fresh; f += teams) {
      if ((i >> 5) >= team * teams) break;  // warps left over
      const uint4* from = p.b + static_cast<int64_t>(slot_adapter[fresh_slot[f]]) * p.b_vecs;
      bool bad = false;
      for (int32_t v0 = rank * per_part + me * 32 + lane; v0 < end; v0 += 16 * threads) {
        uint4 raw[16];  // all on their way at once: what bounds this is the latency of the loads
#pragma unroll
        for (int u = 0; u < 16; ++u)
          raw[u] = v0 + u * threads < end ? __ldg(from + v0 + u * threads) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int u = 0; u < 16; ++u) {
          const uint32_t words[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int q = 0; q < 4; ++q)  // bf16: all eight exponent bits set
            bad |= (words[q] & 0x7f80u) == 0x7f80u || (words[q] & 0x7f800000u) == 0x7f800000u;
        }
      }
      if (bad) seen[f] = 1;
    }
    named_barrier(2, kScanThreads);
    if (i < fresh) p.not_finite[static_cast<int64_t>(slot_adapter[fresh_slot[i]]) * kMaxSplits + rank] = seen[i] != 0 ? 1 : 0;
  } else {
    // ---- this block's part of V: TMEM lane = row
    const int quarter = warp & 3;
    const int lane_row = quarter * 32 + lane;
    // The row a thread drains is its TMEM lane, which is another row than the one it found the slot of.
    named_barrier(1, kTileRows);  // every worker has its slot: `work` may be used again
    work[row] = my_slot;
    named_barrier(1, kTileRows);
    const int32_t slot_here = work[lane_row];
    if (steps == 0 && slot_here >= 0)
      for (int32_t j = 0; j < p.rank; ++j) red[j * kTileRows + lane_row] = 0.0f;
    for (int32_t g = 0; steps > 0 && g < groups; ++g) {
      const uint32_t acc = static_cast<uint32_t>(g) & 1u;
      if (!ptx::mbar_wait_bounded(acc_full_bar + 8 * acc, (static_cast<uint32_t>(g) >> 1) & 1u, abort_word)) {
        give_up(SB_DEV_TIMEOUT_EPILOGUE);
        break;
      }
      ptx::tcgen05_fence_after_sync();
      const int32_t n = min(group_slots, slots - g * group_slots);
      for (int32_t s = 0; s < n; ++s) {
        const bool take = slot_here == g * group_slots + s;
        if (__ballot_sync(0xffffffffu, take) == 0u) continue;
        for (int32_t j = 0; j < p.rank; j += 8) {
          uint32_t v[8];
          ptx::tmem_ld_32x32b_x8(tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * kShrinkCols + s * p.rank + j, v);
          ptx::tmem_ld_wait();
          if (take) {
#pragma unroll
            for (int q = 0; q < 8; ++q) red[(j + q) * kTileRows + lane_row] = __uint_as_float(v[q]);
          }
        }
      }
      ptx::tcgen05_fence_before_sync();
      ptx::mbar_arrive(acc_empty_bar + 8 * acc);
    }
  }
  if (*abort_word != 0u) {
    for (int i = 0; i < 64; ++i) __nanosleep(1000);  // copies in flight land before the shared memory is handed back
  }
  __syncwarp();
  ptx::tcgen05_fence_before_sync();
  if (p.splits > 1) ptx::cluster_sync_all();
  else __syncthreads();
  if (warp == 1) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem_base, 2 * kShrinkCols);
  }
  if (worker && *abort_word == 0u) {
    // Eight values of a row per thread; the block's share of the rows is every splits-th.
    const int32_t pieces = p.rank / 8;
    const int32_t rows = (kTileRows - rank + p.splits - 1) / p.splits;
    for (int32_t i = row; i < rows * pieces; i += kTileRows) {
      const int32_t r = rank + (i % rows) * p.splits;
      const int32_t j0 = i / rows * 8;
      const int32_t a = id[r];
      if (a < 0) continue;
      float v[8];
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = 0.0f;
      for (int32_t part = 0; part < p.splits; ++part) {
        const uint32_t from = ptx::map_to_cta(red_base + static_cast<uint32_t>(j0 * kTileRows + r) * 4u, static_cast<uint32_t>(part));
#pragma unroll
        for (int q = 0; q < 8; ++q) v[q] += ptx::ld_cluster_f32(from + q * kTileRows * 4u);
      }
      const float factor = p.scale != nullptr ? __ldg(p.scale + a) : 1.0f;
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= factor;
      __nv_bfloat16* dst = p.v + static_cast<int64_t>(first_token + r) * p.rank * p.parts + j0;
      for (int32_t part = 0; part < p.parts; ++part) {
        uint32_t packed[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          packed[q] = pack_bf16(v[2 * q], v[2 * q + 1]);
          const float2 held = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&packed[q]));
          v[2 * q] = isfinite(held.x) ? v[2 * q] - held.x : 0.0f;
          v[2 * q + 1] = isfinite(held.y) ? v[2 * q + 1] - held.y : 0.0f;
        }
        *reinterpret_cast<uint4*>(dst + part * p.rank) = make_uint4(packed[0], packed[1], packed[2], packed[3]);
      }
    }
  }
  if (p.splits > 1) ptx::cluster_sync_all();  // nobody's shared memory is read any more
}

// ---- expand -------------------------------------------------------------------------------------------------------
// y on tiles of 128 tokens x 256 columns. The K steps behind D hold V in the columns of its slot: eight K rows at a time
// belong to one adapter, so slots of any rank that is a multiple of 8 share a step, and a tile of few slots has few steps
// (1 of 65 for one adapter of rank 64 at D = 4096). Bound by the tensor cores: T = 8191, 4096 x 4096, rank 64: 211 us,
// 1330 TFLOP/s, 82 % of the measured burst peak and of the issue rate at the clock it ran at. With x gathered by cp.async
// instead of TMA it was 290 us.
// Tiles are walked in bands of 8 row tiles, in a band the row tile changes fastest: 148 tiles in flight are then 8 row
// tiles x 18 column slices, whose x and W are small against L2 (bands of 2 to 16: the same 211 us, 64: 219).
struct LoraExpand {
  static constexpr int32_t kBand = 8;
  struct Params {
    int32_t row_tiles, slices;
    const int32_t* tables;
    const uint8_t* not_finite;
    const __nv_bfloat16* v;
    const __nv_bfloat16* b;
    int32_t num_tokens, width, rank, v_cols, base_steps, adapter_rows, cols, out_fp32, splits;  // v_cols = rank * parts
  };
  struct Tile {
    int32_t k_steps, base_steps, row_tile, n0, slots;
    const int32_t* table;
    bool live;
  };
  struct Rows { int32_t slot[8]; };
  struct Early { int32_t loner; };  // this row's adapter when its B is not finite, else -1
  static constexpr int kStages = 4, kEpilogueWarps = 8, kStaging = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = true, kExtension = true, kAMnMajor = false, kBMnMajor = true;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) { return p.row_tiles * p.slices; }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t;
    const int32_t band = index / (kBand * p.slices);
    const int32_t inside = index - band * (kBand * p.slices);
    const int32_t height = min(kBand, p.row_tiles - band * kBand);
    const int32_t slice = inside / height;
    t.row_tile = band * kBand + inside - slice * height;
    t.n0 = slice * p.cols;
    t.table = p.tables + static_cast<int64_t>(t.row_tile) * kTableInts;
    t.slots = __ldg(t.table);
    t.base_steps = p.base_steps;
    t.k_steps = p.base_steps + (t.slots * p.v_cols + kTileStep - 1) / kTileStep;
    t.live = true;
    return t;
  }
  static __device__ __forceinline__ int columns(const Params& p, const Tile&) { return p.cols; }
  static __device__ __forceinline__ int slabs(const Params& p) { return (p.cols + 63) >> 6; }
  static __device__ __forceinline__ uint32_t tx_bytes(const Params& p, const Tile& t, int32_t ks) {
    return static_cast<uint32_t>(slabs(p)) * TileSmem::kSlabBytes + (ks < t.base_steps ? TileSmem::kABytes : 0);
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    ptx::tma_load_2d(a, &maps.m[3], ks * kTileStep, t.row_tile * kTileRows, bar);
    const int n = slabs(p);
    for (int j = 0; j < n; ++j)
      ptx::tma_load_2d(b + j * TileSmem::kSlabBytes, &maps.m[0], t.n0 + j * 64, ks * kTileStep, bar);
  }
  // Eight K rows at a time: rows of one adapter's B, or of none (past the end, or not finite: zeros).
  static __device__ __forceinline__ int32_t extension_row(const Params& p, const Tile& t, int32_t ks, int piece) {
    const int32_t q = (ks - t.base_steps) * kTileStep + piece * 8;
    const int32_t slot = q / p.v_cols;
    if (slot >= t.slots) return p.adapter_rows;
    const int32_t a = __ldg(t.table + kSlotAdapter + slot);
    if (!adapter_finite(p.not_finite, a, p.splits)) return p.adapter_rows;
    return a * p.rank + (q - slot * p.v_cols) % p.rank;
  }
  static __device__ __forceinline__ void extension_load(const TileMaps& maps, const Params& p, const Tile& t, int piece,
                                                        int32_t row, uint32_t b, uint32_t bar) {
    const int n = slabs(p);
    for (int j = 0; j < n; ++j)
      ptx::tma_load_2d(b + j * TileSmem::kSlabBytes + piece * 1024, &maps.m[1], t.n0 + j * 64, row, bar);
  }
  static __device__ __forceinline__ Rows rows(const Params& p, const Tile& t, int row0) {
    Rows r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r.slot[j] = __ldg(t.table + kRowSlot + row0 + j * 16);
      if (r.slot[j] >= 0 && !adapter_finite(p.not_finite, __ldg(t.table + kSlotAdapter + r.slot[j]), p.splits)) r.slot[j] = -1;
    }
    return r;
  }
  static __device__ __forceinline__ uint4 extension_chunk(const Params& p, const Tile& t, const Rows& r, int j, int row,
                                                          int32_t ks, int chunk) {
    const int32_t q = (ks - t.base_steps) * kTileStep + chunk * 8;
    const int32_t slot = q / p.v_cols;
    if (r.slot[j] != slot) return make_uint4(0u, 0u, 0u, 0u);  // rows past the end have no slot
    const int64_t token = static_cast<int64_t>(t.row_tile) * kTileRows + row;
    return __ldg(reinterpret_cast<const uint4*>(p.v + token * p.v_cols + (q - slot * p.v_cols)));
  }
  static __device__ __forceinline__ Early prefetch(const Params& p, const Tile& t, const EpilogueWarp& w) {
    const int32_t slot = __ldg(t.table + kRowSlot + w.quarter * 32 + w.lane);
    if (slot < 0) return {-1};
    const int32_t a = __ldg(t.table + kSlotAdapter + slot);
    return {adapter_finite(p.not_finite, a, p.splits) ? -1 : a};
  }
  static __device__ __forceinline__ void epilogue(const TileMaps& maps, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    const int32_t row = t.row_tile * kTileRows + w.quarter * 32;
    if (row >= p.num_tokens) return;
    const bool loners = __ballot_sync(0xffffffffu, early.loner >= 0) != 0u;
    const int32_t end = min(t.n0 + p.cols, p.width);
#pragma unroll 1
    for (int32_t col = t.n0 + w.part * 64; col < end; col += 128) {
      uint32_t packed[32];
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint32_t v[32];
        ptx::tmem_ld_32x32b_x32(w.taddr + (col - t.n0) + part * 32, v);
        ptx::tmem_ld_wait();
        if (loners && early.loner >= 0) {
          const __nv_bfloat16* vr = p.v + static_cast<int64_t>(row + w.lane) * p.v_cols;
          for (int32_t j = 0; j < p.rank; ++j) {
            // The parts of V add up to V before they meet B: a part of 0 or of the other sign times infinity is not V's.
            float f = 0.0f;
            for (int32_t q = p.v_cols - p.rank + j; q >= 0; q -= p.rank) f += __bfloat162float(__ldg(vr + q));
            const __nv_bfloat16* br = p.b + (static_cast<int64_t>(early.loner) * p.rank + j) * p.width;
#pragma unroll
            for (int h = 0; h < 32; ++h) {
              const int32_t c = col + part * 32 + h;
              if (c < p.width) v[h] = __float_as_uint(fmaf(f, __bfloat162float(__ldg(br + c)), __uint_as_float(v[h])));
            }
          }
        }
        if (p.out_fp32) {
          if (col + part * 32 < p.width) store_rows_128b(w, &maps.m[2], v, col + part * 32, row);
        } else {
#pragma unroll
          for (int h = 0; h < 16; ++h)
            packed[part * 16 + h] = pack_bf16(__uint_as_float(v[2 * h]), __uint_as_float(v[2 * h + 1]));
        }
      }
      if (!p.out_fp32) store_rows_128b(w, &maps.m[2], packed, col, row);
    }
  }
};

// ---- a decoding step -----------------------------------------------------------------------------------------------

// V[t, j] = scale[a] * x[t] . A[a, j] in fp32, a block each (with one warp the row's loads would wait for each other);
// tokens without an adapter are left out here and later.
constexpr int kRowsThreads = 256;
template <typename index_t>
__global__ void __launch_bounds__(kRowsThreads)
lora_rows_kernel(const uint4* __restrict__ x, const uint4* __restrict__ a, const index_t* __restrict__ adapter_idx,
                 const float* __restrict__ scale, float* __restrict__ v, int32_t num_adapters, int32_t rank, int32_t vecs) {
  __shared__ float warp_sum[kRowsThreads / 32];
  ptx::grid_launch_dependents();
  const int32_t t = static_cast<int32_t>(blockIdx.x);
  const int32_t j = static_cast<int32_t>(blockIdx.y);
  const int64_t id = static_cast<int64_t>(__ldg(adapter_idx + t));
  if (id < 0 || id >= num_adapters) return;
  const uint4* xr = x + static_cast<int64_t>(t) * vecs;
  const uint4* ar = a + (id * rank + j) * vecs;
  float sum = 0.0f;
#pragma unroll 2
  for (int32_t i = static_cast<int32_t>(threadIdx.x); i < vecs; i += kRowsThreads) {
    const uint4 xq = __ldg(xr + i);
    const uint4 aq = __ldg(ar + i);
    const __nv_bfloat162* xp = reinterpret_cast<const __nv_bfloat162*>(&xq);
    const __nv_bfloat162* ap = reinterpret_cast<const __nv_bfloat162*>(&aq);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float2 xf = __bfloat1622float2(xp[q]);
      const float2 af = __bfloat1622float2(ap[q]);
      sum = fmaf(xf.x, af.x, sum);
      sum = fmaf(xf.y, af.y, sum);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kRowsThreads / 32; ++w) sum += warp_sum[w];
    v[static_cast<int64_t>(t) * rank + j] = scale != nullptr ? sum * __ldg(scale + id) : sum;
  }
}

// y: 128 columns of x W by the tensor cores; the workers compute the adapters' term of their share of the tokens while
// the weights stream (thread: 8 columns of every 8th token), and add it to the sums of the splits.
template <int kPasses>
struct SkinnyLora {
  struct Params {
    SkinnyShape shape;
    const void* adapter_idx;
    const float* v;
    const __nv_bfloat16* b;
    void* out;
    int32_t idx_is_i64, num_tokens, num_adapters, rank, width, out_fp32;
  };
  struct Item { int32_t n0, rows; };
  struct Extra { float y[kPasses][8]; };
  static constexpr bool kGather = false;
  static __device__ __forceinline__ bool begin(const Params& p, Item& item, int32_t block_item, int32_t*, int32_t*) {
    item.n0 = block_item * kSkinnyCols;
    item.rows = p.num_tokens;
    return true;
  }
  static __device__ __forceinline__ void load_w(const SkinnyMaps& maps, const Params&, const Item& item, int32_t ks, uint32_t dst,
                                                uint32_t bar) {
    ptx::tma_load_2d(dst, &maps.w[0], item.n0, ks * kSkinnyStep, bar);
    ptx::tma_load_2d(dst + kSkinnyWBytes / 2, &maps.w[0], item.n0 + 64, ks * kSkinnyStep, bar);
  }
  static __device__ __forceinline__ int32_t token(const Params& p, int32_t rank, int worker, int pass) {
    return rank + p.shape.splits * (pass * 8 + (worker >> 4));
  }
  static __device__ __forceinline__ void extra(const Params& p, const Item& item, int32_t rank, int worker, Extra& e) {
    const int32_t col = item.n0 + (worker & 15) * 8;
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
#pragma unroll
      for (int q = 0; q < 8; ++q) e.y[pass][q] = 0.0f;
      const int32_t t = token(p, rank, worker, pass);
      if (t >= p.num_tokens || col >= p.width) continue;
      const int64_t a = p.idx_is_i64 ? __ldg(static_cast<const long long*>(p.adapter_idx) + t)
                                     : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(p.adapter_idx) + t));
      if (a < 0 || a >= p.num_adapters) continue;
      const uint4* b = reinterpret_cast<const uint4*>(p.b + a * p.rank * p.width + col);
      const float* v = p.v + static_cast<int64_t>(t) * p.rank;
      const int32_t stride = p.width / 8;
      for (int32_t j = 0; j < p.rank; j += 8) {
        uint4 raw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) raw[i] = __ldg(b + static_cast<int64_t>(j + i) * stride);
        float f[8];
        *reinterpret_cast<float4*>(f) = __ldcg(reinterpret_cast<const float4*>(v + j));
        *reinterpret_cast<float4*>(f + 4) = __ldcg(reinterpret_cast<const float4*>(v + j + 4));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const __nv_bfloat162* pair = reinterpret_cast<const __nv_bfloat162*>(&raw[i]);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 bf = __bfloat1622float2(pair[q]);
            e.y[pass][2 * q] = fmaf(f[i], bf.x, e.y[pass][2 * q]);
            e.y[pass][2 * q + 1] = fmaf(f[i], bf.y, e.y[pass][2 * q + 1]);
          }
        }
      }
    }
  }
  static __device__ __forceinline__ void finish(const Params& p, const Item& item, const int32_t*, int32_t rank, int worker,
                                                const SkinnySums& red, const Extra& e) {
    const int32_t c = (worker & 15) * 8;
    if (item.n0 + c >= p.width) return;
#pragma unroll
    for (int pass = 0; pass < kPasses; ++pass) {
      const int32_t t = token(p, rank, worker, pass);
      if (t >= p.num_tokens) break;
      float v[8];
      red.sum(t, c, v);
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] += e.y[pass][q];
      const int64_t at = static_cast<int64_t>(t) * p.width + item.n0 + c;
      if (p.out_fp32) {
        float4* dst = reinterpret_cast<float4*>(static_cast<float*>(p.out) + at);
        dst[0] = make_float4(v[0], v[1], v[2], v[3]);
        dst[1] = make_float4(v[4], v[5], v[6], v[7]);
      } else {
        *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.out) + at) =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      }
    }
  }
};

template <int kPasses>
int launch_lora_small(const SkinnyMaps& maps, const SkinnyShape& shape, const void* adapter_idx, int idx_is_i64, const float* v,
                      const void* lora_b, void* out, int out_fp32, int32_t num_tokens, int32_t width, int32_t rank,
                      int32_t num_adapters, int64_t items, int32_t* dev_status, cudaStream_t stream) {
  typename SkinnyLora<kPasses>::Params p{};
  p.shape = shape;
  p.adapter_idx = adapter_idx;
  p.v = v;
  p.b = static_cast<const __nv_bfloat16*>(lora_b);
  p.out = out;
  p.idx_is_i64 = idx_is_i64;
  p.num_tokens = num_tokens;
  p.num_adapters = num_adapters;
  p.rank = rank;
  p.width = width;
  p.out_fp32 = out_fp32;
  return launch_skinny<SkinnyLora<kPasses>>(maps, p, items, true, dev_status, stream, "lora_linear (small)");
}

int lora_small(const void* x, const void* weight, const void* lora_a, const void* lora_b, const void* adapter_idx,
               int idx_is_i64, const float* scale, void* out, int out_fp32, int32_t num_tokens, int32_t d_model, int32_t width,
               int32_t rank, int32_t num_adapters, float* v, const DeviceInfo* info, int32_t* dev_status, cudaStream_t stream) {
  const int64_t items = (width + kSkinnyCols - 1) / kSkinnyCols;
  const SkinnyShape shape = skinny_shape(items, (d_model + kSkinnyStep - 1) / kSkinnyStep, num_tokens, info->sm_count);
  SkinnyMaps maps{};
  if (int rc = encode_2d_map(&maps.w[0], weight, d_model, width, 64, 64, 2, "lora_linear (weight)")) return rc;
  if (int rc = encode_2d_map(&maps.x, x, num_tokens, d_model, shape.rows_pad, 64, 2, "lora_linear (x)")) return rc;
  const dim3 grid(static_cast<unsigned>(num_tokens), static_cast<unsigned>(rank));
  if (idx_is_i64)
    lora_rows_kernel<long long><<<grid, kRowsThreads, 0, stream>>>(static_cast<const uint4*>(x), static_cast<const uint4*>(lora_a),
        static_cast<const long long*>(adapter_idx), scale, v, num_adapters, rank, d_model / 8);
  else
    lora_rows_kernel<int32_t><<<grid, kRowsThreads, 0, stream>>>(static_cast<const uint4*>(x), static_cast<const uint4*>(lora_a),
        static_cast<const int32_t*>(adapter_idx), scale, v, num_adapters, rank, d_model / 8);
  if (int rc = check_launch("lora_linear (rows)")) return rc;
  const int32_t per_rank = (num_tokens + shape.splits - 1) / shape.splits;  // tokens of a block, 8 at a time
#define SB_LORA_SMALL(PASSES)                                                                                               \
  launch_lora_small<PASSES>(maps, shape, adapter_idx, idx_is_i64, v, lora_b, out, out_fp32, num_tokens, width, rank,         \
                            num_adapters, items, dev_status, stream)
  if (per_rank <= 8) return SB_LORA_SMALL(1);
  if (per_rank <= 16) return SB_LORA_SMALL(2);
  if (per_rank <= 32) return SB_LORA_SMALL(4);
  return SB_LORA_SMALL(8);
#undef SB_LORA_SMALL
}

struct LoraSizes {
  int64_t row_tiles, tables, not_finite, v, total;  // bytes of each part, 256-byte aligned, then all
  int32_t splits, steps, total_steps, parts;
};

LoraSizes lora_sizes(int64_t num_tokens, int32_t d_model, int32_t rank, int32_t num_adapters, int out_fp32, int sm_count) {
  LoraSizes s{};
  if (num_tokens <= kSmallTokens) {
    s.v = align256(num_tokens * rank * 4);
    s.total = s.v;
    return s;
  }
  s.row_tiles = (num_tokens + kTileRows - 1) / kTileRows;
  s.parts = out_fp32 ? 3 : 1;
  s.total_steps = (d_model + kTileStep - 1) / kTileStep;
  // Parts of D for few row tiles: up to a block per SM, each of at least 4 K steps.
  s.splits = 1;
  while (s.splits < kMaxSplits && s.row_tiles * s.splits * 2 <= sm_count && s.total_steps >= 8 * s.splits) s.splits *= 2;
  s.steps = (s.total_steps + s.splits - 1) / s.splits;
  s.tables = align256(s.row_tiles * kTableInts * 4);
  s.not_finite = align256(static_cast<int64_t>(num_adapters) * kMaxSplits);
  s.v = align256(num_tokens * rank * s.parts * 2);
  s.total = s.tables + s.not_finite + s.v;
  return s;
}

int check_lora(int64_t num_tokens, int32_t d_model, int32_t width, int32_t rank, int32_t num_adapters) {
  if (num_tokens < 0 || num_tokens > INT32_MAX - kTileRows) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: T must fit 31 bits");
  if (d_model <= 0 || d_model % 8 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: D (%d) must be a positive multiple of 8", d_model);
  if (width <= 0 || width % 8 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: N (%d) must be a positive multiple of 8", width);
  // Column and K indexes run up to a tile past the end; an adapter's B is counted in pieces of 16 bytes, up to 16 per thread
  // of the scan past its end.
  if (d_model > INT32_MAX - kTileCols || width > INT32_MAX - kTileCols)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: D (%d) or N (%d) is too large", d_model, width);
  if (rank <= 0 || rank % 8 != 0 || rank > 128)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the rank (%d) must be a multiple of 8 in [8, 128]", rank);
  if (num_tokens > kSmallTokens && static_cast<int64_t>(rank) * (width / 8) > INT32_MAX - 16 * kScanThreads)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the rank (%d) times N (%d) is too large", rank, width);
  if (num_adapters <= 0 || static_cast<int64_t>(num_adapters) * rank > INT32_MAX - kTileCols)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the number of adapters (%d) must be positive, and times the rank fit 31 bits", num_adapters);
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int64_t sb_lora_workspace_bytes(int64_t num_tokens, int32_t d_model, int32_t width, int32_t rank,
                                           int32_t num_adapters, int out_fp32) {
  clear_error();
  if (check_lora(num_tokens, d_model, width, rank, num_adapters) != SB_OK) return -1;
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return -1;
  return lora_sizes(num_tokens, d_model, rank, num_adapters, out_fp32, info->sm_count).total;
}

extern "C" int sb_lora_linear(const void* x, const void* weight, const void* lora_a, const void* lora_b,
                              const void* adapter_idx, int idx_is_i64, const float* scale, void* out, int out_fp32,
                              int64_t num_tokens, int32_t d_model, int32_t width, int32_t rank, int32_t num_adapters,
                              void* workspace, int64_t workspace_bytes, int32_t* dev_status, sb_stream_t stream) {
  clear_error();
  if (int rc = check_lora(num_tokens, d_model, width, rank, num_adapters)) return rc;
  if (num_tokens == 0) return SB_OK;
  if (!x || !weight || !lora_a || !lora_b || !adapter_idx || !out || !workspace)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: NULL buffer");
  for (const void* q : {x, weight, lora_a, lora_b, static_cast<const void*>(out), static_cast<const void*>(workspace)})
    if (!aligned16(q)) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: buffers must be 16-byte aligned");
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const LoraSizes s = lora_sizes(num_tokens, d_model, rank, num_adapters, out_fp32, info->sm_count);
  if (workspace_bytes < s.total)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the workspace has %lld bytes, %lld are needed",
                (long long)workspace_bytes, (long long)s.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (num_tokens <= kSmallTokens)
    return lora_small(x, weight, lora_a, lora_b, adapter_idx, idx_is_i64, scale, out, out_fp32, static_cast<int32_t>(num_tokens),
                      d_model, width, rank, num_adapters, reinterpret_cast<float*>(ws), info, dev_status, as_stream(stream));
  int32_t* tables = reinterpret_cast<int32_t*>(ws);
  uint8_t* not_finite = ws + s.tables;
  __nv_bfloat16* v = reinterpret_cast<__nv_bfloat16*>(not_finite + s.not_finite);
  const cudaStream_t st = as_stream(stream);
  const int32_t tokens = static_cast<int32_t>(num_tokens);
  const int32_t row_tiles = static_cast<int32_t>(s.row_tiles);
  {
    ShrinkMaps maps{};
    if (int rc = encode_2d_map(&maps.x, x, num_tokens, d_model, kTileRows, 64, 2, "lora_linear (x)")) return rc;
    if (int rc = encode_2d_map(&maps.a, lora_a, static_cast<uint64_t>(num_adapters) * rank, d_model, rank, 64, 2, "lora_linear (A)")) return rc;
    ShrinkParams p{};
    p.adapter_idx = adapter_idx;
    p.b = static_cast<const uint4*>(lora_b);
    p.scale = scale;
    p.tables = tables;
    p.not_finite = not_finite;
    p.v = v;
    p.idx_is_i64 = idx_is_i64;
    p.num_tokens = tokens;
    p.num_adapters = num_adapters;
    p.rank = rank;
    p.parts = s.parts;
    p.splits = s.splits;
    p.steps = s.steps;
    p.total_steps = s.total_steps;
    p.b_vecs = rank * (width / 8);
    p.stages = std::min(6, (225 * 1024 - 1024 - kShrinkHeadBytes - kTileRows * rank * 4) / kShrinkStageBytes);
    int device = 0;
    if (current_device_info(&device) == nullptr) return SB_ERR_CUDA;
    static std::atomic<bool> done[kMaxDevices] = {};
    if (!done[device].load(std::memory_order_acquire)) {
      const cudaError_t err = cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 225 * 1024);
      if (err != cudaSuccess) return fail(SB_ERR_CUDA, "lora_linear: shared memory opt-in: %s", cudaGetErrorString(err));
      done[device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(row_tiles * s.splits));
    cfg.blockDim = dim3(kShrinkThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(shrink_smem_bytes(p.stages, rank));
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(s.splits);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, lora_shrink_kernel, maps, p, dev_status);
    if (err != cudaSuccess) return fail(SB_ERR_CUDA, "lora_linear (shrink): %s", cudaGetErrorString(err));
  }

  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], weight, d_model, width, 64, 64, 2, "lora_linear (weight)")) return rc;
  if (int rc = encode_2d_map(&maps.m[1], lora_b, static_cast<uint64_t>(num_adapters) * rank, width, 8, 64, 2, "lora_linear (B)")) return rc;
  if (int rc = encode_2d_map(&maps.m[2], out, num_tokens, width, 32, out_fp32 ? 32 : 64, out_fp32 ? 4 : 2, "lora_linear (out)")) return rc;
  if (int rc = encode_2d_map(&maps.m[3], x, num_tokens, d_model, kTileRows, 64, 2, "lora_linear (x)")) return rc;
  LoraExpand::Params p{};
  // Columns of a tile: 256, and fewer where not even a quarter of the SMs has one: a step's bytes come sooner (with four
  // adapters of rank 16, T = 128, D = N = 4096: 38.9 -> 34.9 us; T = 342, D = 2336, N = 264, 17 adapters: 47.1 -> 35.0 us).
  // With more tiles than that the rows of x, read once more per tile, cost more (T = 512, D = N = 4096: 41.0 -> 56.8 us).
  int32_t cols = kTileCols;
  while (cols > 64 && 4 * s.row_tiles * ((width + cols - 1) / cols) <= info->sm_count) cols /= 2;
  const int32_t slices = (width + cols - 1) / cols;
  p.row_tiles = row_tiles;
  p.slices = slices;
  p.tables = tables;
  p.not_finite = not_finite;
  p.splits = s.splits;
  p.v = v;
  p.b = static_cast<const __nv_bfloat16*>(lora_b);
  p.num_tokens = tokens;
  p.width = width;
  p.rank = rank;
  p.v_cols = rank * s.parts;
  p.base_steps = s.total_steps;
  p.adapter_rows = num_adapters * rank;
  p.cols = width >= cols ? cols : (width + 15) & ~15;
  p.out_fp32 = out_fp32 ? 1 : 0;
  return launch_tile_gemm<LoraExpand>(maps, p, static_cast<int64_t>(row_tiles) * slices, dev_status, st, "lora_linear (expand)");
}
