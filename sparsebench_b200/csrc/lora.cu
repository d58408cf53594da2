// A projection with the low-rank adapters of many requests at once:
//
//   y[t] = x[t] W + scale[a] * sum_j (x[t] . A[a, j]) B[a, j],   a = adapter_idx[t]   (outside [0, L): no second term)
//
// The products run on tiles of 128 consecutive tokens. A tile's distinct adapters are its slots, in order of first
// appearance (a batch is its requests' tokens one after another, so a tile has few). Per call:
//
//   plan     slots of every tile; which of the used adapters have a B that is not finite
//   shrink   V = x A[a]^T: the rows of all slots' A side by side are the columns of one product, of which each token
//            keeps its own slot's; split over D, joined in a fixed order with the scale
//   expand   y = [x | V in its slot's columns, zeros elsewhere] [W ; B of the slots]: the second term is a few more K
//            steps of the projection itself, so y is written once and never read back
//
// Up to 64 tokens (a decoding step) the weights are streamed by the kernel of skinny.cuh and the second term is plain
// fp32 arithmetic on each token's own rows of A and B (lora_rows_kernel, SkinnyLora): no plan, no pairing of tokens.
//
// In the products V is rounded to bf16 for y in bf16; for y in fp32 it travels as a pair of bf16 (V and what rounding took from it,
// against the same rows of B), 2^-17 of V off.
//
// There a zero of V meets B of other requests' adapters: an infinity or NaN in one adapter would reach its neighbours'
// rows. So an adapter whose B is not finite stays out of the product (plan finds it, reading B once, on its way into
// L2) and its own rows get their term from the epilogue, number by number.

#include <algorithm>
#include <initializer_list>

#include "skinny.cuh"
#include "tile_gemm.cuh"

namespace sb {
namespace {

constexpr int kMaxSlots = kTileRows;
// Per tile: the slot count, the adapter of each slot, the slot of each row (-1: none), and again the adapter of each slot,
// or -1 where its B is not finite.
constexpr int kSlotAdapter = 1, kRowSlot = kSlotAdapter + kMaxSlots, kSlotShared = kRowSlot + kTileRows;
constexpr int kTableInts = kSlotShared + kMaxSlots;
constexpr int kPlanThreads = 256;

// ---- plan ---------------------------------------------------------------------------------------------------------

// Block (tile, part): the tile's slots; part 0 writes them down, and every part looks through its part of the B of those
// of the tile's adapters that the tile before does not have (they are being looked through there, or further up). For a
// batch of whole requests that is once per request; in any order it is at most what expand reads of B anyway. Tiles that
// share an adapter write the same answer.
template <typename index_t>
__global__ void __launch_bounds__(kPlanThreads)
lora_plan_kernel(const index_t* __restrict__ adapter_idx, const uint4* __restrict__ b, int32_t* __restrict__ tables,
                 uint8_t* __restrict__ not_finite, int32_t num_tokens, int32_t num_adapters, int32_t vecs_per_adapter) {
  __shared__ alignas(16) int32_t id[kTileRows];
  __shared__ int32_t slot_adapter[kMaxSlots];
  __shared__ int32_t slot_of_first[kTileRows];
  __shared__ int32_t warp_count[4];
  __shared__ int32_t seen[kMaxSlots];
  ptx::grid_launch_dependents();
  const int i = static_cast<int>(threadIdx.x);
  const int32_t first_token = static_cast<int32_t>(blockIdx.x) * kTileRows;
  int32_t mine = -1;
  if (i < kTileRows) {
    if (first_token + i < num_tokens) {
      const int64_t a = static_cast<int64_t>(__ldg(adapter_idx + first_token + i));
      if (a >= 0 && a < num_adapters) mine = static_cast<int32_t>(a);
    }
    id[i] = mine;
    seen[i] = 0;
  }
  __syncthreads();
  int first = i;
  if (i < kTileRows && mine >= 0) {
    for (int j = 0; j < i; j += 4) {
      const int4 four = *reinterpret_cast<const int4*>(id + j);
      if (four.x == mine) { first = j; break; }
      if (four.y == mine) { first = j + 1; break; }
      if (four.z == mine) { first = j + 2; break; }
      if (four.w == mine) { first = j + 3; break; }
    }
  }
  const bool leads = i < kTileRows && mine >= 0 && first == i;  // first never lies behind i: id[i] itself matches
  const unsigned ballot = __ballot_sync(0xffffffffu, leads);
  if (i < kTileRows && (i & 31) == 0) warp_count[i >> 5] = __popc(ballot);
  __syncthreads();
  int32_t slots = 0, slot = __popc(ballot & ((1u << (i & 31)) - 1u));
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < (i >> 5)) slot += warp_count[w];
    slots += warp_count[w];
  }
  if (leads) {
    slot_adapter[slot] = mine;
    slot_of_first[i] = slot;
  }
  __syncthreads();
  if (blockIdx.y == 0) {
    int32_t* table = tables + static_cast<int64_t>(blockIdx.x) * kTableInts;
    if (i == 0) table[0] = slots;
    if (i < slots) table[kSlotAdapter + i] = slot_adapter[i];
    if (i < kTileRows) table[kRowSlot + i] = mine >= 0 ? slot_of_first[first] : -1;
  }
  if (i < kTileRows && first_token > 0) {
    const int64_t a = static_cast<int64_t>(__ldg(adapter_idx + first_token - kTileRows + i));
    for (int32_t s = 0; s < slots; ++s)
      if (slot_adapter[s] == a) seen[s] = 1;
  }
  __syncthreads();
  const int32_t parts = static_cast<int32_t>(gridDim.y);
  const int32_t per_part = (vecs_per_adapter + parts - 1) / parts;
  const int32_t begin = static_cast<int32_t>(blockIdx.y) * per_part;
  const int32_t end = min(vecs_per_adapter, begin + per_part);
  for (int32_t s = 0; s < slots; ++s) {
    if (seen[s] != 0) continue;
    const int32_t a = slot_adapter[s];
    const uint4* rows = b + static_cast<int64_t>(a) * vecs_per_adapter;
    bool bad = false;
#pragma unroll 4
    for (int32_t v = begin + i; v < end; v += kPlanThreads) {
      const uint4 raw = __ldg(rows + v);
      const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int q = 0; q < 4; ++q)  // bf16: all eight exponent bits set
        bad |= (words[q] & 0x7f80u) == 0x7f80u || (words[q] & 0x7f800000u) == 0x7f800000u;
    }
    const int any = __syncthreads_or(bad);
    if (i == 0) not_finite[static_cast<int64_t>(a) * parts + blockIdx.y] = any ? 1 : 0;
  }
}

// ---- shrink -------------------------------------------------------------------------------------------------------
// One tile = 128 tokens x the slots of one group (as many as fit 256 columns) x one part of D.
struct LoraShrink {
  struct Params {
    const int32_t* tables;
    float* partial;  // [splits, T, r]
    int32_t num_tokens, rank, row_tiles, groups, group_slots, splits, steps, total_steps;  // steps: per split
  };
  struct Tile {
    int32_t k_steps, row_tile, first_slot, slots, step0, split;
    const int32_t* adapters;
    bool live;
  };
  struct Early { int32_t slot; };
  static constexpr int kStages = 4, kEpilogueWarps = 8, kBuffers = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = true, kExtension = false, kAMnMajor = false, kBMnMajor = false;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) { return p.row_tiles * p.groups * p.splits; }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t;
    // Groups past a tile's slots are dead: the group is the slowest index, so the live tiles come first.
    const int32_t group = index / (p.row_tiles * p.splits);
    const int32_t rest = index - group * (p.row_tiles * p.splits);
    t.row_tile = rest / p.splits;
    t.split = rest - t.row_tile * p.splits;
    const int32_t* table = p.tables + static_cast<int64_t>(t.row_tile) * kTableInts;
    t.first_slot = group * p.group_slots;
    t.slots = min(p.group_slots, __ldg(table) - t.first_slot);
    t.adapters = table + kSlotAdapter + t.first_slot;
    t.step0 = t.split * p.steps;
    t.live = t.slots > 0;
    t.k_steps = t.live ? min(p.steps, p.total_steps - t.step0) : 0;
    return t;
  }
  static __device__ __forceinline__ int columns(const Params& p) { return (p.group_slots * p.rank + 15) & ~15; }
  static __device__ __forceinline__ uint32_t tx_bytes(const Params& p, const Tile& t, int32_t) {
    return TileSmem::kABytes + static_cast<uint32_t>(t.slots * p.rank) * 128u;
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    const int32_t k = (t.step0 + ks) * kTileStep;
    ptx::tma_load_2d(a, &maps.m[0], k, t.row_tile * kTileRows, bar);
    for (int32_t s = 0; s < t.slots; ++s)
      ptx::tma_load_2d(b + static_cast<uint32_t>(s * p.rank) * 128u, &maps.m[1], k, __ldg(t.adapters + s) * p.rank, bar);
  }
  static __device__ __forceinline__ Early prefetch(const Params& p, const Tile& t, const EpilogueWarp& w) {
    return {__ldg(p.tables + static_cast<int64_t>(t.row_tile) * kTableInts + kRowSlot + w.quarter * 32 + w.lane)};
  }
  static __device__ __forceinline__ void epilogue(const TileMaps&, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    const int32_t token = t.row_tile * kTileRows + w.quarter * 32 + w.lane;
    float* dst = p.partial + (static_cast<int64_t>(t.split) * p.num_tokens + token) * p.rank;
    for (int32_t s = w.part; s < t.slots; s += 2) {  // the two warps of a quarter share the slots
      const bool mine = early.slot == t.first_slot + s;
      if (__ballot_sync(0xffffffffu, mine) == 0u) continue;
      for (int32_t j = 0; j < p.rank; j += 8) {
        uint32_t v[8];
        ptx::tmem_ld_32x32b_x8(w.taddr + s * p.rank + j, v);
        ptx::tmem_ld_wait();
        if (mine) {
          *reinterpret_cast<uint4*>(dst + j) = make_uint4(v[0], v[1], v[2], v[3]);
          *reinterpret_cast<uint4*>(dst + j + 4) = make_uint4(v[4], v[5], v[6], v[7]);
        }
      }
    }
  }
};

// V[t] = scale * sum over the parts, in order, as one bf16 (parts = 1) or as a pair (parts = 2: r values, then r
// remainders). Tokens without an adapter are not read later and not written. Also the last column of the tables.
template <typename index_t>
__global__ void __launch_bounds__(256)
lora_join_kernel(const float* __restrict__ partial, const index_t* __restrict__ adapter_idx, const float* __restrict__ scale,
                 __nv_bfloat16* __restrict__ v, int32_t num_tokens, int32_t num_adapters, int32_t rank, int32_t splits,
                 int32_t parts, int32_t* __restrict__ tables, const uint8_t* __restrict__ not_finite, int32_t row_tiles,
                 int32_t scan_parts) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  const int64_t start = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (int64_t i = start; i < static_cast<int64_t>(row_tiles) * kMaxSlots; i += stride) {
    int32_t* table = tables + i / kMaxSlots * kTableInts;
    const int32_t s = static_cast<int32_t>(i % kMaxSlots);
    if (s >= __ldcg(table)) continue;
    int32_t a = __ldcg(table + kSlotAdapter + s);
    const uint8_t* flags = not_finite + static_cast<int64_t>(a) * scan_parts;
    unsigned bad = 0;
    for (int32_t q = 0; q < scan_parts; ++q) bad |= __ldcg(flags + q);
    table[kSlotShared + s] = bad != 0 ? -1 : a;
  }
  const int64_t total = static_cast<int64_t>(num_tokens) * rank;
  for (int64_t i = start; i < total; i += stride) {
    const int32_t t = static_cast<int32_t>(i / rank);
    const int32_t j = static_cast<int32_t>(i - static_cast<int64_t>(t) * rank);
    const int64_t a = static_cast<int64_t>(__ldg(adapter_idx + t));
    if (a < 0 || a >= num_adapters) continue;
    float sum = 0.0f;
    for (int32_t s = 0; s < splits; ++s) sum += __ldcg(partial + s * total + i);
    if (scale != nullptr) sum *= __ldg(scale + a);
    const __nv_bfloat16 high = __float2bfloat16_rn(sum);
    __nv_bfloat16* row = v + static_cast<int64_t>(t) * rank * parts;
    row[j] = high;
    if (parts == 2) row[rank + j] = __float2bfloat16_rn(isfinite(__bfloat162float(high)) ? sum - __bfloat162float(high) : 0.0f);
  }
}

// ---- expand -------------------------------------------------------------------------------------------------------
struct LoraExpand {
  struct Params {
    BandOrder order;
    const int32_t* tables;
    const __nv_bfloat16* v;
    const __nv_bfloat16* b;
    int32_t num_tokens, width, rank, v_cols, base_steps, adapter_rows, cols, out_fp32;  // v_cols = rank * parts
  };
  struct Tile {
    int32_t k_steps, base_steps, row_tile, n0, slots;
    const int32_t* table;
    bool live;
  };
  struct Rows { int32_t slot[8]; };
  struct Early { int32_t loner; };  // this row's adapter when its B is not finite, else -1
  static constexpr int kStages = 4, kEpilogueWarps = 8, kBuffers = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = true, kExtension = true, kAMnMajor = false, kBMnMajor = true;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) { return p.order.num_row_blocks * p.order.num_slices; }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t;
    int32_t slice;
    p.order.at(index, &t.row_tile, &slice);
    t.n0 = slice * kTileCols;
    t.table = p.tables + static_cast<int64_t>(t.row_tile) * kTableInts;
    t.slots = __ldg(t.table);
    t.base_steps = p.base_steps;
    t.k_steps = p.base_steps + (t.slots * p.v_cols + kTileStep - 1) / kTileStep;
    t.live = true;
    return t;
  }
  static __device__ __forceinline__ int columns(const Params& p) { return p.cols; }
  static __device__ __forceinline__ int slabs(const Params& p) { return (p.cols + 63) >> 6; }
  static __device__ __forceinline__ uint32_t tx_bytes(const Params& p, const Tile& t, int32_t ks) {
    return static_cast<uint32_t>(slabs(p)) * TileSmem::kSlabBytes + (ks < t.base_steps ? TileSmem::kABytes : 0);
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    const int n = slabs(p);
    if (ks < t.base_steps) {
      ptx::tma_load_2d(a, &maps.m[3], ks * kTileStep, t.row_tile * kTileRows, bar);
      for (int j = 0; j < n; ++j)
        ptx::tma_load_2d(b + j * TileSmem::kSlabBytes, &maps.m[0], t.n0 + j * 64, ks * kTileStep, bar);
      return;
    }
    // Eight K rows at a time: rows of one adapter's B, or of none (past the end, or not finite: zeros).
    int32_t row[8];
#pragma unroll
    for (int g = 0; g < 8; ++g) {
      const int32_t q = (ks - t.base_steps) * kTileStep + g * 8;
      const int32_t slot = q / p.v_cols;
      const int32_t a_id = slot < t.slots ? __ldg(t.table + kSlotShared + slot) : -1;
      int32_t j = q - slot * p.v_cols;
      if (j >= p.rank) j -= p.rank;
      row[g] = a_id >= 0 ? a_id * p.rank + j : p.adapter_rows;
    }
#pragma unroll
    for (int g = 0; g < 8; ++g)
      for (int j = 0; j < n; ++j)
        ptx::tma_load_2d(b + j * TileSmem::kSlabBytes + g * 1024, &maps.m[1], t.n0 + j * 64, row[g], bar);
  }
  static __device__ __forceinline__ Rows rows(const Params&, const Tile& t, int row0) {
    Rows r;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      r.slot[j] = __ldg(t.table + kRowSlot + row0 + j * 16);
      if (r.slot[j] >= 0 && __ldg(t.table + kSlotShared + r.slot[j]) < 0) r.slot[j] = -1;
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
    if (slot < 0 || __ldg(t.table + kSlotShared + slot) >= 0) return {-1};
    return {__ldg(t.table + kSlotAdapter + slot)};
  }
  static __device__ __forceinline__ void epilogue(const TileMaps& maps, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    const int32_t row = t.row_tile * kTileRows + w.quarter * 32;
    if (row >= p.num_tokens) return;
    const bool loners = __ballot_sync(0xffffffffu, early.loner >= 0) != 0u;
    const int32_t end = min(t.n0 + (p.cols > 128 ? (w.part + 1) * 128 : (w.part == 0 ? 128 : 0)), p.width);
#pragma unroll 1
    for (int32_t col = t.n0 + w.part * 128; col < end; col += 64) {
      uint32_t packed[32];
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        uint32_t v[32];
        ptx::tmem_ld_32x32b_x32(w.taddr + (col - t.n0) + part * 32, v);
        ptx::tmem_ld_wait();
        if (loners && early.loner >= 0) {
          const __nv_bfloat16* vr = p.v + static_cast<int64_t>(row + w.lane) * p.v_cols;
          for (int32_t q = 0; q < p.v_cols; ++q) {
            const float f = __bfloat162float(__ldg(vr + q));
            const __nv_bfloat16* br = p.b + (static_cast<int64_t>(early.loner) * p.rank + (q >= p.rank ? q - p.rank : q)) * p.width;
#pragma unroll
            for (int h = 0; h < 32; ++h) {
              const int32_t c = col + part * 32 + h;
              if (c < p.width) v[h] = __float_as_uint(fmaf(f, __bfloat162float(__ldg(br + c)), __uint_as_float(v[h])));
            }
          }
        }
        if (p.out_fp32) {
          if (col + part * 32 < p.width) store_rows_128b<kBuffers>(w, &maps.m[2], v, col + part * 32, row);
        } else {
#pragma unroll
          for (int h = 0; h < 16; ++h)
            packed[part * 16 + h] = pack_bf16(__uint_as_float(v[2 * h]), __uint_as_float(v[2 * h + 1]));
        }
      }
      if (!p.out_fp32) store_rows_128b<kBuffers>(w, &maps.m[2], packed, col, row);
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
  int64_t row_tiles, tables, not_finite, partial, v, total;  // bytes of each part, 256-byte aligned, then all
  int32_t splits, steps, total_steps, parts, scan_parts;
};

int64_t align256(int64_t n) { return (n + 255) & ~static_cast<int64_t>(255); }

LoraSizes lora_sizes(int64_t num_tokens, int32_t d_model, int32_t width, int32_t rank, int32_t num_adapters, int out_fp32, int sm_count) {
  LoraSizes s{};
  if (num_tokens <= kSkinnyMaxRows) {
    s.v = align256(num_tokens * rank * 4);
    s.total = s.v;
    return s;
  }
  s.row_tiles = (num_tokens + kTileRows - 1) / kTileRows;
  s.parts = out_fp32 ? 2 : 1;
  s.total_steps = (d_model + kTileStep - 1) / kTileStep;
  // Parts of D for few row tiles: enough to fill the GPU, each of at least 8 K steps.
  const int64_t want = std::max<int64_t>(1, sm_count / std::max<int64_t>(1, s.row_tiles));
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(want, s.total_steps / 8));
  s.steps = static_cast<int32_t>((s.total_steps + parts - 1) / parts);
  s.splits = (s.total_steps + s.steps - 1) / s.steps;
  s.tables = align256(s.row_tiles * kTableInts * 4);
  // Thread blocks that look through one adapter's B: about four per SM over all tiles, each for 8 KB at least.
  const int64_t b_bytes = static_cast<int64_t>(rank) * width * 2;
  s.scan_parts = static_cast<int32_t>(std::max<int64_t>(1, std::min<int64_t>({64, 4 * sm_count / s.row_tiles, b_bytes / 8192})));
  s.not_finite = align256(static_cast<int64_t>(num_adapters) * s.scan_parts);
  s.partial = align256(static_cast<int64_t>(s.splits) * num_tokens * rank * 4);
  s.v = align256(num_tokens * rank * s.parts * 2);
  s.total = s.tables + s.not_finite + s.partial + s.v;
  return s;
}

int check_lora(int64_t num_tokens, int32_t d_model, int32_t width, int32_t rank, int32_t num_adapters) {
  if (num_tokens < 0 || num_tokens > INT32_MAX - kTileRows) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: T must fit 31 bits");
  if (d_model <= 0 || d_model % 8 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: D (%d) must be a positive multiple of 8", d_model);
  if (width <= 0 || width % 8 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: N (%d) must be a positive multiple of 8", width);
  if (rank <= 0 || rank % 8 != 0 || rank > 128)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the rank (%d) must be a multiple of 8 in [8, 128]", rank);
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
  return lora_sizes(num_tokens, d_model, width, rank, num_adapters, out_fp32, info->sm_count).total;
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
  const LoraSizes s = lora_sizes(num_tokens, d_model, width, rank, num_adapters, out_fp32, info->sm_count);
  if (workspace_bytes < s.total)
    return fail(SB_ERR_INVALID_ARGUMENT, "lora_linear: the workspace has %lld bytes, %lld are needed",
                (long long)workspace_bytes, (long long)s.total);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (num_tokens <= kSkinnyMaxRows)
    return lora_small(x, weight, lora_a, lora_b, adapter_idx, idx_is_i64, scale, out, out_fp32, static_cast<int32_t>(num_tokens),
                      d_model, width, rank, num_adapters, reinterpret_cast<float*>(ws), info, dev_status, as_stream(stream));
  int32_t* tables = reinterpret_cast<int32_t*>(ws);
  uint8_t* not_finite = ws + s.tables;
  float* partial = reinterpret_cast<float*>(not_finite + s.not_finite);
  __nv_bfloat16* v = reinterpret_cast<__nv_bfloat16*>(not_finite + s.not_finite + s.partial);
  const cudaStream_t st = as_stream(stream);
  const int32_t tokens = static_cast<int32_t>(num_tokens);
  const int32_t row_tiles = static_cast<int32_t>(s.row_tiles);

  const dim3 plan_grid(static_cast<unsigned>(row_tiles), static_cast<unsigned>(s.scan_parts));
  const int32_t b_vecs = rank * (width / 8);
  if (idx_is_i64)
    lora_plan_kernel<int64_t><<<plan_grid, kPlanThreads, 0, st>>>(static_cast<const int64_t*>(adapter_idx),
        static_cast<const uint4*>(lora_b), tables, not_finite, tokens, num_adapters, b_vecs);
  else
    lora_plan_kernel<int32_t><<<plan_grid, kPlanThreads, 0, st>>>(static_cast<const int32_t*>(adapter_idx),
        static_cast<const uint4*>(lora_b), tables, not_finite, tokens, num_adapters, b_vecs);
  if (int rc = check_launch("lora_linear (plan)")) return rc;

  {
    TileMaps maps{};
    if (int rc = encode_2d_map(&maps.m[0], x, num_tokens, d_model, kTileRows, 64, 2, "lora_linear (x)")) return rc;
    if (int rc = encode_2d_map(&maps.m[1], lora_a, static_cast<uint64_t>(num_adapters) * rank, d_model, rank, 64, 2, "lora_linear (A)")) return rc;
    LoraShrink::Params p{};
    p.tables = tables;
    p.partial = partial;
    p.num_tokens = tokens;
    p.rank = rank;
    p.row_tiles = row_tiles;
    const int32_t most = static_cast<int32_t>(std::min<int64_t>({kMaxSlots, num_adapters, num_tokens}));
    p.group_slots = std::min(kTileCols / rank, most);
    p.groups = (most + p.group_slots - 1) / p.group_slots;
    p.splits = s.splits;
    p.steps = s.steps;
    p.total_steps = s.total_steps;
    if (int rc = launch_tile_gemm<LoraShrink>(maps, p, static_cast<int64_t>(row_tiles) * p.groups * p.splits, dev_status, st, "lora_linear (shrink)")) return rc;
  }
  {
    const int64_t values = std::max<int64_t>(num_tokens * rank, static_cast<int64_t>(row_tiles) * kMaxSlots);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>((values + 255) / 256, static_cast<int64_t>(info->sm_count) * 8)));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const float* parts = partial;
    const uint8_t* flags = not_finite;
    const cudaError_t err =
        idx_is_i64 ? cudaLaunchKernelEx(&cfg, lora_join_kernel<int64_t>, parts, static_cast<const int64_t*>(adapter_idx), scale, v, tokens,
                                        num_adapters, rank, s.splits, s.parts, tables, flags, row_tiles, s.scan_parts)
                   : cudaLaunchKernelEx(&cfg, lora_join_kernel<int32_t>, parts, static_cast<const int32_t*>(adapter_idx), scale, v, tokens,
                                        num_adapters, rank, s.splits, s.parts, tables, flags, row_tiles, s.scan_parts);
    if (err != cudaSuccess) return fail(SB_ERR_CUDA, "lora_linear (join): %s", cudaGetErrorString(err));
  }

  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], weight, d_model, width, 64, 64, 2, "lora_linear (weight)")) return rc;
  if (int rc = encode_2d_map(&maps.m[1], lora_b, static_cast<uint64_t>(num_adapters) * rank, width, 8, 64, 2, "lora_linear (B)")) return rc;
  if (int rc = encode_2d_map(&maps.m[2], out, num_tokens, width, 32, out_fp32 ? 32 : 64, out_fp32 ? 4 : 2, "lora_linear (out)")) return rc;
  if (int rc = encode_2d_map(&maps.m[3], x, num_tokens, d_model, kTileRows, 64, 2, "lora_linear (x)")) return rc;
  LoraExpand::Params p{};
  const int32_t slices = (width + kTileCols - 1) / kTileCols;
  p.order = {row_tiles, slices, 8};
  p.tables = tables;
  p.v = v;
  p.b = static_cast<const __nv_bfloat16*>(lora_b);
  p.num_tokens = tokens;
  p.width = width;
  p.rank = rank;
  p.v_cols = rank * s.parts;
  p.base_steps = s.total_steps;
  p.adapter_rows = num_adapters * rank;
  p.cols = width >= kTileCols ? kTileCols : (width + 15) & ~15;
  p.out_fp32 = out_fp32 ? 1 : 0;
  return launch_tile_gemm<LoraExpand>(maps, p, static_cast<int64_t>(row_tiles) * slices, dev_status, st, "lora_linear (expand)");
}
