// The gated expert block of the MoE layer and its backward pass, on the block-sparse layout of sb_route.
//
//   forward    G = X Wg[e], U = X Wu[e], H = act(G) * U            (GatedUp), Y = H Wd[e] (RowsProduct)
//   backward   with dO = grad_out of the row's token and w the gate of its copy:
//              dgate = dO . Y, dH = w (dO Wd[e]^T), dU = dH act(G), dG = dH U act'(G)     (grad rows kernel, GradHidden)
//              dWd = H^T (w dO), dWg = X^T dG, dWu = X^T dU                               (GradWeights)
//              dx[t] = sum over the token's copies of dG Wg^T + dU Wu^T                   (RowsProduct, join)
//
// The forward keeps X (rows in layout order), G, U, H and Y. What is an operand of a product is bf16, as the weights are:
// H, w dO, dG and dU are each rounded once, and so are G and U, which the backward pass reads back (in fp32 they would be
// most of its traffic). Y, the rows of dx, all sums, the activation and its derivative are in fp32. dgate takes Y, not
// H dH / w, which a gate of 0 would spoil.
//
// A decoding step (at most 128 copies, nothing kept) takes another way: no layout, the weights of the picked experts
// streamed by the kernels of skinny.cuh (SkinnyUp, SkinnyDown, gated_small_combine_kernel).
//
// act is SiLU, v / (1 + exp(-v)), or the erf form of GELU. exp and the reciprocal are the hardware's approximations (a few
// units of 2^-23) and erf is within 1.5e-7: errors of 1e-6 of |v| at most, far below half a step of the bf16 results (2^-8).

#include <algorithm>
#include <initializer_list>

#include "skinny.cuh"
#include "tile_gemm.cuh"

namespace sb {
namespace {

constexpr float kInvSqrt2Pi = 0.3989422804014327f;

__device__ __forceinline__ float fast_rcp(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// exp(-v) overflows to inf below v = -88: the reciprocal is then 0, the limit.
__device__ __forceinline__ float sigmoid(float v) { return fast_rcp(1.0f + __expf(-v)); }

template <int kActivation>
__device__ __forceinline__ float act_value(float v) {
  return kActivation == SB_ACT_SILU ? v * sigmoid(v) : gelu_erf(v);
}

// act(v) and its derivative.
template <int kActivation>
__device__ __forceinline__ void act_and_slope(float v, float* value, float* slope) {
  if (kActivation == SB_ACT_SILU) {
    const float s = sigmoid(v);
    *value = v * s;
    *slope = s * fmaf(v, 1.0f - s, 1.0f);
  } else {
    // Phi(v) = (1 + erf(v / sqrt 2)) / 2 by Abramowitz-Stegun 7.1.26 (absolute error below 1.5e-7), whose exponential
    // exp(-v^2 / 2) is also the one of the density in the derivative Phi(v) + v phi(v).
    const float a = fabsf(v) * 0.70710678118654752f;
    const float t = fast_rcp(fmaf(0.3275911f, a, 1.0f));
    float poly = fmaf(1.061405429f, t, -1.453152027f);
    poly = fmaf(poly, t, 1.421413741f);
    poly = fmaf(poly, t, -0.284496736f);
    poly = fmaf(poly, t, 0.254829592f);
    const float e = __expf(-a * a);
    const float phi_abs = 1.0f - 0.5f * poly * t * e;  // Phi(|v|)
    const float cdf = v >= 0.0f ? phi_abs : 1.0f - phi_abs;
    *value = v * cdf;
    *slope = fmaf(v * kInvSqrt2Pi, e, cdf);
  }
}

// The 64-row half of the row block that a warp's 32 rows lie in holds real rows (padding sits at the end of a row
// block). The weight gradients read the rows of an expert in steps of 64: halves without real rows are never read.
__device__ __forceinline__ bool half_has_rows(const int32_t* row_token, int32_t row_block, int quarter) {
  return __ldg(row_token + static_cast<int64_t>(row_block) * kTileRows + (quarter & 2) * 32) >= 0;
}

// A lane's row of the tile is no padding. Rows of padding are zeros in X and w dO, and an infinite weight makes NaN of them in
// H, dG and dU (0 * inf), which the weight gradients would sum up with the rest: they are stored as zeros, whatever came out.
__device__ __forceinline__ bool row_is_real(const int32_t* row_token, int32_t row_block, const EpilogueWarp& w) {
  return __ldg(row_token + static_cast<int64_t>(row_block) * kTileRows + w.quarter * 32 + w.lane) >= 0;
}

// Tile order of the products over (row block, column slice): expert by expert, in an expert bands of up to kBand row
// blocks, in a band the row block changes fastest. The thread blocks that run at the same time then work on few column
// slices of one expert's weights for all of its row blocks: a weight tile comes from memory once and from L2 for the
// other row blocks. (Bands of a fixed height over all row blocks straddled the experts: about twice the weight traffic
// with nine row blocks per expert.) Every row block of an expert has `slices` tiles, so the tiles of an expert are
// consecutive, and tile / slices is one of its row blocks: no search.
struct ExpertOrder {
  const int32_t* row_block_expert;
  const int32_t* padded_offsets;
  const int32_t* tokens_per_expert;
  int32_t num_experts, slices;
  static constexpr int32_t kBand = 16;
  __device__ __forceinline__ int32_t live_tiles() const { return __ldg(padded_offsets + num_experts) / kTileRows * slices; }
  // False: not a row block of any expert.
  // groups: how many of the row block's four groups of 32 rows hold real rows (padding sits at the end).
  __device__ __forceinline__ bool at(int32_t tile, int32_t* row_block, int32_t* slice, int32_t* expert, int32_t* groups) const {
    const int32_t e = __ldg(row_block_expert + tile / slices);
    if (e < 0) return false;
    const int32_t begin = __ldg(padded_offsets + e) / kTileRows;
    const int32_t end = __ldg(padded_offsets + e + 1) / kTileRows;
    const int32_t count = __ldg(tokens_per_expert + e);
    int32_t inside = tile - begin * slices;
    const int32_t band = inside / (kBand * slices);
    inside -= band * (kBand * slices);
    const int32_t first = begin + band * kBand;
    const int32_t height = min(kBand, end - first);
    *slice = inside / height;
    *row_block = first + inside - *slice * height;
    *expert = e;
    *groups = max(1, min(4, (count - (*row_block - begin) * kTileRows + 31) / 32));
    return true;
  }
};

// 64 inner columns of the first `groups` x 32 rows of a row block. The rest of the stage keeps what it held, and the
// accumulator rows that come of it are never stored. With a row or two per expert (a small batch) the full 128 rows would
// be a third of all bytes.
template <bool kOnce>  // read once: first out of L2
__device__ __forceinline__ void load_rows(uint32_t a, const CUtensorMap* all, const CUtensorMap* rows32, int32_t col, int32_t row,
                                          int32_t groups, uint32_t bar) {
  const CUtensorMap* map = groups == 4 ? all : rows32;
  const int32_t boxes = groups == 4 ? 1 : groups;
  for (int32_t g = 0; g < boxes; ++g) {
    if (kOnce) ptx::tma_load_2d_hint(a + g * 4096, map, col, row + g * 32, bar, ptx::policy_evict_first());
    else ptx::tma_load_2d(a + g * 4096, map, col, row + g * 32, bar);
  }
}

// ---- forward: both projections, the activation and the product ----------------------------------------------------
// The tile's 256 accumulator columns are 128 columns of G next to the same 128 of U, so a thread that drains column c
// finds its partner 128 columns on and H leaves the chip as the only result (plus G and U for training).
// Padding rows of x are loaded as the zeros they are: multiplying zeros takes less of the power limit, which sets the clock
// of a longer run, than what a stage happens to hold (395 against 406 us a pass of the layer below, one after another).
// Bound by the weights' way from memory where experts have few rows (T = 4096, D = 1024, F = 4096, E = 64: 1.07 GB of
// weights in 193 us, 5.6 TB/s of a measured 6.56 copy peak; 235 us with G and U kept) and by the tensor cores where they
// have many (T = 4096, D = 4096, F = 14336, E = 8: 1.45 ms, 1490 TFLOP/s executed, at the clock that the power limit leaves).
struct GatedUp {
  struct Params {
    ExpertOrder order;
    const int32_t* row_token;
    int32_t d_model;
    int32_t activation;
    int32_t skip_padding;  // 32-row groups of padding are not stored
    int32_t keep;          // G and U are stored too, and every row that the backward pass reads
  };
  struct Tile {
    int32_t k_steps, row_block, n0, expert, first_block;
    bool live;
  };
  struct Early {
    bool store;
    bool real;  // this lane's row is no padding
  };
  static constexpr int kStages = 4, kEpilogueWarps = 8, kStaging = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = false, kExtension = false, kAMnMajor = false, kBMnMajor = true;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) { return p.order.live_tiles(); }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t{};
    int32_t slice, groups;  // all rows are loaded, see above
    t.live = p.order.at(index, &t.row_block, &slice, &t.expert, &groups);
    if (!t.live) return t;
    t.n0 = slice * 128;
    t.first_block = t.row_block * p.order.slices;  // of the layout's blocks, F / 128 per row block
    t.k_steps = p.d_model / kTileStep;
    return t;
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    const uint64_t once = ptx::policy_evict_first();
    ptx::tma_load_2d(a, &maps.m[5], ks * kTileStep, t.row_block * kTileRows, bar);
    const int32_t row = t.expert * p.d_model + ks * kTileStep;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      ptx::tma_load_2d_hint(b + j * TileSmem::kSlabBytes, &maps.m[j >> 1], t.n0 + (j & 1) * 64, row, bar, once);
  }
  static __device__ __forceinline__ Early prefetch(const Params& p, const Tile& t, const EpilogueWarp& w) {
    const bool real = row_is_real(p.row_token, t.row_block, w);
    if (p.keep) return {half_has_rows(p.row_token, t.row_block, w.quarter), real};
    return {!p.skip_padding || __any_sync(0xffffffffu, real), real};
  }
  template <int kActivation>
  static __device__ __forceinline__ void product(uint32_t gate, uint32_t up, uint32_t (&packed)[32]) {
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      uint32_t g[32], u[32];
      ptx::tmem_ld_32x32b_x32(gate + part * 32, g);
      ptx::tmem_ld_32x32b_x32(up + part * 32, u);
      ptx::tmem_ld_wait();
#pragma unroll
      for (int h = 0; h < 16; ++h)
        packed[part * 16 + h] =
            pack_bf16(act_value<kActivation>(__uint_as_float(g[2 * h])) * __uint_as_float(u[2 * h]),
                      act_value<kActivation>(__uint_as_float(g[2 * h + 1])) * __uint_as_float(u[2 * h + 1]));
    }
  }
  static __device__ __forceinline__ void epilogue(const TileMaps& maps, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    if (!early.store) return;
    const int32_t col = w.part * 64;
    const int32_t row = (t.first_block + (t.n0 >> 7)) * kTileRows + w.quarter * 32;
    const uint32_t gate = w.taddr + w.part * 64;
    const uint32_t up = gate + 128;
    uint32_t packed[32];
    if (p.keep) {
      load_packed_x64(gate, packed);
      store_rows_128b(w, &maps.m[3], packed, col, row);
      load_packed_x64(up, packed);
      store_rows_128b(w, &maps.m[4], packed, col, row);
    }
    if (p.activation == SB_ACT_SILU) product<SB_ACT_SILU>(gate, up, packed);
    else product<SB_ACT_GELU>(gate, up, packed);
#pragma unroll
    for (int h = 0; h < 32; ++h) packed[h] = early.real ? packed[h] : 0u;
    store_rows_128b(w, &maps.m[2], packed, col, row);
  }
};

// ---- backward: gradients of G and U -----------------------------------------------------------------
// dH = w (dO Wd^T) over 256 hidden columns; Wd [F, D] is read as the K-major operand it is. In the epilogue a lane has a row
// to itself: it reads G and U and writes dG and dU a sector (16 columns) at a time, the next sector on its way while it
// works on one. What bounds it is the latency of those reads, so sixteen warps share the tile (8: 226 us, 16: 196 us at
// T = 4096, D = 1024, F = 4096, E = 64; at 96 registers a thread the 256 columns spill 44 bytes). Staging the results for TMA stores costs a stage of the ring and is slower (1000
// against 850 us on the Mixtral-like layer).
template <int kCols>
struct GradHidden {
  struct Params {
    ExpertOrder order;
    const int32_t* row_token;
    const float* row_gate;
    const __nv_bfloat16* g;
    const __nv_bfloat16* u;
    __nv_bfloat16* dg;
    __nv_bfloat16* du;
    int32_t d_model, ffn_dim;
    int32_t activation;
  };
  static constexpr int kPart = 16;                // columns at a time: 32 bytes of a row, one sector
  static constexpr int kWarpCols = kCols / 4;     // of the tile's, per epilogue warp
  struct Tile {
    int32_t k_steps, row_block, n0, expert, groups;
    bool live;
  };
  struct Early {
    bool store;
    bool real;  // no padding
    float gate;
    int64_t at;  // of this row's columns in G and U, and in the results
    uint32_t first[2][8];  // G and U of the first part
  };
  static constexpr int kStages = 4, kEpilogueWarps = 16, kStaging = 0;
  static constexpr bool kAhead = true;
  static constexpr bool kVariable = true, kExtension = false, kAMnMajor = false, kBMnMajor = false;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) { return p.order.live_tiles(); }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t{};
    int32_t slice;
    t.live = p.order.at(index, &t.row_block, &slice, &t.expert, &t.groups);
    if (!t.live) return t;
    t.n0 = slice * kCols;
    t.groups = (t.groups + 1) & ~1;  // whole halves: their padding rows are stored, as zeros
    t.k_steps = p.d_model / kTileStep;
    return t;
  }
  static __device__ __forceinline__ int columns(const Params&, const Tile&) { return kCols; }
  static __device__ __forceinline__ uint32_t tx_bytes(const Params&, const Tile& t, int32_t) {
    return static_cast<uint32_t>(t.groups) * 4096u + kCols * 128u;
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    load_rows<false>(a, &maps.m[1], &maps.m[2], ks * kTileStep, t.row_block * kTileRows, t.groups, bar);
    // With F an odd multiple of 128 the last tile's upper 128 columns are rows of the next expert (or zeros past the
    // end): computed, never stored.
    ptx::tma_load_2d_hint(b, &maps.m[0], ks * kTileStep, t.expert * p.ffn_dim + t.n0, bar, ptx::policy_evict_first());
  }
  static __device__ __forceinline__ Early prefetch(const Params& p, const Tile& t, const EpilogueWarp& w) {
    Early e;
    const int32_t n = t.n0 + w.part * kWarpCols;
    e.store = n < p.ffn_dim && half_has_rows(p.row_token, t.row_block, w.quarter);
    if (!e.store) return e;
    e.real = row_is_real(p.row_token, t.row_block, w);
    e.gate = __ldg(p.row_gate + static_cast<int64_t>(t.row_block) * kTileRows + w.quarter * 32 + w.lane);
    e.at = ((static_cast<int64_t>(t.row_block) * (p.ffn_dim >> 7) + (n >> 7)) * kTileRows + w.quarter * 32 + w.lane) * 128 + (n & 127);
    ptx::ld_global_v8(p.g + e.at, e.first[0]);
    ptx::ld_global_v8(p.u + e.at, e.first[1]);
    return e;
  }
  // 32 rows of a block are 8 KB in one piece: the next tile's are asked into L2 before this one is worked on,
  // because what a warp can hold in flight in registers does not cover the way to memory.
  static __device__ __forceinline__ void ahead(const Params& p, const Tile& next, const EpilogueWarp& w) {
    const int32_t n = next.n0 + w.part * kWarpCols;
    if ((w.part != 0 && (n & 127) != 0) || !next.live || n >= p.ffn_dim || w.lane != 0 || !half_has_rows(p.row_token, next.row_block, w.quarter)) return;
    const int64_t at = ((static_cast<int64_t>(next.row_block) * (p.ffn_dim >> 7) + (n >> 7)) * kTileRows + w.quarter * 32) * 128;
    ptx::bulk_prefetch_l2(p.g + at, 32 * 256);
    ptx::bulk_prefetch_l2(p.u + at, 32 * 256);
  }
  static __device__ __forceinline__ void epilogue(const TileMaps&, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    if (!early.store) return;
    if (p.activation == SB_ACT_SILU) work<SB_ACT_SILU>(p, w, early);
    else work<SB_ACT_GELU>(p, w, early);
  }
  template <int kActivation>
  static __device__ __forceinline__ void work(const Params& p, const EpilogueWarp& w, const Early& early) {
    uint32_t held[2][2][8];  // G and U of this part and the next
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      held[0][0][q] = early.first[0][q];
      held[0][1][q] = early.first[1][q];
    }
#pragma unroll
    for (int part = 0; part < kWarpCols / kPart; ++part) {
      uint32_t s[16];
      ptx::tmem_ld_32x32b_x16(w.taddr + w.part * kWarpCols + part * kPart, s);
      if (part + 1 < kWarpCols / kPart) {
        ptx::ld_global_v8(p.g + early.at + (part + 1) * kPart, held[(part + 1) & 1][0]);
        ptx::ld_global_v8(p.u + early.at + (part + 1) * kPart, held[(part + 1) & 1][1]);
      }
      ptx::tmem_ld_wait();
      uint32_t dg[8], du[8];
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        const float2 gf = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&held[part & 1][0][h]));
        const float2 uf = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&held[part & 1][1][h]));
        float a0, a1, d0, d1;
        act_and_slope<kActivation>(gf.x, &a0, &d0);
        act_and_slope<kActivation>(gf.y, &a1, &d1);
        const float s0 = __uint_as_float(s[2 * h]) * early.gate;
        const float s1 = __uint_as_float(s[2 * h + 1]) * early.gate;
        dg[h] = early.real ? pack_bf16(s0 * uf.x * d0, s1 * uf.y * d1) : 0u;
        du[h] = early.real ? pack_bf16(s0 * a0, s1 * a1) : 0u;
      }
      ptx::st_global_v8(p.dg + early.at + part * kPart, dg);
      ptx::st_global_v8(p.du + early.at + part * kPart, du);
    }
  }
};

// ---- the products that give rows: the down projection, and the backward pass's rows of dx ---------------------------
// Down (kBack false): Y = H Wd, Wd [F, D] an MN-major operand. Back: dG Wg^T + dU Wu^T as one product with 2 F inner
// columns, Wg and Wu [D, F] K-major operands. Either way the weights lie as the tensor cores read them. The rows stay in
// fp32: each token's rows are summed, and rounded once, behind this.
// At T = 4096, D = 1024, F = 4096, E = 64: 108 us (0.54 GB of weights, 5.0 TB/s) and 219 us (4.9 TB/s); what is left is the
// last wave, 368 tiles of 256 columns on 148 SMs. Tiles of 128 columns fill it but keep fewer bytes in flight: 141 and
// 285 us. On the Mixtral-like layer (T = 4096, D = 4096, F = 14336, E = 8) 745 us and 1.50 ms, 1450 TFLOP/s executed.
template <bool kBack>
struct RowsProduct {
  struct Params {
    ExpertOrder order;
    const int32_t* row_token;
    int32_t d_model, ffn_dim, cols;
  };
  struct Tile {
    int32_t k_steps, row_block, n0, cols, expert, first_block, groups;
    bool live;
  };
  struct Early { bool store; };
  static constexpr int kStages = 4, kEpilogueWarps = 8, kStaging = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = true, kExtension = false, kAMnMajor = false, kBMnMajor = !kBack;

  // Down: the tiles of the last wave, where they would leave half of the thread blocks or more without one, are cut into
  // two or four by columns (not below 64); `whole` tiles come before them. (176 tiles of a batch of 37 tokens: 76 -> 72 us.
  // Back reads its weights in boxes as tall as the tile is wide, one TMA load per step; cutting those cost 3 %.)
  static __device__ __forceinline__ void waves(const Params& p, int32_t* whole, int32_t* rest, int32_t* cut) {
    const int32_t total = p.order.live_tiles();
    const int32_t blocks = static_cast<int32_t>(gridDim.x);
    *rest = total % blocks;
    *whole = total - *rest;
    *cut = 1;
    while (!kBack && *rest > 0 && *rest * *cut * 2 <= blocks && p.cols / (*cut * 2) >= 64) *cut *= 2;
  }
  static __device__ __forceinline__ int32_t total_tiles(const Params& p) {
    int32_t whole, rest, cut;
    waves(p, &whole, &rest, &cut);
    return whole + rest * cut;
  }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t{};
    int32_t whole, rest, cut, slice, piece = 0;
    waves(p, &whole, &rest, &cut);
    t.cols = p.cols;
    if (index >= whole) {
      piece = (index - whole) % cut;
      index = whole + (index - whole) / cut;
      t.cols /= cut;
    }
    t.live = p.order.at(index, &t.row_block, &slice, &t.expert, &t.groups);
    if (!t.live) return t;
    t.n0 = slice * p.cols + piece * t.cols;
    t.first_block = t.row_block * (p.ffn_dim >> 7);
    // A piece that lies behind D (an odd multiple of 128) has nothing to do.
    t.live = t.n0 < p.d_model;
    t.k_steps = t.live ? (kBack ? 2 : 1) * (p.ffn_dim / kTileStep) : 0;
    return t;
  }
  static __device__ __forceinline__ int columns(const Params&, const Tile& t) { return t.cols; }
  static __device__ __forceinline__ uint32_t tx_bytes(const Params&, const Tile& t, int32_t) {
    return static_cast<uint32_t>(t.groups) * 4096u + static_cast<uint32_t>(t.cols) * 128u;
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    const uint64_t once = ptx::policy_evict_first();
    const int32_t steps = p.ffn_dim / kTileStep;
    const int which = kBack && ks >= steps ? 1 : 0;
    const int32_t k = (ks - which * steps) * kTileStep;
    load_rows<true>(a, &maps.m[which], &maps.m[5 + which], k & 127, (t.first_block + (k >> 7)) * kTileRows, t.groups, bar);
    if (kBack) {
      ptx::tma_load_2d_hint(b, &maps.m[2 + which], k, t.expert * p.d_model + t.n0, bar, once);
    } else {
      for (int32_t j = 0; j < t.cols / 64; ++j)
        ptx::tma_load_2d_hint(b + j * TileSmem::kSlabBytes, &maps.m[2], t.n0 + j * 64, t.expert * p.ffn_dim + k, bar, once);
    }
  }
  static __device__ __forceinline__ Early prefetch(const Params& p, const Tile& t, const EpilogueWarp& w) {
    return {__ldg(p.row_token + static_cast<int64_t>(t.row_block) * kTileRows + w.quarter * 32) >= 0};
  }
  static __device__ __forceinline__ void epilogue(const TileMaps& maps, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early& early) {
    if (!early.store) return;
#pragma unroll 1
    for (int32_t c = w.part * 32; c < t.cols; c += 64) {
      if (t.n0 + c >= p.d_model) break;
      uint32_t v[32];
      ptx::tmem_ld_32x32b_x32(w.taddr + c, v);
      ptx::tmem_ld_wait();
      store_rows_128b(w, &maps.m[4], v, t.n0 + c, t.row_block * kTileRows + w.quarter * 32);
    }
  }
};

// ---- backward: the three weight gradients -------------------------------------------------------------------------
// The rows of an expert are the inner dimension, so both operands are MN-major: X, w dO, H, dG and dU as they lie.
// An expert's rows end inside a step of 64; the rest of that step is zero rows in X and w dO against finite ones (zeros) in
// H, dG and dU. An expert without rows gets zeros. Bound by writing: with two or three K steps per tile the kernel moves
// 5.1 TB/s (T = 4096, D = 1024, F = 4096, E = 64: 365 us). Tried and slower: two staging tiles per warp or sixteen warps for
// a stage of the ring (385 us), stores from registers (444 us); no gain: fetching only the real rows of the last step.
struct GradWeights {
  struct Params {
    const int32_t* padded_offsets;
    const int32_t* tokens_per_expert;
    int32_t num_experts, d_model, ffn_dim;
    int32_t down_cols, down_tiles;  // column tiles of dWd [F, D], its tiles per expert
    int32_t up_cols, up_tiles;      // the same of dWg and dWu [D, F]
  };
  struct Tile {
    int32_t k_steps, which, expert, m0, n0, row0, block0;  // which: 0 dWd, 1 dWg, 2 dWu
    bool live;
  };
  struct Early {};
  static constexpr int kStages = 4, kEpilogueWarps = 8, kStaging = 1;
  static constexpr bool kAhead = false;
  static constexpr bool kVariable = false, kExtension = false, kAMnMajor = true, kBMnMajor = true;

  static __device__ __forceinline__ int32_t total_tiles(const Params& p) {
    return p.num_experts * (p.down_tiles + 2 * p.up_tiles);
  }
  static __device__ __forceinline__ Tile tile(const Params& p, int32_t index) {
    Tile t;
    const int32_t per_expert = p.down_tiles + 2 * p.up_tiles;
    t.expert = index / per_expert;
    int32_t i = index - t.expert * per_expert;
    t.which = 0;
    int32_t cols = p.down_cols;
    if (i >= p.down_tiles) {
      i -= p.down_tiles;
      t.which = i >= p.up_tiles ? 2 : 1;
      i -= (t.which - 1) * p.up_tiles;
      cols = p.up_cols;
    }
    const int32_t m = i / cols;
    t.m0 = m * kTileRows;
    t.n0 = (i - m * cols) * kTileCols;
    t.live = true;
    t.k_steps = (__ldg(p.tokens_per_expert + t.expert) + kTileStep - 1) / kTileStep;
    t.row0 = __ldg(p.padded_offsets + t.expert);
    t.block0 = t.row0 / kTileRows * (p.ffn_dim >> 7);  // the layout's row_offsets, which are regular where rows are
    return t;
  }
  static __device__ __forceinline__ void load(const TileMaps& maps, const Params& p, const Tile& t, int32_t ks, uint32_t a,
                                              uint32_t b, uint32_t bar) {
    const int32_t row = t.row0 + ks * kTileStep;                        // of X and w dO
    const int32_t block = t.block0 + (ks >> 1) * (p.ffn_dim >> 7);      // first of the row block's blocks
    const int32_t inside = (ks & 1) * kTileStep;
    const int32_t slab = TileSmem::kSlabBytes;
    if (t.which == 0) {
      const int32_t h_row = (block + (t.m0 >> 7)) * kTileRows + inside;
#pragma unroll
      for (int j = 0; j < 2; ++j) ptx::tma_load_2d(a + j * slab, &maps.m[2], j * 64, h_row, bar);
#pragma unroll
      for (int j = 0; j < 4; ++j) ptx::tma_load_2d(b + j * slab, &maps.m[1], t.n0 + j * 64, row, bar);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) ptx::tma_load_2d(a + j * slab, &maps.m[0], t.m0 + j * 64, row, bar);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        // With F an odd multiple of 128 the last tile's upper blocks are the next row block's: never stored.
        const int32_t n = t.n0 + j * 64;
        ptx::tma_load_2d(b + j * slab, &maps.m[2 + t.which], n & 127, (block + (n >> 7)) * kTileRows + inside, bar);
      }
    }
  }
  static __device__ __forceinline__ Early prefetch(const Params&, const Tile&, const EpilogueWarp&) { return {}; }
  static __device__ __forceinline__ void epilogue(const TileMaps& maps, const Params& p, const Tile& t, EpilogueWarp& w,
                                                  const Early&) {
    const int32_t width = t.which == 0 ? p.d_model : p.ffn_dim;
    const int32_t row = t.expert * (t.which == 0 ? p.ffn_dim : p.d_model) + t.m0 + w.quarter * 32;
#pragma unroll 1
    for (int g = 0; g < 2; ++g) {
      const int32_t col = t.n0 + w.part * 128 + g * 64;
      if (col >= width) break;
      uint32_t packed[32];
      if (t.k_steps > 0) {
        load_packed_x64(w.taddr + w.part * 128 + g * 64, packed);
      } else {
#pragma unroll
        for (int h = 0; h < 32; ++h) packed[h] = 0u;
      }
      store_rows_128b(w, &maps.m[5 + t.which], packed, col, row);
    }
  }
};

// ---- a decoding step -----------------------------------------------------------------------------------------------
// The blocks are numbered (picked expert in order of first appearance, column tile, split); every block finds its
// expert and that expert's copies from the ids by itself, so there is no routing kernel in front.

struct ExpertItem { int32_t expert, tile, rows; };

// False: fewer distinct experts than block items. list: the expert's copies, ascending.
__device__ __forceinline__ bool find_expert(const void* expert_idx, int idx_is_i64, int32_t copies, int32_t num_experts,
                                            int32_t which, ExpertItem& item, int32_t* ids, int32_t* list) {
  constexpr int kWarps = kSkinnyMaxRows / 32;
  __shared__ int32_t lead_count[kWarps], match_count[kWarps];
  __shared__ int32_t found;
  const int c = static_cast<int>(threadIdx.x);
  int32_t mine = -1;
  if (c < copies) {
    const int64_t id = idx_is_i64 ? __ldg(static_cast<const long long*>(expert_idx) + c)
                                  : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(expert_idx) + c));
    if (id >= 0 && id < num_experts) mine = static_cast<int32_t>(id);
  }
  if (c < kSkinnyMaxRows) ids[c] = mine;
  __syncthreads();
  bool leads = mine >= 0;
  int j = 0;
  for (; leads && j + 4 <= c; j += 4) {
    const int4 four = *reinterpret_cast<const int4*>(ids + j);
    leads = four.x != mine && four.y != mine && four.z != mine && four.w != mine;
  }
  for (; leads && j < c; ++j) leads = ids[j] != mine;
  const int warp = c >> 5;
  const unsigned below = (1u << (c & 31)) - 1u;
  const unsigned lead_mask = __ballot_sync(0xffffffffu, leads);
  if (warp < kWarps && (c & 31) == 0) lead_count[warp] = __popc(lead_mask);
  __syncthreads();
  int32_t distinct = 0, before = __popc(lead_mask & below);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) before += lead_count[w];
    distinct += lead_count[w];
  }
  if (leads && before == which) found = mine;
  if (which >= distinct) return false;
  __syncthreads();
  item.expert = found;
  const bool match = c < kSkinnyMaxRows && mine == item.expert;
  const unsigned match_mask = __ballot_sync(0xffffffffu, match);
  if (warp < kWarps && (c & 31) == 0) match_count[warp] = __popc(match_mask);
  __syncthreads();
  int32_t place = __popc(match_mask & below);
  item.rows = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) place += match_count[w];
    item.rows += match_count[w];
  }
  if (match) list[place] = c;
  return true;  // the caller's next barrier publishes the list
}

// H[copy] = act(x Wg) * (x Wu): the tile's 128 weight columns are 64 of Wg next to the same 64 of Wu.
struct SkinnyUp {
  struct Params {
    SkinnyShape shape;
    const void* expert_idx;
    const __nv_bfloat16* x;
    __nv_bfloat16* h;  // [copies, F]
    int32_t idx_is_i64, copies, k, num_experts, d_model, ffn_dim, tiles, activation;
  };
  using Item = ExpertItem;
  struct Extra {};
  static constexpr bool kGather = true;
  static __device__ __forceinline__ bool begin(const Params& p, Item& item, int32_t block_item, int32_t* ids, int32_t* list) {
    const int32_t which = block_item / p.tiles;
    item.tile = block_item - which * p.tiles;
    return find_expert(p.expert_idx, p.idx_is_i64, p.copies, p.num_experts, which, item, ids, list);
  }
  static __device__ __forceinline__ void load_w(const SkinnyMaps& maps, const Params& p, const Item& item, int32_t ks,
                                                uint32_t dst, uint32_t bar) {
    const int32_t row = item.expert * p.d_model + ks * kSkinnyStep;
    ptx::tma_load_2d(dst, &maps.w[0], item.tile * 64, row, bar);
    ptx::tma_load_2d(dst + kSkinnyWBytes / 2, &maps.w[1], item.tile * 64, row, bar);
  }
  static __device__ __forceinline__ const __nv_bfloat16* gather_row(const Params& p, const Item&, const int32_t* list, int row) {
    return p.x + static_cast<int64_t>(list[row] / p.k) * p.d_model;
  }
  static __device__ __forceinline__ void extra(const Params&, const Item&, int32_t, int, Extra&) {}
  static __device__ __forceinline__ void finish(const Params& p, const Item& item, const int32_t* list, int32_t rank,
                                                int worker, const SkinnySums& red, const Extra&) {
    const int32_t c = (worker & 7) * 8;
    for (int32_t r = rank + p.shape.splits * (worker >> 3); r < item.rows; r += p.shape.splits * 16) {
      float g[8], u[8];
      red.sum(r, c, g);
      red.sum(r, 64 + c, u);
      uint32_t packed[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        packed[q] = p.activation == SB_ACT_SILU
                        ? pack_bf16(act_value<SB_ACT_SILU>(g[2 * q]) * u[2 * q], act_value<SB_ACT_SILU>(g[2 * q + 1]) * u[2 * q + 1])
                        : pack_bf16(act_value<SB_ACT_GELU>(g[2 * q]) * u[2 * q], act_value<SB_ACT_GELU>(g[2 * q + 1]) * u[2 * q + 1]);
      *reinterpret_cast<uint4*>(p.h + static_cast<int64_t>(list[r]) * p.ffn_dim + item.tile * 64 + c) =
          make_uint4(packed[0], packed[1], packed[2], packed[3]);
    }
  }
};

// Y[copy] = H[copy] Wd in fp32.
struct SkinnyDown {
  struct Params {
    SkinnyShape shape;
    const void* expert_idx;
    const __nv_bfloat16* h;
    float* y;  // [copies, D]
    int32_t idx_is_i64, copies, num_experts, d_model, ffn_dim, tiles;
  };
  using Item = ExpertItem;
  struct Extra {};
  static constexpr bool kGather = true;
  static __device__ __forceinline__ bool begin(const Params& p, Item& item, int32_t block_item, int32_t* ids, int32_t* list) {
    const int32_t which = block_item / p.tiles;
    item.tile = block_item - which * p.tiles;
    return find_expert(p.expert_idx, p.idx_is_i64, p.copies, p.num_experts, which, item, ids, list);
  }
  static __device__ __forceinline__ void load_w(const SkinnyMaps& maps, const Params& p, const Item& item, int32_t ks,
                                                uint32_t dst, uint32_t bar) {
    const int32_t row = item.expert * p.ffn_dim + ks * kSkinnyStep;
    ptx::tma_load_2d(dst, &maps.w[0], item.tile * 128, row, bar);
    ptx::tma_load_2d(dst + kSkinnyWBytes / 2, &maps.w[0], item.tile * 128 + 64, row, bar);
  }
  static __device__ __forceinline__ const __nv_bfloat16* gather_row(const Params& p, const Item&, const int32_t* list, int row) {
    return p.h + static_cast<int64_t>(list[row]) * p.ffn_dim;
  }
  static __device__ __forceinline__ void extra(const Params&, const Item&, int32_t, int, Extra&) {}
  static __device__ __forceinline__ void finish(const Params& p, const Item& item, const int32_t* list, int32_t rank,
                                                int worker, const SkinnySums& red, const Extra&) {
    const int32_t c = (worker & 15) * 8;
    for (int32_t r = rank + p.shape.splits * (worker >> 4); r < item.rows; r += p.shape.splits * 8) {
      float v[8];
      red.sum(r, c, v);
      float4* dst = reinterpret_cast<float4*>(p.y + static_cast<int64_t>(list[r]) * p.d_model + item.tile * 128 + c);
      dst[0] = make_float4(v[0], v[1], v[2], v[3]);
      dst[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  }
};

// ---- small kernels ------------------------------------------------------------------------------------------------

constexpr int kSmallThreads = 256;

__device__ __forceinline__ float gate_at(const void* gate, int gate_dtype, int64_t i) {
  return gate_dtype == 1 ? __ldg(static_cast<const float*>(gate) + i)
                         : __bfloat162float(__ldg(static_cast<const __nv_bfloat16*>(gate) + i));
}

// out[t] = sum over the picks j of gate[t, j] * Y[t k + j], in order, from the fp32 rows of a decoding step.
__global__ void __launch_bounds__(128)
gated_small_combine_kernel(const float4* __restrict__ y, const void* __restrict__ expert_idx, int idx_is_i64,
                           const void* __restrict__ gate, int gate_dtype, uint2* __restrict__ out, int32_t k,
                           int32_t num_experts, int32_t quads) {
  ptx::grid_dependency_wait();
  const int32_t t = static_cast<int32_t>(blockIdx.y);
  const int32_t v = static_cast<int32_t>(blockIdx.x) * 128 + static_cast<int32_t>(threadIdx.x);
  if (v >= quads) return;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  for (int32_t j = 0; j < k; ++j) {
    const int32_t c = t * k + j;
    const int64_t id = idx_is_i64 ? __ldg(static_cast<const long long*>(expert_idx) + c)
                                  : static_cast<int64_t>(__ldg(static_cast<const int32_t*>(expert_idx) + c));
    if (id < 0 || id >= num_experts) continue;
    const float w = gate_at(gate, gate_dtype, c);
    const float4 r = __ldcg(y + static_cast<int64_t>(c) * quads + v);
    acc.x = fmaf(w, r.x, acc.x);
    acc.y = fmaf(w, r.y, acc.y);
    acc.z = fmaf(w, r.z, acc.z);
    acc.w = fmaf(w, r.w, acc.w);
  }
  out[static_cast<int64_t>(t) * quads + v] = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
}

// The same from the fp32 rows of the layout: out[t] = sum over the picks j, in order, of gate[t, j] * Y[copy_row[t, j]].
__global__ void __launch_bounds__(kSmallThreads)
gated_combine_kernel(const float4* __restrict__ y, const int32_t* __restrict__ copy_row, const void* __restrict__ gate,
                     int gate_dtype, uint2* __restrict__ out, int64_t num_tokens, int32_t k, int32_t quads) {
  ptx::grid_dependency_wait();
  const int64_t total = num_tokens * quads;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kSmallThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kSmallThreads + threadIdx.x; i < total; i += stride) {
    const int64_t t = i / quads;
    const int32_t v = static_cast<int32_t>(i - t * quads);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int32_t j = 0; j < k; ++j) {
      const int32_t row = __ldg(copy_row + t * k + j);
      if (row < 0) continue;
      const float w = gate_at(gate, gate_dtype, t * k + j);
      const float4 r = __ldcg(y + static_cast<int64_t>(row) * quads + v);
      acc.x = fmaf(w, r.x, acc.x);
      acc.y = fmaf(w, r.y, acc.y);
      acc.z = fmaf(w, r.z, acc.z);
      acc.w = fmaf(w, r.w, acc.w);
    }
    out[i] = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
  }
}

// One warp per row of the layout: x_rows[r] = x[token], zeros for padding and for tokens that x does not have (with the
// layout of a larger batch nothing is read past x). The products' TMA loads want the rows side by side; gathering them inside
// the products with cp.async took a quarter of their time instead.
__global__ void __launch_bounds__(kSmallThreads)
gated_rows_kernel(const uint4* __restrict__ x, const int32_t* __restrict__ row_token, const int32_t* __restrict__ num_rows,
                  uint4* __restrict__ x_rows, int32_t num_tokens, int32_t vecs) {
  ptx::grid_launch_dependents();
  ptx::grid_dependency_wait();
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int32_t rows = __ldg(num_rows);
  const int32_t warps = static_cast<int32_t>(gridDim.x * (kSmallThreads / 32));
  for (int32_t r = static_cast<int32_t>(blockIdx.x * (kSmallThreads / 32) + (threadIdx.x >> 5)); r < rows; r += warps) {
    const int32_t token = __ldg(row_token + r);
    const bool real = token >= 0 && token < num_tokens;
    uint4* dst = x_rows + static_cast<int64_t>(r) * vecs;
    const uint4* src = x + static_cast<int64_t>(real ? token : 0) * vecs;
#pragma unroll 4
    for (int32_t v = lane; v < vecs; v += 32) dst[v] = real ? __ldg(src + v) : make_uint4(0u, 0u, 0u, 0u);
  }
}

// One warp per row of the layout, for the copy that it is: grad_rows[r] = grad_out[token], scaled_rows[r] = w times that,
// rounded to bf16 (what dWd is summed from; dH takes the unscaled rows and w in fp32, one rounding less), row_gate[r] = w,
// zeros for padding; and dgate = grad_out[token] . Y[r] in fp32.
__global__ void __launch_bounds__(kSmallThreads)
gated_grad_rows_kernel(const uint4* __restrict__ grad_out, const float4* __restrict__ y_rows, const void* __restrict__ gate,
                       int gate_dtype, const int32_t* __restrict__ row_token, const int32_t* __restrict__ copy_row,
                       const int32_t* __restrict__ num_rows, uint4* __restrict__ grad_rows, uint4* __restrict__ scaled_rows,
                       float* __restrict__ row_gate, void* __restrict__ dgate, int32_t k, int32_t vecs) {
  ptx::grid_launch_dependents();
  const int lane = static_cast<int>(threadIdx.x & 31);
  const int32_t rows = __ldg(num_rows);
  const int32_t warps = static_cast<int32_t>(gridDim.x * (kSmallThreads / 32));
  for (int32_t r = static_cast<int32_t>(blockIdx.x * (kSmallThreads / 32) + (threadIdx.x >> 5)); r < rows; r += warps) {
    const int32_t token = __ldg(row_token + r);
    uint4* plain = grad_rows + static_cast<int64_t>(r) * vecs;
    uint4* scaled = scaled_rows + static_cast<int64_t>(r) * vecs;
    if (token < 0) {
      for (int32_t v = lane; v < vecs; v += 32) plain[v] = scaled[v] = make_uint4(0u, 0u, 0u, 0u);
      if (lane == 0) row_gate[r] = 0.0f;
      continue;
    }
    // The copy of the token that this row is: the one whose row it is (rows are unique).
    int64_t copy = 0;
    for (int32_t j0 = 0; j0 < k; j0 += 32) {
      const int32_t j = j0 + lane;
      const bool mine = j < k && __ldg(copy_row + static_cast<int64_t>(token) * k + j) == r;
      const unsigned who = __ballot_sync(0xffffffffu, mine);
      if (who != 0u) {
        copy = static_cast<int64_t>(token) * k + j0 + __ffs(who) - 1;
        break;
      }
    }
    const float w = gate_at(gate, gate_dtype, copy);
    const uint4* gs = grad_out + static_cast<int64_t>(token) * vecs;
    const float4* ys = y_rows + static_cast<int64_t>(r) * vecs * 2;
    float dot = 0.0f;
#pragma unroll 4
    for (int32_t v = lane; v < vecs; v += 32) {
      const uint4 raw = __ldg(gs + v);
      const float4 y0 = __ldg(ys + 2 * v), y1 = __ldg(ys + 2 * v + 1);
      const uint32_t gq[4] = {raw.x, raw.y, raw.z, raw.w};
      const float yq[8] = {y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w};
      uint32_t q[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&gq[c]));
        dot = fmaf(f.x, yq[2 * c], dot);
        dot = fmaf(f.y, yq[2 * c + 1], dot);
        q[c] = pack_bf16(f.x * w, f.y * w);
      }
      plain[v] = raw;
      scaled[v] = make_uint4(q[0], q[1], q[2], q[3]);
    }
    if (lane == 0) row_gate[r] = w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
    if (lane == 0) {
      if (gate_dtype == 1) static_cast<float*>(dgate)[copy] = dot;
      else static_cast<__nv_bfloat16*>(dgate)[copy] = __float2bfloat16_rn(dot);
    }
  }
}

// dx[t] = sum over the token's copies of their rows, in copy order in fp32; and zeros into the dgate of copies that have
// no row. A thread per four columns: with a warp per token, few tokens left most SMs idle (T = 179, D = 2688: 28 us).
__global__ void __launch_bounds__(kSmallThreads)
gated_join_kernel(const float4* __restrict__ dx_rows, const int32_t* __restrict__ copy_row, uint2* __restrict__ dx,
                  void* __restrict__ dgate, int gate_dtype, int64_t num_tokens, int32_t k, int32_t quads) {
  ptx::grid_dependency_wait();
  const int64_t total = num_tokens * quads;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kSmallThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kSmallThreads + threadIdx.x; i < total; i += stride) {
    const int64_t t = i / quads;
    const int32_t v = static_cast<int32_t>(i - t * quads);
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int32_t j = 0; j < k; ++j) {
      const int32_t row = __ldg(copy_row + t * k + j);
      if (row < 0) {
        if (v != 0) continue;
        if (gate_dtype == 1) static_cast<float*>(dgate)[t * k + j] = 0.0f;
        else static_cast<__nv_bfloat16*>(dgate)[t * k + j] = __float2bfloat16_rn(0.0f);
        continue;
      }
      const float4 r = __ldcg(dx_rows + static_cast<int64_t>(row) * quads + v);
      acc.x += r.x;
      acc.y += r.y;
      acc.z += r.z;
      acc.w += r.w;
    }
    dx[i] = make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
  }
}

// ---- host side ----------------------------------------------------------------------------------------------------

// Size rules all the products of the gated layer share.
int check_gated(const char* what, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int32_t num_row_blocks,
                int32_t activation) {
  if (d_model <= 0 || d_model % 128 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "%s: D (%d) must be a positive multiple of 128", what, d_model);
  if (ffn_dim <= 0 || ffn_dim % 128 != 0) return fail(SB_ERR_INVALID_ARGUMENT, "%s: F (%d) must be a positive multiple of 128", what, ffn_dim);
  if (num_experts <= 0 || num_row_blocks < 0) return fail(SB_ERR_INVALID_ARGUMENT, "%s: bad sizes", what);
  if (activation != SB_ACT_SILU && activation != SB_ACT_GELU)
    return fail(SB_ERR_INVALID_ARGUMENT, "%s: activation must be 0 (SiLU) or 1 (GELU), got %d", what, activation);
  const int64_t most = static_cast<int64_t>(num_row_blocks) * ffn_dim;  // rows of the block arrays seen as [nnz * 128, 128]
  if (most > INT32_MAX - 4 * kTileRows || static_cast<int64_t>(num_experts) * d_model > INT32_MAX - kTileCols ||
      static_cast<int64_t>(num_experts) * ffn_dim > INT32_MAX - kTileCols ||
      static_cast<int64_t>(num_row_blocks) * kTileRows > INT32_MAX)
    return fail(SB_ERR_INVALID_ARGUMENT, "%s: problem too large", what);
  return SB_OK;
}

bool any_misaligned(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!aligned16(p)) return true;
  return false;
}
bool any_null(std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (p == nullptr) return true;
  return false;
}

// Launches one of the small kernels with programmatic dependence.
template <class... Params, class... Args>
int launch_small(void (*kernel)(Params...), int64_t blocks, int threads, cudaStream_t stream, const char* what, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, static_cast<Params>(args)...);
  if (err != cudaSuccess) return fail(SB_ERR_CUDA, "%s: %s", what, cudaGetErrorString(err));
  return SB_OK;
}

// x_rows, then H (and G, U) on the layout.
int sdd_gated(const void* x, const void* w_gate, const void* w_up, const int32_t* row_token, const int32_t* row_block_expert,
              const int32_t* padded_offsets, const int32_t* tokens_per_expert, void* x_rows, void* h_blocks, void* g_blocks,
              void* u_blocks, int64_t num_tokens, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int32_t num_row_blocks,
              int32_t activation, int skip_padding_rows, int32_t* dev_status, cudaStream_t stream) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const uint64_t w_rows = static_cast<uint64_t>(num_experts) * d_model;
  const uint64_t b_rows = static_cast<uint64_t>(num_row_blocks) * ffn_dim;  // nnz * 128
  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], w_gate, w_rows, ffn_dim, 64, 64, 2, "sdd_gated (w_gate)")) return rc;
  if (int rc = encode_2d_map(&maps.m[1], w_up, w_rows, ffn_dim, 64, 64, 2, "sdd_gated (w_up)")) return rc;
  if (int rc = encode_2d_map(&maps.m[2], h_blocks, b_rows, 128, 32, 64, 2, "sdd_gated (blocks)")) return rc;
  if (g_blocks != nullptr) {
    if (int rc = encode_2d_map(&maps.m[3], g_blocks, b_rows, 128, 32, 64, 2, "sdd_gated (kept gate)")) return rc;
    if (int rc = encode_2d_map(&maps.m[4], u_blocks, b_rows, 128, 32, 64, 2, "sdd_gated (kept up)")) return rc;
  }
  if (int rc = encode_2d_map(&maps.m[5], x_rows, static_cast<uint64_t>(num_row_blocks) * kTileRows, d_model, 128, 64, 2, "sdd_gated (rows)")) return rc;
  const int64_t blocks = std::min<int64_t>(static_cast<int64_t>(num_row_blocks) * (kTileRows / 8), info->sm_count * 8);
  if (int rc = launch_small(gated_rows_kernel, blocks, kSmallThreads, stream, "sdd_gated (rows)", static_cast<const uint4*>(x),
                            row_token, padded_offsets + num_experts, static_cast<uint4*>(x_rows),
                            static_cast<int32_t>(std::min<int64_t>(num_tokens, INT32_MAX)), d_model / 8))
    return rc;
  GatedUp::Params p{};
  p.order = {row_block_expert, padded_offsets, tokens_per_expert, num_experts, ffn_dim / 128};
  p.row_token = row_token;
  p.d_model = d_model;
  p.activation = activation;
  p.skip_padding = skip_padding_rows ? 1 : 0;
  p.keep = g_blocks != nullptr ? 1 : 0;
  return launch_tile_gemm<GatedUp>(maps, p, static_cast<int64_t>(num_row_blocks) * (ffn_dim / 128), dev_status, stream, "sdd_gated");
}

int gated_grad_rows_of(const void* grad_out, const void* y_rows, const void* gate, int gate_dtype, const int32_t* row_token,
                       const int32_t* copy_row, const int32_t* num_rows, void* grad_rows, void* scaled_rows, float* row_gate,
                       void* dgate, int32_t k, int32_t d_model, int32_t num_row_blocks, cudaStream_t stream) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const int64_t blocks = std::min<int64_t>(static_cast<int64_t>(num_row_blocks) * (kTileRows / 8), info->sm_count * 8);
  gated_grad_rows_kernel<<<static_cast<unsigned>(blocks), kSmallThreads, 0, stream>>>(
      static_cast<const uint4*>(grad_out), static_cast<const float4*>(y_rows), gate, gate_dtype, row_token, copy_row, num_rows,
      static_cast<uint4*>(grad_rows), static_cast<uint4*>(scaled_rows), row_gate, dgate, k, d_model / 8);
  return check_launch("moe_gated_backward (rows)");
}

// Columns of a tile: 256, and fewer where that leaves every second SM without a tile. A tile of 128 (64) columns moves 1.3
// (2) times the operand bytes per result: halving as soon as one SM has no tile took longer (forward and backward at T = 100,
// D = 4096, F = 2048, E = 4: 195 against 172 us; T = 179, D = 2688, F = 1536, E = 10: 214 against 200), and so did waiting
// for three quarters without one (T = 1000, D = F = 1024, E = 4: 90 against 84.5).
int32_t tile_cols(int64_t num_row_blocks, int32_t width, int sm_count) {
  int32_t cols = kTileCols;
  while (cols > 64 && 2 * num_row_blocks * ((width + cols - 1) / cols) < sm_count) cols /= 2;
  return cols;
}

template <int kCols>
int gated_grad_hidden(const void* grad_rows, const float* row_gate, const void* w_down, const void* g_blocks, const void* u_blocks,
                      const int32_t* row_token, const int32_t* row_block_expert, const int32_t* padded_offsets,
                      const int32_t* tokens_per_expert, void* dg_blocks,
                      void* du_blocks, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int32_t num_row_blocks,
                      int32_t activation, int32_t* dev_status, cudaStream_t stream) {
  const char* what = "moe_gated_backward (hidden)";
  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], w_down, static_cast<uint64_t>(num_experts) * ffn_dim, d_model, kCols, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[1], grad_rows, static_cast<uint64_t>(num_row_blocks) * kTileRows, d_model, 128, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[2], grad_rows, static_cast<uint64_t>(num_row_blocks) * kTileRows, d_model, 32, 64, 2, what)) return rc;
  typename GradHidden<kCols>::Params p{};
  p.row_gate = row_gate;
  const int32_t slices = (ffn_dim + kCols - 1) / kCols;
  p.order = {row_block_expert, padded_offsets, tokens_per_expert, num_experts, slices};
  p.row_token = row_token;
  p.g = static_cast<const __nv_bfloat16*>(g_blocks);
  p.u = static_cast<const __nv_bfloat16*>(u_blocks);
  p.dg = static_cast<__nv_bfloat16*>(dg_blocks);
  p.du = static_cast<__nv_bfloat16*>(du_blocks);
  p.d_model = d_model;
  p.ffn_dim = ffn_dim;
  p.activation = activation;
  return launch_tile_gemm<GradHidden<kCols>>(maps, p, static_cast<int64_t>(num_row_blocks) * slices, dev_status, stream, what);
}

int gated_grad_weights(const void* x_rows, const void* grad_rows, const void* h_blocks, const void* dg_blocks,
                       const void* du_blocks, const int32_t* padded_offsets, const int32_t* tokens_per_expert, void* dw_gate,
                       void* dw_up, void* dw_down, int32_t d_model, int32_t ffn_dim, int32_t num_experts,
                       int32_t num_row_blocks, int32_t* dev_status, cudaStream_t stream) {
  const char* what = "moe_gated_backward (weights)";
  const uint64_t rows = static_cast<uint64_t>(num_row_blocks) * kTileRows;
  const uint64_t b_rows = static_cast<uint64_t>(num_row_blocks) * ffn_dim;
  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], x_rows, rows, d_model, 64, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[1], grad_rows, rows, d_model, 64, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[2], h_blocks, b_rows, 128, 64, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[3], dg_blocks, b_rows, 128, 64, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[4], du_blocks, b_rows, 128, 64, 64, 2, what)) return rc;
  const uint64_t up_rows = static_cast<uint64_t>(num_experts) * d_model;
  const uint64_t down_rows = static_cast<uint64_t>(num_experts) * ffn_dim;
  if (int rc = encode_2d_map(&maps.m[5], dw_down, down_rows, d_model, 32, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[6], dw_gate, up_rows, ffn_dim, 32, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[7], dw_up, up_rows, ffn_dim, 32, 64, 2, what)) return rc;
  GradWeights::Params p{};
  p.padded_offsets = padded_offsets;
  p.tokens_per_expert = tokens_per_expert;
  p.num_experts = num_experts;
  p.d_model = d_model;
  p.ffn_dim = ffn_dim;
  p.down_cols = (d_model + kTileCols - 1) / kTileCols;
  p.down_tiles = ffn_dim / kTileRows * p.down_cols;
  p.up_cols = (ffn_dim + kTileCols - 1) / kTileCols;
  p.up_tiles = d_model / kTileRows * p.up_cols;
  const int64_t tiles = static_cast<int64_t>(num_experts) * (p.down_tiles + 2ll * p.up_tiles);
  return launch_tile_gemm<GradWeights>(maps, p, tiles, dev_status, stream, what);
}

// Y = H Wd (back: false; a0 = H, w0 = Wd), or the rows of dx = dG Wg^T + dU Wu^T (a0, a1, w0, w1).
template <bool kBack>
int rows_product(const void* a0, const void* a1, const void* w0, const void* w1, const int32_t* row_token,
                 const int32_t* row_block_expert, const int32_t* padded_offsets, const int32_t* tokens_per_expert, void* rows,
                 int32_t d_model, int32_t ffn_dim,
                 int32_t num_experts, int32_t num_row_blocks, int32_t* dev_status, cudaStream_t stream) {
  const char* what = kBack ? "moe_gated_backward (x)" : "moe_gated (down)";
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const int32_t cols = tile_cols(num_row_blocks, d_model, info->sm_count);
  const uint64_t b_rows = static_cast<uint64_t>(num_row_blocks) * ffn_dim;
  TileMaps maps{};
  if (int rc = encode_2d_map(&maps.m[0], a0, b_rows, 128, 128, 64, 2, what)) return rc;
  if (int rc = encode_2d_map(&maps.m[5], a0, b_rows, 128, 32, 64, 2, what)) return rc;
  if (kBack) {
    const uint64_t w_rows = static_cast<uint64_t>(num_experts) * d_model;
    if (int rc = encode_2d_map(&maps.m[1], a1, b_rows, 128, 128, 64, 2, what)) return rc;
    if (int rc = encode_2d_map(&maps.m[6], a1, b_rows, 128, 32, 64, 2, what)) return rc;
    if (int rc = encode_2d_map(&maps.m[2], w0, w_rows, ffn_dim, cols, 64, 2, what)) return rc;
    if (int rc = encode_2d_map(&maps.m[3], w1, w_rows, ffn_dim, cols, 64, 2, what)) return rc;
  } else {
    if (int rc = encode_2d_map(&maps.m[2], w0, static_cast<uint64_t>(num_experts) * ffn_dim, d_model, 64, 64, 2, what)) return rc;
  }
  if (int rc = encode_2d_map(&maps.m[4], rows, static_cast<uint64_t>(num_row_blocks) * kTileRows, d_model, 32, 32, 4, what)) return rc;
  typename RowsProduct<kBack>::Params p{};
  const int32_t slices = (d_model + cols - 1) / cols;
  p.order = {row_block_expert, padded_offsets, tokens_per_expert, num_experts, slices};
  p.row_token = row_token;
  p.d_model = d_model;
  p.ffn_dim = ffn_dim;
  p.cols = cols;
  return launch_tile_gemm<RowsProduct<kBack>>(maps, p, static_cast<int64_t>(num_row_blocks) * slices, dev_status, stream, what);
}

int gated_join(const void* dx_rows, const int32_t* copy_row, void* dx, void* dgate, int gate_dtype, int64_t num_tokens,
               int32_t k, int32_t d_model, cudaStream_t stream) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const int64_t blocks = std::min<int64_t>((num_tokens * (d_model / 4) + kSmallThreads - 1) / kSmallThreads, info->sm_count * 16);
  return launch_small(gated_join_kernel, blocks, kSmallThreads, stream, "moe_gated_backward (join)",
                      static_cast<const float4*>(dx_rows), copy_row, static_cast<uint2*>(dx), dgate, gate_dtype, num_tokens, k,
                      d_model / 4);
}

bool aligned256(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 255u) == 0; }

// The two ways of the forward pass. The decoding way needs no layout and splits K over clusters; it starts a block per
// 64 (128) weight columns of every picked expert. From 129 copies on (and wherever the backward pass needs the layout's
// blocks) the persistent kernels of the layout are at least as fast.
constexpr int64_t kSmallCopies = 128;

// Parts of the buffers, in bytes from their start.
struct GatedBuffers {
  bool small;
  int32_t row_blocks, ffn_blocks;
  // state (keep) or scratch: the layout's arrays, then the blocks
  int64_t tokens_per_expert, padded_offsets, row_token, copy_row, row_block_expert, row_offsets, col_indices, error, work;
  int64_t x_rows, h, g, u, y;
  int64_t state_bytes, scratch_bytes;
  // scratch of the backward pass
  int64_t grad_rows, scaled_rows, row_gate, dg, du, backward_bytes;
};

int gated_buffers(int64_t num_tokens, int32_t k, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int keep,
                  GatedBuffers* b) {
  if (num_tokens <= 0 || k <= 0) return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: T and k must be positive");
  if (num_tokens > INT32_MAX / k) return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: problem too large");
  if (int rc = check_gated("moe_gated", d_model, ffn_dim, num_experts, 0, 0)) return rc;
  const int64_t n = num_tokens * k;
  int64_t row_blocks = 0, rows = 0, ffn_blocks = 0;
  if (int rc = sb_route_sizes(n, num_experts, ffn_dim, 128, &row_blocks, &rows, &ffn_blocks)) return rc;
  if (int rc = check_gated("moe_gated", d_model, ffn_dim, num_experts, static_cast<int32_t>(row_blocks), 0)) return rc;
  *b = GatedBuffers{};
  b->row_blocks = static_cast<int32_t>(row_blocks);
  b->ffn_blocks = static_cast<int32_t>(ffn_blocks);
  b->small = !keep && n <= kSmallCopies;
  int64_t at = 0;
  auto take = [&at](int64_t bytes) {
    const int64_t here = at;
    at += align256(bytes);
    return here;
  };
  if (b->small) {
    b->h = take(n * ffn_dim * 2);
    b->y = take(n * d_model * 4);
    b->scratch_bytes = at;
    return SB_OK;
  }
  b->tokens_per_expert = take(num_experts * 4ll);
  b->padded_offsets = take((num_experts + 1ll) * 4);
  b->row_token = take(rows * 4);
  b->copy_row = take(n * 4);
  b->row_block_expert = take(row_blocks * 4);
  b->row_offsets = take((row_blocks + 1) * 4);
  b->col_indices = take(row_blocks * ffn_blocks * 4);
  b->error = take(4);
  b->x_rows = take(rows * d_model * 2);
  b->y = take(rows * d_model * 4);
  b->h = take(rows * ffn_dim * 2);
  if (keep) {
    b->g = take(rows * ffn_dim * 2);
    b->u = take(rows * ffn_dim * 2);
    b->state_bytes = at;
    at = 0;
  }
  b->work = take(std::max<int64_t>(4, static_cast<int64_t>(sb_route_workspace_bytes(n, num_experts))));  // never NULL
  b->scratch_bytes = at;
  at = 0;
  b->grad_rows = take(rows * d_model * 2);
  b->scaled_rows = take(rows * d_model * 2);
  b->row_gate = take(rows * 4);
  b->dg = take(rows * ffn_dim * 2);
  b->du = take(rows * ffn_dim * 2);
  b->backward_bytes = at;
  return SB_OK;
}

int forward_small(const GatedBuffers& b, const void* x, const void* expert_idx, int idx_is_i64, const void* gate,
                  int gate_dtype, const void* w_gate, const void* w_up, const void* w_down, void* out, int32_t num_tokens,
                  int32_t k, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int32_t activation, uint8_t* scratch,
                  int32_t* dev_status, cudaStream_t stream) {
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const int32_t copies = num_tokens * k;
  const int32_t experts = std::min(copies, num_experts);  // at most so many different ones are picked
  __nv_bfloat16* h = reinterpret_cast<__nv_bfloat16*>(scratch + b.h);
  float* y = reinterpret_cast<float*>(scratch + b.y);
  const uint64_t up_rows = static_cast<uint64_t>(num_experts) * d_model;
  const uint64_t down_rows = static_cast<uint64_t>(num_experts) * ffn_dim;
  SkinnyMaps maps{};
  if (int rc = encode_2d_map(&maps.w[0], w_gate, up_rows, ffn_dim, 64, 64, 2, "moe_gated (w_gate)")) return rc;
  if (int rc = encode_2d_map(&maps.w[1], w_up, up_rows, ffn_dim, 64, 64, 2, "moe_gated (w_up)")) return rc;
  SkinnyUp::Params up{};
  up.tiles = ffn_dim / 64;
  up.shape = skinny_shape(static_cast<int64_t>(experts) * up.tiles, d_model / kSkinnyStep, copies, info->sm_count);
  up.expert_idx = expert_idx;
  up.x = static_cast<const __nv_bfloat16*>(x);
  up.h = h;
  up.idx_is_i64 = idx_is_i64;
  up.copies = copies;
  up.k = k;
  up.num_experts = num_experts;
  up.d_model = d_model;
  up.ffn_dim = ffn_dim;
  up.activation = activation;
  if (int rc = launch_skinny<SkinnyUp>(maps, up, static_cast<int64_t>(experts) * up.tiles, false, dev_status, stream, "moe_gated (up)")) return rc;
  SkinnyMaps down_maps{};
  if (int rc = encode_2d_map(&down_maps.w[0], w_down, down_rows, d_model, 64, 64, 2, "moe_gated (w_down)")) return rc;
  SkinnyDown::Params down{};
  down.tiles = d_model / 128;
  down.shape = skinny_shape(static_cast<int64_t>(experts) * down.tiles, ffn_dim / kSkinnyStep, copies, info->sm_count);
  down.expert_idx = expert_idx;
  down.h = h;
  down.y = y;
  down.idx_is_i64 = idx_is_i64;
  down.copies = copies;
  down.num_experts = num_experts;
  down.d_model = d_model;
  down.ffn_dim = ffn_dim;
  if (int rc = launch_skinny<SkinnyDown>(down_maps, down, static_cast<int64_t>(experts) * down.tiles, true, dev_status, stream, "moe_gated (down)")) return rc;
  cudaLaunchConfig_t cfg = {};
  const int32_t quads = d_model / 4;
  cfg.gridDim = dim3(static_cast<unsigned>((quads + 127) / 128), static_cast<unsigned>(num_tokens));
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&cfg, gated_small_combine_kernel, reinterpret_cast<const float4*>(y), expert_idx,
                                             idx_is_i64, gate, gate_dtype, static_cast<uint2*>(out), k, num_experts, quads);
  if (err != cudaSuccess) return fail(SB_ERR_CUDA, "moe_gated (combine): %s", cudaGetErrorString(err));
  return SB_OK;
}

}  // namespace
}  // namespace sb

using namespace sb;

extern "C" int sb_sdd_gated(const void* x, const void* w_gate, const void* w_up, const int32_t* row_token,
                            const int32_t* row_block_expert, const int32_t* padded_offsets, const int32_t* tokens_per_expert, void* x_rows, void* h_blocks, int64_t num_tokens, int32_t d_model, int32_t ffn_dim,
                            int32_t num_experts, int32_t num_row_blocks, int32_t activation, int skip_padding_rows,
                            int32_t* dev_status, sb_stream_t stream) {
  clear_error();
  if (int rc = check_gated("sdd_gated", d_model, ffn_dim, num_experts, num_row_blocks, activation)) return rc;
  if (num_row_blocks == 0) return SB_OK;
  if (any_null({x, w_gate, w_up, row_token, row_block_expert, padded_offsets, tokens_per_expert, x_rows, h_blocks}))
    return fail(SB_ERR_INVALID_ARGUMENT, "sdd_gated: NULL buffer");
  if (num_tokens <= 0) return fail(SB_ERR_INVALID_ARGUMENT, "sdd_gated: T must be positive");
  if (any_misaligned({x, w_gate, w_up, x_rows, h_blocks}))
    return fail(SB_ERR_INVALID_ARGUMENT, "sdd_gated: x, the weights, the rows and the blocks must be 16-byte aligned");
  return sdd_gated(x, w_gate, w_up, row_token, row_block_expert, padded_offsets, tokens_per_expert, x_rows, h_blocks,
                   nullptr, nullptr, num_tokens, d_model, ffn_dim, num_experts, num_row_blocks, activation, skip_padding_rows, dev_status,
                   as_stream(stream));
}

extern "C" int sb_moe_gated_bytes(int64_t num_tokens, int32_t k, int32_t d_model, int32_t ffn_dim, int32_t num_experts,
                                  int keep, int64_t* bytes) {
  clear_error();
  if (bytes == nullptr) return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated_bytes: NULL output");
  GatedBuffers b;
  if (int rc = gated_buffers(num_tokens, k, d_model, ffn_dim, num_experts, keep, &b)) return rc;
  bytes[0] = b.state_bytes;
  bytes[1] = b.scratch_bytes;
  bytes[2] = keep ? b.backward_bytes : 0;
  return SB_OK;
}

extern "C" int sb_moe_gated_forward(const void* x, const void* expert_idx, int idx_is_i64, const void* gate, int gate_dtype,
                                    const void* w_gate, const void* w_up, const void* w_down, void* out, int64_t num_tokens,
                                    int32_t k, int32_t d_model, int32_t ffn_dim, int32_t num_experts, int32_t activation,
                                    void* state, int64_t state_bytes, void* scratch, int64_t scratch_bytes,
                                    int32_t* dev_status, sb_stream_t stream) {
  clear_error();
  const int keep = state != nullptr ? 1 : 0;
  GatedBuffers b;
  if (int rc = gated_buffers(num_tokens, k, d_model, ffn_dim, num_experts, keep, &b)) return rc;
  if (int rc = check_gated("moe_gated", d_model, ffn_dim, num_experts, b.row_blocks, activation)) return rc;
  if (any_null({x, expert_idx, gate, w_gate, w_up, w_down, out, scratch})) return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: NULL buffer");
  if (any_misaligned({x, w_gate, w_up, w_down, out}) || !aligned256(state) || !aligned256(scratch))
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: buffers must be 16-byte aligned, state and scratch 256-byte aligned");
  if (gate_dtype != 0 && gate_dtype != 1) return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: gate_dtype must be 0 (bf16) or 1 (fp32)");
  if ((keep && state_bytes < b.state_bytes) || scratch_bytes < b.scratch_bytes)
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated: the buffers have %lld and %lld bytes, %lld and %lld are needed",
                (long long)state_bytes, (long long)scratch_bytes, (long long)b.state_bytes, (long long)b.scratch_bytes);
  uint8_t* temp = static_cast<uint8_t*>(scratch);
  if (b.small)
    return forward_small(b, x, expert_idx, idx_is_i64, gate, gate_dtype, w_gate, w_up, w_down, out,
                         static_cast<int32_t>(num_tokens), k, d_model, ffn_dim, num_experts, activation, temp, dev_status,
                         as_stream(stream));
  uint8_t* base = keep ? static_cast<uint8_t*>(state) : temp;
  auto ints = [base](int64_t at) { return reinterpret_cast<int32_t*>(base + at); };
  if (int rc = sb_route(expert_idx, idx_is_i64, num_tokens * k, k, num_experts, b.ffn_blocks, 128, b.row_blocks,
                        ints(b.tokens_per_expert), ints(b.padded_offsets), ints(b.row_token), ints(b.copy_row),
                        ints(b.row_block_expert), ints(b.row_offsets), ints(b.col_indices), ints(b.error), temp + b.work, stream))
    return rc;
  if (int rc = sdd_gated(x, w_gate, w_up, ints(b.row_token), ints(b.row_block_expert), ints(b.padded_offsets),
                         ints(b.tokens_per_expert), base + b.x_rows, base + b.h, keep ? base + b.g : nullptr,
                         keep ? base + b.u : nullptr, num_tokens, d_model, ffn_dim, num_experts, b.row_blocks, activation, 1, dev_status,
                         as_stream(stream)))
    return rc;
  if (int rc = rows_product<false>(base + b.h, nullptr, w_down, nullptr, ints(b.row_token), ints(b.row_block_expert),
                                   ints(b.padded_offsets), ints(b.tokens_per_expert), base + b.y, d_model, ffn_dim, num_experts, b.row_blocks, dev_status,
                                   as_stream(stream)))
    return rc;
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const int64_t blocks = std::min<int64_t>((num_tokens * (d_model / 4) + kSmallThreads - 1) / kSmallThreads, info->sm_count * 16);
  return launch_small(gated_combine_kernel, blocks, kSmallThreads, as_stream(stream), "moe_gated (combine)",
                      reinterpret_cast<const float4*>(base + b.y), ints(b.copy_row), gate, gate_dtype, static_cast<uint2*>(out),
                      num_tokens, k, d_model / 4);
}

extern "C" int sb_moe_gated_backward(const void* grad_out, const void* gate, int gate_dtype,
                                     const void* w_gate, const void* w_up, const void* w_down, const void* state,
                                     int64_t state_bytes, void* dx, void* dgate, void* dw_gate, void* dw_up, void* dw_down,
                                     int64_t num_tokens, int32_t k, int32_t d_model, int32_t ffn_dim, int32_t num_experts,
                                     int32_t activation, void* scratch, int64_t scratch_bytes, int32_t* dev_status,
                                     sb_stream_t stream) {
  clear_error();
  GatedBuffers b;
  if (int rc = gated_buffers(num_tokens, k, d_model, ffn_dim, num_experts, 1, &b)) return rc;
  if (int rc = check_gated("moe_gated_backward", d_model, ffn_dim, num_experts, b.row_blocks, activation)) return rc;
  if (gate_dtype != 0 && gate_dtype != 1)
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated_backward: gate_dtype must be 0 (bf16) or 1 (fp32)");
  if (any_null({grad_out, gate, w_gate, w_up, w_down, state, dx, dgate, dw_gate, dw_up, dw_down, scratch}))
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated_backward: NULL buffer");
  if (any_misaligned({grad_out, w_gate, w_up, w_down, dx, dw_gate, dw_up, dw_down}) || !aligned256(state) || !aligned256(scratch))
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated_backward: buffers must be 16-byte aligned, state and scratch 256-byte aligned");
  if (state_bytes < b.state_bytes || scratch_bytes < b.backward_bytes)
    return fail(SB_ERR_INVALID_ARGUMENT, "moe_gated_backward: the buffers have %lld and %lld bytes, %lld and %lld are needed",
                (long long)state_bytes, (long long)scratch_bytes, (long long)b.state_bytes, (long long)b.backward_bytes);
  const uint8_t* base = static_cast<const uint8_t*>(state);
  uint8_t* temp = static_cast<uint8_t*>(scratch);
  const cudaStream_t st = as_stream(stream);
  auto ints = [base](int64_t at) { return reinterpret_cast<const int32_t*>(base + at); };
  const int32_t* row_token = ints(b.row_token);
  float* row_gate = reinterpret_cast<float*>(temp + b.row_gate);
  if (int rc = gated_grad_rows_of(grad_out, base + b.y, gate, gate_dtype, row_token, ints(b.copy_row),
                                  ints(b.padded_offsets) + num_experts, temp + b.grad_rows, temp + b.scaled_rows, row_gate, dgate, k,
                                  d_model, b.row_blocks, st))
    return rc;
  const DeviceInfo* info = current_device_info();
  if (info == nullptr) return SB_ERR_CUDA;
  const auto grad_hidden = tile_cols(b.row_blocks, ffn_dim, info->sm_count) == kTileCols ? gated_grad_hidden<kTileCols> : gated_grad_hidden<64>;
  if (int rc = grad_hidden(temp + b.grad_rows, row_gate, w_down, base + b.g, base + b.u, row_token, ints(b.row_block_expert),
                           ints(b.padded_offsets), ints(b.tokens_per_expert), temp + b.dg, temp + b.du, d_model, ffn_dim, num_experts, b.row_blocks,
                           activation, dev_status, st))
    return rc;
  if (int rc = gated_grad_weights(base + b.x_rows, temp + b.scaled_rows, base + b.h, temp + b.dg, temp + b.du,
                                  ints(b.padded_offsets), ints(b.tokens_per_expert), dw_gate, dw_up, dw_down, d_model,
                                  ffn_dim, num_experts, b.row_blocks, dev_status, st))
    return rc;
  // The rows of dx (fp32) take the place of grad_rows and scaled_rows (bf16, one behind the other), which the hidden
  // and the weight gradients were the last to read.
  if (int rc = rows_product<true>(temp + b.dg, temp + b.du, w_gate, w_up, row_token, ints(b.row_block_expert),
                                  ints(b.padded_offsets), ints(b.tokens_per_expert), temp + b.grad_rows, d_model, ffn_dim, num_experts, b.row_blocks,
                                  dev_status, st))
    return rc;
  return gated_join(temp + b.grad_rows, ints(b.copy_row), dx, dgate, gate_dtype, num_tokens, k, d_model, st);
}
