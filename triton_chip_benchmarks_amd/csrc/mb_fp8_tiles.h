// Products of FP8 operands with block scales by tiles: persistent workgroups on the
// ring GEMM's loads (mb_gemm_ring.h), a scale for each row and step.
#pragma once

#include "mb_fp8_few.h"
#include "mb_mx_stream.h"

namespace mb {

// The epilogues of Fp8Epilogue, and gated with the gate and up kept.
enum Fp8TileEpilogue { kTilePlain = kFp8Plain, kTileGated = kFp8Gated, kTileGatedFp8 = kFp8GatedFp8, kTileGatedKept };

// A tile of BM rows of W (gated: 32 gates and their 32 ups in turn) by BN of X, a step
// of K of 128 elements: whole blocks. Per stage of the ring, the operands (the layout of
// RingTile) and the scales of the step's four blocks, a dword each row or block of rows:
// 1024 bytes of W's (gated: the gates'), of X's, and (gated) of the ups'.
template <int EPILOGUE, int BM, int BN, int STAGES>
struct Fp8Tile {
  static constexpr bool GATED = EPILOGUE != kTilePlain;
  static constexpr int ROWB = 128, WM = BM / 2, WN = BN / 2, FM = WM / 32, FN = WN / 32, CHUNKS = 4;
  static constexpr int DMA_A = BM / 32, DMA_B = BN / 32, DMAS = DMA_A + DMA_B + 1;  // per wave and step
  static constexpr int OPERANDS = (BM + BN) * ROWB, STAGE = OPERANDS + (GATED ? 3 : 2) * 1024;
  static constexpr int MFMAS = FM * FN * 2, READS = (FM + FN) * CHUNKS;
  static constexpr int SHARED = STAGES * STAGE + (EPILOGUE == kTileGatedFp8 ? 2 * BN * 4 : 0);
  static constexpr int RESIDENT = 160 * 1024 / SHARED;  // workgroups a CU's LDS holds
  static_assert(BM % 64 == 0 && BN % 64 == 0 && BM <= 256 && BN <= 256, "whole instructions; scales of a DMA");
  static_assert(!GATED || BM == 256, "a gated tile is 128 columns of the output: whole blocks of it");
  static_assert(STAGES >= 2 && (STAGES - 1) * DMAS < 64 && RESIDENT >= 1, "vmcnt counts the DMAs in flight; LDS");
  // 256 accumulators a lane leave room for one set of fragments, refilled in place.
  static constexpr bool ROLLED = FM * FN == 16;
  static_assert(!ROLLED || STAGES == 2, "the rolled step");
  // Stores of a lane and tile, 16 bytes each but for the scales.
  static constexpr int stores(int item) {
    return EPILOGUE == kTilePlain     ? FM * FN * item
           : EPILOGUE == kTileGated   ? FM * FN / 2 * item
           : EPILOGUE == kTileGatedFp8 ? FM * FN / 2 + 4 * FN
                                       : FM * FN / 2 * item + FM * FN * item;
  }
};

// A number of the workgroup's that is seldom needed, in a vector register: the scalar
// ones are short.
struct Kept {
  int lanes;
  __device__ __forceinline__ explicit Kept(int v) : lanes(v) { asm volatile("" : "+v"(lanes)); }
  __device__ __forceinline__ operator int() const { return __builtin_amdgcn_readfirstlane(lanes); }
};

// Y = X . W^T, or the gated pair of it: the loads, fragments and counted waits of
// mx_product_stream_kernel (mb_mx_stream.h), whose loads run on over the ends of tiles
// while a tile is stored from its registers. A step is one block of K: a lane reads one
// scale byte for each of its fragments, and v_mfma_scale_f32_32x32x64_f8f6f4 applies
// them, so that the sums over blocks stay in the accumulators. For fp32 outputs a
// fragment goes to bf16 in registers (see Fp8Codes) and v_mfma_f32_32x32x16_bf16.
//
// Gated: W's tile holds 32 gates and the 32 ups of the same columns in turn, so that a
// lane has both of an output in two accumulators, and 128 columns are a tile and a block
// of the FP8 output; the two waves of a row exchange its largest magnitude in LDS.
//
// ROLLED (256x256): the 32 products of a step run row of fragments by row; a fragment
// of the next step is read over the one that was used last, six products or more before
// it is needed. The step's barrier lies after its first products: by then the last
// fragments of this step have arrived, so that its stage may be loaded again, and the
// next step's loads, issued behind the last barrier, have had a step's time to land.
//
// The matrix cores bound it, and the clock that the power limit leaves them: 8192^3 from
// operands in the caches takes 388 us (2.83 PFLOP/s; this library's FP8 product without
// scales 376 to 404), with cold ones 418 to 450. With the barrier after the fourth
// product instead of the second 433 cold, with two barriers a step, each for half of the
// operands, 464. By 256x128 the same product takes 474: its loads are half as many again.
//
// There are at most kStreamExperts experts.
template <class Y, int EPILOGUE, int BM, int BN, int STAGES>
__global__ void __launch_bounds__(256, (Fp8Tile<EPILOGUE, BM, BN, STAGES>::RESIDENT))
    fp8_tiles_kernel(Fp8Product p, int band) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Tile = Fp8Tile<EPILOGUE, BM, BN, STAGES>;
  constexpr bool GATED = Tile::GATED, WIDE = sizeof(Y) == 4;
  constexpr int ROWB = Tile::ROWB, FM = Tile::FM, FN = Tile::FN, CH = Tile::CHUNKS;
  constexpr int STORES = Tile::stores(sizeof(Y));
  static_assert((STAGES - 2) * Tile::DMAS + STORES < 64, "vmcnt counts DMAs and stores in flight");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * Tile::STAGE];
  __shared__ uint32_t row_largest[2][EPILOGUE == kTileGatedFp8 ? BN : 1];
  const int n = p.n, k = p.k, rows = p.rows;
  if (k < 0) lds[threadIdx.x] = 0;  // keeps DMA-written reads live; never executed
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  RowTiles<BN> row_tiles;
  row_tiles.init(p.offsets, p.experts, rows, lane);
  // XCD c (workgroups c, c + 8, ..) takes a contiguous share of the tiles, its
  // workgroups one after the other.
  constexpr int COLUMNS = GATED ? BM / 2 : BM;  // of the output
  const int columns = (n + COLUMNS - 1) / COLUMNS;
  const int count = row_tiles.total * columns, xcd = blockIdx.x % kXcds;
  const Kept columns_kept(columns);
  const Kept share(count / kXcds + (xcd < count % kXcds));
  const Kept share0(xcd * (count / kXcds) + min(xcd, count % kXcds));
  const Kept workers((static_cast<int>(gridDim.x) - xcd + kXcds - 1) / kXcds);
  const int row_bytes = (k + 15) / 16 * 16, k_steps = (k + ROWB - 1) / ROWB;
  const int width = GATED ? 2 * n : n;
  const int w_scales = (width + (1 << p.w_shift) - 1) >> p.w_shift;
  const int x_scales = (rows + (1 << p.x_shift) - 1) >> p.x_shift;
  const int scale_steps = (k_steps + 3) / 4;

  // Tile `index` of the share: bands of row tiles, the rows of a band first.
  struct At {
    int expert, m0, n0, live;  // m0: the first column of the output
  };
  auto locate = [&](int index) __attribute__((always_inline)) {
    const int pid = share0 + index, columns = columns_kept;
    const int per_band = band * columns, first_tile = pid / per_band * band;
    const int in_band = min(row_tiles.total - first_tile, band);
    int expert, row, end;
    row_tiles.find(__builtin_amdgcn_readfirstlane(first_tile + pid % per_band % in_band), expert, row, end);
    return At{__builtin_amdgcn_readfirstlane(expert),
              __builtin_amdgcn_readfirstlane(pid % per_band / in_band * COLUMNS), __builtin_amdgcn_readfirstlane(row),
              __builtin_amdgcn_readfirstlane(min(BN, end - row))};
  };

  // ---- the DMA stream: step `dma_step` of tile `dma_index` is loaded next
  const int drow = lane >> 3;
  const int chunk0 = (lane & 7) ^ (drow >> 1), chunk1 = chunk0 ^ 4;
  const int limit0 = row_bytes - 16 * chunk0, limit1 = row_bytes - 16 * chunk1;
  int va[Tile::DMA_A], vb[Tile::DMA_B];
#pragma unroll
  for (int i = 0; i < Tile::DMA_A; ++i) {
    // Gated, a wave's 64 rows are 32 gates and their ups: rows 32 wave .. of each.
    const int row = GATED ? wave * 32 + 8 * (i & 3) : wave * (BM / 4) + 8 * i;
    va[i] = (row + drow) * row_bytes + 16 * ((i & 1) ? chunk1 : chunk0);
  }
#pragma unroll
  for (int i = 0; i < Tile::DMA_B; ++i)
    vb[i] = (wave * (BN / 4) + 8 * i + drow) * row_bytes + 16 * ((i & 1) ? chunk1 : chunk0);
  const uint32_t lds_base =
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
  // Waves 0 and 2 move W's scales (gated: the gates' and the ups'), 1 and 3 X's.
  const int scale_rows = (wave & 1) ? x_scales : w_scales;
  const uint32_t scale_to = lds_base + Tile::OPERANDS + ((wave & 1) ? 1024 : GATED && wave == 2 ? 2048 : 0);
  int dma_step = 0;
  struct Source {
    __amdgpu_buffer_rsrc_t a[GATED ? 2 : 1], b, scales;
    int scale_row0;
  };
  auto source = [&](const At& at) __attribute__((always_inline)) {
    const int64_t e = at.expert;
    Source from;
    const int taken = min(COLUMNS, n - at.m0) * row_bytes;
    from.a[0] = buffer_rsrc(p.w + (e * width + at.m0) * row_bytes, taken);
    if constexpr (GATED) from.a[1] = buffer_rsrc(p.w + (e * width + n + at.m0) * row_bytes, taken);
    from.b = buffer_rsrc(static_cast<const uint8_t*>(p.x) + static_cast<int64_t>(at.n0) * row_bytes,
                         at.live * row_bytes);
    from.scales = (wave & 1) ? buffer_rsrc(p.sx, scale_steps * x_scales * 4)
                             : buffer_rsrc(p.sw + e * scale_steps * w_scales * 4, scale_steps * w_scales * 4);
    from.scale_row0 = (wave & 1) ? at.n0 >> p.x_shift : ((GATED && wave == 2 ? n : 0) + at.m0) >> p.w_shift;
    return from;
  };
  Kept index(blockIdx.x / kXcds);
  if (index >= share) return;
  // The DMAs run ahead of the products by STAGES steps, and tiles by as many as
  // those make; past the last tile they load it once more.
  const At begin = locate(index);
  Source from = source(begin);
  Kept here_m0(begin.m0), here_n0(begin.n0), here_live(begin.live);
  Kept dma_index(index);
  auto dma = [&](auto i_c, uint32_t stage) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int kb = dma_step * ROWB;
    if constexpr (i < Tile::DMA_A) {
      dma16(from.a[GATED ? i >> 2 : 0], kb < ((i & 1) ? limit1 : limit0) ? va[i] : kOutOfRange, kb,
            lds_base + (wave * (BM / 4) + 8 * i) * ROWB, stage);
    } else if constexpr (i < Tile::DMA_A + Tile::DMA_B) {
      constexpr int j = i - Tile::DMA_A;
      dma16(from.b, kb < ((j & 1) ? limit1 : limit0) ? vb[j] : kOutOfRange, kb,
            lds_base + (BM + wave * (BN / 4) + 8 * j) * ROWB, stage);
    } else {
      dma16(from.scales, lane * 16,
            __builtin_amdgcn_readfirstlane(((dma_step >> 2) * scale_rows + from.scale_row0) * 4), scale_to, stage);
    }
  };
  // After a step's DMAs: the next one, in the tile after at the end of a tile.
  auto dma_advance = [&]() __attribute__((always_inline)) {
    if (++dma_step == k_steps) {
      dma_step = 0;
      dma_index = Kept(dma_index + workers);
      from = source(locate(min(static_cast<int>(dma_index), static_cast<int>(share) - 1)));
    }
  };

  // ---- fragments, as in ring_accumulate
  const int wm = wave & 1, wn = wave >> 1;
  const int lrow = lane % 32, lgroup = lane / 32;
  const int swizzle = ((lrow >> 1) & 7) ^ lgroup;
  const uint32_t la = (wm * Tile::WM + lrow) * ROWB + (swizzle << 4);
  const uint32_t lb = (BM + wn * Tile::WN + lrow) * ROWB + (swizzle << 4);
  struct Set {
    i32x4 a[FM][CH], b[FN][CH];
    uint32_t sa[FM], sb[FN];
  };
  auto read = [&](auto r_c, Set& set, uint32_t stage) __attribute__((always_inline)) {
    constexpr int r = decltype(r_c)::value, c = r / (FM + FN), f = r % (FM + FN);
    if constexpr (f < FM)
      set.a[f][c] = *reinterpret_cast<const i32x4*>(lds + stage + (la ^ (c * 2 << 4)) + f * 32 * ROWB);
    else
      set.b[f - FM][c] = *reinterpret_cast<const i32x4*>(lds + stage + (lb ^ (c * 2 << 4)) + (f - FM) * 32 * ROWB);
  };
  // Bytes of the scales in a stage: tiles start on whole blocks of rows, but for the ups.
  int sa_at[FM], sb_at[FN];
#pragma unroll
  for (int f = 0; f < FM; ++f) {
    if constexpr (GATED) {
      const int row = (wm * FM + f) / 2 * 32 + lrow;
      sa_at[f] = Tile::OPERANDS + (f % 2 ? 2048 + ((((n & ((1 << p.w_shift) - 1)) + row) >> p.w_shift) * 4)
                                         : (row >> p.w_shift) * 4);
    } else {
      sa_at[f] = Tile::OPERANDS + ((wm * Tile::WM + f * 32 + lrow) >> p.w_shift) * 4;
    }
  }
#pragma unroll
  for (int f = 0; f < FN; ++f)
    sb_at[f] = Tile::OPERANDS + 1024 + ((wn * Tile::WN + f * 32 + lrow) >> p.x_shift) * 4;
  auto read_scales = [&](Set& set, int kt, uint32_t stage) __attribute__((always_inline)) {
    const uint8_t* at = lds + stage + (kt & 3);
#pragma unroll
    for (int f = 0; f < FM; ++f) set.sa[f] = at[sa_at[f]];
#pragma unroll
    for (int f = 0; f < FN; ++f) set.sb[f] = at[sb_at[f]];
  };
  f32x16 acc[FM][FN];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x16{};
  };
  // Fragment f of W (f < FM) or X with its scale.
  [[maybe_unused]] auto refill = [&](auto f_c, Set& set, int kt, uint32_t stage) __attribute__((always_inline)) {
    constexpr int f = decltype(f_c)::value;
    static_for<0, CH>([&](auto c_c) __attribute__((always_inline)) {
      read(std::integral_constant<int, decltype(c_c)::value * (FM + FN) + f>{}, set, stage);
    });
    const uint8_t* at = lds + stage + (kt & 3);
    if constexpr (f < FM)
      set.sa[f] = at[sa_at[f]];
    else
      set.sb[f - FM] = at[sb_at[f - FM]];
  };
  // Products q of a step, half of its K after the other. Wide operands are made at the
  // head of a half.
  Fp8Wide wide_a[WIDE ? FM : 1], wide_b[WIDE ? FN : 1];
  auto mma = [&](auto q_c, const Set& set) __attribute__((always_inline)) {
    constexpr int q = decltype(q_c)::value, h = q / (FM * FN), i = q % (FM * FN) / FN, j = q % FN;
    if constexpr (WIDE) {
      if constexpr (q % (FM * FN) == 0) {
#pragma unroll
        for (int f = 0; f < FM; ++f) wide_a[f] = fp8_widen(Fp8Codes{set.a[f][2 * h], set.a[f][2 * h + 1]}, set.sa[f]);
#pragma unroll
        for (int f = 0; f < FN; ++f) wide_b[f] = fp8_widen(Fp8Codes{set.b[f][2 * h], set.b[f][2 * h + 1]}, set.sb[f]);
      }
#pragma unroll
      for (int g = 0; g < 4; ++g)
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wide_a[i].at[g], wide_b[j].at[g], acc[i][j], 0, 0, 0);
    } else {
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(
          __builtin_shufflevector(set.a[i][2 * h], set.a[i][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7),
          __builtin_shufflevector(set.b[j][2 * h], set.b[j][2 * h + 1], 0, 1, 2, 3, 4, 5, 6, 7), acc[i][j], 0, 0, 0,
          static_cast<int>(set.sa[i]), 0, static_cast<int>(set.sb[j]));
    }
  };

  // ---- the output tile: 16 bytes a lane and store, eight (fp32: four) columns
  constexpr int ES = sizeof(Y), PIECE = 16 / ES;
  // An accumulator stays one up to here: taken out of it early, all of them exceed the
  // vector registers.
  auto pin = [&](f32x16& sums) __attribute__((always_inline)) { asm volatile("" : "+a"(sums)); };
  int side = wave;  // the wave's number, made anew at each tile with all that follows from it
  // Accumulators ODD, STEP + ODD, .. of COUNT blocks of 32 columns a wave to rows of
  // `pitch` elements, `limit` columns of them inside.
  auto store_block = [&](auto step_c, auto odd_c, Y* to, int pitch, int limit, int live)
                         __attribute__((always_inline)) {
    constexpr int STEP = decltype(step_c)::value, ODD = decltype(odd_c)::value, COUNT = FM / STEP;
    const int wm = side & 1, wn = side >> 1;
    int here_lane = lane;
    asm volatile("" : "+v"(here_lane), "+s"(pitch));  // offsets are made at each tile: kept over it, they take its registers
    const int lrow = here_lane % 32, lgroup = here_lane / 32;
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
        to, (short)0, ((live - 1) * pitch + min(2 * COUNT * 32, limit)) * ES, kBufferWord3);
    // put(row in elements, column, its piece) for every piece of the lane.
    auto pieces = [&](auto&& put) __attribute__((always_inline)) {
      auto f = [&](int row, int column, i32x4 v) __attribute__((always_inline)) {
        asm volatile("" : "+v"(column));  // one piece's masks at a time: all of them exceed the SGPRs
        put(row, column, v);
        __builtin_amdgcn_sched_barrier(0);  // and one piece's accumulators
      };
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int row = (wn * Tile::WN + j * 32 + lrow) * pitch;
#pragma unroll
        for (int i = 0; i < COUNT; ++i) {
          const int column = (wm * COUNT + i) * 32;
          f32x16& sums = acc[STEP * i + ODD][j];
          pin(sums);
          if constexpr (ES == 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 v = {sums[4 * q], sums[4 * q + 1], sums[4 * q + 2], sums[4 * q + 3]};
              f(row, column + out_row_32(here_lane, 4 * q), __builtin_bit_cast(i32x4, v));
            }
          } else {
            // Lanes 0-31 hold columns 8q .. 8q + 3 of their row, lanes 32-63 the next four of the same rows.
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
              uint32_t word[2][2];
#pragma unroll
              for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const Y pair[2] = {static_cast<Y>(sums[4 * (q + s) + 2 * h]),
                                     static_cast<Y>(sums[4 * (q + s) + 2 * h + 1])};
                  __builtin_memcpy(&word[s][h], pair, 4);
                }
              const auto low = __builtin_amdgcn_permlane32_swap(word[0][0], word[1][0], false, false);
              const auto high = __builtin_amdgcn_permlane32_swap(word[0][1], word[1][1], false, false);
              f(row, column + 8 * (q + lgroup),
                i32x4{static_cast<int>(low[0]), static_cast<int>(high[0]), static_cast<int>(low[1]),
                      static_cast<int>(high[1])});
            }
          }
        }
      }
    };
    // Rows past `live` lie past the buffer. Every wave issues the same STORES,
    // which vmcnt counts; those of an edge beside them only make it wait for more.
    const bool ragged = limit < 2 * COUNT * 32 && limit % PIECE;  // the rows end inside a piece
    pieces([&](int row, int column, i32x4 v) __attribute__((always_inline)) {
      __builtin_amdgcn_raw_buffer_store_b128(v, rc, column + PIECE <= limit ? (row + column) * ES : kOutOfRange, 0, 0);
      if (ragged) {
#pragma unroll
        for (int c = 0; c < PIECE - 1; ++c) {
          const bool inside = column + PIECE > limit && column + c < limit;
          const int offset = inside ? (row + column + c) * ES : kOutOfRange;
          const int word = v[c * ES / 4];
          if constexpr (ES == 4)
            __builtin_amdgcn_raw_buffer_store_b32(word, rc, offset, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b16(static_cast<short>(c % 2 ? word >> 16 : word), rc, offset, 0, 0);
        }
      }
    });
  };
  auto store = [&](const At& at) __attribute__((always_inline)) {
    int n = p.n;
    asm volatile("" : "+s"(side), "+s"(n));
    [[maybe_unused]] const int wm = side & 1, wn = side >> 1;
    const int limit = n - at.m0;  // columns of the tile inside n, at least
    const int64_t row0 = at.n0;
    constexpr std::integral_constant<int, 0> kFirst{};
    constexpr std::integral_constant<int, 1> kSecond{};
    constexpr std::integral_constant<int, 2> kPairs{};
    if constexpr (EPILOGUE == kTilePlain) {
      store_block(kSecond, kFirst, static_cast<Y*>(p.y) + row0 * n + at.m0, n, limit, at.live);
    } else {
      if constexpr (EPILOGUE == kTileGatedKept) {
        Y* pair = static_cast<Y*>(p.gate_up) + row0 * 2 * n + at.m0;
        store_block(kPairs, kFirst, pair, 2 * n, limit, at.live);
        store_block(kPairs, kSecond, pair + n, 2 * n, limit, at.live);
      }
#pragma unroll
      for (int i = 0; i < FM / 2; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          pin(acc[2 * i][j]);
          pin(acc[2 * i + 1][j]);
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            acc[2 * i][j][r] = gated(acc[2 * i][j][r], acc[2 * i + 1][j][r]);
            if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // four gates' signs at a time: all exceed the SGPRs
          }
          pin(acc[2 * i][j]);
        }
      if constexpr (EPILOGUE != kTileGatedFp8) {
        store_block(kPairs, kFirst, static_cast<Y*>(p.y) + row0 * n + at.m0, n, limit, at.live);
      } else {
        const int pitch = (n + 15) / 16 * 16, block = at.m0 / 128, past = (n + 127) / 128;
        int here_lane = lane;
        asm volatile("" : "+v"(here_lane));
        const int lrow = here_lane % 32, lgroup = here_lane / 32;
        // Columns past n have codes of zero, but scales of other rows or steps: a NaN among those is not the block's.
        if (limit < COLUMNS) {
#pragma unroll
          for (int i = 0; i < FM / 2; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) {
              int left = limit - (wm * (FM / 2) + i) * 32;
              pin(acc[2 * i][j]);
              asm volatile("" : "+v"(left));
#pragma unroll
              for (int r = 0; r < 16; ++r) {
                if (out_row_32(here_lane, r) >= left) acc[2 * i][j][r] = 0.0f;
                __builtin_amdgcn_sched_barrier(0);
              }
              pin(acc[2 * i][j]);
            }
        }
        uint32_t largest[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          largest[j] = 0;
#pragma unroll
          for (int i = 0; i < FM / 2; ++i) {
            pin(acc[2 * i][j]);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float v = acc[2 * i][j][r];
              largest[j] = max(largest[j], float_bits(v) & 0x7fffffffu);
            }
            __builtin_amdgcn_sched_barrier(0);
          }
          const auto other = __builtin_amdgcn_permlane32_swap(largest[j], largest[j], false, false);
          largest[j] = max(static_cast<uint32_t>(other[0]), static_cast<uint32_t>(other[1]));
          row_largest[wm][wn * Tile::WN + j * 32 + lrow] = largest[j];
        }
        lds_barrier();
        const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
            static_cast<uint8_t*>(p.y) + row0 * pitch + at.m0, (short)0, at.live * pitch - at.m0, kBufferWord3);
        uint32_t scales[FN];
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          int row = wn * Tile::WN + j * 32 + lrow;
          const uint32_t scale = fp8_scale_byte(max(largest[j], row_largest[wm ^ 1][row]));
          asm volatile("" : "+v"(row));
          scales[j] = scale;
#pragma unroll
          for (int i = 0; i < FM / 2; ++i) {
            // Lanes 0-31 take columns 0 .. 15 of the 32, lanes 32-63 the rest.
            pin(acc[2 * i][j]);
            uint32_t word[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              word[q] = fp8_encode4(acc[2 * i][j][4 * q], acc[2 * i][j][4 * q + 1], acc[2 * i][j][4 * q + 2],
                                    acc[2 * i][j][4 * q + 3], scale);
            const auto even = __builtin_amdgcn_permlane32_swap(word[0], word[2], false, false);
            const auto odd = __builtin_amdgcn_permlane32_swap(word[1], word[3], false, false);
            int column = (wm * (FM / 2) + i) * 32 + 16 * lgroup;
            asm volatile("" : "+v"(column));
            __builtin_amdgcn_raw_buffer_store_b128(
                i32x4{static_cast<int>(even[0]), static_cast<int>(even[1]), static_cast<int>(odd[0]),
                      static_cast<int>(odd[1])},
                rc, at.m0 + column < pitch ? row * pitch + column : kOutOfRange, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        // A byte of each of `live` rows' dwords, and 127 in the rest of a last one.
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
            p.sy + (int64_t{block / 4} * rows + row0) * 4, (short)0, at.live * 4, kBufferWord3);
        int low = block % 4, high = block + 1 == past ? 3 : low;
        asm volatile("" : "+v"(low), "+v"(high));
#pragma unroll
        for (int j = 0; j < FN; ++j) {
          const int scale_at = lgroup == 0 && wm == 0 ? (wn * Tile::WN + j * 32 + lrow) * 4 : kOutOfRange;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            __builtin_amdgcn_raw_buffer_store_b8(static_cast<char>(b == low ? scales[j] : 127u), rs,
                                                 b >= low && b <= high ? scale_at + b : kOutOfRange, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
    }
  };

#pragma unroll 1  // one copy of dma_advance
  for (uint32_t at = 0; at < STAGES * Tile::STAGE; at += Tile::STAGE) {
    static_for<0, Tile::DMAS>([&](auto i_c) __attribute__((always_inline)) { dma(i_c, at); });
    dma_advance();
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only((STAGES - 1) * Tile::DMAS));
  lds_barrier();
  Set set0, set1;
  static_for<0, Tile::READS>([&](auto r_c) __attribute__((always_inline)) { read(r_c, set0, 0); });
  read_scales(set0, 0, 0);

  int with_stores = 0;  // steps whose DMAs a tile's stores have followed
  uint32_t stage = 0;
  auto step = [&](int kt, const Set& set, Set& next) __attribute__((always_inline)) {
    if (with_stores > 0)
      __builtin_amdgcn_s_waitcnt(vmcnt_only((STAGES - 2) * Tile::DMAS + STORES));
    else
      __builtin_amdgcn_s_waitcnt(vmcnt_only((STAGES - 2) * Tile::DMAS));
    --with_stores;
    asm("" : "+s"(with_stores));  // one copy of the loop for both waits
    lds_barrier();
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t next_stage = stage == (STAGES - 1) * Tile::STAGE ? 0 : stage + Tile::STAGE;
    read_scales(next, kt + 1 == k_steps ? 0 : kt + 1, next_stage);
    constexpr int NQ = Tile::MFMAS, NR = Tile::READS, READ_Q = NQ - NQ / 4;
    static_for<0, NQ>([&](auto q_c) __attribute__((always_inline)) {
      constexpr int q = decltype(q_c)::value;
      constexpr int r0 = q < READ_Q ? q * NR / READ_Q : NR, r1 = q + 1 < READ_Q ? (q + 1) * NR / READ_Q : NR;
      static_for<r0, r1>([&](auto r_c) __attribute__((always_inline)) { read(r_c, next, next_stage); });
      static_for<q * Tile::DMAS / NQ, (q + 1) * Tile::DMAS / NQ>(
          [&](auto i_c) __attribute__((always_inline)) { dma(i_c, stage); });
      mma(q_c, set);
      __builtin_amdgcn_sched_barrier(0);
    });
    // The products stay between their loads, whatever branches follow.
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+a"(acc[i][j]));
    stage = next_stage;
    dma_advance();
  };
  [[maybe_unused]] auto rolled = [&](int kt, Set& set) __attribute__((always_inline)) {
    constexpr int NQ = Tile::MFMAS, BARRIER = 2, SPREAD = 22;
    const uint32_t next_stage = stage == 0 ? Tile::STAGE : 0;
    const int next = kt + 1 == k_steps ? 0 : kt + 1;
    static_for<0, NQ>([&](auto q_c) __attribute__((always_inline)) {
      constexpr int q = decltype(q_c)::value, i = q / (2 * FN), j = q / 2 % FN, h = q % 2;
      if constexpr (q == BARRIER) {
        if (with_stores > 0)
          __builtin_amdgcn_s_waitcnt(vmcnt_only(STORES));
        else
          __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
        --with_stores;
        lds_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (q >= BARRIER && q < BARRIER + SPREAD)
        static_for<(q - BARRIER) * Tile::DMAS / SPREAD, (q - BARRIER + 1) * Tile::DMAS / SPREAD>(
            [&](auto i_c) __attribute__((always_inline)) { dma(i_c, stage); });
      mma(std::integral_constant<int, (h * FM + i) * FN + j>{}, set);
      if constexpr (j == FN - 1 && h == 1) refill(std::integral_constant<int, i>{}, set, next, next_stage);
      if constexpr (i == FM - 1 && h == 1) refill(std::integral_constant<int, FM + j>{}, set, next, next_stage);
      __builtin_amdgcn_sched_barrier(0);
    });
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) asm volatile("" : "+a"(acc[i][j]));
    stage = next_stage;
    dma_advance();
  };
  while (true) {
    clear();
    if constexpr (Tile::ROLLED) {
#pragma unroll 1
      for (int kt = 0; kt < k_steps; ++kt) rolled(kt, set0);
    } else {
      int kt = 0;
      do {
        step(kt, set0, set1);
        if (kt + 1 < k_steps)
          step(kt + 1, set1, set0);
        else
          set0 = set1;  // the next tile's first fragments
        kt += 2;
      } while (kt < k_steps);
    }
    store(At{0, here_m0, here_n0, here_live});
    with_stores = STAGES - 1;
    index = Kept(index + workers);
    if (index >= share) break;
    const At here = locate(index);
    here_m0 = Kept(here.m0);
    here_n0 = Kept(here.n0);
    here_live = Kept(here.live);
    if constexpr (Tile::ROLLED && GATED) {
      // The next tile's first fragments again: kept over the gates, they exceed the registers.
      static_for<0, Tile::READS>([&](auto r_c) __attribute__((always_inline)) { read(r_c, set0, stage); });
      read_scales(set0, 0, stage);
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // no DMA of a step past the last may land in a later workgroup's LDS
#endif
}

}  // namespace mb
