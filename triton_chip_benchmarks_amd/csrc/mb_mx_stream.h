// Persistent MXFP4 product kernel: the ring GEMM's K loop run on over a
// workgroup's tiles without a pause between them.
#pragma once

#include "mb_elem.h"
#include "mb_gemm_ring.h"

namespace mb {

// Rows first .. last - 1 of expert `e`; all of them without offsets. Clamped, so
// that whatever `offsets` holds, no row outside 0 .. rows - 1 is touched.
__device__ __forceinline__ void expert_rows(const int32_t* __restrict__ offsets, uint32_t e, int rows, int& first,
                                            int& last) {
  first = offsets ? max(0, min(offsets[e], rows)) : 0;
  last = offsets ? max(first, min(offsets[e + 1], rows)) : rows;
}

constexpr int kStreamExperts = 256;  // four a lane

// Row tiles (BN rows each, an expert's rows starting a tile of their own) in the
// order of the experts: lane l holds experts l, 64 + l, ...
template <int BN>
struct RowTiles {
  int end[kStreamExperts / 64];    // tiles up to and with this expert
  int tiles[kStreamExperts / 64];  // its own
  int first[kStreamExperts / 64], last[kStreamExperts / 64];  // its rows
  int total, rows;
  bool dense;

  __device__ __forceinline__ void init(const int32_t* __restrict__ offsets, int experts, int all_rows, int lane) {
    rows = all_rows;
    dense = offsets == nullptr;
    total = (rows + BN - 1) / BN;
    if (dense) return;
    total = 0;
#pragma unroll
    for (int b = 0; b < kStreamExperts / 64; ++b) {
      const int e = b * 64 + lane;
      first[b] = last[b] = 0;
      if (e < experts) expert_rows(offsets, e, rows, first[b], last[b]);
      tiles[b] = (last[b] - first[b] + BN - 1) / BN;
      int scan = tiles[b];
#pragma unroll
      for (int offset = 1; offset < 64; offset <<= 1) {
        const int v = __shfl_up(scan, offset, 64);
        if (lane >= offset) scan += v;
      }
      end[b] = total + scan;
      total += __builtin_amdgcn_readlane(scan, 63);
    }
  }

  // Expert, first row and last row of row tile `tile` < total.
  __device__ __forceinline__ void find(int tile, int& expert, int& row, int& row_end) const {
    expert = 0;
    row = tile * BN;
    row_end = rows;
    if (dense) return;
    bool found = false;
#pragma unroll
    for (int b = 0; b < kStreamExperts / 64; ++b) {
      const uint64_t past = __ballot(end[b] > tile);
      if (!found && past) {
        found = true;
        const int at = __builtin_ctzll(past);
        expert = b * 64 + at;
        row = __builtin_amdgcn_readlane(first[b], at) +
              (tile - __builtin_amdgcn_readlane(end[b] - tiles[b], at)) * BN;
        row_end = __builtin_amdgcn_readlane(last[b], at);
      }
    }
  }
};

// Y = X . W^T with BM features of BN rows a tile, as mx_product_ring_kernel, a
// workgroup for all the tiles of its place on a CU. That kernel's workgroup of
// 256x128 spends 5.9 us
// beside the 16 of a K of 4096: it waits for its first operands, and nothing else
// runs on the CU while it stores. Here the DMAs run STAGES steps ahead of the
// products over the ends of tiles, and a tile is stored from its registers, whose
// halves of eight neighbouring features meet by v_permlane32_swap, while the next
// one's operands arrive.
//
// vmcnt counts a tile's stores too, in order with the DMAs: a step needs the DMAs
// issued two steps before, after which one step's DMAs and, in the first two
// steps of a tile, the stores of the tile before have been issued.
//
// There are at most kStreamExperts experts.
template <class T, int BM, int BN, int STAGES>
__global__ void __launch_bounds__(256)
    mx_product_stream_kernel(const uint8_t* __restrict__ x, const uint8_t* __restrict__ sx,
                             const uint8_t* __restrict__ w, const uint8_t* __restrict__ sw, T* __restrict__ y,
                             int rows, int n, int k, const int32_t* __restrict__ offsets, int experts, int band) {
#if defined(__HIP_DEVICE_COMPILE__)
  using Op = MfmaMxfp4;
  using Tile = RingTile<Op, BM, BN, STAGES>;
  constexpr int ROWB = Tile::ROWB, FM = Tile::FM, FN = Tile::FN, CH = Tile::CHUNKS;
  constexpr int STORES = FM * FN * 16 * sizeof(T) / 16;  // of a lane and tile
  static_assert((STAGES - 2) * Tile::DMAS + STORES < 64, "vmcnt counts DMAs and stores in flight");
  __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * Tile::STAGE];
  if (k < 0) lds[threadIdx.x] = 0;  // keeps DMA-written reads live; never executed
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

  RowTiles<BN> row_tiles;
  row_tiles.init(offsets, experts, rows, lane);
  // XCD c (workgroups c, c + 8, ..) takes a contiguous share of the tiles, its
  // workgroups one after the other.
  const int columns = (n + BM - 1) / BM;
  const int count = row_tiles.total * columns, xcd = blockIdx.x % kXcds;
  const int share = count / kXcds + (xcd < count % kXcds);
  const int share0 = xcd * (count / kXcds) + min(xcd, count % kXcds);
  const int workers = (static_cast<int>(gridDim.x) - xcd + kXcds - 1) / kXcds;
  const int row_bytes = k / 2, k_steps = (row_bytes + ROWB - 1) / ROWB;

  // Tile `index` of the share: bands of row tiles, the rows of a band first.
  struct At {
    int expert, m0, n0, live;
  };
  auto locate = [&](int index) __attribute__((always_inline)) {
    const int pid = share0 + index;
    const int per_band = band * columns, first_tile = pid / per_band * band;
    const int in_band = min(row_tiles.total - first_tile, band);
    int expert, row, end;
    row_tiles.find(__builtin_amdgcn_readfirstlane(first_tile + pid % per_band % in_band), expert, row, end);
    return At{__builtin_amdgcn_readfirstlane(expert), __builtin_amdgcn_readfirstlane(pid % per_band / in_band * BM),
              __builtin_amdgcn_readfirstlane(row), __builtin_amdgcn_readfirstlane(min(BN, end - row))};
  };

  // ---- the DMA stream: step `dma_step` of tile `dma_index` is loaded next
  const int drow = lane >> 3;
  const int chunk0 = (lane & 7) ^ (drow >> 1), chunk1 = chunk0 ^ 4;
  const int limit0 = row_bytes - 16 * chunk0, limit1 = row_bytes - 16 * chunk1;
  int va[Tile::DMA_A], vb[Tile::DMA_B];
#pragma unroll
  for (int i = 0; i < Tile::DMA_A; ++i)
    va[i] = (wave * (BM / 4) + 8 * i + drow) * row_bytes + 16 * ((i & 1) ? chunk1 : chunk0);
#pragma unroll
  for (int i = 0; i < Tile::DMA_B; ++i)
    vb[i] = (wave * (BN / 4) + 8 * i + drow) * row_bytes + 16 * ((i & 1) ? chunk1 : chunk0);
  const uint32_t lds_base =
      static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) uint8_t*)lds));
  const int scale_half = BM > 128 && !(wave & 1) ? wave >> 1 : 0;
  const int scale_rows = (wave & 1) ? rows : n;
  int dma_step = 0;
  struct Source {
    __amdgpu_buffer_rsrc_t a, b, scales;
    int scale_row0;
  };
  auto source = [&](const At& at) __attribute__((always_inline)) {
    const int64_t e = at.expert;
    return Source{buffer_rsrc(w + (e * n + at.m0) * row_bytes, min(BM, n - at.m0) * row_bytes),
                  buffer_rsrc(x + static_cast<int64_t>(at.n0) * row_bytes, at.live * row_bytes),
                  (wave & 1) ? buffer_rsrc(sx, k_steps * rows * 8)
                             : buffer_rsrc(sw + e * k_steps * n * 8, k_steps * n * 8),
                  scale_first_row(BM, wave, at.m0, at.n0)};
  };
  int index = blockIdx.x / kXcds;
  if (index >= share) return;
  // The DMAs run ahead of the products by STAGES steps, and tiles by as many as
  // those make; past the last tile they load it once more.
  At here = locate(index);
  Source from = source(here);
  int dma_index = index;
  auto dma = [&](auto i_c, uint32_t stage) __attribute__((always_inline)) {
    constexpr int i = decltype(i_c)::value;
    const int kb = dma_step * ROWB;
    if constexpr (i < Tile::DMA_A) {
      dma16(from.a, kb < ((i & 1) ? limit1 : limit0) ? va[i] : kOutOfRange, kb,
            lds_base + (wave * (BM / 4) + 8 * i) * ROWB, stage);
    } else if constexpr (i < Tile::DMA_A + Tile::DMA_B) {
      constexpr int j = i - Tile::DMA_A;
      dma16(from.b, kb < ((j & 1) ? limit1 : limit0) ? vb[j] : kOutOfRange, kb,
            lds_base + (BM + wave * (BN / 4) + 8 * j) * ROWB, stage);
    } else {
      const DmaOffsets at = scale_offsets(dma_step, k_steps, scale_rows, from.scale_row0, lane);
      dma16(from.scales, at.lane, __builtin_amdgcn_readfirstlane(at.scalar),
            lds_base + Tile::OPERANDS + ((wave & 1) ? Tile::SCALES_A : scale_half * 1024), stage);
    }
  };
  // After a step's DMAs: the next one, in the tile after at the end of a tile.
  auto dma_advance = [&]() __attribute__((always_inline)) {
    if (++dma_step == k_steps) {
      dma_step = 0;
      dma_index += workers;
      from = source(locate(min(dma_index, share - 1)));
    }
  };

  // ---- fragments, as in ring_accumulate
  const int wm = wave & 1, wn = wave >> 1;
  const int lrow = lane % Op::M, lgroup = lane / Op::M;
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
      set.a[f][c] = *reinterpret_cast<const i32x4*>(lds + stage + (la ^ (c * Tile::GROUPS << 4)) + f * Op::M * ROWB);
    else
      set.b[f - FM][c] =
          *reinterpret_cast<const i32x4*>(lds + stage + (lb ^ (c * Tile::GROUPS << 4)) + (f - FM) * Op::M * ROWB);
  };
  const uint32_t pick = 0x06040200u + 0x01010101u * static_cast<uint32_t>(lgroup);
  uint32_t tail_mask = 0;
#pragma unroll
  for (int p = 0; p < 4; ++p)
    if (((k_steps - 1) * 8 + 2 * p + lgroup) * 32 < k) tail_mask |= 0xffu << (8 * p);
  auto read_scales = [&](Set& set, int kt, uint32_t stage) __attribute__((always_inline)) {
    const uint32_t mask = kt == k_steps - 1 ? tail_mask : 0xffffffffu;
    auto scale = [&](int row) __attribute__((always_inline)) {
      const i32x2 v = *reinterpret_cast<const i32x2*>(lds + stage + Tile::OPERANDS + row * 8);
      return __builtin_amdgcn_perm(static_cast<uint32_t>(v[1]), static_cast<uint32_t>(v[0]), pick) & mask;
    };
#pragma unroll
    for (int f = 0; f < FM; ++f) set.sa[f] = scale(wm * Tile::WM + f * Op::M + lrow);
#pragma unroll
    for (int f = 0; f < FN; ++f) set.sb[f] = scale(Tile::SCALES_A / 8 + wn * Tile::WN + f * Op::M + lrow);
  };
  typename Op::Acc acc[FM][FN];
  auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = typename Op::Acc{};
  };

  // ---- the output tile: 16 bytes a lane and store, eight (fp32: four) features
  constexpr int PIECE = 16 / sizeof(T);
  auto store = [&](const At& at) __attribute__((always_inline)) {
    constexpr int ES = sizeof(T);
    const int width = n - at.m0;  // features of the tile inside n, at least
    const __amdgpu_buffer_rsrc_t rc = __builtin_amdgcn_make_buffer_rsrc(
        y + static_cast<int64_t>(at.n0) * n + at.m0, (short)0, ((at.live - 1) * n + min(BM, width)) * ES, kBufferWord3);
    // put(row of Y in elements, feature, its piece) for every piece of the lane.
    auto pieces = [&](auto&& put) __attribute__((always_inline)) {
      auto f = [&](int row, int feature, i32x4 value) __attribute__((always_inline)) {
        asm volatile("" : "+v"(feature));  // one piece's masks at a time: all of them exceed the SGPRs
        put(row, feature, value);
      };
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int row = (wn * Tile::WN + j * 32 + (lane & 31)) * n;
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          const int column = wm * Tile::WM + i * 32;
          if constexpr (ES == 4) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const f32x4 v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
              f(row, column + Op::out_row(lane, 4 * q), __builtin_bit_cast(i32x4, v));
            }
          } else {
            // Lanes 0-31 hold features 8q .. 8q + 3 of their row, lanes 32-63 the next four of the same rows.
#pragma unroll
            for (int q = 0; q < 4; q += 2) {
              uint32_t word[2][2];
#pragma unroll
              for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const T pair[2] = {static_cast<T>(acc[i][j][4 * (q + p) + 2 * h]),
                                     static_cast<T>(acc[i][j][4 * (q + p) + 2 * h + 1])};
                  __builtin_memcpy(&word[p][h], pair, 4);
                }
              const auto low = __builtin_amdgcn_permlane32_swap(word[0][0], word[1][0], false, false);
              const auto high = __builtin_amdgcn_permlane32_swap(word[0][1], word[1][1], false, false);
              f(row, column + 8 * (q + (lane >> 5)),
                i32x4{static_cast<int>(low[0]), static_cast<int>(high[0]), static_cast<int>(low[1]),
                      static_cast<int>(high[1])});
            }
          }
        }
      }
    };
    // Rows past `live` lie past the buffer. Every wave issues the same STORES,
    // which vmcnt counts; those of an edge below only make it wait for more.
    pieces([&](int row, int feature, i32x4 value) __attribute__((always_inline)) {
      const int offset = feature + PIECE <= width ? (row + feature) * ES : kOutOfRange;
      __builtin_amdgcn_raw_buffer_store_b128(value, rc, offset, 0, 0);
    });
    if (width < BM && n % PIECE)  // the pieces that n ends in
      pieces([&](int row, int feature, i32x4 value) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < PIECE - 1; ++c) {
          const bool inside = feature + PIECE > width && feature + c < width;
          const int offset = inside ? (row + feature + c) * ES : kOutOfRange;
          const int word = value[c * ES / 4];
          if constexpr (ES == 4)
            __builtin_amdgcn_raw_buffer_store_b32(word, rc, offset, 0, 0);
          else
            __builtin_amdgcn_raw_buffer_store_b16(static_cast<short>(c % 2 ? word >> 16 : word), rc, offset, 0, 0);
        }
      });
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
      constexpr int p = q / (FM * FN), i = q % (FM * FN) / FN, j = q % FN;
      acc[i][j] = Op::template mma_byte<p>(set.a[i][p], set.b[j][p], acc[i][j], set.sa[i], set.sb[j]);
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
  while (true) {
    clear();
    int kt = 0;
    do {
      step(kt, set0, set1);
      if (kt + 1 < k_steps)
        step(kt + 1, set1, set0);
      else
        set0 = set1;  // the next tile's first fragments
      kt += 2;
    } while (kt < k_steps);
    store(here);
    with_stores = STAGES - 1;
    index += workers;
    if (index >= share) break;
    here = locate(index);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));  // no DMA of a step past the last may land in a later workgroup's LDS
#endif
}

}  // namespace mb
