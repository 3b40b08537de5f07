// Products of FP8 operands with block scales: linear layers, their gradients and the
// gated pair of projections, of one weight or one for each expert.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "mb_fp8.h"
#include "mb_fp8_tiles.h"

namespace mb {
namespace {

// ---- the kernels of products -----------------------------------------------------

// Microseconds of a quantisation's launch before a product's (with what an operand in
// memory costs the product over one in LDS), and of 4096 elements that a workgroup of
// eight waves quantises in the product's own, alone on a CU or for every workgroup that
// the CU has. Inside and before, in graphs: 14336 x 4096, 1, 4 and 8 rows 13.8 and 16.9,
// 16.4 and 18.4, 20.5 and 18.7; the gated pair of it 26.1 and 27.0, 27.4 and 27.5, 33.4
// and 27.8; 1024 x 4096, 1, 4 and 8 rows 5.4 and 6.7, 7.2 and 7.2, 9.5 and 7.5.
constexpr double kQuantizeLaunch = 2.5, kStagingAlone = 0.22, kStaging = 0.3;

constexpr int kE4m3 = 3;  // after MB_DTYPE_*: X an operand, or Y one

template <class T>
constexpr int type_code() {
  return sizeof(T) == 1 ? kE4m3 : sizeof(T) == 4 ? MB_DTYPE_F32 : __is_same(T, __bf16) ? MB_DTYPE_BF16 : MB_DTYPE_F16;
}

// What a launch takes, in microseconds. Of tiles: `launch` once; for every round of the
// chip's workgroups `tile`, `ragged` more where the rows of Y are not on 16 bytes, and for
// every 128 elements of K from `step_empty` to `step` with the filled share of the round
// (the L2s and the power limit slow a step down as more CUs run), and kMegabyte for every
// 10^6 bytes of weights at least. Of few rows: `launch`, and the root of the squares of
// `tile` and, for every 256 elements of K that a wave takes, `step` a round, and of
// `megabyte` for every 10^6 bytes of weights (either alone where the other is small).
constexpr double kMegabyte = 0.25;
struct ProductCost {
  float launch, tile, ragged, step_empty, step, megabyte;
};

// A kernel for X of `x` and Y of `y` by `epilogue` (Fp8TileEpilogue): of few rows, or of
// tiles of `features` columns of W by `rows` rows.
struct ProductKernel {
  const char* name;
  int x, y, epilogue;
  bool tiles;
  int features, rows;  // of a workgroup: columns of the output, rows
  int resident;        // workgroups a CU holds
  int band;            // row tiles that share their weight's panels in an XCD's L2
  int split;           // waves that share a tile's K
  ProductCost cost;
  void (*launch)(const Fp8Product&, uint32_t grid, int band, hipStream_t);
};

// Workgroups of a kernel of few rows: columns, experts (rows, if there are fewer) and
// chunks of an expert's rows.
dim3 few_grid(uint32_t n, uint32_t columns, uint32_t rows, uint32_t chunk, uint32_t experts, bool routed) {
  const uint32_t chunks = (rows / (routed ? experts : 1) + chunk - 1) / chunk;
  return dim3((n + columns - 1) / columns, routed ? (rows < experts ? rows : experts) : 1,
              chunks < 1 ? 1 : chunks < 256 ? chunks : 256);
}

template <class X, class Y, int EPILOGUE, int FB, int SPLIT>
void launch_few(const Fp8Product& p, uint32_t, int, hipStream_t stream) {
  constexpr uint32_t kColumns = fp8_few_waves(SPLIT) / SPLIT * FB * 16 / (EPILOGUE == kFp8Plain ? 1 : 2);
  constexpr uint32_t kRows = kFp8FewRows;
  const uint32_t rows = static_cast<uint32_t>(p.rows), lds_rows = rows < kRows ? rows : kRows;
  const uint64_t lds =
      std::max(sizeof(X) > 1 ? fp8_few_lds(static_cast<uint32_t>(p.k), lds_rows) : 0, fp8_few_parts(fp8_few_waves(SPLIT), FB * 16));
  fp8_few_kernel<X, Y, EPILOGUE, FB, SPLIT>
      <<<few_grid(static_cast<uint32_t>(p.n), kColumns, rows, kRows, static_cast<uint32_t>(p.experts), p.offsets),
         dim3(64 * fp8_few_waves(SPLIT)), static_cast<uint32_t>(lds), stream>>>(p, static_cast<int>(lds_rows));
}

template <class Y, int EPILOGUE, int BM, int BN, int STAGES>
void launch_tiles(const Fp8Product& p, uint32_t grid, int band, hipStream_t stream) {
  constexpr uint32_t kPlaces = 256 * Fp8Tile<EPILOGUE, BM, BN, STAGES>::RESIDENT;
  fp8_tiles_kernel<Y, EPILOGUE, BM, BN, STAGES>
      <<<dim3(grid < kPlaces ? grid : kPlaces), dim3(256), 0, stream>>>(p, band);
}

#define MB_FP8_FEW(X, X_NAME, Y, Y_NAME, EPILOGUE, NAME, FB, SPLIT, ...)                                       \
  ProductKernel {                                                                                              \
    "fp8_few_" NAME "_" X_NAME "_" Y_NAME "_" #FB "x" #SPLIT, type_code<X>(), type_code<Y>(), EPILOGUE, false, \
        fp8_few_waves(SPLIT) / SPLIT * FB * 16 / (EPILOGUE == kFp8Plain ? 1 : 2), kFp8FewRows, fp8_few_resident(FB, SPLIT), 0, SPLIT, \
        {__VA_ARGS__}, launch_few<X, Y, EPILOGUE, FB, SPLIT>                                                   \
  }
#define MB_FP8_TILES(Y, Y_NAME, EPILOGUE, NAME, BM, BN, STAGES, BAND, ...)                                     \
  ProductKernel {                                                                                              \
    "fp8_tiles_" NAME "_" Y_NAME "_" #BM "x" #BN, kE4m3, type_code<Y>(), EPILOGUE, true,                       \
        EPILOGUE == kTilePlain ? BM : BM / 2, BN, Fp8Tile<EPILOGUE, BM, BN, STAGES>::RESIDENT, BAND, 1,        \
        {__VA_ARGS__}, launch_tiles<Y, EPILOGUE, BM, BN, STAGES>                                               \
  }
// The forms, for a list M(arguments) of kernels and for their registration alike. Costs
// are fitted to sizes timed on an MI355X, two of five off the tiles: of tiles to 8700 (1
// to 16384 rows, n and K from 64 to 8192, one weight or 8 to 128 experts of uneven
// popularity), where the cheapest estimate costs 1.3% over the fastest on average for
// products and 0.3% for gated ones; of few rows to 17800 in graphs (up to 40 rows of one
// weight and six an expert), where it costs 1.4% over the fastest of all and 4% at the
// ninth decile; the worst are up to twice the time, 30 us, where K is 128 or 256.
#define MB_FP8_FEW_16(M, X, X_NAME, Y, Y_NAME)                                           \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 1, 8, 1.89f, 0.33f, 0, 0, 1.18f, 0.243f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 1, 4, 2.04f, 0.61f, 0, 0, 0.64f, 0.220f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 2, 4, 1.80f, 0.69f, 0, 0, 1.07f, 0.211f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Gated, "gated", 2, 8, 2.13f, 0, 0, 0, 1.60f, 0.230f)       \
  M(X, X_NAME, Y, Y_NAME, kFp8Gated, "gated", 2, 4, 1.82f, 0.81f, 0, 0, 1.04f, 0.207f)
#define MB_FP8_TILES_16(M, Y, Y_NAME)                                                                 \
  M(Y, Y_NAME, kTilePlain, "product", 256, 256, 2, 4, 4.56f, 3.81f, 4.15f, 0.958f, 1.700f, 0)         \
  M(Y, Y_NAME, kTilePlain, "product", 256, 128, 3, 4, 3.83f, 2.87f, 2.05f, 0.620f, 1.095f, 0)         \
  M(Y, Y_NAME, kTilePlain, "product", 128, 128, 4, 6, 4.51f, 1.71f, 0.69f, 0.391f, 0.594f, 0)         \
  M(Y, Y_NAME, kTilePlain, "product", 128, 64, 3, 8, 4.48f, 1.72f, 0.10f, 0.214f, 0.740f, 0)          \
  M(Y, Y_NAME, kTilePlain, "product", 64, 64, 3, 8, 5.16f, 1.14f, 0.05f, 0.134f, 0.417f, 0)           \
  M(Y, Y_NAME, kTileGated, "gated", 256, 256, 2, 4, 4.90f, 6.88f, 1.70f, 1.005f, 1.755f, 0)           \
  M(Y, Y_NAME, kTileGated, "gated", 256, 128, 3, 4, 4.55f, 3.70f, 0.77f, 0.613f, 1.043f, 0)           \
  M(Y, Y_NAME, kTileGated, "gated", 256, 64, 3, 8, 4.50f, 2.24f, 0.27f, 0.427f, 0.746f, 0)            \
  M(Y, Y_NAME, kTileGatedKept, "gated_kept", 256, 256, 2, 4, 3.99f, 10.97f, 5.85f, 0.989f, 1.719f, 0) \
  M(Y, Y_NAME, kTileGatedKept, "gated_kept", 256, 128, 3, 4, 3.75f, 6.17f, 2.81f, 0.614f, 1.010f, 0)  \
  M(Y, Y_NAME, kTileGatedKept, "gated_kept", 256, 64, 3, 8, 3.70f, 3.74f, 1.41f, 0.429f, 0.712f, 0)
#define MB_FP8_FEW_32(M, X, X_NAME, Y, Y_NAME)                                           \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 1, 8, 1.91f, 0.41f, 0, 0, 1.21f, 0.243f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 1, 4, 2.01f, 0.48f, 0, 0, 0.94f, 0.223f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Plain, "product", 2, 4, 1.80f, 0.47f, 0, 0, 1.46f, 0.220f) \
  M(X, X_NAME, Y, Y_NAME, kFp8Gated, "gated", 2, 8, 2.22f, 0, 0, 0, 1.73f, 0.239f)       \
  M(X, X_NAME, Y, Y_NAME, kFp8Gated, "gated", 2, 4, 1.94f, 0.45f, 0, 0, 1.46f, 0.209f)
#define MB_FP8_TILES_32(M, Y, Y_NAME)                                                         \
  M(Y, Y_NAME, kTilePlain, "product", 256, 128, 3, 4, 1.98f, 5.02f, 0.85f, 1.290f, 1.771f, 0) \
  M(Y, Y_NAME, kTilePlain, "product", 128, 128, 4, 6, 3.53f, 2.70f, 0.06f, 0.720f, 0.946f, 0) \
  M(Y, Y_NAME, kTilePlain, "product", 128, 64, 3, 8, 3.25f, 2.81f, 0, 0.423f, 1.040f, 0)      \
  M(Y, Y_NAME, kTilePlain, "product", 64, 64, 3, 8, 4.76f, 1.41f, 0, 0.256f, 0.622f, 0)       \
  M(Y, Y_NAME, kTileGated, "gated", 256, 64, 3, 8, 3.98f, 2.87f, 0.04f, 0.820f, 1.108f, 0)    \
  M(Y, Y_NAME, kTileGatedKept, "gated_kept", 256, 64, 3, 8, 2.83f, 4.91f, 0.71f, 0.825f, 1.105f, 0)
#define MB_FP8_FEW_ALL(M)                                                                                 \
  MB_FP8_FEW_32(M, uint8_t, "e4m3", float, "f32")                                                         \
  MB_FP8_FEW_16(M, uint8_t, "e4m3", _Float16, "f16")                                                      \
  MB_FP8_FEW_16(M, uint8_t, "e4m3", __bf16, "bf16")                                                       \
  MB_FP8_FEW_32(M, float, "f32", float, "f32")                                                            \
  MB_FP8_FEW_16(M, _Float16, "f16", _Float16, "f16")                                                      \
  MB_FP8_FEW_16(M, __bf16, "bf16", __bf16, "bf16")                                                        \
  M(uint8_t, "e4m3", uint8_t, "e4m3", kFp8GatedFp8, "gated_fp8", 2, 1, 0.74f, 3.04f, 0, 0, 1.99f, 0.217f) \
  M(float, "f32", uint8_t, "e4m3", kFp8GatedFp8, "gated_fp8", 2, 1, 0.74f, 3.04f, 0, 0, 1.99f, 0.217f)    \
  M(_Float16, "f16", uint8_t, "e4m3", kFp8GatedFp8, "gated_fp8", 2, 1, 0.74f, 3.04f, 0, 0, 1.99f, 0.217f) \
  M(__bf16, "bf16", uint8_t, "e4m3", kFp8GatedFp8, "gated_fp8", 2, 1, 0.74f, 3.04f, 0, 0, 1.99f, 0.217f)
#define MB_FP8_TILES_ALL(M)                                                                          \
  MB_FP8_TILES_32(M, float, "f32")                                                                   \
  MB_FP8_TILES_16(M, _Float16, "f16")                                                                \
  MB_FP8_TILES_16(M, __bf16, "bf16")                                                                 \
  M(uint8_t, "e4m3", kTileGatedFp8, "gated_fp8", 256, 256, 2, 4, 4.51f, 7.60f, 0, 1.018f, 1.830f, 0) \
  M(uint8_t, "e4m3", kTileGatedFp8, "gated_fp8", 256, 128, 3, 4, 4.38f, 4.14f, 0, 0.631f, 1.061f, 0) \
  M(uint8_t, "e4m3", kTileGatedFp8, "gated_fp8", 256, 64, 3, 8, 4.20f, 2.60f, 0, 0.452f, 0.729f, 0)

#define MB_FP8_FEW_ENTRY(...) MB_FP8_FEW(__VA_ARGS__),
#define MB_FP8_TILES_ENTRY(...) MB_FP8_TILES(__VA_ARGS__),
const ProductKernel kKernels[] = {MB_FP8_FEW_ALL(MB_FP8_FEW_ENTRY) MB_FP8_TILES_ALL(MB_FP8_TILES_ENTRY)};

#define MB_FP8_FEW_REGISTER(X, X_NAME, Y, Y_NAME, EPILOGUE, NAME, FB, SPLIT, ...)          \
  MB_REGISTER_KERNEL("fp8_few_" NAME "_" X_NAME "_" Y_NAME "_" #FB "x" #SPLIT,             \
                     (fp8_few_kernel<X, Y, EPILOGUE, FB, SPLIT>));
#define MB_FP8_TILES_REGISTER(Y, Y_NAME, EPILOGUE, NAME, BM, BN, STAGES, BAND, ...)        \
  MB_REGISTER_KERNEL("fp8_tiles_" NAME "_" Y_NAME "_" #BM "x" #BN, (fp8_tiles_kernel<Y, EPILOGUE, BM, BN, STAGES>));
MB_FP8_FEW_ALL(MB_FP8_FEW_REGISTER)
MB_FP8_TILES_ALL(MB_FP8_TILES_REGISTER)

constexpr uint32_t kMostExperts = 4096;

int check_shape(const char* entry, int dtype, uint64_t rows, uint64_t n, uint64_t k, uint32_t experts) {
  if (!elem_bytes(dtype)) return fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (experts == 0 || experts > kMostExperts)
    return fail(MB_ERR_INVALID, "%s: %u experts outside 1..%u", entry, experts, kMostExperts);
  if (rows > kFp8MostRows || n > kFp8MostK || k > kFp8MostK)
    return fail(MB_ERR_UNSUPPORTED, "%s: %llu x %llu x %llu: at most %u rows, %u columns and %u elements of K", entry,
                (unsigned long long)rows, (unsigned long long)n, (unsigned long long)k, kFp8MostRows, kFp8MostK,
                kFp8MostK);
  return MB_OK;
}

int check_offsets(const char* entry, const int32_t* offsets, uint64_t offsets_bytes, uint32_t experts) {
  if (offsets == nullptr)
    return experts == 1 ? MB_OK : fail(MB_ERR_INVALID, "%s: several experts need offsets", entry);
  if (offsets_bytes < (uint64_t{experts} + 1) * 4)
    return fail(MB_ERR_INVALID, "%s: offsets must hold %u entries", entry, experts + 1);
  if (!aligned(offsets, 4)) return fail(MB_ERR_ALIGNMENT, "%s: offsets must lie on 4 bytes", entry);
  return MB_OK;
}

// X's rows as a routed product gathers them.
int check_routes(const char* entry, const int32_t* offsets, const int32_t* order, const int32_t* slots,
                 uint64_t slots_bytes, uint64_t rows) {
  if (slots && (offsets == nullptr || order == nullptr || slots_bytes < rows * 4))
    return fail(MB_ERR_INVALID, "%s: slots need offsets, order and, in both, an entry for each of %llu rows", entry,
                (unsigned long long)rows);
  if (!aligned(slots, 4) || !aligned(order, 4))
    return fail(MB_ERR_ALIGNMENT, "%s: order and slots must lie on 4 bytes", entry);
  return MB_OK;
}

int shift_of(uint32_t block) { return block == 1 ? 0 : 7; }

// Row tiles of `tile` rows, at most: an expert's rows start one of their own.
uint64_t most_row_tiles(uint32_t rows, uint32_t experts, int tile) {
  return experts > 1 ? rows / tile + (rows < experts ? rows : experts) : (rows + uint64_t{1} * tile - 1) / tile;
}

// Experts with rows, if all were as popular.
double used_experts(uint32_t rows, uint32_t experts) {
  return experts == 1 ? 1.0 : experts * (1.0 - std::exp(-static_cast<double>(rows) / experts));
}

double mean_row_tiles(uint32_t rows, uint32_t experts, int tile) {
  if (experts == 1) return static_cast<double>(most_row_tiles(rows, 1, tile));
  const double each = static_cast<double>(rows) / experts;
  return experts * (each >= tile ? each / tile + 0.5 : each >= 1 ? 1.0 : each);
}

// Estimated microseconds of a launch (see ProductCost).
double product_cost(const ProductKernel& kernel, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts) {
  const ProductCost& cost = kernel.cost;
  const double across = (n + uint64_t{1} * kernel.features - 1) / kernel.features;
  const double used = used_experts(rows, experts);
  const double megabytes = used * (kernel.epilogue == kTilePlain ? 1 : 2) * n * k * 1e-6;  // of weights
  if (!kernel.tiles) {
    const double each = rows / used;
    const double chunks = experts == 1 ? (rows + kFp8FewRows - 1) / kFp8FewRows : std::max(1.0, each / kFp8FewRows);
    const double rounds = std::max(1.0, across * used * chunks / (256.0 * kernel.resident));
    const double turns = ((k + 255) / 256 + kernel.split - 1) / kernel.split;
    // Every workgroup quantises its rows.
    const double each_cu = across * used * chunks / 256.0, waves = fp8_few_waves(kernel.split);
    const double staging = kernel.x == kE4m3 ? 0
                                             : std::min(each, 1.0 * kFp8FewRows) * k / 4096 *
                                                   std::max(kStagingAlone * 8 / waves, kStaging * each_cu);
    return cost.launch + staging +
           std::hypot(rounds * (cost.tile + turns * cost.step), megabytes * chunks * cost.megabyte);
  }
  const double tiles = mean_row_tiles(rows, experts, kernel.rows) * across;
  const double round = 256.0 * kernel.resident, whole = static_cast<double>(static_cast<uint64_t>(tiles / round));
  const double rest = tiles / round - whole, steps = (k + 127) / 128;
  const bool ragged = kernel.y != kE4m3 && uint64_t{n} * elem_bytes(kernel.y) % 16 != 0;
  auto one = [&](double filled) {
    return cost.tile + (ragged ? cost.ragged : 0.0f) +
           steps * (cost.step_empty + (cost.step - cost.step_empty) * filled);
  };
  const double all = cost.launch + whole * one(1.0) + (rest > 0 ? one(rest) : 0.0);
  return std::max(all, 1.0 + megabytes * kMegabyte) + 0.01 * all;  // of two that memory bounds the quicker
}

struct ProductChoice {
  const ProductKernel* kernel = nullptr;
  uint32_t grid = 0;  // of tiles
  double cost = 0;
};

// The kernel for X of type `x` by the rule or, with `wanted`, the one of that name; none
// if it does not take the sizes.
ProductChoice choose_product(int x, int y, int epilogue, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts,
                             const char* wanted) {
  ProductChoice best;
  const uint64_t width = epilogue == kTilePlain ? n : uint64_t{2} * n, steps = (k + uint64_t{511}) / 512;
  for (const ProductKernel& kernel : kKernels) {
    // A kernel of few rows keeps the gate and up, if it is given where to.
    const int asked = epilogue == kTileGatedKept && !kernel.tiles ? static_cast<int>(kTileGated) : epilogue;
    if (kernel.x != x || kernel.y != y || kernel.epilogue != asked) continue;
    if (wanted && strcmp(wanted, kernel.name) != 0) continue;
    uint64_t grid = 0;
    if (kernel.tiles) {
      if (experts > kStreamExperts) continue;
      // The tiles address a matrix's scales, and a tile's rows, with 32-bit offsets.
      if (steps * (rows > width ? rows : width) * 4 > 0x7fffffffu) continue;
      if (fp8_pitch(k) * 256 > 0x7fffffffu || uint64_t{1} * kernel.rows * width * 4 > 0x7fffffffu) continue;
      const uint64_t tiles =
          most_row_tiles(rows, experts, kernel.rows) * ((n + uint64_t{1} * kernel.features - 1) / kernel.features);
      grid = (tiles + kXcds - 1) / kXcds * kXcds;
      if (grid > 0xffffff) continue;
    } else {
      // A row's codes fit the LDS, and the workgroups of 512 a launch's 2^32 - 1.
      if (x != kE4m3 && fp8_few_lds(k, rows < kFp8FewRows ? rows : kFp8FewRows) > 96 * 1024) continue;
      const dim3 few = few_grid(n, static_cast<uint32_t>(kernel.features), rows, kFp8FewRows, experts, experts > 1);
      if (uint64_t{few.x} * few.y * few.z > 0x7fffff) continue;
    }
    const double cost = product_cost(kernel, rows, n, k, experts);
    if (best.kernel && cost >= best.cost) continue;
    best = ProductChoice{&kernel, static_cast<uint32_t>(grid), cost};
  }
  return best;
}

// Whether X, of `dtype`, is quantised in the product's launch, and the choice for either.
bool choose_linear(int dtype, int y, int epilogue, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts,
                   ProductChoice& choice) {
  const ProductChoice inside = choose_product(dtype, y, epilogue, rows, n, k, experts, nullptr);
  choice = choose_product(kE4m3, y, epilogue, rows, n, k, experts, nullptr);
  if (inside.kernel == nullptr || (choice.kernel && inside.cost > choice.cost + kQuantizeLaunch)) return false;
  choice = inside;
  return true;
}

int kind_of(Fp8Epilogue epilogue, const Fp8Product& p) {
  return epilogue == kFp8Gated && p.gate_up ? static_cast<int>(kTileGatedKept) : static_cast<int>(epilogue);
}

int launch_choice(const char* entry, const ProductChoice& choice, const char* wanted, const Fp8Product& p,
                  hipStream_t stream) {
  if (choice.kernel == nullptr)
    return fail(MB_ERR_UNSUPPORTED, "%s: no kernel %s that takes %d x %d x %d and %d experts", entry,
                wanted ? wanted : "", p.rows, p.n, p.k, p.experts);
  choice.kernel->launch(p, choice.grid, choice.kernel->band, stream);
  return launch_status(choice.kernel->name);
}

// X an operand.
int launch_product(const char* entry, const char* wanted, int dtype, Fp8Epilogue epilogue, const Fp8Product& p,
                   hipStream_t stream) {
  const ProductChoice choice = choose_product(
      kE4m3, epilogue == kFp8GatedFp8 ? kE4m3 : dtype, kind_of(epilogue, p), static_cast<uint32_t>(p.rows),
      static_cast<uint32_t>(p.n), static_cast<uint32_t>(p.k), static_cast<uint32_t>(p.experts), wanted);
  return launch_choice(entry, choice, wanted, p, stream);
}

uint64_t workspace_codes(uint64_t rows, uint64_t k) { return (fp8_code_bytes(rows, k) + 15) / 16 * 16; }
uint64_t workspace_bytes_of(uint64_t rows, uint64_t k) { return workspace_codes(rows, k) + fp8_scale_bytes(rows, k, 1); }

// Quantises X (rows of tokens, to their slots, or rows in order) and multiplies. p holds
// all but X's operand.
int run_linear(const char* entry, int dtype, Fp8Epilogue epilogue, Fp8Product p, const int32_t* slots, void* workspace,
               uint64_t workspace_bytes, hipStream_t stream) {
  const uint32_t rows = static_cast<uint32_t>(p.rows), k = static_cast<uint32_t>(p.k);
  const uint64_t needed = workspace_bytes_of(rows, k);
  if (workspace == nullptr || workspace_bytes < needed)
    return fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                (unsigned long long)needed);
  if (!aligned(workspace, 16)) return fail(MB_ERR_ALIGNMENT, "%s: the workspace must lie on 16 bytes", entry);
  ProductChoice choice;
  if (choose_linear(dtype, epilogue == kFp8GatedFp8 ? kE4m3 : dtype, kind_of(epilogue, p), rows,
                    static_cast<uint32_t>(p.n), k, static_cast<uint32_t>(p.experts), choice))
    return launch_choice(entry, choice, nullptr, p, stream);
  uint8_t* codes = static_cast<uint8_t*>(workspace);
  uint8_t* scales = codes + workspace_codes(rows, k);
  if (int rc = fp8_launch_quantize(dtype, p.x, static_cast<uint32_t>(p.tokens), k, p.row_stride, slots,
                                   static_cast<uint32_t>(p.copies), rows, codes, scales, stream))
    return rc;
  p.x = codes;
  p.sx = scales;
  p.x_shift = 0;
  return launch_choice(entry, choice, nullptr, p, stream);
}

// The outputs of a gated product.
int check_gated_outputs(const char* entry, int dtype, void* y, uint64_t y_bytes, void* y_scales, uint64_t y_scales_bytes,
                        void* gate_up, uint64_t gate_up_bytes, uint64_t rows, uint64_t n) {
  if (y_scales) {
    if (int rc = fp8_check_operand(entry, "the output", rows, n, 1, 1, y, y_bytes, y_scales, y_scales_bytes)) return rc;
    if (gate_up)
      return fail(MB_ERR_UNSUPPORTED, "%s: gate and up are kept beside an output of the tensors' type, not FP8", entry);
    return MB_OK;
  }
  if (int rc = fp8_check_output(entry, "the output", dtype, y, y_bytes, rows, n)) return rc;
  return gate_up ? fp8_check_output(entry, "gate_up", dtype, gate_up, gate_up_bytes, rows, 2 * n) : MB_OK;
}

// Operands of a product's gradients in its workspace: d's rows [rows][n], and the
// columns of d [n][depth] and of x [k][depth].
struct GradientSpace {
  uint64_t codes[3], scales[3], end;
};

// K of d_w's operands: whole blocks past the first, so that their rows lie on lines.
uint32_t gradient_depth(uint32_t rows) { return rows > 128 ? (rows + 127) / 128 * 128 : (rows + 15) / 16 * 16; }

GradientSpace gradient_space(uint32_t rows, uint32_t n, uint32_t k) {
  const uint32_t depth = gradient_depth(rows);
  const uint64_t sizes[3][2] = {{rows, n}, {n, depth}, {k, depth}};
  GradientSpace space{};
  for (int i = 0; i < 3; ++i) {
    space.codes[i] = space.end;
    space.scales[i] = space.codes[i] + (fp8_code_bytes(sizes[i][0], sizes[i][1]) + 15) / 16 * 16;
    space.end = space.scales[i] + (fp8_scale_bytes(sizes[i][0], sizes[i][1], 1) + 15) / 16 * 16;
  }
  return space;
}

// d_x [rows][k] and d_w [n][k] of a product of x [rows][k] with W [n][k] for the
// gradient d [rows][n], or, with gate_up, d_out [rows][n / 2] of the gated product.
int run_backward(const char* entry, int dtype, const void* d_out, uint64_t d_out_bytes, uint64_t d_stride,
                 const void* gate_up, uint64_t gate_up_bytes, bool gated, const void* x, uint64_t x_bytes,
                 uint64_t x_stride, const void* w, uint64_t w_bytes, const void* sw, uint64_t sw_bytes,
                 uint32_t w_block, void* d_x, uint64_t d_x_bytes, void* d_w, uint64_t d_w_bytes, uint32_t rows,
                 uint32_t n, uint32_t k, void* workspace, uint64_t workspace_bytes, hipStream_t stream) {
  if (int rc = check_shape(entry, dtype, rows, n, k, 1)) return rc;
  if (rows == 0 || n == 0 || k == 0) return fail(MB_ERR_INVALID, "%s: rows, n and K must be positive", entry);
  if (rows > kFp8MostK)
    return fail(MB_ERR_UNSUPPORTED, "%s: at most %u rows, which d_w sums over", entry, kFp8MostK);
  if (int rc = fp8_check_rows(entry, "d_out", dtype, d_out, d_out_bytes, rows, gated ? n / 2 : n, d_stride)) return rc;
  if (gated)
    if (int rc = fp8_check_output(entry, "gate_up", dtype, gate_up, gate_up_bytes, rows, n)) return rc;
  if (int rc = fp8_check_rows(entry, "x", dtype, x, x_bytes, rows, k, x_stride)) return rc;
  if (int rc = fp8_check_operand(entry, "the weight's columns'", k, n, 1, w_block, w, w_bytes, sw, sw_bytes)) return rc;
  if (int rc = fp8_check_output(entry, "d_x", dtype, d_x, d_x_bytes, rows, k)) return rc;
  if (int rc = fp8_check_output(entry, "d_w", dtype, d_w, d_w_bytes, n, k)) return rc;
  const GradientSpace at = gradient_space(rows, n, k);
  uint8_t* const space = static_cast<uint8_t*>(workspace);
  if (space == nullptr || workspace_bytes < at.end)
    return fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                (unsigned long long)at.end);
  if (!aligned(space, 16)) return fail(MB_ERR_ALIGNMENT, "%s: the workspace must lie on 16 bytes", entry);
  const uint32_t depth = gradient_depth(rows);
  Fp8Out out[3];
  for (int i = 0; i < 3; ++i) out[i] = Fp8Out{space + at.codes[i], space + at.scales[i]};
  if (int rc = fp8_launch_gradient(dtype, d_out, d_stride, gated ? gate_up : nullptr, x, x_stride, rows, n, k, depth,
                                   out[0], out[1], out[2], stream))
    return rc;
  Fp8Product p{};
  p.copies = p.experts = 1;
  p.x = out[0].codes;
  p.sx = out[0].scales;
  p.w = static_cast<const uint8_t*>(w);
  p.sw = static_cast<const uint8_t*>(sw);
  p.w_shift = shift_of(w_block);
  p.y = d_x;
  p.rows = p.tokens = static_cast<int>(rows);
  p.n = static_cast<int>(k);
  p.k = static_cast<int>(n);
  if (int rc = launch_product(entry, nullptr, dtype, kFp8Plain, p, stream)) return rc;
  p.x = out[1].codes;
  p.sx = out[1].scales;
  p.w = out[2].codes;
  p.sw = out[2].scales;
  p.w_shift = 0;
  p.y = d_w;
  p.rows = p.tokens = static_cast<int>(n);
  p.n = static_cast<int>(k);
  p.k = static_cast<int>(depth);
  return launch_product(entry, nullptr, dtype, kFp8Plain, p, stream);
}

}  // namespace
}  // namespace mb

extern "C" {

int mb_fp8_product(int dtype, const void* a, uint64_t a_bytes, const void* scale_a, uint64_t scale_a_bytes,
                   uint32_t a_block, const void* b, uint64_t b_bytes, const void* scale_b, uint64_t scale_b_bytes,
                   uint32_t b_block, void* c, uint64_t c_bytes, uint32_t rows, uint32_t n, uint32_t k,
                   const int32_t* offsets, uint64_t offsets_bytes, uint32_t experts, const char* kernel,
                   void* stream) {
  const char* entry = "mb_fp8_product";
  if (int rc = mb::check_shape(entry, dtype, rows, n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (offsets && a_block != 1)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: rows of several experts have a scale each", entry);
  if (int rc = mb::fp8_check_operand(entry, "a's", rows, k, 1, a_block, a, a_bytes, scale_a, scale_a_bytes)) return rc;
  if (int rc = mb::fp8_check_operand(entry, "b's", n, k, experts, b_block, b, b_bytes, scale_b, scale_b_bytes))
    return rc;
  if (int rc = mb::fp8_check_output(entry, "the output", dtype, c, c_bytes, rows, n)) return rc;
  mb::Fp8Product p{};
  p.x = a;
  p.sx = static_cast<const uint8_t*>(scale_a);
  p.x_shift = mb::shift_of(a_block);
  p.w = static_cast<const uint8_t*>(b);
  p.sw = static_cast<const uint8_t*>(scale_b);
  p.w_shift = mb::shift_of(b_block);
  p.y = c;
  p.rows = p.tokens = static_cast<int>(rows);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.offsets = offsets;
  p.copies = 1;
  p.experts = static_cast<int>(experts);
  return mb::launch_product(entry, kernel, dtype, mb::kFp8Plain, p, static_cast<hipStream_t>(stream));
}

const char* mb_fp8_product_kernel(int dtype, uint32_t rows, uint32_t n, uint32_t k, uint32_t experts, uint32_t linear,
                                  uint32_t gated) {
  const char* entry = "mb_fp8_product_kernel";
  const bool fp8 = gated == MB_FP8_GATED_FP8;
  if (mb::check_shape(entry, dtype, rows, gated ? uint64_t{2} * n : n, k, experts)) return nullptr;
  if (rows == 0 || n == 0 || k == 0 || gated > MB_FP8_GATED_FP8) {
    mb::fail(MB_ERR_INVALID, "%s: no product of %u x %u x %u and kind %u", entry, rows, n, k, gated);
    return nullptr;
  }
  const int kinds[] = {mb::kTilePlain, mb::kTileGated, mb::kTileGatedKept, mb::kTileGatedFp8};
  const int y = fp8 ? mb::kE4m3 : dtype;
  mb::ProductChoice choice;
  if (linear)
    mb::choose_linear(dtype, y, kinds[gated], rows, n, k, experts, choice);
  else
    choice = mb::choose_product(mb::kE4m3, y, kinds[gated], rows, n, k, experts, nullptr);
  if (choice.kernel) return choice.kernel->name;
  mb::fail(MB_ERR_UNSUPPORTED, "%s: no kernel that takes %u x %u x %u and %u experts", entry, rows, n, k, experts);
  return nullptr;
}

uint64_t mb_fp8_linear_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  (void)n;
  return mb::workspace_bytes_of(rows, k);
}

int mb_fp8_linear(int dtype, const void* x, uint64_t x_bytes, uint32_t tokens, uint64_t row_stride, const void* w,
                  uint64_t w_bytes, const void* scale_w, uint64_t scale_w_bytes, uint32_t w_block, void* y,
                  uint64_t y_bytes, uint32_t n, uint32_t k, const int32_t* offsets, uint64_t offsets_bytes,
                  const int32_t* order, const int32_t* slots, uint64_t slots_bytes, uint32_t copies, uint32_t experts,
                  void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_fp8_linear";
  if (slots && (copies == 0 || copies > 64))
    return mb::fail(MB_ERR_INVALID, "%s: %u slots a token outside 1..64", entry, copies);
  const uint64_t rows = uint64_t{tokens} * (slots ? copies : 1);
  if (int rc = mb::check_shape(entry, dtype, rows, n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (int rc = mb::check_routes(entry, offsets, order, slots, slots_bytes, rows)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (int rc = mb::fp8_check_rows(entry, "x", dtype, x, x_bytes, tokens, k, row_stride)) return rc;
  if (int rc = mb::fp8_check_operand(entry, "the weight's", n, k, experts, w_block, w, w_bytes, scale_w, scale_w_bytes))
    return rc;
  if (int rc = mb::fp8_check_output(entry, "the output", dtype, y, y_bytes, rows, n)) return rc;
  mb::Fp8Product p{};
  p.x = x;
  p.row_stride = row_stride;
  p.w = static_cast<const uint8_t*>(w);
  p.sw = static_cast<const uint8_t*>(scale_w);
  p.w_shift = mb::shift_of(w_block);
  p.y = y;
  p.rows = static_cast<int>(rows);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.offsets = offsets;
  p.order = slots ? order : nullptr;
  p.copies = slots ? static_cast<int>(copies) : 1;
  p.tokens = static_cast<int>(tokens);
  p.experts = static_cast<int>(experts);
  return mb::run_linear(entry, dtype, mb::kFp8Plain, p, slots, workspace, workspace_bytes,
                        static_cast<hipStream_t>(stream));
}

uint64_t mb_fp8_linear_backward_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  return mb::gradient_space(rows < mb::kFp8MostRows ? rows : mb::kFp8MostRows, n, k).end;
}

int mb_fp8_linear_backward(int dtype, const void* d_out, uint64_t d_out_bytes, uint64_t d_out_stride, const void* x,
                           uint64_t x_bytes, uint64_t x_stride, const void* w_columns, uint64_t w_columns_bytes,
                           const void* scale_w, uint64_t scale_w_bytes, uint32_t w_block, void* d_x,
                           uint64_t d_x_bytes, void* d_w, uint64_t d_w_bytes, uint32_t rows, uint32_t n, uint32_t k,
                           void* workspace, uint64_t workspace_bytes, void* stream) {
  return mb::run_backward("mb_fp8_linear_backward", dtype, d_out, d_out_bytes, d_out_stride, nullptr, 0, false, x,
                          x_bytes, x_stride, w_columns, w_columns_bytes, scale_w, scale_w_bytes, w_block, d_x,
                          d_x_bytes, d_w, d_w_bytes, rows, n, k, workspace, workspace_bytes,
                          static_cast<hipStream_t>(stream));
}

int mb_fp8_gated_product(int dtype, const void* a, uint64_t a_bytes, const void* scale_a, uint64_t scale_a_bytes,
                         uint32_t a_block, const void* b, uint64_t b_bytes, const void* scale_b, uint64_t scale_b_bytes,
                         uint32_t b_block, void* y, uint64_t y_bytes, void* y_scales, uint64_t y_scales_bytes,
                         void* gate_up, uint64_t gate_up_bytes, uint32_t rows, uint32_t n, uint32_t k,
                         const int32_t* offsets, uint64_t offsets_bytes, uint32_t experts, const char* kernel,
                         void* stream) {
  const char* entry = "mb_fp8_gated_product";
  if (int rc = mb::check_shape(entry, dtype, rows, uint64_t{2} * n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (offsets && a_block != 1)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: rows of several experts have a scale each", entry);
  if (int rc = mb::fp8_check_operand(entry, "a's", rows, k, 1, a_block, a, a_bytes, scale_a, scale_a_bytes)) return rc;
  if (int rc = mb::fp8_check_operand(entry, "b's", uint64_t{2} * n, k, experts, b_block, b, b_bytes, scale_b,
                                     scale_b_bytes))
    return rc;
  if (int rc = mb::check_gated_outputs(entry, dtype, y, y_bytes, y_scales, y_scales_bytes, gate_up, gate_up_bytes, rows,
                                       n))
    return rc;
  mb::Fp8Product p{};
  p.x = a;
  p.sx = static_cast<const uint8_t*>(scale_a);
  p.x_shift = mb::shift_of(a_block);
  p.w = static_cast<const uint8_t*>(b);
  p.sw = static_cast<const uint8_t*>(scale_b);
  p.w_shift = mb::shift_of(b_block);
  p.y = y;
  p.sy = static_cast<uint8_t*>(y_scales);
  p.gate_up = gate_up;
  p.rows = p.tokens = static_cast<int>(rows);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.offsets = offsets;
  p.copies = 1;
  p.experts = static_cast<int>(experts);
  return mb::launch_product(entry, kernel, dtype, y_scales ? mb::kFp8GatedFp8 : mb::kFp8Gated, p,
                            static_cast<hipStream_t>(stream));
}

int mb_fp8_gated(int dtype, const void* x, uint64_t x_bytes, uint32_t tokens, uint64_t row_stride, const void* w,
                 uint64_t w_bytes, const void* scale_w, uint64_t scale_w_bytes, uint32_t w_block, void* y,
                 uint64_t y_bytes, void* y_scales, uint64_t y_scales_bytes, void* gate_up, uint64_t gate_up_bytes,
                 uint32_t n, uint32_t k, const int32_t* offsets, uint64_t offsets_bytes, const int32_t* order,
                 const int32_t* slots, uint64_t slots_bytes, uint32_t copies, uint32_t experts, void* workspace,
                 uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_fp8_gated";
  if (slots && (copies == 0 || copies > 64))
    return mb::fail(MB_ERR_INVALID, "%s: %u slots a token outside 1..64", entry, copies);
  const uint64_t rows = uint64_t{tokens} * (slots ? copies : 1);
  if (int rc = mb::check_shape(entry, dtype, rows, uint64_t{2} * n, k, experts)) return rc;
  if (int rc = mb::check_offsets(entry, offsets, offsets_bytes, experts)) return rc;
  if (int rc = mb::check_routes(entry, offsets, order, slots, slots_bytes, rows)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (k == 0) return mb::fail(MB_ERR_INVALID, "%s: K must be positive", entry);
  if (int rc = mb::fp8_check_rows(entry, "x", dtype, x, x_bytes, tokens, k, row_stride)) return rc;
  if (int rc = mb::fp8_check_operand(entry, "the weight's", uint64_t{2} * n, k, experts, w_block, w, w_bytes, scale_w,
                                     scale_w_bytes))
    return rc;
  if (int rc = mb::check_gated_outputs(entry, dtype, y, y_bytes, y_scales, y_scales_bytes, gate_up, gate_up_bytes, rows,
                                       n))
    return rc;
  mb::Fp8Product p{};
  p.x = x;
  p.row_stride = row_stride;
  p.w = static_cast<const uint8_t*>(w);
  p.sw = static_cast<const uint8_t*>(scale_w);
  p.w_shift = mb::shift_of(w_block);
  p.y = y;
  p.sy = static_cast<uint8_t*>(y_scales);
  p.gate_up = gate_up;
  p.rows = static_cast<int>(rows);
  p.n = static_cast<int>(n);
  p.k = static_cast<int>(k);
  p.offsets = offsets;
  p.order = slots ? order : nullptr;
  p.copies = slots ? static_cast<int>(copies) : 1;
  p.tokens = static_cast<int>(tokens);
  p.experts = static_cast<int>(experts);
  return mb::run_linear(entry, dtype, y_scales ? mb::kFp8GatedFp8 : mb::kFp8Gated, p, slots, workspace, workspace_bytes,
                        static_cast<hipStream_t>(stream));
}

uint64_t mb_fp8_gated_backward_workspace(uint32_t rows, uint32_t n, uint32_t k) {
  const uint64_t width = uint64_t{2} * n < mb::kFp8MostK ? uint64_t{2} * n : mb::kFp8MostK;
  return mb::gradient_space(rows < mb::kFp8MostRows ? rows : mb::kFp8MostRows, static_cast<uint32_t>(width), k).end;
}

int mb_fp8_gated_backward(int dtype, const void* d_out, uint64_t d_out_bytes, uint64_t d_out_stride,
                          const void* gate_up, uint64_t gate_up_bytes, const void* x, uint64_t x_bytes,
                          uint64_t x_stride, const void* w_columns, uint64_t w_columns_bytes, const void* scale_w,
                          uint64_t scale_w_bytes, uint32_t w_block, void* d_x, uint64_t d_x_bytes, void* d_w,
                          uint64_t d_w_bytes, uint32_t rows, uint32_t n, uint32_t k, void* workspace,
                          uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_fp8_gated_backward";
  if (n > mb::kFp8MostK / 2)
    return mb::fail(MB_ERR_UNSUPPORTED, "%s: n = %u: at most %u columns", entry, n, mb::kFp8MostK / 2);
  return mb::run_backward(entry, dtype, d_out, d_out_bytes, d_out_stride, gate_up, gate_up_bytes, true, x, x_bytes,
                          x_stride, w_columns, w_columns_bytes, scale_w, scale_w_bytes, w_block, d_x, d_x_bytes, d_w,
                          d_w_bytes, rows, 2 * n, k, workspace, workspace_bytes, static_cast<hipStream_t>(stream));
}

}  // extern "C"
