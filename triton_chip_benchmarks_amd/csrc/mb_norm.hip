// Root-mean-square norm of rows, with the residual's addition before it and an output
// in the rows' type, in FP8 with block scales, or both; and its gradients.
//
//   t = x + residual, rounded to the rows' type (the residual stream, an output)
//   y = t r w,  r = 1 / sqrt(mean t^2 + eps)
//   d_t = r (w dy - t r^2 mean(w dy t)) + d_total,  d_w = sum over rows of dy t r
//
// The norm is taken of t as it is rounded, so that the gradient, which reads the stream
// again, differentiates what was computed. The norm's sum, root and products are of 64
// bits, at the rate of fp32's and under the loads: an FP8 code beside a border is then the
// exact value's, but for fp32's rounding. The gradients' sums are of fp32, of a row that is
// scaled by a power of two where its squares pass fp32's range.
#include <type_traits>

#include "mb_fp8.h"
#include "mb_fp8_device.h"

namespace mb {
namespace {

typedef float norm_f32x4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kMostColumns = 16384;  // of a row, which a workgroup holds in its registers

// Sum over a row's WAVES waves, the same in every lane; `parts` has a place for each.
template <int WAVES>
__device__ __forceinline__ double row_sum(double v, double* parts, uint32_t wave) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, 64);
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) parts[wave] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += parts[w];
  }
  return v;
}

struct NormArguments {
  const void* x;
  uint64_t x_stride;
  const void* residual;
  uint64_t residual_stride;
  const void* weight;
  float eps;
  void *total, *out;
  uint8_t *codes, *scales;
  uint32_t rows, n;
  double per_column;  // 1 / n
};

// A row by WAVES waves, each lane P pieces of eight neighbouring elements: the row is
// read once and stays in registers. 16 lanes hold a block of the FP8 output, a wave a
// dword of its scales. Memory bounds it: 16384 rows of 8192 in bf16 with the residual,
// its sum and the FP8 output take 156 to 164 us, 5.8 to 6.0 TB/s.
template <class T, int WAVES, int P>
__global__ void __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) rms_norm_kernel(NormArguments a) {
  constexpr uint32_t PER_GROUP = WAVES == 1 ? 4 : 1;  // rows of a workgroup
  __shared__ double parts[WAVES];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t row = blockIdx.x * PER_GROUP + (WAVES == 1 ? wave : 0);
  if (row >= a.rows) return;
  const uint32_t n = a.n, thread = WAVES == 1 ? lane : threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* residual = static_cast<const T*>(a.residual) + row * a.residual_stride;
  Raw8<T> raw[P], added[P], weight[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t c = (p * WAVES * 64 + thread) * 8;
    const int live = static_cast<int>(n > c ? n - c : 0);
    raw[p].load(x + c, live);
    if (a.residual) added[p].load(residual + c, live);
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t c = (p * WAVES * 64 + thread) * 8;
    weight[p].load(static_cast<const T*>(a.weight) + c, static_cast<int>(n > c ? n - c : 0));
  }
  float t[P][8];
  double sum = 0.0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      t[p][i] = raw[p][i];
      if (a.residual) t[p][i] = widen(static_cast<T>(t[p][i] + added[p][i]));
      sum = fma(static_cast<double>(t[p][i]), static_cast<double>(t[p][i]), sum);
    }
  }
  if (a.total) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t c = (p * WAVES * 64 + thread) * 8;
      if (c < n) store8<false>(static_cast<T*>(a.total) + static_cast<uint64_t>(row) * n + c, t[p], static_cast<int>(n - c));
    }
  }
  sum = row_sum<WAVES>(sum, parts, wave);
  const double mean = sum * a.per_column + a.eps;
  double inverse;
  if (mean > 1e-30 && mean < 1e30) {  // a step of Newton from fp32's: within 2^-44 of it
    inverse = __builtin_amdgcn_rsqf(static_cast<float>(mean));
    inverse *= 1.5 - 0.5 * mean * inverse * inverse;
  } else {
    inverse = 1.0 / sqrt(mean);
  }
  const uint32_t pitch = (n + 15) / 16 * 16;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t c = (p * WAVES * 64 + thread) * 8;
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      y[i] = static_cast<float>(t[p][i] * inverse * static_cast<double>(weight[p][i]));
    if (a.out && c < n)
      store8<false>(static_cast<T*>(a.out) + static_cast<uint64_t>(row) * n + c, y, static_cast<int>(n - c));
    if (a.codes) {
      const uint32_t scale = fp8_scale_byte(row16_magnitude<float>(float8_magnitude(y)));
      if (c < pitch)
        *reinterpret_cast<elem_u32x2*>(a.codes + static_cast<uint64_t>(row) * pitch + c) =
            elem_u32x2{fp8_encode4(y[0], y[1], y[2], y[3], scale), fp8_encode4(y[4], y[5], y[6], y[7], scale)};
      const uint32_t kept = c - lane % 16 * 8 < n ? scale : 127;
      uint32_t four = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        four |= static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(kept), 16 * b)) << (8 * b);
      if (lane == 0 && c < n)
        *reinterpret_cast<uint32_t*>(a.scales + (c / 512 * uint64_t{a.rows} + row) * 4) = four;
    }
  }
}

__host__ __device__ constexpr uint32_t partial_pitch(uint32_t n) { return (n + 7) / 8 * 8; }

struct NormGradient {
  const void* d_out;
  uint64_t d_stride;
  const void* total;
  uint64_t total_stride;
  const void* weight;
  float eps;
  const void* d_total;
  uint64_t d_total_stride;
  void* d_x;
  float* partial;  // [workers][partial_pitch(n)] of d_w
  uint32_t rows, n, workers;
};

// A row of the gradient is summed as it is where its mean square and eps are between these:
// past the first its squares may overflow fp32, under the second its products with a small
// gradient may vanish. Other rows are summed again, scaled. (Sums of 64 bits hold them all:
// 8192 rows of 8192 in bf16 134 us with them and 107 so, 20000 of 2048 in fp16 118 and 70.)
constexpr float kMeanMost = 0x1p110f, kMeanLeast = 0x1p-40f;

// Rows worker, worker + workers, .. of the gradient, by WAVES waves as above: both sums
// of a row in one pass over it, and the worker's part of d_w in registers. Memory bounds
// it: 8192 rows of 8192 in bf16, three read and one written, take 104 to 112 us, 4.8 to 5.2
// TB/s, and the sum below 4.6.
template <class T, int WAVES, int P>
__global__ void __launch_bounds__(WAVES > 4 ? 64 * WAVES : 256) rms_norm_backward_kernel(NormGradient a) {
  constexpr uint32_t PER_GROUP = WAVES == 1 ? 4 : 1;
  __shared__ float parts[2][2][WAVES];  // sums of even and odd rows in turn
  __shared__ float scaled_parts[3][WAVES];
  // Where a lane's registers hold no more (16 waves have 128 each), d_total is read when
  // it is added, and the parts of d_w lie in LDS, each lane's its own.
  constexpr bool LATE = WAVES * P == 32 && sizeof(T) == 4;
  __shared__ float kept[LATE ? P * 8 * WAVES * 64 : 1];
  const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t worker = blockIdx.x * PER_GROUP + (WAVES == 1 ? wave : 0);
  if (worker >= a.workers) return;
  const uint32_t n = a.n, thread = WAVES == 1 ? lane : threadIdx.x;
  Raw8<T> weight[P];
  float d_weight[LATE ? 1 : P][8];
  auto sum_at = [&](int p, int i) __attribute__((always_inline)) -> float& {
    if constexpr (LATE)
      return kept[(p * 8 + i) * (WAVES * 64) + threadIdx.x];
    else
      return d_weight[p][i];
  };
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t c = (p * WAVES * 64 + thread) * 8;
    weight[p].load(static_cast<const T*>(a.weight) + c, static_cast<int>(n > c ? n - c : 0));
#pragma unroll
    for (int i = 0; i < 8; ++i) sum_at(p, i) = 0.0f;
  }
  uint32_t turn = 0;
  for (uint32_t row = worker; row < a.rows; row += a.workers, turn ^= 1) {
    Raw8<T> t[P], d[P], d_total[LATE ? 1 : P];
    int rest = static_cast<int>(n);
    asm volatile("" : "+v"(rest));  // the masks of a row's end are made anew in each: all of them exceed the SGPRs
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t c = (p * WAVES * 64 + thread) * 8;
      const int live = rest - static_cast<int>(c);
      t[p].load(static_cast<const T*>(a.total) + row * a.total_stride + c, live);
      d[p].load(static_cast<const T*>(a.d_out) + row * a.d_stride + c, live);
      if (!LATE && a.d_total) d_total[p].load(static_cast<const T*>(a.d_total) + row * a.d_total_stride + c, live);
    }
    // Sums of squares and of dy w t over the row times `scale`.
    auto sums = [&](float scale, float (*shared)[WAVES], float& squares, float& along) __attribute__((always_inline)) {
      squares = along = 0.0f;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = t[p][i] * scale;
          squares = fmaf(v, v, squares);
          along = fmaf(d[p][i] * weight[p][i], v, along);
        }
      squares = wave_add(squares);
      along = wave_add(along);
      if constexpr (WAVES > 1) {
        if (lane == 0) {
          shared[0][wave] = squares;
          shared[1][wave] = along;
        }
        __syncthreads();
        squares = along = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
          squares += shared[0][w];
          along += shared[1][w];
        }
      }
    };
    float squares, along, scale = 1.0f;
    sums(1.0f, parts[turn], squares, along);
    float mean = squares / static_cast<float>(n) + a.eps;
    // (The same in every lane of the row's waves. fp16's squares and products all fit fp32.)
    if (!__is_same(T, _Float16) && !(mean < kMeanMost && mean > kMeanLeast)) {
      // The power of two that takes the larger of the row's largest and eps's root to 1 .. 4.
      float largest = 0.0f;
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(t[p][i]));
      largest = team_max<64>(largest);
      if constexpr (WAVES > 1) {
        if (lane == 0) scaled_parts[2][wave] = largest;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < WAVES; ++w) largest = fmaxf(largest, scaled_parts[2][w]);
      }
      largest = fmaxf(largest, sqrtf(a.eps));
      const int field = static_cast<int>(float_bits(largest) >> 23);
      scale = __builtin_bit_cast(float, static_cast<uint32_t>(max(254 - field, 1)) << 23);
      sums(scale, scaled_parts, squares, along);
      mean = squares / static_cast<float>(n) + a.eps * scale * scale;
    }
    float inverse = 1.0f / sqrtf(mean);
    const float share = along / static_cast<float>(n) * inverse;
    inverse *= scale;  // of t itself: past fp32 only where all of a row lies below 2^-126, and eps with it
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const uint32_t c = (p * WAVES * 64 + thread) * 8;
      const int live = rest - static_cast<int>(c);
      if (LATE && a.d_total) d_total[0].load(static_cast<const T*>(a.d_total) + row * a.d_total_stride + c, live);
      float d_x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float normed = t[p][i] * inverse;
        sum_at(p, i) = fmaf(d[p][i], normed, sum_at(p, i));
        d_x[i] = inverse * (d[p][i] * weight[p][i] - normed * share);
        if (a.d_total) d_x[i] += d_total[LATE ? 0 : p][i];
      }
      if (live > 0) store8<false>(static_cast<T*>(a.d_x) + static_cast<uint64_t>(row) * n + c, d_x, live);
    }
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const uint32_t c = (p * WAVES * 64 + thread) * 8;
    float sums[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) sums[i] = sum_at(p, i);
    if (c < n) store8<false>(a.partial + uint64_t{worker} * partial_pitch(n) + c, sums, 8);  // 0 behind n
  }
}

// d_w from its parts: 64 columns a workgroup, in 64 slices of the workers, each with
// eight loads in flight, joined in a fixed order.
template <class T>
__global__ void __launch_bounds__(1024)
    rms_norm_weight_kernel(const float* __restrict__ partial, T* __restrict__ d_weight, uint32_t workers, uint32_t n) {
  __shared__ float parts[64][64 + 4];
  const uint32_t place = threadIdx.x % 16 * 4, column = blockIdx.x * 64 + place, slice = threadIdx.x / 16;
  const uint32_t pitch = partial_pitch(n);
  float sum[4] = {};
  if (column < pitch)
    for (uint32_t w = slice; w < workers; w += 8 * 64) {
      norm_f32x4 v[8];
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
        v[j] = w + j * 64 < workers
                   ? *reinterpret_cast<const norm_f32x4*>(partial + uint64_t{w + j * 64} * pitch + column)
                   : norm_f32x4{};
#pragma unroll
      for (uint32_t j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i] += v[j][i];
    }
#pragma unroll
  for (int i = 0; i < 4; ++i) parts[slice][place + i] = sum[i];
  __syncthreads();
  if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < n) {
    float all = 0.0f;
#pragma unroll 8
    for (int s = 0; s < 64; ++s) all += parts[s][threadIdx.x];
    d_weight[blockIdx.x * 64 + threadIdx.x] = static_cast<T>(all);
  }
}

// call(integral_constant<WAVES>, integral_constant<P>) for a row of n elements: one wave
// up to 1024, four up to 8192, else 16; with `spread`, as many as have a piece each.
template <class F>
void for_width(uint32_t n, bool spread, F&& call) {
  auto with = [&](auto waves, auto pieces) { call(waves, pieces); };
#define MB_NORM_FORM(W, P) with(std::integral_constant<int, W>{}, std::integral_constant<int, P>{})
  if (n <= 512)
    MB_NORM_FORM(1, 1);
  else if (n <= 1024 && !spread)
    MB_NORM_FORM(1, 2);
  else if (n <= 2048)
    MB_NORM_FORM(4, 1);
  else if (n <= 4096 && !spread)
    MB_NORM_FORM(4, 2);
  else if (n <= 8192 && !spread)
    MB_NORM_FORM(4, 4);
  else if (n <= 8192)
    MB_NORM_FORM(16, 1);
  else
    MB_NORM_FORM(16, 2);
#undef MB_NORM_FORM
}

template <class T>
int launch_norm(const char* entry, const NormArguments& a, hipStream_t stream) {
  int status = MB_OK;
  // Few rows are spread: one of 8192 takes 3.6 us by 16 waves, 0.8 of them for the sums
  // of 64 bits.
  for_width(a.n, a.rows <= 512, [&](auto waves, auto pieces) {
    constexpr int W = decltype(waves)::value, P = decltype(pieces)::value;
    constexpr uint32_t kThreads = W > 4 ? 64 * W : 256;
    const uint32_t grid = W == 1 ? (a.rows + 3) / 4 : a.rows;
    if (uint64_t{grid} * kThreads > 0xffffffffu) {
      status = fail(MB_ERR_UNSUPPORTED, "%s: %u rows of %u exceed one launch", entry, a.rows, a.n);
      return;
    }
    rms_norm_kernel<T, W, P><<<dim3(grid), dim3(kThreads), 0, stream>>>(a);
    status = launch_status("rms_norm");
  });
  return status;
}

template <class T>
void launch_norm_backward(const NormGradient& a, T* d_weight, hipStream_t stream) {
  // Past 4096 columns 16 waves a row, half as many workers for the same waves: 4096 rows
  // of 8192 in fp32 100 to 103 us, by four waves 108; 1000 of 5003 20 to 23 and 24; 8192
  // of 8192 in bf16 108 to 112 by both.
  for_width(a.n, a.n > 4096, [&](auto waves, auto pieces) {
    constexpr int W = decltype(waves)::value, P = decltype(pieces)::value;
    if constexpr (W != 4 || P != 4)
      rms_norm_backward_kernel<T, W, P>
          <<<dim3(W == 1 ? (a.workers + 3) / 4 : a.workers), dim3(W > 4 ? 64 * W : 256), 0, stream>>>(a);
  });
  rms_norm_weight_kernel<T><<<dim3((a.n + 63) / 64), dim3(1024), 0, stream>>>(a.partial, d_weight, a.workers, a.n);
}

// Workers of the gradient: as many waves as hide the memory's latency, and no more, for
// each worker's part of d_w is written and read again. Microseconds with 256, 512, 1024
// and 2048 of them: 512 columns of bf16 by one wave 419, 222, 124, 85 (100000 rows); 4096
// by four 128, 105, 111, 118 (16384 rows); 16384 by 16: 109, 115, 127, 155 (4096).
uint32_t norm_workers(uint32_t rows, uint32_t n) {
  const uint32_t most = n <= 1024 ? 2048 : n <= 4096 ? 512 : 256;
  return rows < most ? rows : most;
}

#define MB_NORM_REGISTER_FORM(T, NAME, W, P)                                                  \
  MB_REGISTER_KERNEL("rms_norm_" NAME "_" #W "x" #P, (rms_norm_kernel<T, W, P>))
#define MB_NORM_REGISTER_BACKWARD(T, NAME, W, P)                                              \
  MB_NORM_REGISTER_FORM(T, NAME, W, P);                                                       \
  MB_REGISTER_KERNEL("rms_norm_backward_" NAME "_" #W "x" #P, (rms_norm_backward_kernel<T, W, P>))
#define MB_NORM_REGISTER(T, NAME)                \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 1, 1);      \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 1, 2);      \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 4, 1);      \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 4, 2);      \
  MB_NORM_REGISTER_FORM(T, NAME, 4, 4);          \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 16, 1);     \
  MB_NORM_REGISTER_BACKWARD(T, NAME, 16, 2);     \
  MB_REGISTER_KERNEL("rms_norm_weight_" NAME, rms_norm_weight_kernel<T>)
MB_NORM_REGISTER(float, "f32");
MB_NORM_REGISTER(_Float16, "f16");
MB_NORM_REGISTER(__bf16, "bf16");

int check_columns(const char* entry, uint32_t n) {
  return n <= kMostColumns ? MB_OK : fail(MB_ERR_UNSUPPORTED, "%s: rows of %u: at most %u elements", entry, n, kMostColumns);
}

int check_weight(const char* entry, int dtype, const void* weight, uint64_t weight_bytes, uint32_t n) {
  return fp8_check_rows(entry, "the weight", dtype, weight, weight_bytes, 1, n, n);
}

}  // namespace
}  // namespace mb

extern "C" {

int mb_rms_norm(int dtype, const void* x, uint64_t x_bytes, uint64_t x_stride, const void* residual,
                uint64_t residual_bytes, uint64_t residual_stride, const void* weight, uint64_t weight_bytes, float eps,
                void* total, uint64_t total_bytes, void* out, uint64_t out_bytes, void* codes, uint64_t codes_bytes,
                void* scales, uint64_t scales_bytes, uint32_t rows, uint32_t n, void* stream) {
  const char* entry = "mb_rms_norm";
  if (!mb::elem_bytes(dtype)) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (int rc = mb::check_columns(entry, n)) return rc;
  if (rows == 0 || n == 0) return MB_OK;
  if (!(eps >= 0.0f)) return mb::fail(MB_ERR_INVALID, "%s: eps must not be negative", entry);
  if (int rc = mb::fp8_check_rows(entry, "x", dtype, x, x_bytes, rows, n, x_stride)) return rc;
  if (residual)
    if (int rc = mb::fp8_check_rows(entry, "the residual", dtype, residual, residual_bytes, rows, n, residual_stride))
      return rc;
  if ((residual == nullptr) != (total == nullptr))
    return mb::fail(MB_ERR_INVALID, "%s: a residual and its sum with x go together", entry);
  if (int rc = mb::check_weight(entry, dtype, weight, weight_bytes, n)) return rc;
  if (total)
    if (int rc = mb::fp8_check_output(entry, "total", dtype, total, total_bytes, rows, n)) return rc;
  if (out == nullptr && codes == nullptr) return mb::fail(MB_ERR_INVALID, "%s: no output", entry);
  if (out)
    if (int rc = mb::fp8_check_output(entry, "out", dtype, out, out_bytes, rows, n)) return rc;
  if (codes)
    if (int rc = mb::fp8_check_operand(entry, "the output's", rows, n, 1, 1, codes, codes_bytes, scales, scales_bytes))
      return rc;
  const mb::NormArguments a{x,     x_stride, residual, residual_stride, weight, eps, total, out,
                            static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales), rows, n, 1.0 / n};
  int status = MB_OK;
  MB_FOR_DTYPE(dtype, status = mb::launch_norm<T>(entry, a, static_cast<hipStream_t>(stream)));
  return status;
}

uint64_t mb_rms_norm_backward_workspace(uint32_t rows, uint32_t n) {
  return uint64_t{mb::norm_workers(rows, n)} * mb::partial_pitch(n) * 4;
}

int mb_rms_norm_backward(int dtype, const void* d_out, uint64_t d_out_bytes, uint64_t d_out_stride, const void* total,
                         uint64_t total_bytes, uint64_t total_stride, const void* weight, uint64_t weight_bytes,
                         float eps, const void* d_total, uint64_t d_total_bytes, uint64_t d_total_stride, void* d_x,
                         uint64_t d_x_bytes, void* d_weight, uint64_t d_weight_bytes, uint32_t rows, uint32_t n,
                         void* workspace, uint64_t workspace_bytes, void* stream) {
  const char* entry = "mb_rms_norm_backward";
  if (!mb::elem_bytes(dtype)) return mb::fail(MB_ERR_INVALID, "%s: unknown element type %d", entry, dtype);
  if (int rc = mb::check_columns(entry, n)) return rc;
  if (rows == 0 || n == 0) return mb::fail(MB_ERR_INVALID, "%s: rows and their elements must be positive", entry);
  if (!(eps >= 0.0f)) return mb::fail(MB_ERR_INVALID, "%s: eps must not be negative", entry);
  if (int rc = mb::fp8_check_rows(entry, "d_out", dtype, d_out, d_out_bytes, rows, n, d_out_stride)) return rc;
  if (int rc = mb::fp8_check_rows(entry, "total", dtype, total, total_bytes, rows, n, total_stride)) return rc;
  if (int rc = mb::check_weight(entry, dtype, weight, weight_bytes, n)) return rc;
  if (d_total)
    if (int rc = mb::fp8_check_rows(entry, "d_total", dtype, d_total, d_total_bytes, rows, n, d_total_stride)) return rc;
  if (int rc = mb::fp8_check_output(entry, "d_x", dtype, d_x, d_x_bytes, rows, n)) return rc;
  if (int rc = mb::fp8_check_output(entry, "d_weight", dtype, d_weight, d_weight_bytes, 1, n)) return rc;
  const uint64_t needed = mb_rms_norm_backward_workspace(rows, n);
  if (workspace == nullptr || workspace_bytes < needed)
    return mb::fail(MB_ERR_INVALID, "%s: the workspace is NULL or too small: %llu bytes needed", entry,
                    (unsigned long long)needed);
  if (!mb::aligned(workspace, 16)) return mb::fail(MB_ERR_ALIGNMENT, "%s: the workspace must lie on 16 bytes", entry);
  const uint32_t workers = mb::norm_workers(rows, n);
  const mb::NormGradient a{d_out, d_out_stride, total, total_stride, weight, eps, d_total, d_total_stride, d_x,
                           static_cast<float*>(workspace), rows, n, workers};
  MB_FOR_DTYPE(dtype, mb::launch_norm_backward<T>(a, static_cast<T*>(d_weight), static_cast<hipStream_t>(stream)));
  return mb::launch_status("rms_norm_backward");
}

}  // extern "C"
