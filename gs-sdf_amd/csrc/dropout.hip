// dropout.hip — y = [residual +] x * keep / (1 - q): the mask of a counter-based generator, made again in the backward pass and never stored.
//
// Streams x (and residual) once and writes y once: bound by memory at 32-bit elements; at 16-bit elements the generator's integer products
// (20 per 8 elements, a quarter of the full rate) take about as long as the bytes.  One thread owns the 8 neighbouring elements of one Philox block,
// 16 bits for each: the finest split that throws no random bits away.  16384 x 8192 bf16: 147 us with a residual (805 MB, 5.5 TB/s), 94 us without (537 MB,
// 5.75 TB/s); a copy of 1 GiB moves 5.2 TB/s.  Rows whose width is no multiple of 8 end element by element, and a wave with an end in it runs the generator in
// both branches: 30011 x 333 fp16 12.2 us (40 MB, 3.3 TB/s).  Where x is dropped y is exactly 0 (or residual): an infinity or NaN there is gone.
#include <type_traits>

#include "adapter_common.h"

namespace gsdf {

static constexpr int64_t DROPOUT_PAST = 64 << 20;      // bytes of y from which on it is written past the caches

// row = block index / blocks per row, by a multiplication: exact for numerators below 2^31
struct FastDiv {
  uint32_t mul, shift, d;
};
static FastDiv fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return FastDiv{(uint32_t)((((1ull << 31) << l) + d - 1) / d), l, d};
}
__device__ __forceinline__ uint32_t fdiv(uint32_t n, FastDiv f) { return (uint32_t)(((uint64_t)n * f.mul) >> 31 >> f.shift); }

// PAST: y goes past the caches
template <typename T, bool RESIDUAL, bool PAST>
__global__ void __launch_bounds__(256)
    dropout_kernel(uint32_t n_blocks, FastDiv per_row, uint32_t row0, int64_t cols, const T *__restrict__ x, int64_t x_stride,
                   const T *__restrict__ residual, int64_t r_stride, Dropout d, T *__restrict__ y, int64_t y_stride) {
  dropout_counter(d);
  for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n_blocks; i += gridDim.x * 256) {
    const uint32_t row_in = fdiv(i, per_row), block = i - row_in * per_row.d;
    const int64_t row = (int64_t)row0 + row_in, col = (int64_t)block * 8;
    const T *px = x + row * x_stride + col;
    const T *pr = RESIDUAL ? residual + row * r_stride + col : nullptr;
    T *py = y + row * y_stride + col;
    uint32_t w[4];
    if (col + 8 <= cols) {
      T v[8], r[8];
      load_piece<T, 8>(px, v);
      if (RESIDUAL) load_piece<T, 8>(pr, r);
      dropout_bits(d, block, (uint32_t)row, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float keep = dropout_keeps(d, w, j) ? (float)v[j] * d.scale : 0.f;
        v[j] = (T)(RESIDUAL ? keep + (float)r[j] : keep);
      }
      store_piece<T, 8, PAST>(py, v);
    } else {
      dropout_bits(d, block, (uint32_t)row, w);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < cols) {
          const float keep = dropout_keeps(d, w, j) ? (float)px[j] * d.scale : 0.f;
          py[j] = (T)(RESIDUAL ? keep + (float)pr[j] : keep);
        }
    }
  }
}

template <typename T>
static void dropout_launch(int64_t rows, int64_t cols, const T *x, int64_t x_stride, const T *residual, int64_t r_stride, const Dropout &d, T *y,
                           int64_t y_stride, hipStream_t stream) {
  const int64_t per_row = ceil_div(cols, 8), most_rows = ((1ll << 31) - 1) / per_row;
  for (int64_t row0 = 0; row0 < rows; row0 += most_rows) {      // one launch unless the matrix has 2^34 elements
    const uint32_t n = (uint32_t)((rows - row0 < most_rows ? rows - row0 : most_rows) * per_row);
    const unsigned grid = (unsigned)ceil_div(n, 256) < 8192u ? (unsigned)ceil_div(n, 256) : 8192u;
    auto run = [&](auto res, auto past) {
      dropout_kernel<T, decltype(res)::value, decltype(past)::value><<<grid, 256, 0, stream>>>(n, fast_div((uint32_t)per_row), (uint32_t)row0, cols, x, x_stride, residual,
                                                                                            r_stride, d, y, y_stride);
    };
    const bool past = rows * cols * (int64_t)sizeof(T) >= DROPOUT_PAST;
    if (residual != nullptr && past) run(std::true_type{}, std::true_type{});
    else if (residual != nullptr) run(std::true_type{}, std::false_type{});
    else if (past) run(std::false_type{}, std::true_type{});
    else run(std::false_type{}, std::false_type{});
  }
}

}  // namespace gsdf

extern "C" int gsdf_dropout(int64_t rows, int64_t cols, int dtype, const void *x, int64_t x_stride, const void *residual, int64_t residual_stride,
                            double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev, void *y, int64_t y_stride, gsdf_stream_t stream_) {
  hipStream_t stream = (hipStream_t)stream_;
  GSDF_REQUIRE(rows >= 0 && rows < (1ll << 32), "dropout: %lld rows outside [0, 2^32)", (long long)rows);
  GSDF_REQUIRE(cols >= 0 && cols < (1ll << 33), "dropout: %lld columns outside [0, 2^33)", (long long)cols);
  GSDF_REQUIRE(gsdf::known_dtype(dtype), "dropout: unknown element type %d", dtype);
  GSDF_REQUIRE(p >= 0.0 && p <= 1.0, "dropout: p = %g outside [0, 1]", p);
  if (rows == 0 || cols == 0) return GSDF_OK;
  GSDF_REQUIRE(x != nullptr && y != nullptr, "dropout: x and y are required");
  GSDF_REQUIRE(rows == 1 || (x_stride >= 0 && y_stride >= cols && (residual == nullptr || residual_stride >= 0)),
               "dropout: row strides %lld -> %lld of %lld columns", (long long)x_stride, (long long)y_stride, (long long)cols);
  GSDF_TIMED("gsdf_dropout");
  const gsdf::Dropout d = gsdf::make_dropout(p, seed, offset, offset_dev);
  GSDF_BY_DTYPE(dtype, gsdf::dropout_launch<T>(rows, cols, (const T *)x, x_stride, (const T *)residual, residual_stride, d, (T *)y, y_stride, stream));
  GSDF_CHECK_LAUNCH("dropout");
  return GSDF_OK;
}
