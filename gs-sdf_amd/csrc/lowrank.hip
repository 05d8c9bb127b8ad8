// lowrank.hip — low-rank adapters of many requests at once beside a shared projection:
//     y_t = base_t + s_g B_g h_t,   h_t = A_g drop(x_t),   g = ids[t]
// backward:  dh_t = s_g B_g^T dy_t,  dx_t = drop'(A_g^T dh_t),  dA_g = sum_t dh_t drop(x_t)^T,  dB_g = s_g sum_t dy_t h_t^T.
#include "adapter_common.h"

namespace gsdf {

struct Lowrank {      // gsdf_lowrank_args as the kernels take it
  int64_t rows, x_stride;
  int n_in, n_out, rank, n_adapters, ids_64;
  const void *ids;
  const float *scales;
  Dropout drop;
};
__device__ __forceinline__ int adapter_of(const Lowrank &q, int64_t row) {      // -1: none
  const int64_t g = load_id(q.ids, q.ids_64, row);
  return g >= 0 && g < q.n_adapters ? (int)g : -1;
}

// h[row][j] = sum_k drop(x)[row][k] a[g][j][k]: a wave per (row, j)
template <typename T>
__global__ void __launch_bounds__(256) lowrank_shrink_kernel(Lowrank q, const T *__restrict__ x, const T *__restrict__ a, float *__restrict__ h) {
  dropout_counter(q.drop);
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, g = adapter_of(q, row);
  for (int j = threadIdx.x >> 6; j < q.rank; j += 4) {
    float s = 0.f;
    if (g >= 0)
      for (int k = lane; k < q.n_in; k += 64) {
        float v = (float)x[row * q.x_stride + k];
        if (q.drop.threshold != 0) {
          uint32_t w[4];
          dropout_bits(q.drop, k >> 3, (uint32_t)row, w);
          v = dropout_keeps(q.drop, w, k & 7) ? v * q.drop.scale : 0.f;
        }
        s = fmaf(v, (float)a[((int64_t)g * q.rank + j) * q.n_in + k], s);
      }
    s = wave_sum_to_lane63(s);
    if (lane == 63) h[row * q.rank + j] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) lowrank_expand_kernel(Lowrank q, const float *__restrict__ h, const T *__restrict__ b, const T *base, int64_t base_stride,
                                                             T *y, int64_t y_stride) {
  const int64_t row = blockIdx.x;
  const int g = adapter_of(q, row);
  const float s = g < 0 || q.scales == nullptr ? 1.f : q.scales[g];
  for (int n = blockIdx.y * 256 + threadIdx.x; n < q.n_out; n += gridDim.y * 256) {
    float v = 0.f;
    if (g >= 0)
      for (int j = 0; j < q.rank; ++j) v = fmaf(h[row * q.rank + j], (float)b[((int64_t)g * q.n_out + n) * q.rank + j], v);
    y[row * y_stride + n] = (T)((base != nullptr ? (float)base[row * base_stride + n] : 0.f) + s * v);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) lowrank_dh_kernel(Lowrank q, const T *__restrict__ dy, int64_t dy_stride, const T *__restrict__ b, float *__restrict__ dh) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, g = adapter_of(q, row);
  for (int j = threadIdx.x >> 6; j < q.rank; j += 4) {
    float s = 0.f;
    if (g >= 0)
      for (int n = lane; n < q.n_out; n += 64) s = fmaf((float)dy[row * dy_stride + n], (float)b[((int64_t)g * q.n_out + n) * q.rank + j], s);
    s = wave_sum_to_lane63(s) * (g < 0 || q.scales == nullptr ? 1.f : q.scales[g]);
    if (lane == 63) dh[row * q.rank + j] = s;
  }
}
template <typename T>
__global__ void __launch_bounds__(256) lowrank_dx_kernel(Lowrank q, const float *__restrict__ dh, const T *__restrict__ a, T *__restrict__ dx, int64_t dx_stride) {
  dropout_counter(q.drop);
  const int64_t row = blockIdx.x;
  const int g = adapter_of(q, row);
  for (int k = blockIdx.y * 256 + threadIdx.x; k < q.n_in; k += gridDim.y * 256) {
    float v = 0.f;
    if (g >= 0)
      for (int j = 0; j < q.rank; ++j) v = fmaf(dh[row * q.rank + j], (float)a[((int64_t)g * q.rank + j) * q.n_in + k], v);
    if (q.drop.threshold != 0) {
      uint32_t w[4];
      dropout_bits(q.drop, k >> 3, (uint32_t)row, w);
      v = dropout_keeps(q.drop, w, k & 7) ? v * q.drop.scale : 0.f;
    }
    dx[row * dx_stride + k] = (T)v;
  }
}
// out[g][j][c] (or [g][c][j]) = sum over g's rows of u[t][j] v[t][c]: a thread per element
template <typename T, bool DROP>
__global__ void __launch_bounds__(256) lowrank_outer_kernel(Lowrank q, const float *__restrict__ u, const T *__restrict__ v, int64_t v_stride, int width,
                                                            bool scaled, bool columns_first, T *__restrict__ out) {
  dropout_counter(q.drop);
  const int c = blockIdx.x * 256 + threadIdx.x, j = blockIdx.y, g = blockIdx.z;
  if (c >= width) return;
  float s = 0.f;
  for (int64_t row = 0; row < q.rows; ++row) {
    if (adapter_of(q, row) != g) continue;
    float t = (float)v[row * v_stride + c];
    if (DROP && q.drop.threshold != 0) {
      uint32_t w[4];
      dropout_bits(q.drop, c >> 3, (uint32_t)row, w);
      t = dropout_keeps(q.drop, w, c & 7) ? t * q.drop.scale : 0.f;
    }
    s = fmaf(u[row * q.rank + j], t, s);
  }
  if (scaled && q.scales != nullptr) s *= q.scales[g];
  out[columns_first ? ((int64_t)g * width + c) * q.rank + j : ((int64_t)g * q.rank + j) * width + c] = (T)s;
}

static int lowrank_check(const gsdf_lowrank_args *a, Lowrank *q) {
  GSDF_REQUIRE(a != nullptr, "lowrank: args is NULL");
  GSDF_REQUIRE(a->rows >= 0 && a->rows < (1ll << 31), "lowrank: %lld rows outside [0, 2^31)", (long long)a->rows);
  GSDF_REQUIRE(a->n_in >= 1 && a->n_out >= 1 && a->n_in < (1 << 24) && a->n_out < (1 << 24), "lowrank: widths %d -> %d outside [1, 2^24)", a->n_in, a->n_out);
  GSDF_REQUIRE(a->rank >= 1 && a->rank <= GSDF_LOWRANK_MAX_RANK, "lowrank: rank %d outside [1, %d]", a->rank, GSDF_LOWRANK_MAX_RANK);
  GSDF_REQUIRE(a->n_adapters >= 1 && a->n_adapters <= GSDF_LOWRANK_MAX_ADAPTERS, "lowrank: %d adapters outside [1, %d]", a->n_adapters, GSDF_LOWRANK_MAX_ADAPTERS);
  GSDF_REQUIRE(known_dtype(a->dtype), "lowrank: unknown element type %d", a->dtype);
  GSDF_REQUIRE(a->p >= 0.0 && a->p <= 1.0, "lowrank: p = %g outside [0, 1]", a->p);
  GSDF_REQUIRE(a->rows == 0 || (a->x != nullptr && a->ids != nullptr), "lowrank: x and ids are required");
  GSDF_REQUIRE(a->a != nullptr && a->b != nullptr, "lowrank: a and b are required");
  GSDF_REQUIRE(a->rows <= 1 || a->x_stride >= 0, "lowrank: row stride %lld of x", (long long)a->x_stride);
  q->rows = a->rows; q->x_stride = a->x_stride; q->n_in = a->n_in; q->n_out = a->n_out; q->rank = a->rank; q->n_adapters = a->n_adapters;
  q->ids_64 = a->ids_64; q->ids = a->ids; q->scales = a->scales;
  q->drop = make_dropout(a->p, a->seed, a->offset, a->offset_dev);
  return GSDF_OK;
}

}  // namespace gsdf

extern "C" size_t gsdf_lowrank_save_bytes(const gsdf_lowrank_args *a) {
  gsdf::Lowrank q;
  if (gsdf::lowrank_check(a, &q) != GSDF_OK) return 0;
  return gsdf::align_up((size_t)q.rows * q.rank * 4 + 16, 256);
}
extern "C" size_t gsdf_lowrank_fwd_ws_bytes(const gsdf_lowrank_args *a) { return gsdf_lowrank_save_bytes(a); }
extern "C" size_t gsdf_lowrank_bwd_ws_bytes(const gsdf_lowrank_args *a) { return gsdf_lowrank_save_bytes(a); }

extern "C" int gsdf_lowrank_fwd(const gsdf_lowrank_args *args, const void *base, int64_t base_stride, void *y, int64_t y_stride, void *save, void *ws,
                                gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  Lowrank q;
  if (const int e = lowrank_check(args, &q)) return e;
  if (q.rows == 0) return GSDF_OK;
  GSDF_REQUIRE(y != nullptr && ws != nullptr, "lowrank_fwd: y and the workspace are required");
  GSDF_REQUIRE(q.rows == 1 || (y_stride >= q.n_out && (base == nullptr || base_stride >= 0)), "lowrank_fwd: row strides %lld -> %lld of %d columns",
               (long long)base_stride, (long long)y_stride, q.n_out);
  GSDF_TIMED("gsdf_lowrank_fwd");
  float *h = (float *)(save != nullptr ? save : ws);
  GSDF_BY_DTYPE(args->dtype, {
    lowrank_shrink_kernel<T><<<(unsigned)q.rows, 256, 0, stream>>>(q, (const T *)args->x, (const T *)args->a, h);
    lowrank_expand_kernel<T><<<dim3((unsigned)q.rows, 1), 256, 0, stream>>>(q, h, (const T *)args->b, (const T *)base, base_stride, (T *)y, y_stride);
  });
  GSDF_CHECK_LAUNCH("lowrank_fwd");
  return GSDF_OK;
}

extern "C" int gsdf_lowrank_bwd(const gsdf_lowrank_args *args, const void *dy, int64_t dy_stride, const void *save, void *dx, int64_t dx_stride, void *da,
                                void *db, void *ws, gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  Lowrank q;
  if (const int e = lowrank_check(args, &q)) return e;
  GSDF_REQUIRE(ws != nullptr && (q.rows == 0 || (dy != nullptr && save != nullptr)), "lowrank_bwd: dy, the forward's saved buffer and the workspace are required");
  GSDF_REQUIRE(q.rows <= 1 || (dy_stride >= 0 && (dx == nullptr || dx_stride >= q.n_in)), "lowrank_bwd: row strides %lld, %lld", (long long)dy_stride,
               (long long)dx_stride);
  GSDF_TIMED("gsdf_lowrank_bwd");
  float *dh = (float *)ws;
  const float *h = (const float *)save;
  GSDF_BY_DTYPE(args->dtype, {
    if (q.rows > 0 && (dx != nullptr || da != nullptr)) lowrank_dh_kernel<T><<<(unsigned)q.rows, 256, 0, stream>>>(q, (const T *)dy, dy_stride, (const T *)args->b, dh);
    if (q.rows > 0 && dx != nullptr) lowrank_dx_kernel<T><<<dim3((unsigned)q.rows, 1), 256, 0, stream>>>(q, dh, (const T *)args->a, (T *)dx, dx_stride);
    if (da != nullptr)
      lowrank_outer_kernel<T, true><<<dim3((unsigned)ceil_div(q.n_in, 256), q.rank, q.n_adapters), 256, 0, stream>>>(
          q, dh, (const T *)args->x, q.x_stride, q.n_in, false, false, (T *)da);
    if (db != nullptr)
      lowrank_outer_kernel<T, false><<<dim3((unsigned)ceil_div(q.n_out, 256), q.rank, q.n_adapters), 256, 0, stream>>>(
          q, h, (const T *)dy, dy_stride, q.n_out, true, true, (T *)db);
  });
  GSDF_CHECK_LAUNCH("lowrank_bwd");
  return GSDF_OK;
}
