// router_balance.hip — the balance loss of a router and the rows each expert got.
//
// With p_t = softmax(logits_t), V the valid rows (mask), k choices a row, counts_e = choices of expert e among the valid rows:
//     loss = E sum_e f_e P_e,   f_e = counts_e / (k V),   P_e = (sum over valid rows of p_te) / V
// f is not differentiated (whole numbers), so  d loss / d logits_te = p_te (c_e - sum_j c_j p_tj)  with c_e = E f_e / V.  A constant taken off every
// c_e changes nothing there (the p of a row sum to 1): c_e = (E counts_e - k V) / (k V^2) is stored instead, from whole numbers, because an even
// router has E f_e close to 1 and the difference would lose its digits in 32 bits.
//
// One read of the logits forward and one backward (the gradient waits for the counts of all rows), one write: bound by memory.  A row lives in
// LPR neighbouring lanes of a wave, up to 8 (16 above 512 experts) consecutive logits each; a lane owns the same columns of every row it meets, so the
// column sums stay in its registers and cross lanes once, at the end.  Counts are whole numbers, and the workgroups' partial column sums are added in
// the order of the workgroups: the results do not change from launch to launch.  A workgroup's rows are added in 32 bits (a lane has few of them), the workgroups in 64.
// 761 x 1024 rows of 32 32-bit logits (97 MB): partial sums 26.8 us (3.7 TB/s: 256 groups of 1024 threads; twice as many take 24.6 and cost the finish the
// same 2.2), finish 5.9 us (latency), backward 34 us for a read and a write (5.7 TB/s).  The sums and maxima over a row without LDS: partial 27.6 -> 26.8.
// The next row's logits asked for ahead took 31.6 us: 16 waves a unit already cover the loads.
#include "adapter_common.h"

namespace gsdf {

static constexpr int RB_THREADS = 1024, RB_MAX_BLOCKS = 256, RB_MAX_EXPERTS = GSDF_ROUTER_MAX_EXPERTS;

// exp(x), x <= 0, in a few units in the last place: the product's rounding error goes back in (exp2's own is one unit)
__device__ __forceinline__ float exp_fast(float x) {
  const float t = x * 1.44269504f, lo = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269504f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return x < -104.f ? 0.f : fmaf(e, lo * 0.693147181f, e);      // below: no 32-bit number, and lo of a type's lowest value is no number at all
}

template <typename T, int VPL, bool WHOLE>
__device__ __forceinline__ void load_logits(const T *__restrict__ row, int c0, int n_experts, float (&v)[VPL]) {
  constexpr int W = 16 / sizeof(T) < VPL ? 16 / sizeof(T) : VPL;      // elements of one 16-byte access
#pragma unroll
  for (int i = 0; i < VPL; i += W) {
    if (WHOLE || c0 + i + W <= n_experts) {
      if (!WHOLE || c0 + i < n_experts) {      // WHOLE: n_experts is a multiple of W, so a piece is in or out
        T t[W];
        load_piece<T, W>(row + c0 + i, t);
#pragma unroll
        for (int j = 0; j < W; ++j) v[i + j] = (float)t[j];
      } else {
#pragma unroll
        for (int j = 0; j < W; ++j) v[i + j] = -INFINITY;
      }
    } else {
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = c0 + i + j < n_experts ? (float)row[c0 + i + j] : -INFINITY;
    }
  }
}

// the value of all LPR lanes of a row from its lanes' values, by `op`: 1, 2, 4 and 8 lanes apart without LDS (lanes that have met hold the same value, so a
// mirrored row of 8 or 16 lanes brings the other half's)
template <int LPR, typename Op>
__device__ __forceinline__ float over_row(float v, Op op) {
  if (LPR > 1) v = op(v, dpp_mov<0xB1>(v));        // quad_perm 1 0 3 2
  if (LPR > 2) v = op(v, dpp_mov<0x4E>(v));        // quad_perm 2 3 0 1
  if (LPR > 4) v = op(v, dpp_mov<0x141>(v));       // row_half_mirror
  if (LPR > 8) v = op(v, dpp_mov<0x140>(v));       // row_mirror
  if (LPR > 16) v = op(v, __shfl_xor(v, 16));
  if (LPR > 32) v = op(v, __shfl_xor(v, 32));
  return v;
}
// v: a lane's logits -> its probabilities.  A row without a finite or larger logit (all -inf) has probability 0 everywhere.
template <int VPL, int LPR>
__device__ __forceinline__ void softmax_row(float (&v)[VPL]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < VPL; ++i) m = fmaxf(m, v[i]);
  m = over_row<LPR>(m, [](float a, float b) { return fmaxf(a, b); });
  m = m == -INFINITY ? 0.f : m;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < VPL; ++i) { v[i] = exp_fast(v[i] - m); s += v[i]; }
  s = over_row<LPR>(s, [](float a, float b) { return a + b; });
  const float inv = s == 0.f ? 0.f : 1.f / s;
#pragma unroll
  for (int i = 0; i < VPL; ++i) v[i] *= inv;
}

struct BalancePartials {      // the workspace: one row of each per workgroup
  float *psum;                // [n_blocks][E]
  int *counts;                // [n_blocks][E]
  int *valid;                 // [n_blocks]
};

template <typename T, int VPL, int LPR, bool WHOLE>
__global__ void __launch_bounds__(RB_THREADS)
    balance_partial_kernel(int64_t rows, int64_t rows_per_block, int n_experts, int k, const T *__restrict__ logits, int64_t stride,
                           const void *__restrict__ ids, int ids_64, const uint8_t *__restrict__ mask, BalancePartials ws) {
  __shared__ int s_count[RB_MAX_EXPERTS + 1];
  __shared__ float s_sum[RB_THREADS / 64][64 * VPL];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane % LPR, c0 = sub * VPL;
  for (int e = threadIdx.x; e <= n_experts; e += RB_THREADS) s_count[e] = 0;      // [n_experts]: valid rows
  __syncthreads();
  float sum[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) sum[i] = 0.f;
  int valid = 0;
  const int64_t first = (int64_t)blockIdx.x * rows_per_block, last = first + rows_per_block < rows ? first + rows_per_block : rows;
  for (int64_t row = first + threadIdx.x / LPR; row < last; row += RB_THREADS / LPR) {
    if (mask != nullptr && mask[row] == 0) continue;      // (the whole row's lanes go together: no lane waits for one that left)
    float v[VPL];
    load_logits<T, VPL, WHOLE>(logits + row * stride, c0, n_experts, v);
    for (int j = sub; j < k; j += LPR) {
      const int64_t e = load_id(ids, ids_64, row * k + j);
      if (e >= 0 && e < n_experts) atomicAdd(&s_count[e], 1);
    }
    softmax_row<VPL, LPR>(v);
#pragma unroll
    for (int i = 0; i < VPL; ++i) sum[i] += v[i];
    valid += sub == 0;
  }
#pragma unroll
  for (int i = 0; i < VPL; ++i) {      // the rows of a wave: lanes with the same columns
#pragma unroll
    for (int o = LPR; o < 64; o <<= 1) sum[i] += __shfl_xor(sum[i], o);
    if (lane < LPR) s_sum[wave][c0 + i] = sum[i];
  }
  if (valid > 0) atomicAdd(&s_count[n_experts], valid);
  __syncthreads();
  for (int e = threadIdx.x; e < n_experts; e += RB_THREADS) {
    float t = 0.f;
#pragma unroll
    for (int w = 0; w < RB_THREADS / 64; ++w) t += s_sum[w][e];
    ws.psum[(int64_t)blockIdx.x * n_experts + e] = t;
    ws.counts[(int64_t)blockIdx.x * n_experts + e] = s_count[e];
  }
  if (threadIdx.x == 0) ws.valid[blockIdx.x] = s_count[n_experts];
}

// one workgroup: the partials in the order of the workgroups, sums of whole numbers and of doubles
__global__ void __launch_bounds__(1024)
    balance_finish_kernel(int n_blocks, int n_experts, int k, BalancePartials ws, float *__restrict__ loss, int64_t *__restrict__ counts,
                          float *__restrict__ pull) {
  __shared__ double s_p[1024];
  __shared__ int64_t s_c[1024];
  __shared__ int64_t s_valid;
  const int t = threadIdx.x;
  s_c[t] = 0;
  if (t < n_blocks) s_c[t] = ws.valid[t];
  __syncthreads();
  if (t < 64) {
    int64_t v = 0;
    for (int b = t; b < n_blocks; b += 64) v += s_c[b];
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    if (t == 0) s_valid = v;
  }
  __syncthreads();
  const int64_t valid = s_valid;
  // `width` >= n_experts threads read one workgroup's row, 1024 / width rows at a time; the rows' sums meet in LDS
  int width = 1;
  while (width < n_experts) width <<= 1;
  const int e = t & (width - 1), slice = t / width, slices = 1024 / width;
  double p = 0.0;
  int64_t c = 0;
  if (e < n_experts) {
    int b = slice;
    for (; b + 15 * slices < n_blocks; b += 16 * slices) {      // sixteen loads of each on their way together: what this kernel waits for
      float tp[16];
      int tc[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) { tp[i] = ws.psum[(b + i * slices) * n_experts + e]; tc[i] = ws.counts[(b + i * slices) * n_experts + e]; }
#pragma unroll
      for (int i = 0; i < 16; ++i) { p += (double)tp[i]; c += tc[i]; }
    }
    for (; b < n_blocks; b += slices) { p += (double)ws.psum[b * n_experts + e]; c += ws.counts[b * n_experts + e]; }
  }
  s_p[t] = p; s_c[t] = c;
  __syncthreads();
  for (int s = slices >> 1; s > 0; s >>= 1) {
    if (slice < s) { s_p[t] += s_p[t + s * width]; s_c[t] += s_c[t + s * width]; }
    __syncthreads();
  }
  p = 0.0;
  if (t < n_experts) {
    c = s_c[t];
    const double v = valid > 0 ? (double)valid : 1.0, kv = (double)k * v;
    counts[t] = c;
    pull[t] = valid > 0 ? (float)(((double)n_experts * (double)c - kv) / (kv * v)) : 0.f;
    p = (double)n_experts * ((double)c / kv) * (s_p[t] / v);
  }
  __syncthreads();
  s_p[t] = p;
  __syncthreads();
  for (int s = 512; s > 0; s >>= 1) {
    if (t < s) s_p[t] += s_p[t + s];
    __syncthreads();
  }
  if (t == 0) loss[0] = (float)s_p[0];
}

template <typename T, int VPL, int LPR, bool WHOLE>
__global__ void __launch_bounds__(256)
    balance_bwd_kernel(int64_t rows, int n_experts, const T *__restrict__ logits, int64_t stride, const uint8_t *__restrict__ mask,
                       const float *__restrict__ pull, const float *__restrict__ v_loss, T *__restrict__ v_logits) {
  const int sub = threadIdx.x % LPR, c0 = sub * VPL;
  const float vl = v_loss[0];
  float c[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) c[i] = c0 + i < n_experts ? pull[c0 + i] : 0.f;
  for (int64_t row = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR; row < rows; row += (int64_t)gridDim.x * (256 / LPR)) {
    T *out = v_logits + row * n_experts;
    float v[VPL];
    const bool valid = mask == nullptr || mask[row] != 0;
    if (valid) {
      load_logits<T, VPL, WHOLE>(logits + row * stride, c0, n_experts, v);
      softmax_row<VPL, LPR>(v);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i) dot = fmaf(v[i], c[i], dot);
      dot = over_row<LPR>(dot, [](float a, float b) { return a + b; });
#pragma unroll
      for (int i = 0; i < VPL; ++i) v[i] = vl * (v[i] * (c[i] - dot));
    } else {
#pragma unroll
      for (int i = 0; i < VPL; ++i) v[i] = 0.f;
    }
    constexpr int W = 16 / sizeof(T) < VPL ? 16 / sizeof(T) : VPL;
#pragma unroll
    for (int i = 0; i < VPL; i += W) {
      if (c0 + i + W <= n_experts) {
        T t[W];
#pragma unroll
        for (int j = 0; j < W; ++j) t[j] = (T)v[i + j];
        store_piece<T, W>(out + c0 + i, t);
      } else if (!WHOLE) {
#pragma unroll
        for (int j = 0; j < W; ++j)
          if (c0 + i + j < n_experts) out[c0 + i + j] = (T)v[i + j];
      }
    }
  }
}

// lanes of a row and logits of a lane: 8 logits a lane (two 16-byte accesses at 32 bits), the fewest lanes that hold the row
#define GSDF_BALANCE_SHAPE(n_experts, whole, ...)                                                                              \
  if (whole) { constexpr bool WHOLE = true; GSDF_BALANCE_LANES(n_experts, __VA_ARGS__) }                                       \
  else { constexpr bool WHOLE = false; GSDF_BALANCE_LANES(n_experts, __VA_ARGS__) }
#define GSDF_BALANCE_LANES(n_experts, ...)                                                       \
  if (n_experts <= 8) { constexpr int VPL = 8, LPR = 1; __VA_ARGS__; }                           \
  else if (n_experts <= 16) { constexpr int VPL = 8, LPR = 2; __VA_ARGS__; }                     \
  else if (n_experts <= 32) { constexpr int VPL = 8, LPR = 4; __VA_ARGS__; }                     \
  else if (n_experts <= 64) { constexpr int VPL = 8, LPR = 8; __VA_ARGS__; }                     \
  else if (n_experts <= 128) { constexpr int VPL = 8, LPR = 16; __VA_ARGS__; }                   \
  else if (n_experts <= 256) { constexpr int VPL = 8, LPR = 32; __VA_ARGS__; }                   \
  else if (n_experts <= 512) { constexpr int VPL = 8, LPR = 64; __VA_ARGS__; }                   \
  else { constexpr int VPL = 16, LPR = 64; __VA_ARGS__; }

static int lanes_per_row(int n_experts) {
  int l = 1;
  while (l * 8 < n_experts && l < 64) l <<= 1;
  return l;
}
static int64_t balance_blocks(int64_t rows, int n_experts) {
  const int64_t b = ceil_div(rows, RB_THREADS / lanes_per_row(n_experts));
  return b < 1 ? 1 : (b < RB_MAX_BLOCKS ? b : RB_MAX_BLOCKS);
}

}  // namespace gsdf

extern "C" size_t gsdf_router_balance_ws_bytes(int64_t rows, int n_experts) {
  if (rows < 0 || n_experts < 1 || n_experts > gsdf::RB_MAX_EXPERTS) return 0;
  return (size_t)gsdf::balance_blocks(rows, n_experts) * ((size_t)n_experts * 8 + 4);
}

extern "C" int gsdf_router_balance_fwd(int64_t rows, int n_experts, int k, int dtype, const void *logits, int64_t stride, const void *ids,
                                       int ids_64, const uint8_t *mask, float *loss, int64_t *counts, float *pull, void *ws,
                                       gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  GSDF_REQUIRE(rows >= 0 && rows < (1ll << 31), "router_balance: %lld rows outside [0, 2^31)", (long long)rows);
  GSDF_REQUIRE(n_experts >= 1 && n_experts <= RB_MAX_EXPERTS, "router_balance: %d experts outside [1, %d]", n_experts, RB_MAX_EXPERTS);
  GSDF_REQUIRE(k >= 1 && k <= n_experts, "router_balance: %d choices of %d experts", k, n_experts);
  GSDF_REQUIRE(known_dtype(dtype), "router_balance: unknown element type %d", dtype);
  GSDF_REQUIRE(loss != nullptr && counts != nullptr && pull != nullptr && ws != nullptr, "router_balance: outputs and workspace are required");
  GSDF_REQUIRE(rows == 0 || (logits != nullptr && ids != nullptr), "router_balance: logits and ids are required");
  GSDF_REQUIRE(rows <= 1 || stride >= 0, "router_balance: row stride %lld", (long long)stride);
  GSDF_TIMED("gsdf_router_balance_fwd");
  const int64_t blocks = balance_blocks(rows, n_experts), per_block = ceil_div(rows, blocks);
  BalancePartials part;
  part.psum = (float *)ws;
  part.counts = (int *)(part.psum + blocks * n_experts);
  part.valid = part.counts + blocks * n_experts;
  GSDF_BY_DTYPE(dtype, {
    const bool whole = n_experts % (int)(16 / sizeof(T)) == 0;
    GSDF_BALANCE_SHAPE(n_experts, whole, (balance_partial_kernel<T, VPL, LPR, WHOLE><<<(unsigned)blocks, RB_THREADS, 0, stream>>>(
        rows, per_block, n_experts, k, (const T *)logits, stride, ids, ids_64, mask, part)))
  });
  balance_finish_kernel<<<1, 1024, 0, stream>>>((int)blocks, n_experts, k, part, loss, counts, pull);
  GSDF_CHECK_LAUNCH("router_balance_fwd");
  return GSDF_OK;
}

extern "C" int gsdf_router_balance_bwd(int64_t rows, int n_experts, int dtype, const void *logits, int64_t stride, const uint8_t *mask,
                                       const float *pull, const float *v_loss, void *v_logits, gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  GSDF_REQUIRE(rows >= 0 && rows < (1ll << 31), "router_balance_bwd: %lld rows outside [0, 2^31)", (long long)rows);
  GSDF_REQUIRE(n_experts >= 1 && n_experts <= RB_MAX_EXPERTS, "router_balance_bwd: %d experts outside [1, %d]", n_experts, RB_MAX_EXPERTS);
  GSDF_REQUIRE(known_dtype(dtype), "router_balance_bwd: unknown element type %d", dtype);
  if (rows == 0) return GSDF_OK;
  GSDF_REQUIRE(logits != nullptr && pull != nullptr && v_loss != nullptr && v_logits != nullptr, "router_balance_bwd: a required pointer is NULL");
  GSDF_REQUIRE(rows == 1 || stride >= 0, "router_balance_bwd: row stride %lld", (long long)stride);
  GSDF_TIMED("gsdf_router_balance_bwd");
  const int64_t want = ceil_div(rows, 256 / lanes_per_row(n_experts));
  const unsigned grid = (unsigned)(want < 8192 ? want : 8192);
  GSDF_BY_DTYPE(dtype, {
    const bool whole = n_experts % (int)(16 / sizeof(T)) == 0;
    GSDF_BALANCE_SHAPE(n_experts, whole, (balance_bwd_kernel<T, VPL, LPR, WHOLE><<<grid, 256, 0, stream>>>(
        rows, n_experts, (const T *)logits, stride, mask, pull, v_loss, (T *)v_logits)))
  });
  GSDF_CHECK_LAUNCH("router_balance_bwd");
  return GSDF_OK;
}
