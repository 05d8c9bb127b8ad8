// lowrank_kernels.h — the products of the low-rank adapters; lowrank_f32.hip, lowrank_f16.hip and lowrank_bf16.hip compile it for their element type.
//
// The adapters' weights are small beside x, base and y, so the operator is bound by the bytes of its rows.  The rows are put in the order of
// their adapters first (`lowrank_plan_*`): a range of 16 to 64 rows then has one adapter, and each product is tiles of matrix instructions whose
// operands come from global memory in the layout that the instruction wants:
//   shrink   contracts a row's elements (x with A, dy with B^T).  The order of the contraction is free: an instruction's lanes take 64 neighbouring bytes of
//            each of 16 rows.  The waves of a workgroup split the row and meet in LDS.
//   expand   contracts ranks (h with B, dh with A^T): the instruction's rows are columns of y, permuted so that a lane holds 16 neighbouring bytes and four lanes 64.
//   outer    contracts rows (dh with x, h with dy): a lane holds 8 rows x 16 bytes and turns them in registers.
// h and dh are held in 32 bits.  In front of 16-bit instructions they are split into three parts of the weights' type, which hold all 24 bits between
// them: the instructions are not the bound.
//
// Measured beside the bytes that a product cannot do without (a copy of 1 GiB moves 5.2 TB/s):
//   8192 rows, 4096 -> 4096, rank 16, bf16, dropout: shrink 22 us (64 MB, 3.0 TB/s: the generator's products are half of it; without dropout 18, 3.8 TB/s), expand 33 us
//     (128 MB, 4.1 TB/s), dx 27 us (64 MB and the generator again), outer 32 us (128 MB, 4.2 TB/s), the sum of its chunks 4 us, plan and layout 11 to 12 us (latency)
//   6007 rows, 4096 -> 4096, rank 64, bf16: shrink 18.5 us (47 MB, and 0.13 GB of A from the L2: its ranges are 24 rows), expand 28.9 us (98 MB, 3.4 TB/s, and 0.12 GB of B from the L2), plan and
//     layout 10.5 us
//   300000 rows, 64 -> 64, rank 8, 32 bits: both products 53 us forward (230 MB, 4.3 TB/s), 43 backward (154 MB, 3.6 TB/s), outer 45 us (173 MB, 3.8 TB/s), sum 5.3 us
#pragma once
#include <type_traits>

#include "lowrank.h"

namespace gsdf {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ---- pieces of rows ---------------------------------------------------------------------------------------------------------------------------
// 16 bytes of a row in registers.  Fragments stay whole vectors: as single 16-bit values they would be taken apart, waited for and put together again
// wherever two paths of the code meet.
template <typename T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(N)));
};
template <typename T>
__device__ __forceinline__ typename Vec<T>::vec load_vec(const T *__restrict__ p) {
  return *reinterpret_cast<const typename Piece<T, Vec<T>::N>::any *>(p);
}
// v moved down by n elements (0 .. N), zeros behind
template <typename T>
__device__ __forceinline__ typename Vec<T>::vec move_down(typename Vec<T>::vec v, int n) {
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  u64x2 u = __builtin_bit_cast(u64x2, v);
  const int bits = n * 8 * (int)sizeof(T), in = bits & 63;
  const uint64_t low = bits >= 128 ? 0 : bits >= 64 ? u[1] : u[0], high = bits >= 64 ? 0 : u[1];
  u[0] = (low >> in) | ((high << 1) << (63 - in));
  u[1] = high >> in;
  return __builtin_bit_cast(typename Vec<T>::vec, u);
}
// the elements of a row from k on, 0 behind its end: the row's last 16 bytes, moved down (one element after the other took a kernel from 8 to 18 us)
template <typename T>
__device__ __forceinline__ typename Vec<T>::vec load_vec_end(const T *__restrict__ row, int k, int width) {
  constexpr int N = Vec<T>::N;
  if (width >= N) {
    const int at = k + N <= width ? k : width - N, by = k - at;
    return move_down<T>(load_vec<T>(row + at), by < N ? by : N);
  }
  typename Vec<T>::vec v;      // a row of less than 16 bytes
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = row[k + i < width ? k + i : 0];
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = k + i < width ? v[i] : (T)0.f;
  return v;
}
// the first `valid` (less than all) elements of v: by halves
template <typename T>
__device__ __forceinline__ void store_vec_end(T *p, int valid, typename Vec<T>::vec v) {
  constexpr int N = Vec<T>::N;
  if (N == 8 && (valid & 4)) {
    typename Piece<T, 4>::vec t = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<typename Piece<T, 4>::any *>(p) = t;
    v = move_down<T>(v, 4);
    p += 4;
  }
  if (valid & 2) {
    typename Piece<T, 2>::vec t = {v[0], v[1]};
    *reinterpret_cast<typename Piece<T, 2>::any *>(p) = t;
    v = move_down<T>(v, 2);
    p += 2;
  }
  if (valid & 1) p[0] = v[0];
}
template <typename T>
__device__ __forceinline__ typename Vec<T>::vec zero_unless(bool keep, typename Vec<T>::vec v) {
  u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = keep ? u[i] : 0u;
  return __builtin_bit_cast(typename Vec<T>::vec, u);
}
// N (4, or 16 bytes) neighbouring results, `valid` of them
template <typename T, int N>
__device__ __forceinline__ void store_some(T *__restrict__ p, int valid, const float (&v)[N]) {
  if constexpr (N == Vec<T>::N) {
    typename Vec<T>::vec o;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = (T)v[i];
    if (valid >= N) *reinterpret_cast<typename Piece<T, N>::any *>(p) = o;
    else if (valid > 0) store_vec_end<T>(p, valid, o);
  } else {
    if (valid >= N) {
#pragma unroll
      for (int i = 0; i < N; i += 4) {
        const T t[4] = {(T)v[i], (T)v[i + 1], (T)v[i + 2], (T)v[i + 3]};
        store_piece<T, 4>(p + i, t);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i < valid) p[i] = (T)v[i];
    }
  }
}
// all ones in the half word (16-bit elements) of each element that stays: sat(bits - (threshold - 1)) is 0 exactly below the threshold
__device__ __forceinline__ uint32_t keep_mask16(const Dropout &d, uint32_t w) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  const unsigned short below = (unsigned short)(d.threshold - 1u);
  u16x2 t = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, w), u16x2{below, below});
  t = __builtin_elementwise_min(t, u16x2{1, 1});
  return __builtin_bit_cast(uint32_t, (u16x2)(u16x2{0, 0} - t));
}
// zeros where dropped: the 16 bytes of `row` from column `col` on; the survivors' factor goes into the sums
template <typename V>
__device__ __forceinline__ V drop8_16(const Dropout &d, uint32_t row, int col, V v) {
  uint32_t w[4];
  dropout_bits(d, (uint32_t)col >> 3, row, w);
  u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] &= keep_mask16(d, w[i]);
  return __builtin_bit_cast(V, u);
}
__device__ __forceinline__ void drop_vec(const Dropout &d, uint32_t row, int col, bf16x8 &v) { v = drop8_16(d, row, col, v); }
__device__ __forceinline__ void drop_vec(const Dropout &d, uint32_t row, int col, f16x8 &v) { v = drop8_16(d, row, col, v); }
__device__ __forceinline__ void drop_vec(const Dropout &d, uint32_t row, int col, f32x4 &v) {      // half a block
  uint32_t w[4];
  dropout_bits(d, (uint32_t)col >> 3, row, w);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = ((i & 1) ? (((col & 4) ? w[2 + i / 2] : w[i / 2]) >> 16) : (((col & 4) ? w[2 + i / 2] : w[i / 2]) & 0xFFFFu)) >= d.threshold ? v[i] : 0.f;
}

// acc += a b over the 16 bytes of each lane: one 16-bit instruction, or four of 32 bits (any order of the contraction is as good)
__device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 acc) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0); }
__device__ __forceinline__ f32x4 mma(f32x4 a, f32x4 b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 4; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
  return acc;
}
// v = hi + mid + lo: eight bits each, cut off and not rounded, so that no part of a finite number is infinite (bf16); eleven (fp16).  An infinity leaves nothing.
__device__ __forceinline__ void split(float v, bf16_t &hi, bf16_t &mid, bf16_t &lo) {
  auto top = [](float t) { return __float_as_uint(t) & 0xFFFF0000u; };
  auto part = [](uint32_t t) { return __builtin_bit_cast(bf16_t, (unsigned short)(t >> 16)); };
  const uint32_t h = top(v);
  const float r = fabsf(v) == INFINITY ? 0.f : v - __uint_as_float(h);
  const uint32_t m = top(r);
  hi = part(h); mid = part(m); lo = part(top(r - __uint_as_float(m)));
}
__device__ __forceinline__ void split(float v, f16_t &hi, f16_t &mid, f16_t &lo) {
  hi = (f16_t)v;
  const float r = fabsf((float)hi) == INFINITY ? 0.f : v - (float)hi;
  mid = (f16_t)r;
  lo = (f16_t)(r - (float)mid);
}
// In front of fp16 parts: a power of two that brings `largest` into [2^14, 2^15), where neither it nor what is 2^38 times smaller runs over or vanishes;
// times `scale_back` of it everything is as before.  Infinities and what is all zeros stay.
__device__ __forceinline__ float scale_up(float largest) {
  const int e = (__float_as_int(largest) >> 23) & 255, up = 268 - e;
  return e == 0 || e == 255 ? 1.f : __int_as_float((up < 253 ? up : 253) << 23);
}
__device__ __forceinline__ float scale_back(float scale) { return __int_as_float((254 << 23) - __float_as_int(scale)); }

// ---- shrink: H[place][j] = factor sum_k drop(x)[row][k] W[g][j][k] -------------------------------------------------------------------------
// A workgroup of `split` waves has a range of rows and its waves take the steps of 128 bytes in turn (one wave: four ranges a workgroup).
// RT: tiles of 16 ranks.  H: [places][16 RT] (for `expand`; zeros behind the rank) and / or HT: [rank][ht_ld] (for `outer`).
struct ShrinkArgs {
  const void *x, *w;
  int64_t x_stride;               // elements between rows
  int width, rank, split;         // w: fragments (PackArgs)
  const float *scales;            // per adapter, or null
  float factor;
  float *h, *ht;
  int64_t ht_ld;
  Dropout drop;
  Plan plan;
};
template <typename T, int RT, int TT, bool DROP, bool RAGGED>      // TT: tiles of 16 rows in the range
__device__ __forceinline__ void shrink_sums(const ShrinkArgs &q, int4 range, int which, int part, f32x4 (&acc)[RT][TT]) {
  typedef typename Vec<T>::vec V;
  constexpr int N = Vec<T>::N, STEP = 8 * N;
  const int lane = threadIdx.x & 63, c = lane & 15, quad = lane >> 4;
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < TT; ++t) acc[r][t] = f32x4{0.f, 0.f, 0.f, 0.f};
  const T *px[TT];
  uint32_t row[TT];
#pragma unroll
  for (int t = 0; t < TT; ++t) {      // a place behind the range reads its last row: its sums are not written
    const int i = t * 16 + c;
    row[t] = (uint32_t)q.plan.order[range.y + (i < range.z ? i : range.z - 1)];
    px[t] = (const T *)q.x + (int64_t)row[t] * q.x_stride;
  }
  const V *pw = (const V *)q.w + (int64_t)range.x * ((q.width + STEP - 1) / STEP) * RT * 128 + lane;
  // Ranges begin at different steps: rows of 2^n bytes at the same step would all ask the same memory channels (19 against 15 us for 64 MB).
  const int full = q.width / STEP, turn = full > 0 ? (int)((unsigned)which % (unsigned)full) : 0;
  auto place = [&](int step) { return step + turn < full ? step + turn : step + turn - full; };
  auto load = [&](int step, V (&xs)[TT][2], V (&ws)[RT][2]) {
    const int k = step * STEP + quad * N;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int t = 0; t < TT; ++t) xs[t][i] = load_vec<T>(px[t] + k + i * 4 * N);
#pragma unroll
      for (int r = 0; r < RT; ++r) ws[r][i] = pw[((int64_t)step * RT + r) * 128 + i * 64];
    }
  };
  auto add = [&](int step, V (&xs)[TT][2], V (&ws)[RT][2]) {
    if (DROP) {
      const int k = step * STEP + quad * N;
#pragma unroll
      for (int t = 0; t < TT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) drop_vec(q.drop, row[t], k + i * 4 * N, xs[t][i]);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < TT; ++t) acc[r][t] = mma(ws[r][i], xs[t][i], acc[r][t]);
  };
  int s = part;
  auto steps = [&](auto ahead) {      // steps whose loads are on their way together
    constexpr int AHEAD = decltype(ahead)::value;
    for (; s + (AHEAD - 1) * q.split < full; s += AHEAD * q.split) {
      V xs[AHEAD][TT][2], ws[AHEAD][RT][2];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) load(place(s + u * q.split), xs[u], ws[u]);
      __builtin_amdgcn_sched_barrier(0);      // (left alone, the compiler saves registers and lets two loads go at a time)
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) add(place(s + u * q.split), xs[u], ws[u]);
    }
  };
  if (RT == 1 && TT < 3) steps(std::integral_constant<int, 4>{});
  if (RT <= 4) steps(std::integral_constant<int, 2>{});
  steps(std::integral_constant<int, 1>{});
  if (RAGGED && full * STEP < q.width && part == full % q.split) {      // the rows' last elements (RAGGED may be for y's width alone)
    const int k = full * STEP + quad * N;
    V xs[TT][2], ws[RT][2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int r = 0; r < RT; ++r) ws[r][i] = pw[((int64_t)full * RT + r) * 128 + i * 64];
#pragma unroll
      for (int t = 0; t < TT; ++t) xs[t][i] = load_vec_end<T>(px[t], k + i * 4 * N, q.width);
    }
    add(full, xs, ws);
  }
}
template <typename T, int RT, int TT, bool DROP, bool RAGGED>
__device__ __forceinline__ void shrink_range(const ShrinkArgs &q, int4 range, int which, int part, f32x4 *s_sum) {
  constexpr int RR = RT < 2 ? RT : 2;      // tiles of ranks that meet in LDS at a time
  const int lane = threadIdx.x & 63, c = lane & 15, quad = lane >> 4;
  f32x4 acc[RT][TT];
  shrink_sums<T, RT, TT, DROP, RAGGED>(q, range, which, part, acc);
  const float f = q.factor * (q.scales != nullptr ? q.scales[range.x] : 1.f);
  auto put = [&](int r, int t, f32x4 v) {
    const int i0 = t * 16 + c, j0 = r * 16 + quad * 4;
    if (i0 >= range.z) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = j0 + i < q.rank ? v[i] * f : 0.f;
    if (q.h != nullptr) *reinterpret_cast<f32x4 *>(q.h + (int64_t)(range.y + i0) * (16 * RT) + j0) = v;
    if (q.ht != nullptr) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (j0 + i < q.rank) q.ht[(int64_t)(j0 + i) * q.ht_ld + range.y + i0] = v[i];
    }
  };
  if (q.split == 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) put(r, t, acc[r][t]);
    return;
  }
#pragma unroll
  for (int r0 = 0; r0 < RT; r0 += RR) {      // the waves share the adding and the writing
    if (r0 > 0) __syncthreads();
#pragma unroll
    for (int r = 0; r < RR; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) s_sum[(part * RR * TT + r * TT + t) * 64 + lane] = acc[r0 + r][t];
    __syncthreads();
    for (int i = part; i < RR * TT; i += q.split) {
      f32x4 v = s_sum[i * 64 + lane];
      for (int w = 1; w < q.split; ++w) v += s_sum[(w * RR * TT + i) * 64 + lane];
      put(r0 + i / TT, i % TT, v);
    }
  }
}
template <typename T, int RT, bool DROP, bool RAGGED>      // RAGGED: the width is no multiple of a step
__global__ void __launch_bounds__(512) lowrank_shrink_kernel(ShrinkArgs q) {
  extern __shared__ f32x4 s_sum[];      // [split][min(RT, 2)][3][64]
  const int wave = threadIdx.x >> 6, which = q.split == 1 ? blockIdx.x * 4 + wave : blockIdx.x, part = q.split == 1 ? 0 : wave;
  if (which >= q.plan.n_ranges) return;
  const int4 range = q.plan.range[which];
  if (range.z == 0 || range.x == q.plan.n_adapters) return;
  if (DROP) dropout_counter(q.drop);
  if (range.z > 32) shrink_range<T, RT, 3, DROP, RAGGED>(q, range, which, part, s_sum);
  else if (range.z > 16) shrink_range<T, RT, 2, DROP, RAGGED>(q, range, which, part, s_sum);
  else shrink_range<T, RT, 1, DROP, RAGGED>(q, range, which, part, s_sum);
}

// ---- expand: y[row][n] = base[row][n] + sum_j H[place][j] W[g][n][j] -------------------------------------------------------------------------
// A wave takes 64 columns of 16, 32 or 64 rows (the weights come from the L2 once for all of them; ranks above 32 stop at 32 rows, whose h leaves room for
// more waves: rank 64, 6007 rows of 8 KB 28.9 us against 32.6 with 64 rows).  Loads of the next columns are on their way while the last are stored.  The instruction's rows are columns of y in the order that leaves a lane pieces of 16 neighbouring bytes, four lanes 64 of
// them; lanes of rows c and c + 8 then change pieces, so that an access covers 128 bytes of each of 8 rows instead of 64 of 16 (30 against 34 us for
// a plain copy of 8192 rows of 8 KB in this manner).
struct ExpandArgs {
  const float *h;
  const void *w, *base;
  void *y;
  int64_t w_group, base_stride, y_stride;
  int width, w_ld, rank, parts;      // parts: waves that share a range's columns
  Dropout drop;      // on the result (dx), DROP only
  Plan plan;
};
// lanes c and c + 8 of each 16: a of the lower and b of the upper one stay, the lower one's b and the upper one's a change places.  Its own inverse.
template <typename V>
__device__ __forceinline__ void change_halves(V &a_, V &b_, bool upper) {
  u32x4 a = __builtin_bit_cast(u32x4, a_), b = __builtin_bit_cast(u32x4, b_);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t away = upper ? a[i] : b[i], come = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)away, 0x128, 0xF, 0xF, true);      // row_ror:8
    a[i] = upper ? come : a[i];
    b[i] = upper ? b[i] : come;
  }
  a_ = __builtin_bit_cast(V, a);
  b_ = __builtin_bit_cast(V, b);
}
// HERE: h comes from the wave's own sums, whose layout (a lane has 4 ranks of its row) an instruction takes as it is when the ranks of the contraction
// are told the weights in that order: four ranks' first and second parts a lane at 16 bits, and their third beside zeros.  Else it is read from H.  `source`
// fills f.
template <typename T, int RT, int TT, bool DROP, bool RAGGED, bool PAST, bool HERE, typename Source>
__device__ __forceinline__ void expand_range(const ExpandArgs &q, int4 range, int part, int turn, int chunks, Source source) {
  typedef typename Vec<T>::vec V;
  constexpr int N = Vec<T>::N, NP = 8 / N;      // pairs of pieces of a lane's 16 columns: piece p at column 4 N p + N quad of the 64
  constexpr bool WIDE = sizeof(T) == 4;
  const int lane = threadIdx.x & 63, c = lane & 15, quad = lane >> 4;
  const bool upper = c >= 8, idle = range.x == q.plan.n_adapters, add = q.base != nullptr;
  const int *order = q.plan.order + range.y;
  // access 2 t + half: rows 16 t + 8 half + c % 8, the lower lanes their first 64 bytes of a pair, the upper ones the second
  const T *base[2 * TT];
  T *y[2 * TT];
  const int column = (upper ? 4 * N : 0) + quad * N;
#pragma unroll
  for (int i = 0; i < 2 * TT; ++i) {
    const int at = i * 8 + (c & 7);
    const int64_t row = order[at < range.z ? at : range.z - 1];
    base[i] = (const T *)q.base + row * q.base_stride;
    y[i] = (T *)q.y + row * q.y_stride;
  }
  auto load_base = [&](int ch, V (&b)[2 * TT][NP]) {
#pragma unroll
    for (int i = 0; i < 2 * TT; ++i)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const int n = ch * 64 + p * 8 * N + column;
        if (!add) b[i][p] = V{};
        else if (!RAGGED || n + N <= q.width) b[i][p] = load_vec<T>(base[i] + n);
        else b[i][p] = load_vec_end<T>(base[i], n, q.width);
      }
  };
  auto store = [&](int i, int n, V v) {
    if (i * 8 + (c & 7) >= range.z) return;
    if (!RAGGED || n + N <= q.width) {
      if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<typename Piece<T, N>::any *>(y[i] + n));
      else *reinterpret_cast<typename Piece<T, N>::any *>(y[i] + n) = v;
    } else if (n < q.width) {
      store_vec_end<T>(y[i] + n, q.width - n, v);
    }
  };
  if (idle) {
    for (int i = part; i < chunks; i += q.parts) {
      const int ch = i + turn < chunks ? i + turn : i + turn - chunks;
      V b[2 * TT][NP];
      load_base(ch, b);
#pragma unroll
      for (int r = 0; r < 2 * TT; ++r)
#pragma unroll
        for (int p = 0; p < NP; ++p) store(r, ch * 64 + p * 8 * N + column, b[r][p]);
    }
    return;
  }
  const T *w = (const T *)q.w + range.x * q.w_group;
  // h of the lane's row as the instruction wants it.  16 bits: 8 ranks a lane, 32 an instruction, one for each part (a rank of at most 16: two parts in
  // one instruction).  32 bits: 4 ranks a lane, 16 a group of four instructions.
  constexpr bool BOTH = !WIDE && (HERE || RT == 1);      // first and second parts in one instruction
  constexpr int KB = WIDE || HERE ? RT : (RT == 1 ? 1 : RT / 2), FN = WIDE || HERE ? 1 : 2;
  auto rank_of = [&](int k) { return WIDE || HERE ? k * 16 + quad * 4 : (RT == 1 ? (quad & 1) * 8 : k * 32 + quad * 8); };
  V b[2 * TT][NP], u[4][KB];
  auto load_weights = [&](int ch) {
    const bool whole = !RAGGED || (ch * 64 + 64 <= q.width && (HERE || q.rank % N == 0));
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int col = ch * 64 + m * 4 / N * 4 * N + (c >> 2) * N + m * 4 % N + (c & 3);      // the column that this lane's weights belong to
      const T *pw = w + (int64_t)(whole || col < q.width ? col : q.width - 1) * q.w_ld;
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int j = rank_of(k);
        if constexpr (HERE && !WIDE) {      // (a rank that is a multiple of 4)
          const typename Piece<T, 4>::vec four = *reinterpret_cast<const typename Piece<T, 4>::any *>(pw + (j < q.rank ? j : 0));
          u[m][k] = V{four[0], four[1], four[2], four[3], four[0], four[1], four[2], four[3]};
        } else if (whole || HERE) {
          u[m][k] = load_vec<T>(pw + (j < q.rank ? j : 0));
        } else {
          u[m][k] = load_vec_end<T>(pw, j, q.rank);
        }
      }
    }
  };
  auto chunk_of = [&](int i) { return i + turn < chunks ? i + turn : i + turn - chunks; };
  load_weights(chunk_of(part));
  load_base(chunk_of(part), b);
  V hi[TT][KB], mid[TT][KB], lo[TT][KB];
  float back[TT];
  uint32_t row_of[TT];
  f32x4 f[TT][KB][FN];
  source(f);
#pragma unroll
  for (int t = 0; t < TT; ++t) {
    if (DROP) row_of[t] = (uint32_t)order[t * 16 + c < range.z ? t * 16 + c : range.z - 1];
    float largest = 0.f;
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int e = 0; e < FN; ++e) {
        if (DROP) f[t][k][e] *= q.drop.scale;
#pragma unroll
        for (int l = 0; l < 4; ++l) largest = fmaxf(largest, fabsf(f[t][k][e][l]));
      }
    float scale = 1.f;
    back[t] = 1.f;
    if (__is_same(T, f16_t)) {
      largest = fmaxf(largest, __shfl_xor(largest, 16));
      largest = fmaxf(largest, __shfl_xor(largest, 32));
      scale = scale_up(largest);
      back[t] = scale_back(scale);
    }
#pragma unroll
    for (int k = 0; k < KB; ++k)
#pragma unroll
      for (int e = 0; e < FN * 4; ++e) {
        const float v = f[t][k][e / 4][e % 4] * scale;
        if constexpr (WIDE) {
          hi[t][k][e] = v;
        } else {
          T h, m, l;
          split(v, h, m, l);
          if (HERE) {
            hi[t][k][e] = h; hi[t][k][e + 4] = m;
            lo[t][k][e] = l; lo[t][k][e + 4] = (T)0.f;
          } else {
            hi[t][k][e] = BOTH && quad >= 2 ? m : h;
            mid[t][k][e] = m;
            lo[t][k][e] = BOTH && quad >= 2 ? (T)0.f : l;
          }
        }
      }
  }
  for (int i = part; i < chunks; i += q.parts) {
    const int ch = chunk_of(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int k = 0; k < KB; ++k) u[m][k] = zero_unless<T>(rank_of(k) < q.rank, u[m][k]);
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      f32x4 acc[4];
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        acc[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < KB; ++k) {
          if (!WIDE) acc[m] = mma(u[m][k], lo[t][k], acc[m]);
          if (!WIDE && !BOTH) acc[m] = mma(u[m][k], mid[t][k], acc[m]);
          acc[m] = mma(u[m][k], hi[t][k], acc[m]);
        }
      }
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        V o[2];
        if (add) change_halves(b[2 * t][p], b[2 * t + 1][p], upper);      // now the pieces 2 p and 2 p + 1 of the lane's own row
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int piece = 2 * p + s, n = ch * 64 + piece * 4 * N + quad * N;
          float v[N];
#pragma unroll
          for (int e = 0; e < N; ++e) {
            v[e] = acc[(piece * N + e) / 4][e % 4] * back[t];
            if (add) v[e] += (float)b[2 * t + s][p][e];
          }
          if (DROP) {
            uint32_t bits[4];
            dropout_bits(q.drop, (uint32_t)n >> 3, row_of[t], bits);
            if (N == 4 && (n & 4)) { bits[0] = bits[2]; bits[1] = bits[3]; }
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = dropout_keeps(q.drop, bits, e) ? v[e] : 0.f;
          }
#pragma unroll
          for (int e = 0; e < N; ++e) o[s][e] = (T)v[e];
        }
        change_halves(o[0], o[1], upper);
        store(2 * t, ch * 64 + p * 8 * N + column, o[0]);
        store(2 * t + 1, ch * 64 + p * 8 * N + column, o[1]);
      }
    }
    if (i + q.parts < chunks) {
      load_weights(chunk_of(i + q.parts));
      load_base(chunk_of(i + q.parts), b);
    }
  }
}
// `source` of a range whose h is in memory: pieces of the lane's ranks
template <typename T, int RT, int TT>
struct FromMemory {
  static constexpr bool WIDE = sizeof(T) == 4;
  static constexpr int KB = WIDE ? RT : (RT == 1 ? 1 : RT / 2), FN = WIDE ? 1 : 2;
  const float *h;      // of the range
  int rows;
  __device__ __forceinline__ void operator()(f32x4 (&f)[TT][KB][FN]) const {
    const int c = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4;
#pragma unroll
    for (int t = 0; t < TT; ++t) {
      const float *p = h + (int64_t)(t * 16 + c < rows ? t * 16 + c : rows - 1) * (16 * RT) + (WIDE ? quad * 4 : RT == 1 ? (quad & 1) * 8 : quad * 8);
#pragma unroll
      for (int k = 0; k < KB; ++k)
#pragma unroll
        for (int e = 0; e < FN; ++e) f[t][k][e] = *reinterpret_cast<const f32x4 *>(p + k * (16 * FN) + e * 4);
    }
  }
};
// RAGGED: the width is no multiple of 64 or the rank none of a lane's piece; PAST: y goes past the caches
template <typename T, int RT, bool DROP, bool RAGGED, bool PAST>
__global__ void __launch_bounds__(256, RAGGED || RT == 8 ? 1 : 2) lowrank_expand_kernel(ExpandArgs q) {
  const unsigned id = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6)), which = id / (unsigned)q.parts;
  if (which >= (unsigned)q.plan.n_wide) return;
  const int4 range = q.plan.wide[which];
  if (range.z == 0 || (range.x == q.plan.n_adapters && q.base == q.y)) return;      // (in place a row without an adapter is not touched)
  const int chunks = (q.width + 63) / 64, part = (int)(id % (unsigned)q.parts);
  const int turn = (int)(which % (unsigned)chunks);      // ranges begin at different columns: not all at the same memory channels
  if (DROP) dropout_counter(q.drop);
  const float *h = q.h + (int64_t)range.y * (16 * RT);
  if constexpr (RT <= 2) {      // (a wider rank's h would leave room for two waves a SIMD)
    if (range.z > 32) {
      expand_range<T, RT, 4, DROP, RAGGED, PAST, false>(q, range, part, turn, chunks, FromMemory<T, RT, 4>{h, range.z});
      return;
    }
  }
  if (range.z > 16) expand_range<T, RT, 2, DROP, RAGGED, PAST, false>(q, range, part, turn, chunks, FromMemory<T, RT, 2>{h, range.z});
  else expand_range<T, RT, 1, DROP, RAGGED, PAST, false>(q, range, part, turn, chunks, FromMemory<T, RT, 1>{h, range.z});
}

// ---- both: many rows leave no unit idle when a wave takes a range through `shrink` and `expand` by itself; h stays in its registers -------------
// Workgroups of one wave: a range is begun as soon as another ends (four waves a workgroup: 55.2 us against 53.7; ranges of 16 rows instead of 32: 61).
template <typename T, int RT, int TT, bool DROP_X, bool DROP_Y, bool RAGGED, bool PAST>
__device__ __forceinline__ void both_range(const ShrinkArgs &s, const ExpandArgs &q, int4 range, int which) {
  const int c = threadIdx.x & 15, quad = (threadIdx.x & 63) >> 4;
  auto source = [&](f32x4 (&f)[TT][RT][1]) {
    f32x4 acc[RT][TT];
    shrink_sums<T, RT, TT, DROP_X, RAGGED>(s, range, which, 0, acc);
    const float factor = s.factor * (s.scales != nullptr ? s.scales[range.x] : 1.f);
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < TT; ++t) {
        const int i0 = t * 16 + c, j0 = r * 16 + quad * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[t][r][0][i] = j0 + i < s.rank ? acc[r][t][i] * factor : 0.f;
        if (s.ht != nullptr && i0 < range.z) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + i < s.rank) s.ht[(int64_t)(j0 + i) * s.ht_ld + range.y + i0] = f[t][r][0][i];
        }
      }
  };
  expand_range<T, RT, TT, DROP_Y, RAGGED, PAST, true>(q, range, 0, which % ((q.width + 63) / 64), (q.width + 63) / 64, source);
}
template <typename T, int RT, bool DROP_X, bool DROP_Y, bool RAGGED, bool PAST>
__global__ void __launch_bounds__(64) lowrank_both_kernel(ShrinkArgs s, ExpandArgs q) {
  const int which = (int)__builtin_amdgcn_readfirstlane(blockIdx.x);
  if (which >= q.plan.n_wide) return;
  const int4 range = q.plan.wide[which];
  if (range.z == 0 || (range.x == q.plan.n_adapters && q.base == q.y)) return;
  if (DROP_X) dropout_counter(s.drop);
  if (DROP_Y) dropout_counter(q.drop);
  if (range.z > 16) both_range<T, RT, 2, DROP_X, DROP_Y, RAGGED, PAST>(s, q, range, which);
  else both_range<T, RT, 1, DROP_X, DROP_Y, RAGGED, PAST>(s, q, range, which);
}

// ---- outer: sum over an adapter's rows of UT[j][place] V[row][c] ----------------------------------------------------------------------------
// A workgroup of 8 waves owns a chunk of rows and 16 lanes x 16 bytes of columns; its waves take 32 rows in turn and meet in LDS.  Chunks of 512 rows instead of
// 1024 make more workgroups of few columns, but more partial sums: 45 us against 44 for 300000 rows of 64 columns, 33 against 31 for 8192 rows of 4096.
struct OuterSide {
  const float *ut;      // [..][ut_ld]
  const void *v;
  int64_t v_stride;
  int width, drop;
  int columns_first;    // result [g][c][j] (B) instead of [g][j][c] (A)
  void *out;
  float *part;          // [slots][16 RT ranks][width] or [slots][width][16 RT]
};
struct OuterArgs {
  OuterSide side[2];
  int64_t ut_ld;
  int rank, rank_padded, blocks0, blocks;      // column blocks of side 0, of both
  Dropout drop;
  Plan plan;
};
// element e of 8 rows as one fragment
__device__ __forceinline__ u32x4 column_of(const u32x4 (&v)[8], int e) {
  u32x4 o;
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __builtin_amdgcn_perm(v[2 * i + 1][e >> 1], v[2 * i][e >> 1], (e & 1) ? 0x07060302u : 0x05040100u);
  return o;
}
template <typename T, int RT, bool RAGGED>      // RAGGED: a width is no multiple of COLS
__global__ void __launch_bounds__(LR_OUTER_THREADS) lowrank_outer_kernel(OuterArgs q) {
  typedef typename Vec<T>::vec V;
  constexpr int VE = Vec<T>::N, COLS = 16 * VE;      // elements of a lane's piece, columns of a workgroup
  __shared__ f32x4 s_sum[4][VE][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, quad = lane >> 4;
  const int block = blockIdx.x % q.blocks;
  const int4 chunk = q.plan.chunk[blockIdx.x / q.blocks];
  if (chunk.x < 0) return;
  const bool second = block >= q.blocks0;
  const OuterSide &s = q.side[second];
  const int col0 = (block - (second ? q.blocks0 : 0)) * COLS, col = col0 + c * VE, valid = s.width - col;
  const int rank0 = blockIdx.y * 64;
  const bool drop = s.drop != 0;
  if (drop) dropout_counter(q.drop);
  f32x4 acc[RT][VE];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[r][e] = f32x4{0.f, 0.f, 0.f, 0.f};
  // fp16: the power of two in front of the split of rank c of a tile, and of its sums until the waves meet.  One for each rank: an infinity, or values that are far
  // larger, are nothing to the others.  It comes down where a step has more (with room for four times as much).
  constexpr bool HALF = __is_same(T, f16_t);
  float scale[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) scale[r] = __int_as_float(253 << 23);
  auto times_of_ranks = [&](f32x4 (&v)[VE], float f) {      // a lane's sums are of ranks quad * 4 ..
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float t = __shfl(f, quad * 4 + i);
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e][i] *= t;
    }
  };
  const int steps = (chunk.z + 31) / 32;
  const int *order = q.plan.order + chunk.y;
  const bool columns_whole = !RAGGED || col0 + COLS <= s.width;
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  i32x4 next[2] = {};
  auto load_rows = [&](int st) {      // the lane's 8 rows of a step
    const int at = st * 32 + quad * 8;
    if (st * 32 + 32 <= chunk.z) {
#pragma unroll
      for (int i = 0; i < 2; ++i) next[i] = *reinterpret_cast<const Piece<int, 4>::any *>(order + at + i * 4);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) next[i / 4][i % 4] = order[at + i < chunk.z ? at + i : chunk.z - 1];
    }
  };
  if (wave < steps) load_rows(wave);
  for (int st = wave; st < steps; st += 8) {
    const int at = st * 32 + quad * 8;
    int row[8];
    V v[8];
    f32x4 u[RT][2];
#pragma unroll
    for (int i = 0; i < 8; ++i) row[i] = next[i / 4][i % 4];
#pragma unroll
    for (int r = 0; r < RT; ++r) {      // (places behind the chunk are in the buffer, which has room behind its last)
      const int j = rank0 + r * 16 + c;
      const float *pu = s.ut + (int64_t)(j < q.rank ? j : 0) * q.ut_ld + chunk.y;
#pragma unroll
      for (int i = 0; i < 2; ++i) u[r][i] = zero_unless<float>(rank0 + r * 16 + c < q.rank, load_vec<float>(pu + at + i * 4));
    }
    if (columns_whole) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load_vec<T>((const T *)s.v + (int64_t)row[i] * s.v_stride + col);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load_vec_end<T>((const T *)s.v + (int64_t)row[i] * s.v_stride, col, s.width);
    }
    if (st + 8 < steps) load_rows(st + 8);
    __builtin_amdgcn_sched_barrier(0);
    if (drop) {
#pragma unroll
      for (int i = 0; i < 8; ++i) drop_vec(q.drop, (uint32_t)row[i], col, v[i]);
    }
    if (st * 32 + 32 > chunk.z) {      // rows behind the chunk: nothing, whatever was read in their place
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = zero_unless<T>(at + i < chunk.z, v[i]);
#pragma unroll
        for (int r = 0; r < RT; ++r) u[r][i / 4][i % 4] = at + i < chunk.z ? u[r][i / 4][i % 4] : 0.f;
      }
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[r][i / 4][i % 4], v[i][e], acc[r][e], 0, 0, 0);
    } else {
      if (HALF) {
        float fresh[RT];
        bool any = false;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          float largest = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(u[r][i / 4][i % 4]));
          largest = fmaxf(largest, __shfl_xor(largest, 16));
          largest = fmaxf(largest, __shfl_xor(largest, 32));
          const bool more = largest * scale[r] >= 32768.f && largest != INFINITY;
          fresh[r] = more ? 0.25f * scale_up(largest) : scale[r];
          any |= more;
        }
        if (__any(any)) {
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            times_of_ranks(acc[r], fresh[r] * scale_back(scale[r]));
            scale[r] = fresh[r];
          }
        }
      }
      V hi[RT], mid[RT], lo[RT];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          T h, m, l;
          split(HALF ? u[r][i / 4][i % 4] * scale[r] : u[r][i / 4][i % 4], h, m, l);
          hi[r][i] = h; mid[r][i] = m; lo[r][i] = l;
        }
      u32x4 words[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) words[i] = __builtin_bit_cast(u32x4, v[i]);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const V b = __builtin_bit_cast(V, column_of(words, e));
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          acc[r][e] = mma(lo[r], b, acc[r][e]);
          acc[r][e] = mma(mid[r], b, acc[r][e]);
          acc[r][e] = mma(hi[r], b, acc[r][e]);
        }
      }
    }
  }
  if (HALF) {
#pragma unroll
    for (int r = 0; r < RT; ++r) times_of_ranks(acc[r], scale_back(scale[r]));
  }
  // the waves' sums: 4 + 4, 2 + 2, 1 + 1, one tile of ranks at a time
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    for (int half = 4; half > 0; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int e = 0; e < VE; ++e) s_sum[wave - half][e][lane] = acc[r][e];
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[r][e] += s_sum[wave][e][lane];
      }
    }
  }
  if (wave != 0 || valid <= 0) return;
  const float f = drop ? q.drop.scale : 1.f;
  const int RP = q.rank_padded;
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    const int j0 = rank0 + r * 16 + quad * 4;
    if (j0 >= q.rank) continue;
    if (!s.columns_first) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (j0 + i >= q.rank) continue;
        float o[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) o[e] = acc[r][e][i] * f;
        if (chunk.w < 0) store_some<T, VE>((T *)s.out + ((int64_t)chunk.x * q.rank + j0 + i) * s.width + col, valid, o);
        else store_some<float, VE>(s.part + ((int64_t)chunk.w * RP + j0 + i) * s.width + col, valid, o);
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        if (e >= valid) continue;
        const float o[4] = {acc[r][e][0] * f, acc[r][e][1] * f, acc[r][e][2] * f, acc[r][e][3] * f};
        if (chunk.w < 0) store_some<T, 4>((T *)s.out + ((int64_t)chunk.x * s.width + col + e) * q.rank + j0, q.rank - j0, o);
        else store_some<float, 4>(s.part + ((int64_t)chunk.w * s.width + col + e) * RP + j0, 4, o);
      }
    }
  }
}
// the adapters that `outer` did not finish: the sum of several chunks in a fixed order, by `W` threads where there are many (300 chunks of six adapters, 1024
// results: 7.6 us by single threads, 5.5 by four; 16 chunks of eight, 2^20 results: 4.1 against 5.5)
struct SumArgs {
  OuterSide side[2];
  int rank, rank_padded, blocks0;
  Plan plan;
};
template <typename T, int W>
__global__ void __launch_bounds__(256) lowrank_sum_kernel(SumArgs q) {
  constexpr int PER = 256 / W;
  __shared__ float s_part[W][PER];
  const bool second = (int)blockIdx.x >= q.blocks0;
  const OuterSide &s = q.side[second];
  const int g = blockIdx.y, at = threadIdx.x % PER, slice = threadIdx.x / PER;
  const int2 slots = q.plan.slots[g];
  if (slots.y <= 1) return;
  const unsigned i = (blockIdx.x - (second ? q.blocks0 : 0)) * PER + at, n = (unsigned)q.rank * s.width, o = i < n ? i : n - 1;
  const int64_t each = (int64_t)q.rank_padded * s.width;
  const float *p = s.part + slots.x * each + (s.columns_first ? o / (unsigned)q.rank * q.rank_padded + o % (unsigned)q.rank : o);
  const int share = (slots.y + W - 1) / W, last = (slice + 1) * share < slots.y ? (slice + 1) * share : slots.y;
  float v = 0.f;
  int k = slice * share;
  for (; k + 8 <= last; k += 8) {
    float t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = p[(k + e) * each];
    v += ((t[0] + t[1]) + (t[2] + t[3])) + ((t[4] + t[5]) + (t[6] + t[7]));
  }
  for (; k < last; ++k) v += p[k * each];
  if (W > 1) {
    s_part[slice][at] = v;
    __syncthreads();
    for (int w = 1; w < W; ++w) v += s_part[w][at];      // (slice 0's own is in v)
  }
  if (slice == 0 && i < n) ((T *)s.out)[(int64_t)g * n + i] = (T)v;
}

// ---- a few rows without gradients: no order, workgroups of a row ---------------------------------------------------------------------------
struct RowArgs {
  Ids ids;
  const void *x, *a, *b, *base;
  void *y;
  float *h;
  int64_t x_stride, base_stride, y_stride;
  int n_in, n_out, rank;
  const float *scales;
  Dropout drop;
};
// h_j of the row, in lane 63 of the wave.  EIGHT: eight pieces on their way together, then four (48 rows of 4096, rank 32, fp16: 5.1 against 5.4 us; in the
// one-launch kernel, one row of rank 16, eight took 6.1 us against 5.8)
template <typename T, bool EIGHT>
__device__ __forceinline__ float row_rank(const RowArgs &q, const Dropout &drop, int64_t row, int g, int j) {
  typedef typename Vec<T>::vec V;
  constexpr int N = Vec<T>::N;
  const int lane = threadIdx.x & 63, width = q.n_in;
  const T *px = (const T *)q.x + row * q.x_stride, *pa = (const T *)q.a + ((int64_t)g * q.rank + j) * width;
  float s = 0.f;
  auto add = [&](int k, V u, V v) {
    if (drop.threshold != 0) drop_vec(drop, (uint32_t)row, k, u);
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf((float)u[i], (float)v[i], s);
  };
  int k = lane * N;
  auto pieces = [&](auto ahead) {      // pieces on their way together
    constexpr int AHEAD = decltype(ahead)::value;
    for (; k + (AHEAD - 1) * 64 * N + N <= width; k += AHEAD * 64 * N) {
      V u[AHEAD], v[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) { u[i] = load_vec<T>(px + k + i * 64 * N); v[i] = load_vec<T>(pa + k + i * 64 * N); }
      if (EIGHT) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) add(k + i * 64 * N, u[i], v[i]);
    }
  };
  if (EIGHT) pieces(std::integral_constant<int, 8>{});
  pieces(std::integral_constant<int, 4>{});
  for (; k + N <= width; k += 64 * N) add(k, load_vec<T>(px + k), load_vec<T>(pa + k));
  if (k < width) add(k, load_vec_end<T>(px, k, width), load_vec_end<T>(pa, k, width));
  return wave_sum_to_lane63(s) * (q.scales != nullptr ? q.scales[g] : 1.f) * (drop.threshold != 0 ? drop.scale : 1.f);
}
// columns n, n + step, .. of the row: LPC lanes a column, a lane 16 bytes of its weights at a time; h in LDS or in memory
template <typename T, int LPC>
__device__ __forceinline__ void row_columns(const RowArgs &q, int64_t row, int g, int n, int step, const float *h) {
  typedef typename Vec<T>::vec V;
  constexpr int N = Vec<T>::N;
  const int sub = threadIdx.x % LPC, rank = q.rank;
  const bool has = g < q.ids.n_adapters;
  const T *base = (const T *)q.base + row * q.base_stride, *pb = (const T *)q.b + (int64_t)g * q.n_out * rank;
  T *y = (T *)q.y + row * q.y_stride;
  constexpr int C = 4;      // columns on their way together
  float v[C];
  V w[C];
  auto weights = [&](int j) {      // of ranks j .. j + N
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const T *p = pb + (int64_t)(n + c * step < q.n_out ? n + c * step : n) * rank;
      w[c] = j + N <= rank ? load_vec<T>(p + j) : load_vec_end<T>(p, j, rank);
    }
  };
  auto begin = [&]() {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int at = n + c * step;
      v[c] = q.base != nullptr && at < q.n_out ? (float)base[at] : 0.f;
    }
    if (has && sub * N < rank) weights(sub * N);
  };
  if (n < q.n_out) begin();
  while (n < q.n_out) {
    float s[C];
#pragma unroll
    for (int c = 0; c < C; ++c) s[c] = 0.f;
    if (has) {
      for (int j = sub * N; j < rank; j += LPC * N) {
        if (j != sub * N) weights(j);
        float t[N];
        if (j + N <= rank) {
#pragma unroll
          for (int i = 0; i < N; i += 4) {
            const Vec<float>::vec four = load_vec<float>(h + j + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) t[i + e] = four[e];
          }
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) t[i] = j + i < rank ? h[j + i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int c = 0; c < C; ++c) s[c] = fmaf(t[i], (float)w[c][i], s[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int o = 1; o < LPC; o <<= 1) s[c] += __shfl_xor(s[c], o);
      if (sub == 0 && n + c * step < q.n_out) y[n + c * step] = (T)(s[c] + v[c]);
    }
    n += C * step;
    if (n < q.n_out) begin();
  }
}
template <typename T>
__device__ __forceinline__ void row_columns_by_rank(const RowArgs &q, int64_t row, int g, int block, int blocks, const float *h) {
  constexpr int N = Vec<T>::N;
  const int t = threadIdx.x, threads = blockDim.x;
  if (q.rank <= N) row_columns<T, 1>(q, row, g, block * threads + t, blocks * threads, h);
  else if (q.rank <= 2 * N) row_columns<T, 2>(q, row, g, (block * threads + t) / 2, blocks * threads / 2, h);
  else row_columns<T, 4>(q, row, g, (block * threads + t) / 4, blocks * threads / 4, h);
}
template <typename T>
__global__ void __launch_bounds__(1024) lowrank_row_shrink_kernel(RowArgs q) {
  const int64_t row = blockIdx.x;
  const int j = blockIdx.y * 16 + (threadIdx.x >> 6), g = group_of(q.ids, row);
  if (j >= q.rank || g == q.ids.n_adapters) return;
  dropout_counter(q.drop);
  const float v = row_rank<T, true>(q, q.drop, row, g, j);
  if ((threadIdx.x & 63) == 63) q.h[row * q.rank + j] = v;
}
template <typename T>
__global__ void __launch_bounds__(256) lowrank_row_expand_kernel(RowArgs q) {
  const int64_t row = blockIdx.x;
  const int g = group_of(q.ids, row);
  if (g == q.ids.n_adapters && q.base == q.y) return;
  row_columns_by_rank<T>(q, row, g, blockIdx.y, gridDim.y, q.h + row * q.rank);
}
// both in one launch: every workgroup of a row makes its h again
template <typename T>
__global__ void __launch_bounds__(1024) lowrank_row_kernel(RowArgs q) {
  __shared__ float s_h[GSDF_LOWRANK_MAX_RANK];
  const int64_t row = blockIdx.x;
  const int g = group_of(q.ids, row);
  if (g == q.ids.n_adapters && q.base == q.y) return;
  if (g < q.ids.n_adapters) {
    dropout_counter(q.drop);
    for (int j = threadIdx.x >> 6; j < q.rank; j += 16) {
      const float v = row_rank<T, false>(q, q.drop, row, g, j);
      if ((threadIdx.x & 63) == 63) s_h[j] = v;
    }
  }
  __syncthreads();
  row_columns_by_rank<T>(q, row, g, blockIdx.y, gridDim.y, s_h);
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------------
// Without gradients, few rows take no plan, which costs 10 us and the layout of every adapter's A before the first product, but read the weights again for every row.
// Up to 64 rows always (bf16, 4096 -> 4096, rank 64: 13 to 15 us against 23); up to 512, or four an adapter, while what the rows read is no more than 32 MB and
// twice the weights of all adapters (a choice between rows that are all of one adapter, and stay in a cache, and rows that are of all).  bf16, 4096 -> 4096: 8 adapters of rank 16, 128 rows 11 us
// against 17; 1024 of rank 64, 2048 rows 191 us against 247 where they are of one adapter and 361 against 413 where they are of all, 4096 rows 352 against 253 and 679 against 445; 128 of
// rank 64, 256 rows 28 and 47 against 42 and 52, 512 rows 49 and 80 against 43 and 55.  64 -> 4096, 1000 of rank 16, 800 rows: 20 and 29 against 33 and 45.
static constexpr int64_t LR_FEW_BYTES = 32 << 20;
static constexpr int64_t LR_FEW_ROWS = 64;
// bytes of A that may be read to make every row's h again in each of its workgroups, for a launch less
static constexpr int64_t LR_ROW_AGAIN = 4 << 20;
static constexpr int64_t LR_PAST = 32 << 20;      // bytes of a result from which on it is written past the caches

#define GSDF_BY_RANK(rt, ...)                                 \
  switch (rt) {                                               \
    case 1: { constexpr int RT = 1; __VA_ARGS__; break; }     \
    case 2: { constexpr int RT = 2; __VA_ARGS__; break; }     \
    case 4: { constexpr int RT = 4; __VA_ARGS__; break; }     \
    default: { constexpr int RT = 8; __VA_ARGS__; break; }    \
  }

static ShrinkArgs shrink_args(const Lowrank &q, const void *x, int64_t x_stride, int width, const void *w, const float *scales, bool drop, float *h, float *ht) {
  ShrinkArgs s;
  s.x = x; s.w = w; s.x_stride = x_stride; s.width = width; s.rank = q.a.rank; s.split = 1;
  s.scales = scales; s.factor = drop ? q.drop.scale : 1.f; s.h = h; s.ht = ht; s.ht_ld = q.ht_ld; s.drop = q.drop; s.plan = q.plan;
  return s;
}
static ExpandArgs expand_args(const Lowrank &q, const float *h, const void *w, int64_t w_group, int w_ld, int ranks, int width, const void *base, int64_t base_stride,
                              void *y, int64_t y_stride) {
  ExpandArgs s;
  s.h = h; s.w = w; s.base = base; s.y = y; s.w_group = w_group; s.base_stride = base_stride; s.y_stride = y_stride; s.width = width; s.w_ld = w_ld; s.rank = ranks;
  s.parts = 1; s.drop = q.drop; s.plan = q.plan;
  return s;
}
// y from x: `shrink` and `expand`, or both at once; `shrink` alone where no y is wanted
template <typename T>
static void products_launch(const Lowrank &q, ShrinkArgs s, ExpandArgs e, bool drop_x, bool drop_y, hipStream_t stream) {
  constexpr int STEP = 128 / (int)sizeof(T), N = 16 / (int)sizeof(T);
  const bool past = (int64_t)q.a.rows * e.width * (int64_t)sizeof(T) >= LR_PAST;
  if (q.both && e.y != nullptr) {
    const unsigned grid = (unsigned)q.plan.n_wide;
    const bool ragged = s.width % STEP != 0 || e.width % 64 != 0;
    auto run = [&](auto rt, auto dx, auto dy) {
      constexpr int RT = decltype(rt)::value;
      constexpr bool DX = decltype(dx)::value, DY = decltype(dy)::value;
      if (ragged) lowrank_both_kernel<T, RT, DX, DY, true, false><<<grid, 64, 0, stream>>>(s, e);
      else if (past) lowrank_both_kernel<T, RT, DX, DY, false, true><<<grid, 64, 0, stream>>>(s, e);
      else lowrank_both_kernel<T, RT, DX, DY, false, false><<<grid, 64, 0, stream>>>(s, e);
    };
    auto by_drop = [&](auto rt) {
      if (drop_x) run(rt, std::true_type{}, std::false_type{});
      else if (drop_y) run(rt, std::false_type{}, std::true_type{});
      else run(rt, std::false_type{}, std::false_type{});
    };
    if (q.rt == 1) by_drop(std::integral_constant<int, 1>{});
    else by_drop(std::integral_constant<int, 2>{});
    return;
  }
  {
    const int steps = (int)ceil_div(s.width, STEP);
    s.split = steps >= 8 ? 8 : steps >= 4 ? 4 : steps >= 2 ? 2 : 1;
    const unsigned grid = (unsigned)(s.split == 1 ? ceil_div(q.plan.n_ranges, 4) : q.plan.n_ranges), threads = s.split == 1 ? 256 : 64 * s.split;
    const bool ragged = s.width % STEP != 0;
    GSDF_BY_RANK(q.rt, {
      const size_t lds = s.split == 1 ? 0 : (size_t)s.split * (RT < 2 ? 1 : 2) * 3 * 64 * sizeof(f32x4);
      if (drop_x && ragged) lowrank_shrink_kernel<T, RT, true, true><<<grid, threads, lds, stream>>>(s);
      else if (drop_x) lowrank_shrink_kernel<T, RT, true, false><<<grid, threads, lds, stream>>>(s);
      else if (ragged) lowrank_shrink_kernel<T, RT, false, true><<<grid, threads, lds, stream>>>(s);
      else lowrank_shrink_kernel<T, RT, false, false><<<grid, threads, lds, stream>>>(s);
    });
  }
  if (e.y == nullptr) return;      // dh alone: x wants no gradient
  const int64_t chunks = ceil_div(e.width, 64);
  // one chunk of 64 columns a wave until there are more than eight waves a SIMD, then more
  e.parts = (int)ceil_div(chunks, ceil_div(chunks * q.plan.n_wide, LR_CUS * 4 * 8));
  const unsigned grid = (unsigned)ceil_div((int64_t)q.plan.n_wide * e.parts, 4);
  const bool ragged = e.width % 64 != 0 || e.rank % N != 0;
  auto run = [&](auto rt, auto drop) {
    constexpr int RT = decltype(rt)::value;
    constexpr bool DROP = decltype(drop)::value;
    if (ragged) lowrank_expand_kernel<T, RT, DROP, true, false><<<grid, 256, 0, stream>>>(e);
    else if (past) lowrank_expand_kernel<T, RT, DROP, false, true><<<grid, 256, 0, stream>>>(e);
    else lowrank_expand_kernel<T, RT, DROP, false, false><<<grid, 256, 0, stream>>>(e);
  };
  GSDF_BY_RANK(q.rt, {
    if (drop_y) run(std::integral_constant<int, RT>{}, std::true_type{});
    else run(std::integral_constant<int, RT>{}, std::false_type{});
  });
}

template <typename T>
void lowrank_fwd(const Lowrank &q, const void *base, int64_t base_stride, void *y, int64_t y_stride, bool training, hipStream_t stream) {
  const gsdf_lowrank_args &a = q.a;
  const Ids ids = {a.ids, a.ids_64, a.n_adapters};
  const int64_t read = a.rows * a.rank * ((int64_t)a.n_in + a.n_out) * (int64_t)sizeof(T);      // of the adapters' weights, row by row
  const int64_t bank = (int64_t)a.n_adapters * q.rp * ((int64_t)a.n_in + a.n_out) * (int64_t)sizeof(T);      // all weights, ranks in whole tiles
  const int64_t most = 4 * (int64_t)a.n_adapters > 8 * LR_FEW_ROWS ? 4 * (int64_t)a.n_adapters : 8 * LR_FEW_ROWS;
  if (!training && (a.rows <= LR_FEW_ROWS || (a.rows <= most && read <= LR_FEW_BYTES + 2 * bank))) {
    constexpr int N = 16 / (int)sizeof(T);
    RowArgs r;
    r.ids = ids; r.x = a.x; r.a = a.a; r.b = a.b; r.base = base; r.y = y; r.h = q.h; r.x_stride = a.x_stride; r.base_stride = base_stride; r.y_stride = y_stride;
    r.n_in = a.n_in; r.n_out = a.n_out; r.rank = a.rank; r.scales = a.scales; r.drop = q.drop;
    const int lanes = a.rank <= N ? 1 : a.rank <= 2 * N ? 2 : 4;
    const int64_t wide = ceil_div((int64_t)a.n_out * lanes, 1024), weights = (int64_t)a.rank * a.n_in * (int64_t)sizeof(T);
    if (a.rows * wide * weights <= LR_ROW_AGAIN) {
      lowrank_row_kernel<T><<<dim3((unsigned)a.rows, (unsigned)wide), 1024, 0, stream>>>(r);
      return;
    }
    const int64_t narrow = ceil_div((int64_t)a.n_out * lanes, 256), most = ceil_div(2048, a.rows);
    lowrank_row_shrink_kernel<T><<<dim3((unsigned)a.rows, (unsigned)ceil_div(a.rank, 16)), 1024, 0, stream>>>(r);
    lowrank_row_expand_kernel<T><<<dim3((unsigned)a.rows, (unsigned)(narrow < most ? narrow : most)), 256, 0, stream>>>(r);
    return;
  }
  lowrank_plan_launch(q.plan, ids, lowrank_pack_args(q, training), stream);
  products_launch<T>(q, shrink_args(q, a.x, a.x_stride, a.n_in, q.a_frag, a.scales, q.drop.threshold != 0, q.h, training ? q.ht : nullptr),
                     expand_args(q, q.h, a.b, (int64_t)a.n_out * a.rank, a.rank, a.rank, a.n_out, base, base_stride, y, y_stride), q.drop.threshold != 0, false, stream);
}

template <typename T>
void lowrank_bwd(const Lowrank &q, const void *dy, int64_t dy_stride, void *dx, int64_t dx_stride, void *da, void *db, hipStream_t stream) {
  const gsdf_lowrank_args &a = q.a;
  const bool drop = q.drop.threshold != 0;
  const unsigned G = (unsigned)a.n_adapters;
  if (a.rows > 0 && (dx != nullptr || da != nullptr))
    products_launch<T>(q, shrink_args(q, dy, dy_stride, a.n_out, q.b_frag, a.scales, false, dx != nullptr ? q.dh : nullptr, da != nullptr ? q.dht : nullptr),
                       expand_args(q, q.dh, q.a_turned, (int64_t)a.n_in * q.rp, q.rp, q.rp, a.n_in, nullptr, 0, dx, dx_stride), false, drop, stream);
  if (da == nullptr && db == nullptr) return;
  constexpr int COLS = 16 * (16 / (int)sizeof(T));
  OuterArgs o;
  o.side[0] = {q.dht, a.x, a.x_stride, a.n_in, drop, 0, da, q.part[0]};
  o.side[1] = {q.ht, dy, dy_stride, a.n_out, 0, 1, db, q.part[1]};
  o.ut_ld = q.ht_ld; o.rank = a.rank; o.rank_padded = q.rp; o.drop = q.drop; o.plan = q.plan;
  o.blocks0 = da != nullptr ? (int)ceil_div(a.n_in, COLS) : 0;
  const unsigned blocks1 = db != nullptr ? (unsigned)ceil_div(a.n_out, COLS) : 0;
  o.blocks = o.blocks0 + (int)blocks1;
  {
    const dim3 grid((unsigned)o.blocks * (unsigned)q.plan.max_chunks, q.rt == 8 ? 2 : 1);
    const bool ragged = a.n_in % COLS != 0 || a.n_out % COLS != 0;
    switch (q.rt) {
      case 1: ragged ? lowrank_outer_kernel<T, 1, true><<<grid, LR_OUTER_THREADS, 0, stream>>>(o) : lowrank_outer_kernel<T, 1, false><<<grid, LR_OUTER_THREADS, 0, stream>>>(o); break;
      case 2: ragged ? lowrank_outer_kernel<T, 2, true><<<grid, LR_OUTER_THREADS, 0, stream>>>(o) : lowrank_outer_kernel<T, 2, false><<<grid, LR_OUTER_THREADS, 0, stream>>>(o); break;
      default: ragged ? lowrank_outer_kernel<T, 4, true><<<grid, LR_OUTER_THREADS, 0, stream>>>(o) : lowrank_outer_kernel<T, 4, false><<<grid, LR_OUTER_THREADS, 0, stream>>>(o); break;
    }
  }
  if (a.rows <= q.plan.chunk_rows) return;      // no adapter has two chunks
  SumArgs s;
  s.side[0] = o.side[0]; s.side[1] = o.side[1]; s.rank = a.rank; s.rank_padded = q.rp; s.plan = q.plan;
  const bool many = a.rows / LR_CHUNK > 4 * (int64_t)G;      // chunks of an adapter, on average
  const int per = many ? 64 : 256;
  s.blocks0 = da != nullptr ? (int)ceil_div((int64_t)a.rank * a.n_in, per) : 0;
  const unsigned sum1 = db != nullptr ? (unsigned)ceil_div((int64_t)a.rank * a.n_out, per) : 0;
  if (many) lowrank_sum_kernel<T, 4><<<dim3((unsigned)s.blocks0 + sum1, G), 256, 0, stream>>>(s);
  else lowrank_sum_kernel<T, 1><<<dim3((unsigned)s.blocks0 + sum1, G), 256, 0, stream>>>(s);
}


}  // namespace gsdf
