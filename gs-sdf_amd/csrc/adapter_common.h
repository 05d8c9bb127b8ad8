// adapter_common.h — what the adapter operators (lowrank.hip, dropout.hip, router_balance.hip) share: element types, vectors of elements at
// any alignment, and the counter-based generator behind the dropout mask.
#pragma once
#include <math.h>

#include "common.h"

namespace gsdf {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// N consecutive elements at the alignment of ONE: global memory takes 16-byte accesses at any multiple of the element, so a row that
// starts anywhere is still read and written in 16-byte pieces
template <typename T, int N>
struct Piece {
  typedef T vec __attribute__((ext_vector_type(N)));
  typedef vec any __attribute__((aligned(sizeof(T)), may_alias));
};
template <typename T, int N>
__device__ __forceinline__ void load_piece(const T *__restrict__ p, T (&out)[N]) {
  const typename Piece<T, N>::vec t = *reinterpret_cast<const typename Piece<T, N>::any *>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = t[i];
}
template <typename T, int N, bool PAST = false>      // PAST: past the caches
__device__ __forceinline__ void store_piece(T *__restrict__ p, const T (&in)[N]) {
  typename Piece<T, N>::vec t;
#pragma unroll
  for (int i = 0; i < N; ++i) t[i] = in[i];
  if (PAST && N * sizeof(T) > 16) {      // (two accesses of 16 bytes)
    typename Piece<T, N / 2>::vec a, b;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) { a[i] = t[i]; b[i] = t[N / 2 + i]; }
    __builtin_nontemporal_store(a, reinterpret_cast<typename Piece<T, N / 2>::any *>(p));
    __builtin_nontemporal_store(b, reinterpret_cast<typename Piece<T, N / 2>::any *>(p + N / 2));
  } else if (PAST) {
    __builtin_nontemporal_store(t, reinterpret_cast<typename Piece<T, N>::any *>(p));
  } else {
    *reinterpret_cast<typename Piece<T, N>::any *>(p) = t;
  }
}

// ---- the dropout mask ---------------------------------------------------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): ten rounds of two 32x32 -> 64-bit products.
// One block = 128 bits = 16 bits for each of 8 neighbouring elements of a row.  Counter: (col / 8, row, offset), key: seed — an element's bits depend
// on its place in the matrix alone, never on the launch, so the backward pass makes them again instead of reading a stored mask.
struct Dropout {
  uint32_t key0, key1, off0, off1;
  const uint64_t *offset_dev;      // added to the offset where it is not null (a captured graph's counter)
  uint32_t threshold;              // an element is dropped where its 16 bits are below: round(65536 p), 0 .. 65536
  float scale;                     // 65536 / (65536 - threshold); 0 where everything is dropped
};
static inline Dropout make_dropout(double p, uint64_t seed, uint64_t offset, const uint64_t *offset_dev) {
  Dropout d;
  d.key0 = (uint32_t)seed; d.key1 = (uint32_t)(seed >> 32);
  d.off0 = (uint32_t)offset; d.off1 = (uint32_t)(offset >> 32);
  d.offset_dev = offset_dev;
  d.threshold = (uint32_t)floor(p * 65536.0 + 0.5);
  d.scale = d.threshold >= 65536u ? 0.f : (float)(65536.0 / (65536.0 - d.threshold));
  return d;
}
#ifdef __HIPCC__
__device__ __forceinline__ void dropout_counter(Dropout &d) {
  if (d.offset_dev != nullptr) {
    const uint64_t o = (((uint64_t)d.off1 << 32) | d.off0) + *d.offset_dev;
    d.off0 = (uint32_t)o; d.off1 = (uint32_t)(o >> 32);
  }
}
// the 16-bit pieces of the 8 elements [8 block, 8 block + 8) of `row`, two per word, the lower column in the lower half
__device__ __forceinline__ void dropout_bits(const Dropout &d, uint32_t block, uint32_t row, uint32_t (&w)[4]) {
  uint32_t c0 = block, c1 = row, c2 = d.off0, c3 = d.off1, k0 = d.key0, k1 = d.key1;
#pragma unroll
  for (int i = 0; i < 10; ++i) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0; c1 = (uint32_t)p1;
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1; c3 = (uint32_t)p0;
    k0 += 0x9E3779B9u; k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}
__device__ __forceinline__ bool dropout_keeps(const Dropout &d, const uint32_t (&w)[4], int i) {
  return ((i & 1) ? (w[i >> 1] >> 16) : (w[i >> 1] & 0xFFFFu)) >= d.threshold;
}
#endif

#ifdef __HIPCC__
__device__ __forceinline__ int64_t load_id(const void *__restrict__ ids, int ids_64, int64_t i) {
  return ids_64 ? static_cast<const int64_t *>(ids)[i] : (int64_t) static_cast<const int32_t *>(ids)[i];
}
#endif

// runs `body` with T = the element type of `dtype`
#define GSDF_BY_DTYPE(dtype, ...)                                          \
  switch (dtype) {                                                         \
    case GSDF_F32: { typedef float T; __VA_ARGS__; break; }                \
    case GSDF_F16: { typedef gsdf::f16_t T; __VA_ARGS__; break; }          \
    default: { typedef gsdf::bf16_t T; __VA_ARGS__; break; }               \
  }

static inline bool known_dtype(int dtype) { return dtype == GSDF_F32 || dtype == GSDF_F16 || dtype == GSDF_BF16; }
static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

}  // namespace gsdf
