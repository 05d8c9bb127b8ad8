// lowrank.hip — low-rank adapters of many requests at once beside a shared projection:
//     y_t = base_t + s_g B_g h_t,   h_t = A_g drop(x_t),   g = ids[t]
// backward:  dh_t = s_g B_g^T dy_t,  dx_t = drop'(A_g^T dh_t),  dA_g = sum_t dh_t drop(x_t)^T,  dB_g = s_g sum_t dy_t h_t^T.
//
// The adapters' weights are small beside x, base and y, so the operator is bound by the bytes of its rows.  The rows are put in the order of
// their adapters first (`plan_*`): a tile of 32 rows then has one adapter, and each product is a tile of matrix instructions whose operands
// come from global memory in the layout that the instruction wants:
//   shrink   contracts a row's elements (x with A, dy with B^T).  The order of the contraction is free: four lanes take 32 neighbouring bytes each of a
//            row's 128, so that a row is read in whole cache lines.  The waves of a workgroup split the row and meet in LDS.
//   expand   contracts ranks (h with B, dh with A^T): the instruction's rows are columns of y, permuted so that a lane holds 16 neighbours.
//   outer    contracts rows (dh with x, h with dy): a lane holds 8 rows x 16 bytes and turns them in registers.
// h and dh are held in 32 bits.  In front of 16-bit instructions they are split into a high and a low part of the weights' type (16 or 22 bits of the
// value's), which costs instructions that are not the bound; rounding them once would cost as much precision again as the result's own rounding.
#include "adapter_common.h"

namespace gsdf {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

static constexpr int LR_TILE = 32;          // rows of a tile: two matrix tiles, so that weights are read once for 32 rows
static constexpr int LR_CHUNK = 1024;       // rows of one sum in `outer`
static constexpr int LR_PLAN_ROWS = 16384;  // rows of one workgroup of the plan

// ---- the rows in the order of their adapters ----------------------------------------------------------------------------------------------
// All in one int32 buffer.  Group n_adapters holds the rows without an adapter.
struct Plan {
  int *order;      // [rows]: the row at each place, adapters one behind the other, rows of one adapter in their own order
  int4 *tile;      // [max_tiles]: adapter, first place, rows (0: unused), -
  int4 *chunk;     // [max_chunks]: adapter, first place, rows, slot of its partial sums (-1: the adapter's only chunk)
  int2 *slots;     // [n_adapters]: first slot, chunks
  int *start;      // [n_adapters + 2]
  int *tile0;      // [n_adapters + 2]: first tile of each group
  int *chunk0;     // [n_adapters + 1]
  int *hist;       // [blocks][n_adapters + 1]: rows of each group in front of each workgroup's share
  int max_tiles, max_chunks, blocks, n_adapters;
  int64_t rows;
};
static size_t plan_layout(Plan *p, void *mem, int64_t rows, int n_adapters) {
  p->rows = rows; p->n_adapters = n_adapters;
  p->blocks = (int)ceil_div(rows > 0 ? rows : 1, LR_PLAN_ROWS);
  p->max_tiles = (int)(rows / LR_TILE + n_adapters + 1);
  p->max_chunks = (int)(rows / LR_CHUNK + n_adapters);
  char *at = (char *)mem;
  auto take = [&](size_t bytes) { char *r = at; at += align_up(bytes, 16); return r; };
  p->tile = (int4 *)take((size_t)p->max_tiles * 16);
  p->chunk = (int4 *)take((size_t)p->max_chunks * 16);
  p->slots = (int2 *)take((size_t)n_adapters * 8);
  p->start = (int *)take((size_t)(n_adapters + 2) * 4);
  p->tile0 = (int *)take((size_t)(n_adapters + 2) * 4);
  p->chunk0 = (int *)take((size_t)(n_adapters + 1) * 4);
  p->hist = (int *)take((size_t)p->blocks * (n_adapters + 1) * 4);
  p->order = (int *)take((size_t)rows * 4);
  return (size_t)(at - (char *)mem);
}
// slots for the chunks of adapters with more than one: such an adapter has more than LR_CHUNK rows, so there are at most twice rows / LR_CHUNK of them
static int64_t plan_max_slots(int64_t rows, int n_adapters) {
  const int64_t twice = 2 * (rows / LR_CHUNK) + 1, all = rows / LR_CHUNK + n_adapters;
  return rows <= LR_CHUNK ? 0 : (twice < all ? twice : all);
}

struct Ids {
  const void *p;
  int is_64, n_adapters;
};
__device__ __forceinline__ int group_of(Ids ids, int64_t row) {
  const int64_t g = load_id(ids.p, ids.is_64, row);
  return g >= 0 && g < ids.n_adapters ? (int)g : ids.n_adapters;
}

// exclusive sums of (a, b, c) over the 1024 threads of the workgroup; totals in `sum`
__device__ __forceinline__ int3 block_scan3(int3 v, int3 *sum, int (*s_w)[3]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int3 i = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(i.x, o), b = __shfl_up(i.y, o), c = __shfl_up(i.z, o);
    if (lane >= o) { i.x += a; i.y += b; i.z += c; }
  }
  if (lane == 63) { s_w[wave][0] = i.x; s_w[wave][1] = i.y; s_w[wave][2] = i.z; }
  __syncthreads();
  int3 before = {0, 0, 0}, all = {0, 0, 0};
  for (int w = 0; w < 16; ++w) {
    if (w == wave) before = all;
    all.x += s_w[w][0]; all.y += s_w[w][1]; all.z += s_w[w][2];
  }
  *sum = all;
  return {before.x + i.x - v.x, before.y + i.y - v.y, before.z + i.z - v.z};
}

// lengths of the groups -> starts, tiles, chunks, slots (one workgroup of 1024; thread g has adapter g's rows)
__device__ __forceinline__ void plan_tables(const Plan &p, int rows_of, int (*s_w)[3]) {
  const int G = p.n_adapters, g = threadIdx.x;
  const int n = g < G ? rows_of : 0, chunks = (n + LR_CHUNK - 1) / LR_CHUNK;
  int3 sum, sum2;
  const int3 at = block_scan3({n, (n + LR_TILE - 1) / LR_TILE, chunks}, &sum, s_w);
  __syncthreads();
  const int3 slot = block_scan3({chunks > 1 ? chunks : 0, 0, 0}, &sum2, s_w);
  if (g < G) {
    p.start[g] = at.x; p.tile0[g] = at.y; p.chunk0[g] = at.z;
    p.slots[g] = {slot.x, chunks};
  }
  if (g == 0) {
    const int idle = (int)p.rows - sum.x;
    p.start[G] = sum.x; p.start[G + 1] = (int)p.rows;
    p.tile0[G] = sum.y; p.tile0[G + 1] = sum.y + (idle + LR_TILE - 1) / LR_TILE;
    p.chunk0[G] = sum.z;
  }
}
// the last group that begins at or before i
__device__ __forceinline__ int find_group(const int *first, int n, int i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= i) lo = mid; else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ void plan_lists(const Plan &p, int first, int step) {
  const int G = p.n_adapters;
  const int tiles = p.tile0[G + 1], chunks = p.chunk0[G];
  for (int i = first; i < p.max_tiles; i += step) {
    int4 t = {0, 0, 0, 0};
    if (i < tiles) {
      const int g = find_group(p.tile0, G + 1, i), at = p.start[g] + (i - p.tile0[g]) * LR_TILE, left = p.start[g + 1] - at;
      t = {g, at, left < LR_TILE ? left : LR_TILE, 0};
    }
    p.tile[i] = t;
  }
  for (int i = first; i < p.max_chunks; i += step) {
    int4 t = {0, 0, 0, -1};
    if (i < chunks) {
      const int g = find_group(p.chunk0, G, i), k = i - p.chunk0[g], at = p.start[g] + k * LR_CHUNK, left = p.start[g + 1] - at;
      t = {g, at, left < LR_CHUNK ? left : LR_CHUNK, p.slots[g].y > 1 ? p.slots[g].x + k : -1};
    }
    p.chunk[i] = t;
  }
}
// counts of the workgroup's rows by wave: s_hist[wave][group]; each wave owns a run of rows, so that places follow the rows' order
__device__ __forceinline__ void plan_count(const Ids &ids, int64_t first, int64_t last, int *s_hist, int G1) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  for (int i = threadIdx.x; i < 16 * G1; i += 1024) s_hist[i] = 0;
  __syncthreads();
  const int64_t run = (last - first + 1023) / 1024 * 64, from = first + wave * run, to = from + run < last ? from + run : last;
  for (int64_t i = from + lane; i < to; i += 64) atomicAdd(&s_hist[wave * G1 + group_of(ids, i)], 1);
  __syncthreads();
}
__device__ __forceinline__ void plan_place(const Ids &ids, int64_t first, int64_t last, int *s_next, int G1, int *order) {
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t run = (last - first + 1023) / 1024 * 64, from = first + wave * run, to = from + run < last ? from + run : last;
  int bits = 0;
  while ((1 << bits) < G1) ++bits;
  for (int64_t i0 = from; i0 < to; i0 += 64) {
    const int64_t i = i0 + lane;
    const bool in = i < to;
    const int g = in ? group_of(ids, i) : 0;
    uint64_t same = __ballot(in);      // the lanes with my group
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((g >> b) & 1);
      same &= ((g >> b) & 1) ? set : ~set;
    }
    if (in) {
      int *next = &s_next[wave * G1 + g];
      const int base = __hip_atomic_load(next, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      const int before = __popcll(same & ((1ull << lane) - 1));
      order[base + before] = (int)i;
      __builtin_amdgcn_wave_barrier();      // every lane has read the place before its first lane moves it on
      if (before == 0) __hip_atomic_store(next, base + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// up to LR_PLAN_ROWS rows: all in one workgroup
__global__ void __launch_bounds__(1024) lowrank_plan_kernel(Plan p, Ids ids) {
  extern __shared__ int s_hist[];      // [16][G + 1]
  __shared__ int s_w[16][3];
  const int G = p.n_adapters, G1 = G + 1, t = threadIdx.x;
  plan_count(ids, 0, p.rows, s_hist, G1);
  int n = 0;
  if (t < G)
    for (int w = 0; w < 16; ++w) n += s_hist[w * G1 + t];
  plan_tables(p, n, s_w);
  __syncthreads();      // (the tables are read back below: same workgroup, same CU, behind a barrier that waits for the stores)
  for (int g = t; g < G1; g += 1024) {
    int at = p.start[g];
    for (int w = 0; w < 16; ++w) { const int c = s_hist[w * G1 + g]; s_hist[w * G1 + g] = at; at += c; }
  }
  __syncthreads();
  plan_place(ids, 0, p.rows, s_hist, G1, p.order);
  plan_lists(p, t, 1024);
}
// more rows: counts of each workgroup's share, their sums, the places
__global__ void __launch_bounds__(1024) lowrank_plan_count_kernel(Plan p, Ids ids) {
  extern __shared__ int s_hist[];
  const int G1 = p.n_adapters + 1;
  const int64_t first = (int64_t)blockIdx.x * LR_PLAN_ROWS, last = first + LR_PLAN_ROWS < p.rows ? first + LR_PLAN_ROWS : p.rows;
  plan_count(ids, first, last, s_hist, G1);
  for (int g = threadIdx.x; g < G1; g += 1024) {
    int n = 0;
    for (int w = 0; w < 16; ++w) n += s_hist[w * G1 + g];
    p.hist[(int64_t)blockIdx.x * G1 + g] = n;
  }
}
__global__ void __launch_bounds__(1024) lowrank_plan_scan_kernel(Plan p) {
  __shared__ int s_w[16][3];
  const int G1 = p.n_adapters + 1;
  int mine = 0;
  for (int g = threadIdx.x; g < G1; g += 1024) {
    int n = 0;
    for (int b = 0; b < p.blocks; ++b) { const int c = p.hist[(int64_t)b * G1 + g]; p.hist[(int64_t)b * G1 + g] = n; n += c; }
    if (g == threadIdx.x) mine = n;
  }
  plan_tables(p, mine, s_w);
}
__global__ void __launch_bounds__(1024) lowrank_plan_place_kernel(Plan p, Ids ids) {
  extern __shared__ int s_hist[];
  const int G1 = p.n_adapters + 1;
  const int64_t first = (int64_t)blockIdx.x * LR_PLAN_ROWS, last = first + LR_PLAN_ROWS < p.rows ? first + LR_PLAN_ROWS : p.rows;
  plan_count(ids, first, last, s_hist, G1);
  for (int g = threadIdx.x; g < G1; g += 1024) {
    int at = p.start[g] + p.hist[(int64_t)blockIdx.x * G1 + g];
    for (int w = 0; w < 16; ++w) { const int c = s_hist[w * G1 + g]; s_hist[w * G1 + g] = at; at += c; }
  }
  __syncthreads();
  plan_place(ids, first, last, s_hist, G1, p.order);
  plan_lists(p, blockIdx.x * 1024 + threadIdx.x, gridDim.x * 1024);
}

static void plan_launch(const Plan &p, const Ids &ids, hipStream_t stream) {
  const size_t lds = (size_t)16 * (p.n_adapters + 1) * 4;
  if (p.blocks == 1) {
    lowrank_plan_kernel<<<1, 1024, lds, stream>>>(p, ids);
  } else {
    lowrank_plan_count_kernel<<<p.blocks, 1024, lds, stream>>>(p, ids);
    lowrank_plan_scan_kernel<<<1, 1024, 0, stream>>>(p);
    lowrank_plan_place_kernel<<<p.blocks, 1024, lds, stream>>>(p, ids);
  }
}

// ---- pieces of rows ---------------------------------------------------------------------------------------------------------------------------
// 32 bytes of a row: what a lane contracts in one step of `shrink`
template <typename T>
struct Span {
  static constexpr int N = 32 / sizeof(T);
  T v[N];
};
// the first `valid` of its elements, 0 behind them
template <typename T, int N>
__device__ __forceinline__ void load_part(const T *__restrict__ p, int valid, T (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < valid ? p[i] : (T)0.f;
}
template <typename T, int N>
__device__ __forceinline__ void load_some(const T *__restrict__ p, int valid, T (&v)[N]) {
  constexpr int W = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  if (valid >= N) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
      T t[W];
      load_piece<T, W>(p + i, t);
#pragma unroll
      for (int j = 0; j < W; ++j) v[i + j] = t[j];
    }
  } else {
    load_part<T, N>(p, valid, v);
  }
}
// N (a multiple of 4) neighbouring results, `valid` of them
template <typename T, int N>
__device__ __forceinline__ void store_some(T *__restrict__ p, int valid, const float (&v)[N]) {
  constexpr int W = 16 / sizeof(T) < N ? 16 / sizeof(T) : N;
  if (valid >= N) {
#pragma unroll
    for (int i = 0; i < N; i += W) {
      T t[W];
#pragma unroll
      for (int j = 0; j < W; ++j) t[j] = (T)v[i + j];
      store_piece<T, W>(p + i, t);
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}
// zero where dropped: N elements of `row` from column `col`, a multiple of N (N = 4: half a block); the survivors' factor goes into the sums
template <typename T, int N>
__device__ __forceinline__ void drop_some(const Dropout &d, uint32_t row, int col, T (&v)[N]) {
#pragma unroll
  for (int b = 0; b < N; b += 8) {
    uint32_t w[4];
    dropout_bits(d, (uint32_t)(col + b) >> 3, row, w);
    if (N == 4 && (col & 4)) { w[0] = w[2]; w[1] = w[3]; }
#pragma unroll
    for (int i = 0; i < (N < 8 ? N : 8); ++i) v[b + i] = dropout_keeps(d, w, i) ? v[b + i] : (T)0.f;
  }
}

// acc += a b over 8 contracted elements of each lane: one 16-bit instruction, or eight of 32 bits (any order of the contraction is as good)
__device__ __forceinline__ f32x4 mma8(const bf16_t *a, const bf16_t *b, f32x4 acc) {
  bf16x8 u, v;
#pragma unroll
  for (int i = 0; i < 8; ++i) { u[i] = a[i]; v[i] = b[i]; }
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(u, v, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma8(const f16_t *a, const f16_t *b, f32x4 acc) {
  f16x8 u, v;
#pragma unroll
  for (int i = 0; i < 8; ++i) { u[i] = a[i]; v[i] = b[i]; }
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(u, v, acc, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma8(const float *a, const float *b, f32x4 acc) {
#pragma unroll
  for (int i = 0; i < 8; ++i) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], acc, 0, 0, 0);
  return acc;
}
// a power of two that brings the largest of the wave's |v| (over lanes that `same` joins) into [1, 2): 16-bit numbers of fp16 would run over or vanish
__device__ __forceinline__ float scale_to_one(float largest) {
  const int e = (__float_as_int(largest) >> 23) & 255;
  return e == 0 || e == 255 ? 1.f : __int_as_float((254 - e < 1 ? 1 : 254 - e) << 23);
}

// ---- shrink: H[place][j] = factor sum_k drop(x)[row][k] W[g][j][k] -------------------------------------------------------------------------
// A workgroup of 8 waves; `split` of them share a tile of rows and take its steps of 128 bytes in turn.  RT: tiles of 16 ranks.
// H: [places][16 RT] (for `expand`) and / or HT: [16 RT][ht_ld] (for `outer`), zeros behind the rank.
struct ShrinkArgs {
  const void *x, *w;
  int64_t x_stride, w_group;      // elements between rows; between the adapters' matrices
  int width, w_ld, rank, split;
  const float *scales;            // per adapter, or null
  float factor;
  float *h, *ht;
  int64_t ht_ld;
  Dropout drop;
  Plan plan;
};
template <typename T, int RT, bool DROP>
__global__ void __launch_bounds__(512) lowrank_shrink_kernel(ShrinkArgs q) {
  __shared__ float s_sum[8][RT * 2 * 4][64];
  constexpr int NE = Span<T>::N, STEP = 4 * NE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, quad = lane >> 4;
  const int part = wave % q.split, which = blockIdx.x * (8 / q.split) + wave / q.split;
  int4 tile = {0, 0, 0, 0};
  if (which < q.plan.max_tiles) tile = q.plan.tile[which];
  const bool live = tile.z > 0 && tile.x < q.plan.n_adapters;
  f32x4 acc[RT][2];
#pragma unroll
  for (int r = 0; r < RT; ++r) acc[r][0] = acc[r][1] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (live) {
    if (DROP) dropout_counter(q.drop);
    const T *px[2];
    uint32_t row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {      // a place behind the tile reads its last row: its sums are not written
      const int i = t * 16 + c;
      row[t] = (uint32_t)q.plan.order[tile.y + (i < tile.z ? i : tile.z - 1)];
      px[t] = (const T *)q.x + (int64_t)row[t] * q.x_stride;
    }
    const T *pw[RT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int j = r * 16 + c;
      pw[r] = (const T *)q.w + tile.x * q.w_group + (int64_t)(j < q.rank ? j : q.rank - 1) * q.w_ld;
    }
    const int steps = (q.width + STEP - 1) / STEP;
    for (int s = part; s < steps; s += q.split) {
      const int k = s * STEP + quad * NE, valid = q.width - k;
      Span<T> xs[2], ws[RT];
      if ((s + 1) * STEP <= q.width) {
#pragma unroll
        for (int t = 0; t < 2; ++t) load_some<T, NE>(px[t] + k, NE, xs[t].v);
#pragma unroll
        for (int r = 0; r < RT; ++r) load_some<T, NE>(pw[r] + k, NE, ws[r].v);
      } else {
#pragma unroll
        for (int t = 0; t < 2; ++t) load_part<T, NE>(px[t] + k, valid, xs[t].v);
#pragma unroll
        for (int r = 0; r < RT; ++r) load_part<T, NE>(pw[r] + k, valid, ws[r].v);
      }
      if (DROP) {
#pragma unroll
        for (int t = 0; t < 2; ++t) drop_some<T, NE>(q.drop, row[t], k, xs[t].v);
      }
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < NE; i += 8) acc[r][t] = mma8(ws[r].v + i, xs[t].v + i, acc[r][t]);
    }
  }
  if (q.split > 1) {
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) s_sum[wave][(r * 2 + t) * 4 + i][lane] = acc[r][t][i];
    __syncthreads();
    if (part != 0) return;
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = acc[r][t][i];
          for (int w = 1; w < q.split; ++w) v += s_sum[wave + w][(r * 2 + t) * 4 + i][lane];
          acc[r][t][i] = v;
        }
  }
  if (!live) return;
  const float f = q.factor * (q.scales != nullptr ? q.scales[tile.x] : 1.f);
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int i0 = t * 16 + c;
    if (i0 >= tile.z) continue;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      f32x4 v;
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = r * 16 + quad * 4 + i < q.rank ? acc[r][t][i] * f : 0.f;
      if (q.h != nullptr) *reinterpret_cast<f32x4 *>(q.h + (int64_t)(tile.y + i0) * (16 * RT) + r * 16 + quad * 4) = v;
      if (q.ht != nullptr) {
#pragma unroll
        for (int i = 0; i < 4; ++i) q.ht[(int64_t)(r * 16 + quad * 4 + i) * q.ht_ld + tile.y + i0] = v[i];
      }
    }
  }
}

// ---- expand: y[row][n] = base[row][n] + sum_j H[place][j] W[g][n][j] -------------------------------------------------------------------------
// A wave takes 64 columns of a tile at a time: four matrix tiles whose rows are columns of y in the order that leaves a lane 16 neighbours.
struct ExpandArgs {
  const float *h;
  const void *w, *base;
  void *y;
  int64_t w_group, base_stride, y_stride;
  int width, w_ld, rank;
  const float *scales;
  Dropout drop;      // on the result (dx), DROP only
  Plan plan;
};
template <typename T, int RT, bool DROP>
__global__ void __launch_bounds__(256) lowrank_expand_kernel(ExpandArgs q) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, quad = lane >> 4;
  const int4 tile = q.plan.tile[blockIdx.x];
  if (tile.z == 0) return;
  const bool idle = tile.x == q.plan.n_adapters;
  if (idle && q.base == q.y) return;      // in place: not touched
  int64_t row[2];
  bool mine[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int i = t * 16 + c;
    mine[t] = i < tile.z;
    row[t] = q.plan.order[tile.y + (mine[t] ? i : tile.z - 1)];
  }
  const int chunks = (q.width + 63) / 64;
  const T *base = (const T *)q.base;
  T *y = (T *)q.y;
  if (idle) {
    for (int ch = blockIdx.y * 4 + wave; ch < chunks; ch += gridDim.y * 4) {
      const int n = ch * 64 + quad * 16, valid = q.width - n;
      if (valid <= 0) continue;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        T b[16];
        if (base != nullptr) load_some<T, 16>(base + row[t] * q.base_stride + n, valid, b);
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = base != nullptr ? (float)b[i] : 0.f;
        if (mine[t]) store_some<T, 16>(y + row[t] * q.y_stride + n, valid, v);
      }
    }
    return;
  }
  if (DROP) dropout_counter(q.drop);
  const float scale = (q.scales != nullptr ? q.scales[tile.x] : 1.f) * (DROP ? q.drop.scale : 1.f);
  const T *w = (const T *)q.w + tile.x * q.w_group;
  // h of the lane's row as the instruction wants it.  16 bits: 8 ranks a lane, 32 an instruction, high and low parts (a rank of at most 16: both in
  // one instruction).  32 bits: 4 ranks a lane, 16 a group of four instructions.
  constexpr bool WIDE = sizeof(T) == 4;
  constexpr int KB = WIDE ? RT : (RT == 1 ? 1 : RT / 2), PER = WIDE ? 4 : 8;
  T hi[2][KB][PER], lo[2][KB][PER];
  float back[2];
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const float *ph = q.h + (int64_t)(tile.y + (mine[t] ? t * 16 + c : tile.z - 1)) * (16 * RT);
    float f[KB][PER];
    float largest = 0.f;
#pragma unroll
    for (int b = 0; b < KB; ++b) {
      const int j = WIDE ? b * 16 + quad * 4 : (RT == 1 ? (quad & 1) * 8 : b * 32 + quad * 8);
#pragma unroll
      for (int i = 0; i < PER; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(ph + j + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[b][i + e] = v[e] * scale; largest = fmaxf(largest, fabsf(f[b][i + e])); }
      }
    }
    float down = 1.f;
    back[t] = 1.f;
    if (sizeof(T) == 2 && __is_same(T, f16_t)) {
      largest = fmaxf(largest, __shfl_xor(largest, 16));
      largest = fmaxf(largest, __shfl_xor(largest, 32));
      down = scale_to_one(largest);
      back[t] = 1.f / down;
    }
#pragma unroll
    for (int b = 0; b < KB; ++b)
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const float v = f[b][i] * down;
        hi[t][b][i] = (T)v;
        lo[t][b][i] = (T)(v - (float)hi[t][b][i]);
        if (!WIDE && RT == 1) hi[t][b][i] = quad < 2 ? hi[t][b][i] : lo[t][b][i];
      }
  }
  for (int ch = blockIdx.y * 4 + wave; ch < chunks; ch += gridDim.y * 4) {
    const int n = ch * 64 + quad * 16, valid = q.width - n;
    T b[2][16];
    if (base != nullptr && valid > 0) {
#pragma unroll
      for (int t = 0; t < 2; ++t) load_some<T, 16>(base + row[t] * q.base_stride + n, valid, b[t]);
    }
    float v[2][16];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int col = ch * 64 + (c >> 2) * 16 + m * 4 + (c & 3);      // the column that this lane's weights belong to
      const T *pw = w + (int64_t)(col < q.width ? col : q.width - 1) * q.w_ld;
      f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        const int j = WIDE ? k * 16 + quad * 4 : (RT == 1 ? (quad & 1) * 8 : k * 32 + quad * 8);
        T u[PER];
        load_some<T, PER>(pw + j, q.rank - j, u);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[i], hi[t][k][i], acc[t], 0, 0, 0);
          } else {
            acc[t] = mma8(u, hi[t][k], acc[t]);
            if (RT > 1) acc[t] = mma8(u, lo[t][k], acc[t]);
          }
        }
      }
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[t][m * 4 + i] = acc[t][i];
    }
    if (valid <= 0) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if (!mine[t]) continue;
#pragma unroll
      for (int i = 0; i < 16; ++i) v[t][i] = v[t][i] * back[t] + (base != nullptr ? (float)b[t][i] : 0.f);
      if (DROP) drop_some<float, 16>(q.drop, (uint32_t)row[t], n, v[t]);
      store_some<T, 16>(y + row[t] * q.y_stride + n, valid, v[t]);
    }
  }
}

// ---- outer: sum over an adapter's rows of UT[j][place] V[row][c] ----------------------------------------------------------------------------
// A workgroup of 8 waves owns a chunk of rows and 16 lanes x 16 bytes of columns; its waves take 32 rows in turn and meet in LDS.
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
template <typename T, int RT>
__global__ void __launch_bounds__(512) lowrank_outer_kernel(OuterArgs q) {
  constexpr int VE = 16 / sizeof(T), COLS = 16 * VE;      // elements of a lane's piece, columns of a workgroup
  __shared__ float s_sum[4][VE * 4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, quad = lane >> 4;
  const int block = blockIdx.x % q.blocks;
  const int4 chunk = q.plan.chunk[blockIdx.x / q.blocks];
  if (chunk.z == 0) return;
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
  const int steps = (chunk.z + 31) / 32;
  const bool columns_whole = col0 + COLS <= s.width;
  for (int st = wave; st < steps; st += 8) {
    const int at = st * 32 + quad * 8;      // the lane's 8 rows
    const bool whole = st * 32 + 32 <= chunk.z;
    T v[8][VE];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int k = whole || at + i < chunk.z ? at + i : chunk.z - 1;
      const uint32_t row = (uint32_t)q.plan.order[chunk.y + k];
      const T *pv = (const T *)s.v + (int64_t)row * s.v_stride + col;
      if (columns_whole) load_piece<T, VE>(pv, v[i]);
      else load_part<T, VE>(pv, valid, v[i]);
      if (drop) drop_some<T, VE>(q.drop, row, col, v[i]);
      if (!whole) {      // rows behind the chunk: nothing, whatever the row read in their place holds
#pragma unroll
        for (int e = 0; e < VE; ++e) v[i][e] = at + i < chunk.z ? v[i][e] : (T)0.f;
      }
    }
    float u[RT][8];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const float *pu = s.ut + (int64_t)(rank0 + r * 16 + c) * q.ut_ld + chunk.y + at;
      load_some<float, 8>(pu, whole ? 8 : chunk.z - at, u[r]);
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 8; ++i) acc[r][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(u[r][i], v[i][e], acc[r][e], 0, 0, 0);
    } else {
      constexpr bool HALF = __is_same(T, f16_t);
      float down = 1.f, up = 1.f;
      if (HALF) {      // one power of two for the step: the sums of other steps keep their own
        float largest = 0.f;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
          for (int i = 0; i < 8; ++i) largest = fmaxf(largest, fabsf(u[r][i]));
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) largest = fmaxf(largest, __shfl_xor(largest, o));
        down = scale_to_one(largest);
        up = 1.f / down;
      }
      T hi[RT][8], lo[RT][8];
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float t = u[r][i] * down;
          hi[r][i] = (T)t;
          lo[r][i] = (T)(t - (float)hi[r][i]);
        }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        T b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) b[i] = v[i][e];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          if (HALF) {
            f32x4 t = mma8(lo[r], b, f32x4{0.f, 0.f, 0.f, 0.f});
            t = mma8(hi[r], b, t);
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[r][e][i] = fmaf(t[i], up, acc[r][e][i]);
          } else {
            acc[r][e] = mma8(lo[r], b, acc[r][e]);
            acc[r][e] = mma8(hi[r], b, acc[r][e]);
          }
        }
      }
    }
  }
  // the waves' sums: 4 + 4, 2 + 2, 1 + 1, one tile of ranks at a time
#pragma unroll
  for (int r = 0; r < RT; ++r) {
    for (int half = 4; half > 0; half >>= 1) {
      __syncthreads();
      if (wave >= half && wave < 2 * half) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) s_sum[wave - half][e * 4 + i][lane] = acc[r][e][i];
      }
      __syncthreads();
      if (wave < half) {
#pragma unroll
        for (int e = 0; e < VE; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[r][e][i] += s_sum[wave][e * 4 + i][lane];
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
// the adapters that `outer` did not finish: the sum of several chunks, in their order, or zeros where there are no rows
struct SumArgs {
  OuterSide side[2];
  int rank, rank_padded, blocks0;
  Plan plan;
};
template <typename T>
__global__ void __launch_bounds__(256) lowrank_sum_kernel(SumArgs q) {
  const bool second = (int)blockIdx.x >= q.blocks0;
  const OuterSide &s = q.side[second];
  const int g = blockIdx.y;
  const int2 slots = q.plan.slots[g];
  if (slots.y == 1) return;
  const int64_t i = (int64_t)((int)blockIdx.x - (second ? q.blocks0 : 0)) * 256 + threadIdx.x, n = (int64_t)q.rank * s.width;
  if (i >= n) return;
  float v = 0.f;
  if (slots.y > 1) {
    const int64_t each = (int64_t)q.rank_padded * s.width;
    const int64_t at = s.columns_first ? i / q.rank * q.rank_padded + i % q.rank : i;
    const float *p = s.part + slots.x * each + at;
    for (int k = 0; k < slots.y; ++k) v += p[k * each];
  }
  ((T *)s.out)[g * n + i] = (T)v;
}

// ---- weights turned for the backward pass: A [g][r][k] -> [g][k][RP] (zeros behind the rank), B [g][n][r] -> [g][RP'][n] ----------------------
struct TurnArgs {
  const void *in[2];
  void *out[2];
  int rows[2], cols[2], out_ld[2];      // of one adapter's matrix, and of the turned one
  int blocks0;
  Plan plan;
};
template <typename T>
__global__ void __launch_bounds__(256) lowrank_turn_kernel(TurnArgs q) {
  __shared__ T s[64][65];
  const int g = blockIdx.y;
  if (q.plan.slots[g].y == 0) return;      // nobody reads it
  const int k = (int)blockIdx.x >= q.blocks0;
  const int tiles_c = (q.cols[k] + 63) / 64, b = (int)blockIdx.x - (k ? q.blocks0 : 0), r0 = b / tiles_c * 64, c0 = b % tiles_c * 64;
  const T *in = (const T *)q.in[k] + (int64_t)g * q.rows[k] * q.cols[k];
  T *out = (T *)q.out[k] + (int64_t)g * q.cols[k] * q.out_ld[k];
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int r = r0 + i / 64, c = c0 + i % 64;
    s[i / 64][i % 64] = r < q.rows[k] && c < q.cols[k] ? in[(int64_t)r * q.cols[k] + c] : (T)0.f;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 4096; i += 256) {
    const int c = c0 + i / 64, r = r0 + i % 64;
    if (c < q.cols[k] && r < q.out_ld[k]) out[(int64_t)c * q.out_ld[k] + r] = s[i % 64][i / 64];
  }
}

// ---- a few rows without gradients: no order, a workgroup per row ----------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(1024) lowrank_row_shrink_kernel(Ids ids, const T *__restrict__ x, int64_t x_stride, const T *__restrict__ a, int width, int rank,
                                                                  const float *__restrict__ scales, Dropout drop, float *__restrict__ h) {
  constexpr int NE = 16 / sizeof(T);
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, j = blockIdx.y * 16 + (threadIdx.x >> 6), g = group_of(ids, row);
  if (j >= rank || g == ids.n_adapters) return;
  dropout_counter(drop);
  const T *px = x + row * x_stride, *pa = a + ((int64_t)g * rank + j) * width;
  float s = 0.f;
#pragma unroll 4
  for (int k = lane * NE; k < width; k += 64 * NE) {
    T u[NE], v[NE];
    load_some<T, NE>(px + k, width - k, u);
    load_some<T, NE>(pa + k, width - k, v);
    if (drop.threshold != 0) drop_some<T, NE>(drop, (uint32_t)row, k, u);
#pragma unroll
    for (int i = 0; i < NE; ++i) s = fmaf((float)u[i], (float)v[i], s);
  }
  s = wave_sum_to_lane63(s);
  if (lane == 63) h[row * rank + j] = s * (scales != nullptr ? scales[g] : 1.f) * (drop.threshold != 0 ? drop.scale : 1.f);
}
// 16 columns a wave and step, four lanes to a column
template <typename T>
__global__ void __launch_bounds__(256) lowrank_row_expand_kernel(Ids ids, const float *__restrict__ h, const T *__restrict__ b, int width, int rank, const T *base,
                                                                 int64_t base_stride, T *y, int64_t y_stride) {
  const int64_t row = blockIdx.x;
  const int g = group_of(ids, row), sub = threadIdx.x & 3;
  if (g == ids.n_adapters && base == y) return;
  const float *ph = h + row * rank;
  for (int n = blockIdx.y * 64 + (threadIdx.x >> 2); n < width; n += gridDim.y * 64) {
    float s = 0.f;
    if (g < ids.n_adapters) {
      const T *pb = b + ((int64_t)g * width + n) * rank;
      for (int j = sub * 8; j < rank; j += 32) {
        T v[8];
        load_some<T, 8>(pb + j, rank - j, v);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (j + i < rank) s = fmaf(ph[j + i], (float)v[i], s);
      }
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    if (sub == 0) y[row * y_stride + n] = (T)(s + (base != nullptr ? (float)base[row * base_stride + n] : 0.f));
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------------------------
static constexpr int64_t LR_FEW_ROWS = 64;

static int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
#define GSDF_BY_RANK(rt, ...)                                 \
  switch (rt) {                                               \
    case 1: { constexpr int RT = 1; __VA_ARGS__; break; }     \
    case 2: { constexpr int RT = 2; __VA_ARGS__; break; }     \
    case 4: { constexpr int RT = 4; __VA_ARGS__; break; }     \
    default: { constexpr int RT = 8; __VA_ARGS__; break; }    \
  }

// a buffer in pieces of 256 bytes
struct Carve {
  char *at;
  size_t used = 0;
  explicit Carve(void *p) : at((char *)p) {}
  template <typename P>
  P *take(size_t bytes) { P *r = (P *)(at + used); used += align_up(bytes, 256); return r; }
};

struct Lowrank {
  gsdf_lowrank_args a;
  Dropout drop;
  Plan plan;
  int rt, rp, es;
  int64_t ht_ld;
  // saved by the forward pass
  float *ht;
  // workspace
  float *h, *dh, *dht, *part[2];
  void *turned[2];
  size_t save_bytes, fwd_ws_bytes, bwd_ws_bytes;
};
static int lowrank_check(const gsdf_lowrank_args *a) {
  GSDF_REQUIRE(a != nullptr, "lowrank: args is NULL");
  GSDF_REQUIRE(a->rows >= 0 && a->rows < (1ll << 28), "lowrank: %lld rows outside [0, 2^28)", (long long)a->rows);
  GSDF_REQUIRE(a->n_in >= 1 && a->n_out >= 1 && a->n_in < (1 << 22) && a->n_out < (1 << 22), "lowrank: widths %d -> %d outside [1, 2^22)", a->n_in, a->n_out);
  GSDF_REQUIRE(a->rank >= 1 && a->rank <= GSDF_LOWRANK_MAX_RANK, "lowrank: rank %d outside [1, %d]", a->rank, GSDF_LOWRANK_MAX_RANK);
  GSDF_REQUIRE(a->n_adapters >= 1 && a->n_adapters <= GSDF_LOWRANK_MAX_ADAPTERS, "lowrank: %d adapters outside [1, %d]", a->n_adapters, GSDF_LOWRANK_MAX_ADAPTERS);
  GSDF_REQUIRE(known_dtype(a->dtype), "lowrank: unknown element type %d", a->dtype);
  GSDF_REQUIRE(a->p >= 0.0 && a->p <= 1.0, "lowrank: p = %g outside [0, 1]", a->p);
  GSDF_REQUIRE(a->rows == 0 || (a->x != nullptr && a->ids != nullptr), "lowrank: x and ids are required");
  GSDF_REQUIRE(a->a != nullptr && a->b != nullptr, "lowrank: a and b are required");
  GSDF_REQUIRE(a->rows <= 1 || a->x_stride >= 0, "lowrank: row stride %lld of x", (long long)a->x_stride);
  return GSDF_OK;
}
// where everything lies in the saved buffer and in the workspace (`training`: the plan is in the saved buffer, else in the workspace)
static void lowrank_layout(Lowrank *q, const gsdf_lowrank_args *a, void *save, void *ws, bool training) {
  q->a = *a;
  q->drop = make_dropout(a->p, a->seed, a->offset, a->offset_dev);
  q->rt = rank_tiles(a->rank);
  q->rp = 16 * q->rt;
  q->es = a->dtype == GSDF_F32 ? 4 : 2;
  q->ht_ld = (int64_t)align_up((size_t)a->rows, 4);
  Plan unused;
  const size_t plan_bytes = plan_layout(&unused, nullptr, a->rows, a->n_adapters), h_bytes = (size_t)a->rows * q->rp * 4, ht_bytes = (size_t)q->ht_ld * q->rp * 4;
  Carve s(save), f(ws), b(ws);
  void *plan_saved = s.take<char>(plan_bytes);
  q->ht = s.take<float>(ht_bytes);
  q->save_bytes = s.used;
  void *plan_ws = f.take<char>(plan_bytes);
  q->h = f.take<float>(h_bytes);
  q->fwd_ws_bytes = f.used;
  plan_layout(&q->plan, training ? plan_saved : plan_ws, a->rows, a->n_adapters);
  const size_t weights = (size_t)a->n_adapters * q->rp * q->es, part = (size_t)plan_max_slots(a->rows, a->n_adapters) * q->rp * 4;
  q->dh = b.take<float>(h_bytes);
  q->dht = b.take<float>(ht_bytes);
  q->turned[0] = b.take<char>(weights * a->n_in);
  q->turned[1] = b.take<char>(weights * a->n_out);
  q->part[0] = b.take<float>(part * a->n_in);
  q->part[1] = b.take<float>(part * a->n_out);
  q->bwd_ws_bytes = b.used;
}

template <typename T>
static void shrink_launch(const Lowrank &q, const void *x, int64_t x_stride, int width, const void *w, int64_t w_group, int w_ld, const float *scales, bool drop, float *h,
                          float *ht, hipStream_t stream) {
  ShrinkArgs s;
  s.x = x; s.w = w; s.x_stride = x_stride; s.w_group = w_group; s.width = width; s.w_ld = w_ld; s.rank = q.a.rank;
  s.scales = scales; s.factor = drop ? q.drop.scale : 1.f; s.h = h; s.ht = ht; s.ht_ld = q.ht_ld; s.drop = q.drop; s.plan = q.plan;
  const int steps = (int)ceil_div(width, 128 / (int)sizeof(T));
  s.split = steps >= 8 ? 8 : steps >= 4 ? 4 : steps >= 2 ? 2 : 1;
  const unsigned grid = (unsigned)ceil_div(q.plan.max_tiles, 8 / s.split);
  GSDF_BY_RANK(q.rt, {
    if (drop) lowrank_shrink_kernel<T, RT, true><<<grid, 512, 0, stream>>>(s);
    else lowrank_shrink_kernel<T, RT, false><<<grid, 512, 0, stream>>>(s);
  });
}
template <typename T>
static void expand_launch(const Lowrank &q, const float *h, const void *w, int64_t w_group, int w_ld, int ranks, int width, const float *scales, const void *base,
                          int64_t base_stride, void *y, int64_t y_stride, bool drop, hipStream_t stream) {
  ExpandArgs s;
  s.h = h; s.w = w; s.base = base; s.y = y; s.w_group = w_group; s.base_stride = base_stride; s.y_stride = y_stride; s.width = width; s.w_ld = w_ld; s.rank = ranks;
  s.scales = scales; s.drop = q.drop; s.plan = q.plan;
  const int64_t chunks = ceil_div(width, 64);
  const dim3 grid((unsigned)q.plan.max_tiles, (unsigned)ceil_div(chunks, chunks >= 16 ? 16 : 4));
  GSDF_BY_RANK(q.rt, {
    if (drop) lowrank_expand_kernel<T, RT, true><<<grid, 256, 0, stream>>>(s);
    else lowrank_expand_kernel<T, RT, false><<<grid, 256, 0, stream>>>(s);
  });
}

template <typename T>
static void lowrank_fwd(const Lowrank &q, const void *base, int64_t base_stride, void *y, int64_t y_stride, bool training, hipStream_t stream) {
  const gsdf_lowrank_args &a = q.a;
  const Ids ids = {a.ids, a.ids_64, a.n_adapters};
  if (!training && a.rows <= LR_FEW_ROWS) {
    lowrank_row_shrink_kernel<T><<<dim3((unsigned)a.rows, (unsigned)ceil_div(a.rank, 16)), 1024, 0, stream>>>(ids, (const T *)a.x, a.x_stride, (const T *)a.a, a.n_in, a.rank,
                                                                                                         a.scales, q.drop, q.h);
    lowrank_row_expand_kernel<T><<<dim3((unsigned)a.rows, (unsigned)(ceil_div(a.n_out, 64) < 4096 ? ceil_div(a.n_out, 64) : 4096)), 256, 0, stream>>>(
        ids, q.h, (const T *)a.b, a.n_out, a.rank, (const T *)base,
                                                                                                         base_stride, (T *)y, y_stride);
    return;
  }
  plan_launch(q.plan, ids, stream);
  shrink_launch<T>(q, a.x, a.x_stride, a.n_in, a.a, (int64_t)a.rank * a.n_in, a.n_in, a.scales, q.drop.threshold != 0, q.h, training ? q.ht : nullptr, stream);
  expand_launch<T>(q, q.h, a.b, (int64_t)a.n_out * a.rank, a.rank, a.rank, a.n_out, nullptr, base, base_stride, y, y_stride, false, stream);
}

template <typename T>
static void lowrank_bwd(const Lowrank &q, const void *dy, int64_t dy_stride, void *dx, int64_t dx_stride, void *da, void *db, hipStream_t stream) {
  const gsdf_lowrank_args &a = q.a;
  const bool drop = q.drop.threshold != 0;
  const unsigned G = (unsigned)a.n_adapters;
  if (a.rows > 0 && (dx != nullptr || da != nullptr)) {
    TurnArgs t;
    t.in[0] = a.a; t.out[0] = q.turned[0]; t.rows[0] = a.rank; t.cols[0] = a.n_in; t.out_ld[0] = q.rp;
    t.in[1] = a.b; t.out[1] = q.turned[1]; t.rows[1] = a.n_out; t.cols[1] = a.rank; t.out_ld[1] = a.n_out;
    t.blocks0 = dx != nullptr ? (int)(ceil_div(q.rp, 64) * ceil_div(a.n_in, 64)) : 0;
    t.plan = q.plan;
    const unsigned blocks1 = (unsigned)(ceil_div(a.n_out, 64) * ceil_div(a.rank, 64));
    lowrank_turn_kernel<T><<<dim3((unsigned)t.blocks0 + blocks1, G), 256, 0, stream>>>(t);
    shrink_launch<T>(q, dy, dy_stride, a.n_out, q.turned[1], (int64_t)a.rank * a.n_out, a.n_out, a.scales, false, q.dh, da != nullptr ? q.dht : nullptr, stream);
  }
  if (a.rows > 0 && dx != nullptr)
    expand_launch<T>(q, q.dh, q.turned[0], (int64_t)a.n_in * q.rp, q.rp, q.rp, a.n_in, nullptr, nullptr, 0, dx, dx_stride, drop, stream);
  if (da == nullptr && db == nullptr) return;
  constexpr int COLS = 16 * (16 / (int)sizeof(T));
  OuterArgs o;
  o.side[0] = {q.dht, a.x, a.x_stride, a.n_in, drop, 0, da, q.part[0]};
  o.side[1] = {q.ht, dy, dy_stride, a.n_out, 0, 1, db, q.part[1]};
  o.ut_ld = q.ht_ld; o.rank = a.rank; o.rank_padded = q.rp; o.drop = q.drop; o.plan = q.plan;
  o.blocks0 = da != nullptr ? (int)ceil_div(a.n_in, COLS) : 0;
  const unsigned blocks1 = db != nullptr ? (unsigned)ceil_div(a.n_out, COLS) : 0;
  o.blocks = o.blocks0 + (int)blocks1;
  if (a.rows > 0) {
    const dim3 grid((unsigned)o.blocks * (unsigned)q.plan.max_chunks, q.rt == 8 ? 2 : 1);
    switch (q.rt) {
      case 1: lowrank_outer_kernel<T, 1><<<grid, 512, 0, stream>>>(o); break;
      case 2: lowrank_outer_kernel<T, 2><<<grid, 512, 0, stream>>>(o); break;
      default: lowrank_outer_kernel<T, 4><<<grid, 512, 0, stream>>>(o); break;
    }
  }
  SumArgs s;
  s.side[0] = o.side[0]; s.side[1] = o.side[1]; s.rank = a.rank; s.rank_padded = q.rp; s.plan = q.plan;
  s.blocks0 = da != nullptr ? (int)ceil_div((int64_t)a.rank * a.n_in, 256) : 0;
  const unsigned sum1 = db != nullptr ? (unsigned)ceil_div((int64_t)a.rank * a.n_out, 256) : 0;
  lowrank_sum_kernel<T><<<dim3((unsigned)s.blocks0 + sum1, G), 256, 0, stream>>>(s);
}

}  // namespace gsdf

extern "C" size_t gsdf_lowrank_save_bytes(const gsdf_lowrank_args *a) {
  gsdf::Lowrank q;
  if (gsdf::lowrank_check(a) != GSDF_OK) return 0;
  gsdf::lowrank_layout(&q, a, nullptr, nullptr, true);
  return q.save_bytes;
}
extern "C" size_t gsdf_lowrank_fwd_ws_bytes(const gsdf_lowrank_args *a) {
  gsdf::Lowrank q;
  if (gsdf::lowrank_check(a) != GSDF_OK) return 0;
  gsdf::lowrank_layout(&q, a, nullptr, nullptr, true);
  return q.fwd_ws_bytes;
}
extern "C" size_t gsdf_lowrank_bwd_ws_bytes(const gsdf_lowrank_args *a) {
  gsdf::Lowrank q;
  if (gsdf::lowrank_check(a) != GSDF_OK) return 0;
  gsdf::lowrank_layout(&q, a, nullptr, nullptr, true);
  return q.bwd_ws_bytes;
}

extern "C" int gsdf_lowrank_fwd(const gsdf_lowrank_args *args, const void *base, int64_t base_stride, void *y, int64_t y_stride, void *save, void *ws,
                                gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  if (const int e = lowrank_check(args)) return e;
  GSDF_REQUIRE(args->rows == 0 || (y != nullptr && ws != nullptr), "lowrank_fwd: y and the workspace are required");
  GSDF_REQUIRE(args->rows <= 1 || (y_stride >= args->n_out && (base == nullptr || base_stride >= 0)), "lowrank_fwd: row strides %lld -> %lld of %d columns",
               (long long)base_stride, (long long)y_stride, args->n_out);
  GSDF_REQUIRE(base != y || args->rows <= 1 || base_stride == y_stride, "lowrank_fwd: y is base, but their row strides are not the same");
  GSDF_TIMED("gsdf_lowrank_fwd");
  if (args->rows == 0 && save == nullptr) return GSDF_OK;
  Lowrank q;
  lowrank_layout(&q, args, save, ws, save != nullptr);
  if (args->rows == 0) {      // the backward pass asks the plan which adapters have rows
    plan_launch(q.plan, Ids{args->ids, args->ids_64, args->n_adapters}, stream);
  } else {
    GSDF_BY_DTYPE(args->dtype, lowrank_fwd<T>(q, base, base_stride, y, y_stride, save != nullptr, stream));
  }
  GSDF_CHECK_LAUNCH("lowrank_fwd");
  return GSDF_OK;
}

extern "C" int gsdf_lowrank_bwd(const gsdf_lowrank_args *args, const void *dy, int64_t dy_stride, const void *save, void *dx, int64_t dx_stride, void *da,
                                void *db, void *ws, gsdf_stream_t stream_) {
  using namespace gsdf;
  hipStream_t stream = (hipStream_t)stream_;
  if (const int e = lowrank_check(args)) return e;
  GSDF_REQUIRE(ws != nullptr && save != nullptr && (args->rows == 0 || dy != nullptr), "lowrank_bwd: dy, the forward's saved buffer and the workspace are required");
  GSDF_REQUIRE(args->rows <= 1 || (dy_stride >= 0 && (dx == nullptr || dx_stride >= args->n_in)), "lowrank_bwd: row strides %lld, %lld", (long long)dy_stride,
               (long long)dx_stride);
  GSDF_TIMED("gsdf_lowrank_bwd");
  Lowrank q;
  lowrank_layout(&q, args, const_cast<void *>(save), ws, true);
  GSDF_BY_DTYPE(args->dtype, lowrank_bwd<T>(q, dy, dy_stride, dx, dx_stride, da, db, stream));
  GSDF_CHECK_LAUNCH("lowrank_bwd");
  return GSDF_OK;
}
