// lowrank.hip — low-rank adapters of many requests at once beside a shared projection:
//     y_t = base_t + s_g B_g h_t,   h_t = A_g drop(x_t),   g = ids[t]
// backward:  dh_t = s_g B_g^T dy_t,  dx_t = drop'(A_g^T dh_t),  dA_g = sum_t dh_t drop(x_t)^T,  dB_g = s_g sum_t dy_t h_t^T.
// The products are in lowrank_kernels.h; here are the order of the rows and the C entries.
#include "lowrank.h"

namespace gsdf {

// inclusive sums over the lanes of the wave, without LDS
__device__ __forceinline__ int wave_scan(int v) {
  v += (int)dpp_mov_u<0x111>((unsigned)v);                   // row_shr:1, 2, 4, 8: inside rows of 16 lanes
  v += (int)dpp_mov_u<0x112>((unsigned)v);
  v += (int)dpp_mov_u<0x114>((unsigned)v);
  v += (int)dpp_mov_u<0x118>((unsigned)v);
  v += (int)dpp_mov_u<0x142, 0xA, 0xF, false>((unsigned)v);  // row_bcast:15 into rows 1 and 3
  v += (int)dpp_mov_u<0x143, 0xC, 0xF, false>((unsigned)v);  // row_bcast:31 into rows 2 and 3
  return v;
}
// exclusive sums of C numbers (at most 4) over the 1024 threads of the workgroup; totals in `sum`
template <int C>
__device__ __forceinline__ void block_scan(int (&v)[C], int (&sum)[C], int4 *s_w) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int i[C], before[C];
#pragma unroll
  for (int c = 0; c < C; ++c) { i[c] = wave_scan(v[c]); before[c] = sum[c] = 0; }
  if (lane == 63) s_w[wave] = int4{i[0], C > 1 ? i[C > 1 ? 1 : 0] : 0, C > 2 ? i[C > 2 ? 2 : 0] : 0, C > 3 ? i[C > 3 ? 3 : 0] : 0};
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const int4 t = s_w[w];
    const int part[4] = {t.x, t.y, t.z, t.w};
#pragma unroll
    for (int c = 0; c < C; ++c) {
      before[c] = w == wave ? sum[c] : before[c];
      sum[c] += part[c];
    }
  }
  __syncthreads();
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = before[c] + i[c] - v[c];
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

template <typename E>
__device__ __forceinline__ void pack_block(const PackArgs &q, int block) {
  typedef E vec __attribute__((ext_vector_type(16 / sizeof(E))));
  constexpr int N = 16 / sizeof(E);
  const int each = q.blocks[0] + q.blocks[1] + q.blocks[2], g = block / each;
  int b = block % each;
  const E *a = (const E *)q.a + (int64_t)g * q.rank * q.n_in, *bm = (const E *)q.b + (int64_t)g * q.n_out * q.rank;
  vec v;
  if (b < q.blocks[0] + q.blocks[1]) {      // fragments of A, or of B^T
    const bool second = b >= q.blocks[0];
    const int p = (b - (second ? q.blocks[0] : 0)) * 1024 + threadIdx.x, width = second ? q.n_out : q.n_in, steps = (width + 8 * N - 1) / (8 * N);
    const int lane = p & 63, r = (p >> 7) & (q.rt - 1), step = (p >> 7) / q.rt;
    if (step >= steps) return;
    const int j = r * 16 + (lane & 15), k = step * 8 * N + ((p >> 6) & 1) * 4 * N + (lane >> 4) * N;
    if (!second && j < q.rank && k + N <= width) v = *reinterpret_cast<const typename Piece<E, N>::any *>(a + (int64_t)j * width + k);
    else
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const bool in = j < q.rank && k + i < width;
      const int64_t at = in ? (second ? (int64_t)(k + i) * q.rank + j : (int64_t)j * width + k + i) : 0;
      const E t = second ? bm[at] : a[at];
      v[i] = in ? t : (E)0;
    }
    reinterpret_cast<vec *>(second ? q.b_frag : q.a_frag)[((int64_t)g * steps * q.rt << 7) + p] = v;
  } else {                                   // A^T: neighbouring lanes have neighbouring columns of A
    b -= q.blocks[0] + q.blocks[1];
    const int p = b * 1024 + threadIdx.x, jp = p / q.n_in, k = p % q.n_in, per_row = q.rt * 16 / N;
    if (jp >= per_row) return;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int j = jp * N + i;
      const E t = a[j < q.rank ? (int64_t)j * q.n_in + k : 0];
      v[i] = j < q.rank ? t : (E)0;
    }
    reinterpret_cast<vec *>(q.a_turned)[((int64_t)g * q.n_in + k) * per_row + jp] = v;
  }
}

// The plan takes two launches: each workgroup counts its share of the rows; then each adds up the counts of all (they are few), finds where its own rows
// go and puts them there.  Up to 16384 rows each workgroup counts all rows instead, in one launch.  A chain of waits, not bytes: 1111 rows of 5 adapters 7.6 us,
// 8192 of 8 11 us, 300000 of 6 4.7 and 9.4 us.
__global__ void __launch_bounds__(1024) lowrank_plan_count_kernel(Plan p, Ids ids, PackArgs pack) {
  extern __shared__ int s_hist[];      // [n_adapters + 1]
  if ((int)blockIdx.x >= p.blocks) {
    if (pack.es == 4) pack_block<uint32_t>(pack, blockIdx.x - p.blocks);
    else pack_block<unsigned short>(pack, blockIdx.x - p.blocks);
    return;
  }
  for (int g = threadIdx.x; g <= p.n_adapters; g += 1024) s_hist[g] = 0;
  __syncthreads();
  const int first = blockIdx.x * p.block_rows, last = first + p.block_rows < p.rows ? first + p.block_rows : p.rows;
  for (int i = first + threadIdx.x; i < last; i += 1024) atomicAdd(&s_hist[group_of(ids, i)], 1);
  __syncthreads();
  for (int g = threadIdx.x; g < p.n_adapters; g += 1024) p.hist[(int64_t)blockIdx.x * p.n_adapters + g] = s_hist[g];
}
struct PlanLds {      // of lowrank_plan_place_kernel: all [n_adapters + 2], next [16][n_adapters + 1]
  int *first, *mine, *range0, *wide0, *chunk0, *slot0, *next;
  __host__ __device__ static size_t bytes(int G) { return (size_t)(6 * (G + 2) + 16 * (G + 1)) * 4; }
  __device__ explicit PlanLds(int *s, int G) : first(s), mine(s + G + 2), range0(s + 2 * (G + 2)), wide0(s + 5 * (G + 2)), chunk0(s + 3 * (G + 2)), slot0(s + 4 * (G + 2)), next(s + 6 * (G + 2)) {}
};
// ONE: no counts came before; each workgroup looks through all rows (LDS counters of 16 lanes each, so that rows of one adapter do not queue)
template <bool ONE>
__global__ void __launch_bounds__(1024) lowrank_plan_place_kernel(Plan p, Ids ids, PackArgs pack) {
  extern __shared__ int s_mem[];
  if (ONE && (int)blockIdx.x >= p.blocks) {
    if (pack.es == 4) pack_block<uint32_t>(pack, blockIdx.x - p.blocks);
    else pack_block<unsigned short>(pack, blockIdx.x - p.blocks);
    return;
  }
  __shared__ int4 s_w[16];
  __shared__ int s_all[1024], s_mine[1024], s_per;
  const int G = p.n_adapters, G1 = G + 1, t = threadIdx.x, lane = t & 63, wave = t >> 6, me = blockIdx.x;
  PlanLds s(s_mem, G);
  // the share's rows: each wave owns a run of them, so that places follow the rows' order
  const int first_row = me * p.block_rows, last_row = first_row + p.block_rows < p.rows ? first_row + p.block_rows : p.rows, run = p.block_rows / 16;
  const int from = first_row + wave * run, to = from + run < last_row ? from + run : last_row;
  const int h0 = from + lane < to ? group_of(ids, from + lane) : 0;      // (most shares have one row a lane: read once)
  if (t == 0) s_per = LR_RANGE;
  if (ONE) {
    int *before = s.next, *others = s.next + 16 * G1;
    for (int i = t; i < 32 * G1; i += 1024) before[i] = 0;
    __syncthreads();
#pragma unroll 4
    for (int i = t; i < p.rows; i += 1024) {
      const int h = group_of(ids, i);
      atomicAdd((i < first_row ? before : others) + (t & 15) * G1 + h, 1);
    }
    __syncthreads();
    for (int h = t >> 4; h < G; h += 64) {
      int b = before[(t & 15) * G1 + h], a = b + others[(t & 15) * G1 + h];
#pragma unroll
      for (int o = 1; o < 16; o <<= 1) { b += __shfl_xor(b, o, 16); a += __shfl_xor(a, o, 16); }
      if ((t & 15) == 0) { s_all[h] = a; s_mine[h] = b; }
    }
    __syncthreads();
  }
  for (int i = t; i < 16 * G1; i += 1024) s.next[i] = 0;
  // the adapters' rows in all shares and in the shares before this one
  int width = 1, slices = 1;
  if (!ONE) {
    while (width < G) width <<= 1;
    while (slices < p.blocks && slices * width < 1024) slices <<= 1;
  }
  const int slice = t / width, g = t & (width - 1);
  int all = 0, mine = 0;
  if (!ONE && g < G && slice < slices) {
#pragma unroll 4
    for (int b = slice; b < p.blocks; b += slices) {
      const int c = p.hist[(int64_t)b * G + g];
      all += c; mine += b < me ? c : 0;
    }
  }
  if (!ONE) { s_all[t] = all; s_mine[t] = mine; }
  __syncthreads();
  if (from + lane < to) atomicAdd(&s.next[wave * G1 + h0], 1);
  for (int i = from + 64 + lane; i < to; i += 64) atomicAdd(&s.next[wave * G1 + group_of(ids, i)], 1);
  for (int h = slices >> 1; h > 0; h >>= 1) {
    if (!ONE && slice < h) { s_all[t] += s_all[t + h * width]; s_mine[t] += s_mine[t + h * width]; }
    __syncthreads();
  }
  const int n = t < G ? s_all[t] : 0, chunks = t >= G ? 0 : n > p.chunk_rows ? (n + p.chunk_rows - 1) / p.chunk_rows : 1;
  int at[4] = {n, chunks, chunks > 1 ? chunks : 0, t < G ? s_mine[t] : 0}, sum[4];
  block_scan(at, sum, s_w);
  const int idle = p.rows - sum[0];
  // the smallest size of a range that makes no more of them than are wanted: a wave tries a size
  for (int per = p.per + wave; per < LR_RANGE; per += 16) {
    int k = 0;
    for (int i = lane; i < G; i += 64) k += (int)((unsigned)(s_all[i] + per - 1) / (unsigned)per);
    k = __builtin_amdgcn_readlane(wave_scan(k), 63) + (int)((unsigned)(idle + per - 1) / (unsigned)per);
    if (k <= p.wanted) {      // sizes behind it make no more
      if (lane == 0) atomicMin(&s_per, per);
      break;
    }
  }
  if (t < G) { s.first[t] = at[0]; s.chunk0[t] = at[1]; s.slot0[t] = at[2]; s.mine[t] = s_mine[t]; }
  if (t == 0) { s.first[G] = sum[0]; s.first[G + 1] = p.rows; s.chunk0[G] = sum[1]; s.mine[G] = first_row - sum[3]; }
  __syncthreads();
  const unsigned per = (unsigned)s_per;
  int rat[2] = {(int)((unsigned)(n + per - 1) / per), (n + p.wide_rows - 1) / p.wide_rows}, rsum[2];
  block_scan(rat, rsum, s_w);
  if (t < G) { s.range0[t] = rat[0]; s.wide0[t] = rat[1]; }
  if (t == 0) {
    s.wide0[G] = rsum[1]; s.wide0[G + 1] = rsum[1] + (idle + p.wide_rows - 1) / p.wide_rows;
    s.range0[G] = rsum[0]; s.range0[G + 1] = rsum[0] + (int)((unsigned)(idle + per - 1) / per);
  }
  // where each wave's rows of each group go: 16 lanes a group
  for (int h = t >> 4; h < G1; h += 64) {
    const int w = t & 15, c = s.next[w * G1 + h];
    int i = c;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
      const int u = __shfl_up(i, o, 16);
      i += w >= o ? u : 0;
    }
    s.next[w * G1 + h] = s.first[h] + s.mine[h] + i - c;
  }
  __syncthreads();
  // (nothing is written to memory before the last barrier: a barrier waits for it)
  if (t < G && me == 0) p.slots[t] = {at[2], chunks};
  for (int i = me * 1024 + t; i < p.n_ranges + p.n_wide + p.max_chunks; i += p.blocks * 1024) {
    const bool chunk = i >= p.n_ranges + p.n_wide, wide = !chunk && i >= p.n_ranges;
    const int *of = chunk ? s.chunk0 : wide ? s.wide0 : s.range0;
    const int at_list = i - (chunk ? p.n_ranges + p.n_wide : wide ? p.n_ranges : 0), count = of[chunk ? G : G1];
    int4 r = {chunk ? -1 : 0, 0, 0, -1};
    if (at_list < count) {
      const int h = find_group(of, chunk ? G : G1, at_list);
      const unsigned k = at_list - of[h], m = of[h + 1] - of[h], rows = s.first[h + 1] - s.first[h];
      unsigned from, to;
      if (chunk) {      // the chunks of an adapter are of one size, whole steps of 32 rows
        const unsigned size = ((rows + m - 1) / m + 31) / 32 * 32;
        from = k * size < rows ? k * size : rows;
        to = from + size < rows ? from + size : rows;
      } else {          // its ranges are of about one size
        const unsigned size = rows / m, more = rows % m;
        from = k * size + (k < more ? k : more);
        to = from + size + (k < more ? 1u : 0u);
      }
      r = {h, s.first[h] + (int)from, (int)(to - from), chunk && m > 1 ? s.slot0[h] + (int)k : -1};
    }
    (chunk ? p.chunk : wide ? p.wide : p.range)[at_list] = r;
  }
  int bits = 0;
  while ((1 << bits) < G1) ++bits;
  for (int i0 = from; i0 < to; i0 += 64) {
    const bool in = i0 + lane < to;
    const int h = i0 == from ? h0 : in ? group_of(ids, i0 + lane) : 0;
    uint64_t same = __ballot(in);      // the lanes with my group
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __ballot((h >> b) & 1);
      same &= ((h >> b) & 1) ? set : ~set;
    }
    if (in) {
      int *next = &s.next[wave * G1 + h];
      const int base = __hip_atomic_load(next, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      const int before = __popcll(same & ((1ull << lane) - 1));
      p.order[base + before] = i0 + lane;
      __builtin_amdgcn_wave_barrier();      // every lane has read the place before its first lane moves it on
      if (before == 0) __hip_atomic_store(next, base + __popcll(same), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
    __builtin_amdgcn_wave_barrier();
  }
}

void lowrank_plan_launch(const Plan &p, const Ids &ids, const PackArgs &pack, hipStream_t stream) {
  const size_t lds = PlanLds::bytes(p.n_adapters);
  if (p.rows <= LR_PLAN_ONE && p.n_adapters <= 256) {
    lowrank_plan_place_kernel<true><<<(unsigned)(p.blocks + pack.n_blocks), 1024, lds + (size_t)16 * (p.n_adapters + 1) * 4, stream>>>(p, ids, pack);
    return;
  }
  lowrank_plan_count_kernel<<<(unsigned)(p.blocks + pack.n_blocks), 1024, (size_t)(p.n_adapters + 1) * 4, stream>>>(p, ids, pack);
  lowrank_plan_place_kernel<false><<<p.blocks, 1024, lds, stream>>>(p, ids, pack);
}

// a buffer in pieces of 256 bytes
struct Carve {
  char *at;
  size_t used = 0;
  explicit Carve(void *p) : at((char *)p) {}
  template <typename P>
  P *take(size_t bytes) { P *r = (P *)(at + used); used += align_up(bytes, 256); return r; }
};

static int rank_tiles(int rank) { return rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8; }
static int lowrank_check(const gsdf_lowrank_args *a) {
  GSDF_REQUIRE(a != nullptr, "lowrank: args is NULL");
  GSDF_REQUIRE(a->rows >= 0 && a->rows < (1ll << 28), "lowrank: %lld rows outside [0, 2^28)", (long long)a->rows);
  GSDF_REQUIRE(a->n_in >= 1 && a->n_out >= 1 && a->n_in < (1 << 22) && a->n_out < (1 << 22), "lowrank: widths %d -> %d outside [1, 2^22)", a->n_in, a->n_out);
  GSDF_REQUIRE(a->rank >= 1 && a->rank <= GSDF_LOWRANK_MAX_RANK, "lowrank: rank %d outside [1, %d]", a->rank, GSDF_LOWRANK_MAX_RANK);
  GSDF_REQUIRE(a->n_adapters >= 1 && a->n_adapters <= GSDF_LOWRANK_MAX_ADAPTERS, "lowrank: %d adapters outside [1, %d]", a->n_adapters, GSDF_LOWRANK_MAX_ADAPTERS);
  const int64_t weights = (int64_t)a->n_adapters * 16 * rank_tiles(a->rank) * (2 * (int64_t)a->n_in + a->n_out);
  GSDF_REQUIRE(weights < (1ll << 32), "lowrank: %lld elements of weights (ranks in whole tiles of matrix instructions) are more than a launch can lay out", (long long)weights);
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
  q->ht_ld = (int64_t)align_up((size_t)a->rows + 32, 4);      // `outer` reads whole steps of 32 places
  Plan unused;
  q->both = a->rows >= LR_BOTH && q->rt <= 2 && a->rank % 4 == 0;
  // 64 rows of `expand` read the weights once; fewer rows where there are not enough waves otherwise
  const int64_t chunks = ceil_div(a->n_in > a->n_out ? a->n_in : a->n_out, 64);
  const int wide = q->both || q->rt > 2 || a->rows / 64 * chunks < 2048 ? (!q->both && a->rows / 32 * chunks < 2048 ? 16 : 32) : 64;
  const int least = 4 * q->rt;      // (an adapter's weights are read once a range: the wider, the more rows have to share them)
  const size_t plan_bytes = plan_layout(&unused, nullptr, a->rows, a->n_adapters, least, wide), h_bytes = (size_t)a->rows * q->rp * 4, ht_bytes = (size_t)q->ht_ld * q->rp * 4;
  Carve s(save), f(ws), b(ws);
  void *plan_saved = s.take<char>(plan_bytes);
  q->ht = s.take<float>(ht_bytes);
  const size_t weights = (size_t)a->n_adapters * q->rp * q->es, part = (size_t)plan_max_slots(a->rows, a->n_adapters) * q->rp * 4;
  const int step = 128 / q->es;
  q->a_turned = s.take<char>(weights * a->n_in);
  q->b_frag = s.take<char>(weights * align_up((size_t)a->n_out, step));
  q->save_bytes = s.used;
  void *plan_ws = f.take<char>(plan_bytes);
  q->h = f.take<float>(h_bytes);
  q->a_frag = f.take<char>(weights * align_up((size_t)a->n_in, step));
  q->fwd_ws_bytes = f.used;      // the plan at least: never 0
  plan_layout(&q->plan, training ? plan_saved : plan_ws, a->rows, a->n_adapters, least, wide);
  q->dh = b.take<float>(h_bytes);
  q->dht = b.take<float>(ht_bytes);
  q->part[0] = b.take<float>(part * a->n_in);
  q->part[1] = b.take<float>(part * a->n_out);
  q->bwd_ws_bytes = b.used > 0 ? b.used : 256;      // (a buffer that a caller can point to)
}

PackArgs lowrank_pack_args(const Lowrank &q, bool training) {
  const gsdf_lowrank_args &a = q.a;
  const int step = 128 / q.es;
  PackArgs t;
  t.a = a.a; t.b = a.b; t.a_frag = q.a_frag; t.b_frag = q.b_frag; t.a_turned = q.a_turned;
  t.n_in = a.n_in; t.n_out = a.n_out; t.rank = a.rank; t.rt = q.rt; t.es = q.es;
  t.blocks[0] = (int)ceil_div(ceil_div(a.n_in, step) * q.rt * 128, 1024);
  t.blocks[1] = training ? (int)ceil_div(ceil_div(a.n_out, step) * q.rt * 128, 1024) : 0;
  t.blocks[2] = training ? (int)ceil_div((int64_t)a.n_in * q.rp / (16 / q.es), 1024) : 0;
  t.n_blocks = a.rows > 0 ? (t.blocks[0] + t.blocks[1] + t.blocks[2]) * a.n_adapters : 0;
  return t;
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
    lowrank_plan_launch(q.plan, Ids{args->ids, args->ids_64, args->n_adapters}, lowrank_pack_args(q, false), stream);
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
  Lowrank q;
  lowrank_layout(&q, args, const_cast<void *>(save), ws, true);
  // (only rows that lie on one another are so many and so wide)
  const int64_t columns = 256 / q.es, outer = (int64_t)q.plan.max_chunks * (ceil_div(args->n_in, columns) + ceil_div(args->n_out, columns));
  GSDF_REQUIRE((da == nullptr && db == nullptr) || outer * LR_OUTER_THREADS < (1ll << 32), "lowrank_bwd: %lld workgroups for the weights' gradients are more than a launch holds",
               (long long)outer);
  GSDF_TIMED("gsdf_lowrank_bwd");
  GSDF_BY_DTYPE(args->dtype, lowrank_bwd<T>(q, dy, dy_stride, dx, dx_stride, da, db, stream));
  GSDF_CHECK_LAUNCH("lowrank_bwd");
  return GSDF_OK;
}
