// lowrank.h — what lowrank.hip (the plan, the C entries) and lowrank_kernels.h (the products, compiled once for each element type) share.
#pragma once
#include "adapter_common.h"

namespace gsdf {

static constexpr int LR_CUS = 256;          // compute units the ranges are dealt to
static constexpr int LR_AIM = 40;           // rows of a range that are aimed at, at most
static constexpr int LR_RANGE = 48;         // most rows of a range: three matrix tiles
static constexpr int LR_BOTH = 65536;        // rows from which on a wave takes a range through both products
static constexpr int LR_PLAN_ONE = 16384;    // rows up to which the plan is one launch
static constexpr int LR_CHUNK = 1024;       // most rows of one sum in `outer`
static constexpr int LR_OUTER_THREADS = 512;
static constexpr int LR_CHUNK_FEW = 2048;   // the same where all rows are no more: then no adapter has two, and nothing is left to add up

// ---- the rows in the order of their adapters ----------------------------------------------------------------------------------------------
// All in one int32 buffer.  Group n_adapters holds the rows without an adapter.
struct Plan {
  int *order;      // [rows]: the row at each place, adapters one behind the other, rows of one adapter in their own order
  int4 *range;     // [n_ranges]: adapter, first place, rows (0: unused), -
  int4 *wide;      // [n_wide]: the same of up to wide_rows rows, for `expand`
  int4 *chunk;     // [max_chunks]: adapter (-1: unused), first place, rows (0: an adapter without any), slot of its partial sums (-1: its only chunk)
  int2 *slots;     // [n_adapters]: first slot, chunks
  int *hist;       // [blocks][n_adapters]: rows of each adapter in each workgroup's share
  int rows, n_adapters, blocks, block_rows;
  int per, wanted, n_ranges, wide_rows, n_wide, chunk_rows, max_chunks;
};
// Every range costs a compute unit about the bytes of its rows and of its adapter's weights, and ends with its adapter: `per` is the smallest size from
// this one on that makes no more ranges than a multiple of the units (8192 rows of 8 KB, rank 16: 264 ranges of 32 rows took 28 us on 256 units, 249 of up to 34 took 20).
// `least`: rows that share the weights at least.  `wide_rows`: rows of a range of `expand`, 16, 32 or 64.
static size_t plan_layout(Plan *p, void *mem, int64_t rows, int n_adapters, int least, int wide_rows) {
  p->rows = (int)rows; p->n_adapters = n_adapters;
  p->block_rows = rows <= LR_CUS * 1024 ? 1024 : (int)align_up((size_t)ceil_div(rows, LR_CUS), 1024);
  p->blocks = (int)ceil_div(rows > 0 ? rows : 1, p->block_rows);
  const int64_t waves = ceil_div(rows > 0 ? rows : 1, LR_CUS * LR_AIM);
  p->wanted = (int)(LR_CUS * waves);
  p->per = (int)ceil_div(rows > 0 ? rows : 1, p->wanted);
  if (p->per < least) p->per = least;
  const int64_t most = rows / LR_RANGE + n_adapters + 1;
  p->n_ranges = (int)(p->wanted > most ? p->wanted : most);
  p->wide_rows = wide_rows;
  p->n_wide = (int)(rows / wide_rows + n_adapters + 1);
  p->chunk_rows = rows <= LR_CHUNK_FEW ? LR_CHUNK_FEW : LR_CHUNK;
  p->max_chunks = (int)(rows / p->chunk_rows + n_adapters);
  char *at = (char *)mem;
  auto take = [&](size_t bytes) { char *r = at; at += align_up(bytes, 16); return r; };
  p->range = (int4 *)take((size_t)p->n_ranges * 16);
  p->wide = (int4 *)take((size_t)p->n_wide * 16);
  p->chunk = (int4 *)take((size_t)p->max_chunks * 16);
  p->slots = (int2 *)take((size_t)n_adapters * 8);
  p->hist = (int *)take((size_t)p->blocks * n_adapters * 4);
  p->order = (int *)take((size_t)rows * 4);
  return (size_t)(at - (char *)mem);
}
// slots for the chunks of adapters with more than one: such an adapter has more than LR_CHUNK rows, so there are at most twice rows / LR_CHUNK of them
static int64_t plan_max_slots(int64_t rows, int n_adapters) {
  const int64_t twice = 2 * (rows / LR_CHUNK) + 1, all = rows / LR_CHUNK + n_adapters;
  return rows <= LR_CHUNK_FEW ? 0 : (twice < all ? twice : all);
}

struct Ids {
  const void *p;
  int is_64, n_adapters;
};
__device__ __forceinline__ int group_of(Ids ids, int64_t row) {
  const int64_t g = load_id(ids.p, ids.is_64, row);
  return g >= 0 && g < ids.n_adapters ? (int)g : ids.n_adapters;
}

// ---- weights laid out for the matrix instructions ----------------------------------------------------------------------------------------
// `shrink` reads fragments: [adapter][step][tile of 16 ranks][2][64 lanes] pieces of 16 bytes, lane (c, quad) of half i with the elements
// step 8N + i 4N + quad N .. of rank c of the tile (N elements in 16 bytes; zeros behind the width and the rank).  A wave's load is 1 KB of neighbours, where 16 rows
// 2^n bytes apart ask one channel of the L2 (rank 64, 8192 rows of 8 KB: 26 us against 22; rank 128: 41 against 28).  `expand` of the backward pass
// reads A^T as [adapter][n_in][RP].  They are made beside the plan, whose few workgroups leave the card idle.
struct PackArgs {
  const void *a, *b;
  void *a_frag, *b_frag, *a_turned;      // a_turned, b_frag: null without a backward pass
  int n_in, n_out, rank, rt, es;
  int blocks[3], n_blocks;               // workgroups of each for one adapter; of all for all
};

// a call, with everything in its place
struct Lowrank {
  gsdf_lowrank_args a;
  Dropout drop;
  Plan plan;
  int rt, rp, es;
  bool both;      // `shrink` and `expand` in one kernel
  int64_t ht_ld;
  // saved by the forward pass (beside the plan)
  float *ht;
  void *b_frag, *a_turned;
  // workspace
  float *h, *dh, *dht, *part[2];
  void *a_frag;
  size_t save_bytes, fwd_ws_bytes, bwd_ws_bytes;
};

void lowrank_plan_launch(const Plan &p, const Ids &ids, const PackArgs &pack, hipStream_t stream);
PackArgs lowrank_pack_args(const Lowrank &q, bool training);
template <typename T>
void lowrank_fwd(const Lowrank &q, const void *base, int64_t base_stride, void *y, int64_t y_stride, bool training, hipStream_t stream);
template <typename T>
void lowrank_bwd(const Lowrank &q, const void *dy, int64_t dy_stride, void *dx, int64_t dx_stride, void *da, void *db, hipStream_t stream);

}  // namespace gsdf
