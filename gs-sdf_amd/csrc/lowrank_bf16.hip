// lowrank_bf16.hip — the products of the low-rank adapters (lowrank_kernels.h) for one element type.
#include "lowrank_kernels.h"

namespace gsdf {
template void lowrank_fwd<bf16_t>(const Lowrank &, const void *, int64_t, void *, int64_t, bool, hipStream_t);
template void lowrank_bwd<bf16_t>(const Lowrank &, const void *, int64_t, void *, int64_t, void *, void *, hipStream_t);
}  // namespace gsdf
