// gsdf_adapters.h — one decoder for many maps: low-rank adapters chosen row by row beside a shared projection, dropout on their input, and the balance loss
// of the router that chooses them (include/gsdf_hip.h: L1-L3).  No reference counterpart: the reference trains one network per map
// (include/neural_net/local_map.cpp:29-55).  gs_sdf_amd.adapters (Python) calls these functions and documents them in full.
//
// fp32, fp16 or bf16 elements, one type per call.  Differentiable once.  Every call runs on the current stream of its tensors' device, takes its workspace from
// the caching allocator, synchronises nothing and can be captured into a graph.  Errors are c10::Error.
#pragma once
#include <torch/torch.h>

#include <optional>
#include <tuple>

namespace gsdf_adapters {

// where a dropout mask begins: a number, plus a device word (int64, one element) if there is one — a captured graph's counter
struct Offset {
  uint64_t number = 0;
  std::optional<torch::Tensor> word;
};

// base + s_g B_g A_g drop(x) for every row, g = ids[row]: x [..., k], a [g, r, k], b [g, n, r], ids [...] (int32 / int64; outside [0, g): base alone),
// scales [g] fp32 constants, base [..., n] -> [..., n].  Gradients for x, a, b, base.
torch::Tensor lowrank_adapt(const torch::Tensor &x, const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &ids,
                            const std::optional<torch::Tensor> &scales = std::nullopt, const std::optional<torch::Tensor> &base = std::nullopt, double p = 0.0,
                            uint64_t seed = 0, const Offset &offset = {});
// y += s_g B_g A_g x in place, rows without an adapter untouched; y shares no memory with what the call reads (else: error); no gradients
void lowrank_adapt_(const torch::Tensor &y, const torch::Tensor &x, const torch::Tensor &a, const torch::Tensor &b, const torch::Tensor &ids,
                    const std::optional<torch::Tensor> &scales = std::nullopt);
// [residual +] x with elements dropped at probability round(65536 p) / 65536, the others multiplied by 1 / (1 - that)
torch::Tensor dropout(const torch::Tensor &x, double p, uint64_t seed, const Offset &offset = {}, const std::optional<torch::Tensor> &residual = std::nullopt);
// logits [..., e], ids [...] or [..., k], mask [...] (bool / uint8) -> (loss, counts int64 [e])
std::tuple<torch::Tensor, torch::Tensor> router_balance(const torch::Tensor &logits, const torch::Tensor &ids, const std::optional<torch::Tensor> &mask = std::nullopt);

}  // namespace gsdf_adapters
