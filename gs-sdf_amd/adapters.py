"""One decoder for many maps: low-rank adapters chosen row by row beside a shared projection, dropout on their input, and the balance loss of
the router that chooses them (include/gsdf_hip.h: L1-L3).  No reference counterpart: the reference trains one network per map
(include/neural_net/local_map.cpp:29-55).

    y = lowrank_adapt(x, a, b, ids, scales, base)          # base + s_g B_g A_g x, g = ids[row]
    y = dropout(x, p, seed, offset, residual)              # Philox mask, never stored
    loss, counts = router_balance(logits, ids, mask)

Elements are fp32, fp16 or bf16 (one type per call), sums are held in 32 bits and a result is rounded once.  Rows may be strided (a slice of a wider
buffer is read in place); any other layout is copied first.  Every call runs on the current stream of its tensors' device, allocates its
workspace from torch's caching allocator and can be captured into a graph; nothing synchronises.  Derivatives are those of one backward pass: a second one
through a gradient raises (through base and residual, which are added as they are, it goes on), an input with a forward-mode tangent is refused.  As with every operator of torch, a backward pass is captured
only while no eager graph of the same leaves lives: torch would wait for that graph's stream, which ends the capture and may end the process.
"""
import importlib.util
import math
import os
import sysconfig

import torch

from . import capi

MAX_RANK, MAX_ADAPTERS, MAX_EXPERTS = 128, 1024, 1024      # include/gsdf_hip.h

_mod = None


def _ops():
    """The C++ operators (host/gsdf_adapters/gsdf_adapters.h); fails loudly, there is no fallback."""
    global _mod
    if _mod is None:
        capi.lib()      # the kernels' library, with its version check
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "lib", "_gsdf_adapters" + sysconfig.get_config_var("EXT_SUFFIX"))
        if not os.path.exists(path):
            raise RuntimeError(f"{path} not found: build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        spec = importlib.util.spec_from_file_location("_gsdf_adapters", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        _mod = mod
    return _mod


def lowrank_adapt(x, a, b, ids, scales=None, base=None, p=0.0, seed=0, offset=0):
    """y = base + s_g B_g A_g drop(x) for every row, g = ids[row]: x [..., k], a [g, r, k], b [g, n, r], ids [...] (int32 / int64), scales [g] fp32
    constants (None: 1), base [..., n] (None: 0) -> y [..., n].  A row whose id is outside [0, g) has no adapter: y is base there.  p > 0 drops elements of
    x as dropout(x, p, seed, offset) would.  Gradients for x, a, b and base (once; a rank up to 128, up to 1024 adapters).  h keeps its 32 bits beside
    16-bit elements, as a sum of three of them: where a factor is infinite the result is not finite, but may be NaN where the formula has an infinity."""
    return (_mod or _ops()).lowrank_adapt(x, a, b, ids, scales, base, p, seed, offset)


def lowrank_adapt_(y, x, a, b, ids, scales=None):
    """In place, for serving: y += s_g B_g A_g x in every row that has an adapter; the other rows are not touched.  y [..., n] has neighbouring elements in a row
    (a slice of a wider buffer is fine) and shares no memory with what the call reads.  No gradients."""
    (_mod or _ops()).lowrank_adapt_(y, x, a, b, ids, scales)
    return y


class LowRankAdapters:
    """Adapters for a shared network (sdf.TCNNNetwork.forward takes them): leaves `a_` [n_adapters, rank, n_in] (uniform, bound 1 / sqrt(n_in)) and `b_`
    [n_adapters, n_out, rank] (zeros: a new adapter changes nothing), scale alpha / rank.  p > 0: dropout on their input in every call that makes gradients, until eval() (a normal taken for an
    answer makes gradients too; train() turns it on again);
    its masks go by `seed` and `calls_`, which counts such calls: both belong into a checkpoint beside the leaves.  Without a `seed` every bank has another, out of
    torch's default generator (torch.manual_seed makes them again; processes that train one bank give one seed), since two banks of one seed drop the same elements.  `calls_` is a host number: a
    captured call replays one mask and a call that is made again for its gradients (activation checkpoints) takes another, so give `offset` (a number of the program's own, or a
    device word that it counts up) there."""

    def __init__(self, n_adapters, n_in, n_out, rank, alpha=None, p=0.0, dtype=torch.float32, device="cuda", seed=None):
        if not (1 <= rank <= MAX_RANK and 1 <= n_adapters <= MAX_ADAPTERS):
            raise RuntimeError(f"LowRankAdapters: rank {rank} or {n_adapters} adapters out of range")
        if not 0.0 <= float(p) <= 1.0:
            raise RuntimeError(f"p: expected a probability in [0, 1], got {p}")
        if seed is None:
            seed = int(torch.randint(0, 1 << 62, (), device="cpu"))
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.a_ = ((torch.rand(n_adapters, rank, n_in, generator=g) * 2 - 1) / math.sqrt(n_in)).to(dtype).to(device).requires_grad_(True)
        self.b_ = torch.zeros(n_adapters, n_out, rank, dtype=dtype, device=device).requires_grad_(True)
        self.scales = torch.full((n_adapters,), float(rank if alpha is None else alpha) / rank, dtype=torch.float32, device=device)
        self.p, self.seed, self.calls_, self.training = float(p), int(seed), 0, True

    def train(self, mode=True):
        self.training = bool(mode)
        return self

    def eval(self):
        return self.train(False)

    def forward(self, x, ids, base=None, offset=None):
        gradients = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, self.a_, self.b_, base))
        p = self.p if self.training and gradients else 0.0
        if offset is None:
            offset = self.calls_
            self.calls_ += p > 0
        return lowrank_adapt(x, self.a_, self.b_, ids, self.scales, base, p, self.seed, offset)

    __call__ = forward


def dropout(x, p, seed, offset=0, residual=None):
    """[residual +] x with elements dropped at probability round(65536 p) / 65536 and the others multiplied by 1 / (1 - that): x [..., cols] of any shape,
    seen as a matrix of rows of its last dimension.  The mask goes by (seed, offset, row, column) alone (include/gsdf_hip.h: gsdf_dropout): the same
    numbers give the same mask on any layout, and the backward pass makes it again.  offset: a number, or a device word (int64, one element) that is read when
    the kernel runs; it has to hold the same value in the backward pass.  A dropped element is exactly 0 (or residual), whatever x holds there."""
    return (_mod or _ops()).dropout(x, p, seed, offset, residual)


def router_balance(logits, ids, mask=None):
    """Balance loss of a router and its experts' counts: logits [..., e], ids [...] or [..., k] (int32 / int64) the experts that each row went to, mask [...] (bool or
    uint8; None: all) the rows that count -> (loss fp32 scalar, counts int64 [e]).  With f_e = counts_e / (k V), P_e the mean of softmax(logits) over the
    V valid rows, loss = e sum_e f_e P_e: 1 for an even router.  The gradient goes to the logits through P; rows outside the mask get 0.  ids outside
    [0, e) count for nobody.  Without a valid row loss and gradient are 0."""
    return (_mod or _ops()).router_balance(logits, ids, mask)
