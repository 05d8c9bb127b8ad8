"""One decoder for many maps: low-rank adapters chosen row by row beside a shared projection, dropout on their input, and the balance loss of
the router that chooses them (include/gsdf_hip.h: L1-L3).  No reference counterpart: the reference trains one network per map
(include/neural_net/local_map.cpp:29-55).

    y = lowrank_adapt(x, a, b, ids, scales, base)          # base + s_g B_g A_g x, g = ids[row]
    y = dropout(x, p, seed, offset, residual)              # Philox mask, never stored
    loss, counts = router_balance(logits, ids, mask)

Elements are fp32, fp16 or bf16 (one type per call), sums are held in 32 bits and a result is rounded once.  Rows may be strided (a slice of a wider
buffer is read in place); any other layout is copied first.  Every call runs on the current stream of its tensors' device, allocates its
workspace from torch's caching allocator and can be captured into a graph; nothing synchronises.
"""
import ctypes as C
import math

import torch

from . import capi

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}      # include/gsdf_hip.h: GSDF_F32 / _F16 / _BF16
MAX_RANK, MAX_ADAPTERS, MAX_EXPERTS = 128, 1024, 1024


def _need(cond, what):
    if not cond:
        raise RuntimeError(what)


def _same(ref, t, name, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise RuntimeError(f"{name}: expected a tensor")
    if t.device != ref.device:
        raise RuntimeError(f"{name}: expected a tensor on {ref.device}, got one on {t.device}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name}: expected dtype {dtype}, got {t.dtype}")


def _elements(t, name):
    if not (isinstance(t, torch.Tensor) and t.is_cuda):
        raise RuntimeError(f"{name}: expected a device tensor (the HIP path has no CPU fallback)")
    d = _DTYPES.get(t.dtype)
    if d is None:
        raise RuntimeError(f"{name}: expected fp32, fp16 or bf16 elements, got {t.dtype}")
    return d


def _rows(t):
    """-> (a [rows, width] tensor whose rows are neighbours' elements, its row stride); a view where the layout allows it"""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1] if t.dim() else 1) if t.numel() else t.new_empty(math.prod(t.shape[:-1]), t.shape[-1] if t.dim() else 1)
    if t.stride(1) != 1 and t.shape[1] != 1:
        t = t.contiguous()
    return t, t.stride(0)


def _index(t, ref, name):
    _same(ref, t, name)
    if t.dtype not in (torch.int32, torch.int64):
        raise RuntimeError(f"{name}: expected int32 or int64, got {t.dtype}")
    return t.contiguous()


def _offset(offset, ref):
    """-> (number, device word or None)"""
    if isinstance(offset, torch.Tensor):
        _same(ref, offset, "offset", torch.int64)
        _need(offset.numel() == 1, "offset: expected one device word")
        return 0, offset
    if not 0 <= int(offset) < 2 ** 64:
        raise RuntimeError("offset: expected a number in [0, 2^64)")
    return int(offset), None


def _check_p(p, seed):
    if not 0.0 <= float(p) <= 1.0:
        raise RuntimeError(f"p: expected a probability in [0, 1], got {p}")
    if not 0 <= int(seed) < 2 ** 64:
        raise RuntimeError("seed: expected a number in [0, 2^64)")


def _run(dev, fn, *args):
    """fn(*args, stream) on the current stream of `dev`, with `dev` current while it launches"""
    if dev.index == torch.cuda.current_device():
        code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, torch._C._cuda_getCurrentRawStream(dev.index))
    if code != 0:
        capi.check(code, fn.__name__)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _grad_wanted(*ts):
    if torch.is_grad_enabled():
        for t in ts:
            if t is not None and t.requires_grad:
                return True
    return False


def _once(backward):
    """a backward pass that is not differentiated again (torch.autograd.function.once_differentiable, whose cost only a call with create_graph pays)"""
    checked = torch.autograd.function.once_differentiable(backward)

    def run(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)
    return run


# ------------------------------------------------------------------------------------------------
# L1  low-rank adapters
# ------------------------------------------------------------------------------------------------
def _lowrank_args(x, x_stride, a, b, ids, scales, dtype, p, seed, offset, word):
    return capi.LowrankArgs(x.shape[0], x_stride, a.shape[2], b.shape[1], a.shape[1], a.shape[0], dtype, ids.dtype == torch.int64, x.data_ptr(),
                            a.data_ptr(), b.data_ptr(), ids.data_ptr(), _ptr(scales), p, seed, offset, _ptr(word))


def _lowrank_fwd(x, x_stride, a, b, ids, scales, base, y, dtype, p, seed, offset, word, keep):
    L = capi.lib()
    args = _lowrank_args(x, x_stride, a, b, ids, scales, dtype, p, seed, offset, word)
    ref = C.byref(args)
    ws = torch.empty(L.gsdf_lowrank_fwd_ws_bytes(ref), dtype=torch.uint8, device=x.device)
    save = torch.empty(L.gsdf_lowrank_save_bytes(ref), dtype=torch.uint8, device=x.device) if keep else None
    base, base_stride = (None, 0) if base is None else _rows(base)
    _run(x.device, L.gsdf_lowrank_fwd, ref, _ptr(base), base_stride, y.data_ptr(), y.stride(0), _ptr(save), ws.data_ptr())
    return save


class _Lowrank(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, base, ids, scales, dtype, p, seed, offset, word):
        x, x_stride = _rows(x)
        y = torch.empty(x.shape[0], b.shape[1], dtype=x.dtype, device=x.device)
        save = _lowrank_fwd(x, x_stride, a, b, ids, scales, base, y, dtype, p, seed, offset, word, True)
        ctx.save_for_backward(x, a, b, ids, scales, save, word)
        ctx.rest = (dtype, p, seed, offset)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        x, a, b, ids, scales, save, word = ctx.saved_tensors
        dtype, p, seed, offset = ctx.rest
        need_x, need_a, need_b, need_base = ctx.needs_input_grad[:4]
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need_x else None
        da = torch.empty_like(a) if need_a else None
        db = torch.empty_like(b) if need_b else None
        if need_x or need_a or need_b:
            L = capi.lib()
            g, g_stride = _rows(dy)
            args = _lowrank_args(x, x.stride(0), a, b, ids, scales, dtype, p, seed, offset, word)
            ref = C.byref(args)
            ws = torch.empty(L.gsdf_lowrank_bwd_ws_bytes(ref), dtype=torch.uint8, device=x.device)
            _run(x.device, L.gsdf_lowrank_bwd, ref, g.data_ptr(), g_stride, save.data_ptr(), _ptr(dx), 0 if dx is None else dx.stride(0), _ptr(da), _ptr(db),
                 ws.data_ptr())
        return dx, da, db, (dy if need_base else None), None, None, None, None, None, None, None


def _lowrank_checked(x, a, b, ids, scales, base, p, seed, offset):
    dtype = _elements(x, "x")
    _same(x, a, "a", x.dtype)
    _same(x, b, "b", x.dtype)
    if x.dim() < 1 or a.dim() != 3 or b.dim() != 3:
        raise RuntimeError("lowrank_adapt: expected x [..., k], a [g, r, k], b [g, n, r]")
    (g, r, k), lead = a.shape, x.shape[:-1]
    n = b.shape[1]
    if x.shape[-1] != k or b.shape[0] != g or b.shape[2] != r:
        raise RuntimeError(f"lowrank_adapt: x {tuple(x.shape)}, a {tuple(a.shape)}, b {tuple(b.shape)} do not fit (x [..., k], a [g, r, k], b [g, n, r])")
    if not (1 <= r <= MAX_RANK and 1 <= g <= MAX_ADAPTERS and k >= 1 and n >= 1):
        raise RuntimeError(f"lowrank_adapt: rank {r} outside [1, {MAX_RANK}], {g} adapters outside [1, {MAX_ADAPTERS}], or an empty projection {k} -> {n}")
    ids = _index(ids, x, "ids")
    if ids.shape != lead:
        raise RuntimeError(f"ids: expected shape {tuple(lead)}, got {tuple(ids.shape)}")
    if scales is not None:
        _same(x, scales, "scales", torch.float32)
        if scales.dim() != 1 or scales.shape[0] != g:
            raise RuntimeError(f"scales: expected shape ({g},), got {tuple(scales.shape)}")
        if scales.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("scales: constants, no gradient is offered for them")
        scales = scales.contiguous()
    if base is not None:
        _same(x, base, "base", x.dtype)
        if base.dim() != x.dim() or base.shape[-1] != n or base.shape[:-1] != lead:
            raise RuntimeError(f"base: expected shape {tuple(lead) + (n,)}, got {tuple(base.shape)}")
    _check_p(p, seed)
    return dtype, a.contiguous(), b.contiguous(), ids, scales, _offset(offset, x)


def lowrank_adapt(x, a, b, ids, scales=None, base=None, p=0.0, seed=0, offset=0):
    """y = base + s_g B_g A_g drop(x) for every row, g = ids[row]: x [..., k], a [g, r, k], b [g, n, r], ids [...] (int32 / int64), scales [g] fp32
    constants (None: 1), base [..., n] (None: 0) -> y [..., n].  A row whose id is outside [0, g) has no adapter: y is base there.  p > 0 drops elements of
    x as dropout(x, p, seed, offset) would.  Gradients for x, a, b and base (once; a rank up to 128, up to 1024 adapters)."""
    dtype, a, b, ids, scales, (offset, word) = _lowrank_checked(x, a, b, ids, scales, base, p, seed, offset)
    shape = x.shape[:-1] + (b.shape[1],)
    if _grad_wanted(x, a, b, base):
        rows = math.prod(x.shape[:-1])
        y = _Lowrank.apply(x.reshape(rows, x.shape[-1]) if x.dim() != 2 else x, a, b,
                           base if base is None or x.dim() == 2 else base.reshape(rows, shape[-1]), ids, scales, dtype, float(p), int(seed), offset, word)
        return y if x.dim() == 2 else y.view(shape)
    x, x_stride = _rows(x)
    y = torch.empty(shape, dtype=x.dtype, device=x.device)
    _lowrank_fwd(x, x_stride, a, b, ids, scales, base, y if y.dim() == 2 else y.view(x.shape[0], shape[-1]), dtype, float(p), int(seed), offset, word, False)
    return y


def lowrank_adapt_(y, x, a, b, ids, scales=None):
    """In place, for serving: y += s_g B_g A_g x in every row that has an adapter; the other rows are not touched.  y [..., n] has neighbouring elements in a row
    (a slice of a wider buffer is fine).  No gradients."""
    dtype, a, b, ids, scales, _ = _lowrank_checked(x, a, b, ids, scales, y, 0.0, 0, 0)
    _need(not _grad_wanted(y, x, a, b), "lowrank_adapt_: no gradients in place; use lowrank_adapt")
    n = b.shape[1]
    out = y if y.dim() == 2 else y.view(math.prod(y.shape[:-1]), n)
    _need(out.stride(1) == 1 or n == 1, "lowrank_adapt_: the elements of a row of y have to be neighbours")
    _need(out.shape[0] <= 1 or out.stride(0) >= n, "lowrank_adapt_: the rows of y overlap")
    x, x_stride = _rows(x)
    _lowrank_fwd(x, x_stride, a, b, ids, scales, out, out, dtype, 0.0, 0, 0, None, False)
    torch.autograd.graph.increment_version(y)
    return y


class LowRankAdapters:
    """Adapters for a shared network (sdf.TCNNNetwork.forward takes them): leaves `a_` [n_adapters, rank, n_in] (uniform, bound 1 / sqrt(n_in)) and `b_`
    [n_adapters, n_out, rank] (zeros: a new adapter changes nothing), scale alpha / rank.  p > 0: dropout on their input in every call that makes gradients;
    its masks go by `seed` and `calls_`, which counts such calls.  `calls_` is a host number: a captured call replays one mask, so give
    `offset` (a device word that the program counts up) there."""

    def __init__(self, n_adapters, n_in, n_out, rank, alpha=None, p=0.0, dtype=torch.float32, device="cuda", seed=0):
        _need(1 <= rank <= MAX_RANK and 1 <= n_adapters <= MAX_ADAPTERS, f"LowRankAdapters: rank {rank} or {n_adapters} adapters out of range")
        _check_p(p, seed)
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.a_ = ((torch.rand(n_adapters, rank, n_in, generator=g) * 2 - 1) / math.sqrt(n_in)).to(dtype).to(device).requires_grad_(True)
        self.b_ = torch.zeros(n_adapters, n_out, rank, dtype=dtype, device=device).requires_grad_(True)
        self.scales = torch.full((n_adapters,), float(rank if alpha is None else alpha) / rank, dtype=torch.float32, device=device)
        self.p, self.seed, self.calls_ = float(p), int(seed), 0

    def forward(self, x, ids, base=None, offset=None):
        p = self.p if _grad_wanted(x, self.a_, self.b_, base) else 0.0
        if offset is None:
            offset = self.calls_
            self.calls_ += p > 0
        return lowrank_adapt(x, self.a_, self.b_, ids, self.scales, base, p, self.seed, offset)

    __call__ = forward


# ------------------------------------------------------------------------------------------------
# L2  dropout
# ------------------------------------------------------------------------------------------------
def _dropout(x, residual, dtype, p, seed, offset, word):
    m, stride = _rows(x)
    r, r_stride = (None, 0) if residual is None else _rows(residual)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _run(x.device, capi.lib().gsdf_dropout, m.shape[0], m.shape[1], dtype, m.data_ptr(), stride, _ptr(r), r_stride, p, seed, offset, _ptr(word),
         y.data_ptr(), m.shape[1])
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, dtype, p, seed, offset, word):
        ctx.save_for_backward(word)
        ctx.rest = (dtype, p, seed, offset)
        return _dropout(x, residual, dtype, p, seed, offset, word)

    @staticmethod
    @_once
    def backward(ctx, dy):
        word, = ctx.saved_tensors
        dtype, p, seed, offset = ctx.rest
        return (_dropout(dy, None, dtype, p, seed, offset, word) if ctx.needs_input_grad[0] else None), (dy if ctx.needs_input_grad[1] else None), \
            None, None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """[residual +] x with elements dropped at probability round(65536 p) / 65536 and the others multiplied by 1 / (1 - that): x [..., cols] of any shape,
    seen as a matrix of rows of its last dimension.  The mask goes by (seed, offset, row, column) alone (include/gsdf_hip.h: gsdf_dropout): the same
    numbers give the same mask on any layout, and the backward pass makes it again.  offset: a number, or a device word (int64, one element) that is read when
    the kernel runs; it has to hold the same value in the backward pass.  A dropped element is exactly 0 (or residual), whatever x holds there."""
    dtype = _elements(x, "x")
    _check_p(p, seed)
    if residual is not None:
        _same(x, residual, "residual", x.dtype)
        _need(residual.shape == x.shape, f"residual: expected shape {tuple(x.shape)}, got {tuple(residual.shape)}")
    offset, word = _offset(offset, x)
    if _grad_wanted(x, residual):
        return _Dropout.apply(x, residual, dtype, float(p), int(seed), offset, word)
    return _dropout(x, residual, dtype, float(p), int(seed), offset, word)


# ------------------------------------------------------------------------------------------------
# L3  balance loss
# ------------------------------------------------------------------------------------------------
def _balance_fwd(logits, stride, ids, k, mask, dtype):
    L = capi.lib()
    rows, e = logits.shape
    dev = logits.device
    loss, pull = torch.empty((), dtype=torch.float32, device=dev), torch.empty(e, dtype=torch.float32, device=dev)
    counts = torch.empty(e, dtype=torch.int64, device=dev)
    ws = torch.empty(L.gsdf_router_balance_ws_bytes(rows, e), dtype=torch.uint8, device=dev)
    _run(dev, L.gsdf_router_balance_fwd, rows, e, k, dtype, logits.data_ptr(), stride, ids.data_ptr(), ids.dtype == torch.int64, _ptr(mask), loss.data_ptr(),
         counts.data_ptr(), pull.data_ptr(), ws.data_ptr())
    return loss, counts, pull


class _Balance(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, k, mask, dtype):
        m, stride = _rows(logits)
        loss, counts, pull = _balance_fwd(m, stride, ids, k, mask, dtype)
        ctx.save_for_backward(m, mask, pull)
        ctx.dtype = dtype
        ctx.mark_non_differentiable(counts)
        return loss, counts

    @staticmethod
    @_once
    def backward(ctx, v_loss, _v_counts):
        m, mask, pull = ctx.saved_tensors
        rows, e = m.shape
        v_logits = torch.empty(rows, e, dtype=m.dtype, device=m.device)
        _run(m.device, capi.lib().gsdf_router_balance_bwd, rows, e, ctx.dtype, m.data_ptr(), m.stride(0), _ptr(mask), pull.data_ptr(),
             v_loss.contiguous().data_ptr(), v_logits.data_ptr())
        return v_logits, None, None, None, None


def router_balance(logits, ids, mask=None):
    """Balance loss of a router and its experts' counts: logits [..., e], ids [...] or [..., k] (int32 / int64) the experts that each row went to, mask [...] (bool or
    uint8; None: all) the rows that count -> (loss fp32 scalar, counts int64 [e]).  With f_e = counts_e / (k V), P_e the mean of softmax(logits) over the
    V valid rows, loss = e sum_e f_e P_e: 1 for an even router.  The gradient goes to the logits through P; rows outside the mask get 0.  ids outside
    [0, e) count for nobody.  Without a valid row loss and gradient are 0."""
    dtype = _elements(logits, "logits")
    _need(logits.dim() >= 1 and 1 <= logits.shape[-1] <= MAX_EXPERTS, f"logits: expected [..., e] with 1 to {MAX_EXPERTS} experts, got {tuple(logits.shape)}")
    lead, e = logits.shape[:-1], logits.shape[-1]
    ids = _index(ids, logits, "ids")
    _need(ids.shape == lead or ids.shape[:-1] == lead, f"ids: expected shape {tuple(lead)} or {tuple(lead)} + (k,), got {tuple(ids.shape)}")
    k = 1 if ids.shape == lead else ids.shape[-1]
    _need(1 <= k <= e, f"ids: {k} choices of {e} experts")
    if mask is not None:
        _same(logits, mask, "mask")
        _need(mask.dtype in (torch.bool, torch.uint8) and mask.shape == lead, f"mask: expected bool or uint8 of shape {tuple(lead)}, got {mask.dtype} "
              f"{tuple(mask.shape)}")
        mask = mask.contiguous()
    if _grad_wanted(logits):
        return _Balance.apply(logits if logits.dim() == 2 else logits.reshape(math.prod(lead), e), ids, k, mask, dtype)
    m, stride = _rows(logits)
    loss, counts, _ = _balance_fwd(m, stride, ids, k, mask, dtype)
    return loss, counts
