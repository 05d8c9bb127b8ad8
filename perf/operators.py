"""Cases and plain forms of the operators of gs_sdf_amd.adapters, for timing and for comparison.

  lowrank_adapt    y = base + s_g B_g A_g drop(x) with the adapter g = ids[row] of each row, beside a shared projection
  dropout          y = [residual +] drop(x) with the mask of a counter-based generator (Philox4x32-10), never stored
  router_balance   the balance loss of a router and the rows that each expert got

`own` False: elementary torch operations in 32 bits; `own` True: the calls a user makes of the framework.

The mask: element (row, col) of a matrix looks at 16 bits of the Philox block with the counter (col / 8, row, offset mod 2^32, offset / 2^32)
and the key (seed mod 2^32, seed / 2^32): bits 16 (col % 2) of word (col % 8) / 2.  It is dropped where they are below round(65536 p); what stays
is multiplied by 65536 / (65536 - round(65536 p)).
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"fp32": 4, "fp16": 2, "bf16": 2}

# the most that a drawn case costs, per operator: the largest listed case of it
LOWRANK_MOST = 8192 * (4096 + 4096)              # rows * (k + n) of a training step
LOWRANK_MOST_PLAIN = 8192 * (4096 + 4096) * 768  # ... times the rows of all adapters: what the plain form multiplies
DROPOUT_MOST = 16384 * 8192
BALANCE_MOST = 1000003 * 24


def listed():
    return [
        # one token of one request while it is answered: nothing but latency
        dict(name="serve_one", op="lowrank", rows=1, k=4096, n=4096, r=16, g=8, dtype="bf16", train=False, p=0.0, packed=False, idle=0.0),
        # a batch of requests at one token each, some of them without an adapter
        dict(name="serve_batch", op="lowrank", rows=48, k=4096, n=8192, r=32, g=16, dtype="fp16", train=False, p=0.0, packed=False, idle=0.2),
        # the prompts of a dozen requests, packed one behind the other
        dict(name="prompts", op="lowrank", rows=6007, k=4096, n=4096, r=64, g=12, dtype="bf16", train=False, p=0.0, packed=True, idle=0.05),
        # a training step of adapters that a router chooses row by row, dropout on their input
        dict(name="train_wide", op="lowrank", rows=8192, k=4096, n=4096, r=16, g=8, dtype="bf16", train=True, p=0.1, packed=False, idle=0.0),
        # adapters of six maps beside one hidden layer (64 wide) of a shared SDF decoder, at the samples of 0.3 M visible splats
        dict(name="train_decoder", op="lowrank", rows=300000, k=64, n=64, r=8, g=6, dtype="fp32", train=True, p=0.0, packed=False, idle=0.0),
        # nothing divides anything
        dict(name="train_odd", op="lowrank", rows=1111, k=1001, n=777, r=12, g=5, dtype="fp16", train=True, p=0.25, packed=False, idle=0.15),
        # a small hidden layer: the launches are what it costs
        dict(name="dropout_small", op="dropout", rows=64, cols=64, pad=0, dtype="fp32", p=0.1, residual=False),
        # ragged rows out of a wider buffer
        dict(name="dropout_ragged", op="dropout", rows=30011, cols=333, pad=19, dtype="fp16", p=0.3, residual=False),
        # the largest activation of a step, added to its residual stream
        dict(name="dropout_large", op="dropout", rows=16384, cols=8192, pad=0, dtype="bf16", p=0.1, residual=True),
        # a router's smallest batch
        dict(name="balance_small", op="balance", rows=64, e=8, k=2, dtype="fp32", idle=0.0),
        # many small experts, a padded batch
        dict(name="balance_tokens", op="balance", rows=16411, e=128, k=8, dtype="bf16", idle=0.1),
        # the points of a batch over the maps of a scene, one map for each
        dict(name="balance_points", op="balance", rows=1000003, e=24, k=1, dtype="fp32", idle=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lowrank", "lowrank", "dropout", "balance"])
    dtype = rng.choice(["fp32", "fp16", "bf16", "bf16"])
    if op == "lowrank":
        k, n = _log(rng, 32, 8192), _log(rng, 16, 8192)
        if rng.random() < 0.7:      # most layers are whole multiples of 64
            k, n = max(64, k // 64 * 64), max(64, n // 64 * 64)
        r, g = rng.choice([4, 8, 12, 16, 16, 32, 64, 96, 128]), _log(rng, 1, 48)
        g = max(1, min(g, 1536 // r))
        train = rng.random() < 0.5
        most = min(300000, LOWRANK_MOST * (1 if train else 2) // (k + n) // (2 if dtype == "fp32" else 1),
                   LOWRANK_MOST_PLAIN // ((k + n) * r * g))
        return dict(op="lowrank", rows=_log(rng, 1, max(2, most)), k=k, n=n, r=r, g=g, dtype=dtype, train=train,
                    p=rng.choice([0.0, 0.05, 0.1, 0.3]) if train else 0.0, packed=rng.random() < 0.5, idle=rng.choice([0.0, 0.0, 0.1, 0.5]))
    if op == "dropout":
        cols = _log(rng, 1, 16384)
        rows = _log(rng, 1, max(2, min(1 << 20, DROPOUT_MOST // cols // (2 if dtype == "fp32" else 1))))
        return dict(op="dropout", rows=rows, cols=cols, pad=rng.choice([0, 0, 0, 5, 8, 24]), dtype=dtype, p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                    residual=rng.random() < 0.5)
    e = _log(rng, 2, 512)
    k = rng.randint(1, min(8, e))
    return dict(op="balance", rows=_log(rng, 1, BALANCE_MOST // (e * k)), e=e, k=k, dtype=dtype, idle=rng.choice([0.0, 0.1, 0.4]))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    randn = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    rand = lambda *s: torch.rand(*s, generator=g, device=dev)  # noqa: E731
    rows = case["rows"]
    st = dict(case, seed=seed * 7919 + 12345, offset=seed % 1000)
    if case["op"] == "lowrank":
        k, n, r, ng = case["k"], case["n"], case["r"], case["g"]
        st["x"] = randn(rows, k).to(dt)
        st["base"] = randn(rows, n).to(dt)
        st["a"] = (randn(ng, r, k) / math.sqrt(k)).to(dt)
        st["b"] = (randn(ng, n, r) / math.sqrt(r)).to(dt)
        st["scales"] = 0.25 + 1.5 * rand(ng)
        if case["packed"]:      # requests one behind the other: pieces of unequal lengths, each with the adapter of its request
            cuts = (rand(max(1, 2 * ng - 1)) * rows).long().sort().values
            piece = torch.searchsorted(cuts, torch.arange(rows, device=dev), right=True)
            of = torch.randint(0, ng, (2 * ng,), generator=g, device=dev)
            idle = rand(2 * ng) < case["idle"]
            ids = torch.where(idle[piece], -1, of[piece])
        else:                   # some adapters are wanted more than others
            ids = (ng * rand(rows).square()).long().clamp_(max=ng - 1)
            ids = torch.where(rand(rows) < case["idle"], -1, ids)
        st["ids"] = ids.to(torch.int32)
        if case["train"]:
            st["dy"] = randn(rows, n).to(dt)
            for name in ("x", "a", "b"):
                st[name].requires_grad_(True)
    elif case["op"] == "dropout":
        cols = case["cols"]
        st["x"] = randn(rows, cols + case["pad"]).to(dt)[:, :cols].detach().requires_grad_(True)
        st["residual"] = randn(rows, cols).to(dt) if case["residual"] else None
        st["dy"] = randn(rows, cols).to(dt)
    else:
        e, k = case["e"], case["k"]
        logits = (1.5 * randn(rows, e) + randn(e)).to(dt)
        st["ids"] = logits.float().topk(k, dim=1).indices.to(torch.int32)
        st["mask"] = rand(rows) >= case["idle"] if case["idle"] else None
        st["logits"] = logits.requires_grad_(True)
        st["dloss"] = 0.5 + rand(())
    return st


# ---- the plain forms ------------------------------------------------------------------------------------------------------------------------
def _times(m, v):
    """The high and the low half of the 64-bit product of two 32-bit numbers, in integers that hold 63 bits."""
    t = m * (v & 0xFFFF)
    u = m * (v >> 16) + (t >> 16)
    return u >> 16, ((u & 0xFFFF) << 16) | (t & 0xFFFF)


def _keep(rows, cols, p, seed, offset, device):
    blocks = -(-cols // 8)
    c0 = torch.arange(blocks, device=device).expand(rows, blocks)
    c1 = torch.arange(rows, device=device)[:, None].expand(rows, blocks)
    c2, c3 = torch.full_like(c0, offset & 0xFFFFFFFF), torch.full_like(c0, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):     # the rounds of Philox4x32-10: each needs the one before
        h0, l0 = _times(0xD2511F53, c0)
        h1, l1 = _times(0xCD9E8D57, c2)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack((c0, c1, c2, c3), dim=-1)
    pieces = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(rows, blocks * 8)
    return pieces[:, :cols] >= _threshold(p)


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _rescale(p):
    return 65536.0 / (65536 - _threshold(p))


def _plain_lowrank(st):
    dt, dev = st["x"].dtype, st["x"].device
    rows, ng, r = st["rows"], st["g"], st["r"]
    x, a, b = st["x"].detach().float(), st["a"].detach().float(), st["b"].detach().float()
    if st["p"] > 0:
        keep = _keep(rows, st["k"], st["p"], st["seed"], st["offset"], dev)
        x = torch.where(keep, x * _rescale(st["p"]), 0.0)
    # every row through every adapter, and all but its own left out: two products, no loop over adapters
    mine = (st["ids"][:, None] == torch.arange(ng, device=dev, dtype=torch.int32))[..., None]
    down, up = a.reshape(ng * r, -1), b.permute(0, 2, 1).reshape(ng * r, -1)
    scales = st["scales"][:, None]
    h = torch.where(mine, (x @ down.t()).view(rows, ng, r) * scales, 0.0).view(rows, ng * r)
    out = {"y": (st["base"].float() + h @ up).to(dt)}
    if st["train"]:
        dy = st["dy"].float()
        dh = torch.where(mine, (dy @ up.t()).view(rows, ng, r) * scales, 0.0).view(rows, ng * r)
        dx = dh @ down
        if st["p"] > 0:
            dx = torch.where(keep, dx * _rescale(st["p"]), 0.0)
        out["dx"] = dx.to(dt)
        out["da"] = (dh.t() @ x).view(ng, r, -1).to(dt)
        out["db"] = (h.t() @ dy).view(ng, r, -1).permute(0, 2, 1).contiguous().to(dt)
    return out


def _plain_dropout(st):
    x, dt = st["x"].detach().float(), st["x"].dtype
    keep = _keep(st["rows"], st["cols"], st["p"], st["seed"], st["offset"], x.device)
    y = torch.where(keep, x * _rescale(st["p"]), 0.0)
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return {"y": y.to(dt), "dx": torch.where(keep, st["dy"].float() * _rescale(st["p"]), 0.0).to(dt)}


def _plain_balance(st):
    logits, e, k = st["logits"].detach().float(), st["e"], st["k"]
    z = (logits - logits.amax(dim=1, keepdim=True)).exp()
    p = z / z.sum(dim=1, keepdim=True)
    hit = st["ids"][..., None] == torch.arange(e, device=logits.device, dtype=torch.int32)
    if st["mask"] is not None:
        p = torch.where(st["mask"][:, None], p, 0.0)
        hit = hit & st["mask"][:, None, None]
        valid = st["mask"].sum().clamp(min=1).double()
    else:
        valid = torch.full((), float(st["rows"]), dtype=torch.float64, device=logits.device)
    counts = hit.sum(dim=(0, 1))
    # 64 bits: the sum over all rows, and the shares' distance from even ones, which is small beside them
    share = counts.double() / (k * valid)
    loss = e * (share * (p.sum(dim=0, dtype=torch.float64) / valid)).sum()
    pull = (((e * share - 1) / valid) * st["dloss"].double()).float()
    dlogits = p * (pull - (p * pull).sum(dim=1, keepdim=True))
    return {"loss": loss.float(), "counts": counts, "dlogits": dlogits.to(st["logits"].dtype)}


def run(st):
    if not own:
        return {"lowrank": _plain_lowrank, "dropout": _plain_dropout, "balance": _plain_balance}[st["op"]](st)
    from gs_sdf_amd import adapters
    if st["op"] == "lowrank":
        if not st["train"]:
            return {"y": adapters.lowrank_adapt(st["x"], st["a"], st["b"], st["ids"], scales=st["scales"], base=st["base"])}
        y = adapters.lowrank_adapt(st["x"], st["a"], st["b"], st["ids"], scales=st["scales"], base=st["base"], p=st["p"], seed=st["seed"],
                                   offset=st["offset"])
        dx, da, db = torch.autograd.grad(y, (st["x"], st["a"], st["b"]), st["dy"])
        return {"y": y.detach(), "dx": dx, "da": da, "db": db}
    if st["op"] == "dropout":
        y = adapters.dropout(st["x"], st["p"], st["seed"], st["offset"], residual=st["residual"])
        return {"y": y.detach(), "dx": torch.autograd.grad(y, st["x"], st["dy"])[0]}
    loss, counts = adapters.router_balance(st["logits"], st["ids"], mask=st["mask"])
    return {"loss": loss.detach(), "counts": counts, "dlogits": torch.autograd.grad(loss, st["logits"], st["dloss"])[0]}


def work(case):
    s, rows = BYTES[case["dtype"]], case["rows"]
    if case["op"] == "lowrank":
        k, n, r = case["k"], case["n"], case["r"]
        busy, weights = rows * (1 - case["idle"]), min(case["g"], rows) * r * (k + n)
        nbytes, flops = s * (busy * k + 2 * rows * n + weights) + 4 * rows, 2 * busy * r * (k + n)
        if case["train"]:       # dy and x once each, dx; the adapters again, and their gradients whole
            nbytes += s * (busy * (n + k) + rows * k + weights + case["g"] * r * (k + n))
            flops *= 3
        return {"bytes": nbytes, "flops": flops}
    if case["op"] == "dropout":
        n = rows * case["cols"]
        return {"bytes": s * n * (5 if case["residual"] else 4), "flops": 2 * n}
    e, k = case["e"], case["k"]     # logits once for the loss and once for its gradient, which waits for the counts of all rows
    return {"bytes": s * rows * e * 3 + 4 * rows * k + 16 * e, "flops": 12 * rows * e}


# ---- 64 bits, from the definitions ----------------------------------------------------------------------------------------------------------
def _exact_keep(rows, cols, p, seed, offset):
    """numpy's unsigned 64-bit integers: a product of two 32-bit numbers is whole in one of them"""
    shape = (rows, (cols + 7) // 8)
    low = np.uint64(0xFFFFFFFF)
    ctr = [np.broadcast_to(np.arange(shape[1], dtype=np.uint64), shape), np.broadcast_to(np.arange(rows, dtype=np.uint64)[:, None], shape),
           np.full((1, 1), offset & 0xFFFFFFFF, dtype=np.uint64), np.full((1, 1), offset >> 32, dtype=np.uint64)]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        first, second = ctr[0] * np.uint64(0xD2511F53), ctr[2] * np.uint64(0xCD9E8D57)
        ctr = [(second >> np.uint64(32)) ^ ctr[1] ^ np.uint64(key[0]), second & low, (first >> np.uint64(32)) ^ ctr[3] ^ np.uint64(key[1]), first & low]
        key = [(key[0] + 0x9E3779B9) % 2 ** 32, (key[1] + 0xBB67AE85) % 2 ** 32]
    out = np.empty(shape + (8,), dtype=bool)
    border = np.uint64(int(math.floor(p * 65536 + 0.5)))
    for i in range(8):
        out[..., i] = ((ctr[i // 2] >> np.uint64(16 * (i % 2))) & np.uint64(0xFFFF)) >= border
    return torch.from_numpy(out.reshape(rows, -1)[:, :cols])


def exact(case, seed):
    st = prepare(case, seed)
    dev = torch.device("cuda")
    if case["op"] == "lowrank":
        x, a, b, y = (st[name].detach().double() for name in ("x", "a", "b", "base"))
        factor = None
        if case["p"] > 0:
            dropped = int(math.floor(case["p"] * 65536 + 0.5))
            factor = _exact_keep(case["rows"], case["k"], case["p"], st["seed"], st["offset"]).to(dev).double() * (65536 / (65536 - dropped))
            x = x * factor
        dx, da, db = torch.zeros_like(x), torch.zeros_like(a), torch.zeros_like(b)
        for g in range(case["g"]):
            at = (st["ids"] == g).nonzero()[:, 0]
            if not at.numel():
                continue
            s = st["scales"][g].double()
            h = x[at] @ a[g].t().contiguous()
            y[at] += s * (h @ b[g].t().contiguous())
            if case["train"]:
                dy = st["dy"][at].double()
                dh = s * (dy @ b[g])
                dx[at] = dh @ a[g]
                da[g] = dh.t().contiguous() @ x[at]
                db[g] = s * (dy.t().contiguous() @ h)
        if not case["train"]:
            return {"y": y}
        return {"y": y, "dx": dx if factor is None else dx * factor, "da": da, "db": db}
    if case["op"] == "dropout":
        dropped = int(math.floor(case["p"] * 65536 + 0.5))
        factor = _exact_keep(case["rows"], case["cols"], case["p"], st["seed"], st["offset"]).to(dev).double() * (65536 / (65536 - dropped))
        y = st["x"].detach().double() * factor
        return {"y": y if st["residual"] is None else y + st["residual"].double(), "dx": st["dy"].double() * factor}
    logits, e, k = st["logits"].detach().double(), case["e"], case["k"]
    p = torch.softmax(logits, dim=1)
    rows = st["mask"].nonzero()[:, 0] if st["mask"] is not None else torch.arange(case["rows"], device=dev)
    valid = max(1, rows.numel())
    counts = torch.bincount(st["ids"][rows].reshape(-1).long(), minlength=e)
    share = counts.double() / (valid * k)
    loss = e * (share * p[rows].sum(dim=0) / valid).sum()
    c = st["dloss"].double() * e * share / valid
    dlogits = torch.zeros_like(p)
    dlogits[rows] = p[rows] * (c - (p[rows] * c).sum(dim=1, keepdim=True))
    return {"loss": loss, "counts": counts, "dlogits": dlogits}
