"""Plain 64-bit statements of the adapter operators (gs_sdf_amd.adapters), on the CPU: what the kernels are compared with."""
import math

import numpy as np
import torch

# half a step of each type, relative to the value: what one rounding may be off
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# the products of h and dh (32 bits) with 16-bit weights go through the matrix instructions as a high and a low part of the weights' type: what two
# roundings leave is half a step of half a step, relative to the largest value that shares the scale of the split
SPLIT = {torch.float32: 0.0, torch.float16: 2.0 ** -22, torch.bfloat16: 2.0 ** -16}


def philox(ctr, key):
    """Philox4x32-10 of numpy uint64 arrays that hold 32-bit numbers"""
    low = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) for v in ctr]
    k = list(key)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def keep_factor(rows, cols, p, seed, offset, row0=0):
    """[rows, cols] doubles: 0 where dropped, 1 / (1 - q) elsewhere"""
    t = threshold(p)
    if t >= 65536:
        return torch.zeros(rows, cols, dtype=torch.float64)
    blocks = (cols + 7) // 8
    shape = (rows, blocks)
    w = philox([np.broadcast_to(np.arange(blocks, dtype=np.uint64), shape), np.broadcast_to(np.arange(row0, row0 + rows, dtype=np.uint64)[:, None], shape),
                np.full(shape, offset % 2 ** 32, dtype=np.uint64), np.full(shape, offset >> 32, dtype=np.uint64)], (seed % 2 ** 32, seed >> 32))
    bits = np.stack([(w[i // 2] >> np.uint64(16 * (i % 2))) & np.uint64(0xFFFF) for i in range(8)], axis=-1).reshape(rows, blocks * 8)[:, :cols]
    return torch.from_numpy((bits >= np.uint64(t)).astype(np.float64)) * (65536.0 / (65536 - t))


def _d(t):
    return t.detach().cpu().double()


class Lowrank:
    """y and the gradients, and beside each the magnitudes its error goes by: `*_mag` = the sum of the absolute products, `*_split` = the same
    with the split factor replaced by its largest value"""

    def __init__(self, x, a, b, ids, scales=None, base=None, dy=None, p=0.0, seed=0, offset=0):
        x, a, b, ids = _d(x), _d(a), _d(b), ids.cpu().long()
        (G, r, K), N, T = a.shape, b.shape[1], x.shape[0]
        s = torch.ones(G, dtype=torch.float64) if scales is None else _d(scales)
        f = keep_factor(T, K, p, seed, offset) if threshold(p) else torch.ones(T, K, dtype=torch.float64)
        x = torch.where(f != 0, x * f, torch.zeros(()).double())
        self.y = torch.zeros(T, N).double() if base is None else _d(base)
        self.y_mag, self.y_split = self.y.abs(), torch.zeros(T, N).double()
        self.dx, self.da, self.db = torch.zeros(T, K).double(), torch.zeros_like(a), torch.zeros_like(b)
        self.dx_mag, self.da_mag, self.db_mag = torch.zeros(T, K).double(), torch.zeros_like(a), torch.zeros_like(b)
        self.dx_split, self.da_split, self.db_split = torch.zeros(T, K).double(), torch.zeros_like(a), torch.zeros_like(b)
        dy = None if dy is None else _d(dy)
        for g in range(G):
            at = (ids == g).nonzero()[:, 0]
            if not len(at):
                continue
            xg, sg = x[at], s[g]
            h, hm = xg @ a[g].T, xg.abs() @ a[g].abs().T
            self.y[at] += sg * (h @ b[g].T)
            self.y_mag[at] += sg.abs() * (hm @ b[g].abs().T)
            self.y_split[at] += sg.abs() * h.abs().max(dim=1, keepdim=True).values * b[g].abs().sum(dim=1)
            if dy is None:
                continue
            dyg = dy[at]
            dh, dhm = sg * (dyg @ b[g]), sg.abs() * (dyg.abs() @ b[g].abs())
            self.dx[at], self.dx_mag[at] = (dh @ a[g]) * f[at], (dhm @ a[g].abs()) * f[at]
            self.dx_split[at] = dh.abs().max(dim=1, keepdim=True).values * a[g].abs().sum(dim=0) * f[at]
            self.da[g], self.da_mag[g] = dh.T @ xg, dhm.T @ xg.abs()
            self.da_split[g] = dh.abs().max() * xg.abs().sum(dim=0)
            self.db[g], self.db_mag[g] = sg * (dyg.T @ h), sg.abs() * (dyg.abs().T @ hm)
            self.db_split[g] = (sg.abs() * h.abs().max() * dyg.abs().sum(dim=0))[:, None]

    def check(self, name, got, terms):
        """`terms`: how many products are added one after the other at most, over all sums on the way (each addition and each product one 32-bit rounding)"""
        want, mag, split = getattr(self, name), getattr(self, name + "_mag"), getattr(self, name + "_split")
        bound = HALF[got.dtype] * want.abs() + (1 + HALF[got.dtype]) * ((terms + 16) * 2.0 ** -24 * mag + SPLIT[got.dtype] * split)
        within(got, want, bound, name, got.dtype)


def within(got, want, bound, name, dtype):
    got = _d(got)
    assert got.shape == want.shape, f"{name}: shape {tuple(got.shape)}, expected {tuple(want.shape)}"
    tiny = torch.finfo(dtype).smallest_normal if dtype != torch.float32 else 1e-37      # results below the normal numbers keep fewer bits
    off = (got - want).abs() - bound
    bad = ~(off <= tiny * 2.0 ** -8 if dtype == torch.float16 else off <= tiny)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} outside their bounds, worst {off[bad].max() if torch.isfinite(off[bad]).any() else off[bad][:3]} " \
                          f"at {bad.nonzero()[0].tolist()}: got {got[bad][0]}, expected {want[bad][0]}"


class Balance:
    def __init__(self, logits, ids, mask=None, v_loss=1.0):
        z, E = _d(logits), logits.shape[-1]
        T = z.shape[0]
        ids = ids.cpu().long().reshape(T, -1)
        k = ids.shape[1]
        ok = torch.ones(T, dtype=torch.bool) if mask is None else mask.cpu() != 0
        V = max(1, int(ok.sum()))
        z = torch.where(ok[:, None], z, torch.zeros(()).double())
        m = z.max(dim=1, keepdim=True).values
        e = torch.exp(z - torch.where(m == -math.inf, torch.zeros(()).double(), m))
        p = e / torch.where(e.sum(dim=1, keepdim=True) == 0, torch.ones(()).double(), e.sum(dim=1, keepdim=True)) * ok[:, None]
        chosen = ids[ok].reshape(-1)
        self.counts = torch.bincount(chosen[(chosen >= 0) & (chosen < E)], minlength=E)
        share = self.counts.double() / (k * V)
        self.loss = E * (share * p.sum(dim=0) / V).sum()
        c = (E * share - 1) / V if ok.any() else torch.zeros(E).double()
        dot = (p * c).sum(dim=1, keepdim=True)
        self.v = v_loss * p * (c - dot)
        # p: a few roundings of exp, of the sum over the row, of the quotient; c and the sum over p c likewise
        self.v_bound = (3 * E + 48) * 2.0 ** -24 * abs(v_loss) * p * (c.abs() + (p * c.abs()).sum(dim=1, keepdim=True))
        self.loss_bound = (E + T + 48) * 2.0 ** -24 * self.loss
