"""The adapter operators (gs_sdf_amd.adapters) on the GPU against plain 64-bit statements of them (adapters_ref.py).  Bounds: half a step of the result's type,
the 32-bit roundings of the sums, the split of 32-bit factors in front of 16-bit matrix instructions; derived there, none is fitted."""
import math

import pytest
import torch

import adapters_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[1] for d in DTYPES]


@pytest.fixture(scope="module")
def ad():
    from gs_sdf_amd import adapters
    return adapters


def make(rows, k, n, r, g, dtype, idle=0.0, packed=False, seed=0, dev="cuda", ids_dtype=torch.int32):
    gen = torch.Generator().manual_seed(seed + 31 * rows + k)
    x = torch.randn(rows, k, generator=gen)
    a, b = torch.randn(g, r, k, generator=gen) / math.sqrt(k), torch.randn(g, n, r, generator=gen) / math.sqrt(r)
    ids = torch.randint(0, g, (rows,), generator=gen)
    if packed:
        ids = ids.sort().values[torch.arange(rows).roll(rows // 3)]
    ids = torch.where(torch.rand(rows, generator=gen) < idle, -1, ids)
    scales = 0.25 + 1.5 * torch.rand(g, generator=gen)
    base, dy = torch.randn(rows, n, generator=gen), torch.randn(rows, n, generator=gen)
    return [t.to(dtype).to(dev) for t in (x, a, b)] + [ids.to(ids_dtype).to(dev), scales.to(dev)] + [t.to(dtype).to(dev) for t in (base, dy)]


#        rows, k, n, r, g, idle, packed: one token to many; whole and odd widths; a rank of one to the largest; adapters without rows
SHAPES = [(1, 64, 64, 16, 1, 0.0, False), (1, 1, 1, 1, 1, 0.0, False), (2, 7, 5, 3, 4, 0.0, False), (3, 4096, 33, 16, 8, 0.0, False), (16, 33, 2050, 8, 3, 0.3, False),
          (17, 129, 65, 17, 5, 0.0, False), (63, 200, 100, 64, 7, 0.2, True), (64, 256, 128, 32, 2, 0.0, True), (65, 72, 80, 128, 3, 0.0, False),
          (130, 1000, 1001, 12, 40, 0.1, False), (257, 40, 24, 100, 2, 0.5, False), (700, 136, 264, 16, 6, 0.05, False), (2500, 64, 64, 8, 6, 0.0, False),
          (5000, 32, 16, 4, 12, 0.1, True), (1500, 512, 96, 48, 9, 0.0, True), (3000, 16, 300, 20, 1000, 0.1, False), (900, 300, 16, 65, 1, 0.0, False),
          (20000, 24, 40, 16, 9, 0.05, False), (40000, 8, 8, 2, 1024, 0.1, False), (70000, 64, 64, 8, 6, 0.05, False), (66000, 24, 72, 20, 5, 0.1, True), (65600, 72, 8, 4, 3, 0.0, False),
          (9500, 136, 72, 20, 3, 0.0, False), (9800, 72, 136, 64, 2, 0.0, True), (10000, 64, 64, 128, 3, 0.02, False), (8200, 1040, 1024, 16, 5, 0.0, False),
          (8200, 64, 2112, 8, 5, 0.0, False), (48, 2048, 1024, 32, 4, 0.1, False), (2048, 64, 48, 8, 3, 0.0, False), (2049, 64, 48, 8, 1, 0.0, False), (4500, 264, 136, 96, 3, 0.0, True)]


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_lowrank_forward(ad, shape, dtype):
    rows, k, n, r, g, idle, packed = shape
    x, a, b, ids, scales, base, _ = make(rows, k, n, r, g, dtype, idle, packed)
    want = ref.Lowrank(x, a, b, ids, scales, base)
    got = ad.lowrank_adapt(x, a, b, ids, scales, base)
    want.check("y", got, k + r)
    none = (ids < 0).cpu()
    assert torch.equal(got.cpu()[none], base.cpu()[none])      # no adapter: base itself
    got = ad.lowrank_adapt(x, a, b, ids.long())                # no base, no scales, 64-bit ids
    ref.Lowrank(x, a, b, ids).check("y", got, k + r)
    assert (got.cpu()[none] == 0).all()


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s[:5])))
def test_lowrank_gradients(ad, shape, dtype, p):
    rows, k, n, r, g, idle, packed = shape
    x, a, b, ids, scales, base, dy = make(rows, k, n, r, g, dtype, idle, packed, seed=1)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy, p, 99, 12345678901)
    for t in (x, a, b, base):
        t.requires_grad_(True)
    y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=p, seed=99, offset=12345678901)
    dx, da, db, dbase = torch.autograd.grad(y, (x, a, b, base), dy)
    want.check("y", y, k + r)
    want.check("dx", dx, n + r)
    want.check("da", da, n + rows)
    want.check("db", db, k + rows)
    assert torch.equal(dbase, dy)
    empty = torch.tensor([i for i in range(g) if not (ids == i).any()], dtype=torch.long, device=x.device)
    assert (da[empty] == 0).all() and (db[empty] == 0).all() and (dx[ids < 0] == 0).all()


@pytest.mark.parametrize("which", ["x", "a", "b"])
def test_lowrank_one_gradient_at_a_time(ad, which):
    x, a, b, ids, scales, base, dy = make(200, 96, 80, 16, 4, torch.bfloat16, 0.1)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    leaf = {"x": x, "a": a, "b": b}[which].requires_grad_(True)
    y = ad.lowrank_adapt(x, a, b, ids, scales, base)
    want.check("d" + which, torch.autograd.grad(y, leaf, dy)[0], 96 + 80 + 200)


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("rows,r", [(65536, 8), (66000, 24), (70001, 6), (9000, 64)])
@pytest.mark.parametrize("which", ["x", "a", "b", "ab", "xb"])
def test_lowrank_some_gradients_of_many_rows(ad, which, rows, r, p):
    """the factors that want no gradient are left out on every path, the one that takes rows through both products at once among them"""
    x, a, b, ids, scales, base, dy = make(rows, 40, 72, r, 5, torch.bfloat16, 0.1)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy, p, 5, 6)
    leaves = [{"x": x, "a": a, "b": b}[w].requires_grad_(True) for w in which]
    grads = torch.autograd.grad(ad.lowrank_adapt(x, a, b, ids, scales, base, p=p, seed=5, offset=6), leaves, dy)
    for w, g in zip(which, grads):
        want.check("d" + w, g, 40 + 72 + rows)


def test_lowrank_gradients_against_differences(ad):
    """d/de of sum(y dy) along random directions, by differences of the 64-bit forward, against the kernels' gradients"""
    x, a, b, ids, scales, base, dy = make(90, 37, 29, 9, 5, torch.float32, 0.1)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    grads = torch.autograd.grad(ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.2, seed=3, offset=4), leaves, dy)
    gen = torch.Generator().manual_seed(5)
    for i in range(3):
        d = torch.randn(leaves[i].shape, generator=gen).double()
        at = lambda e: float((ref.Lowrank(*[leaves[j].detach().cpu().double() + (e * d if j == i else 0) for j in range(3)], ids, scales, base, p=0.2, seed=3,  # noqa: E731
                                          offset=4).y * dy.cpu().double()).sum())
        slope = (at(1e-3) - at(-1e-3)) / 2e-3      # y is linear in each factor: the difference is exact but for 64-bit roundings
        got = float((grads[i].cpu().double() * d).sum())
        scale = float((grads[i].cpu().double() * d).abs().sum())
        assert abs(got - slope) < 200 * 2.0 ** -24 * scale + 1e-9 * abs(at(0.0))


def test_lowrank_without_base(ad):
    x, a, b, ids, scales, _, dy = make(90, 40, 56, 8, 3, torch.float32, 0.1)
    want = ref.Lowrank(x, a, b, ids, scales, None, dy)
    x = x.view(30, 3, 40).requires_grad_(True)
    y = ad.lowrank_adapt(x, a, b, ids.view(30, 3), scales)
    want.check("y", y.view(90, 56), 48)
    want.check("dx", torch.autograd.grad(y, x, dy.view(y.shape))[0].view(90, 40), 64)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n", [(5, 41, 23), (300, 41, 23), (300, 128, 64)])
def test_lowrank_strided_rows_and_any_alignment(ad, dtype, rows, k, n):
    """rows out of wider buffers that begin at any element, an upstream gradient that is one expanded row"""
    x, a, b, ids, scales, base, dy = make(rows, k, n, 8, 3, dtype, 0.1)
    wide = lambda t, before, after: torch.cat([torch.full((rows, before), math.nan, dtype=dtype, device=t.device), t,  # noqa: E731
                                               torch.full((rows, after), math.nan, dtype=dtype, device=t.device)], 1)[:, before:before + t.shape[1]]
    xs, bs = wide(x, 3, 6), wide(base, 1, 0)
    shift = lambda t: torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)  # noqa: E731      one element off any alignment
    one = dy[:1].expand(rows, n)
    want = ref.Lowrank(x, a, b, ids, scales, base, one, 0.1, 7, 8)
    xs.requires_grad_(True)
    a1, b1 = shift(a).requires_grad_(True), shift(b).requires_grad_(True)
    y = ad.lowrank_adapt(xs, a1, b1, ids, scales, bs, p=0.1, seed=7, offset=8)
    dx, da, db = torch.autograd.grad(y, (xs, a1, b1), one)
    want.check("y", y, k + 8)
    want.check("dx", dx, n + 8)
    want.check("da", da, n + rows)
    want.check("db", db, k + rows)
    with torch.no_grad():
        ref.Lowrank(x, a, b, ids, scales, base).check("y", ad.lowrank_adapt(xs, a1, b1, ids, scales, bs), k + 8)


@pytest.mark.parametrize("rows", [3, 200])
def test_lowrank_leading_dimensions_and_columns_first(ad, rows):
    x, a, b, ids, scales, base, dy = make(rows * 4, 48, 56, 8, 3, torch.float32)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    x4, b4 = x.view(rows, 2, 2, 48).requires_grad_(True), base.view(rows, 2, 2, 56)
    y = ad.lowrank_adapt(x4, a, b, ids.view(rows, 2, 2), scales, b4)
    assert y.shape == (rows, 2, 2, 56)
    want.check("y", y.view(-1, 56), 56)
    want.check("dx", torch.autograd.grad(y, x4, dy.view(y.shape))[0].view(-1, 48), 64)
    xt = x.detach().t().contiguous().t()      # column-major
    want.check("y", ad.lowrank_adapt(xt, a, b, ids, scales, base), 56)
    one = ad.lowrank_adapt(x[0].detach(), a, b, ids[0], scales, base[0])
    assert one.shape == (56,) and torch.allclose(one, y.view(-1, 56)[0], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("rows", [0, 1])
def test_lowrank_no_rows_and_no_adapters(ad, rows):
    x, a, b, ids, scales, base, dy = make(rows, 24, 40, 8, 3, torch.float32)
    ids = torch.full_like(ids, -1)
    for t in (x, a, b):
        t.requires_grad_(True)
    y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.5, seed=1)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    assert torch.equal(y, base) and (dx == 0).all() and (da == 0).all() and (db == 0).all() and dx.shape == x.shape
    assert torch.equal(ad.lowrank_adapt(x.detach(), a, b, ids, scales, base), base)


@pytest.mark.parametrize("rows", [9, 500])
def test_lowrank_ids_outside_the_adapters_take_none(ad, rows):
    x, a, b, ids, scales, base, dy = make(rows, 40, 24, 8, 3, torch.float32, ids_dtype=torch.int64)
    wild = ids.clone()
    wild[1::4] = torch.tensor([3, -1, 2 ** 40, -2 ** 62], device=ids.device)[torch.arange(len(wild[1::4]), device=ids.device) % 4]
    plain = torch.where((wild >= 0) & (wild < 3), wild, -1)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = ad.lowrank_adapt(x, a, b, wild, scales, base)
    assert torch.equal(y, ad.lowrank_adapt(x, a, b, plain, scales, base))
    ref.Lowrank(x, a, b, plain, scales, base).check("y", y, 48)
    for got, want in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(ad.lowrank_adapt(x, a, b, plain, scales, base), leaves, dy)):
        assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [6, 300])
def test_lowrank_infinities_stay_in_their_rows_and_adapters(ad, rows, dtype):
    x, a, b, ids, scales, base, dy = make(rows, 72, 40, 16, 4, dtype)
    ids = torch.arange(rows, device=ids.device, dtype=torch.int32) % 4
    clean = ref.Lowrank(x, a, b, ids, scales, base, dy)
    x[2], dy[2] = math.nan, math.inf      # a row of adapter 2
    a[3], b[3] = math.nan, -math.inf      # adapter 3 as a whole
    for t in (x, a, b):
        t.requires_grad_(True)
    y = ad.lowrank_adapt(x, a, b, ids, scales, base)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    rows_ok = (ids.cpu() != 3) & (torch.arange(rows) != 2)
    for name, got, terms in (("y", y, 88), ("dx", dx, 56)):
        w = ref.HALF[dtype] * getattr(clean, name).abs() + (terms + 16) * 2.0 ** -23 * getattr(clean, name + "_mag") + 2 * ref.SPLIT[dtype] * getattr(clean, name + "_split")
        ref.within(got[rows_ok], getattr(clean, name)[rows_ok], w[rows_ok], name, dtype)
    assert torch.isfinite(da[:2].float()).all() and torch.isfinite(db[:2].float()).all()
    assert not torch.isfinite(y[2].float()).any() and not torch.isfinite(da[2].float()).any()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("shape", [(1, 64, 64, 16, 1), (5, 33, 70, 20, 3), (48, 256, 128, 32, 4), (300, 41, 23, 12, 3), (300, 128, 64, 8, 9), (700, 264, 1024, 100, 2), (3000, 64, 40, 8, 5),
                                   (20000, 24, 64, 64, 7), (65567, 8, 128, 24, 200), (65567, 128, 8, 24, 200), (66000, 64, 64, 8, 6), (66000, 72, 100, 4, 3), (66000, 128, 64, 7, 3)],
                         ids=lambda s: "x".join(map(str, s)))
def test_lowrank_reads_nothing_it_did_not_write(ad, shape, dtype):
    """the saved buffer, the workspaces and what lies behind them hold NaN: the results are those of buffers of zeros"""
    import ctypes as C
    from gs_sdf_amd import capi
    L, (rows, k, n, r, g) = capi.lib(), shape
    x, a, b, ids, scales, base, dy = make(rows, k, n, r, g, dtype, 0.1, rows > 20000)
    d = dict(rows=rows, x_stride=k, n_in=k, n_out=n, rank=r, n_adapters=g, dtype=DTYPES.index(dtype), ids_64=0, x=x.data_ptr(), a=a.data_ptr(), b=b.data_ptr(), ids=ids.data_ptr(),
             scales=scales.data_ptr(), p=0.1, seed=1, offset=2, offset_dev=None)
    args = C.byref(capi.LowrankArgs(*[d[name] for name, _ in capi.LowrankArgs._fields_]))
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    got = []
    for fill in (0, 255):
        hold = lambda size: torch.full((size + 65536,), fill, dtype=torch.uint8, device="cuda")  # noqa: E731
        save, ws, wb = hold(L.gsdf_lowrank_save_bytes(args)), hold(L.gsdf_lowrank_fwd_ws_bytes(args)), hold(L.gsdf_lowrank_bwd_ws_bytes(args))
        y, alone, dx, da, db = (torch.full_like(t, math.nan) for t in (base, base, x, a, b))
        assert L.gsdf_lowrank_fwd(args, base.data_ptr(), n, y.data_ptr(), n, save.data_ptr(), ws.data_ptr(), stream) == 0
        assert L.gsdf_lowrank_bwd(args, dy.data_ptr(), n, save.data_ptr(), dx.data_ptr(), k, da.data_ptr(), db.data_ptr(), wb.data_ptr(), stream) == 0
        assert L.gsdf_lowrank_fwd(args, base.data_ptr(), n, alone.data_ptr(), n, None, hold(L.gsdf_lowrank_fwd_ws_bytes(args)).data_ptr(), stream) == 0
        torch.cuda.synchronize()
        got.append((y, alone, dx, da, db))
    for u, v in zip(*got):
        assert torch.isfinite(u).all() and torch.equal(u, v)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("k,n", [(8, 128), (128, 8), (64, 72)])
def test_lowrank_infinities_of_many_rows_stay_in_their_adapters(ad, k, n, dtype):
    x, a, b, ids, scales, base, dy = make(65600, k, n, 8, 3, dtype, 0.05)
    want = ref.Lowrank(x, a[:2], b[:2], torch.where(ids == 2, -1, ids), scales[:2], base, dy)
    a[2], b[2] = math.inf, math.inf
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = ad.lowrank_adapt(x, a, b, ids, scales, base)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    ok = (ids != 2).cpu()
    for name, t in (("y", y), ("dx", dx)):
        for suffix in ("", "_mag", "_split"):
            setattr(want, name + suffix, getattr(want, name + suffix)[ok])
        want.check(name, t[ok.cuda()], k + n)
    want.check("da", da[:2], n + 65600)
    want.check("db", db[:2], k + 65600)


def test_lowrank_dropped_infinities_are_gone(ad):
    x, a, b, ids, scales, base, dy = make(64, 80, 40, 8, 2, torch.bfloat16)
    f = ref.keep_factor(64, 80, 0.5, 11, 3)
    hole = torch.where(f == 0, torch.tensor(math.nan), x.float().cpu()).to(x.dtype).to(x.device)
    for t in (hole, a, b):
        t.requires_grad_(True)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy, 0.5, 11, 3)
    y = ad.lowrank_adapt(hole, a, b, ids, scales, base, p=0.5, seed=11, offset=3)
    dx, da, db = torch.autograd.grad(y, (hole, a, b), dy)
    want.check("y", y, 88)
    want.check("dx", dx, 48)
    want.check("da", da, 104)
    want.check("db", db, 144)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["float16", "bfloat16"])
@pytest.mark.parametrize("size", [1e-4, 300.0])
def test_lowrank_small_and_large_inner_values(ad, dtype, size):
    """h and dh far from 1: below the normal 16-bit numbers, or above the largest of them, where y is not"""
    x, a, b, ids, scales, base, dy = make(150, 512, 48, 16, 3, dtype)
    x, b, dy = x * size, b / size, dy * (1e-3 if size < 1 else 1.0)
    a = a * (1e-2 if size < 1 else 20.0)
    b = b * (1.0 if size < 1 else 0.05)
    for t in (x, a, b):
        t.requires_grad_(True)
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    assert size < 1 or float((x.detach().double() @ a.detach()[0].double().t()).abs().max()) > 2e4
    y = ad.lowrank_adapt(x, a, b, ids, scales, base)
    dx, da, db = torch.autograd.grad(y, (x, a, b), dy)
    want.check("y", y, 528)
    want.check("dx", dx, 64)
    want.check("da", da, 198)
    if float(want.db.abs().max()) < 6e4 or dtype == torch.bfloat16:
        want.check("db", db, 662)


@pytest.mark.parametrize("rows", [7, 300])
def test_lowrank_in_place(ad, rows):
    x, a, b, ids, scales, base, _ = make(rows, 64, 48, 16, 3, torch.bfloat16, 0.4)
    buf = torch.full((rows + 5, 60), 3.0, dtype=torch.bfloat16, device=x.device)
    buf[:rows, 4:52] = base
    before = buf.clone()
    y = buf[:rows, 4:52]
    version = y._version
    out = ad.lowrank_adapt_(y, x, a, b, ids, scales)
    assert out is y and y._version > version
    assert torch.equal(y, ad.lowrank_adapt(x, a, b, ids, scales, base))
    buf[:rows, 4:52] = before[:rows, 4:52]
    assert torch.equal(buf, before)      # the columns beside, the rows behind


@pytest.mark.parametrize("rows", [1, 5, 300])
def test_lowrank_in_place_beside_its_own_input(ad, rows):
    """y and x are columns of one buffer: apart they may be, on one another they may not"""
    x, a, b, ids, scales, base, _ = make(rows, 40, 24, 8, 3, torch.bfloat16, 0.1)
    want = ref.Lowrank(x, a, b, ids, scales, base)
    for x0, y0 in ((0, 40), (24, 0), (30, 3)):
        big = torch.zeros(rows, 72, dtype=x.dtype, device="cuda")
        big[:, x0:x0 + 40], big[:, y0:y0 + 24] = x, base
        want.check("y", ad.lowrank_adapt_(big[:, y0:y0 + 24], big[:, x0:x0 + 40], a, b, ids, scales), 48)
        assert torch.equal(big[:, x0:x0 + 40], x)
    big = torch.zeros(rows + 1, 72, dtype=x.dtype, device="cuda")
    for x0, y0 in ((0, 39), (23, 0), (30, 7), (10, 20), (0, 0)):
        with pytest.raises(RuntimeError, match="share memory"):
            ad.lowrank_adapt_(big[:rows, y0:y0 + 24], big[:rows, x0:x0 + 40], a, b, ids, scales)
    flat = big.view(-1)
    with pytest.raises(RuntimeError, match="share memory"):      # rows of different strides
        ad.lowrank_adapt_(flat[39:39 + rows * 24].view(rows, 24), flat[:rows * 40].view(rows, 40), a, b, ids, scales)
    if rows == 1:
        return
    with pytest.raises(RuntimeError, match="share memory"):      # x is one row, and it lies in y
        ad.lowrank_adapt_(big[:rows, :24], big[1:2, :40].expand(rows, 40), a, b, ids, scales)


def test_lowrank_rows_behind_32_bits(ad):
    """element offsets above 2^32 in x, base, y and dx"""
    rows, stride, k, n = 9, 1 << 29, 72, 40
    x, a, b, ids, scales, base, dy = make(rows, k, n, 8, 3, torch.float16)
    big = torch.empty(rows * stride, dtype=torch.float16, device=x.device).view(rows, stride)
    big[:, :k], big[:, 1024:1024 + n] = x, base
    xs, bs = big[:, :k], big[:, 1024:1024 + n]
    want = ref.Lowrank(x, a, b, ids, scales, base, dy, 0.2, 1, 2)
    y = ad.lowrank_adapt(xs.detach(), a, b, ids, scales, bs)
    ref.Lowrank(x, a, b, ids, scales, base).check("y", y, k + 8)
    ad.lowrank_adapt_(bs, xs.detach(), a, b, ids, scales)
    assert torch.equal(bs, y)
    bs.copy_(base)
    xs = xs.detach().requires_grad_(True)
    y = ad.lowrank_adapt(xs, a, b, ids, scales, bs, p=0.2, seed=1, offset=2)
    want.check("y", y, k + 8)
    want.check("dx", torch.autograd.grad(y, xs, dy)[0], n + 8)
    d = ad.dropout(big[:, :k].detach(), 0.3, 5)
    assert torch.equal(d, ad.dropout(x, 0.3, 5))


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n,r", [(5, 200, 96, 16), (60, 2048, 1024, 32), (900, 136, 72, 12), (66000, 64, 64, 8)])
def test_lowrank_one_mask_on_every_path(ad, rows, k, n, r, dtype):
    """with and without gradients, few rows and many: the same elements are dropped"""
    x, a, b, ids, scales, base, _ = make(rows, k, n, r, 4, dtype, 0.1)
    want = ref.Lowrank(x, a, b, ids, scales, base, None, 0.3, 21, 22)
    want.check("y", ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.3, seed=21, offset=22), k + r)
    want.check("y", ad.lowrank_adapt(x.requires_grad_(True), a, b, ids, scales, base, p=0.3, seed=21, offset=torch.tensor([22], device="cuda")), k + r)


def test_lowrank_backward_twice_and_a_moved_counter(ad):
    x, a, b, ids, scales, base, dy = make(300, 64, 48, 8, 3, torch.float32)
    x.requires_grad_(True)
    word = torch.tensor([5], device="cuda")
    y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.3, seed=1, offset=word)
    z = ad.dropout(x, 0.3, 1, word)
    first = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(y, x, dy, retain_graph=True)[0])
    word += 1      # the masks of the forward passes are gone
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z.sum(), x)


def test_lowrank_infinite_factors(ad):
    """32 bits: what the formula gives; 16 bits: not finite there, and nowhere else"""
    for dtype in DTYPES:
        for rows in (3, 200):
            x, a, b, ids, scales, base, _ = make(rows, 40, 24, 1, 2, dtype)
            a, b, x = a.abs() + 0.1, b.abs() + 0.1, x.abs() + 0.1
            ids[:2] = torch.tensor([0, 1], device="cuda", dtype=torch.int32)
            x[0, 7], b[1, 5] = math.inf, math.inf
            y = ad.lowrank_adapt(x, a, b, ids, scales, base).float()
            assert (y[0] == math.inf).all()
            hit = torch.zeros_like(y, dtype=torch.bool)
            hit[0], hit[ids == 1, 5] = True, True
            assert torch.equal(~torch.isfinite(y), hit) and (dtype != torch.float32 or (y[hit] == math.inf).all())


def test_lowrank_results_do_not_change_from_run_to_run(ad):
    x, a, b, ids, scales, base, dy = make(3000, 256, 192, 16, 7, torch.bfloat16, 0.1)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]

    def step():
        y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.1, seed=1)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, dy))
    first = step()
    for _ in range(5):
        assert all(torch.equal(u, v) for u, v in zip(first, step()))


# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,p", [(1, 1, 0.5), (1, 100003, 0.1), (70001, 1, 0.5), (3, 8, 0.9), (257, 333, 0.3), (64, 64, 0.1), (40, 4096, 0.0), (5, 77, 1.0),
                                         (9, 16, 1e-6), (1000, 7, 0.25)])
def test_dropout(ad, rows, cols, p, dtype):
    gen = torch.Generator().manual_seed(rows + cols)
    x, res, dy = [torch.randn(rows, cols, generator=gen).to(dtype).cuda() for _ in range(3)]
    f = ref.keep_factor(rows, cols, p, 2 ** 63 + 5, 2 ** 33 + 1)
    x.requires_grad_(True)
    res.requires_grad_(True)
    y = ad.dropout(x, p, 2 ** 63 + 5, 2 ** 33 + 1)
    want = x.detach().cpu().double() * f
    rounds = (ref.HALF[dtype] + 2.0 ** -23) * want.abs()      # the factor's rounding, the product's, the result's
    ref.within(y, want, rounds, "y", dtype)
    assert torch.equal((y.cpu() == 0), (f == 0) | (x.detach().cpu() == 0) | (y.cpu() == 0) & (f != 0))
    ref.within(torch.autograd.grad(y, x, dy)[0], dy.cpu().double() * f, (ref.HALF[dtype] + 2.0 ** -23) * (dy.cpu().double() * f).abs(), "dx", dtype)
    y = ad.dropout(x, p, 2 ** 63 + 5, 2 ** 33 + 1, residual=res)
    total = want + res.detach().cpu().double()
    ref.within(y, total, ref.HALF[dtype] * total.abs() + 2.0 ** -22 * (want.abs() + res.detach().cpu().double().abs()), "y", dtype)
    assert torch.equal(y.detach().cpu()[f == 0], res.detach().cpu()[f == 0])
    dx, dres = torch.autograd.grad(y, (x, res), dy)
    assert torch.equal(dres, dy) and ((dx.cpu() == 0) | (f != 0)).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_dropout_goes_by_place_and_not_by_layout(ad, dtype):
    x = torch.randn(37, 50, device="cuda").to(dtype)
    want = ad.dropout(x, 0.4, 8, 9)
    wide = torch.full((37, 71), math.nan, dtype=dtype, device="cuda")
    wide[:, 3:53] = x
    assert torch.equal(ad.dropout(wide[:, 3:53], 0.4, 8, 9), want)
    assert torch.equal(ad.dropout(x.t().contiguous().t(), 0.4, 8, 9), want)
    assert torch.equal(ad.dropout(x.view(37, 1, 50), 0.4, 8, 9).view(37, 50), want)
    assert torch.equal(ad.dropout(x, 0.4, 8, torch.tensor([9], device="cuda")), want)
    assert torch.equal(ad.dropout(x[:1].expand(37, 50), 0.4, 8, 9), ad.dropout(x[:1].expand(37, 50).contiguous(), 0.4, 8, 9))
    assert not torch.equal(ad.dropout(x, 0.4, 8, 10) == 0, want == 0) and not torch.equal(ad.dropout(x, 0.4, 9, 9) == 0, want == 0)
    x[want == 0] = math.inf
    assert torch.equal(ad.dropout(x, 0.4, 8, 9), want)      # what is dropped is gone
    assert ad.dropout(x[:0], 0.4, 8).shape == (0, 50) and ad.dropout(x[:, :0], 0.4, 8).shape == (37, 0)


def test_dropout_many_elements(ad):
    """more than 2^31 elements: rows at the end, and columns at the end of one long row, are those of the definition"""
    rows, cols = 300007, 8192
    x = torch.ones(rows, cols, dtype=torch.bfloat16, device="cuda")
    y = ad.dropout(x, 0.25, 3, 1)
    for r0 in (0, 262143, rows - 2):
        assert torch.equal(y[r0:r0 + 2].cpu() == 0, ref.keep_factor(2, cols, 0.25, 3, 1, row0=r0) == 0)
    line = ad.dropout(x.view(-1), 0.25, 3, 1)
    n = rows * cols
    blocks = torch.arange(n // 8 - 64, n // 8).numpy().astype("uint64")
    w = ref.philox([blocks, blocks * 0, blocks * 0 + 1, blocks * 0], (3, 0))
    bits = torch.stack([torch.from_numpy(((w[i // 2] >> (16 * (i % 2))) & 0xFFFF).astype("int64")) for i in range(8)], dim=1).reshape(-1)
    assert torch.equal(line[-512:].cpu() == 0, bits < 16384)


# ------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,e,k,idle", [(1, 1, 1, 0.0), (1, 2, 2, 0.0), (5, 3, 1, 0.0), (64, 8, 2, 0.0), (100, 9, 3, 0.3), (1000, 24, 1, 0.0), (333, 64, 8, 0.1),
                                           (700, 100, 4, 0.0), (513, 128, 8, 0.2), (90, 255, 6, 0.0), (77, 500, 8, 0.5), (50, 513, 2, 0.0), (40, 1024, 8, 0.1),
                                           (20000, 16, 2, 0.4), (70000, 5, 1, 0.0)])
def test_balance(ad, rows, e, k, idle, dtype):
    gen = torch.Generator().manual_seed(rows + e)
    logits = (2 * torch.randn(rows, e, generator=gen) + torch.randn(e, generator=gen)).to(dtype)
    ids = logits.float().topk(k, dim=1).indices
    mask = torch.rand(rows, generator=gen) >= idle if idle else None
    if mask is not None:
        logits[~mask] = math.nan      # what a padded row holds is nobody's business
    want = ref.Balance(logits, ids, mask, 1.75)
    lg = logits.cuda().requires_grad_(True)
    for idt in (torch.int32, torch.int64):
        loss, counts = ad.router_balance(lg, ids.to(idt).cuda(), None if mask is None else mask.cuda())
        assert torch.equal(counts.cpu(), want.counts) and counts.dtype == torch.int64
        assert abs(float(loss.detach()) - float(want.loss)) <= float(want.loss_bound) + 1e-30
        g, = torch.autograd.grad(loss, lg, torch.tensor(1.75, device="cuda"))
        ref.within(g, want.v, ref.HALF[dtype] * want.v.abs() + 1.01 * want.v_bound, "dlogits", dtype)
        if mask is not None:
            assert (g.cpu()[~mask] == 0).all()
    with torch.no_grad():
        again, c2 = ad.router_balance(lg, ids.cuda(), None if mask is None else mask.cuda())
        assert torch.equal(again, loss) and torch.equal(c2, counts)


def test_balance_edges(ad):
    lowest = torch.finfo(torch.float32).min
    gen = torch.Generator().manual_seed(6)
    z = torch.randn(40, 12, generator=gen)
    z[:, 5] = -math.inf          # an expert that nobody may choose
    z[3] = lowest                # even, that expert too
    z[4] = -math.inf             # nothing left: no probability, no gradient
    z[6, :11] = lowest           # one expert left
    ids = torch.randint(0, 12, (40, 2), generator=gen)
    ids[7] = torch.tensor([-1, 12])      # dropped choices
    ids[8] = torch.tensor([3, 3])        # the same expert twice
    want = ref.Balance(z, ids)
    lg = z.cuda().requires_grad_(True)
    loss, counts = ad.router_balance(lg, ids.cuda())
    assert torch.equal(counts.cpu(), want.counts) and abs(float(loss.detach()) - float(want.loss)) <= float(want.loss_bound)
    g, = torch.autograd.grad(loss, lg)
    ref.within(g, want.v, ref.HALF[torch.float32] * want.v.abs() + 1.01 * want.v_bound, "dlogits", torch.float32)
    assert (g[4] == 0).all() and (g[torch.arange(40) != 3, 5] == 0).all()
    for rows in (0, 40):         # nobody is there
        none = torch.zeros(rows, dtype=torch.uint8, device="cuda")
        lg = z[:rows].cuda().requires_grad_(True)
        loss, counts = ad.router_balance(lg, ids[:rows].cuda(), none)
        assert float(loss) == 0 and (counts == 0).all() and (torch.autograd.grad(loss, lg)[0] == 0).all()
    wide = torch.full((40, 20), math.nan, device="cuda")
    wide[:, 3:15] = z.cuda()
    assert torch.equal(ad.router_balance(wide[:, 3:15], ids.cuda())[0], ad.router_balance(z.cuda(), ids.cuda())[0])
    one = z[:1].expand(40, 12)
    lg = z[:1].cuda().requires_grad_(True)
    got = ad.router_balance(lg.expand(40, 12), ids.cuda())[0]
    want = ref.Balance(one, ids)
    assert abs(float(got.detach()) - float(want.loss)) <= float(want.loss_bound)
    assert torch.allclose(torch.autograd.grad(got, lg)[0].cpu().double()[0], want.v.sum(dim=0), rtol=1e-4, atol=1e-7)
    lead = ad.router_balance(z.cuda().view(5, 8, 12), ids.cuda().view(5, 8, 2))
    assert torch.equal(lead[0], ad.router_balance(z.cuda(), ids.cuda())[0])


def test_balance_gradient_against_differences(ad):
    gen = torch.Generator().manual_seed(4)
    z = torch.randn(30, 10, generator=gen)
    ids = z.topk(2, dim=1).indices
    lg = z.cuda().requires_grad_(True)
    g = torch.autograd.grad(ad.router_balance(lg, ids.cuda())[0], lg)[0].cpu().double()
    d = torch.randn(30, 10, generator=gen).double()
    at = lambda e: float(ref.Balance(z.double() + e * d, ids).loss)  # noqa: E731
    slope = (8 * (at(1e-3) - at(-1e-3)) - (at(2e-3) - at(-2e-3))) / 12e-3      # error of the fourth order in 1e-3
    assert abs(slope - float((g * d).sum())) < 1e-9 + 1e-5 * float((g * d).abs().sum())


# ------------------------------------------------------------------------------------------------
def routed_step(ad, p_in, p_out, seed, x, w, a, b, wr, mask):
    """a router picks one adapter a row; the shared projection and the adapters; dropout into the residual stream; the balance loss beside"""
    logits = x @ wr.t()
    ids = logits.detach().argmax(dim=1)
    y = ad.lowrank_adapt(x, a, b, ids, None, x @ w.t(), p=p_in, seed=seed, offset=1)
    out = ad.dropout(y, p_out, seed, 2, residual=x)
    loss, counts = ad.router_balance(logits, ids, mask)
    return out, loss, counts, ids


def test_a_routed_layer_as_it_is_used(ad):
    gen = torch.Generator().manual_seed(8)
    rows, k, r, g = 600, 64, 8, 5
    x, w, a, b, wr, dy = [t.cuda() for t in (torch.randn(rows, k, generator=gen), torch.randn(k, k, generator=gen) / 8, torch.randn(g, r, k, generator=gen) / 8,
                                             torch.randn(g, k, r, generator=gen) / 3, torch.randn(g, k, generator=gen) / 8, torch.randn(rows, k, generator=gen))]
    mask = torch.rand(rows, generator=gen).cuda() > 0.1
    leaves = [t.requires_grad_(True) for t in (x, w, a, b, wr)]
    out, loss, counts, ids = routed_step(ad, 0.1, 0.2, 77, x, w, a, b, wr, mask)
    got = torch.autograd.grad((out * dy).sum() + 3.0 * loss, leaves)
    # the same in 64 bits by torch's own differentiation
    x2, w2, a2, b2, wr2 = [t.detach().cpu().double().requires_grad_(True) for t in leaves]
    i2, m2 = ids.cpu(), mask.cpu()
    f1, f2 = ref.keep_factor(rows, k, 0.1, 77, 1), ref.keep_factor(rows, k, 0.2, 77, 2)
    h = ((x2 * f1)[:, None, :] * a2[i2]).sum(-1)
    y2 = x2 @ w2.T + (h[:, None, :] * b2[i2]).sum(-1)
    prob = torch.softmax(x2 @ wr2.T, dim=1)
    share = torch.bincount(i2[m2], minlength=g).double() / m2.sum()
    loss2 = g * (share * prob[m2].mean(dim=0)).sum()
    out2 = y2 * f2 + x2
    want = torch.autograd.grad((out2 * dy.cpu().double()).sum() + 3.0 * loss2, (x2, w2, a2, b2, wr2))
    assert torch.equal(counts.cpu(), torch.bincount(i2[m2], minlength=g))
    close = lambda u, v: float((u.detach().cpu().double() - v.detach()).norm() / v.detach().norm()) < 3e-6  # noqa: E731      fp32 sums of 64 to 600 terms: (600)^0.5 2^-24
    assert close(out, out2) and close(loss, loss2) and all(close(u, v) for u, v in zip(got, want))


def test_shared_decoder_with_adapters(ad):
    """sdf.TCNNNetwork takes the adapters: the shared network's own output where there is none, gradients for both"""
    import gs_sdf_amd.sdf as sdf
    net = sdf.TCNNNetwork(32, 2, dict(otype="FullyFusedMLP", activation="ReLU", output_activation="None", n_neurons=64, n_hidden_layers=4), device="cuda", bias=True, seed=2)
    bank = ad.LowRankAdapters(4, 32, 2, 8, alpha=16, p=0.1, seed=3)
    x = torch.randn(3000, 32, device="cuda").requires_grad_(True)
    ids = torch.randint(-1, 4, (3000,), device="cuda", dtype=torch.int32)
    plain = net(x)
    assert torch.equal(net(x, bank, ids), plain)      # a new bank changes nothing
    with torch.no_grad():
        bank.b_.normal_()
    assert bank.calls_ == 1
    out = net(x, bank, ids)
    assert bank.calls_ == 2 and torch.equal(out[ids < 0], plain[ids < 0])
    dy = torch.randn_like(out)
    want = ref.Lowrank(x, bank.a_, bank.b_, ids, bank.scales, plain, dy, 0.1, 3, 1)
    want.check("y", out, 48)
    dx, da, db, dw = torch.autograd.grad(out, (x, bank.a_, bank.b_, net.params_), dy)
    want.check("da", da, 3100)
    want.check("db", db, 3100)
    dx0, dw0 = torch.autograd.grad(net(x), (x, net.params_), dy)
    assert torch.allclose(dw, dw0, rtol=1e-5, atol=1e-5 * float(dw0.abs().max()))
    assert float(((dx - dx0).cpu().double() - want.dx).norm() / want.dx.norm()) < 1e-5
    with torch.no_grad():      # serving: no dropout, no count
        ref.Lowrank(x, bank.a_, bank.b_, ids, bank.scales, plain).check("y", net(x, bank, ids), 48)
        assert bank.calls_ == 2
    with pytest.raises(RuntimeError, match="go together"):
        net(x, bank)


def test_other_streams(ad):
    """two streams at once: each call's workspace is its own"""
    cases = [make(800, 128, 96, 16, 5, torch.bfloat16, seed=s) for s in range(2)]
    want = []
    for x, a, b, ids, scales, base, dy in cases:
        xs = x.clone().requires_grad_(True)
        y = ad.lowrank_adapt(xs, a, b, ids, scales, base, p=0.1, seed=1)
        want.append((y.detach(), torch.autograd.grad(y, xs, dy)[0], ad.router_balance(base.detach(), ids)[0]))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(10):
        for i, (x, a, b, ids, scales, base, dy) in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                xs = x.clone().requires_grad_(True)
                y = ad.lowrank_adapt(xs, a, b, ids, scales, base, p=0.1, seed=1)
                got[i].append((y.detach(), torch.autograd.grad(y, xs, dy)[0], ad.router_balance(base.detach(), ids)[0]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(u, v) for one in got[i] for u, v in zip(one, want[i]))


def test_captured_graph_replays(ad):
    """forward and backward of a routed layer in one graph: new inputs, new ids and a new mask (its counter is a device word) with every replay"""
    dev = "cuda"
    rows, k, g = 500, 64, 4
    x, a, b, _, scales, base, dy = make(rows, k, 48, 8, g, torch.float32)
    ids = torch.randint(0, g, (rows,), device=dev, dtype=torch.int32)
    word = torch.zeros(1, dtype=torch.int64, device=dev)
    x, a, b = [t.detach().requires_grad_(True) for t in (x, a, b)]
    logits = torch.randn(rows, g, device=dev, requires_grad=True)

    def step():
        y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=0.2, seed=5, offset=word)
        out = ad.dropout(y, 0.3, 6, word)
        loss, counts = ad.router_balance(logits, ids)
        grads = torch.autograd.grad((out, loss), (x, a, b, logits), (dy, torch.ones_like(loss)))
        return [out.detach(), loss.detach(), counts] + list(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    masks = []
    for i in range(4):
        with torch.no_grad():
            x.copy_(torch.randn(rows, k, device=dev))
            ids.copy_(torch.randint(-1, g, (rows,), device=dev, dtype=torch.int32))
            word.fill_(i)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        want = step()
        assert all(torch.equal(u, v) for u, v in zip(got, want))
        masks.append(got[0] == 0)
    assert not torch.equal(masks[0], masks[1])


def test_refusals(ad):
    x, a, b, ids, scales, base, dy = make(8, 16, 12, 4, 2, torch.float32)
    for bad in (lambda: ad.lowrank_adapt(x.double(), a, b, ids), lambda: ad.lowrank_adapt(x, a.half(), b, ids), lambda: ad.lowrank_adapt(x, a[:, :, :8], b, ids),
                lambda: ad.lowrank_adapt(x, a, b[:1], ids), lambda: ad.lowrank_adapt(x, a, b, ids[:4]), lambda: ad.lowrank_adapt(x, a, b, ids.float()),
                lambda: ad.lowrank_adapt(x, a, b, ids.cpu()), lambda: ad.lowrank_adapt(x, a, b, ids, scales.half()), lambda: ad.lowrank_adapt(x, a, b, ids, scales[:1]),
                lambda: ad.lowrank_adapt(x, a, b, ids, scales.clone().requires_grad_(True)), lambda: ad.lowrank_adapt(x, a, b, ids, scales, base[:, :4]),
                lambda: ad.lowrank_adapt(x, a, b, ids, scales, base[0]), lambda: ad.lowrank_adapt(x, a, b, ids, p=2.0), lambda: ad.lowrank_adapt(x, a, b, ids, seed=-1),
                lambda: ad.lowrank_adapt(x, a, b, ids, offset=-1), lambda: ad.lowrank_adapt(x, a, b, ids, offset=torch.zeros(1, device="cuda")),
                lambda: ad.lowrank_adapt(x, torch.zeros(2, 129, 16, device="cuda"), torch.zeros(2, 12, 129, device="cuda"), ids),
                lambda: ad.lowrank_adapt_(base, x.clone().requires_grad_(True), a, b, ids), lambda: ad.lowrank_adapt_(base[:1].expand(8, 12), x, a, b, ids),
                lambda: ad.lowrank_adapt_(base.t().contiguous().t(), x, a, b, ids),
                lambda: ad.dropout(x.long(), 0.5, 1), lambda: ad.dropout(x, -0.5, 1), lambda: ad.dropout(x, 0.5, 2 ** 64), lambda: ad.dropout(x, 0.5, 1, residual=base),
                lambda: ad.router_balance(x.long(), ids), lambda: ad.router_balance(x, ids[:3]), lambda: ad.router_balance(x, ids, ids), lambda: ad.router_balance(
                    x, torch.zeros(8, 17, dtype=torch.int32, device="cuda")), lambda: ad.router_balance(torch.zeros(2, 1025, device="cuda"), ids[:2])):
        with pytest.raises(RuntimeError):
            bad()
    leaf = x.clone().requires_grad_(True)
    y = ad.dropout(leaf, 0.5, 1)
    with pytest.raises(RuntimeError):      # once differentiable
        torch.autograd.grad((y * y).sum(), leaf, create_graph=True)[0].sum().backward()
