"""The adapter operators (gs_sdf_amd.adapters) at their edges, on the GPU: inner values that need all 32 bits, ranks of very different sizes, what a call has to
refuse before it writes, derivatives of other kinds than one backward pass."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import adapters_ref as ref
from test_gpu_adapters import make

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = [str(d).split(".")[1] for d in DTYPES]


@pytest.fixture(scope="module")
def ad():
    from gs_sdf_amd import adapters
    return adapters


def whole_numbers(dtype, rows, width, gen, *lead):
    """[*lead, rows, width] whole numbers of the type whose products, summed over `width`, need 24 bits and fit them: every 32-bit sum of them is exact"""
    lo, hi = (128, 255) if dtype == torch.bfloat16 else (1200, 1448)
    return torch.randint(lo, hi + 1, (*lead, rows, width), generator=gen).double()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["float16", "bfloat16"])
@pytest.mark.parametrize("rows,r", [(40, 8), (300, 2), (300, 16), (300, 24), (700, 64), (900, 128), (65600, 4), (65600, 16), (65600, 32)])
def test_lowrank_inner_values_keep_32_bits(ad, rows, r, dtype):
    """h (dh) of 24 bits whose last digits alone are left: neighbouring ranks differ by x[., 0] (dy[., 0]) and are taken from one another, and so are neighbouring
    rows in the weights' gradients.  All sums are whole numbers below 2^24 and the results fit the type: they are equal, not close."""
    gen = torch.Generator().manual_seed(rows + r)
    wide, n, g = 256 if dtype == torch.bfloat16 else 8, 72, 3
    ids = torch.randint(-1, g, (rows // 2,), generator=gen).repeat_interleave(2)      # pairs of rows share an adapter
    rich = whole_numbers(dtype, rows, wide, gen)
    rich[1::2] = rich[0::2]
    rich[1::2, 0] -= 1
    weights = whole_numbers(dtype, r, wide, gen, g)
    weights[:, 1::2] = weights[:, 0::2]
    weights[:, 1::2, 0] -= 1
    rich[:, 0], weights[:, :, 0] = rich[:, 0].clamp(min=130 if wide == 256 else 1202), weights[:, :, 0].clamp(max=254 if wide == 256 else 1447)
    rich[1::2, 0] = rich[0::2, 0] - 1
    weights[:, 1::2, 0] = weights[:, 0::2, 0] - 1
    pick = torch.zeros(g, n, r, dtype=torch.float64)      # column i takes the two ranks of pair i mod r / 2 from one another
    for i in range(n):
        pick[:, i, 2 * (i % (r // 2))], pick[:, i, 2 * (i % (r // 2)) + 1] = 1, -1
    pairs = torch.zeros(rows, n, dtype=torch.float64)     # column i takes the two rows of pair i from one another
    for i in range(min(n, rows // 2)):
        pairs[2 * i, i], pairs[2 * i + 1, i] = 1, -1
    on = (ids >= 0).double()[:, None]
    first = torch.zeros(g, n, dtype=torch.float64)        # the adapter of pair i
    for i in range(min(n, rows // 2)):
        if ids[2 * i] >= 0:
            first[ids[2 * i], i] = 1
    d = lambda t: t.to(dtype).cuda().requires_grad_(True)  # noqa: E731
    assert float((rich[:64] @ weights[0].T).max()) < 2 ** 24 and float((rich[:64] @ weights[0].T).max()) > 2 ** 23
    x, a, b, dy, ids = d(rich), d(weights), d(pick), d(pairs), ids.to(torch.int32).cuda()
    y = ad.lowrank_adapt(x, a, b, ids)
    assert torch.equal(y.detach().cpu().double(), (rich[:, :1] * on).expand(rows, n))
    db, = torch.autograd.grad(y, b, dy)      # h of row 2 i less h of row 2 i + 1: a[., 0]
    assert torch.equal(db.cpu().double(), first[:, :, None] * weights[:, None, :, 0])
    x, a, b, dy = d(pairs), d(pick.transpose(1, 2)), d(weights.transpose(1, 2)), d(rich)
    y = ad.lowrank_adapt(x, a, b, ids)
    dx, da = torch.autograd.grad(y, (x, a), dy)
    assert torch.equal(dx.cpu().double(), (rich[:, :1] * on).expand(rows, n))
    assert torch.equal(da.cpu().double(), first[:, None, :] * weights[:, :, :1])


def check_alone(want, name, got, terms, rank_dim=None, ranks=None):
    """as Lowrank.check, but nothing is allowed for values that do not take part in an element's own sum: what is left of the split of h is 2^-38 of the largest h"""
    w, mag, split = getattr(want, name), getattr(want, name + "_mag"), getattr(want, name + "_split")
    if rank_dim is not None:
        at = torch.tensor(ranks)
        got, w, mag, split = got.index_select(rank_dim, at.to(got.device)), w.index_select(rank_dim, at), mag.index_select(rank_dim, at), 0.0
    ref.within(got, w, ref.HALF[got.dtype] * w.abs() + (1 + ref.HALF[got.dtype]) * ((3 * terms + 16) * 2.0 ** -24 * mag + 2.0 ** -38 * split), name, got.dtype)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,r", [(300, 12), (300, 24), (700, 64), (900, 100), (65600, 16)])
def test_lowrank_small_ranks_beside_large_ones(ad, rows, r, dtype):
    """a rank whose h and dh are 1e-5 of the others' keeps its own digits in the weights' gradients"""
    x, a, b, ids, scales, base, dy = make(rows, 64, 72, r, 3, dtype, 0.1)
    small = [1, r - 3]
    with torch.no_grad():
        a[:, small] *= 2e-5
        b[:, :, small] *= 2e-5
        if dtype != torch.float32:
            x *= 4.0
            dy *= 4.0
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    dx, da, db = torch.autograd.grad(ad.lowrank_adapt(x, a, b, ids, scales, base), leaves, dy)
    check_alone(want, "da", da, 72 + rows, 1, small)
    check_alone(want, "db", db, 64 + rows, 2, small)
    check_alone(want, "dx", dx, 72 + r)


@pytest.mark.parametrize("rows,r", [(300, 12), (300, 24), (700, 64), (65600, 16)])
def test_lowrank_small_ranks_in_a_row_of_large_ones(ad, rows, r):
    """fp16: y from a rank whose h is 3e-7 of another's, which has no part in y"""
    x, a, b, ids, scales, base, _ = make(rows, 64, 72, r, 3, torch.float16, 0.1)
    a[:, 0] *= 1e4
    b[:, :, 0] = 0
    a[:, 1:] *= 2e-3
    check_alone(ref.Lowrank(x, a, b, ids, scales), "y", ad.lowrank_adapt(x.requires_grad_(True), a, b, ids, scales), 64 + r)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,r", [(300, 12), (300, 24), (700, 64), (900, 100), (65600, 16)])
def test_lowrank_an_infinity_in_one_rank_stays_there(ad, rows, r, dtype):
    """an infinite weight of one rank: the gradients of the others are what they are without that rank, above the largest fp16 number too"""
    x, a, b, ids, scales, base, dy = make(rows, 64, 72, r, 3, dtype, 0.1)
    few = 2e-3 if rows < 1000 else 2e-4      # (sums of all rows that fit the type)
    x, dy, b = x * few, dy * 400, b * 60
    keep = [i for i in range(r) if i != 2]
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    b[1, 5, 2] = math.inf
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    da, = torch.autograd.grad(ad.lowrank_adapt(x, a, b, ids, scales, base), leaves[1:2], dy)
    assert not torch.isfinite(da[1, 2].float()).any()
    check_alone(want, "da", da, 72 + rows, 1, keep)
    x, a, b, ids, scales, base, dy = make(rows, 64, 72, r, 3, dtype, 0.1)
    x, a, dy = x * 400, a * 200, dy * few
    want = ref.Lowrank(x, a, b, ids, scales, base, dy)
    a[1, 2, 7] = -math.inf
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    db, = torch.autograd.grad(ad.lowrank_adapt(x, a, b, ids, scales, base), leaves[2:], dy)
    assert not torch.isfinite(db[1, :, 2].float()).any()
    check_alone(want, "db", db, 64 + rows, 2, keep)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows", [65, 1170, 1200, 1300, 1320, 2119])
@pytest.mark.parametrize("used", [1, 530])
def test_lowrank_few_adapters_of_a_large_bank(ad, rows, used, dtype):
    """on both sides of the border between the path of few rows and the plan, which goes by the bytes of weights that either reads"""
    x, a, b, ids, scales, base, _ = make(rows, 64, 1000, 64, 530, dtype, 0.1)
    ids = torch.where(ids < 0, ids, ids % used + (530 - used))
    want = ref.Lowrank(x, a[530 - used:], b[530 - used:], torch.where(ids < 0, ids, ids - (530 - used)), scales[530 - used:], base)
    got = ad.lowrank_adapt(x, a, b, ids, scales, base)
    want.check("y", got, 64 + 64)
    assert torch.equal(got[ids < 0], base[ids < 0])


def test_forward_mode_is_refused(ad):
    """a dual tensor does not ask for a gradient, and its tangent would be lost without an error"""
    x, a, b, ids, scales, base, _ = make(30, 16, 12, 4, 2, torch.float32)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for grad in (True, False):
            with torch.set_grad_enabled(grad):
                for call in (lambda: ad.lowrank_adapt(dual(x), a, b, ids, scales, base), lambda: ad.lowrank_adapt(x, dual(a), b, ids, scales, base),
                             lambda: ad.lowrank_adapt(x, a, dual(b), ids, scales, base), lambda: ad.lowrank_adapt(x, a, b, ids, dual(scales), base),
                             lambda: ad.lowrank_adapt(x, a, b, ids, scales, dual(base)), lambda: ad.lowrank_adapt_(dual(base.clone()), x, a, b, ids, scales),
                             lambda: ad.lowrank_adapt_(base.clone(), dual(x), a, b, ids, scales), lambda: ad.dropout(dual(x), 0.5, 1),
                             lambda: ad.dropout(x, 0.5, 1, residual=dual(x)), lambda: ad.router_balance(dual(x), ids)):
                    with pytest.raises(RuntimeError, match="forward-mode"):
                        call()
        leaf = x.clone().requires_grad_(True)
        for y in (ad.lowrank_adapt(leaf, a, b, ids, scales, base), ad.dropout(leaf, 0.5, 1), ad.router_balance(leaf, ids)[0]):
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, dual(y.detach()), retain_graph=True)
            torch.autograd.grad(y, leaf, y.detach())      # nobody is dual: as ever


class Cut(torch.autograd.Function):
    """hands its input on and no gradient back"""

    @staticmethod
    def forward(ctx, x):
        return x.clone()

    @staticmethod
    def backward(ctx, g):
        return None


def test_no_gradient_upstream_is_no_gradient(ad):
    x, a, b, ids, scales, base, _ = make(300, 16, 12, 4, 2, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, a, b, base)]
    for y, of in ((ad.lowrank_adapt(x, a, b, ids, scales, base), leaves), (ad.dropout(x, 0.5, 1), [x]), (ad.dropout(x, 0.5, 1, residual=x * 2), [x]),
                  (ad.router_balance(x, ids)[0], [x])):
        assert all(g is None for g in torch.autograd.grad(Cut.apply(y).sum(), of, allow_unused=True))


@pytest.mark.parametrize("strided", [False, True])
def test_second_derivatives_raise_and_are_not_taken_for_nothing(ad, strided):
    """by backward() and by grad(), which asks for some leaves alone: beside a term of its own a missing one would go unseen"""
    x, a, b, ids, scales, base, _ = make(300, 16, 12, 4, 2, torch.float32)
    x = x.t().contiguous().t() if strided else x
    leaf = lambda t: t.clone().requires_grad_(True)  # noqa: E731
    for call, leaves in ((lambda t, u, v: ad.lowrank_adapt(t, u, v, ids, scales, base), [leaf(x), leaf(a), leaf(b)]),
                         (lambda t, u, v: ad.lowrank_adapt(t.view(30, 10, 16), u, v, ids.view(30, 10), scales), [leaf(x).contiguous().detach().requires_grad_(True), leaf(a), leaf(b)]),
                         (lambda t: ad.dropout(t, 0.5, 1), [leaf(x)]), (lambda t: ad.router_balance(t, ids)[0], [leaf(x)])):
        for i in range(len(leaves)):      # the gradient of one factor
            first, = torch.autograd.grad((call(*leaves) ** 2).sum(), leaves[i], create_graph=True)
            with pytest.raises(RuntimeError, match="differentiable once"):
                first.sum().backward(retain_graph=True)
            for other in leaves:
                with pytest.raises(RuntimeError, match="differentiable once"):
                    torch.autograd.grad(first.sum() + (other ** 2).sum(), other, retain_graph=True)
    x, a, b = [t.detach() for t in (x, a, b)]
    t = leaf(x)
    first, = torch.autograd.grad(ad.lowrank_adapt(t, a, b, ids).sum(), t, create_graph=True)      # a constant: there is nothing to refuse
    assert torch.equal(torch.autograd.grad((t ** 2).sum() + first.sum(), t)[0], 2 * t)


def test_what_is_added_stays_differentiable(ad):
    """base and residual go into the sum as they are, and so do derivatives of every order"""
    x, a, b, ids, scales, _, _ = make(300, 16, 16, 4, 2, torch.float32)
    z = torch.randn(300, 16, device="cuda", requires_grad=True)
    for call in (lambda t: ad.lowrank_adapt(x, a, b, ids, scales, t), lambda t: ad.dropout(x, 0.5, 1, residual=t)):
        y = call(z ** 3)
        first, = torch.autograd.grad((y ** 2).sum(), z, create_graph=True)
        assert torch.allclose(first, 6 * y * z ** 2)
        assert torch.allclose(torch.autograd.grad(first.sum(), z)[0], 18 * z ** 4 + 12 * y * z, rtol=1e-4, atol=1e-4)


def test_lazily_negated_tensors(ad):
    x, a, b, ids, scales, base, dy = make(300, 16, 16, 4, 2, torch.float32)
    neg = torch._neg_view
    assert neg(x).is_neg()
    want = ad.lowrank_adapt(-x, a, -b, ids, -scales, -base)
    assert torch.equal(ad.lowrank_adapt(neg(x), a, neg(b), ids, neg(scales), neg(base)), want)
    assert torch.equal(ad.lowrank_adapt(x, neg(a), b, ids), ad.lowrank_adapt(x, -a, b, ids))
    assert torch.equal(ad.dropout(neg(x), 0.5, 1, residual=neg(dy)), ad.dropout(-x, 0.5, 1, residual=-dy))
    assert torch.equal(ad.router_balance(neg(x), ids)[0], ad.router_balance(-x, ids)[0])
    leaf = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(ad.lowrank_adapt(neg(leaf), a, b, ids), leaf, neg(dy))
    assert torch.equal(got, torch.autograd.grad(ad.lowrank_adapt(-leaf, a, b, ids), leaf, -dy)[0])
    out = base.clone()
    with pytest.raises(RuntimeError, match="negat"):
        ad.lowrank_adapt_(neg(out), x, a, b, ids)
    assert torch.equal(out, base)


@pytest.mark.parametrize("rows", [6, 300])
def test_lowrank_in_place_refuses_before_it_writes(ad, rows):
    x, a, b, ids, scales, base, _ = make(rows, 40, 24, 8, 3, torch.float32, 0.1)
    with torch.inference_mode():
        y = base.clone()
        ad.lowrank_adapt_(y, x, a, b, ids, scales)      # in inference mode: as torch's own operators in place
        y.copy_(base)
    with pytest.raises(RuntimeError, match="inference"):
        ad.lowrank_adapt_(y, x, a, b, ids, scales)
    assert torch.equal(y, base)
    big = torch.zeros(max(rows * 24, a.numel(), b.numel()) + 64, device="cuda")
    y = big[16:16 + rows * 24].view(rows, 24)
    for name, t in (("a", a), ("b", b), ("scales", scales)):
        inside = big[20:20 + t.numel()].view(t.shape)
        inside.copy_(t)
        held = big.clone()
        with pytest.raises(RuntimeError, match="share memory"):
            ad.lowrank_adapt_(y, x, inside if name == "a" else a, inside if name == "b" else b, ids, inside if name == "scales" else scales)
        assert torch.equal(big, held)
    inside = big.view(torch.int32)[20:20 + rows]
    inside.copy_(ids)
    with pytest.raises(RuntimeError, match="share memory"):
        ad.lowrank_adapt_(y, x, a, b, inside, scales)
    # weights between the rows of a strided y share nothing with it
    wide = torch.zeros(rows, 40, device="cuda")
    wide[0, 30:33] = scales
    wide[:, :24] = base
    assert torch.equal(ad.lowrank_adapt_(wide[:, :24], x, a, b, ids, wide[0, 30:33]), ad.lowrank_adapt(x, a, b, ids, scales, base))


def test_banks_made_without_a_seed_differ(ad):
    """two layers' banks drop different elements and begin with different weights; torch's own seed makes them again"""
    x = torch.ones(200, 64, device="cuda", requires_grad=True)
    ids = torch.zeros(200, dtype=torch.int32, device="cuda")

    def mask(bank):      # through weights that change nothing
        with torch.no_grad():
            bank.a_[0].copy_(torch.eye(64)), bank.b_[0].copy_(torch.eye(64))
        return bank(x, ids).detach() == 0
    torch.manual_seed(5)
    banks = [ad.LowRankAdapters(2, 64, 64, 64, p=0.5) for _ in range(2)]
    assert banks[0].seed != banks[1].seed and not torch.equal(banks[0].a_, banks[1].a_)
    torch.manual_seed(5)
    again = ad.LowRankAdapters(2, 64, 64, 64, p=0.5)
    assert again.seed == banks[0].seed and torch.equal(again.a_, banks[0].a_)
    assert not torch.equal(mask(banks[0]), mask(banks[1]))
    assert torch.equal(ad.LowRankAdapters(2, 64, 64, 64, seed=3).a_, ad.LowRankAdapters(2, 64, 64, 64, seed=3).a_)


def test_a_bank_that_answers_drops_nothing_even_with_gradients(ad):
    """a normal at inference is a gradient: eval() takes the dropout out and holds the counter"""
    bank = ad.LowRankAdapters(3, 32, 8, 4, p=0.5, seed=7)
    with torch.no_grad():
        bank.b_.normal_()
    x = torch.randn(100, 32, device="cuda", requires_grad=True)
    ids = torch.randint(0, 3, (100,), device="cuda", dtype=torch.int32)
    assert bank.training and bank.eval() is bank and not bank.training
    y = bank(x, ids)
    assert torch.equal(y, ad.lowrank_adapt(x, bank.a_, bank.b_, ids, bank.scales)) and bank.calls_ == 0
    assert bank.train() is bank and bank.training
    assert torch.equal(bank(x, ids), ad.lowrank_adapt(x, bank.a_, bank.b_, ids, bank.scales, p=0.5, seed=7, offset=0)) and bank.calls_ == 1
    bank.train(False)
    assert torch.equal(bank(x, ids), y) and bank.calls_ == 1


@pytest.mark.parametrize("p", [1.0, 65535 / 65536, 1 / 65536])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,k,n,r", [(5, 200, 96, 16), (60, 2048, 1024, 32), (900, 136, 72, 12), (66000, 64, 64, 8)])
def test_lowrank_masks_at_the_ends_of_p(ad, rows, k, n, r, dtype, p):
    """everything dropped, all but one element in 65536, that one alone: on the path of few rows, behind the plan, and through both products at once"""
    x, a, b, ids, scales, base, dy = make(rows, k, n, r, 4, dtype, 0.1)
    if 0.5 < p < 1:
        a = a / 256      # the factor of what stays is 65536
    want = ref.Lowrank(x, a, b, ids, scales, base, dy, p, 21, 22)
    want.check("y", ad.lowrank_adapt(x, a, b, ids, scales, base, p=p, seed=21, offset=22), k + r)
    leaves = [t.requires_grad_(True) for t in (x, a, b)]
    y = ad.lowrank_adapt(x, a, b, ids, scales, base, p=p, seed=21, offset=22)
    want.check("y", y, k + r)
    dx, da, db = torch.autograd.grad(y, leaves, dy)
    f = ref.keep_factor(rows, k, p, 21, 22)
    assert (dx.cpu()[f == 0] == 0).all()
    if p == 1.0:
        assert torch.equal(y, base) and (da == 0).all() and (db == 0).all()
    if dtype != torch.float16 or p < 0.5 or p == 1.0:      # (65536 times a gradient passes the largest fp16 number)
        want.check("dx", dx, n + r)
        want.check("da", da, n + rows)
        want.check("db", db, k + rows)


@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("rows,cols,p", [(257, 333, 0.3), (64, 64, 0.1), (1, 100003, 0.5), (300, 8, 65535 / 65536), (70, 1001, 1 / 65536)])
def test_dropout_mask_is_the_definition(ad, rows, cols, p, dtype):
    """of ones: 0 exactly where the definition drops, the rounded factor everywhere else"""
    f = ref.keep_factor(rows, cols, p, 3, 4)
    y = ad.dropout(torch.ones(rows, cols, dtype=dtype, device="cuda"), p, 3, 4)
    assert torch.equal(y.cpu() != 0, f != 0) and torch.equal(y.cpu(), f.float().to(dtype))
    res = torch.full((rows, cols), 0.5, dtype=dtype, device="cuda")
    assert torch.equal(ad.dropout(torch.ones_like(res), p, 3, 4, residual=res).cpu(), (f.float() + 0.5).to(dtype))


@pytest.mark.parametrize("rows,e,k,idle", [(70000, 5, 1, 0.0), (20000, 16, 2, 0.4), (16411, 128, 8, 0.1), (300007, 24, 1, 0.2)])
def test_balance_loss_counts_every_row(ad, rows, e, k, idle):
    """the longest chain of 32-bit sums is a row, the rows of a lane, the lanes of a wave and the waves of a workgroup: a loss of one valid row more or less is outside"""
    gen = torch.Generator().manual_seed(rows)
    logits = 2 * torch.randn(rows, e, generator=gen) + torch.randn(e, generator=gen)
    ids = logits.topk(k, dim=1).indices
    mask = torch.rand(rows, generator=gen) >= idle if idle else None
    want = ref.Balance(logits, ids, mask)
    lanes = 1
    while lanes * 8 < e and lanes < 64:
        lanes *= 2
    groups = min(256, -(-rows * lanes // 1024))
    of_a_lane = -(-(-(-rows // groups)) * lanes // 1024)
    spread = float((logits.max(dim=1).values - logits.min(dim=1).values).max())      # half a step of it in exp's argument
    # exp: 3 units; the sum of a row, its quotient and product; the rows of a lane; the lanes of a wave and the waves; the result
    bound = (spread / 2 + 3 + e + 2 + of_a_lane + 6 + 16 + 2) * 2.0 ** -23 * float(want.loss)
    assert bound < 0.9 * 2 / rows * float(want.loss) or rows > 100000 or e > 100
    loss, _ = ad.router_balance(logits.cuda(), ids.cuda(), None if mask is None else mask.cuda())
    assert abs(float(loss) - float(want.loss)) <= bound
