"""The adapter operators without a GPU: the mask's generator, refusals of the C ABI and of the Python entry points (nothing is launched)."""
import ctypes as C

import numpy as np
import pytest
import torch

import adapters_ref as ref


def test_reference_generator_gives_the_published_answers():
    """known answers published with the generator (ctr, key -> block)"""
    full = 0xFFFFFFFF
    for ctr, key, want in (([0] * 4, (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
                           ([full] * 4, (full, full), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
                           ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0), (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = ref.philox([np.array([c], dtype=np.uint64) for c in ctr], key)
        assert tuple(int(v[0]) for v in got) == want


def test_reference_mask_has_the_share_it_says():
    f = ref.keep_factor(400, 1001, 0.3, 77, 5)
    q = ref.threshold(0.3) / 65536
    share = float((f == 0).double().mean())
    assert abs(share - q) < 5 * (q * (1 - q) / f.numel()) ** 0.5
    assert torch.equal(ref.keep_factor(3, 5, 0.0, 1, 1), torch.ones(3, 5).double())


@pytest.fixture(scope="module")
def capi():
    import gs_sdf_amd.capi as capi
    capi.lib()
    return capi


def _args(capi, **kw):
    d = dict(rows=4, x_stride=8, n_in=8, n_out=8, rank=4, n_adapters=2, dtype=0, ids_64=0, x=64, a=64, b=64, ids=64, scales=None, p=0.0, seed=0, offset=0,
             offset_dev=None)
    d.update(kw)
    return capi.LowrankArgs(*[d[n] for n, _ in capi.LowrankArgs._fields_])


@pytest.mark.parametrize("bad,said", [(dict(rank=0), "rank 0"), (dict(rank=129), "rank 129"), (dict(n_adapters=0), "0 adapters"),
                                      (dict(n_adapters=1025), "1025 adapters"), (dict(dtype=3), "element type 3"), (dict(p=1.5), "p = 1.5"),
                                      (dict(p=float("nan")), "p = "), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(n_in=0), "widths"),
                                      (dict(x=None), "required"), (dict(ids=None), "required"), (dict(a=None), "required"), (dict(b=None), "required")])
def test_lowrank_refuses(capi, bad, said):
    args = _args(capi, **bad)
    L = capi.lib()
    assert L.gsdf_lowrank_fwd(C.byref(args), None, 0, 64, 8, None, 64, None) == -1
    assert said in L.gsdf_last_error().decode()
    assert L.gsdf_lowrank_bwd(C.byref(args), 64, 8, 64, 64, 8, 64, 64, 64, None) == -1
    assert said in L.gsdf_last_error().decode()


def test_lowrank_refuses_weights_behind_a_launch(capi):
    L = capi.lib()
    for bad in (dict(n_adapters=1024, n_in=1 << 21, rank=1, x_stride=1 << 21), dict(n_adapters=1024, n_out=1 << 21, rank=4), dict(n_adapters=700, n_in=1 << 14, n_out=1 << 14, rank=65)):
        args = _args(capi, **bad)
        assert L.gsdf_lowrank_fwd(C.byref(args), None, 0, 64, 1 << 21, None, 64, None) == -1
        assert "weights" in L.gsdf_last_error().decode()
        assert L.gsdf_lowrank_fwd_ws_bytes(C.byref(args)) == 0 and L.gsdf_lowrank_save_bytes(C.byref(args)) == 0 and L.gsdf_lowrank_bwd_ws_bytes(C.byref(args)) == 0
    for good in (dict(n_adapters=600, n_in=1 << 14, n_out=1 << 14, rank=65), dict(n_adapters=1024, n_in=4096, n_out=4096, rank=64)):      # 3.8e9 and 0.8e9 elements
        assert L.gsdf_lowrank_fwd_ws_bytes(C.byref(_args(capi, **good))) > 0


def test_lowrank_refuses_missing_buffers(capi):
    L, args = capi.lib(), _args(capi)
    assert L.gsdf_lowrank_fwd(None, None, 0, 64, 8, None, 64, None) == -1
    assert L.gsdf_lowrank_fwd(C.byref(args), None, 0, None, 8, None, 64, None) == -1
    assert L.gsdf_lowrank_fwd(C.byref(args), None, 0, 64, 8, None, None, None) == -1
    assert L.gsdf_lowrank_fwd(C.byref(args), None, 0, 64, 7, None, 64, None) == -1      # rows of y that overlap
    assert L.gsdf_lowrank_bwd(C.byref(args), 64, 8, None, 64, 8, 64, 64, 64, None) == -1
    assert L.gsdf_lowrank_bwd(C.byref(args), None, 8, 64, 64, 8, 64, 64, 64, None) == -1
    assert L.gsdf_lowrank_bwd(C.byref(args), 64, 8, 64, 64, 7, 64, 64, 64, None) == -1


def test_dropout_refuses(capi):
    L = capi.lib()
    call = lambda rows=4, cols=8, dtype=0, x=64, xs=8, p=0.5, y=64, ys=8: L.gsdf_dropout(rows, cols, dtype, x, xs, None, 0, p, 0, 0, None, y, ys, None)  # noqa: E731
    for bad in (dict(rows=-1), dict(rows=1 << 32), dict(cols=1 << 33), dict(cols=-1), dict(dtype=7), dict(p=-0.1), dict(p=1.01), dict(p=float("nan")), dict(x=None),
                dict(y=None), dict(ys=7), dict(xs=-1)):
        assert call(**bad) == -1, bad
    assert call(rows=0) == 0 and call(cols=0) == 0      # nothing to do, nothing launched


def test_balance_refuses(capi):
    L = capi.lib()
    f = lambda rows=4, e=8, k=1, dtype=0, logits=64, s=8, ids=64, loss=64, ws=64: L.gsdf_router_balance_fwd(  # noqa: E731
        rows, e, k, dtype, logits, s, ids, 0, None, loss, 64, 64, ws, None)
    for bad in (dict(rows=-1), dict(rows=1 << 31), dict(e=0), dict(e=1025), dict(k=0), dict(k=9), dict(dtype=-1), dict(logits=None), dict(ids=None), dict(loss=None),
                dict(ws=None), dict(s=-1)):
        assert f(**bad) == -1, bad
    b = lambda rows=4, e=8, dtype=0, logits=64, s=8, pull=64, v=64: L.gsdf_router_balance_bwd(rows, e, dtype, logits, s, None, pull, 64, v, None)  # noqa: E731
    for bad in (dict(rows=-1), dict(e=0), dict(e=1025), dict(dtype=9), dict(logits=None), dict(pull=None), dict(v=None), dict(s=-1)):
        assert b(**bad) == -1, bad
    assert b(rows=0) == 0


def test_python_entries_refuse_host_tensors():
    from gs_sdf_amd import adapters
    x, a, b, ids = torch.zeros(4, 8), torch.zeros(2, 3, 8), torch.zeros(2, 5, 3), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adapters.lowrank_adapt(x, a, b, ids)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adapters.lowrank_adapt_(torch.zeros(4, 5), x, a, b, ids)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adapters.dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        adapters.router_balance(x, ids)
    with pytest.raises(RuntimeError, match="out of range"):
        adapters.LowRankAdapters(2, 8, 5, 129, device="cpu")
    with pytest.raises(RuntimeError, match="probability"):
        adapters.LowRankAdapters(2, 8, 5, 4, p=1.5, device="cpu")


def test_lowrank_refuses_weight_gradients_behind_a_launch(capi):
    """rows that are one row again and again make more workgroups of 512 threads than a launch holds (2^32 threads) out of little memory"""
    L = capi.lib()
    for bad in (dict(rows=(1 << 28) - 1, n_in=1 << 21, x_stride=0, n_out=8, rank=1, n_adapters=1), dict(rows=1 << 26, n_in=8, n_out=1 << 21, rank=4, n_adapters=1, dtype=2)):
        args = _args(capi, **bad)
        assert L.gsdf_lowrank_bwd(C.byref(args), 64, 0, 64, None, 0, 64, 64, 64, None) == -1
        assert "a launch" in L.gsdf_last_error().decode()
