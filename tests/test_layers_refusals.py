"""What layer norm, embedding and the orthogonalized updates refuse, before anything is launched (no GPU needed)."""
import ctypes
import os

import pytest
import torch

OK, OFF = 0x10000, 0x10001
NAN = float("nan")


@pytest.fixture(scope="module")
def lib():
    from rwkv_kernel import _native

    if not os.path.exists(_native.LIB_PATH):
        import __graft_entry__

        __graft_entry__.build()
    return _native.load()


def _norm(lib, **change):
    a = dict(dtype=2, branch=0, params=2, rows=10, C=64, x=OK, xs=64, add=OK, adds=64, w=OK, b=OK, eps=1e-5, total=OK, y=OK, stats=OK)
    a.update(change)
    return lib.wkv6_layer_norm(None, a["dtype"], a["branch"], a["params"], a["rows"], a["C"], a["x"], a["xs"], a["add"], a["adds"], a["w"], a["b"], a["eps"], a["total"], a["y"], a["stats"])


def _norm_backward(lib, **change):
    a = dict(dtype=2, branch=0, params=2, rows=10, C=64, total=OK, ts=64, stats=OK, w=OK, gy=OK, gt=OK, gx=OK, ga=OK, gw=OK, gb=OK, ws=OK, n=1 << 30)
    a.update(change)
    return lib.wkv6_layer_norm_backward(None, a["dtype"], a["branch"], a["params"], a["rows"], a["C"], a["total"], a["ts"], a["stats"], a["w"], a["gy"], a["gt"], a["gx"], a["ga"],
                                        a["gw"], a["gb"], a["ws"], a["n"])


def test_layer_norm(lib):
    for bad in (dict(dtype=3), dict(dtype=0, branch=2), dict(dtype=0, branch=1), dict(branch=5), dict(params=-1), dict(rows=0), dict(rows=-1), dict(C=0)):
        assert _norm(lib, **bad) == 1 and _norm_backward(lib, **bad) == 1, bad
    for bad in (dict(x=None), dict(y=None), dict(add=None), dict(total=None), dict(xs=-1), dict(adds=-1), dict(eps=-1.0), dict(eps=NAN), dict(x=OK + 2), dict(add=OFF), dict(y=OFF), dict(total=OK + 2),
                dict(w=OK + 2), dict(b=OFF), dict(stats=OK + 4)):
        assert _norm(lib, **bad) == 1, bad
    for bad in (dict(total=None), dict(stats=None), dict(gy=None), dict(ts=-1), dict(total=OK + 2), dict(gt=OFF), dict(gx=OK + 2), dict(gy=OFF), dict(ga=OFF), dict(w=OFF), dict(gw=OK + 2),
                dict(gb=OFF), dict(stats=OK + 4)):
        assert _norm_backward(lib, **bad) == 1, bad
    for bad in (dict(C=32769), dict(rows=1 << 62)):
        assert _norm(lib, **bad) == 2 and _norm_backward(lib, **bad) == 2, bad
    need = lib.wkv6_layer_norm_backward_workspace_bytes(10, 64)
    assert need > 0 and lib.wkv6_layer_norm_backward_workspace_bytes(0, 64) == 0 and lib.wkv6_layer_norm_backward_workspace_bytes(10, 32769) == 0
    for bad in (dict(ws=None), dict(ws=OK + 8), dict(n=need - 1)):
        assert _norm_backward(lib, **bad) == 3 and _norm_backward(lib, gw=None, **bad) == 3, bad


def test_embedding(lib):
    def forward(dtype=2, out=0, N=10, V=50, C=64, ids=OK, w=OK, stride=64, scale=1.0, o=OK):
        return lib.wkv6_embedding(None, dtype, out, N, V, C, ids, w, stride, scale, o)

    def backward(dtype=2, out=0, N=10, V=50, C=64, ids=OK, w=OK, scale=1.0, o=OK, ws=OK, n=1 << 40):
        return lib.wkv6_embedding_backward(None, dtype, out, N, V, C, ids, o, scale, -1, w, ws, n)

    for bad in (dict(dtype=3), dict(dtype=0, out=2), dict(dtype=1, out=0), dict(out=7), dict(N=0), dict(V=0), dict(C=0), dict(N=-1), dict(ids=None), dict(w=None), dict(o=None), dict(ids=OK + 4),
                dict(w=OK + 2), dict(o=OFF)):
        assert forward(**bad) == 1 and backward(**bad) == 1, bad
    assert forward(stride=-1) == 1
    for bad in (dict(N=1 << 31), dict(V=1 << 31), dict(C=(1 << 24) + 1), dict(V=1 << 30, C=1 << 20)):
        assert forward(**bad) == 2 and backward(**bad) == 2, bad
    need = lib.wkv6_embedding_backward_workspace_bytes(10, 50, 64)
    assert need > 0 and lib.wkv6_embedding_backward_workspace_bytes(0, 50, 64) == 0 and lib.wkv6_embedding_backward_workspace_bytes(10, 1 << 31, 64) == 0
    for bad in (dict(ws=None), dict(ws=OK + 8), dict(n=need - 1)):
        assert backward(**bad) == 3, bad


def _matrices(*rows):
    from rwkv_kernel import _native

    out = (_native.MuonMatrix * max(1, len(rows)))()
    for m, r in zip(out, rows):
        for k, v in dict(dict(grad=OK, momentum=OK, out=OK, master=None, rows=8, columns=16, rate=1.0), **r).items():
            setattr(m, k, v)
    return out


def test_orthogonalized_updates(lib):
    three = (ctypes.c_double * 15)(*([3.0, -4.0, 2.0] * 5))
    big = 1 << 40

    def step(rows=None, dtype=2, count=1, steps=5, coefficients=three, eps=1e-7, mu=0.9, lr=0.1, lr_device=None, wd=0.0, ws=OK, n=big):
        return lib.wkv6_muon_step(None, dtype, count, _matrices(rows or {}), steps, coefficients, eps, mu, 1, lr, lr_device, wd, ws, n)

    def orth(rows=None, dtype=2, count=1, steps=5, coefficients=three, eps=1e-7, ws=OK, n=big):
        return lib.wkv6_orthogonalize(None, dtype, count, _matrices(dict(dict(momentum=None), **(rows or {}))), steps, coefficients, eps, ws, n)

    for bad in (dict(dtype=3), dict(count=0), dict(count=-1), dict(steps=0), dict(steps=101), dict(coefficients=None), dict(eps=-1.0), dict(eps=NAN), dict(rows=dict(rows=-1)),
                dict(rows=dict(columns=-2)), dict(rows=dict(grad=None)), dict(rows=dict(out=None)), dict(rows=dict(grad=OK + 2)), dict(rows=dict(out=OFF)), dict(rows=dict(master=OK + 2))):
        assert step(**bad) == 1 and orth(**bad) == 1, bad
    for bad in (dict(mu=1.0), dict(mu=-0.1), dict(mu=NAN), dict(lr=-1.0), dict(lr=NAN), dict(wd=-0.1), dict(lr_device=OK + 2), dict(rows=dict(momentum=None)), dict(rows=dict(momentum=OK + 2)),
                dict(rows=dict(rate=-1.0)), dict(rows=dict(rate=NAN))):
        assert step(**bad) == 1, bad
    for bad in (dict(momentum=OK), dict(master=OK)):
        assert orth(rows=bad) == 1, bad
    for bad in (dict(rows=1 << 26, columns=1), dict(rows=1 << 15, columns=1 << 15), dict(rows=40000, columns=40000)):
        assert step(rows=bad) == 2 and orth(rows=bad) == 2, bad
    need = lib.wkv6_muon_workspace_bytes(1, _matrices({}))
    assert need > 0 and lib.wkv6_muon_workspace_bytes(0, _matrices({})) == 0 and lib.wkv6_muon_workspace_bytes(1, None) == 0
    for bad in (dict(ws=None), dict(ws=OK + 16), dict(n=need - 1)):
        assert step(**bad) == 3 and orth(**bad) == 3, bad
    # nothing to do: nothing is asked for
    assert step(rows=dict(rows=0, grad=None, out=None, momentum=None), ws=None, n=0) == 0
    # the workspace of many is bounded, and holds the largest
    many = _matrices(*[dict(rows=4096, columns=4096)] * 40)
    one = lib.wkv6_muon_workspace_bytes(1, many)
    assert one <= lib.wkv6_muon_workspace_bytes(40, many) < 40 * one


def test_tensors_that_are_not_on_the_gpu():
    import rwkv_kernel

    x, ids = torch.zeros(2, 8), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: rwkv_kernel.layer_norm(x), lambda: rwkv_kernel.embedding(ids, x)):
        with pytest.raises(AssertionError, match="GPU"):
            call()
    for call in (lambda: rwkv_kernel.orthogonalize(x), lambda: rwkv_kernel.muon_step([x], [x], [x], 0.1)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()
