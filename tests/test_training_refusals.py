"""What the losses over logits and the optimizer refuse, before anything is launched (no GPU needed)."""
import ctypes
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
OK, OFF = 0x10000, 0x10001


@pytest.fixture(scope="module")
def native():
    from rwkv_kernel import _native

    if not os.path.exists(_native.LIB_PATH):
        import __graft_entry__

        __graft_entry__.build()
    return _native


ROWS = dict(dtype=0, B=2, T=3, V=50, logits=OK, stride_b=150, stride_t=50, ids=OK)
BAD_ROWS = [dict(dtype=3), dict(dtype=-1), dict(B=0), dict(T=0), dict(V=0), dict(B=-1), dict(logits=None), dict(ids=None), dict(logits=OFF),
            dict(ids=OK + 4), dict(stride_b=-1), dict(stride_t=-50), dict(dtype=2, logits=OK + 2)]
TOO_MANY = [dict(B=1 << 16, T=1 << 16), dict(B=1 << 32), dict(V=1 << 31)]


def _rows(**change):
    r = dict(ROWS, **change)
    return [None] + [r[k] for k in ("dtype", "B", "T", "V", "logits", "stride_b", "stride_t", "ids")] + [None]


def _calls(lib, rows, workspace=OK, bytes_=1 << 20, **kw):
    """Every entry on rows of logits, its arguments otherwise in order but for those named."""
    a = dict(temperature=1.0, logps=OK, stats=OK, coef=OK, grad=OK, loss=OK, means=OK, adv=OK, red=1, lo=0.2, hi=0.2, klw=0.1, beta=0.1, ls=0.0, kind=0, text=OK, up=OK, there=0)
    a.update(kw)
    ws = (workspace, bytes_)
    return {
        "logprobs": lambda: lib.wkv6_token_logprobs(*rows, a["temperature"], a["logps"], a["stats"]),
        "cross_entropy": lambda: lib.wkv6_cross_entropy(*rows, a["red"], a["loss"], a["stats"], a["coef"], a["grad"], *ws),
        "policy": lambda: lib.wkv6_policy_loss(*rows, None, a["adv"], 1, 0, None, a["lo"], a["hi"], a["klw"], a["temperature"], a["red"], a["loss"], a["logps"], a["means"],
                                               a["stats"], a["coef"], a["grad"], *ws),
        "preference": lambda: lib.wkv6_preference_loss(*rows, None, a["kind"], a["beta"], a["ls"], 0, a["loss"], a["text"], a["stats"], a["coef"], *ws),
        "backward": lambda: lib.wkv6_logits_backward(*rows, a["temperature"], a["stats"], a["coef"], 1, 0, a["up"], a["there"], a["grad"]),
    }


def test_rows_of_logits(native):
    lib = native.load()
    for bad in BAD_ROWS:
        for name, call in _calls(lib, _rows(**bad)).items():
            assert call() == 1, (name, bad)
    for bad in TOO_MANY:
        for name, call in _calls(lib, _rows(**bad)).items():
            assert call() == 2, (name, bad)
    nan = float("nan")
    for bad, who in ((dict(temperature=0.0), "logprobs policy backward"), (dict(temperature=nan), "logprobs policy backward"),
                     (dict(temperature=float("inf")), "logprobs policy backward"), (dict(logps=None), "logprobs policy"), (dict(loss=None), "cross_entropy policy preference"),
                     (dict(loss=OFF), "cross_entropy policy preference"), (dict(stats=OK + 2), "logprobs cross_entropy policy preference backward"),
                     (dict(grad=OFF), "cross_entropy policy backward"), (dict(stats=None), "cross_entropy policy backward"), (dict(coef=None), "cross_entropy policy backward"),
                     (dict(grad=None), "backward"), (dict(up=None, there=1), "backward"), (dict(red=3), "cross_entropy policy"), (dict(red=2), "cross_entropy"), (dict(red=0), "policy"),
                     (dict(adv=None), "policy"), (dict(means=None), "policy"), (dict(lo=-0.1), "policy"), (dict(hi=nan), "policy"), (dict(klw=nan), "policy"),
                     (dict(kind=3), "preference"), (dict(beta=0.0), "preference"), (dict(beta=nan), "preference"), (dict(ls=0.5), "preference"),
                     (dict(ls=0.1, kind=1), "preference"), (dict(text=None), "preference")):
        calls = _calls(lib, _rows(), **bad)
        for name in who.split():
            assert calls[name]() == 1, (name, bad)
    assert _calls(lib, _rows(B=3))["preference"]() == 1
    need = lib.wkv6_loss_workspace_bytes(2, 3)
    assert need > 0 and lib.wkv6_loss_workspace_bytes(0, 3) == 0 and lib.wkv6_loss_workspace_bytes(1 << 20, 1 << 20) == 0
    for ws in ((None, 1 << 20), (OK + 8, 1 << 20), (OK, need - 1)):
        for name in ("cross_entropy", "policy", "preference"):
            assert _calls(lib, _rows(), *ws)[name]() == 3, (name, ws)


def _tensors(native, *rows):
    return (native.AdamwTensor * len(rows))(*[native.AdamwTensor(**r) for r in rows])


def test_optimizer(native):
    lib = native.load()
    good = dict(param=OK, grad=OK, exp_avg=OK, exp_avg_sq=OK, scales=OK, master=None, numel=10)

    def step(rows=(good,), dtype=0, bits=32, count=None, step=OK, lr_device=None, lr=1e-3, b1=0.9, b2=0.99, eps=1e-8, wd=0.0, clip=0.0, skip=0, norm=None):
        t = _tensors(native, *rows)
        return lib.wkv6_adamw_step(None, dtype, bits, len(rows) if count is None else count, t if rows else None, step, lr_device, lr, b1, b2, eps, wd, clip, skip, norm, 0)

    nan = float("nan")
    for bad in (dict(dtype=3), dict(bits=16), dict(count=0), dict(count=1 << 31), dict(step=None), dict(step=OK + 4), dict(lr=-1.0), dict(lr=nan), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0),
                dict(wd=nan), dict(clip=-1.0), dict(clip=1.0), dict(skip=1), dict(norm=OFF), dict(lr_device=OFF),
                dict(rows=(dict(good, param=None),)), dict(rows=(good, dict(good, grad=None))), dict(rows=(dict(good, exp_avg=None),)), dict(rows=(dict(good, exp_avg_sq=OK + 2),)),
                dict(rows=(dict(good, scales=None),), bits=8), dict(rows=(dict(good, scales=OK + 4),), bits=8), dict(rows=(dict(good, master=OFF),)),
                dict(rows=(dict(good, numel=-1),)), dict(rows=(dict(good, numel=1 << 40),)), dict(rows=(dict(good, param=OFF),)), dict(dtype=2, rows=(dict(good, grad=OK + 2),))):
        assert step(**bad) == 1, bad
    rows = _tensors(native, dict(grad=OK, numel=10))
    n = lib.wkv6_grad_norm_workspace_bytes(1)
    assert n > 0 and lib.wkv6_grad_norm_workspace_bytes(0) == 0
    assert lib.wkv6_grad_norm(None, 5, 1, rows, OK, OK, n) == 1 and lib.wkv6_grad_norm(None, 0, 1, rows, None, OK, n) == 1
    assert lib.wkv6_grad_norm(None, 0, 0, rows, OK, OK, n) == 1 and lib.wkv6_grad_norm(None, 0, 1, rows, OK, OK, n - 1) == 3
    assert lib.wkv6_grad_norm(None, 0, 1, _tensors(native, dict(grad=None, numel=10)), OK, OK, n) == 1
    assert ctypes.sizeof(native.AdamwTensor) == 56


def test_python_layer():
    import rwkv_kernel as k
    x, ids = torch.zeros(2, 3, 5), torch.zeros(2, 3, dtype=torch.int64)
    for call in (lambda: k.cross_entropy(x, ids), lambda: k.token_logprobs(x, ids), lambda: k.preference_loss(x, ids), lambda: k.policy_loss(x, ids, None, None, torch.zeros(2))):
        with pytest.raises(AssertionError, match="GPU"):
            call()
    p = torch.nn.Parameter(torch.zeros(4))
    for kw in (dict(moment_bits=4), dict(max_grad_norm=0.0), dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(weight_decay=-1.0)):
        with pytest.raises(AssertionError):
            k.AdamW([p], **kw)
    opt = k.AdamW([p])
    p.grad = torch.zeros(4)
    with pytest.raises(AssertionError, match="GPU"):
        opt.step()
    with pytest.raises(RuntimeError, match="GPU"):
        k.adamw_step([p.detach()], [p.grad], [p.grad], [p.grad], torch.zeros((), dtype=torch.int64), 1e-3)
    with pytest.raises(RuntimeError, match="GPU"):
        k.grad_norm([p.grad])


def test_masters_are_not_lost_or_gained_by_loading():
    """A state whose masters are not what the optimizer asks for is refused before anything is taken from it (no GPU needed)."""
    import rwkv_kernel as k
    params = lambda: [torch.nn.Parameter(torch.ones(5, dtype=d)) for d in (torch.bfloat16, torch.float32)]  # noqa: E731

    def saved(masters):
        """What an optimizer over the two has saved behind a step, with or without a master of the first."""
        state = {i: dict(step=torch.tensor(3), exp_avg=torch.full((5,), 0.5), exp_avg_sq=torch.full((5,), 0.25)) for i in (0, 1)}
        if masters:
            state[0]["master"] = torch.full((5,), 1.001)
        return dict(k.AdamW(params(), master_weights=masters).state_dict(), state=state)

    for has in (False, True):
        for wants in (False, True):
            opt = k.AdamW(params(), master_weights=wants)
            if has != wants:
                with pytest.raises(AssertionError, match="master"):
                    opt.load_state_dict(saved(has))
                assert not opt.state
                continue
            opt.load_state_dict(saved(has))
            a, b = (opt.state[p] for p in opt.param_groups[0]["params"])
            assert ("master" in a) == wants and "master" not in b and int(a["step"]) == 3
            assert not wants or (a["master"].dtype == torch.float32 and bool((a["master"] == 1.001).all()))
    # parameters of 16 bits that became parameters of 32 have no master either
    with pytest.raises(AssertionError, match="master"):
        k.AdamW([torch.nn.Parameter(p.detach().float()) for p in params()], master_weights=True).load_state_dict(saved(True))
