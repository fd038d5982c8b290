"""orthogonalize, muon_step and the optimizer against the formula in float64.

Tolerances: the iteration multiplies what is lost in small singular values by up to 485, by how much depends on the matrix.  So the same iteration in float32 gives the
measure: a pair of fp16 numbers has 22 bits where float32 has 24, each rounding is at most 4 times as large and there are as many of them, and the results may differ from
float64 by 8 times what float32's does, in the 2-norm and in the largest element (beside 2^-19 of it, or 2^-16 of matrices so small that float32 may
happen to be exact: five steps of some six roundings of 2^-22, doubled on the way).  The result's rounding to its type comes on top."""
import math

import pytest
import torch

import rwkv_kernel
from rwkv_kernel.torch_muon import COEFFICIENTS

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def _iterate(g, steps=5, coefficients=COEFFICIENTS, eps=1e-7, dtype=torch.float64):
    """One matrix, in this dtype, on its device."""
    rows = coefficients if hasattr(coefficients[0], "__len__") else [coefficients] * steps
    x = (g.double() / (g.double().norm() + eps)).to(dtype)
    tall = x.shape[0] > x.shape[1]
    x = x.t().contiguous() if tall else x
    for a, b, c in rows:
        gram = x @ x.t().contiguous()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if tall else x


def _off(g, **kw):
    """(the value in float64, what each element may be off by, and the 2-norm of all)"""
    want, single = _iterate(g, **kw), _iterate(g, dtype=F32, **kw).double()
    floor = 2.0 ** (-16 if min(g.shape) <= 4 else -19)
    return want, 8 * float((single - want).abs().max()) + floor * float(want.abs().max()), 8 * float((single - want).norm()) + floor * float(want.norm())


def _check(got, g, **kw):
    assert got.shape == g.shape and got.dtype == g.dtype and got.is_contiguous()
    want, each, all_ = _off(g, **kw)
    half = torch.finfo(got.dtype).eps / 2
    rounding = want.abs() * half + torch.finfo(got.dtype).smallest_normal * half
    error = (got.double() - want).abs()
    assert bool((error <= each + rounding + each * half).all()), (tuple(g.shape), float(error.max()), each)
    assert float(error.norm()) <= all_ + float(rounding.norm()) * (1 + half), (tuple(g.shape), float(error.norm()), all_)


def _matrix(m, n, seed, kind="gradient", dtype=F32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, n, generator=g)
    if kind == "gradient":     # a few strong directions and many weak ones
        r = min(m, n, 8)
        x = (torch.randn(m, r, generator=g) * torch.exp(-torch.arange(r) / 2.0)) @ torch.randn(r, n, generator=g) + 0.2 * x
    elif kind == "deficient":  # rows that repeat
        x = x[torch.arange(m) // 2]
    elif kind == "sparse":
        x = x * (torch.rand(m, n, generator=g) < 0.01)
        x[0, 0] = 1.0
    return (x * 1e-3).to(dtype).cuda()


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 3), (3, 2), (16, 16), (31, 33), (33, 31), (32, 32), (32, 64), (64, 32), (63, 65), (64, 64), (65, 129), (96, 100), (128, 128), (129, 300),
          (300, 129), (256, 256), (257, 1000), (32, 2048), (2048, 32), (777, 1311), (1500, 600)]


@pytest.mark.parametrize("m,n", SHAPES)
def test_shapes(m, n):
    print("orthogonalize", m, n, flush=True)
    for dtype in (F32, BF16, F16):
        x = _matrix(m, n, m + n, dtype=dtype)
        out = rwkv_kernel.orthogonalize(x)
        _check(out, x)
        assert torch.equal(out, rwkv_kernel.orthogonalize(x))


@pytest.mark.parametrize("kind", ["gradient", "normal", "deficient", "sparse"])
def test_kinds(kind):
    print("orthogonalize", kind, flush=True)
    for m, n in ((100, 300), (300, 100), (200, 200)):
        x = _matrix(m, n, 5, kind)
        _check(rwkv_kernel.orthogonalize(x), x)
        _check(rwkv_kernel.orthogonalize(x, steps=1), x, steps=1)
        triples = [(3.0, -3.2, 1.2), (1.875, -1.25, 0.375)] * 2
        _check(rwkv_kernel.orthogonalize(x, steps=4, coefficients=triples, eps=1e-3), x, steps=4, coefficients=triples, eps=1e-3)


def test_singular_values():
    """What the operator is for: those of a well-conditioned matrix come to 0.65 .. 1.25."""
    x = _matrix(120, 400, 3, "normal")
    s = torch.linalg.svdvals(rwkv_kernel.orthogonalize(x).double().cpu())
    assert 0.65 < float(s.min()) and float(s.max()) < 1.25


def test_lists_and_batches():
    print("orthogonalize, lists", flush=True)
    shapes = [(64, 64), (3, 200, 70), (1, 1), (32, 300), (2, 2, 40, 40), (300, 32), (0, 5), (256, 700), (4, 0, 8)] + [(24 + i, 40) for i in range(70)]
    xs = [_matrix(math.prod(s[:-1]), s[-1], i).view(s) if math.prod(s) else torch.zeros(s, device="cuda") for i, s in enumerate(shapes)]
    out = rwkv_kernel.orthogonalize(xs)
    for x, o in zip(xs, out):
        assert o.shape == x.shape
        if x.numel():
            for a, b in zip(x.reshape(-1, *x.shape[-2:]), o.reshape(-1, *o.shape[-2:])):
                _check(b, a)
    assert rwkv_kernel.orthogonalize([]) == []


@pytest.mark.parametrize("count,m,n", [(4, 2048, 2048), (1, 2048, 2048), (1, 1024, 4096), (2, 4096, 1024), (9, 1000, 1500), (1, 300, 20000)])
def test_large(count, m, n):
    """(in float64 and float32 on the GPU)"""
    print("orthogonalize", count, m, n, flush=True)
    xs = [_matrix(m, n, i, dtype=BF16 if i % 2 else F32) for i in range(count)]
    for dtype in (F32, BF16):
        mine = [x for x in xs if x.dtype == dtype]
        for x, o in zip(mine, rwkv_kernel.orthogonalize(mine)):
            _check(o, x)


@pytest.mark.parametrize("m,n", [(1, 50000), (20, 70001), (64, 100000), (60000, 33), (65, 60000), (9000, 300), (512, 8192), (513, 8300), (130, 8191), (200, 33333)])
def test_long_and_thin(m, n):
    print("orthogonalize", m, n, flush=True)
    x = _matrix(m, n, 4, "normal")
    _check(rwkv_kernel.orthogonalize(x), x)
    few = [x, _matrix(100, 9000, 5), _matrix(40, 20000, 6), _matrix(90, 90, 7), x]
    out = rwkv_kernel.orthogonalize(few)
    for y, o in zip(few, out):
        _check(o, y)


def test_more_than_the_workspace_holds_at_once():
    """30 matrices of 2048 x 2048 go through in parts; and matrices through the C interface with room for one at a time, or for two."""
    print("orthogonalize, in parts", flush=True)
    xs = [_matrix(2048, 2048, i, "normal", BF16) for i in range(3)] * 10
    out = rwkv_kernel.orthogonalize(xs)
    for i in range(3):
        _check(out[i], xs[i])
        assert torch.equal(out[27 + i], rwkv_kernel.orthogonalize(xs)[27 + i])
    del xs, out
    from rwkv_kernel import _native

    lib = _native.load()
    ys = [_matrix(200, 300, 1), _matrix(300, 100, 2), _matrix(40, 500, 3), _matrix(200, 300, 4), _matrix(3, 3, 5)]
    rows = (_native.MuonMatrix * len(ys))()
    outs = [torch.zeros_like(y) for y in ys]
    for r, y, o in zip(rows, ys, outs):
        r.grad, r.out, r.rows, r.columns = y.data_ptr(), o.data_ptr(), y.shape[0], y.shape[1]
    import ctypes
    triples = (ctypes.c_double * 15)(*(list(COEFFICIENTS) * 5))
    all_ = lib.wkv6_muon_workspace_bytes(len(ys), rows)
    one = max(lib.wkv6_muon_workspace_bytes(1, ctypes.byref(r)) for r in rows)
    assert one < all_
    for n in (all_, one, (one + all_) // 2):
        ws = torch.full((n + 4096,), 0x7F, dtype=torch.uint8, device="cuda")
        assert lib.wkv6_orthogonalize(torch.cuda.current_stream().cuda_stream, 2, len(ys), rows, 5, triples, 1e-7, ws.data_ptr(), n) == 0
        torch.cuda.synchronize()
        assert bool((ws[n:] == 0x7F).all())
        for y, o in zip(ys, outs):
            _check(o, y)
            o.zero_()


def test_two_streams_at_once():
    print("orthogonalize, two streams", flush=True)
    xs = [_matrix(300, 500, i) for i in range(2)]
    want = [rwkv_kernel.orthogonalize(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[k].append(rwkv_kernel.orthogonalize(xs[k]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for g, w in zip(got, want) for o in g)


def test_views():
    x = _matrix(50, 120, 1)
    big = torch.zeros(60, 130, device="cuda")
    big[3:53, 7:127] = x
    flat = torch.cat([x.new_zeros(1), x.reshape(-1)])[1:].view(50, 120)
    assert torch.equal(rwkv_kernel.orthogonalize(big[3:53, 7:127]), rwkv_kernel.orthogonalize(x))
    assert torch.equal(rwkv_kernel.orthogonalize(flat), rwkv_kernel.orthogonalize(x))
    _check(rwkv_kernel.orthogonalize(x.t()), x.t())


def test_sizes_of_the_values():
    """Only eps knows how large the elements are: from 1e-18 to 1e18 (their squares leave fp32), and nothing at all."""
    x = _matrix(40, 60, 2, "normal")
    for scale in (1e-18, 1e-10, 1e10, 1e18):
        y = x * scale
        _check(rwkv_kernel.orthogonalize(y, eps=0.0), y, eps=0.0)
    assert not bool(rwkv_kernel.orthogonalize(torch.zeros(40, 60, device="cuda")).any())
    y = x.clone()
    y[3, 3] = float("nan")
    assert bool(rwkv_kernel.orthogonalize(y).isnan().all())
    out = rwkv_kernel.orthogonalize([x, y, x])
    assert torch.equal(out[0], rwkv_kernel.orthogonalize(x)) and torch.equal(out[0], out[2])


def test_norms_far_below_eps():
    """X begins with entries down to 1e-12, where the pairs hold them to 2^-35 (half of fp16's smallest number, 2^-25, over 1024), which grows with the small singular
    values, by 3.4445^5 < 486, like they do: in the 2-norm 486 * 2^-35 * sqrt(number of elements), beside the relative part."""
    x = _matrix(40, 60, 2, "normal")
    for scale in (1e-7, 1e-9, 1e-11):
        y = x * scale
        want, _, all_ = _off(y)
        error = rwkv_kernel.orthogonalize(y).double() - want
        assert float(error.norm()) <= all_ + 2.0 ** -18 * float(want.norm()) + 486 * 2.0 ** -35 * math.sqrt(y.numel()), (scale, float(error.norm()), float(want.norm()))


def _step_inputs(shapes, dtype, seed, masters):
    ps = [_matrix(math.prod(s[:-1]), s[-1], seed + i, "normal").view(s) * 300 for i, s in enumerate(shapes)]
    gs = [_matrix(math.prod(s[:-1]), s[-1], seed + 100 + i).view(s).to(dtype) for i, s in enumerate(shapes)]
    bufs = [_matrix(math.prod(s[:-1]), s[-1], seed + 200 + i).view(s) * 0.3 for i, s in enumerate(shapes)]
    return [p.to(dtype) for p in ps], gs, bufs, ps if masters else None


def _check_step(before, after, lr, momentum, nesterov, decay, scale):
    params, grads, bufs, masters = before
    for i in range(len(params)):
        g, b = grads[i].double(), bufs[i].double()
        new = momentum * b + (1 - momentum) * g
        off = 4 * U * (momentum * b.abs() + (1 - momentum) * g.abs())
        assert bool(((after[2][i].double() - new).abs() <= off).all())
        u = (1 - momentum) * g + momentum * new if nesterov else new
        w = (masters or params)[i].double()
        shape = w.shape
        rate = {"shape": math.sqrt(max(1, shape[-2] / shape[-1])), "rms": 0.2 * math.sqrt(max(shape[-2:]))}.get(scale, scale)
        for j in range(math.prod(shape[:-2])):
            at = lambda t: t.reshape(-1, *shape[-2:])[j]  # noqa: E731
            o, each, _ = _off(at(u))
            want = at(w) * (1 - lr * decay) - lr * rate * o
            off = lr * rate * each + 4 * U * (at(w).abs() + lr * rate * o.abs())
            if masters:
                assert bool(((at(after[3][i]).double() - want).abs() <= off).all())
                assert torch.equal(after[0][i], after[3][i].to(after[0][i].dtype))
            half = torch.finfo(after[0][i].dtype).eps / 2
            off = off + (want.abs() + off) * half
            error = (at(after[0][i]).double() - want).abs()
            assert bool((error <= off).all()), (shape, float((error / off).max()))


@pytest.mark.parametrize("dtype,masters", [(F32, False), (BF16, False), (BF16, True), (F16, True)])
def test_steps(dtype, masters):
    print("muon step", dtype, masters, flush=True)
    shapes = [(64, 64), (300, 70), (70, 300), (2, 40, 50), (1, 9), (128, 256), (33, 33)]
    for momentum, nesterov, decay, scale in ((0.95, True, 0.1, "shape"), (0.9, False, 0.0, "rms"), (0.0, True, 0.5, 0.7)):
        before = _step_inputs(shapes, dtype, 7, masters)
        after = tuple(None if l is None else [t.clone() for t in l] for l in before)
        rwkv_kernel.muon_step(after[0], after[1], after[2], lr=0.02, momentum=momentum, nesterov=nesterov, weight_decay=decay, scale=scale, masters=after[3])
        assert all(torch.equal(a, b) for a, b in zip(before[1], after[1]))
        _check_step(before, after, 0.02, momentum, nesterov, decay, scale)
        again = tuple(None if l is None else [t.clone() for t in l] for l in before)
        rate = torch.tensor(0.02, device="cuda")
        rwkv_kernel.muon_step(again[0], again[1], again[2], lr=rate, momentum=momentum, nesterov=nesterov, weight_decay=decay, scale=scale, masters=again[3])
        assert all(torch.equal(a, b) for a, b in zip(after[0] + after[2], again[0] + again[2]))


def test_optimizer():
    print("Muon", flush=True)
    g = torch.Generator().manual_seed(1)
    make = lambda: [torch.nn.Parameter(p.clone()) for p in _step_inputs([(64, 32), (32, 64)], BF16, 3, False)[0]] + [torch.nn.Parameter(torch.ones(8, 8, device="cuda"))]  # noqa: E731
    ps, qs = make(), make()
    a, b = (rwkv_kernel.Muon([{"params": x[:2]}, {"params": x[2:], "lr": torch.tensor(0.1, device="cuda")}], lr=0.05, weight_decay=0.1, master_weights=True) for x in (ps, qs))
    for step in range(4):
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, generator=g).to(p.dtype).cuda() if step != 1 or p.shape != (8, 8) else None
            q.grad = p.grad
        before = [[p.detach().clone() for p in ps[:2]], [p.grad for p in ps[:2]], [a.state[p]["momentum"].clone() for p in ps[:2]] if step else [torch.zeros(p.shape, device="cuda") for p in ps[:2]],
                  [a.state[p]["master"].clone() for p in ps[:2]] if step else [p.detach().float() for p in ps[:2]]]
        last = ps[2].detach().clone()
        a.step()
        _check_step(before, [[p.detach() for p in ps[:2]], None, [a.state[p]["momentum"] for p in ps[:2]], [a.state[p]["master"] for p in ps[:2]]], 0.05, 0.95, True, 0.1, "shape")
        assert torch.equal(last, ps[2].detach()) == (step == 1)
        assert a.state[ps[0]]["momentum"].dtype == F32 and "master" not in a.state.get(ps[2], {})
        if step == 1:   # the twin goes on from what was saved
            b.load_state_dict(a.state_dict())
            for p, q in zip(ps, qs):
                q.data.copy_(p.data)
        if step > 1:
            b.step()
            assert all(torch.equal(p, q) for p, q in zip(ps, qs))
            assert b.state[qs[0]]["momentum"].dtype == F32 and b.state[qs[0]]["master"].dtype == F32
    with pytest.raises(AssertionError, match="master"):
        rwkv_kernel.Muon([{"params": qs[:2]}, {"params": qs[2:]}], lr=0.05).load_state_dict(a.state_dict())


def test_refused():
    w = torch.zeros(8, 8, device="cuda")
    step = lambda p=w, g=w.clone(), m=w.clone(), lr=0.1, **kw: rwkv_kernel.muon_step([p], [g], [m], lr, **kw)  # noqa: E731
    for call in (lambda: rwkv_kernel.orthogonalize(w, steps=0), lambda: rwkv_kernel.orthogonalize(w, coefficients=(1, 2)), lambda: rwkv_kernel.orthogonalize(w, eps=-1.0),
                 lambda: rwkv_kernel.orthogonalize(w, steps=2, coefficients=[(1, 2, 3)] * 3), lambda: rwkv_kernel.orthogonalize(w, coefficients=(1.0, 2.0, float("nan"))),
                 lambda: step(lr=-1.0), lambda: step(momentum=1.0), lambda: step(scale="other"), lambda: step(scale=-1.0), lambda: step(p=w[0], g=w[0], m=w[0]),
                 lambda: rwkv_kernel.Muon([torch.nn.Parameter(w[0])])):
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: rwkv_kernel.orthogonalize(w.double()), lambda: rwkv_kernel.orthogonalize(w[0]), lambda: rwkv_kernel.orthogonalize([w, w.to(BF16)]),
                 lambda: rwkv_kernel.orthogonalize([w, w.cpu()]), lambda: rwkv_kernel.orthogonalize(w.clone().requires_grad_(True)), lambda: step(p=w.t()[:, :4], g=w[:, :4], m=w[:, :4].contiguous()), lambda: step(m=w.to(BF16)),
                 lambda: step(g=w.to(BF16)), lambda: step(m=w), lambda: rwkv_kernel.muon_step([w, w.clone()], [w.clone()] * 2, [w.clone(), w], 0.1),
                 lambda: step(masters=[w.clone()]), lambda: step(lr=torch.ones(1)), lambda: rwkv_kernel.muon_step([], [], [], 0.1)):
        with pytest.raises(RuntimeError):
            call()


def test_captured_and_on_another_stream():
    print("muon step, captured", flush=True)
    shapes = [(64, 64), (300, 70), (16, 20)]
    state = _step_inputs(shapes, BF16, 9, True)
    twin = tuple([t.clone() for t in l] for l in state)
    rate = torch.tensor(0.02, device="cuda")
    run = lambda s: rwkv_kernel.muon_step(s[0], s[1], s[2], lr=rate, weight_decay=0.1, masters=s[3])  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(state)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            run(state)
    torch.cuda.current_stream().wait_stream(side)
    run(twin)
    for k in range(3):
        rate.fill_(0.01 * (k + 1))
        for a, b in zip(state[1], twin[1]):
            new = _matrix(*a.shape, 50 + k, dtype=BF16)
            a.copy_(new)
            b.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        run(twin)
        for x, y in zip(state, twin):
            assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_tangents_are_refused():
    """orthogonalize has no derivative in forward mode either."""
    import torch.autograd.forward_ad as fwd

    x = _matrix(40, 60, 2)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: rwkv_kernel.orthogonalize(dual), lambda: rwkv_kernel.orthogonalize([x, dual])):
            with pytest.raises(RuntimeError, match="no derivative"):
                call()
        assert torch.equal(rwkv_kernel.orthogonalize(fwd.unpack_dual(dual).primal), rwkv_kernel.orthogonalize(x))


@pytest.mark.parametrize("m,n", [(40, 60), (60, 40), (100, 130), (130, 100), (33, 9000), (100, 9000)])
def test_norms_at_the_ends_of_fp32(m, n):
    """1024 over the norm leaves fp32 at either end where the norm and X do not; an eps below fp32's smallest number is an eps."""
    print("orthogonalize, ends of fp32", m, n, flush=True)
    x = _matrix(m, n, 2, "normal") * 1e3   # of a size of 1
    for scale in (1e-41, 1e-37, 3e-30, 1e30, 3e37):
        y = x * scale
        assert bool(y.isfinite().all()) and bool(y.any())
        _check(rwkv_kernel.orthogonalize(y, eps=0.0), y, eps=0.0)
    y = x * 1e-40
    _check(rwkv_kernel.orthogonalize(y, eps=1e-39), y, eps=1e-39)
    _check(rwkv_kernel.orthogonalize(y, eps=1e-60), y, eps=1e-60)
    for eps in (1e-7, 1e-40, 1e-46, 1e-300):
        assert not bool(rwkv_kernel.orthogonalize(torch.zeros(m, n, device="cuda"), eps=eps).any()), eps
    assert bool(rwkv_kernel.orthogonalize(torch.zeros(m, n, device="cuda"), eps=0.0).isnan().all())


def test_gradients_in_what_is_written_are_refused():
    """Momenta are written before the gradients are read for the second time."""
    w = _matrix(40, 60, 1)
    buf = torch.zeros(3 * 2400, device="cuda")
    g, m, other = (buf[i * 2400:(i + 1) * 2400].view(40, 60) for i in range(3))
    shifted = buf[2500:4900].view(40, 60)
    for call in (lambda: rwkv_kernel.muon_step([w], [g], [g], 0.1), lambda: rwkv_kernel.muon_step([w], [shifted], [m], 0.1), lambda: rwkv_kernel.muon_step([w, g], [w.clone(), g], [m, other], 0.1),
                 lambda: rwkv_kernel.muon_step([w, g], [g, w.clone()], [m, other], 0.1),
                 lambda: rwkv_kernel.muon_step([w.to(BF16)], [g.view(-1).view(BF16)[:2400].view(40, 60)], [m], 0.1, masters=[g])):
        with pytest.raises(RuntimeError, match="gradient shares elements"):
            call()
    assert not bool(buf.any()) and torch.equal(w, _matrix(40, 60, 1))
    g.copy_(_matrix(40, 60, 3))
    rwkv_kernel.muon_step([w, m], [g, g], [other, torch.zeros_like(w)], 0.1)   # (one gradient may be two parameters')
    rwkv_kernel.muon_step([w], [m.view(60, 40).t()], [m], 0.1)                 # (and one that is not contiguous is copied before)


# Products are made in tiles of 64, 128 or 256, by how many tiles a launch has, 64 and 128 in two forms (few tiles, alone on their compute units, have four buffers): each of them
# with rows and columns left over, as results and as steps on weights, and the square of A (its tiles are counted on and above the diagonal).
FORMS = {"64 alone": [(300, 500)], "64 twice": [(1000, 1100)], "128 alone": [(1100, 2000)], "128 twice": [(2100, 1000)] * 2 + [(1000, 2100)], "256": [(1300, 2070), (2070, 1300)] * 10,
         "shared": [(300, 9000), (9000, 300)], "two launches": [(70, 90)] * 30 + [(90, 70)] * 30}
EACH = {"64 alone": [0], "64 twice": [0], "128 alone": [0], "128 twice": [0, 2], "256": [0, 1, 18, 19], "shared": [0, 1], "two launches": [0, 29, 55, 56, 59]}   # of them, what is compared


def _pick(lists, which):
    return tuple(None if l is None else [l[i] for i in which] for l in lists)


@pytest.mark.parametrize("dtype,masters", [(F32, False), (BF16, True), (F16, False)])
@pytest.mark.parametrize("form", list(FORMS))
def test_steps_in_every_tile_form(form, dtype, masters):
    print("muon step, tiles", form, dtype, masters, flush=True)
    before = _step_inputs(FORMS[form], dtype, 11, masters)
    kept = tuple(None if l is None else [t.clone() for t in l] for l in _pick(before, EACH[form]))
    rwkv_kernel.muon_step(before[0], before[1], before[2], lr=0.02, weight_decay=0.1, masters=before[3])
    _check_step(kept, _pick(before, EACH[form]), 0.02, 0.95, True, 0.1, "shape")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shapes", [[(1500, 1600)], [(1600, 1500)], [(1300, 2070)] * 25 + [(2070, 1300)] * 25, [(1290, 1310)] * 56])
def test_results_in_large_tiles(shapes, dtype):
    """One matrix whose A has more than 256 tiles of 64 and fewer than 128 of 128; lists whose A has 1024 tiles of 256."""
    print("orthogonalize, tiles", len(shapes), shapes[0], dtype, flush=True)
    some = {s: _matrix(*s, s[0], dtype=dtype) for s in set(shapes)}
    out = rwkv_kernel.orthogonalize([some[s] for s in shapes])
    for i in {0, len(shapes) // 2, len(shapes) - 1}:
        _check(out[i], some[shapes[i]])


def test_a_list_over_the_workspace():
    """42 matrices of 2048 x 2048 do not fit the workspace together: 31 and 11 go through, as results and as steps."""
    from rwkv_kernel import _native

    print("orthogonalize, over the workspace", flush=True)
    count, most = 42, 2 ** 31
    rows = (_native.MuonMatrix * count)()
    for r in rows:
        r.rows = r.columns = 2048
    lib = _native.load()
    one = lib.wkv6_muon_workspace_bytes(1, rows)
    assert lib.wkv6_muon_workspace_bytes(count, rows) == most < count * one and most // one == 31
    xs = [_matrix(2048, 2048, i, "normal", BF16) for i in range(5)]
    at = [i * 2 % 5 for i in range(count)]
    out = rwkv_kernel.orthogonalize([xs[i] for i in at])
    for i in (0, 30, 31, 32, 41):
        _check(out[i], xs[at[i]])
    assert all(torch.equal(out[i], out[i % 5]) for i in range(31))
    del out
    params, bufs = [xs[at[-1 - i]].clone() for i in range(count)], [torch.zeros(2048, 2048, device="cuda") for _ in range(count)]
    before = _pick((params, [xs[i] for i in at], bufs, None), (0, 30, 31, 41))
    before = (*([t.clone() for t in l] for l in before[:3]), None)
    rwkv_kernel.muon_step(params, [xs[i] for i in at], bufs, lr=0.02, weight_decay=0.1)
    _check_step(before, _pick((params, None, bufs, None), (0, 30, 31, 41)), 0.02, 0.95, True, 0.1, "shape")


@pytest.mark.parametrize("shapes", [[(32, 2048)] * 5 + [(2048, 32)] * 5, [(2048, 2048)], [(777, 1311)], [(300, 9000)]])
def test_calls_repeat_themselves(shapes):
    """Whatever the memory held that a call gets as its workspace; and a result in 16 bits is the fp32 result, rounded once."""
    print("orthogonalize, again", shapes[0], flush=True)
    for dtype in (BF16, F16):
        xs = [_matrix(*s, i, dtype=dtype) for i, s in enumerate(shapes)]
        want = rwkv_kernel.orthogonalize(xs)
        for k in range(6):
            for n in (1 << 18, 1 << 20, 1 << 22, 1 << 24, 1 << 25):
                torch.full((n,), (float("nan"), 3.0, float("inf"))[k % 3], device="cuda")
            assert all(torch.equal(a, b) for a, b in zip(want, rwkv_kernel.orthogonalize(xs)))
        single = rwkv_kernel.orthogonalize([x.float() for x in xs])
        assert all(torch.equal(a, b.to(dtype)) for a, b in zip(want, single))
