"""layer_norm and its gradients against the formula in float64.

Tolerances: with u = 2^-24 a sum over a row is added up in at most 64 steps (32 elements to a lane, 6 steps over a wave, at most 16 over waves), so the mean is off
by 64 u mean|s|, the variance by 64 u of itself and by the square of the mean's error, 1 / deviation by some 36 u; products and differences
add a few u of themselves.  A result is rounded once more, by half a step of its type.  Sums over rows: a wave adds at most rows / 2048 + 1 rows (where a
workgroup takes a row, rows / 512 + 1), then four waves, then workgroups in fp64."""
import gc

import pytest
import torch

import rwkv_kernel

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _round(x, dtype):
    """How far rounding to dtype is off at most: half a step, or half of the smallest number."""
    info = torch.finfo(dtype)
    return x.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2


def _within(name, got, want, off):
    got, want = got.detach().double().cpu(), want.detach().double()
    off = off + _round(want.abs() + off, _within.dtype)
    bad = ~((got - want).abs() <= off)
    assert not bool(bad.any()), (name, int(bad.sum()), float(((got - want).abs() / off).nan_to_num(1e9).max()))


def _check(name, got, want, off):
    _within.dtype = got.dtype
    _within(name, got, want, off)


def _formula(x, add, weight, bias, eps, gy, gtotal):
    """Values in float64 and what they may be off by before they are rounded, from tensors on the GPU."""
    s = x.detach().cpu()
    if add is not None:
        s = (s.float() + add.detach().cpu().float()).to(x.dtype)
    s = s.double().flatten(0, -2) if x.dim() > 1 else s.double()[None]
    rows, C = s.shape
    w = torch.ones(C).double() if weight is None else weight.detach().cpu().double()
    b = torch.zeros(C).double() if bias is None else bias.detach().cpu().double()
    m = s.mean(1, keepdim=True)
    q = 1 / torch.sqrt((s - m).square().mean(1, keepdim=True) + eps)
    h = (s - m) * q
    m_off = 64 * U * s.abs().mean(1, keepdim=True)
    q_off = 40 * U + (m_off * q).square()
    h_off = m_off * q + (q_off + 2 * U) * h.abs()
    y = h * w + b
    out = {"y": (y, h_off * w.abs() + 4 * U * ((h * w).abs() + b.abs())), "total": (s, torch.zeros_like(s))}
    if gy is None:
        return out
    g = gy.detach().cpu().double().reshape(rows, C)
    gw = g * w
    c1, c2 = gw.mean(1, keepdim=True), (gw * h).mean(1, keepdim=True)
    c1_off = 68 * U * gw.abs().mean(1, keepdim=True)
    c2_off = 68 * U * (gw * h).abs().mean(1, keepdim=True) + (gw.abs() * h_off).mean(1, keepdim=True)
    size = gw.abs() + c1.abs() + (h * c2).abs()
    gx = q * (gw - c1 - h * c2)
    off = q * (8 * U * size + c1_off + h_off * c2.abs() + (h.abs() + h_off) * c2_off) + (q_off + 4 * U) * q * size
    if gtotal is not None:
        t = gtotal.detach().cpu().double().reshape(rows, C)
        gx, off = gx + t, off + 2 * U * (gx.abs() + t.abs())
    steps = rows / (2048 if C <= 1024 else 512) + 16
    out["gx"] = out["gadd"] = (gx, off)
    out["gweight"] = ((g * h).sum(0), (g.abs() * h_off).sum(0) + steps * U * (g * h).abs().sum(0))
    out["gbias"] = (g.sum(0), steps * U * g.abs().sum(0))
    return out


def _inputs(shape, stream, branch, params, add, seed, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(shape, generator=g) * torch.exp(torch.randn(shape[-1], generator=g) * 0.5) + mean).to(stream).cuda()
    a = torch.randn(shape, generator=g).to(branch).cuda() if add else None
    w = b = None
    if params is not None:
        w, b = ((torch.randn(shape[-1], generator=g) * 0.3 + k).to(params).cuda() for k in (1.0, 0.0))
    gy, gt = torch.randn(shape, generator=g).to(branch).cuda(), torch.randn(shape, generator=g).to(stream).cuda() if add else None
    return x, a, w, b, gy, gt


def _run(x, a, w, b, gy, gt, branch, eps=1e-5):
    leaves = [None if t is None else t.detach().requires_grad_(True) for t in (x, a, w, b)]
    out = rwkv_kernel.layer_norm(leaves[0], leaves[2], leaves[3], eps=eps, add=leaves[1], dtype=branch)
    out = out if a is not None else (out,)
    grads = torch.autograd.grad(out, [t for t in leaves if t is not None], [gy] if gt is None else [gy, gt])
    res = dict(zip(("y", "total"), out))
    res.update(zip([n for n, t in zip(("gx", "gadd", "gweight", "gbias"), leaves) if t is not None], grads))
    return res


def _all_within(res, want):
    for name, got in res.items():
        value, off = want[name]
        _check(name, got.reshape(value.shape), value, off)


TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]


@pytest.mark.parametrize("stream,branch", TYPES)
@pytest.mark.parametrize("C", [1, 2, 7, 64, 100, 512, 513, 777, 1024, 2048, 2052, 4096, 5001, 8192, 8200, 16384, 16390, 32768])
def test_widths(C, stream, branch):
    print("layer norm", C, stream, branch, flush=True)
    rows = 5 if C > 8192 else 37
    for add, params in ((True, F32), (False, stream)):
        ins = _inputs((rows, C), stream, branch, params, add, C)
        res = _run(*ins, branch)
        x, a, w, b, gy, gt = ins
        _all_within(res, _formula(x, a, w, b, 1e-5, gy, gt))
        assert res["y"].dtype == branch and (not add or (res["total"].dtype == stream and res["gadd"].dtype == branch))
        assert res["gweight"].dtype == params


@pytest.mark.parametrize("rows,C", [(1, 2048), (3, 64), (4, 2048), (129, 777), (5000, 256), (2049, 2048), (1025, 4100), (513, 12000)])
def test_rows(rows, C):
    print("layer norm rows", rows, C, flush=True)
    for stream, branch in ((F32, BF16), (F16, F16)):
        ins = _inputs((rows, C), stream, branch, F32, True, rows)
        x, a, w, b, gy, gt = ins
        res = _run(*ins, branch)
        _all_within(res, _formula(x, a, w, b, 1e-5, gy, gt))
        again = _run(*ins, branch)
        assert all(torch.equal(res[k], again[k]) for k in res)


def test_a_mean_far_from_zero():
    """(values of 1000 and more with a deviation of 1: the sum of squares less the squared mean would keep nothing of it)"""
    for mean in (1e3, -1e5):
        x, a, w, b, gy, gt = _inputs((33, 1000), F32, F32, F32, False, 5, mean)
        _all_within(_run(x, a, w, b, gy, gt, F32), _formula(x, a, w, b, 1e-5, gy, gt))


def test_rows_that_are_constant():
    x = torch.full((3, 100), 7.0).cuda()
    y = rwkv_kernel.layer_norm(x, bias=torch.arange(100.0).cuda())
    assert torch.equal(y, torch.arange(100.0).cuda().expand(3, 100))
    y = rwkv_kernel.layer_norm(torch.zeros(2, 5, device="cuda"), eps=0.0)
    assert bool(y.isnan().all())


def test_slices_views_and_broadcasts():
    print("layer norm, strided", flush=True)
    g = torch.Generator().manual_seed(3)
    base = torch.randn(4, 9, 300, generator=g).cuda()
    w, b = torch.randn(300, generator=g).cuda(), torch.randn(300, generator=g).cuda()
    for x in (base[:, :-1], base[1:3, 2:7], base[:, 3], base.transpose(0, 1), base[:, :, :77], base[..., 1::2], base[0, 0], base[:1, :1, :].expand(4, 9, 300)):
        C = x.shape[-1]
        want = _formula(x, None, w[:C], b[:C], 1e-5, None, None)["y"]
        y = rwkv_kernel.layer_norm(x, w[:C], b[:C])
        assert y.shape == x.shape and y.is_contiguous()
        _check("y", y.reshape(want[0].shape), *want)
        gy = torch.randn(C, generator=g).cuda().expand(x.shape)   # (a gradient that is broadcast)
        leaf = x.detach().clone().requires_grad_(True)
        gx, = torch.autograd.grad(rwkv_kernel.layer_norm(leaf.as_strided(x.shape, leaf.stride()), w[:C], b[:C]), leaf, gy)
        want = _formula(x, None, w[:C], b[:C], 1e-5, gy, None)["gx"]
        _check("gx", gx.reshape(want[0].shape), *want)
        both = rwkv_kernel.layer_norm(x.clone(memory_format=torch.contiguous_format), w[:C], b[:C], add=x)
        want = _formula(x, x, w[:C], b[:C], 1e-5, None, None)
        for name, got in zip(("y", "total"), both):
            _check(name, got.reshape(want[name][0].shape), *want[name])


def test_any_address():
    """Rows, weights and gradients that begin at any element."""
    for dtype in (F32, BF16, F16):
        ins = [None if t is None else torch.cat([t.new_zeros(k + 1), t.reshape(-1)])[k + 1:].view(t.shape) for k, t in
               enumerate(_inputs((11, 130), dtype, dtype, dtype, True, 8))]
        x, a, w, b, gy, gt = ins
        _all_within(_run(*ins, dtype), _formula(x, a, w, b, 1e-5, gy, gt))


def test_types_that_are_not_the_kernels():
    """add and the norm in different types beside a stream in fp32."""
    for add_type, branch in ((F32, BF16), (BF16, F32), (F16, BF16)):
        x, a, w, b, gy, gt = _inputs((9, 256), F32, add_type, F32, True, 4)
        res = _run(x, a, w, b, gy.to(branch), gt, branch)
        want = _formula(x, a, w, b, 1e-5, gy.to(branch), gt)
        assert res["y"].dtype == branch and res["gadd"].dtype == add_type
        _all_within(res, want)


def test_some_gradients_only():
    x, a, w, b, gy, gt = _inputs((40, 500), F32, BF16, F32, True, 6)
    want = _formula(x, a, w, b, 1e-5, gy, gt)
    for names in (("x",), ("add",), ("weight",), ("bias",), ("x", "bias"), ("add", "weight")):
        leaves = {k: t.detach().requires_grad_(k in names) for k, t in dict(x=x, add=a, weight=w, bias=b).items()}
        y, total = rwkv_kernel.layer_norm(leaves["x"], leaves["weight"], leaves["bias"], add=leaves["add"], dtype=BF16)
        outs, arriving = ((y, total), (gy, gt)) if total.requires_grad and ("x" in names or "add" in names) else ((y,), (gy,))
        for k, got in zip(names, torch.autograd.grad(outs, [leaves[k] for k in names], arriving)):
            _check("g" + k, got.reshape(want["g" + k][0].shape), *want["g" + k])
    # a sum of what needs no gradient needs none, whatever the weights do
    y, total = rwkv_kernel.layer_norm(x, w.detach().requires_grad_(True), b, add=a, dtype=BF16)
    assert y.requires_grad and not total.requires_grad
    # one of the two outputs alone
    leaves = [t.detach().requires_grad_(True) for t in (x, a)]
    y, total = rwkv_kernel.layer_norm(leaves[0], w, b, add=leaves[1], dtype=BF16)
    gx, ga = torch.autograd.grad(total, leaves, gt, retain_graph=True)
    assert torch.equal(gx, gt) and torch.equal(ga, gt.to(BF16))
    alone = _formula(x, a, w, b, 1e-5, gy, None)
    gx, ga = torch.autograd.grad(y, leaves, gy)
    _check("gx", gx, *alone["gx"])
    _check("gadd", ga, *alone["gx"])


def test_differences():
    """A gradient against differences of the function itself, in the direction of a random change: fp32 outputs are good to some 2^-22 of their size, and the
    step of 2^-6 leaves a third-order term of about 2^-12 of the slope's size."""
    x, a, w, b, gy, gt = _inputs((6, 96), F32, F32, F32, True, 9)
    res = _run(x, a, w, b, gy, gt, F32)
    g = torch.Generator().manual_seed(1)
    for name, t in (("gx", x), ("gadd", a), ("gweight", w), ("gbias", b)):
        d = torch.randn(t.shape, generator=g).cuda()
        h = 2.0 ** -6

        def value(k):
            args = [t + k * h * d if u is t else u for u in (x, a, w, b)]
            y, total = rwkv_kernel.layer_norm(args[0], args[2], args[3], add=args[1])
            return float((y.double() * gy.double()).sum() + (total.double() * gt.double()).sum())

        slope = (8 * (value(1) - value(-1)) - (value(2) - value(-2))) / (12 * h)
        want = float((res[name].double() * d.double()).sum())
        size = float((res[name].double() * d.double()).abs().sum())
        assert abs(slope - want) <= 2.0 ** -10 * size, (name, slope, want, size)


def test_rows_that_are_no_numbers_stay_apart():
    for bad in (float("nan"), float("inf"), -float("inf")):
        x, a, w, b, gy, gt = _inputs((8, 300), F32, BF16, F32, True, 2)
        x[3, 17] = bad
        res = _run(x, a, w, b, gy, gt, BF16)
        keep = [0, 1, 2, 4, 5, 6, 7]
        want = _formula(x[keep], a[keep], w, b, 1e-5, gy[keep], gt[keep])
        for name in ("y", "total", "gx", "gadd"):
            _check(name, res[name][keep], *want[name])
        assert bool(res["y"][3].isnan().all()) and bool(res["gx"][3].isnan().all())


def test_empty_and_refused():
    x = torch.zeros(0, 8, device="cuda")
    assert rwkv_kernel.layer_norm(x).shape == (0, 8)
    y, total = rwkv_kernel.layer_norm(x, add=x.to(BF16), dtype=BF16)
    assert y.dtype == BF16 and total.dtype == F32
    w = torch.ones(8, device="cuda")
    x = torch.zeros(2, 8, device="cuda")
    for call in (lambda: rwkv_kernel.layer_norm(x.double()), lambda: rwkv_kernel.layer_norm(x, w[:7]), lambda: rwkv_kernel.layer_norm(x, w, w.to(BF16)),
                 lambda: rwkv_kernel.layer_norm(x.to(BF16), dtype=F32), lambda: rwkv_kernel.layer_norm(x, add=x[:1]), lambda: rwkv_kernel.layer_norm(x, eps=-1.0),
                 lambda: rwkv_kernel.layer_norm(x.to(BF16), add=x), lambda: rwkv_kernel.layer_norm(x, w.cpu()),
                 lambda: rwkv_kernel.layer_norm(torch.zeros(1, 32769, device="cuda"))):
        with pytest.raises(AssertionError):
            call()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(rwkv_kernel.layer_norm(leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_nothing_is_kept_of_a_forward_that_is_dropped():
    x, a, w, b, _, _ = _inputs((500, 1024), F32, BF16, F32, True, 3)
    leaves = [t.detach().requires_grad_(True) for t in (x, a, w, b)]
    gc.collect()   # (what other tests have left may go meanwhile)
    before = torch.cuda.memory_allocated()
    for _ in range(5):
        y, total = rwkv_kernel.layer_norm(leaves[0], leaves[2], leaves[3], add=leaves[1], dtype=BF16)
        del y, total
    assert torch.cuda.memory_allocated() <= before


def test_a_sum_that_is_changed_is_noticed():
    """The backward reads the sum that was returned: changed in place, it is refused."""
    x, a, w, b, gy, _ = _inputs((5, 64), F32, F32, F32, True, 3)
    leaf = x.detach().requires_grad_(True)
    y, total = rwkv_kernel.layer_norm(leaf, w, b, add=a)
    with torch.no_grad():
        total.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, leaf, gy)


def test_added_to_itself():
    """layer_norm(x, add=x): x gets both gradients."""
    for dtype in (F32, BF16):
        x, _, w, b, gy, gt = _inputs((21, 200), dtype, dtype, F32, True, 3)
        want = _formula(x, x, w, b, 1e-5, gy, gt)
        leaf = x.detach().requires_grad_(True)
        gx, = torch.autograd.grad(rwkv_kernel.layer_norm(leaf, w, b, add=leaf), leaf, [gy, gt])
        value, off = want["gx"]
        _check("gx", gx, 2 * value, 2 * (off + _round(value.abs() + off, dtype)))


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last rows are those of a call of their own, and the sums over rows those of its parts."""
    print("layer norm, 2^31 elements", flush=True)
    rows, C = 70000, 32768
    x = torch.zeros(rows, C, dtype=BF16, device="cuda")
    g = torch.Generator().manual_seed(2)
    x[-3:], x[0] = torch.randn(3, C, generator=g).to(BF16).cuda(), torch.randn(C, generator=g).to(BF16).cuda()
    w = torch.randn(C, generator=g).cuda()
    gy = torch.zeros(rows, C, dtype=BF16, device="cuda")
    gy[-3:] = torch.randn(3, C, generator=g).to(BF16).cuda()
    some = [0, rows - 3, rows - 2, rows - 1]

    def run(x, gy):
        leaf, weight = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
        y = rwkv_kernel.layer_norm(leaf, weight)
        return (y.detach(), *torch.autograd.grad(y, (leaf, weight), gy))

    y, gx, gw = run(x, gy)
    y4, gx4, gw4 = run(x[some], gy[some])
    assert torch.equal(y[some], y4) and torch.equal(gx[some], gx4)
    assert float((gw - gw4).abs().max()) <= 8 * U * float((gy[some].float().abs() * 8).sum(0).max())
    assert not bool(y[1:-3].view(-1).view(torch.int16).any())


def test_captured_and_on_another_stream():
    print("layer norm, captured", flush=True)
    x, a, w, b, gy, gt = _inputs((300, 512), F32, BF16, F32, True, 7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            _run(x, a, w, b, gy, gt, BF16)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            res = _run(x, a, w, b, gy, gt, BF16)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (11, 12, 13):
        for t, new in zip((x, a, w, b, gy, gt), _inputs((300, 512), F32, BF16, F32, True, seed)):
            t.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager = _run(x, a, w, b, gy, gt, BF16)
        assert all(torch.equal(res[k], eager[k]) for k in res)
        _all_within(res, _formula(x, a, w, b, 1e-5, gy, gt))


def test_second_derivatives_are_refused_for_any_layout():
    """A derivative of a gradient that was taken with create_graph is refused, and not left out, for inputs that the kernels read as they are and for those that are copied."""
    big = _inputs((6, 4, 32), F32, F32, F32, False, 8)[0]
    w = torch.ones(16, device="cuda")
    for view in (lambda t: t, lambda t: t.transpose(0, 1), lambda t: t[:, :, ::2], lambda t: t.permute(2, 0, 1), lambda t: t[1::2, 1:3, :16], lambda t: t[0, 0].expand(3, 32)):
        for how in ("alone", "added", "added to"):
            leaf = big.clone().requires_grad_(True)
            x = view(leaf)
            if how == "alone":
                y = rwkv_kernel.layer_norm(x, w if x.shape[-1] == 16 else None)
            else:
                y, _ = rwkv_kernel.layer_norm(*((x,) if how == "added to" else (torch.ones_like(x),)), add=torch.ones_like(x) if how == "added to" else x)
            g, = torch.autograd.grad(y.sum(), leaf, create_graph=True)
            assert g.requires_grad, how
            with pytest.raises(RuntimeError, match="second derivative"):
                (y.sum() + g.square().sum()).backward()
