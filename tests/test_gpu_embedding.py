"""embedding and the gradient of its table against the formula in float64.

Tolerances: a value of the forward is one product in fp32 and one rounding to its type; a sum over n rows is off by at most n u of the sum of its terms' sizes, u = 2^-24
(fp32, in any order), by u more for the scale, and by the rounding to the table's type."""
import pytest
import torch

import rwkv_kernel

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16), (F16, F16)]


def _round(x, dtype):
    info = torch.finfo(dtype)
    return x.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2


def _check(ids, weight, scale, padding_id, dtype, gout, out, grad):
    """All rows of the result and of the gradient, on the CPU."""
    V, C = weight.shape
    i, w, g = ids.reshape(-1).cpu(), weight.detach().cpu().double(), gout.detach().cpu().double().reshape(-1, C)
    held = (i >= 0) & (i < V)
    want = torch.zeros(len(i), C).double()
    want[held] = w[i[held]] * scale
    want[i >= V] = float("nan")
    got = out.detach().cpu().double().reshape(-1, C)
    off = 2 * U * want.abs()
    off = off + _round(want.abs() + off, dtype)
    assert out.dtype == dtype and out.shape == (*ids.shape, C)
    assert torch.equal(got.isnan(), want.isnan()) and not bool(((got - want).abs() > off).any())
    if scale == 1.0 and weight.dtype == dtype:
        assert torch.equal(got.nan_to_num(7.0), want.nan_to_num(7.0))
    part = held if padding_id is None else held & (i != padding_id)
    total, size, count = torch.zeros(V, C).double(), torch.zeros(V, C).double(), torch.zeros(V).double()
    total.index_add_(0, i[part], g[part])
    size.index_add_(0, i[part], g[part].abs())
    count.index_add_(0, i[part], torch.ones(int(part.sum())).double())
    total, size = total * scale, size * abs(scale)
    off = (count[:, None] + 2) * U * size
    off = off + _round(total.abs() + off, weight.dtype)
    got = grad.cpu().double()
    assert grad.dtype == weight.dtype and grad.shape == weight.shape
    bad = (got - total).abs() > off
    assert not bool(bad.any()) and bool(got.isfinite().all()), (int(bad.sum()), float(((got - total).abs() / off.clamp(min=1e-300)).max()))
    assert not bool(got[count == 0].any())


def _run(ids, weight, scale=1.0, padding_id=None, dtype=None, gout=None):
    leaf = weight.detach().requires_grad_(True)
    out = rwkv_kernel.embedding(ids, leaf, scale=scale, padding_id=padding_id, dtype=dtype)
    grad, = torch.autograd.grad(out, leaf, gout)
    return out, grad


def _case(shape, V, C, seed, table=F32, dtype=F32, kind="uniform", **kw):
    g = torch.Generator().manual_seed(seed)
    weight = torch.randn(V, C, generator=g).to(table).cuda()
    if kind == "uniform":
        ids = torch.randint(0, V, shape, generator=g)
    elif kind == "one":
        ids = torch.full(shape, V // 2)
    elif kind == "text":   # the k-th token as often as 1 / k
        ids = (torch.exp(torch.rand(shape, generator=g).double() * torch.log(torch.tensor(V + 1.0))).long() - 1).clamp(0, V - 1)
    elif kind == "sorted":
        ids = torch.randint(0, V, shape, generator=g).reshape(-1).sort().values.reshape(shape)
    else:   # some outside of the table
        ids = torch.randint(-V // 4 - 1, V + V // 4 + 1, shape, generator=g)
    ids, gout = ids.cuda(), torch.randn(*shape, C, generator=g).to(dtype).cuda()
    kw.setdefault("scale", 1.0)
    out, grad = _run(ids, weight, dtype=dtype, gout=gout, **kw)
    _check(ids, weight, kw["scale"], kw.get("padding_id"), dtype, gout, out, grad)
    out2, grad2 = _run(ids, weight, dtype=dtype, gout=gout, **kw)
    assert torch.equal(grad, grad2)


@pytest.mark.parametrize("table,dtype", TYPES)
def test_types(table, dtype):
    print("embedding", table, dtype, flush=True)
    for C in (1, 3, 8, 64, 130, 777, 1024, 2048, 2500, 4100, 9000):
        _case((3, 41), 50, C, C, table, dtype, "text", scale=3.7)


@pytest.mark.parametrize("kind", ["uniform", "one", "text", "sorted", "outside"])
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 63, 64, 65, 1000, 1024, 1025, 4097, 16383, 16384, 16385, 20000])
def test_numbers_of_tokens(N, kind):
    print("embedding", N, kind, flush=True)
    _case((N,), 300, 40, N, F32, F32, kind)
    _case((N,), 7, 12, N + 1, BF16, BF16, kind)


@pytest.mark.parametrize("V", [1, 2, 511, 512, 513, 65535, 65536, 262143, 262144, 300000])
def test_sizes_of_the_table(V):
    print("embedding, table", V, flush=True)
    for kind in ("uniform", "text", "outside"):
        _case((2500,), V, 20, V, F32, BF16, kind)


def test_many_tokens():
    print("embedding, many tokens", flush=True)
    _case((5, 40001), 65536, 16, 1, BF16, BF16, "text")
    _case((300000,), 3, 8, 2, F32, F32, "uniform")
    _case((70000,), 400000, 8, 3, F32, F32, "outside")


def test_padding_id_and_shapes():
    _case((4, 5, 6), 30, 33, 4, kind="text", padding_id=0)
    _case((4, 5, 6), 30, 33, 4, kind="outside", padding_id=29)
    _case((100,), 30, 33, 4, kind="one", padding_id=15)   # (nothing is left)
    weight = torch.randn(30, 33).cuda()
    out = rwkv_kernel.embedding(torch.tensor(7, device="cuda"), weight)
    assert torch.equal(out, weight[7])
    leaf = weight.clone().requires_grad_(True)
    out = rwkv_kernel.embedding(torch.zeros(2, 0, dtype=torch.int64, device="cuda"), leaf, dtype=BF16)
    assert out.shape == (2, 0, 33) and out.dtype == BF16
    out.sum().backward()
    assert not bool(leaf.grad.any())


def test_strided_tables_ids_and_gradients():
    print("embedding, strided", flush=True)
    g = torch.Generator().manual_seed(5)
    big = torch.randn(60, 50, generator=g).cuda()
    ids = torch.randint(0, 50, (9, 14), generator=g).cuda()
    for w in (big[:, :21], big[::2][:30, 3:], big.t(), big[5:55, 1:2]):
        i = ids % w.shape[0]
        for j in (i, i.t(), i[:, ::3], i[:1].expand(5, 14)):
            gout = torch.randn(j.shape[-1], w.shape[1], generator=g).cuda().expand(*j.shape, w.shape[1])
            out, grad = _run(j, w, scale=0.5, gout=gout)
            _check(j, w, 0.5, None, F32, gout, out, grad)
    flat = torch.randn(1 + 40 * 13, generator=g).cuda()[1:].view(40, 13)   # any address
    gout = torch.randn(1 + 9 * 14 * 13, generator=g).cuda()[1:].view(9, 14, 13)
    out, grad = _run(ids % 40, flat, gout=gout)
    _check(ids % 40, flat, 1.0, None, F32, gout, out, grad)


def test_offsets_beyond_32_bits():
    """A table of more than 2^31 elements: its last rows, and their gradients."""
    V, C = 131073, 16400
    weight = torch.empty(V, C, dtype=BF16, device="cuda")
    rows = torch.tensor([0, 131071, 131072], device="cuda")
    values = torch.randn(3, C, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    weight[rows] = values
    leaf = weight.requires_grad_(True)
    out = rwkv_kernel.embedding(rows[[2, 0, 1, 2]], leaf)
    assert torch.equal(out, values[[2, 0, 1, 2]])
    gout = torch.ones(4, C, dtype=BF16, device="cuda") * torch.tensor([1.0, 2.0, 4.0, 8.0], device="cuda")[:, None].to(BF16)
    grad, = torch.autograd.grad(out, leaf, gout)
    assert torch.equal(grad[rows].float(), torch.tensor([2.0, 4.0, 9.0], device="cuda")[:, None].expand(3, C))
    assert int(torch.count_nonzero(grad[:, 0])) == 3 and int(torch.count_nonzero(grad[:, C - 1])) == 3
    grad[rows] = 0
    assert not bool(grad.view(-1).view(torch.int16).any())


def test_values_that_are_no_numbers_stay_in_their_rows():
    weight = torch.randn(10, 20).cuda()
    ids = torch.tensor([1, 2, 3, 2, 9], device="cuda")
    gout = torch.ones(5, 20, device="cuda")
    gout[1, 4], gout[4, 5] = float("nan"), float("inf")
    _, grad = _run(ids, weight, gout=gout)
    want = torch.zeros(10, 20)
    want[1], want[2], want[3], want[9] = 1.0, 2.0, 1.0, 1.0
    want[2, 4], want[9, 5] = float("nan"), float("inf")
    assert torch.equal(grad.cpu().nan_to_num(5.0), want.nan_to_num(5.0))


def test_refused():
    w, i = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for call in (lambda: rwkv_kernel.embedding(i.int(), w), lambda: rwkv_kernel.embedding(i.cpu(), w), lambda: rwkv_kernel.embedding(i, w.double()),
                 lambda: rwkv_kernel.embedding(i, w[0]), lambda: rwkv_kernel.embedding(i, w.to(BF16), dtype=F32), lambda: rwkv_kernel.embedding(i, w, padding_id=4),
                 lambda: rwkv_kernel.embedding(i, w, padding_id=-1), lambda: rwkv_kernel.embedding(i, w[:0])):
        with pytest.raises(AssertionError):
            call()
    leaf = w.clone().requires_grad_(True)
    g, = torch.autograd.grad(rwkv_kernel.embedding(i, leaf).square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        g.sum().backward()


def test_captured_and_on_another_stream():
    print("embedding, captured", flush=True)
    g = torch.Generator().manual_seed(7)
    for N in (900, 17000):
        weight, gout = torch.randn(500, 64, generator=g).cuda(), torch.randn(N, 64, generator=g).cuda()
        ids = torch.randint(0, 500, (N,), generator=g).cuda()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                _run(ids, weight, gout=gout)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out, grad = _run(ids, weight, gout=gout)
        torch.cuda.current_stream().wait_stream(side)
        for _ in range(3):
            ids.copy_(torch.randint(-3, 500, (N,), generator=g))
            gout.copy_(torch.randn(N, 64, generator=g))
            graph.replay()
            torch.cuda.synchronize()
            _check(ids, weight, 1.0, None, F32, gout, out, grad)
            assert torch.equal(grad, _run(ids, weight, gout=gout)[1])
