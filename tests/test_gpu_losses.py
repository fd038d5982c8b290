"""The losses over logits (token_logprobs, cross_entropy, preference_loss, policy_loss) against their formulas in float64 on the
same rounded logits, with torch's autograd for the gradients.

Tolerances, u = 2^-24.  The kernels keep a row's largest logit and the sum of exp((x - top) / temperature) in fp32.  With R the largest
|x - top| / temperature of the row, an exponent is formed with two roundings (2 R u, as a relative error of its exp), exp itself
has one unit in the last place (2 u).  The sum of V values has as many roundings (u each) as the thread with the most of them adds, and some ten for
what the threads bring together: rows of up to 4096 values belong to 64 threads, longer ones to 256 and more, so at most
n = min(V, 4096) / 64 + V / 256 + 1 (which values a thread adds depends on where the row begins in memory).  E = u (2 R + n + 12), relative, for the
sum, and as an absolute error for log(sum).  lp then is one product
and a difference in 64 bits: |lp| u more where it is stored.  p = exp / sum is off by 2 E p; a gradient c (1[id] - p) by |c| (2 E p + 2 u),
and by what c is off; then it is rounded once to its own type (half its eps, and half the smallest subnormal number)."""
import math

import pytest
import torch

import rwkv_kernel

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}
# vocabularies on either side of what a vector, a wave, a workgroup and the kernels' size classes hold
VOCABULARIES = [1, 2, 7, 8, 9, 63, 64, 255, 1000, 2047, 2048, 2049, 4100, 8191, 16384, 16392, 32768, 50277, 65536, 65537, 131073, 151936, 170001,
                512, 513, 1024, 1025, 4096, 4097, 8193, 12288, 12289, 20481, 24576, 24577, 40961, 49153, 57345, 81920, 81921, 106497, 163840, 163841, 163849,
                20480, 20488, 73000, 73729, 90113, 98304, 98305]


def _case(B, T, V, dtype, seed, std=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, V, generator=g) * std
    ids = torch.randint(0, V, (B, T), generator=g)
    x.scatter_add_(2, ids[..., None], torch.full((B, T, 1), 4.0))
    return x.to(dtype).cuda(), ids.cuda(), (torch.rand(B, T, generator=g) < 0.7).cuda(), g


def _lp64(x, ids, mask, temperature=1.0):
    """lp in float64 on the CPU with a graph to the leaf it returns, and E of each row."""
    leaf = x.detach().cpu().double().requires_grad_(True)
    counted = torch.ones_like(ids.cpu(), dtype=torch.bool) if mask is None else mask.cpu() != 0
    counted = counted & (ids.cpu() >= 0)
    z = torch.where(counted[..., None], leaf, torch.zeros((), dtype=torch.float64)) / temperature
    lse = torch.logsumexp(z, -1)
    lp = z.gather(-1, ids.cpu().clamp(min=0)[..., None])[..., 0] - lse
    lp = torch.where(counted, lp, torch.zeros_like(lp))
    finite = torch.where(torch.isfinite(z), z, z.amax(-1, keepdim=True)).detach()
    R = (finite.amax(-1) - finite.amin(-1))
    V = x.shape[-1]
    E = U * (2 * R + min(V, 4096) / 64 + V / 256 + 1 + 12)
    return leaf, lp, counted, E, torch.exp(z - lse[..., None]).detach()


def _within(name, got, want, tol):
    got, want = got.detach().cpu().double(), want.detach()
    assert got.shape == want.shape, name
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()) and bool(torch.isfinite(got).all()), "%s: %.3e beyond its tolerance" % (name, float(off.max()))


def _grad_within(name, got, want, p, c, c_off, E, dtype, temperature=1.0):
    """c, c_off (B,T): the coefficient of each row and how far it may be off."""
    c, c_off = c.abs()[..., None] / temperature, c_off[..., None] / temperature
    tol = c * (2 * E[..., None] * p + 3 * U) + c_off
    tol = tol + torch.finfo(dtype).eps / 2 * (want.abs() + tol) + SMALLEST[dtype]
    assert got.dtype == dtype, name
    _within(name, got, want, tol)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", VOCABULARIES)
def test_token_logprobs(V, dtype):
    print("token_logprobs", V, dtype, flush=True)
    B, T, tau = 2, 3, 0.7
    x, ids, mask, g = _case(B, T, V, dtype, V)
    mask[0, 0], mask[1, 2] = True, False
    x[1, 2] = float("nan")                       # a row that does not count is not looked at
    gout = torch.randn(B, T, generator=g)
    leaf, lp, counted, E, p = _lp64(x, ids, mask, tau)
    with torch.no_grad():
        alone = rwkv_kernel.token_logprobs(x, ids, mask, temperature=tau)
    xr = x.clone().requires_grad_(True)
    got = rwkv_kernel.token_logprobs(xr, ids, mask, temperature=tau)
    assert torch.equal(alone, got.detach()) and got.dtype == torch.float32
    _within("lp", got, lp, E + 2 * U * lp.abs())
    lp.backward(gout.double())
    got.backward(gout.cuda())
    c = torch.where(counted, gout.double(), torch.zeros(()).double())
    _grad_within("grad", xr.grad, leaf.grad, p, c, 2 * U * c.abs(), E, dtype, tau)
    assert bool((xr.grad[1, 2] == 0).all())


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", [(1, 1, 5), (3, 5, 1000), (2, 33, 4099), (1, 300, 257), (40, 1, 96), (2, 4, 65536), (1, 2, 151936)])
def test_cross_entropy(B, T, V, dtype, reduction):
    print("cross_entropy", B, T, V, dtype, flush=True)
    x, ids, mask, _ = _case(B, T, V, dtype, B * T + V)
    mask[0, 0] = True
    if T > 3:
        ids[0, 2] = -100
    scale = 1.0 if dtype == torch.bfloat16 else 512.0
    for up in (1.0, scale, 0.3):
        leaf, lp, counted, E, p = _lp64(x, ids, mask)
        n = int(counted.sum()) if reduction == "mean" else 1
        loss = -lp.sum() / n
        xr = x.clone().requires_grad_(True)
        got = rwkv_kernel.cross_entropy(xr, ids, mask, reduction=reduction)
        assert got.dtype == torch.float32 and got.shape == ()
        with torch.no_grad():
            assert torch.equal(got.detach(), rwkv_kernel.cross_entropy(x, ids, mask, reduction=reduction))
        _within("loss", got, loss, ((E + 4 * U * lp.abs()) * counted).sum() / n + 2 * U * loss.abs())
        loss.backward(torch.tensor(up).double())
        got.backward(torch.tensor(up).cuda())
        c = torch.where(counted, torch.tensor(float(torch.tensor(up))).double() / n, torch.zeros(()).double())
        _grad_within("grad", xr.grad, leaf.grad, p, c, 4 * U * c, E, dtype)


def test_flat_logits_and_texts_are_one():
    x, ids, mask, _ = _case(3, 7, 500, torch.bfloat16, 1)
    flat = rwkv_kernel.cross_entropy(x.view(21, 500), ids.view(21), mask.view(21))
    assert torch.equal(flat, rwkv_kernel.cross_entropy(x, ids, mask))
    lp = rwkv_kernel.token_logprobs(x.view(21, 500), ids.view(21))
    assert lp.shape == (21,) and torch.equal(lp.view(3, 7), rwkv_kernel.token_logprobs(x, ids))


def _preference(lp, counted, ref, beta, kind, smoothing, average):
    P = lp.shape[0] // 2
    s = lp.sum(1) / (counted.sum(1).clamp(min=1) if average else 1)
    r = torch.zeros_like(s) if ref is None else ref.cpu().double()
    d = s[:P] - s[P:] - (r[:P] - r[P:])
    sig = torch.nn.functional.logsigmoid
    each = {"sigmoid": lambda: -(1 - smoothing) * sig(beta * d) - smoothing * sig(-beta * d),
            "hinge": lambda: torch.relu(1 - beta * d), "ipo": lambda: (d - 0.5 / beta) ** 2}[kind]()
    return each.mean(), s, d


@pytest.mark.parametrize("kind,smoothing,average,with_ref", [("sigmoid", 0.0, False, True), ("sigmoid", 0.1, False, False), ("sigmoid", 0.0, True, True),
                                                             ("hinge", 0.0, False, True), ("ipo", 0.0, True, True)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("P,T,V", [(1, 1, 50), (3, 9, 1000), (20, 70, 130), (1, 3, 65536)])
def test_preference_loss(P, T, V, dtype, kind, smoothing, average, with_ref):
    print("preference_loss", P, T, V, dtype, kind, flush=True)
    x, ids, mask, g = _case(2 * P, T, V, dtype, P + T + V)
    if P > 1:
        mask[1] = False                      # a text of which no token counts
    beta = 0.1
    leaf, lp, counted, E, p = _lp64(x, ids, mask)
    # (away from the hinge's corner, where the gradient jumps)
    ref = (lp.detach().sum(1) + torch.randn(2 * P, generator=g).double() * 3).float().cuda() if with_ref else None
    loss, s, d = _preference(lp, counted, ref, beta, kind, smoothing, average)
    assert kind != "hinge" or float((1 - beta * d.detach()).abs().min()) > 1e-4
    xr = x.clone().requires_grad_(True)
    got, got_s = rwkv_kernel.preference_loss(xr, ids, mask, ref, beta=beta, kind=kind, label_smoothing=smoothing, average=average)
    with torch.no_grad():
        again, _ = rwkv_kernel.preference_loss(x, ids, mask, ref, beta=beta, kind=kind, label_smoothing=smoothing, average=average)
    assert torch.equal(got.detach(), again) and not got_s.requires_grad
    s_off = (E * counted).sum(1) / (counted.sum(1).clamp(min=1) if average else 1)
    _within("s", got_s, s, s_off + 2 * U * s.abs())
    d_off = s_off[:P] + s_off[P:]
    # dl/dd is at most beta or 2 |d - 1 / (2 beta)|, and changes by at most beta^2 / 4 or 2 times what d is off by
    slope = 2 * (d - 0.5 / beta).abs() + 2 * d_off if kind == "ipo" else torch.full_like(d, beta)
    _within("loss", got, loss, (slope * d_off).mean() + 2 * U * loss.abs())
    loss.backward()
    got.backward()
    length = counted.sum(1).clamp(min=1).double() if average else torch.ones(2 * P).double()
    c = (slope.detach().repeat(2) / P / length)[:, None].expand(lp.shape) * counted
    bend = {"sigmoid": beta * beta / 4, "hinge": 0.0, "ipo": 2.0}[kind]
    c_off = (bend * d_off.repeat(2) / P / length)[:, None] * counted + 4 * U * c
    _grad_within("grad", xr.grad, leaf.grad, p, c, c_off, E, dtype)


@pytest.mark.parametrize("reduction", ["mean", "mean_of_texts"])
@pytest.mark.parametrize("old,ref,per_token", [(True, True, False), (False, True, True), (True, False, True)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,T,V", [(1, 1, 30), (4, 9, 1000), (3, 65, 130), (2, 3, 65536), (300, 1, 64)])
def test_policy_loss(B, T, V, dtype, old, ref, per_token, reduction):
    print("policy_loss", B, T, V, dtype, old, ref, reduction, flush=True)
    tau, lo, hi, klw = 0.8, 0.2, 0.28, 0.05
    x, ids, mask, g = _case(B, T, V, dtype, B + T + V)
    if B > 1:
        mask[1] = False
    leaf, lp, counted, E, p = _lp64(x, ids, mask, tau)
    d = torch.randn(B, T, generator=g) * 0.2
    near = ((d.exp() - 1 - hi).abs() < 1e-2) | ((d.exp() - 1 + lo).abs() < 1e-2)
    d = torch.where(near, torch.zeros(()), d)    # away from the corners of the clipping
    old_lp = (lp.detach() - d).float() if old else None
    ref_lp = (lp.detach() + torch.randn(B, T, generator=g) * 0.3).float() if ref else None
    A = torch.randn(*((B, T) if per_token else (B,)), generator=g)
    junk = torch.full((B, T), float("nan"))      # what stands where no token counts is not looked at
    give = lambda v: None if v is None else torch.where(counted, v, junk).cuda()  # noqa: E731
    A_all = A.double() if per_token else A.double()[:, None].expand(B, T)
    ratio = torch.exp(lp - old_lp.double()) if old else torch.exp(lp - lp.detach())
    clipped = torch.where(A_all > 0, ratio > 1 + hi, ratio < 1 - lo)
    each = -torch.minimum(ratio * A_all, ratio.clamp(1 - lo, 1 + hi) * A_all)
    e = ref_lp.double() - lp if ref else torch.zeros_like(lp)
    kl = torch.exp(e) - e - 1
    n = counted.sum(1, keepdim=True).double()
    w = counted / (n.clamp(min=1) * (n > 0).sum() if reduction == "mean_of_texts" else counted.sum()).clamp(min=1)
    loss = ((each + klw * kl) * w).sum()
    xr = x.clone().requires_grad_(True)
    args = (ids, mask, give(old_lp), torch.where(counted, A, junk).cuda() if per_token else A.cuda())
    kw = dict(ref_logps=give(ref_lp), clip_low=lo, clip_high=hi, kl_weight=klw, temperature=tau, reduction=reduction)
    got, got_lp, means = rwkv_kernel.policy_loss(xr, *args, **kw)
    with torch.no_grad():
        again = rwkv_kernel.policy_loss(x, *args, **kw)
    assert all(torch.equal(a, b.detach()) for a, b in zip(again, (got, got_lp, means))) and not (got_lp.requires_grad or means.requires_grad)
    lp_off = E + 4 * U * lp.abs()
    _within("lp", got_lp, lp, lp_off)
    # a term changes by at most (ratio |A| + klw |1 - exp(e)|) times what lp is off by, and its own arithmetic has some ten roundings
    rA, far = (ratio * A_all).detach().abs(), (e.exp() - 1).detach().abs()
    off = (rA + klw * far) * lp_off * 2 + 16 * U * (rA + klw * (e.abs() + kl).detach())
    _within("loss", got, loss, (off * w).sum() + 2 * U * loss.abs())
    kl_off = far * lp_off * 2 + 16 * U * (e.abs() + kl).detach()
    want = torch.stack([(kl * w).sum(), (clipped * w).sum()])
    _within("means", means, want, torch.stack([(kl_off * w).sum(), 8 * U * (w.sum())]) + 2 * U * want.abs())
    loss.backward()
    got.backward()
    c = (rA + klw * far) * w
    c_off = (rA + klw * (1 + far)) * w * (2 * lp_off + 16 * U)
    _grad_within("grad", xr.grad, leaf.grad, p, c, c_off, E, dtype, tau)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_with_banned_tokens_and_far_offsets(dtype):
    """-inf logits have probability zero and no gradient; an offset of all logits changes nothing but their own rounding."""
    x, ids, _, _ = _case(2, 4, 3001, dtype, 5)
    x[:, :, 100:2900] = float("-inf")
    ids[:] = 7
    x[1] = (x[1].float() + 900.0).to(dtype)
    leaf, lp, counted, E, p = _lp64(x, ids, None)
    xr = x.clone().requires_grad_(True)
    got = rwkv_kernel.cross_entropy(xr, ids)
    loss = -lp.mean()
    _within("loss", got, loss, (E + 4 * U * lp.abs()).mean() + 2 * U * loss.abs())
    loss.backward()
    got.backward()
    c = torch.full(lp.shape, 1.0 / 8).double()
    _grad_within("grad", xr.grad, torch.nan_to_num(leaf.grad), p, c, 4 * U * c, E, dtype)
    assert bool((xr.grad[:, :, 100:2900] == 0).all())


@pytest.mark.parametrize("temperature", [0.5, 0.7, 0.8, 1.0, 1.1, 1.3, 2.0, 3.3, 1.0 / 1.44269504])
def test_banned_tokens_at_any_temperature(temperature):
    x, ids, _, _ = _case(1, 2, 300, torch.float32, 16)
    x[:, :, 40:290] = float("-inf")
    ids[:] = 3
    leaf, lp, counted, E, p = _lp64(x, ids, None, float(torch.tensor(temperature)))
    xr = x.clone().requires_grad_(True)
    got = rwkv_kernel.token_logprobs(xr, ids, temperature=temperature)
    _within("lp", got, lp, E + 4 * U * lp.abs())
    lp.sum().backward()
    got.sum().backward()
    c = torch.ones(lp.shape).double()
    _grad_within("grad", xr.grad, torch.nan_to_num(leaf.grad), p, c, 4 * U * c / temperature, E, torch.float32, temperature)


def test_the_wrong_shows():
    """NaN or +inf in a row that counts, an id beyond the vocabulary and a row of nothing but -inf give NaN there and nowhere else; a banned
    token that stands there gives a loss of +inf."""
    V = 2500
    for spoil, ids_of in ((lambda r: r.fill_(float("-inf")), 3), (lambda r: r[9:10].fill_(float("nan")), 3), (lambda r: r[V - 1:].fill_(float("inf")), 3), (lambda r: None, V + 5), (lambda r: None, 2 ** 40)):
        x, ids, _, _ = _case(1, 3, V, torch.bfloat16, 6)
        spoil(x[0, 1])
        ids[0, 1] = ids_of
        xr = x.clone().requires_grad_(True)
        lp = rwkv_kernel.token_logprobs(xr, ids)
        assert torch.isnan(lp).tolist() == [[False, True, False]]
        lp.sum().backward()
        assert bool(torch.isnan(xr.grad[0, 1]).any()) and bool(torch.isfinite(xr.grad[0, [0, 2]]).all())
        assert bool(torch.isnan(rwkv_kernel.cross_entropy(x, ids)))
    x, ids, _, _ = _case(1, 3, V, torch.bfloat16, 6)
    ids[0, 1] = 8
    x[0, 1, 8] = float("-inf")
    assert float(rwkv_kernel.cross_entropy(x, ids)) == float("inf")


def test_no_counted_token_is_a_loss_of_zero():
    x, ids, mask, _ = _case(2, 3, 100, torch.bfloat16, 8)
    x.fill_(float("nan"))
    mask[:] = False
    for call in (lambda v: rwkv_kernel.cross_entropy(v, ids, mask), lambda v: rwkv_kernel.policy_loss(v, ids, mask, None, torch.ones(2).cuda())[0],
                 lambda v: rwkv_kernel.policy_loss(v, ids, mask, None, torch.ones(2).cuda(), reduction="mean_of_texts")[0]):
        xr = x.clone().requires_grad_(True)
        loss = call(xr)
        loss.backward()
        assert float(loss) == 0.0 and bool((xr.grad == 0).all())
    xr = x.clone().requires_grad_(True)
    loss, s = rwkv_kernel.preference_loss(xr, ids, mask) if x.shape[0] % 2 == 0 else None
    loss.backward()
    assert abs(float(loss) - math.log(2.0)) < 1e-6 and s.tolist() == [0.0, 0.0] and bool((xr.grad == 0).all())


def test_no_tokens_at_all():
    x = torch.zeros(2, 0, 50, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    ids = torch.zeros(2, 0, dtype=torch.int64, device="cuda")
    loss = rwkv_kernel.cross_entropy(x, ids)
    loss.backward()
    assert float(loss) == 0.0 and x.grad.shape == x.shape and rwkv_kernel.token_logprobs(x, ids).shape == (2, 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strided_logits(dtype):
    """A slice of a longer sequence, rows off any alignment, a transposed batch, broadcast rows and a vocabulary that is not the last stride."""
    g = torch.Generator().manual_seed(3)
    whole = torch.randn(3, 8, 1031, generator=g).to(dtype).cuda()
    ids = torch.randint(0, 900, (3, 5), generator=g).cuda()
    views = [whole[:, 2:7, 1:1000], whole[:, 2:7, 3:1030], whole.transpose(0, 1)[:3, :, :].transpose(1, 2)[:, :1000, :].transpose(1, 2)[:, :3].repeat(1, 2, 1)[:, :5],
             whole[:1, 2:7, :1003].expand(3, 5, 1003), whole[:, :1, :1003].expand(3, 5, 1003), whole[:, 1:6].transpose(1, 2).contiguous().transpose(1, 2)]
    for v in views:
        assert v.shape[:2] == (3, 5)
        ref, lp, counted, E, p = _lp64(v, ids, None)
        (-lp.mean()).backward()
        leaf = v.detach()
        leaf.requires_grad_(True)
        rwkv_kernel.cross_entropy(leaf, ids).backward()
        c = torch.full(lp.shape, 1.0 / 15).double()
        _grad_within("grad", leaf.grad, ref.grad, p, c, 4 * U * c, E, dtype)
        _within("lp", rwkv_kernel.token_logprobs(v, ids), lp, E + 2 * U * lp.abs())
    # through autograd's own views: every element of the base gets its gradient
    base = whole.clone().requires_grad_(True)
    rwkv_kernel.cross_entropy(base[:, 2:7, 1:1000], ids).backward()
    inner = whole[:, 2:7, 1:1000].detach().requires_grad_(True)
    rwkv_kernel.cross_entropy(inner, ids).backward()
    part = torch.zeros_like(base.grad)
    part[:, 2:7, 1:1000] = inner.grad
    assert torch.equal(base.grad, part)


@pytest.mark.parametrize("dtype", DTYPES)
def test_outputs_stay_inside(dtype):
    """Nothing is written before or behind the gradient's rows: they lie in memory whose surroundings hold a known value (the C entry)."""
    from rwkv_kernel import _native
    lib, code = _native.load(), {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}[dtype]
    B, T, V, room = 2, 3, 4099, 1024
    x, ids, mask, _ = _case(B, T, V, dtype, 9)
    for shift in range(0, 9):
        grad = torch.full((room + B * T * V + room,), 7.0, dtype=dtype, device="cuda")
        at = grad[room + shift:]
        stats, coef, loss = (torch.empty(n, device="cuda") for n in (2 * B * T, B * T, 1))
        n = lib.wkv6_loss_workspace_bytes(B, T)
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        _native.check(lib.wkv6_cross_entropy(torch.cuda.current_stream().cuda_stream, code, B, T, V, x.data_ptr(), T * V, V, ids.data_ptr(), mask.data_ptr(), 1,
                                             loss.data_ptr(), stats.data_ptr(), coef.data_ptr(), at.data_ptr(), ws.data_ptr(), n))
        xr = x.clone().requires_grad_(True)
        rwkv_kernel.cross_entropy(xr, ids, mask).backward(torch.tensor(1.0).cuda())
        assert torch.equal(at[:B * T * V], xr.grad.view(-1))
        assert bool((grad[:room + shift] == 7).all()) and bool((at[B * T * V:] == 7).all())


def test_gradient_by_differences():
    """The policy loss's gradient against central differences of the loss, fp32 logits: steps of 2^-5 in a logit, errors of third order."""
    x, ids, mask, g = _case(2, 3, 12, torch.float32, 11, std=1.0)
    mask[:] = True
    lp = rwkv_kernel.token_logprobs(x, ids)
    old, ref, A = lp - 0.05, lp + 0.1 * torch.randn(2, 3, generator=g).cuda(), torch.randn(2, generator=g).cuda()
    f = lambda v: rwkv_kernel.policy_loss(v, ids, mask, old, A, ref_logps=ref, kl_weight=0.3)[0]  # noqa: E731
    xr = x.clone().requires_grad_(True)
    f(xr).backward()
    h = 2.0 ** -5
    for b, t, j in ((0, 0, 0), (0, 2, 5), (1, 1, 11), (1, 0, int(ids[1, 0]))):
        up, down = x.clone(), x.clone()
        up[b, t, j] += h
        down[b, t, j] -= h
        with torch.no_grad():
            slope = (float(f(up)) - float(f(down))) / (2 * h)
        # |f'''| <= about 4 max|A| / 6 tokens; the loss itself is off by some 2^-22
        assert abs(slope - float(xr.grad[b, t, j])) <= 4 * 2.5 / 6 * h * h / 6 + 2.0 ** -22 / h


def test_backward_twice_and_in_parts():
    """A graph's second backward gives the first one's gradient anew; gradients add up; one that arrives scaled is scaled."""
    for dtype in DTYPES:
        x, ids, mask, _ = _case(2, 5, 700, dtype, 12)
        xr = x.clone().requires_grad_(True)
        loss = rwkv_kernel.cross_entropy(xr, ids, mask)
        first, = torch.autograd.grad(loss, xr, retain_graph=True)
        kept = first.clone()
        first.zero_()                         # what was handed out is the caller's
        second, = torch.autograd.grad(loss, xr, retain_graph=True)
        assert torch.equal(second, kept)
        half, = torch.autograd.grad(loss * 0.5, xr, retain_graph=True)
        if dtype != torch.float16:            # (a power of two: exact but for fp16's subnormal numbers)
            assert torch.equal(half, kept * 0.5)
        with pytest.raises(RuntimeError):
            xr2 = x.clone().requires_grad_(True)
            y = xr2 * 1
            loss = rwkv_kernel.cross_entropy(y, ids, mask)
            y.mul_(2)
            loss.backward()


def test_on_another_stream_and_in_a_graph():
    """Forward and backward captured together, replayed with other logits between eager calls, each time against the eager result."""
    x, ids, mask, g = _case(4, 6, 3000, torch.bfloat16, 13)
    old = rwkv_kernel.token_logprobs(x, ids).clone()
    A = torch.randn(4, generator=g).cuda()
    calls = [lambda v: rwkv_kernel.cross_entropy(v, ids, mask), lambda v: rwkv_kernel.policy_loss(v, ids, mask, old, A, ref_logps=old, kl_weight=0.1)[0],
             lambda v: rwkv_kernel.preference_loss(v, ids, mask, ref_logps=old.sum(1))[0], lambda v: rwkv_kernel.token_logprobs(v, ids, mask).sum()]
    for call in calls:
        static = x.clone().requires_grad_(True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = torch.autograd.grad(call(static), static)[0]
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        assert torch.equal(eager, torch.autograd.grad(call(static), static)[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = call(static)
            grad, = torch.autograd.grad(loss, static)
        for seed in range(4):
            fresh = _case(4, 6, 3000, torch.bfloat16, 20 + seed)[0]
            with torch.no_grad():
                static.copy_(fresh)
            graph.replay()
            torch.cuda.synchronize()
            v = fresh.clone().requires_grad_(True)
            want = call(v)
            want_grad, = torch.autograd.grad(want, v)
            assert torch.equal(loss, want.detach()) and torch.equal(grad, want_grad), seed


def test_many_rows_and_far_rows():
    """More tokens than one counting workgroup, and rows beyond 2^31 elements."""
    x, ids, mask, _ = _case(1, 70000, 24, torch.float32, 14)
    loss = rwkv_kernel.cross_entropy(x, ids, mask)
    _, lp, counted, E, _ = _lp64(x, ids, mask)
    _within("loss", loss, -lp.sum() / counted.sum(), (E + 4 * U * lp.abs()).mean() * 2 + 4 * U * lp.abs().mean())
    V, T = 65536, 33000                       # 2.16e9 elements
    big = torch.zeros(1, T, V, dtype=torch.bfloat16, device="cuda")
    ids = torch.full((1, T), -1, dtype=torch.int64, device="cuda")
    last = torch.randn(V, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    big[0, T - 1] = last
    ids[0, T - 1] = 12345
    big.requires_grad_(True)
    loss = rwkv_kernel.cross_entropy(big, ids)
    loss.backward()
    v = last.clone()[None].requires_grad_(True)
    want = rwkv_kernel.cross_entropy(v, ids[0, T - 1:])
    want.backward()
    assert torch.equal(loss.detach(), want.detach()) and torch.equal(big.grad[0, T - 1], v.grad[0]) and bool((big.grad[0, T - 2] == 0).all())


def test_results_do_not_change_from_run_to_run():
    x, ids, mask, _ = _case(8, 50, 9000, torch.bfloat16, 15)
    runs = []
    for _ in range(3):
        v = x.clone().requires_grad_(True)
        loss, s = rwkv_kernel.preference_loss(v, ids, mask)
        loss.backward()
        runs.append((loss.detach(), s, v.grad))
    for other in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(runs[0], other))


def test_what_stands_beside_the_logits_gets_no_gradient():
    """Log probabilities of other models and advantages may carry a graph: nothing flows into it, and without logits that want one there is no gradient."""
    x, ids, mask, g = _case(4, 5, 300, torch.float32, 17)
    old = rwkv_kernel.token_logprobs(x, ids).requires_grad_(True)
    ref = (old * 1.5)
    A = torch.randn(4, generator=g).cuda().requires_grad_(True)
    for leaf in (x.clone().requires_grad_(True), x):
        loss = rwkv_kernel.policy_loss(leaf, ids, mask, old, A, ref_logps=ref, kl_weight=0.1)[0] + rwkv_kernel.preference_loss(leaf, ids, mask, ref.sum(1))[0]
        assert loss.requires_grad == leaf.requires_grad
        if leaf.requires_grad:
            loss.backward()
            assert leaf.grad is not None
    assert old.grad is None and A.grad is None


def test_more_rows_than_a_launch_counts_threads():
    """2^32 threads and more: rows of 256 threads each, all the same one in memory."""
    rows, V = (1 << 24) + 5, 4104
    row = torch.randn(V, generator=torch.Generator().manual_seed(18)).to(torch.bfloat16).cuda()
    ids = torch.full((1, rows), -1, dtype=torch.int64, device="cuda")
    ids[0, ::4096] = 3
    ids[0, rows - 1] = 11
    lp = rwkv_kernel.token_logprobs(row.expand(1, rows, V), ids)
    want = rwkv_kernel.token_logprobs(row[None, None].expand(1, 2, V), torch.tensor([[3, 11]]).cuda())
    assert bool((lp[0, :rows - 1:4096] == want[0, 0]).all()) and bool(lp[0, rows - 1] == want[0, 1])
    assert int((lp != 0).sum()) == (rows - 2) // 4096 + 2


@pytest.mark.parametrize("reduction", ["mean", "mean_of_texts"])
def test_many_short_texts(reduction):
    """More texts than counting workgroups, and more rows than one workgroup adds up."""
    B, T, V = 70000, 2, 40
    x, ids, mask, g = _case(B, T, V, torch.float32, 19)
    A = torch.randn(B, generator=g).cuda()
    got, got_lp, _ = rwkv_kernel.policy_loss(x, ids, mask, None, A, reduction=reduction)
    _, lp, counted, E, _ = _lp64(x, ids, mask)
    n = counted.sum(1, keepdim=True).double()
    w = counted / (n.clamp(min=1) * (n > 0).sum() if reduction == "mean_of_texts" else counted.sum())
    want = -(A.cpu().double()[:, None] * w).sum()
    # (the ratio is 1: a term is the advantage times its weight, two roundings)
    _within("loss", got, want, 4 * U * (A.cpu().double().abs()[:, None] * w).sum())
    _within("lp", got_lp, lp, E + 2 * U * lp.abs())
    loss, s = rwkv_kernel.preference_loss(x, ids, mask)
    want, s64, d = _preference(lp, counted, None, 0.1, "sigmoid", 0.0, False)
    off = (E * counted).sum(1)
    _within("preference", loss, want, 0.1 * (off[:B // 2] + off[B // 2:]).mean() + 2 * U * want.abs())


def test_two_streams_at_once():
    """The same logits on two streams, and calls of different sizes side by side: each as if alone."""
    cases = [_case(3, 40, V, torch.bfloat16, V) for V in (3000, 40000)]
    alone = []
    for x, ids, mask, _ in cases:
        v = x.clone().requires_grad_(True)
        loss = rwkv_kernel.cross_entropy(v, ids, mask)
        alone.append((loss.detach(), torch.autograd.grad(loss, v)[0]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for i, s in enumerate(streams):
        x, ids, mask, _ = cases[i % 2]
        with torch.cuda.stream(s):
            for _ in range(3):
                v = x.clone().requires_grad_(True)
                loss = rwkv_kernel.cross_entropy(v, ids, mask)
                got.append((i % 2, loss.detach(), torch.autograd.grad(loss, v)[0]))
    torch.cuda.synchronize()
    for which, loss, grad in got:
        assert torch.equal(loss, alone[which][0]) and torch.equal(grad, alone[which][1])


def test_a_backward_captured_after_an_eager_forward():
    """Its replays give the gradient anew each time, whatever became of the last one, and an eager backward behind them too."""
    x, ids, mask, _ = _case(2, 9, 1500, torch.bfloat16, 20)
    y = x.clone().requires_grad_(True)   # (a leaf that only the capturing stream has seen: torch's engine would make any other stream of the graph wait
    side = torch.cuda.Stream()           # for the captured gradient, and so a part of the capture that nothing joins again)
    side.wait_stream(torch.cuda.current_stream())
    up = torch.ones((), device="cuda")
    with torch.cuda.stream(side):
        loss = rwkv_kernel.cross_entropy(y, ids, mask)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grad, = torch.autograd.grad(loss, y, up, retain_graph=True)
    torch.cuda.synchronize()
    w = x.clone().requires_grad_(True)
    rwkv_kernel.cross_entropy(w, ids, mask).backward()
    for scale in (1.0, 1.0, 0.5, 1.0):
        up.fill_(scale)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(grad, w.grad * scale)
        grad.fill_(float("nan"))
        torch.cuda.synchronize()
    up.fill_(1.0)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        eager, = torch.autograd.grad(loss, y, up)
    torch.cuda.synchronize()
    assert torch.equal(eager, w.grad)


def test_refusals_on_the_gpu():
    x, ids, mask, _ = _case(2, 3, 40, torch.bfloat16, 22)
    A = torch.ones(2, device="cuda")
    lp = torch.zeros(2, 3, device="cuda")
    k = rwkv_kernel
    bad_rows = [(x.double(), ids, mask), (x[0, 0], ids[0, 0], None), (x, ids.int(), mask), (x, ids[:, :2], mask), (x, ids.cpu(), mask), (x, ids, mask.float()),
                (x, ids, mask[:1]), (x, ids, mask.cpu()), (x[:, :, :0], ids, mask), (x.cpu(), ids, mask)]
    for rows in bad_rows:
        for call in (lambda r: k.cross_entropy(*r), lambda r: k.token_logprobs(*r), lambda r: k.preference_loss(*r), lambda r: k.policy_loss(*r, lp, A)):
            with pytest.raises(AssertionError):
                call(rows)
    for call in (lambda: k.cross_entropy(x, ids, reduction="none"), lambda: k.token_logprobs(x, ids, temperature=0.0), lambda: k.preference_loss(x[:1], ids[:1]),
                 lambda: k.preference_loss(x, ids, kind="other"), lambda: k.preference_loss(x, ids, beta=0.0), lambda: k.preference_loss(x, ids, label_smoothing=0.5),
                 lambda: k.preference_loss(x, ids, kind="hinge", label_smoothing=0.1), lambda: k.preference_loss(x, ids, ref_logps=lp),
                 lambda: k.preference_loss(x[0], ids[0]), lambda: k.preference_loss(x[:, :0], ids[:, :0]), lambda: k.policy_loss(x[0], ids[0], None, lp[0], A),
                 lambda: k.policy_loss(x, ids, mask, lp[:, :2], A), lambda: k.policy_loss(x, ids, mask, lp.cpu(), A), lambda: k.policy_loss(x, ids, mask, lp, A[:1]),
                 lambda: k.policy_loss(x, ids, mask, lp, A, ref_logps=lp[0]), lambda: k.policy_loss(x, ids, mask, lp, A, reduction="sum"),
                 lambda: k.policy_loss(x, ids, mask, lp, A, clip_low=-0.1), lambda: k.policy_loss(x, ids, mask, lp, A, kl_weight=-1.0),
                 lambda: k.policy_loss(x, ids, mask, lp, A, temperature=0.0), lambda: k.policy_loss(x[:, :0], ids[:, :0], None, lp[:, :0], A)):
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError, match="wkv6"):     # 1 / temperature is no number of fp32
        k.token_logprobs(x, ids, temperature=1e-40)


def test_other_types_beside_the_logits():
    """Masks in bytes, log probabilities and advantages in other types or not contiguous: as their fp32 copies."""
    x, ids, mask, g = _case(4, 6, 500, torch.float32, 23)
    old = rwkv_kernel.token_logprobs(x, ids) - 0.05
    ref, A = old + 0.1, torch.randn(4, 6, generator=g).cuda()
    want = rwkv_kernel.policy_loss(x, ids, mask, old, A, ref_logps=ref, kl_weight=0.1)
    wide = lambda t: t.t().contiguous().t()  # noqa: E731
    for got in (rwkv_kernel.policy_loss(x, wide(ids), wide(mask).to(torch.uint8) * 7, old.double(), wide(A), ref_logps=wide(ref), kl_weight=0.1),
                rwkv_kernel.policy_loss(wide(x.view(4, -1)).view(4, 6, 500), ids, mask, wide(old), A.double(), ref_logps=ref, kl_weight=0.1)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def _banned_case(dtype, seed, B=2, T=4, V=300):
    """Logits of which the token that stands at (0, 1) has -inf, with softmax and E of each row in 64 bits."""
    x, ids, _, g = _case(B, T, V, dtype, seed)
    ids[0, 1] = 8
    x[0, 1, 8] = float("-inf")
    _, lp, _, E, p = _lp64(x, ids, None)
    return x, ids, lp.detach(), E, p, g


def _rows_of(c, ids, p):
    """c (1[id] - p) of each row, in 64 bits."""
    return c[..., None] * (torch.zeros_like(p).scatter_(-1, ids.cpu()[..., None], 1.0) - p)


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_of_a_banned_token_without_old_logps(dtype):
    """The ratio is 1 wherever the log probability is a number or -inf: loss and gradient are the advantages'."""
    x, ids, lp, E, p, g = _banned_case(dtype, 41)
    A = torch.randn(2, 4, generator=g)
    xr = x.clone().requires_grad_(True)
    loss, got_lp, means = rwkv_kernel.policy_loss(xr, ids, None, None, A.cuda())
    want = -A.double().mean()
    _within("loss", loss, want, 4 * U * A.double().abs().mean())
    assert float(got_lp[0, 1]) == float("-inf") and means.tolist() == [0.0, 0.0]
    loss.backward()
    c = -A.double() / 8
    _grad_within("grad", xr.grad, _rows_of(c, ids, p), p, c, 4 * U * c.abs(), E, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_kl_that_is_infinite(dtype):
    """A KL term beyond fp32's range, or of a banned token, is infinite and no NaN; with a weight of 0 it is only reported, and loss and
    gradient are those without a reference model, bit for bit."""
    x, ids, lp, E, p, g = _banned_case(dtype, 42)
    A = torch.randn(2, generator=g).cuda()
    ref = torch.where(torch.isfinite(lp), lp, torch.full_like(lp, -3.0)).float().cuda()   # (a number where lp is -inf: exp(e) is infinite there)
    far = torch.zeros_like(ref)
    far[1, 2] = 200.0
    for r, spoilt in ((ref, (0, 1)), (ref + far, (1, 2))):
        ids_r = ids.clone()
        if spoilt == (1, 2):
            ids_r[0, 1] = -1                               # (the banned token does not count)
        runs = []
        for kw in (dict(), dict(ref_logps=r, kl_weight=0.0), dict(ref_logps=r, kl_weight=0.1)):
            xr = x.clone().requires_grad_(True)
            loss, _, means = rwkv_kernel.policy_loss(xr, ids_r, None, None, A, **kw)
            loss.backward()
            runs.append((loss.detach(), xr.grad, means))
        assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1]) and bool(torch.isfinite(runs[0][1]).all())
        assert runs[0][2].tolist() == [0.0, 0.0] and runs[1][2].tolist() == [float("inf"), 0.0]
        assert float(runs[2][0]) == float("inf") and float(runs[2][2][0]) == float("inf")
        others = torch.ones(2, 4, dtype=torch.bool)
        others[spoilt] = False
        assert bool(torch.isfinite(runs[2][1][others.cuda()]).all()) and not bool(torch.isfinite(runs[2][1][spoilt]).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_policy_ratio_beyond_the_range_with_an_advantage_of_zero(dtype):
    """exp(lp - old) of 100 is beyond fp32: times an advantage of 0 it is 0, as the formula's; of a positive one it is clipped, of a negative one infinite."""
    x, ids, _, g = _case(2, 3, 200, dtype, 43)
    _, lp, _, E, p = _lp64(x, ids, None)
    old = lp.detach().float().cuda()
    old[0, 1] -= 100.0
    A = torch.tensor([[1.0, 0.0, -0.5], [0.25, 2.0, -1.0]])
    xr = x.clone().requires_grad_(True)
    loss, _, means = rwkv_kernel.policy_loss(xr, ids, None, old, A.cuda())
    loss.backward()
    # (elsewhere the ratio is 1 but for what lp and its rounding are off by)
    off = E + 8 * U * (1 + lp.detach().abs())
    _within("loss", loss, -A.double().mean(), (A.double().abs() * off).mean() * 2)
    c = -A.double() / 6
    _grad_within("grad", xr.grad, _rows_of(c, ids, p), p, c, 2 * c.abs() * off, E, dtype)
    assert bool((xr.grad[0, 1] == 0).all()) and means.tolist() == [0.0, 0.0]
    for a, want in ((0.5, False), (-0.5, True)):
        A[0, 1] = a
        loss = rwkv_kernel.policy_loss(x, ids, None, old, A.cuda())[0]
        assert bool(torch.isinf(loss)) == want and not bool(torch.isnan(loss))


@pytest.mark.parametrize("kind", ["hinge", "sigmoid"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_preference_for_a_text_with_a_banned_token(dtype, kind):
    """A chosen text of probability zero: the loss is infinite, and its slope -beta, as the formula's."""
    x, ids, lp, E, p, _ = _banned_case(dtype, 44)
    beta = 0.3
    xr = x.clone().requires_grad_(True)
    loss, s = rwkv_kernel.preference_loss(xr, ids, beta=beta, kind=kind)
    assert float(loss) == float("inf") and float(s[0]) == float("-inf") and math.isfinite(float(s[1]))
    loss.backward()
    c = torch.tensor([-beta, beta]).double()[:, None].expand(2, 4)
    _grad_within("grad", xr.grad, _rows_of(c, ids, p), p, c, 4 * U * c.abs(), E, dtype)
    # rejected instead, it costs nothing
    back = torch.tensor([1, 0]).cuda()
    xr = x[back].clone().requires_grad_(True)
    loss, _ = rwkv_kernel.preference_loss(xr, ids[back], beta=beta, kind=kind)
    loss.backward()
    assert float(loss) == 0.0 and bool((xr.grad == 0).all())


@pytest.mark.parametrize("temperature", [0.7, 0.9, 1.3, 3.3])
def test_temperature_has_no_error_of_its_own(temperature):
    """The log probability is divided by the temperature (as an fp32 number) in 64 bits.  Rows of two logits, 0 and -d with d of 60 and more: the sum of
    exponentials is 1 to the last bit (exp(-60 / 3.3) < 2^-26), so lp is -d / temperature, once rounded: no rounding of 1 / temperature, which has the same sign in each token, adds up
    over a text.  (Half of a last place, 2^-24 of the value at most, and 2^-50 for the arithmetic in 64 bits; at 3.3 what the sum of exponentials leaves out.)"""
    tau = float(torch.tensor(temperature))
    d = torch.linspace(60, 400, 1999)
    x = torch.stack([torch.zeros_like(d), -d], 1)[None].cuda()
    ids = torch.ones(1, d.numel(), dtype=torch.int64, device="cuda")
    want = -d.double() / tau - torch.log1p(torch.exp(-d.double() / tau))
    with torch.no_grad():
        for lp in (rwkv_kernel.token_logprobs(x, ids, temperature=temperature),
                   rwkv_kernel.policy_loss(x, ids, None, None, torch.ones(1).cuda(), temperature=temperature)[1]):
            off = lp.cpu().double()[0] - want
            assert bool((off.abs() <= want.abs() * 2.0 ** -24 * (1 + 2.0 ** -20) + torch.exp(-d.double() / tau)).all()), float((off / want).abs().max())
            # and the errors' mean is that of roundings, each at most 2^-24 of its value either way: 1999 of them, nine standard deviations of their mean
            assert abs(float((off / want).mean())) <= 9 * 2.0 ** -24 / math.sqrt(3 * d.numel())


@pytest.mark.parametrize("temperature", [1e-30, 1e20, 1e29, 3e36, 1e38, 3.4e38])
def test_banned_tokens_at_temperatures_at_the_ends_of_the_range(temperature):
    """All tokens that are not banned are as likely as each other, or the largest logit is all there is."""
    x, ids, _, _ = _case(1, 2, 300, torch.float32, 48)
    x[:, :, 40:290] = float("-inf")
    ids[:] = x.argmax(-1)
    xr = x.clone().requires_grad_(True)
    lp = rwkv_kernel.token_logprobs(xr, ids, temperature=temperature)
    lp.sum().backward()
    want = 0.0 if temperature < 1 else -math.log(50)
    # (of 50 equal terms the sum is exact; log and its rounding)
    assert float((lp.detach().double() - want).abs().max()) <= 2 * U * abs(want)
    assert bool((xr.grad[:, :, 40:290] == 0).all()) and bool(torch.isfinite(xr.grad).all())


def test_no_second_derivative():
    """A gradient taken with create_graph has the plain one's values, and whoever differentiates it is told that there is nothing, instead of losing a term."""
    x, ids, mask, g = _case(2, 5, 300, torch.float32, 45)
    old = rwkv_kernel.token_logprobs(x, ids)
    A = torch.randn(2, generator=g).cuda()
    w = torch.randn(2, 5, generator=g).cuda()
    for call in (lambda v: (rwkv_kernel.token_logprobs(v, ids, mask) * w).sum(), lambda v: rwkv_kernel.cross_entropy(v, ids, mask),
                 lambda v: rwkv_kernel.preference_loss(v, ids, mask, old.sum(1))[0], lambda v: rwkv_kernel.policy_loss(v, ids, mask, old, A, ref_logps=old + 0.1, kl_weight=0.1)[0]):
        leaf = x.clone().requires_grad_(True)
        logits = leaf * 1.0                                # (a leaf, and logits that something made)
        plain, = torch.autograd.grad(call(logits), leaf, retain_graph=True)
        for at in (leaf, logits):
            loss = call(logits)
            grad, = torch.autograd.grad(loss, at, create_graph=True)
            assert torch.equal(grad.detach(), plain) and grad.requires_grad
            with pytest.raises(RuntimeError, match="second derivative"):
                (loss + grad.square().sum()).backward()
        leaf.grad = None
        call(leaf * 1.0).backward()
        assert torch.equal(leaf.grad, plain)


@pytest.mark.parametrize("rows,V,dtype", [(4500, 4100, torch.bfloat16), (4500, 4100, torch.float32), (2500, 20000, torch.bfloat16), (2500, 20000, torch.float32),
                                          (17000, 250, torch.bfloat16), (17000, 1000, torch.float32)])
def test_many_rows_under_a_loss_that_is_scaled(rows, V, dtype):
    """What the forward wrote for an arriving gradient of 1 is written anew for another one, in every row: more of them than the workgroups that look at what arrived (2048,
    of one row, of a piece of one, or of four short ones) take at once.  0.5 and 2 are powers of two: exact."""
    x, ids, mask, g = _case(4, rows // 4, V, dtype, rows + V, std=1.0)
    old = rwkv_kernel.token_logprobs(x, ids) - 0.05
    A = torch.randn(4, generator=g).cuda()
    for call in (lambda v: rwkv_kernel.cross_entropy(v, ids, mask, reduction="sum"), lambda v: rwkv_kernel.policy_loss(v, ids, mask, old, A, ref_logps=old, kl_weight=0.1)[0]):
        grads = []
        for up in (1.0, 0.5, 2.0):
            v = x.clone().requires_grad_(True)
            grads.append(torch.autograd.grad(call(v), v, torch.tensor(up).cuda())[0])
        assert torch.equal(grads[1] * 2, grads[0]) and torch.equal(grads[2], grads[0] * 2)
        assert bool((grads[0][mask].abs().amax(-1) > 0).all()) and bool((grads[0][~mask] == 0).all())


@pytest.mark.parametrize("T,V,dtype", [(1400, 65536, torch.bfloat16), (1300, 70001, torch.float16), (700, 65537, torch.float32), (90000, 1003, torch.bfloat16)])
def test_gradients_past_the_caches(T, V, dtype):
    """A gradient of 160 MiB and more is stored in another way; its rows are those of calls on parts that stay below."""
    assert T * V * torch.finfo(dtype).bits // 8 >= 160 << 20
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.empty(1, T, V, dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=gen)
    ids = torch.randint(0, V, (1, T), generator=gen, device="cuda")
    mask = torch.rand(1, T, generator=gen, device="cuda") < 0.8
    w = torch.randn(1, T, generator=gen, device="cuda")

    def logprobs(a, b):
        v = x[:, a:b].detach().requires_grad_(True)
        lp = rwkv_kernel.token_logprobs(v, ids[:, a:b], mask[:, a:b], temperature=0.9)
        return lp.detach(), torch.autograd.grad(lp, v, w[:, a:b])[0]

    def loss(a, b):   # (a forward that writes the gradient too, or leaves it to the backward: fp16)
        v = x[:, a:b].detach().requires_grad_(True)
        return torch.autograd.grad(rwkv_kernel.cross_entropy(v, ids[:, a:b], mask[:, a:b], reduction="sum"), v)

    for call in (logprobs, loss):
        whole, step = call(0, T), (T + 2) // 3
        for a in range(0, T, step):
            b = min(T, a + step)
            for got, part in zip(whole, call(a, b)):
                assert torch.equal(got[:, a:b], part), (a, b)


def test_preference_gradients_past_the_caches():
    """Two texts of 96 MiB each: the gradient's rows are those that their halves have, of a loss whose slope is the same (the sigmoid's at d = 0, as both texts are one)."""
    T, V = 768, 65536
    gen = torch.Generator(device="cuda").manual_seed(46)
    text = torch.empty(1, T, V, dtype=torch.bfloat16, device="cuda").normal_(0.0, 2.0, generator=gen)
    ids = torch.randint(0, V, (1, T), generator=gen, device="cuda")

    def grad(a, b):
        v = text[:, a:b].repeat(2, 1, 1).requires_grad_(True)
        loss, _ = rwkv_kernel.preference_loss(v, ids[:, a:b].repeat(2, 1), beta=0.25)
        return torch.autograd.grad(loss, v)[0]

    whole = grad(0, T)
    assert whole.numel() * 2 >= 160 << 20
    for a in range(0, T, T // 2):
        assert torch.equal(whole[:, a:a + T // 2], grad(a, a + T // 2))
    assert torch.equal(whole[0], -whole[1]) and bool((whole[0].abs().amax(-1) > 0).all())


def test_other_ways_to_run_them():
    """Inference mode, recomputation, and saved tensors kept on the host: as a plain call."""
    from torch.utils.checkpoint import checkpoint
    whole = torch.randn(4, 9, 400, generator=torch.Generator().manual_seed(49)).cuda()
    _, ids, mask, g = _case(4, 6, 390, torch.float32, 49)
    view = whole[:, 2:8, 3:393]                            # (rows apart: what comes back from the host may lie otherwise)
    old, A = rwkv_kernel.token_logprobs(view, ids) - 0.05, torch.randn(4, generator=g).cuda()
    for call in (lambda v: rwkv_kernel.cross_entropy(v, ids, mask), lambda v: rwkv_kernel.token_logprobs(v, ids, mask).sum(),
                 lambda v: rwkv_kernel.preference_loss(v, ids, mask, old.sum(1))[0], lambda v: rwkv_kernel.policy_loss(v, ids, mask, old, A, ref_logps=old, kl_weight=0.1)[0]):
        leaf = view.detach().requires_grad_(True)
        want = call(leaf)
        want_grad, = torch.autograd.grad(want, leaf)
        with torch.inference_mode():
            assert torch.equal(call(view), want) and torch.equal(call(whole.clone()[:, 2:8, 3:393]), want)   # (rows that begin where they did: the sums' order goes by that)
        with torch.autograd.graph.save_on_cpu():
            loss = call(leaf)
        assert torch.equal(torch.autograd.grad(loss, leaf)[0], want_grad)
        loss = checkpoint(call, leaf, use_reentrant=False)
        assert torch.equal(loss, want) and torch.equal(torch.autograd.grad(loss, leaf)[0], want_grad)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_policy_beside_its_own_log_probabilities(dtype):
    """The ratio is 1 and the KL term 0 to the last bit, so that the loss and its gradient are those without either."""
    x, ids, mask, g = _case(3, 7, 1200, dtype, 50)
    A = torch.randn(3, generator=g).cuda()
    xr, same = (x.clone().requires_grad_(True) for _ in range(2))
    plain, lp, _ = rwkv_kernel.policy_loss(xr, ids, mask, None, A, temperature=0.9)
    loss, _, means = rwkv_kernel.policy_loss(same, ids, mask, lp, A, ref_logps=lp, kl_weight=0.5, clip_low=0.0, clip_high=0.0, temperature=0.9)
    plain.backward()
    loss.backward()
    assert torch.equal(loss, plain) and means.tolist() == [0.0, 0.0] and torch.equal(same.grad, xr.grad)
