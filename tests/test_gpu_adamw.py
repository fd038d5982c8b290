"""AdamW (adamw_step, grad_norm, the optimizer) against its formula in float64.

Tolerances, u = 2^-24.  m and v are formed with three roundings each, of g (1 - b) and m b, and g has one of the clipping's product:
6 u of the larger of the terms' magnitudes.  The update lr / c1 m / (sqrt(v) / sqrt(c2) + eps) has some eight roundings, in whose
square root v's error halves, and the difference that forms p one of p and one of p's decay: 16 u |update| + 4 u |p|.  16-bit parameters
are rounded once more, by half their eps."""
import copy
import math

import pytest
import torch

import rwkv_kernel

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
F8 = torch.float8_e4m3fn
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# on either side of a vector, a scale's block, a workgroup's chunk; one element, none
SHAPES = [(1,), (0,), (7,), (255,), (256,), (257,), (16, 16), (33, 129), (4096,), (4097,), (8191,), (3, 5, 1111), (64, 2048), (70001,)]
LR, BETAS, EPS, WD = 3e-3, (0.9, 0.99), 1e-8, 0.1


def _setup(shapes, dtype, bits, master, seed, step=10):
    g = torch.Generator().manual_seed(seed)
    rand = lambda s, std: torch.randn(*s, generator=g) * std  # noqa: E731
    st = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], scales=[] if bits == 8 else None, masters=[] if master else None)
    for s in shapes:
        n = math.prod(s)
        p = rand(s, 0.1)
        st["params"].append(p.to(dtype).cuda())
        if master:
            st["masters"].append(p.cuda())
        st["grads"].append((rand(s, 1.0) * torch.exp(rand(s, 1.5)) * 1e-2).to(dtype).cuda())
        m, r = rand(s, 1e-2), rand(s, 1e-2).abs()
        if bits == 8:
            blocks = (n + 255) // 256
            sc = torch.rand(blocks, 2, generator=g) * 1e-4 + 1e-6
            wide = sc.repeat_interleave(256, 0)[:n]
            st["scales"].append(sc.cuda())
            st["exp_avgs"].append((m.reshape(-1) / wide[:, 0]).clamp(-448, 448).to(F8).reshape(s).cuda())
            st["exp_avg_sqs"].append((r.reshape(-1) / wide[:, 1]).clamp(0, 448).to(F8).reshape(s).cuda())
        else:
            st["exp_avgs"].append(m.cuda())
            st["exp_avg_sqs"].append((r * r).cuda())
    st["step"] = torch.tensor(step, dtype=torch.int64, device="cuda")
    return st


def _wide(x, scales, column):
    """The values of an 8-bit moment, in float64."""
    n = x.numel()
    return x.detach().float().cpu().double().reshape(-1) * scales.cpu().double().repeat_interleave(256, 0)[:n, column]


def _mix(x):
    x = (x ^ (x >> 16)) * 0xBB67AE85 & 0xFFFFFFFF
    x = (x ^ (x >> 15)) * 0x9E3779B9 & 0xFFFFFFFF
    return x ^ (x >> 16)


def _check(before, after, norm, clip, bits, t, lr=LR):
    scale = 1.0 if clip is None or norm <= clip else clip / norm
    c1, c2 = 1 - BETAS[0] ** t, 1 - BETAS[1] ** t
    for j, p0 in enumerate(before["params"]):
        n = p0.numel()
        if n == 0:
            continue
        flat = lambda name: before[name][j].cpu().double().reshape(-1)  # noqa: E731
        g = flat("grads") * scale
        if bits == 8:
            m0, v0 = _wide(before["exp_avgs"][j], before["scales"][j], 0), _wide(before["exp_avg_sqs"][j], before["scales"][j], 1) ** 2
        else:
            m0, v0 = flat("exp_avgs"), flat("exp_avg_sqs")
        m, v = BETAS[0] * m0 + (1 - BETAS[0]) * g, BETAS[1] * v0 + (1 - BETAS[1]) * g * g
        m_off, v_off = 6 * U * (m0.abs() + g.abs()), 6 * U * (v0 + g * g)
        w = flat("masters" if before["masters"] else "params")
        update = lr / c1 * m / ((v / c2).sqrt() + EPS)
        new = w * (1 - lr * WD) - update
        off = 16 * U * update.abs() + lr / c1 * m_off / ((v / c2).sqrt() + EPS) + 4 * U * w.abs() + 2.0 ** -149
        got = after["params"][j].cpu().double().reshape(-1)
        if before["masters"]:
            master = after["masters"][j].cpu()
            assert bool(((master.double().reshape(-1) - new).abs() <= off).all()), j
            assert torch.equal(master.to(p0.dtype), after["params"][j].cpu()), j
        else:
            if p0.dtype != torch.float32:
                off = off + torch.finfo(p0.dtype).eps / 2 * (new.abs() + off) + (2.0 ** -25 if p0.dtype == torch.float16 else 0.0)
            assert bool(((got - new).abs() <= off).all()), (j, float(((got - new).abs() - off).max()))
        if bits == 32:
            assert bool(((after["exp_avgs"][j].cpu().double().reshape(-1) - m).abs() <= m_off).all()), j
            assert bool(((after["exp_avg_sqs"][j].cpu().double().reshape(-1) - v).abs() <= v_off).all()), j
            continue
        # 8 bits: the scales are the largest magnitudes over 448; a value lies within one step of float8 (an eighth of its power of two, 2^-9 at
        # least) of what it stands for, and which neighbour it is follows from the hash
        r, r_off = v.sqrt(), 6 * U * (v0 + g * g) / (2 * v.sqrt()).clamp(min=1e-30) + U * v.sqrt()
        key = _mix((7 * 0x9E3779B9 + t * 0xBB67AE85 + j) & 0xFFFFFFFF)
        h = _mix((torch.arange(n) * 0x9E3779B9 + key) & 0xFFFFFFFF)
        for column, (name, x, x_off, u16) in enumerate((("exp_avgs", m, m_off, h & 0xFFFF), ("exp_avg_sqs", r, r_off, h >> 16))):
            pad = torch.cat([x, x.new_zeros(-n % 256)]).view(-1, 256)
            top = pad.abs().amax(1).clamp(min=2.0 ** -100)
            sc = after["scales"][j][:, column].cpu().double()
            assert bool(((sc * 448 - top).abs() <= 16 * U * top).all()), j
            y, wide = x.abs() / sc.repeat_interleave(256)[:n], after[name][j].cpu().double().reshape(-1)
            assert bool(((wide == 0) | (torch.sign(wide) == torch.sign(x))).all())
            step = torch.exp2(torch.floor(torch.log2(y.clamp(min=2.0 ** -6))) - 3)
            low = torch.floor(y / step)
            up = (y / step - low) * 65536 + u16.double() >= 65536
            want = (low + up) * step
            want = torch.where((want == 0) & (x > 0), torch.tensor(2.0 ** -9).double(), want) if column == 1 else want
            near = ((y / step - low) * 65536 + u16.double() - 65536).abs() <= 65536 * (x_off / sc.repeat_interleave(256)[:n] + 32 * U * y) / step + 1
            near = near | (y / step - torch.round(y / step)).abs().lt(1e-3)   # (where the step itself may be the next one's)
            differs = (wide.abs() - want.clamp(max=448)).abs() > 1e-9 * want
            assert not bool((differs & ~near).any()), (j, name)
            assert bool(((wide.abs() - y).abs() <= 2 * step).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_eight_bits_to_the_last_bit(dtype):
    """Moments in 8 bits and their scales are what the formula's fp32 operations give one after the other, bit for bit, over several steps."""
    st = _setup([(70001,), (3000,), (64, 2048)], dtype, 8, False, 21)
    for t in (11, 12, 13):
        for x in st["grads"]:
            x.mul_(0.9).add_(1e-3)
        before = _clone(st)
        _step(st)
        for j, g in enumerate(before["grads"]):
            n, g = g.numel(), g.reshape(-1).float()
            sc = before["scales"][j].repeat_interleave(256, 0)[:n]
            m, r = before["exp_avgs"][j].reshape(-1).float() * sc[:, 0], before["exp_avg_sqs"][j].reshape(-1).float() * sc[:, 1]
            m, v = m * BETAS[0] + g * (1 - BETAS[0]), r * r * BETAS[1] + g * g * (1 - BETAS[1])
            key = _mix((7 * 0x9E3779B9 + t * 0xBB67AE85 + j) & 0xFFFFFFFF)
            h = _mix((torch.arange(n, device="cuda") * 0x9E3779B9 + key) & 0xFFFFFFFF)
            for column, (name, x, u16) in enumerate((("exp_avgs", m, h & 0xFFFF), ("exp_avg_sqs", torch.sqrt(v), h >> 16))):
                top = torch.cat([x, x.new_zeros(-n % 256)]).view(-1, 256).abs().amax(1).clamp(min=2.0 ** -100)
                assert torch.equal(st["scales"][j][:, column], top * (1.0 / 448.0)), (j, name)
                y = x.abs() * (torch.reciprocal(top) * 448.0).repeat_interleave(256)[:n]
                code = ((((y * 2.0 ** -120).view(torch.int32).long()) + (u16 << 4)) >> 20).clamp(max=0x7E)
                if column == 1:
                    code = torch.where((code == 0) & (x > 0), torch.ones_like(code), code)
                want = code.to(torch.uint8).view(F8).float() * torch.where(x < 0, -1.0, 1.0)
                assert torch.equal(st[name][j].reshape(-1).float(), want), (j, name)


def _clone(st):
    return {k: [t.clone() for t in v] if isinstance(v, list) else (v.clone() if v is not None else None) for k, v in st.items()}


def _step(st, **kw):
    kw = dict(dict(lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, seed=7), **kw)
    return rwkv_kernel.adamw_step(st["params"], st["grads"], st["exp_avgs"], st["exp_avg_sqs"], st["step"], scales=st["scales"], masters=st["masters"], **kw)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("clip", [None, 1.0, 1e6])
def test_step(dtype, bits, master, clip):
    print("adamw", dtype, bits, master, clip, flush=True)
    if master and dtype == torch.float32:
        return
    st = _setup(SHAPES, dtype, bits, master, 1)
    for t in (11, 12):
        before = _clone(st)
        norm = _step(st, max_grad_norm=clip)
        want = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
        assert (norm is None) == (clip is None) and int(st["step"]) == t
        if clip is not None:
            assert abs(float(norm) - want) <= 2 * U * want
        assert all(torch.equal(a, b) for a, b in zip(before["grads"], st["grads"]))
        _check(before, st, want, clip, bits, t)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 47, 48, 49, 97, 300])
def test_many_tensors(count, bits):
    """More tensors than one launch takes, empty ones among them; each as if it were stepped in a list of its place."""
    shapes = [((i * 37) % 600,) for i in range(count)]
    shapes[0] = (5,)
    st = _setup(shapes, torch.bfloat16, bits, False, count)
    before = _clone(st)
    norm = _step(st, max_grad_norm=0.5)
    want = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
    assert abs(float(norm) - want) <= 2 * U * want
    _check(before, st, want, 0.5, bits, 11)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_any_alignment_and_nothing_beside(dtype, bits):
    """Tensors that begin anywhere in a larger buffer, one behind the other or apart; what lies around them keeps its values."""
    n, room = 5000, 64
    for shift in (0, 1, 2, 3, 5, 8):
        st = _setup([(n,)], dtype, bits, False, 3)
        plain = _clone(st)
        buffers = {}
        for k in ("params", "grads", "exp_avgs", "exp_avg_sqs"):
            fill = torch.full((room + n + room,), 7.0, device="cuda").to(st[k][0].dtype)
            fill[room + shift:room + shift + n].copy_(st[k][0])
            buffers[k], st[k] = fill, [fill[room + shift:room + shift + n]]
        _step(st, max_grad_norm=1.0)
        _step(plain, max_grad_norm=1.0)
        for k, fill in buffers.items():
            assert torch.equal(st[k][0].float(), plain[k][0].float()), k
            assert bool((fill[:room + shift].float() == 7).all()) and bool((fill[room + shift + n:].float() == 7).all()), k


def test_layouts():
    """Parameters in any dense order; a gradient in another order than its parameter."""
    for bits in (32, 8):
        st = _setup([(40, 30)], torch.float32, bits, False, 4)
        turned = _clone(st)
        for k in ("params", "exp_avgs", "exp_avg_sqs"):   # the same memory, read as its transpose
            turned[k] = [turned[k][0].view(40, 30).t()]
        turned["grads"] = [turned["grads"][0].t().contiguous()]
        _step(st)
        _step(turned)
        for k in ("params", "exp_avgs", "exp_avg_sqs"):
            assert torch.equal(turned[k][0].t().float(), st[k][0].float()), k


def test_first_steps_from_nothing():
    """Zero moments, zero gradients, gradients of every magnitude, an element whose gradient has always been zero."""
    for bits in (32, 8):
        p = torch.linspace(-1, 1, 1000).cuda()
        opt = rwkv_kernel.AdamW([torch.nn.Parameter(p.clone())], lr=1e-2, betas=BETAS, weight_decay=0.0, moment_bits=bits)
        q = opt.param_groups[0]["params"][0]
        q.grad = torch.zeros_like(q)
        opt.step()
        assert torch.equal(q.detach(), p)
        g = torch.exp2(torch.linspace(-60, 10, 1000)).cuda()
        g[::7] = 0
        q.grad = g.clone()
        opt.step()
        # m / sqrt(v) of a first gradient in step 2
        t = 2
        want = p.double().cpu() - torch.where(g.cpu() != 0, 1e-2 / (1 - 0.9 ** t) * 0.1 * g.cpu().double() / ((0.01 * g.cpu().double() ** 2 / (1 - 0.99 ** t)).sqrt() + 1e-8), torch.zeros(()).double())
        assert bool(((q.detach().cpu().double() - want).abs() <= 1e-6).all())
        for _ in range(5):
            opt.step()
        assert bool(torch.isfinite(q).all()) and torch.equal(q.detach()[::7], p[::7])
        assert float((q.detach() - p).abs().max()) < 0.2   # (a denominator lost to rounding would throw a weight far away)


def test_rounding_at_random_keeps_the_mean():
    """A moment that changes by far less than a step of its format moves on average as it should: v under a gradient half again as large."""
    n = 1 << 16
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = rwkv_kernel.AdamW([p], lr=0.0, betas=(0.9, 0.999), moment_bits=8)
    p.grad = torch.ones_like(p)
    p.grad[::256] = 4.0      # the largest of each block: the others' values lie between the format's
    opt.step()
    s = opt.state[p]
    value = lambda: (s["exp_avg_sq"].float().view(-1, 256) * s["scales"][:, 1:]).view(-1)  # noqa: E731
    v = 0.001
    p.grad[p.grad == 1] = 1.5
    for _ in range(60):
        opt.step()
        v = 0.999 * v + 0.001 * 2.25
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[::256] = False
    r = value()[others].double()
    # each step adds a rounding of variance at most (step / 2)^2 with step <= r / 8, which decays hardly at all: 60 (r / 16)^2 = (0.48 r)^2 for
    # one element, over 65000 elements 0.2 % of r; its square shifts the mean of r by at most half of 60 (1/16)^2 / 2
    assert abs(float(r.mean()) / math.sqrt(v) - 1) < 0.13
    assert bool((s["exp_avg"].float().abs() > 0).all())


def test_clipping_and_non_finite_gradients():
    for bits in (32, 8):
        for bad in (float("inf"), float("nan")):
            st = _setup([(300,), (500,)], torch.bfloat16, bits, False, 5)
            st["grads"][1][17] = bad
            before = _clone(st)
            norm = _step(st, max_grad_norm=1.0, skip_nonfinite=True)
            assert not math.isfinite(float(norm)) and int(st["step"]) == 10
            for k in ("params", "exp_avgs", "exp_avg_sqs") + (("scales",) if bits == 8 else ()):
                assert all(torch.equal(a.float(), b.float()) for a, b in zip(before[k], st[k])), k
            # without it the damage shows
            st["grads"][0].normal_()
            _step(st)
            assert not bool(torch.isfinite(st["params"][1]).all()) and bool(torch.isfinite(st["params"][0]).all())
            moments = st["exp_avgs"][1].float().view(-1) * (st["scales"][1].repeat_interleave(256, 0)[:500, 0] if bits == 8 else 1.0)
            assert not math.isfinite(float(moments[17]))


def test_a_given_norm_and_a_rate_on_the_device():
    st = _setup([(1000,)], torch.float32, 32, False, 6)
    other = _clone(st)
    norm = rwkv_kernel.grad_norm(st["grads"])
    _step(st, max_grad_norm=0.1)
    _step(other, max_grad_norm=0.1, grad_norm=norm, lr=torch.tensor(LR).cuda())
    # (the rate is rounded to fp32 first: 2 u of an update, which p's own rounding hides or not)
    assert float((st["params"][0] - other["params"][0]).abs().max()) <= 4 * U * (float(st["params"][0].abs().max()) + 0.1)
    assert torch.equal(st["exp_avgs"][0], other["exp_avgs"][0])


def test_grad_norm_over_large_and_small():
    g = torch.Generator().manual_seed(8)
    for dtype in DTYPES:
        grads = [(torch.randn(n, generator=g) * s).to(dtype).cuda() for n, s in ((5_000_001, 1e-3), (3, 100.0), (0, 1.0), (4097, 1.0))]
        want = math.sqrt(sum(float(x.double().square().sum()) for x in grads))
        assert abs(float(rwkv_kernel.grad_norm(grads)) - want) <= 2 * U * want
        assert torch.equal(rwkv_kernel.grad_norm(grads), rwkv_kernel.grad_norm(grads))
    assert float(rwkv_kernel.grad_norm([torch.full((10,), 3e38).cuda()])) == float("inf")
    assert float(rwkv_kernel.grad_norm([torch.zeros(0).cuda()])) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_count_on(bits):
    """A captured step takes the next step count and a new rate in each replay, with eager work between."""
    shapes = [(300,), (64, 65), (5000,)]
    params = [torch.nn.Parameter((torch.randn(*s, generator=torch.Generator().manual_seed(1)) * 0.1).cuda()) for s in shapes]
    lr = torch.tensor(1e-2).cuda()
    opt = rwkv_kernel.AdamW(params, lr=lr, betas=BETAS, max_grad_norm=1.0, moment_bits=bits, seed=3)
    twin_params = [torch.nn.Parameter(p.detach().clone()) for p in params]
    twin_lr = lr.clone()
    twin = rwkv_kernel.AdamW(twin_params, lr=twin_lr, betas=BETAS, max_grad_norm=1.0, moment_bits=bits, seed=3)
    g = torch.Generator().manual_seed(2)
    for p, q in zip(params, twin_params):
        p.grad = torch.randn(*p.shape, generator=g).cuda()
        q.grad = p.grad.clone()
    opt.step()
    twin.step()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(4):
        for p, q in zip(params, twin_params):
            p.grad.copy_(torch.randn(*p.shape, generator=g))
            q.grad.copy_(p.grad)
        lr.mul_(0.7)
        twin_lr.mul_(0.7)
        graph.replay()
        torch.cuda.synchronize()
        twin.step()
        for p, q in zip(params, twin_params):
            assert torch.equal(p, q), i
            for k in opt.state[p]:
                assert torch.equal(opt.state[p][k].float(), twin.state[q][k].float()), (i, k)
        assert torch.equal(opt.last_grad_norm, twin.last_grad_norm)


def _model(dtype=torch.float32, seed=0):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 30), torch.nn.Linear(30, 5)).cuda().to(dtype)


@pytest.mark.parametrize("bits,master,dtype", [(32, False, torch.float32), (8, False, torch.float32), (32, True, torch.bfloat16), (8, True, torch.bfloat16)])
def test_optimizer_saves_and_loads(bits, master, dtype):
    """State dicts, copies and pickles go on as if nothing had happened; parameters without a gradient keep their own step count."""
    import io
    x = torch.randn(16, 20, generator=torch.Generator().manual_seed(1)).cuda().to(dtype)
    make = lambda m: rwkv_kernel.AdamW([{"params": m[0].parameters(), "weight_decay": 0.0}, {"params": list(m[1].parameters()) + list(m[2].parameters())}],  # noqa: E731
                                       lr=1e-2, moment_bits=bits, master_weights=master, max_grad_norm=0.5)

    def train(m, o, steps, skip=False):
        for _ in range(steps):
            o.zero_grad(set_to_none=True)
            m(x).float().square().mean().backward()
            if skip:
                for p in m[1].parameters():
                    p.grad = None
            o.step()

    model = _model(dtype)
    opt = make(model)
    train(model, opt, 3)
    train(model, opt, 2, skip=True)
    train(model, opt, 1)
    steps = [int(opt.state[p]["step"]) for p in model.parameters()]
    assert steps == [6, 6, 4, 4, 6, 6]
    assert opt.state[model[0].weight]["step"] is not opt.state[model[2].weight]["step"]
    other = _model(dtype, 1)
    other.load_state_dict(model.state_dict())
    loaded = make(other)
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    loaded.load_state_dict(torch.load(file, weights_only=True))
    third = copy.deepcopy((model, opt))
    for m, o in ((model, opt), (other, loaded), third):
        train(m, o, 2)
    for p, q, r in zip(model.parameters(), other.parameters(), third[0].parameters()):
        assert torch.equal(p, q) and torch.equal(p, r)
        for k in opt.state[p]:
            assert opt.state[p][k].dtype == loaded.state[q][k].dtype and torch.equal(opt.state[p][k].float(), loaded.state[q][k].float()), k


def test_against_torchs_own_optimizer():
    """Ten steps beside torch.optim.AdamW in float64 from the same weights and gradients: each step's error is some 2^-21 of an update."""
    p64 = [torch.randn(*s, generator=torch.Generator().manual_seed(1)).double() for s in ((30, 40), (7,))]
    ours = [torch.nn.Parameter(p.float().cuda()) for p in p64]
    theirs = [torch.nn.Parameter(p.float().double()) for p in p64]
    a = rwkv_kernel.AdamW(ours, lr=1e-2, weight_decay=0.1)
    b = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.1, foreach=False)
    g = torch.Generator().manual_seed(2)
    for _ in range(10):
        for p, q in zip(ours, theirs):
            q.grad = torch.randn(*q.shape, generator=g).double().float().double()
            p.grad = q.grad.float().cuda()
        a.step()
        b.step()
    for p, q in zip(ours, theirs):
        assert float((p.detach().cpu().double() - q.detach()).abs().max()) <= 10 * (2.0 ** -20 * 2e-2 + 4 * U * 5)


def test_a_parameter_in_use_is_noticed():
    """autograd sees that a weight it saved has changed."""
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    x = torch.ones(4, device="cuda", requires_grad=True)
    y = (p * x).sum()
    opt = rwkv_kernel.AdamW([p])
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals_on_the_gpu():
    st = _setup([(10,)], torch.float32, 32, False, 9)
    bad = dict(params=[st["params"][0].double()], grads=[st["grads"][0].half()], exp_avgs=[st["exp_avgs"][0][:5]], exp_avg_sqs=[st["exp_avg_sqs"][0].cpu()],
               step=st["step"].float())
    for k, v in bad.items():
        with pytest.raises(RuntimeError, match="wkv6"):
            _step(dict(st, **{k: v}))
    with pytest.raises(RuntimeError, match="twice"):
        _step({k: v * 2 if isinstance(v, list) else v for k, v in st.items()})
    with pytest.raises(RuntimeError, match="scales"):
        _step(dict(st, scales=[torch.zeros(1, 2).cuda()]))
    with pytest.raises(RuntimeError, match="master"):
        _step(dict(st, masters=[torch.zeros(10).cuda()]))
    for kw in (dict(lr=-1.0), dict(max_grad_norm=0.0)):
        with pytest.raises(AssertionError):
            _step(st, **kw)
    with pytest.raises(RuntimeError):
        _step(st, betas=(1.0, 0.9))


def test_a_first_step_is_not_captured():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = rwkv_kernel.AdamW([p])
    p.grad = torch.ones_like(p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(AssertionError, match="captured"):
        with torch.cuda.graph(graph):
            opt.step()
    torch.cuda.synchronize()
    opt.step()
    assert int(opt.state[p]["step"]) == 1


def test_a_moment_twice_is_refused():
    st = _setup([(10,), (10,)], torch.float32, 32, False, 9)
    with pytest.raises(RuntimeError, match="twice"):
        _step(dict(st, exp_avgs=[st["exp_avgs"][0]] * 2))
    with pytest.raises(RuntimeError, match="twice"):
        _step(dict(st, exp_avg_sqs=st["exp_avgs"]))
    with pytest.raises(RuntimeError, match="dense"):
        wide = torch.zeros(10, 4, device="cuda")
        _step({k: [wide[:, 0].clone().as_strided((10,), (1,)) if k != "params" else wide[:, 0]] if isinstance(v, list) else v for k, v in st.items()})


def test_steps_on_two_streams():
    """Two optimizers side by side, each as if alone."""
    def run(streams):
        out = []
        for i, stream in enumerate(streams):
            p = torch.nn.Parameter(torch.linspace(-1, 1, 50000 + i).cuda())
            with torch.cuda.stream(stream):
                opt = rwkv_kernel.AdamW([p], lr=1e-2, max_grad_norm=1.0, moment_bits=8)
                for t in range(5):
                    p.grad = torch.sin(p.detach() * (t + 1))
                    opt.step()
            out.append(p)
        torch.cuda.synchronize()
        return [p.detach().clone() for p in out]

    torch.cuda.synchronize()
    alone = run([torch.cuda.current_stream()] * 3)
    side = [torch.cuda.Stream() for _ in range(3)]
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    assert all(torch.equal(a, b) for a, b in zip(alone, run(side)))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_elements_than_32_bits_count(bits):
    """A tensor of more than 2^31 elements: its last ones go as they do in a tensor of their own (in 8 bits: within the two values that the drawn number chooses from)."""
    n, tail = (1 << 31) + 4096 + 77, 4096 + 77
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    st = _setup([(tail,)], torch.bfloat16, bits, False, 31)
    whole = dict(params=[p], grads=[g], masters=None, step=st["step"].clone(), scales=None)
    p[-tail:], g[-tail:] = st["params"][0], st["grads"][0]
    for k in ("exp_avgs", "exp_avg_sqs"):
        m = torch.zeros(n, dtype=torch.uint8 if bits == 8 else torch.float32, device="cuda")
        m[-tail:] = st[k][0].view(torch.uint8) if bits == 8 else st[k][0]
        whole[k] = [m.view(F8) if bits == 8 else m]
    if bits == 8:
        scales = torch.zeros((n + 255) // 256, 2, device="cuda")
        scales[-((tail + 255) // 256):] = st["scales"][0]
        whole["scales"] = [scales]
    norms = [_step(x, max_grad_norm=0.5) for x in (st, whole)]
    assert torch.equal(*norms) and torch.equal(p[-tail:], st["params"][0]) and not bool(p[:-tail].any())
    for k in ("exp_avgs", "exp_avg_sqs"):
        got, want = whole[k][0][-tail:], st[k][0]
        if bits == 32:
            assert torch.equal(got, want)
        else:
            got, want = got.view(torch.uint8).int(), want.view(torch.uint8).int()
            assert int((got - want).abs().max()) <= 1
    if bits == 8:
        assert torch.equal(whole["scales"][0][-((tail + 255) // 256):], st["scales"][0])


def test_tensors_that_overlap_are_refused():
    """Two tensors of a call that share elements would be written by two workgroups at once; neighbours in one buffer are in order."""
    for bits in (32, 8):
        for name in ("params", "exp_avgs", "exp_avg_sqs", "masters"):
            st = _setup([(600,), (600,)], torch.bfloat16, bits, True, 9)
            room = torch.zeros(1200, device="cuda").to(st[name][0].dtype)
            before = _clone(st)
            with pytest.raises(RuntimeError, match="twice"):
                _step(dict(st, **{name: [room[:600], room[300:900]]}))
            with pytest.raises(RuntimeError, match="twice"):
                _step(dict(st, **{name: [room[599:1199], room[:600]]}))
            assert int(st["step"]) == 10 and all(torch.equal(a.float(), b.float()) for a, b in zip(before["params"], st["params"]))
            _step(dict(st, **{name: [room[600:], room[:600]]}))
            assert int(st["step"]) == 11


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [59, 60, 61, 119, 120, 121])
def test_as_many_tensors_as_launches_take(count, bits):
    """On either side of 60 and 120 tensors: one launch, two, three."""
    test_many_tensors(count, bits)


@pytest.mark.parametrize("dtype,bits,master", [(torch.float32, 32, False), (torch.float32, 8, False), (torch.bfloat16, 32, False), (torch.bfloat16, 32, True), (torch.float16, 8, True),
                                               (torch.bfloat16, 8, False)])
def test_steps_past_the_caches(dtype, bits, master):
    """Tensors of 160 MiB and more together are loaded and stored in another way: they become what they do in calls of their own, at the same place of a list."""
    sizes = [9_000_001, 8_999_743, 9_500_123, 3_000_000, 4097]
    es = torch.finfo(dtype).bits // 8
    assert sum(sizes) * (2 * es + bits // 4 + (4 if master else 0)) >= 160 << 20 > max(sizes) * (2 * es + bits // 4 + (4 if master else 0))
    gen = torch.Generator(device="cuda").manual_seed(47)
    rand = lambda n, std: torch.randn(n, generator=gen, device="cuda") * std  # noqa: E731
    st = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[], scales=[] if bits == 8 else None, masters=[] if master else None, step=torch.tensor(10, device="cuda"))
    for n in sizes:
        w = rand(n, 0.1)
        st["params"].append(w.to(dtype))
        if master:
            st["masters"].append(w)
        st["grads"].append(rand(n, 1e-2).to(dtype))
        if bits == 8:
            st["scales"].append(torch.rand((n + 255) // 256, 2, generator=gen, device="cuda") * 1e-4 + 1e-6)
            st["exp_avgs"].append(rand(n, 100.0).clamp(-448, 448).to(F8))
            st["exp_avg_sqs"].append(rand(n, 100.0).abs().clamp(0, 448).to(F8))
        else:
            st["exp_avgs"].append(rand(n, 1e-2))
            st["exp_avg_sqs"].append(rand(n, 1e-2).square())
    alone = _clone(st)
    norm = rwkv_kernel.grad_norm(st["grads"])
    _step(st, max_grad_norm=0.5, grad_norm=norm)
    for j in range(len(sizes)):
        # (empty tensors before it: the place in the list decides what 8-bit moments are rounded to)
        one = {k: [t[:0].clone() for t in v[:j]] + v[j:j + 1] if isinstance(v, list) else v for k, v in alone.items()}
        one["step"] = torch.tensor(10, device="cuda")
        _step(one, max_grad_norm=0.5, grad_norm=norm)
        for k in ("params", "exp_avgs", "exp_avg_sqs", "scales", "masters"):
            if st[k]:
                assert torch.equal(st[k][j].float(), alone[k][j].float()), (j, k)
        assert not torch.equal(st["exp_avgs"][j].float(), torch.zeros_like(st["exp_avgs"][j]).float())
