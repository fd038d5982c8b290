"""The model with the package's embedding and layer norms, trained with its losses and Muon: against the same model in float64 on the CPU, whose operator is the python loop."""
import copy

import pytest
import torch
import torch.utils.checkpoint

import rwkv6_harness as hz
import rwkv_kernel

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
B, T, V = 2, 40, 300
CONFIG = dict(num_layers=2, vocabulary_size=V, hidden_size=128, decomposer_size=32, head_size=64, expand_size=256)


def _models(seed=1):
    torch.manual_seed(seed)
    plain = hz.RWKV6(rwkv_kernel.OPSKernelOperator(64, T), **CONFIG)
    ours = hz.RWKV6(rwkv_kernel.RWKVKernelOperator(64, T), **CONFIG)
    ours.load_state_dict(plain.state_dict())
    return plain.double(), ours.cuda()


def _ids(seed=2):
    return torch.randint(0, V, (B, T + 1), generator=torch.Generator().manual_seed(seed))


def _calls(monkeypatch):
    """How often the model's steps call the package's functions."""
    seen = {}
    for name in ("embedding", "layer_norm", "cross_entropy"):
        def counted(*a, _f=getattr(rwkv_kernel, name), _n=name, **k):
            seen[_n] = seen.get(_n, 0) + 1
            return _f(*a, **k)
        monkeypatch.setattr(rwkv_kernel, name, counted)
    return seen


def test_forward_and_gradients_in_fp32(monkeypatch):
    """Everything in fp32: values and gradients of a loss within 2^-12 of the largest of a tensor (some 100 roundings of 2^-24 on the way, and the operator's own
    1e-4 of its largest value)."""
    seen = _calls(monkeypatch)
    plain, ours = _models()
    ids = _ids()
    w = torch.randn(B, T, V, generator=torch.Generator().manual_seed(3)).double()
    a, b = plain(ids[:, :-1]), ours(ids[:, :-1].cuda())
    assert seen == {"embedding": 1, "layer_norm": 2 + 2 * CONFIG["num_layers"]}
    assert float((b.cpu().double() - a).detach().abs().max()) <= 2.0 ** -12 * float(a.detach().abs().max())
    (a * w).sum().backward()
    (b * w.float().cuda()).sum().backward()
    for (name, p), q in zip(plain.named_parameters(), ours.parameters()):
        assert float((q.grad.cpu().double() - p.grad).abs().max()) <= 2.0 ** -10 * float(p.grad.abs().max()) + 1e-9, name


def test_blocks_are_the_stages():
    _, ours = _models()
    x = torch.randn(B, T, 128, generator=torch.Generator().manual_seed(5)).cuda()
    with torch.no_grad():
        y, branch = ours.blocks[0].stages(x, None)
        assert torch.equal(ours.blocks[0](x), y + branch)
        z, branch = ours.blocks[1].stages(y, branch)
        want = ours.blocks[1](ours.blocks[0](x))
    assert float((z + branch - want).abs().max()) <= 2.0 ** -20 * float(want.abs().max())   # (one kernel adds what two added)


def test_norms_under_autocast():
    """The norms come out in bf16 where their readers round them: the logits are those of the model whose norms are torch's, to the bit wherever no fp32 value lies next
    to the middle between two of bf16; half a step of bf16 (2^-9) of the largest value is left for those."""
    _, ours = _models()
    plain = copy.deepcopy(ours)

    class Own(torch.nn.LayerNorm):   # (not the class that the package's kernel stands in for)
        pass

    for module in list(plain.modules()):
        for name, child in list(module.named_children()):
            if type(child) is torch.nn.LayerNorm:
                own = Own(child.normalized_shape, eps=child.eps).cuda()
                own.load_state_dict(child.state_dict())
                setattr(module, name, own)
    ids = _ids().cuda()[:, :-1]
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        a, b = ours(ids).float(), plain(ids).float()
    assert float((a - b).abs().max()) <= 2.0 ** -6 * float(b.abs().max())
    assert float((a - b).norm()) <= 2.0 ** -8 * float(b.norm())


@pytest.mark.parametrize("dtype", [None, BF16])
def test_steps_with_muon(dtype, monkeypatch):
    """Three steps: each matrix of the layers gets the step that muon_step makes of its gradient and momentum, everything else AdamW's, and the loss is finite."""
    seen = _calls(monkeypatch)
    _, ours = _models()
    opt = hz.muon_and_adamw(ours, lr=0.01, weight_decay=0.1, adamw_lr=1e-3)
    muon, adamw = opt.optimizers
    matrices = [p for g in muon.param_groups for p in g["params"]]
    others = [p for g in adamw.param_groups for p in g["params"]]
    assert len(matrices) + len(others) == len(list(ours.parameters())) and all(p.dim() == 2 for p in matrices)
    assert any(p is ours.embedding.weight for p in others) and any(p is ours.output_layer.weight for p in others)
    for step in range(3):
        before = [p.detach().clone() for p in matrices]
        bufs = [muon.state[p]["momentum"].clone() if step else torch.zeros_like(p) for p in matrices]
        rest = [p.detach().clone() for p in others]
        loss = hz.train_step(ours, opt, _ids(10 + step).cuda(), dtype)
        assert bool(loss.isfinite())
        rwkv_kernel.muon_step(before, [p.grad for p in matrices], bufs, 0.01, weight_decay=0.1)
        assert all(torch.equal(p, q) for p, q in zip(before, matrices))
        assert not any(torch.equal(p, q) for p, q in zip(rest, others) if p.numel() > 1)
    assert seen == {"embedding": 3, "layer_norm": 3 * (2 + 2 * CONFIG["num_layers"]), "cross_entropy": 3}


def test_a_captured_step():
    """Forward, backward and both optimizers in one graph, replayed, against the same steps taken one by one."""
    print("training step with Muon, captured", flush=True)
    _, ours = _models()
    twin = copy.deepcopy(ours)
    opts = [hz.muon_and_adamw(m, lr=0.01) for m in (ours, twin)]
    ids = [_ids(20).cuda() for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step(model, opt, x):
        for p in model.parameters():
            p.grad = None
        loss = rwkv_kernel.cross_entropy(model(x[:, :-1]), x[:, 1:])
        loss.backward()
        opt.step()
        return loss

    with torch.cuda.stream(side):
        step(ours, opts[0], ids[0])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            loss = step(ours, opts[0], ids[0])
    torch.cuda.current_stream().wait_stream(side)
    step(twin, opts[1], ids[1])
    for k in range(3):
        for x in ids:
            x.copy_(_ids(30 + k))
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin, opts[1], ids[1])
        assert torch.equal(loss, want)
        for (name, p), q in zip(ours.named_parameters(), twin.parameters()):
            assert torch.equal(p, q), name


def _reruns(module):
    """The module in another one, which computes its activations again in the backward pass."""
    class Wrap(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.inner = module

        def forward(self, *a):
            return torch.utils.checkpoint.checkpoint(self.inner, *a, use_reentrant=False)

    return Wrap()


@pytest.mark.parametrize("dtype", [None, BF16])
def test_hooks_and_wrappers_in_the_model(dtype):
    """Hooks on the table, the norms, the mixes and the output layer run, with what torch's modules see there (fp32 in and out of the norms), and wrapped modules are called.  The logits
    are the model's: to 2^-12 of the largest in fp32, as above; under bf16 autocast to half a step of bf16, 2^-9, in each of some 10 stages that a flipped rounding goes through: 2^-5."""
    _, ours = _models()
    ids = _ids().cuda()[:, :-1]
    off = 2.0 ** (-12 if dtype is None else -5)

    def run(model):
        with torch.autocast("cuda", dtype=BF16, enabled=dtype is not None):
            return model(ids).float()

    def close(a, b):
        return float((a - b).detach().abs().max()) <= off * float(b.detach().abs().max())

    want = run(ours)
    names = ["embedding", "embedding_ln", "output_ln", "output_layer"] + ["blocks.%d.%s" % (k, n) for k in range(2) for n in ("layer_norm_att", "layer_norm_ffn", "time_mix", "channel_mix")]
    for kind in ("forward", "pre", "backward"):
        model, seen = copy.deepcopy(ours), {}
        for name in names:
            m = model.get_submodule(name)
            if kind == "forward":
                m.register_forward_hook(lambda m, a, out, n=name: seen.update({n: (a[0].dtype, out.dtype)}))
            elif kind == "pre":
                m.register_forward_pre_hook(lambda m, a, n=name: seen.update({n: (a[0].dtype,)}))
            else:
                m.register_full_backward_hook(lambda m, gi, go, n=name: seen.update({n: ()}))
        logits = run(model)
        logits.sum().backward()
        assert close(logits, want) and sorted(seen) == sorted(names), kind
        if kind != "backward":
            assert all(all(t == torch.float32 for t in v) for n, v in seen.items() if "norm" in n or "_ln" in n)
            assert all(v[0] == torch.float32 for n, v in seen.items() if n != "embedding")
    # a hook that changes what comes out does so
    for name in ("embedding", "embedding_ln", "output_ln", "blocks.0.layer_norm_att", "blocks.1.layer_norm_ffn"):
        model = copy.deepcopy(ours)
        model.get_submodule(name).register_forward_hook(lambda m, a, out: torch.zeros_like(out))
        assert not close(run(model), want), name
    # nothing is asked of a module in another one's place
    for name in names:
        model = copy.deepcopy(ours)
        parent, _, child = name.rpartition(".")
        setattr(model.get_submodule(parent), child, _reruns(model.get_submodule(name)))
        logits = run(model)
        assert close(logits, want), name
        logits.sum().backward()


def test_norms_that_are_left_to_torch(monkeypatch):
    """More channels than the kernel takes, several dimensions, branches of other types and shapes: what they were before there was a kernel."""
    seen = _calls(monkeypatch)
    g = torch.Generator().manual_seed(4)
    wide, two = torch.nn.LayerNorm(40000).cuda(), torch.nn.LayerNorm((6, 64)).cuda()
    for norm, shape, branch in ((wide, (2, 3, 40000), None), (wide, (2, 3, 40000), torch.float32), (two, (5, 6, 64), None), (two, (5, 6, 64), torch.float32),
                                (torch.nn.LayerNorm(64).cuda(), (5, 6, 64), "row")):
        x = torch.randn(shape, generator=g).cuda()
        b = None if branch is None else torch.randn(shape if branch != "row" else shape[-1:], generator=g).cuda()
        total, h = hz.add_norm(x, b, norm)
        assert torch.equal(total, x if b is None else x + b) and torch.equal(h, norm(total))
    norm = torch.nn.LayerNorm(64).cuda().double()
    x, b = torch.randn(5, 64, generator=g).cuda(), torch.randn(5, 64, generator=g).double().cuda()
    total, h = hz.add_norm(x, b, norm)
    assert total.dtype == h.dtype == torch.float64 and torch.equal(h, norm(x + b))
    assert seen == {}
    hz.add_norm(x, x, torch.nn.LayerNorm(64).cuda())
    assert seen == {"layer_norm": 1}


def test_ids_outside_of_the_table():
    """An error on the CPU; on the GPU NaN in the logits of their text and no others, and in a step's loss.  What is no id at all is refused on either."""
    plain, ours = _models()
    ids = torch.randint(0, V, (4, T), generator=torch.Generator().manual_seed(6))
    want = ours(ids.cuda())
    for bad in (-1, -V, V, -2 ** 63, 2 ** 63 - 1):
        x = ids.clone()
        x[2, 5] = bad
        with pytest.raises(IndexError):
            plain(x)
        got = ours(x.cuda())
        assert torch.equal(got[[0, 1, 3]], want[[0, 1, 3]]) and bool(got[2, 5:].isnan().all()), bad
        if bad in (-1, V):
            assert bool(ours(x.int().cuda())[2, 5:].isnan().all())
            assert bool(rwkv_kernel.cross_entropy(got, ids.cuda()).isnan())
    assert torch.equal(ours(ids.int().cuda()), want)
    for model, x in ((plain, ids), (ours, ids.cuda())):
        with pytest.raises((RuntimeError, IndexError)):
            model(x.float())


def test_training_goes_on_from_what_was_saved():
    """Muon and AdamW as one optimizer, with a schedule, saved after two steps and loaded."""
    _, ours = _models()
    _, twin = _models(seed=9)
    opt, other = hz.muon_and_adamw(ours, lr=0.01), hz.muon_and_adamw(twin, lr=0.5, adamw_lr=0.3)
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 0.5 ** step)
    for step in range(2):
        hz.train_step(ours, opt, _ids(10 + step).cuda())
        schedule.step()
    assert [g["lr"] for g in opt.param_groups] == [0.0025, 0.25e-4]
    twin.load_state_dict(ours.state_dict())
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    for step in range(2):
        for model, o in ((ours, opt), (twin, other)):
            hz.train_step(model, o, _ids(20 + step).cuda())
    assert all(torch.equal(p, q) for p, q in zip(ours.parameters(), twin.parameters()))
    assert all(torch.equal(opt.state[p][n], other.state[q][n]) for p, q in zip(ours.parameters(), twin.parameters()) for n in opt.state[p])


def test_options_of_both_optimizers():
    _, ours = _models()
    ours = ours.to(BF16)
    opt = hz.muon_and_adamw(ours, lr=0.01, weight_decay=0.1, adamw_lr=1e-3, adamw=dict(moment_bits=8, master_weights=True, max_grad_norm=1e-3, weight_decay=0.0, betas=(0.8, 0.9)), momentum=0.9,
                            master_weights=True)
    muon, adamw = opt.optimizers
    assert [(g["lr"], g["weight_decay"]) for g in opt.param_groups] == [(0.01, 0.1), (1e-3, 0.0)] and opt.param_groups[0]["momentum"] == 0.9 and opt.param_groups[1]["betas"] == (0.8, 0.9)
    ids, w = _ids().cuda(), torch.randn(B, T, V, generator=torch.Generator().manual_seed(3)).cuda()
    for _ in range(2):
        opt.zero_grad()
        with torch.autocast("cuda", dtype=BF16):
            (ours(ids[:, :-1]).float() * w).sum().backward()
        opt.step()
    assert all("master" in s for s in opt.state.values()) and all("scales" in s for s in adamw.state.values()) and float(adamw.last_grad_norm) > 1e-3
    with pytest.raises(AssertionError, match="skip_nonfinite"):
        hz.muon_and_adamw(ours, adamw=dict(skip_nonfinite=True))


class _Torchs(torch.nn.LayerNorm):   # (not the class that the package's kernel stands in for)
    pass


def _with_torchs_norms(model):
    model = copy.deepcopy(model)
    for m in model.modules():
        if type(m) is torch.nn.LayerNorm:
            m.__class__ = _Torchs
    return model


def test_types_of_the_norms_under_autocast(monkeypatch):
    """bf16 where the only reader would round it, fp32 otherwise."""
    seen = []
    kernel = rwkv_kernel.layer_norm
    monkeypatch.setattr(rwkv_kernel, "layer_norm", lambda *a, **k: (seen.append(k["dtype"]), kernel(*a, **k))[1])
    _, ours = _models()
    ids = _ids().cuda()[:, :-1]
    for dtype, want in ((BF16, [torch.float32] + [BF16] * 5), (torch.float16, [torch.float32] * 6), (None, [torch.float32] * 6)):
        del seen[:]
        with torch.autocast("cuda", dtype=dtype, enabled=dtype is not None):
            ours(ids)
        assert seen == want, dtype


@pytest.mark.parametrize("C", [128, 777, 2048])
def test_an_addition_and_its_norm_under_autocast(C):
    """One addition with its norm, kernel and torch, with gradients.  The sum is the same to the bit.  The norm, some 8 roundings of 2^-24 in fp32 (and the channels' sums), goes
    to the other of two neighbours in bf16 only next to the middle between them: in 2^-8 of the elements at most, by a step of 2^-7.  The same for the branch's gradient.  Gradients in
    fp32 differ by roundings of terms up to 2^3 times what is left of them: 2^-18 of the largest, sums over the rows by 2^-16."""
    g = torch.Generator().manual_seed(C)
    norm = torch.nn.LayerNorm(C).cuda()
    with torch.no_grad():
        norm.weight.copy_(torch.randn(C, generator=g))
        norm.bias.copy_(torch.randn(C, generator=g))
    x, gy, gt = (torch.randn(6, 50, C, generator=g).cuda() for _ in range(3))
    branch = torch.randn(6, 50, C, generator=g).to(BF16).cuda()
    res = []
    for module in (norm, _with_torchs_norms(torch.nn.ModuleList([norm]))[0]):
        a, b = x.clone().requires_grad_(True), branch.clone().requires_grad_(True)
        with torch.autocast("cuda", dtype=BF16):
            total, h = hz.add_norm(a, b, module, rounded=True)
        assert h.dtype == (BF16 if module is norm else torch.float32)
        h = h.to(BF16)
        res.append([total, h, *torch.autograd.grad([total, h], [a, b, module.weight, module.bias], [gt, gy.to(BF16)])])
    (total, h, gx, gb, gw, gbias), want = res
    assert torch.equal(total, want[0])
    for p, q in ((h, want[1]), (gb, want[3])):
        assert int((p != q).sum()) <= 2.0 ** -8 * p.numel()
        assert bool(((p.float() - q.float()).abs() <= 2.0 ** -7 * q.float().abs() + 2.0 ** -20).all())
    assert float((gx - want[2]).abs().max()) <= 2.0 ** -18 * float(want[2].abs().max())
    for p, q in ((gw, want[4]), (gbias, want[5])):
        assert float((p - q).abs().max()) <= 2.0 ** -16 * float(q.abs().max())


def test_gradients_under_autocast():
    """The model's gradients under bf16 autocast with the kernel's norms and with torch's.  Either has the errors of its roundings to bf16; these are as large on both sides but not
    the same ones, so that a gradient of one is off from that of the other by about 1.4 times what torch's is off from float64: by 3 times at most, in the 2-norm of each parameter."""
    plain, ours = _models()
    torchs = _with_torchs_norms(ours)
    ids, w = _ids(), torch.randn(B, T, V, generator=torch.Generator().manual_seed(3))
    (plain(ids[:, :-1]) * w.double()).sum().backward()
    for model in (ours, torchs):
        with torch.autocast("cuda", dtype=BF16):
            logits = model(ids[:, :-1].cuda())
        (logits.float() * w.cuda()).sum().backward()
    for (name, e), p, q in zip(plain.named_parameters(), ours.parameters(), torchs.parameters()):
        p, q = p.grad.cpu().double(), q.grad.cpu().double()
        assert float((p - q).norm()) <= 3 * float((q - e.grad).norm()) + 2.0 ** -16 * float(e.grad.norm()), name
