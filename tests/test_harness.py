"""The RWKV-6 model harness around the operator (configuration 4 of the baseline, at toy sizes here):
its layers against independent restatements, a few training steps on the CPU with the python-loop
operator, and -- on the GPU -- the same model with the HIP operator against the python-loop one."""
import os
import sys

import pytest
import torch
import torch.nn.functional as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "star-rwkv6_amd"))
os.environ.setdefault("KERAS_BACKEND", "torch")

import rwkv6_harness as hz  # noqa: E402
from rwkv_kernel import OPSKernelOperator  # noqa: E402

TOY = dict(num_layers=2, vocabulary_size=97, hidden_size=128, decomposer_size=8, head_size=64, expand_size=224)


def _toy(op, seed=0):
    torch.manual_seed(seed)
    return hz.RWKV6(op, **TOY)


def test_time_shift_is_previous_token_minus_token():
    x = torch.arange(24, dtype=torch.float32).reshape(2, 3, 4)
    s = hz.time_shift(x)
    assert torch.equal(s[:, 0], -x[:, 0])                  # nothing before the first token
    assert torch.equal(s[:, 1:], x[:, :-1] - x[:, 1:])


def test_group_norm_normalises_each_head():
    torch.manual_seed(1)
    gn = hz.GroupNorm(128, 64)
    with torch.no_grad():
        gn.scale.uniform_(0.5, 1.5); gn.offset.uniform_(-1, 1)
    x = torch.randn(2, 5, 128)
    y = gn(x)
    xh = x.reshape(2, 5, 2, 64)
    ref = (xh - xh.mean(-1, keepdim=True)) / torch.sqrt(xh.var(-1, unbiased=False, keepdim=True) + 64e-5)
    ref = (gn.scale * ref + gn.offset).reshape(2, 5, 128)
    assert torch.allclose(y, ref, atol=1e-5)


def test_time_mix_follows_the_reference_layer():
    """TimeMix written out step by step (rwkv6_model.py:134-160) with the operator called directly."""
    torch.manual_seed(2)
    op = OPSKernelOperator(64, 16)
    tm = hz.TimeMix(op, 128, 8, 64)
    x = torch.randn(2, 16, 128)
    xs = torch.cat([torch.zeros(2, 1, 128), x[:, :-1]], 1) - x
    xm = x + xs * tm.time_mix_x
    mix = lambda d: x + xs * d(xm)
    r, k, v = tm.dense_r(mix(tm.dense_xr)), tm.dense_k(mix(tm.dense_xk)), tm.dense_v(mix(tm.dense_xv))
    w, g = tm.dense_w(mix(tm.dense_xw)), F.silu(tm.dense_g(mix(tm.dense_xg)))
    y, _ = op(r, k, v, w, tm.time_faaaa)
    ref = tm.dense_o(tm.group_norm(y) * g)
    assert torch.allclose(tm(x), ref, atol=1e-5)
    # a padded position gets w = -1e9 (rwkv6_model.py:152) and k = 0 (what :151 means to do; the
    # reference masks xk after k was computed from it): same call, masked operands
    mask = torch.ones(2, 16, dtype=torch.bool); mask[:, 5] = False
    m = mask.float()[..., None]
    y_m, _ = op(r, k * m, v, w * m + (1 - m) * -1e9, tm.time_faaaa)
    assert torch.allclose(tm(x, mask), tm.dense_o(tm.group_norm(y_m) * g), atol=1e-5)


def test_training_steps_on_cpu_reduce_the_loss():
    model = _toy(OPSKernelOperator(64, 32))
    opt = torch.optim.AdamW(model.parameters(), lr=3e-3)
    torch.manual_seed(3)
    ids = torch.randint(0, TOY["vocabulary_size"], (2, 33))
    losses = [float(hz.train_step(model, opt, ids)) for _ in range(6)]
    assert all(torch.isfinite(torch.tensor(losses)))
    assert losses[-1] < losses[0] - 0.2, losses
    for p in model.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [None, torch.bfloat16])
def test_model_step_hip_operator_matches_python_loop(dtype):
    """Same weights, same tokens: loss and gradients of one step with the HIP operator on the GPU
    (fp32 = per-timestep kernels, bf16 autocast = chunked MFMA kernels) against the python-loop
    operator on the CPU in fp32."""
    from rwkv_kernel import RWKVKernelOperator
    T = 128
    ref = _toy(OPSKernelOperator(64, T), seed=4)
    dev = torch.device("cuda:0")
    gpu = _toy(RWKVKernelOperator(64, T), seed=4).to(dev)
    gpu.load_state_dict(ref.state_dict())
    torch.manual_seed(5)
    ids = torch.randint(0, TOY["vocabulary_size"], (2, T + 1))

    def loss_and_grads(model, ids, autocast):
        model.zero_grad(set_to_none=True)
        with torch.autocast(ids.device.type, dtype=autocast, enabled=autocast is not None):
            logits = model(ids[:, :-1])
        loss = F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), ids[:, 1:].reshape(-1))
        loss.backward()
        return float(loss.detach()), {n: p.grad.detach().float().cpu() for n, p in model.named_parameters()}

    l_ref, g_ref = loss_and_grads(ref, ids, None)
    l_gpu, g_gpu = loss_and_grads(gpu, ids.to(dev), dtype)
    tol = 2e-4 if dtype is None else 3e-2
    assert abs(l_gpu - l_ref) <= tol * max(1.0, abs(l_ref)), (l_gpu, l_ref)
    worst = 0.0
    for n in g_ref:
        denom = float(g_ref[n].abs().max()) + 1e-12
        worst = max(worst, float((g_gpu[n] - g_ref[n]).abs().max()) / denom)
    assert worst <= (2e-3 if dtype is None else 8e-2), worst


@pytest.mark.gpu
def test_inference_forward_uses_the_fused_output_stage():
    """In bf16 the time-mix layer takes group norm and gate from the operator's own output stage,
    without gradients (y never written) and with them (the differentiable fused call); the logits
    agree with the unfused bf16 path and with the fp32 python-loop model on the CPU."""
    from rwkv_kernel import RWKVKernelOperator
    T = 96
    ref = _toy(OPSKernelOperator(64, T), seed=6)
    dev = torch.device("cuda:0")
    gpu = _toy(RWKVKernelOperator(64, T), seed=6).to(dev)
    gpu.load_state_dict(ref.state_dict())
    torch.manual_seed(7)
    ids = torch.randint(0, TOY["vocabulary_size"], (3, T))
    calls = []
    op = gpu.blocks[0].time_mix.rwkv_kernel
    inner = op.forward_gn_gate
    op.forward_gn_gate = lambda *a, **kw: (calls.append(1), inner(*a, **kw))[1]
    with torch.no_grad():
        want = ref(ids).float()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            fused = gpu(ids.to(dev)).float().cpu()
    assert len(calls) == TOY["num_layers"]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        trained = gpu(ids.to(dev)).float().cpu()   # gradients enabled: the differentiable fused call
    assert len(calls) == 2 * TOY["num_layers"] and trained.requires_grad
    op.forward_gn_gate = None                      # the layer then runs operator, group norm and gate one by one
    with torch.autocast("cuda", dtype=torch.bfloat16):
        unfused = gpu(ids.to(dev)).float().cpu()
    assert len(calls) == 2 * TOY["num_layers"]
    scale = float(want.abs().max())
    assert float((fused - want).abs().max()) <= 5e-2 * scale
    assert float((fused - unfused.detach()).abs().max()) <= 3e-2 * scale
    assert float((trained.detach() - unfused.detach()).abs().max()) <= 3e-2 * scale


@pytest.mark.gpu
def test_training_step_uses_the_fused_input_side():
    """With mixers of rank 32 (the rank of configuration 4) the time-mix layer under bf16 autocast takes
    its five mixed inputs from the library's shift-mix kernels: loss and gradients of one step against
    the fp32 python-loop model on the CPU, and against the same GPU model with that path switched off."""
    from rwkv_kernel import RWKVKernelOperator
    T = 128
    cfg = dict(TOY, decomposer_size=32)
    torch.manual_seed(8)
    ref = hz.RWKV6(OPSKernelOperator(64, T), **cfg)
    dev = torch.device("cuda:0")
    gpu = hz.RWKV6(RWKVKernelOperator(64, T), **cfg).to(dev)
    gpu.load_state_dict(ref.state_dict())
    torch.manual_seed(9)
    ids = torch.randint(0, TOY["vocabulary_size"], (2, T + 1))
    calls = []
    op = gpu.blocks[0].time_mix.rwkv_kernel
    inner = op.shift_mix
    op.shift_mix = lambda *a, **kw: (calls.append(1), inner(*a, **kw))[1]

    def loss_and_grads(model, ids, autocast):
        model.zero_grad(set_to_none=True)
        with torch.autocast(ids.device.type, dtype=autocast, enabled=autocast is not None):
            logits = model(ids[:, :-1])
        loss = F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), ids[:, 1:].reshape(-1))
        loss.backward()
        return float(loss.detach()), {n: p.grad.detach().float().cpu() for n, p in model.named_parameters()}

    l_ref, g_ref = loss_and_grads(ref, ids, None)
    l_gpu, g_gpu = loss_and_grads(gpu, ids.to(dev), torch.bfloat16)
    assert len(calls) == TOY["num_layers"]
    op.shift_mix = None
    l_off, g_off = loss_and_grads(gpu, ids.to(dev), torch.bfloat16)
    assert len(calls) == TOY["num_layers"]
    assert abs(l_gpu - l_ref) <= 3e-2 * max(1.0, abs(l_ref)), (l_gpu, l_ref)

    def worst(ga, gb):
        return max(float((ga[n] - gb[n]).abs().max()) / (float(gb[n].abs().max()) + 1e-12) for n in gb)

    w_fused, w_off = worst(g_gpu, g_ref), worst(g_off, g_ref)
    print("worst relative gradient error vs fp32: fused input side %.3e, torch ops %.3e" % (w_fused, w_off))
    assert w_fused <= 8e-2, w_fused
    mix_names = [n for n in g_ref if "dense_x" in n or "time_mix_x" in n]
    assert mix_names and all(torch.isfinite(g_gpu[n]).all() and float(g_gpu[n].abs().max()) > 0 for n in mix_names)


@pytest.mark.gpu
def test_config4_full_size_train_step(oracle):
    """Configuration 4 at its real size through the torch binding: 24 layers, d_model 2048, 32 heads
    of 64, FFN 7168, vocabulary 65536 (rwkv6_model.py:261-276), 8 x 1024 uniform random token ids,
    bf16 autocast, next-token cross entropy, forward + backward + AdamW -- on the calls the training
    benchmark times: the model finds the operator's fused entry points (token-shift mixes on the input
    side, group norm and gate in the operator's output stage) and every layer takes them.  Loss and
    every gradient are finite, and what one mid-stack layer's fused output-stage call saw -- r, k, v,
    w, u, gate coming in, the gradient of its output arriving -- reproduces that call's output and
    its eight gradients against float64 (the oracle's operator, torch's layer_norm autograd), all
    batch rows, at the tolerance and with the conditioning of the fused stage's own parity test."""
    import collections
    import numpy as np
    from _util import check_composite, flat_heads, fused_stage_reference, to_np
    from rwkv_kernel import RWKVKernelOperator

    dev = torch.device("cuda:0")
    B, T, N = 8, 1024, 64
    H = hz.CONFIG4["hidden_size"] // N
    print("config 4 full size", flush=True)
    op = RWKVKernelOperator(N, T)
    layer, rec = hz.CONFIG4["num_layers"] // 2, {}

    class Recording:
        """The operator as the model sees it, counting the calls and keeping the tensors of the fused
        output-stage call number `layer` (0-based)."""

        def __init__(self):
            self.taken = collections.Counter()

        def __call__(self, r, k, v, w, u):
            self.taken["plain"] += 1
            return op(r, k, v, w, u)

        def shift_mix_supported(self, *a, **kw):
            return op.shift_mix_supported(*a, **kw)

        def shift_mix(self, *a, **kw):
            self.taken["shift_mix"] += 1
            return op.shift_mix(*a, **kw)

        def shift_mix_x(self, *a, **kw):
            self.taken["shift_mix_x"] += 1
            return op.shift_mix_x(*a, **kw)

        def forward_gn_gate(self, r, k, v, w, u, gate, scale, offset, eps):
            mine = self.taken["forward_gn_gate"] == layer
            self.taken["forward_gn_gate"] += 1
            if mine:
                for name, x in zip(("r", "k", "v", "w", "u", "gate"), (r, k, v, w, u, gate)):
                    x.retain_grad()
                    rec[name] = x
                rec["scale"], rec["offset"], rec["eps"] = scale.detach().clone(), offset.detach().clone(), eps
                rec["scale_param"], rec["offset_param"] = scale, offset
            out, s = op.forward_gn_gate(r, k, v, w, u, gate, scale, offset, eps)
            if mine:
                rec["out"] = out.detach()
                # As in the fused stage's own parity test, the gradient arriving at this one call is zeroed on the
                # (token, head) groups where the norm is ill-conditioned (a head's standard deviation below 5 % of
                # the median: 1/std magnifies the bf16 rounding of y itself there, whatever computes the gradient);
                # the step goes on with that gradient.
                rec["y_ref"], _ = oracle.forward_c(*[to_np(x) for x in (r, k, v, w, u)], N)
                keep = torch.tensor(~flat_heads(rec["y_ref"], N), device=out.device).view(B, T, H, 1).expand(B, T, H, N).reshape(B, T, H * N)
                rec["flat"] = int((~keep).sum()) // N
                out.register_hook(lambda g: g * keep.to(g.dtype))
                out.register_hook(lambda g: rec.__setitem__("gout", g.detach().clone()))
            return out, s

    torch.manual_seed(11)
    with torch.device(dev):
        recorder = Recording()
        model = hz.RWKV6(recorder, **hz.CONFIG4)
    opt = torch.optim.AdamW(model.parameters(), lr=1e-4, fused=True)
    ids = torch.randint(0, hz.CONFIG4["vocabulary_size"], (B, T + 1), device=dev)
    loss = float(hz.train_step(model, opt, ids, torch.bfloat16))
    torch.cuda.synchronize()
    assert np.isfinite(loss) and abs(loss - np.log(hz.CONFIG4["vocabulary_size"])) < 2.0, loss
    for n, p in model.named_parameters():
        assert p.grad is not None and bool(torch.isfinite(p.grad).all()), n
        assert bool(torch.isfinite(p).all()), n
    L = hz.CONFIG4["num_layers"]
    assert dict(recorder.taken) == {"shift_mix": L, "shift_mix_x": 2 * L, "forward_gn_gate": L}, dict(recorder.taken)
    assert rec["r"].dtype == torch.bfloat16 and tuple(rec["r"].shape) == (B, T, H * N) and "gout" in rec

    ins = [to_np(rec[n]) for n in "rkvw"] + [to_np(rec["u"])]
    print("ill-conditioned (token, head) groups of the recorded call: %d of %d" % (rec["flat"], B * T * H), flush=True)
    want = fused_stage_reference(oracle, ins, to_np(rec["gate"]), to_np(rec["gout"]), to_np(rec["scale"]), to_np(rec["offset"]), N, rec["eps"], rec["y_ref"])
    check_composite("out", rec["out"], want["out"])
    check_composite("ggate", rec["gate"].grad, want["ggate"])
    check_composite("gscale", rec["scale_param"].grad, want["gscale"])
    check_composite("goffset", rec["offset_param"].grad, want["goffset"])
    for name, leaf in zip("gr gk gv gw gu".split(), "rkvwu"):
        check_composite(name, rec[leaf].grad, want[name])


@pytest.mark.gpu
def test_train_step_takes_logits_in_64_bits():
    """A model in double precision trains as it always did: the loss is torch's cross entropy of its logits in fp32."""
    torch.manual_seed(8)
    model = torch.nn.Embedding(31, 31).double().cuda()     # (a model whose logits are looked up)
    ids = torch.randint(0, 31, (3, 9), device="cuda")
    before = model.weight.detach().clone()
    with torch.no_grad():
        want = F.cross_entropy(model(ids[:, :-1]).float().reshape(-1, 31), ids[:, 1:].reshape(-1))
    loss = hz.train_step(model, torch.optim.SGD(model.parameters(), lr=0.1), ids)
    assert torch.equal(loss, want) and not torch.equal(model.weight, before) and bool(torch.isfinite(model.weight).all())


@pytest.mark.gpu
def test_train_step_takes_logits_of_another_shape():
    """Rows of logits one behind the other, or with a dimension between, belong to the texts' tokens in order, as torch's cross entropy takes them."""
    class Shaped(torch.nn.Embedding):
        def forward(self, ids):
            return super().forward(ids).reshape(*self.shape_of(ids), self.num_embeddings)

    torch.manual_seed(9)
    ids = torch.randint(0, 31, (3, 9), device="cuda")
    weight = torch.randn(31, 31, device="cuda")
    grads = []
    for shape_of in (lambda ids: ids.shape, lambda ids: (ids.numel(),), lambda ids: (ids.shape[0], 1, ids.shape[1]), lambda ids: (ids.numel(), 1)):
        model = Shaped(31, 31).cuda()
        model.shape_of = shape_of
        with torch.no_grad():
            model.weight.copy_(weight)
        loss = hz.train_step(model, torch.optim.SGD(model.parameters(), lr=0.1), ids)
        grads.append((loss, model.weight.grad))
    for loss, grad in grads[1:]:
        # (the same rows and sums; the embedding's backward may add them up in another order: 27 terms of less than 1 / 24 each)
        assert torch.equal(loss, grads[0][0]) and float((grad - grads[0][1]).abs().max()) <= 27 * 2.0 ** -24


@pytest.mark.gpu
def test_train_step_takes_tokens_in_bytes():
    """A model over bytes whose ids are held as such: as with the same ids in 64 bits."""
    class Bytes(torch.nn.Embedding):
        def forward(self, ids):
            return super().forward(ids.long())

    torch.manual_seed(10)
    ids = torch.randint(0, 256, (3, 9), device="cuda", dtype=torch.uint8)
    weight = torch.randn(256, 256, device="cuda")
    runs = []
    for tokens in (ids.long(), ids):
        model = Bytes(256, 256).cuda()
        with torch.no_grad():
            model.weight.copy_(weight)
        runs.append(hz.train_step(model, torch.optim.SGD(model.parameters(), lr=0.1), tokens))
    assert torch.equal(*runs)


def test_fine_tuning_steps_say_what_they_need(monkeypatch):
    """Off the GPU, or with another flavour of the package, there are no losses to run them on."""
    model = _toy(OPSKernelOperator(64, 32))
    opt = torch.optim.SGD(model.parameters(), lr=0.1)
    ids = torch.randint(0, TOY["vocabulary_size"], (2, 9))
    mask = torch.ones(2, 8, dtype=torch.bool)
    for backend in ("torch", "jax"):
        monkeypatch.setenv("KERAS_BACKEND", backend)
        for step in (lambda: hz.token_logprobs(model, ids, mask), lambda: hz.preference_step(model, opt, ids, mask, torch.zeros(2)),
                     lambda: hz.policy_step(model, opt, ids, mask, torch.zeros(2, 8), torch.zeros(2))):
            with pytest.raises(AssertionError, match="on the GPU"):
                step()


@pytest.mark.gpu
def test_train_step_takes_several_tokens_at_a_place():
    """Texts of K tokens at each place and logits for each of them: the loss is the mean over all."""
    torch.manual_seed(11)
    model = torch.nn.Embedding(31, 31).cuda()
    ids = torch.randint(0, 31, (3, 9, 4), device="cuda")
    with torch.no_grad():
        want = F.cross_entropy(model(ids[:, :-1]).reshape(-1, 31), ids[:, 1:].reshape(-1))
    loss = hz.train_step(model, torch.optim.SGD(model.parameters(), lr=0.1), ids)
    # (losses of about 4, each off by some 2^-22 of itself)
    assert abs(float(loss) - float(want)) <= 2.0 ** -20 * float(want) and bool(torch.isfinite(model.weight).all())
