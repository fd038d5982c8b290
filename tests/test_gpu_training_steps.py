"""The losses, the model and the optimizer together, as a training uses them (rwkv6_harness's steps): the gradient that reaches the
logits against the loss's formula in float64 on those very logits, and the weights against AdamW's formula on the gradients that reached them."""
import math

import pytest
import torch

import rwkv6_harness as hz
import rwkv_kernel
from test_gpu_adamw import _check as check_adamw
from test_gpu_losses import U, _grad_within, _lp64, _preference, _within

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
B, T, V = 4, 37, 777
LR, BETAS, WD = 3e-3, (0.9, 0.99), 0.1       # what check_adamw goes by


class Tap(torch.nn.Module):
    """A model whose logits can be looked at."""

    def __init__(self, model):
        super().__init__()
        self.model = model

    def forward(self, ids):
        self.logits = self.model(ids)
        if self.logits.requires_grad:
            self.logits.retain_grad()
        return self.logits


def _model(seed):
    torch.manual_seed(seed)
    return Tap(hz.RWKV6(rwkv_kernel.RWKVKernelOperator(64, 64), num_layers=2, vocabulary_size=V, hidden_size=128, decomposer_size=32, head_size=64,
                        expand_size=256).cuda())


def _texts(seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (B, T + 1), generator=g).cuda()
    lengths = torch.tensor([T, T // 2, T - 5, 9])
    mask = ((torch.arange(T)[None] >= 4) & (torch.arange(T)[None] < lengths[:, None])).cuda()
    return ids, mask, g


def _before(model, opt):
    ps = list(model.parameters())
    s = [opt.state[p] for p in ps]
    return ps, dict(params=[p.detach().clone() for p in ps], exp_avgs=[x["exp_avg"].clone() for x in s], exp_avg_sqs=[x["exp_avg_sq"].clone() for x in s],
                    scales=[x["scales"].clone() for x in s] if "scales" in s[0] else None, masters=None)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("kind", ["train", "preference", "policy"])
def test_steps(kind, bits):
    print("training step", kind, bits, flush=True)
    model, reference = _model(1), _model(2)
    ids, mask, g = _texts(3)
    ref = hz.token_logprobs(reference, ids, mask, BF16)
    opt = rwkv_kernel.AdamW(model.parameters(), lr=LR, betas=BETAS, weight_decay=WD, moment_bits=bits, max_grad_norm=0.05, seed=7)
    A = torch.randn(B, generator=g).cuda()
    counted = torch.ones_like(mask) if kind == "train" else mask
    for t in (1, 2, 3):
        old = hz.token_logprobs(model, ids, mask, BF16)
        if t > 1:
            ps, before = _before(model, opt)
        if kind == "train":
            loss = hz.train_step(model, opt, ids, BF16)
        elif kind == "preference":
            loss = hz.preference_step(model, opt, ids, mask, ref.sum(1), BF16, beta=0.2)
        else:
            loss = hz.policy_step(model, opt, ids, mask, old, A, BF16, ref_logps=ref, kl_weight=0.1)
        logits = model.logits
        assert logits.dtype == BF16 and math.isfinite(float(loss))
        leaf, lp, c_mask, E, p = _lp64(logits, ids[:, 1:], counted)
        n = c_mask.sum()
        if kind == "train":
            want, c = -lp.sum() / n, c_mask / n.double()
            c_off, off = 4 * U * c, ((E + 4 * U * lp.abs()) * c_mask).sum() / n
        elif kind == "preference":
            want, s, d = _preference(lp, c_mask, ref.sum(1), 0.2, "sigmoid", 0.0, False)
            d_off = (E * c_mask).sum(1)
            d_off = d_off[:2] + d_off[2:]
            c = 0.2 / 2 * c_mask.double()
            c_off, off = (0.04 / 4 * d_off.repeat(2) / 2)[:, None] * c_mask + 4 * U * c, 0.2 * d_off.mean()
        else:
            # the sampling model's log probabilities are this model's: the ratio is 1 but for their rounding, far from where it is clipped
            ratio = torch.exp(lp - old.cpu().double())
            assert float((ratio.detach() - 1).abs().max()) < 0.1
            e = ref.cpu().double() - lp
            A64 = A.cpu().double()[:, None]
            each = -ratio * A64 + 0.1 * (torch.exp(e) - e - 1)
            want = (each * c_mask).sum() / n
            size = ratio.detach() * A64.abs() + 0.1 * (1 + (e.exp() - 1).detach().abs() + e.detach().abs())
            c = size * c_mask / n
            lp_off = E + 4 * U * lp.abs()
            c_off, off = c * (4 * lp_off + 16 * U), (c * (2 * lp_off + 16 * U)).sum()
        _within("loss", loss, want, off + 4 * U * want.abs())
        want.backward()
        _grad_within("grad", logits.grad, leaf.grad, p, c, c_off, E, BF16)
        if t > 1:
            after = _before(model, opt)[1]
            before["grads"] = [q.grad for q in ps]
            norm = math.sqrt(sum(float(x.double().square().sum()) for x in before["grads"]))
            assert abs(float(opt.last_grad_norm) - norm) <= 2 * U * norm
            check_adamw(before, after, norm, 0.05, bits, t)


def test_train_step_is_the_plain_one():
    """The step's loss and the gradients of the weights beside torch's cross entropy over the same model's logits in fp32: the gradients by the logits
    are the same numbers rounded from fp32 values that differ by less than 2^-17, so a few of them by one step of bf16 (2^-8): in the 2-norm
    less than a tenth of that."""
    model = _model(4)
    ids, _, _ = _texts(5)
    opt = torch.optim.SGD(model.parameters(), lr=0.0)
    loss = hz.train_step(model, opt, ids, BF16)
    ours = model.logits.grad.clone()
    opt.zero_grad(set_to_none=True)
    with torch.autocast("cuda", dtype=BF16):
        logits = model(ids[:, :-1])
    want = torch.nn.functional.cross_entropy(logits.float().reshape(-1, V), ids[:, 1:].reshape(-1))
    want.backward()
    assert abs(float(loss) - float(want)) <= 2.0 ** -20 * float(want)
    assert float((ours.double() - logits.grad.double()).norm() / logits.grad.double().norm()) <= 0.1 * 2.0 ** -8
