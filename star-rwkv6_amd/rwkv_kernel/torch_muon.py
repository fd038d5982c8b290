"""Orthogonalized weight updates and the optimizer with them, on libwkv6_gfx950.so.  Not part of the reference, which takes its optimizer from the framework
above it.

    orthogonalize(matrices)               each brought near to the nearest matrix with orthonormal rows or columns, by Newton-Schulz products
    muon_step(params, grads, momenta, lr) one step of the optimizer: momentum, orthogonalized updates, weight decay
    Muon                                  the optimizer, for a model's weight matrices (AdamW takes the rest: embeddings, norms, biases, the head)

Matrices are (.., rows, columns) in bf16, fp16 or fp32 on the GPU; dimensions before the last two are a batch.  All products have 22 bits whatever the matrices'
dtype (three fp16 products on the matrix instructions, accumulated in fp32): small singular values grow by a^steps, and what a product in
16 bits loses of them with it.  Calls go to the current stream of the tensors' device, allocate nothing but their results and a workspace, never
synchronise, and can be captured into a graph.
"""
import math

import torch

from . import _native

COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # of X, A X and A A X: singular values from 0.003 to 1 come to 0.7 .. 1.2 in five steps


def _coefficients(coefficients, steps):
    """One triple for all steps, or one for each, as a flat list."""
    assert isinstance(steps, int) and 1 <= steps <= 100, "steps must be 1 to 100"
    rows = [tuple(float(x) for x in coefficients)] * steps if not hasattr(coefficients[0], "__len__") else [tuple(float(x) for x in r) for r in coefficients]
    assert len(rows) == steps and all(len(r) == 3 and all(math.isfinite(x) for x in r) for r in rows), "coefficients must be three numbers, or three for each step"
    return [x for r in rows for x in r]


def orthogonalize(matrices, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """X = G / (|G| + eps) with |G| the 2-norm of all elements, then `steps` times X = a X + b A X + c A A X with A = X X^T (of a matrix with more rows than columns its
    transpose's, transposed): the singular vectors of G with singular values near 1.  Without a
    derivative: a matrix that requires a gradient is refused where gradients are recorded, and one with a tangent (forward mode).

    matrices: a tensor (.., rows, columns), or a list of such, of one dtype and any shapes; they go through together.  Returns the same in new tensors of
    their dtype.  Of a G whose norm is far below eps, and so of a result far below 1, an element is good to some 2^-26, and not to its own size.  coefficients:
    (a, b, c), or one such triple for each step; what leaves the range of +-64 on the way (not with coefficients that keep singular values of 0 .. 1.2
    in it) ends as NaN."""
    flat = _coefficients(coefficients, steps)
    assert eps >= 0
    single = isinstance(matrices, torch.Tensor)
    out = _native.load_torch().orthogonalize([matrices] if single else list(matrices), flat, float(eps))
    return out[0] if single else out


def _rate(scale, shape):
    if scale == "shape":
        return math.sqrt(max(1.0, shape[-2] / max(1, shape[-1])))
    if scale == "rms":
        return 0.2 * math.sqrt(max(shape[-2:]))
    assert not isinstance(scale, str) and float(scale) >= 0, "scale must be 'shape', 'rms' or a number that is not negative"
    return float(scale)


def muon_step(params, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, scale="shape", steps=5, coefficients=COEFFICIENTS, eps=1e-7, masters=None):
    """One step over lists of matrices, in place:
        buf = momentum buf + (1 - momentum) g
        u = (1 - momentum) g + momentum buf if nesterov else buf
        p = p (1 - lr weight_decay) - lr rate orthogonalize(u)
    params, grads: of one dtype (bf16, fp16, fp32); params contiguous, none twice and no two with elements in common, and a gradient with none of what is written.  momenta: buf, fp32.  lr: a number, or one
    fp32 value on the device (which a captured graph's replays read anew).  scale: rate is sqrt(max(1, rows / columns)) ("shape"), 0.2
    sqrt(max(rows, columns)) ("rms": an update's elements are then as large as AdamW's), or a number.  masters: fp32 weights that are updated in the params'
    place, the params their rounded copies."""
    params = list(params)
    device_lr = lr if isinstance(lr, torch.Tensor) else None
    assert device_lr is not None or lr >= 0
    assert 0 <= momentum < 1 and weight_decay >= 0 and eps >= 0
    assert all(p.dim() >= 2 for p in params), "parameters must be matrices"
    _native.load_torch().muon_step(params, list(grads), list(momenta), list(masters or ()), [_rate(scale, p.shape) for p in params], _coefficients(coefficients, steps), float(eps),
                                   float(momentum), bool(nesterov), 0.0 if device_lr is not None else float(lr), device_lr, float(weight_decay))


class Muon(torch.optim.Optimizer):
    """The optimizer on ``muon_step``: all matrices of a group in one call, without a synchronisation.

    params: matrices alone (a parameter with fewer than two dimensions is refused).  master_weights: 16-bit parameters are updated in fp32 behind their rounded
    copies.  lr of a group may be an fp32 tensor on the device.  A step can be captured into a graph once every parameter has its state, after a
    first step.  State of a parameter: "momentum", fp32, and where there is one "master"."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, scale="shape", steps=5, coefficients=COEFFICIENTS, eps=1e-7, master_weights=False):
        assert isinstance(lr, torch.Tensor) or lr >= 0
        assert 0 <= momentum < 1 and weight_decay >= 0 and eps >= 0
        _rate(scale, (1, 1))
        _coefficients(coefficients, steps)
        self.master_weights = master_weights
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, scale=scale, steps=steps, coefficients=coefficients, eps=eps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        assert all(p.dim() >= 2 for p in self.param_groups[-1]["params"]), "parameters must be matrices"

    def _has_master(self, p):
        return self.master_weights and p.dtype != torch.float32

    def _state_of(self, p):
        s = self.state[p]
        if "momentum" not in s:
            # (into a graph each replay would begin from nothing again)
            assert not torch.cuda.is_current_stream_capturing(), "a step is captured after a first one that gave every parameter its state"
            s["momentum"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            if self._has_master(p):
                s["master"] = p.detach().to(torch.float32, memory_format=torch.contiguous_format, copy=True)
        return s

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            together = {}
            for p in group["params"]:
                if p.grad is not None:
                    assert p.is_cuda, "parameters must be on the GPU"
                    together.setdefault((p.device, p.dtype), []).append(p)
            for ps in together.values():
                states = [self._state_of(p) for p in ps]
                muon_step(ps, [p.grad for p in ps], [s["momentum"] for s in states], group["lr"], group["momentum"], group["nesterov"], group["weight_decay"],
                          group["scale"], group["steps"], group["coefficients"], group["eps"], masters=[s["master"] for s in states] if "master" in states[0] else None)
        return loss

    def load_state_dict(self, state_dict):
        """As every optimizer's, but states keep their own dtypes.  A state without the masters that this optimizer has, or with others, is refused."""
        theirs = [i for group in state_dict["param_groups"] for i in group["params"]]
        ours = [p for group in self.param_groups for p in group["params"]]
        for i, p in zip(theirs, ours):
            s = state_dict["state"].get(i)
            if s:
                assert ("master" in s) == self._has_master(p), "saved %s master, by an optimizer with other master_weights or parameters of another dtype" % (
                    "with a" if "master" in s else "without a")
        super().load_state_dict(state_dict)
        for i, p in zip(theirs, ours):
            if i in state_dict["state"]:
                self.state[p] = {k: v.detach().clone().to(p.device) if isinstance(v, torch.Tensor) else v for k, v in state_dict["state"][i].items()}

    def __getstate__(self):
        return dict(super().__getstate__(), master_weights=self.master_weights)
