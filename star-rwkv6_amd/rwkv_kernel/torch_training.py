"""What a training step does behind the model's last layer, on libwkv6_gfx950.so: losses over logits with their gradients, and
the optimizer's step.  Not part of the reference, which takes both from the framework above it.

    cross_entropy(logits, ids)                       the next-token loss
    token_logprobs(logits, ids)                      log probabilities of the tokens that stand there
    preference_loss(logits, ids, mask, ...)          pairs of chosen and rejected texts
    policy_loss(logits, ids, mask, ...)              sampled texts and their advantages
    grad_norm(grads), adamw_step(params, ...), AdamW the optimizer

Logits are (B, T, V) or, for the first two, (N, V), in bf16, fp16 or fp32 on the GPU; batch and time may be strided or broadcast (a
slice of a longer sequence is taken as it is).  All arithmetic on them is in fp32, sums over tokens in fp64; the gradient has the
logits' dtype and is rounded once.  `ids` (int64) names the token that stands at each place: for a model's outputs at
positions 0 .. T-1 these are the input ids from position 1 on.  A token counts if its `mask` is not zero (None: all do) and its id is not
negative; the logits of one that does not are never read, and get a gradient of zero.  An id of V or more makes its token's log
probability, and with it the loss, NaN.  A temperature is the fp32 number nearest to what is given; logits are divided by it in 64 bits.

Calls go to the current stream of the tensors' device, allocate nothing but their results and workspaces, never
synchronise, and can be captured into a graph (a backward only where no graph of its leaves is alive that another stream made: torch's engine
would make that stream wait for the capture, and the process ends).

The losses have first derivatives.  A gradient taken with create_graph has its value, and a derivative of it is refused.
"""
import torch

from . import _native

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_REDUCE = {"sum": 0, "mean": 1, "mean_of_texts": 2}
_PREFERENCE = {"sigmoid": 0, "hinge": 1, "ipo": 2}
SCALE_BLOCK = 256   # elements that share a scale where moments are held in 8 bits


def _rows(logits, ids, mask, flat_allowed):
    """(logits (B,T,V) with rows in one piece, ids (B,T), mask (B,T) bytes or None), checked."""
    if _native.load_torch().plain_rows(logits, ids, mask):
        return logits, ids, mask
    assert isinstance(logits, torch.Tensor) and logits.is_cuda, "logits must be on the GPU"
    assert logits.dtype in _DTYPES, "logits must be bfloat16, float16 or float32"
    assert logits.dim() == 3 or (flat_allowed and logits.dim() == 2), "logits must be (batch, time, vocabulary)%s" % (
        " or (tokens, vocabulary)" if flat_allowed else "")
    assert ids.dtype == torch.int64 and ids.shape == logits.shape[:-1] and ids.device == logits.device, \
        "ids must be int64, of the logits' shape without the vocabulary, on their device"
    assert logits.shape[-1] > 0, "the vocabulary is empty"
    if mask is not None:
        assert mask.dtype in (torch.bool, torch.uint8) and mask.shape == ids.shape and mask.device == logits.device, \
            "mask must be bool or uint8, of the ids' shape, on their device"
    if logits.dim() == 2:
        logits, ids, mask = logits[None], ids[None], None if mask is None else mask[None]
    if logits.stride(2) != 1 and logits.shape[2] > 1:
        logits = logits.contiguous()
    return logits, ids.contiguous(), None if mask is None else mask.contiguous()


def _per_token(x, ids, name):
    if x is None:
        return None
    assert x.shape == ids.shape and x.device == ids.device and x.is_floating_point(), "%s must be (batch, time), on the logits' device" % name
    return x if x.dtype == torch.float32 and x.is_contiguous() else x.to(torch.float32).contiguous()


def token_logprobs(logits, ids, mask=None, temperature=1.0):
    """log softmax(logits / temperature) at ids: fp32, of ids' shape, 0 where a token does not count.  Differentiable in logits."""
    shape = ids.shape
    logits, ids, mask = _rows(logits, ids, mask, True)
    assert temperature > 0
    if ids.numel() == 0:
        return logits.float().sum(-1).reshape(shape)
    lp = _native.load_torch().token_logprobs(logits, ids, mask, float(temperature))
    return lp if len(shape) == 2 else lp.reshape(shape)


def cross_entropy(logits, ids, mask=None, reduction="mean"):
    """The mean (or "sum") over the tokens that count of -log softmax(logits) at ids, an fp32 scalar, differentiable in logits; 0 if no
    token counts.  With a gradient wanted the logits are read once, and their gradient is written in the same pass."""
    logits, ids, mask = _rows(logits, ids, mask, True)
    assert reduction in ("mean", "sum"), "reduction must be 'mean' or 'sum'"
    if ids.numel() == 0:
        return logits.float().sum()
    return _native.load_torch().cross_entropy(logits, ids, mask, _REDUCE[reduction])


def preference_loss(logits, ids, mask=None, ref_logps=None, beta=0.1, kind="sigmoid", label_smoothing=0.0, average=False):
    """A loss on pairs of texts: of the batch of 2 P texts, text i is chosen over text P + i.

    With s the sum of a text's token log probabilities (`average`: their mean) and d = (s_chosen - s_rejected) minus the same of
    `ref_logps` (2 P values, a reference model's; None: zero), the loss is the mean over the pairs of
        "sigmoid"  -(1 - label_smoothing) log sigmoid(beta d) - label_smoothing log sigmoid(-beta d)
        "hinge"    max(0, 1 - beta d)
        "ipo"      (d - 1 / (2 beta))^2
    Returns (loss, s): an fp32 scalar, differentiable in logits, and the 2 P values of s, which carry no gradient.  The coefficient of a
    token's gradient depends on both whole texts, so the logits are read twice."""
    logits, ids, mask = _rows(logits, ids, mask, False)
    B = logits.shape[0]
    assert B % 2 == 0 and B > 0, "the batch holds the chosen texts, then as many rejected ones"
    assert kind in _PREFERENCE, "kind must be 'sigmoid', 'hinge' or 'ipo'"
    assert beta > 0 and 0.0 <= label_smoothing < 0.5
    assert label_smoothing == 0.0 or kind == "sigmoid", "label_smoothing belongs to the sigmoid loss"
    if ref_logps is not None:
        assert ref_logps.shape == (B,) and ref_logps.device == logits.device and ref_logps.is_floating_point(), \
            "ref_logps must hold one value for each text, on the logits' device"
        ref_logps = ref_logps.to(torch.float32).contiguous()
    assert ids.numel() > 0, "the texts are empty"
    return _native.load_torch().preference_loss(logits, ids, mask, ref_logps, _PREFERENCE[kind], float(beta), float(label_smoothing), bool(average))


def policy_loss(logits, ids, mask, old_logps, advantages, ref_logps=None, clip_low=0.2, clip_high=0.2, kl_weight=0.0, temperature=1.0,
                reduction="mean"):
    """The clipped policy loss with a KL term.  With lp a token's log probability, ratio = exp(lp - old_logps) (`old_logps` (B, T), the
    sampling model's; None: the sampling model is this one, the ratio 1 with lp's gradient) and e = ref_logps - lp, the loss is the mean of
        kl_weight (exp(e) - e - 1) - min(ratio A, clamp(ratio, 1 - clip_low, 1 + clip_high) A)
    over all tokens that count ("mean"), or over each text's and then over the texts that have any ("mean_of_texts").  `advantages`: (B,)
    or (B, T).  `ref_logps` (B, T): a reference model's; None: no KL term, and with a kl_weight of 0 it is in the means alone.  None of the three gets a gradient.
    Returns (loss, lp, means): an fp32 scalar, differentiable in logits, and without gradients lp (B, T) and the same means of
    exp(e) - e - 1 and of whether the clamped term was the smaller one (2 values).  With a gradient wanted the logits are read once."""
    logits, ids, mask = _rows(logits, ids, mask, False)
    B = logits.shape[0]
    assert temperature > 0 and clip_low >= 0 and clip_high >= 0 and kl_weight >= 0
    assert reduction in ("mean", "mean_of_texts"), "reduction must be 'mean' or 'mean_of_texts'"
    old_logps, ref_logps = _per_token(old_logps, ids, "old_logps"), _per_token(ref_logps, ids, "ref_logps")
    assert advantages.shape in ((B,), ids.shape) and advantages.device == logits.device and advantages.is_floating_point(), \
        "advantages must be (batch,) or (batch, time), on the logits' device"
    assert ids.numel() > 0, "the texts are empty"
    advantages = advantages.to(torch.float32)
    return _native.load_torch().policy_loss(logits, ids, mask, old_logps, advantages, ref_logps, float(clip_low), float(clip_high),
                                            float(kl_weight), float(temperature), _REDUCE[reduction])


def grad_norm(grads):
    """The 2-norm of all tensors of a list together, an fp32 scalar on their device; one dtype.  Added up in fp64, always in the same order."""
    return _native.load_torch().grad_norm(list(grads))


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, scales=None, masters=None,
               max_grad_norm=None, grad_norm=None, skip_nonfinite=False, seed=0):
    """One AdamW step over lists of tensors, in place:
        g = g * max_grad_norm / max(norm, max_grad_norm)                 (max_grad_norm None: g as it is)
        m = b1 m + (1 - b1) g,  v = b2 v + (1 - b2) g^2,  t = step = step + 1
        p = p (1 - lr weight_decay) - lr / (1 - b1^t) m / (sqrt(v / (1 - b2^t)) + eps)
    params, grads: of one dtype (bf16, fp16, fp32), any dense layout, none twice and no two with elements in common.  step: one int64 on the device, that of no other call under way.  lr: a number, or one fp32 value on the
    device (which a captured graph's replays read anew).  masters: fp32 weights that are updated in the params' place, the
    params their rounded copies.  grad_norm: the norm to clip by, one fp32 value on the device; None: that of these gradients.  skip_nonfinite: a
    step whose norm is not finite changes nothing.  Returns the norm, None if nothing asked for it.

    exp_avgs, exp_avg_sqs: m and v in fp32.  Or m and sqrt(v) as float8_e4m3fn, each times its scale: scales, fp32 (ceil(numel / 256), 2), has a scale
    of either for each 256 elements.  They are rounded to one of the two nearest values at random, so that their mean is kept and small
    changes are not lost; `seed`, step and the place in list and tensor decide, so the same call gives the same result."""
    device_lr = lr if isinstance(lr, torch.Tensor) else None
    assert device_lr is not None or lr >= 0
    assert max_grad_norm is None or max_grad_norm > 0, "max_grad_norm must be positive"
    return _native.load_torch().adamw_step(
        list(params), list(grads), list(exp_avgs), list(exp_avg_sqs), step, list(scales or ()), list(masters or ()), device_lr,
        0.0 if device_lr is not None else float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
        float(max_grad_norm or 0.0), bool(skip_nonfinite), grad_norm, int(seed) & 0xFFFFFFFF)


class AdamW(torch.optim.Optimizer):
    """AdamW on ``adamw_step``: the norm of all gradients, where it is asked for, and one step for all parameters of a group in a few
    launches, without a synchronisation.

    moment_bits: 32 or 8 (see adamw_step; a parameter then has 2 bytes of state and a little).  master_weights: 16-bit parameters are
    updated in fp32 behind their rounded copies.  max_grad_norm: gradients of all groups
    together are clipped to it;
    ``last_grad_norm`` is their norm, on the device.  skip_nonfinite: a step whose norm is not finite is left out.  lr of a group may be an
    fp32 tensor on the device.  A step can be captured into a graph once every parameter has its state, after a first step.

    State of a parameter: "step" (shared by parameters with one history), "exp_avg", "exp_avg_sq", and where they are in 8 bits
    "scales", where there is one "master"."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, moment_bits=32, master_weights=False,
                 max_grad_norm=None, skip_nonfinite=False, seed=0):
        assert moment_bits in (8, 32), "moment_bits must be 8 or 32"
        assert max_grad_norm is None or max_grad_norm > 0, "max_grad_norm must be positive"
        assert isinstance(lr, torch.Tensor) or lr >= 0
        assert 0 <= betas[0] < 1 and 0 <= betas[1] < 1 and eps >= 0 and weight_decay >= 0
        self.moment_bits, self.master_weights = moment_bits, master_weights
        self.max_grad_norm, self.skip_nonfinite, self.seed = max_grad_norm, skip_nonfinite, seed
        self.last_grad_norm = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    def _new_state(self, p, step):
        # (into a graph each replay would begin from nothing again)
        assert not torch.cuda.is_current_stream_capturing(), "a step is captured after a first one that gave every parameter its state"
        s = self.state[p]
        s["step"] = step
        dtype = torch.float8_e4m3fn if self.moment_bits == 8 else torch.float32
        for name in ("exp_avg", "exp_avg_sq"):
            if self.moment_bits == 8:
                s[name] = torch.zeros_like(p, dtype=torch.uint8, memory_format=torch.preserve_format).view(dtype)
            else:
                s[name] = torch.zeros_like(p, dtype=dtype, memory_format=torch.preserve_format)
        if self.moment_bits == 8:
            s["scales"] = torch.zeros((p.numel() + SCALE_BLOCK - 1) // SCALE_BLOCK, 2, dtype=torch.float32, device=p.device)
        if self._has_master(p):
            s["master"] = p.detach().to(torch.float32, memory_format=torch.preserve_format)

    def _cohorts(self):
        """Parameters that have a gradient, by (group, device, dtype, what steps they have taken): what one call can take together."""
        cohorts, new = {}, {}
        for i, group in enumerate(self.param_groups):
            for p in group["params"]:
                if p.grad is None:
                    continue
                assert p.is_cuda, "parameters must be on the GPU"
                if p not in self.state or "step" not in self.state[p]:
                    key = (i, p.device, p.dtype)
                    if key not in new:
                        new[key] = torch.zeros((), dtype=torch.int64, device=p.device)
                    self._new_state(p, new[key])
                cohorts.setdefault((i, p.device, p.dtype, id(self.state[p]["step"])), []).append(p)
        # parameters that share a step but do not take this one stay with the old one
        taking = {}
        for key, ps in cohorts.items():
            taking.setdefault(key[3], []).extend(ps)
        for group in self.param_groups:
            for p in group["params"]:
                if p.grad is None and p in self.state and id(self.state[p].get("step")) in taking:
                    for q in taking.pop(id(self.state[p]["step"])):
                        key, old = ("after", q.dtype, id(self.state[q]["step"])), self.state[q]["step"]
                        if key not in new:
                            assert not torch.cuda.is_current_stream_capturing(), "a captured step takes the parameters that the step before it took"
                            new[key] = old.clone()
                        self.state[q]["step"] = new[key]
        return [(key[0], ps) for key, ps in cohorts.items()]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        cohorts = self._cohorts()
        if not cohorts:
            return loss
        norm = None
        if self.max_grad_norm is not None or self.skip_nonfinite:
            by_dtype = {}
            for _, ps in cohorts:
                by_dtype.setdefault((ps[0].device, ps[0].dtype), []).extend(p.grad for p in ps)
            assert len({device for device, _ in by_dtype}) == 1, "gradients that are clipped together must be on one GPU"
            norms = [grad_norm(gs) for gs in by_dtype.values()]
            norm = norms[0] if len(norms) == 1 else torch.stack(norms).double().square().sum().sqrt().float()
        self.last_grad_norm = norm
        for n, (i, ps) in enumerate(cohorts):
            group, states = self.param_groups[i], [self.state[p] for p in ps]
            with torch.cuda.device(ps[0].device):
                adamw_step(ps, [p.grad for p in ps], [s["exp_avg"] for s in states], [s["exp_avg_sq"] for s in states], states[0]["step"], group["lr"],
                           group["betas"], group["eps"], group["weight_decay"],
                           scales=[s["scales"] for s in states] if "scales" in states[0] else None,
                           masters=[s["master"] for s in states] if "master" in states[0] else None,
                           max_grad_norm=self.max_grad_norm, grad_norm=norm, skip_nonfinite=self.skip_nonfinite, seed=self.seed + n)
        return loss

    def _has_master(self, p):
        return self.master_weights and p.dtype != torch.float32

    def load_state_dict(self, state_dict):
        """As every optimizer's, but states keep their own dtypes, and parameters with one step count share it again.  A state with moments in another
        number of bits, without the masters that this optimizer has or with others, is refused."""
        theirs = [i for group in state_dict["param_groups"] for i in group["params"]]
        for i, p in zip(theirs, [p for group in self.param_groups for p in group["params"]]):
            s = state_dict["state"].get(i)
            if s:
                assert ("scales" in s) == (self.moment_bits == 8), "the moments were saved in another number of bits"
                assert ("master" in s) == self._has_master(p), "saved %s master, by an optimizer with other master_weights or parameters of another dtype" % (
                    "with a" if "master" in s else "without a")
        super().load_state_dict(state_dict)
        ours = [(n, p) for n, group in enumerate(self.param_groups) for p in group["params"]]
        shared = {}
        for (n, p), i in zip(ours, theirs):
            if i not in state_dict["state"]:
                continue
            s = {k: v.detach().clone().to(p.device) if isinstance(v, torch.Tensor) else v for k, v in state_dict["state"][i].items()}
            s["step"] = shared.setdefault((n, p.device, p.dtype, int(s["step"])), s["step"].to(torch.int64).reshape(()))
            self.state[p] = s

    def __getstate__(self):
        own = ("moment_bits", "master_weights", "max_grad_norm", "skip_nonfinite", "seed", "last_grad_norm")
        return dict(super().__getstate__(), **{k: getattr(self, k) for k in own})
