"""RWKV-6 model harness in plain torch around the WKV6 operator.

Measurement and test harness only: it exists so that the operator can be exercised the way its
caller does it -- once per layer, forward and backward, inside a real next-token training step --
without the Keras / bert4keras3 stack the reference's model file needs.  The layers restate
rwkv6_model.py of the reference, module by module:

    TimeShift        rwkv6_model.py:37-45    (x shifted right by one token) - x
    DecomposerDense  rwkv6_model.py:11-34    Dense(tanh, no bias) -> Dense(bias): the low-rank mixers
    TimeMix          rwkv6_model.py:117-185  data-dependent token-shift mixing, r/k/v/w/g projections,
                                             x, _ = rwkv_kernel(r, k, v, w, time_faaaa), per-head group
                                             norm (eps 64e-5), output projection of x * g
    ChannelMix       rwkv6_model.py:50-82    relu^2 key, sigmoid receptance
    GroupNorm        rwkv6_model.py:83-115
    Block            rwkv6_model.py:187-208  x + TimeMix(LN(x)); x + ChannelMix(LN(x))
    RWKV6            rwkv6_model.py:259-274  Embedding -> LN -> blocks -> LN -> Dense(vocab)

`rwkv_kernel` is any object with the operator's call signature `x, state = op(r, k, v, w, u)`:
rwkv_kernel.RWKVKernelOperator (the HIP library) on a GPU, rwkv_kernel.OPSKernelOperator (the
python loop) anywhere.  Initialisation is random (small normal / uniform decay range); no
checkpoint format is read or written here.
"""
import math
import os

import torch
from torch import nn
import torch.nn.functional as F


def time_shift(x):
    """rwkv6_model.py:40-43: previous token (zero for the first) minus the token itself."""
    return F.pad(x, (0, 0, 1, 0))[:, :-1, :] - x


def _kernels(x):
    """The operator package where it has kernels for this tensor (its torch flavour, on the GPU, in 16 or 32 bits), else None."""
    if not x.is_cuda or x.dtype not in (torch.bfloat16, torch.float16, torch.float32) or os.environ.get("KERAS_BACKEND") != "torch":
        return None
    import rwkv_kernel

    return rwkv_kernel


def _as_built(module, cls):
    """Whether a call of this module is its class's forward and nothing else, so that what stands in for it is the same: no hooks, no wrapper or
    subclass, no forward of its own, not compiled."""
    return type(module) is cls and "forward" not in module.__dict__ and getattr(module, "_compiled_call_impl", None) is None \
        and not (module._forward_hooks or module._forward_pre_hooks or module._backward_hooks or module._backward_pre_hooks) \
        and not nn.modules.module._has_any_global_hook()


def _bf16_autocast():
    return torch.is_autocast_enabled('cuda') and torch.get_autocast_dtype('cuda') == torch.bfloat16


def _goes_beside(x, branch):
    """Whether the sum is in x's type, and the kernel has the two."""
    return branch.dtype == x.dtype or (x.dtype == torch.float32 and branch.dtype in (torch.bfloat16, torch.float16))


def _rounds(x, reader):
    """Whether this module, the only one to read the norm of x, would round it to bf16 first: under bf16 autocast on the GPU, a projection or what begins with the
    library's input side."""
    if not (x.is_cuda and _bf16_autocast()):
        return False
    return _as_built(reader, nn.Linear) or ((_as_built(reader, TimeMix) or _as_built(reader, ChannelMix)) and reader.rounds_its_input())


def add_norm(x, branch, norm, rounded=False):
    """(x + branch, the norm of it), in one kernel where the package has it; branch None: (x, the norm of x).  rounded: under bf16 autocast the norm's readers
    round it to bf16, and it comes out so there."""
    kernels, autocast = _kernels(x), torch.is_autocast_enabled('cuda')
    if kernels is None or not _as_built(norm, nn.LayerNorm) or norm.normalized_shape != (x.shape[-1],) or x.shape[-1] > kernels.torch_layers.MOST_CHANNELS \
            or (x.dtype != torch.float32 and autocast) or (branch is not None and (branch.shape != x.shape or not _goes_beside(x, branch))):
        x = x if branch is None else x + branch
        return x, norm(x)
    dtype = torch.bfloat16 if rounded and _bf16_autocast() else x.dtype
    if branch is None:
        return x, kernels.layer_norm(x, norm.weight, norm.bias, norm.eps, dtype=dtype)
    h, x = kernels.layer_norm(x, norm.weight, norm.bias, norm.eps, add=branch, dtype=dtype)
    return x, h


class DecomposerDense(nn.Module):
    def __init__(self, hidden_size, decomposer_size, use_bias=False):
        super().__init__()
        self.dense_a = nn.Linear(hidden_size, decomposer_size, bias=False)
        self.dense_b = nn.Linear(decomposer_size, hidden_size, bias=use_bias)

    def forward(self, x):
        return self.dense_b(torch.tanh(self.dense_a(x)))


class GroupNorm(nn.Module):
    """Layer norm over each head's channels with a per-(head, channel) scale and offset."""

    def __init__(self, hidden_size, head_size, epsilon=64e-5):
        super().__init__()
        assert hidden_size % head_size == 0
        self.num_heads, self.head_size, self.epsilon = hidden_size // head_size, head_size, epsilon
        self.scale = nn.Parameter(torch.ones(self.num_heads, head_size))
        self.offset = nn.Parameter(torch.zeros(self.num_heads, head_size))

    def forward(self, x):
        B, T, C = x.shape
        x = x.reshape(B, T, self.num_heads, self.head_size)
        x = F.layer_norm(x.float(), (self.head_size,), None, None, self.epsilon).to(x.dtype)
        return (self.scale.to(x.dtype) * x + self.offset.to(x.dtype)).reshape(B, T, C)


class TimeMix(nn.Module):
    def __init__(self, rwkv_kernel, hidden_size, decomposer_size, head_size):
        super().__init__()
        assert hidden_size % head_size == 0
        self.rwkv_kernel = rwkv_kernel
        self.hidden_size, self.head_size = hidden_size, head_size
        self.time_mix_x = nn.Parameter(torch.rand(hidden_size))
        self.dense_xr = DecomposerDense(hidden_size, decomposer_size, use_bias=True)
        self.dense_xw = DecomposerDense(hidden_size, decomposer_size, use_bias=True)
        self.dense_xk = DecomposerDense(hidden_size, decomposer_size, use_bias=True)
        self.dense_xv = DecomposerDense(hidden_size, decomposer_size, use_bias=True)
        self.dense_xg = DecomposerDense(hidden_size, decomposer_size, use_bias=True)
        self.dense_r = nn.Linear(hidden_size, hidden_size, bias=False)
        self.dense_k = nn.Linear(hidden_size, hidden_size, bias=False)
        self.dense_v = nn.Linear(hidden_size, hidden_size, bias=False)
        self.dense_w = DecomposerDense(hidden_size, head_size, use_bias=True)
        self.dense_g = nn.Linear(hidden_size, hidden_size, bias=False)
        self.time_faaaa = nn.Parameter(0.5 * torch.randn(hidden_size // head_size, head_size))
        self.group_norm = GroupNorm(hidden_size, head_size)
        self.dense_o = nn.Linear(hidden_size, hidden_size, bias=False)
        # the raw decay input w: the bias spreads it over [-6, 1] (decay exp(-exp(w)) from 0.998 to 0.07)
        with torch.no_grad():
            self.dense_w.dense_b.bias.uniform_(-6.0, 1.0)

    def rounds_its_input(self):
        """Whether the input is only read in bf16 under bf16 autocast on the GPU: by the library's input side."""
        return hasattr(self.rwkv_kernel, "shift_mix") and self.hidden_size % 64 == 0 and self.dense_xr.dense_a.out_features in (32, 64)

    def _mixed_inputs(self, x):
        """xr, xk, xv, xw, xg of rwkv6_model.py:134-145."""
        mixers = (self.dense_xr, self.dense_xk, self.dense_xv, self.dense_xw, self.dense_xg)
        fused = getattr(self.rwkv_kernel, "shift_mix", None)
        if fused is not None and x.is_cuda and torch.is_autocast_enabled('cuda') and torch.get_autocast_dtype('cuda') == torch.bfloat16:
            xb = x.to(torch.bfloat16).contiguous()
            if self.rwkv_kernel.shift_mix_supported(xb, mixers[0].dense_a.out_features):
                # token shift, x_mix and the five rank-R expansions in the operator library's kernels
                return fused(xb, self.time_mix_x,
                             torch.cat([m.dense_a.weight for m in mixers]),
                             torch.stack([m.dense_b.weight for m in mixers]),
                             torch.stack([m.dense_b.bias for m in mixers]))
        x_shift = time_shift(x)
        x_mix = x + x_shift * self.time_mix_x.to(x.dtype)
        return tuple(x + x_shift * m(x_mix) for m in mixers)

    def forward(self, x, mask=None):
        xr, xk, xv, xw, xg = self._mixed_inputs(x)
        r, k, v, w, g = self.dense_r(xr), self.dense_k(xk), self.dense_v(xv), self.dense_w(xw), F.silu(self.dense_g(xg))
        if mask is not None:
            # Padded tokens neither write to the state nor decay it.  rwkv6_model.py:149-152 sets
            # w = -1e9 there (decay 1) and multiplies xk by the mask -- after k has already been
            # computed from xk (:148), so in the reference as committed k stays unmasked and a padded
            # token still writes k v^T into the state.  The evident intent is implemented here: k is
            # masked.  (A deliberate deviation; the operator itself is not involved.)
            m = mask.to(x.dtype)[..., None]
            k = k * m
            w = w * m + (1 - m) * -1e9
        u = self.time_faaaa.to(r.dtype)
        fused = getattr(self.rwkv_kernel, "forward_gn_gate", None)
        if fused is not None and r.is_cuda and r.dtype == torch.bfloat16:
            # group norm and gate come out of the operator's own output stage (inference: y is never
            # written; training: y and the norm's statistics are kept for one fused backward kernel)
            x, _ = fused(r.contiguous(), k.contiguous(), v.contiguous(), w.contiguous(), u, g.contiguous(),
                         self.group_norm.scale, self.group_norm.offset, self.group_norm.epsilon)
            return self.dense_o(x)
        y, _ = self.rwkv_kernel(r.contiguous(), k.contiguous(), v.contiguous(), w.contiguous(), u)
        return self.dense_o(self.group_norm(y) * g)


class ChannelMix(nn.Module):
    def __init__(self, hidden_size, expand_size, rwkv_kernel=None):
        super().__init__()
        self.rwkv_kernel = rwkv_kernel   # optional: its shift_mix_x kernel does the two token-shift mixes in bf16
        self.time_mix_k = nn.Parameter(torch.rand(hidden_size))
        self.time_mix_r = nn.Parameter(torch.rand(hidden_size))
        self.dense_key = nn.Linear(hidden_size, expand_size, bias=False)
        self.dense_value = nn.Linear(expand_size, hidden_size, bias=False)
        self.dense_receptance = nn.Linear(hidden_size, hidden_size, bias=False)

    def rounds_its_input(self):
        return hasattr(self.rwkv_kernel, "shift_mix_x") and self.time_mix_k.numel() % 64 == 0

    def forward(self, x):
        fused = getattr(self.rwkv_kernel, "shift_mix_x", None)
        if fused is not None and x.is_cuda and torch.is_autocast_enabled('cuda') and torch.get_autocast_dtype('cuda') == torch.bfloat16 \
                and x.shape[-1] % 64 == 0:
            xb = x.to(torch.bfloat16).contiguous()
            xk, xr = fused(xb, self.time_mix_k), fused(xb, self.time_mix_r)
        else:
            xx = time_shift(x)
            xk = x + xx * self.time_mix_k.to(x.dtype)
            xr = x + xx * self.time_mix_r.to(x.dtype)
        k = torch.square(torch.relu(self.dense_key(xk)))
        return torch.sigmoid(self.dense_receptance(xr)) * self.dense_value(k)


class Block(nn.Module):
    def __init__(self, rwkv_kernel, hidden_size, decomposer_size, head_size, expand_size):
        super().__init__()
        self.layer_norm_att = nn.LayerNorm(hidden_size, eps=1e-5)
        self.layer_norm_ffn = nn.LayerNorm(hidden_size, eps=1e-5)
        self.time_mix = TimeMix(rwkv_kernel, hidden_size, decomposer_size, head_size)
        self.channel_mix = ChannelMix(hidden_size, expand_size, rwkv_kernel)

    def stages(self, x, branch, mask=None):
        """From the stream and the branch that the layer before leaves (or None) to those of this one: each addition goes with the norm that follows it."""
        x, h = add_norm(x, branch, self.layer_norm_att, _rounds(x, self.time_mix))
        x, h = add_norm(x, self.time_mix(h, mask), self.layer_norm_ffn, _rounds(x, self.channel_mix))
        return x, self.channel_mix(h)

    def forward(self, x, mask=None):
        x, branch = self.stages(x, None, mask)
        return x + branch


class RWKV6(nn.Module):
    """ids (B, T) -> logits (B, T, vocabulary).  Ids outside of the table, negative ones among them, are an error on the CPU.  On the GPU, where the host does not see them, their
    rows are NaN, and with them the logits of their texts and a loss over these."""

    def __init__(self, rwkv_kernel, num_layers, vocabulary_size, hidden_size, decomposer_size, head_size, expand_size):
        super().__init__()
        self.embedding = nn.Embedding(vocabulary_size, hidden_size)
        self.embedding_ln = nn.LayerNorm(hidden_size, eps=1e-5)
        self.blocks = nn.ModuleList(Block(rwkv_kernel, hidden_size, decomposer_size, head_size, expand_size)
                                    for _ in range(num_layers))
        self.output_ln = nn.LayerNorm(hidden_size, eps=1e-5)
        self.output_layer = nn.Linear(hidden_size, vocabulary_size, bias=False)
        for m in self.modules():
            if isinstance(m, nn.Linear):
                nn.init.normal_(m.weight, std=0.5 / math.sqrt(m.in_features))
        nn.init.normal_(self.embedding.weight, std=0.02)

    def forward(self, ids, mask=None):
        table = self.embedding
        plain = _as_built(table, nn.Embedding) and table.padding_idx is None and table.max_norm is None and not table.sparse and not table.scale_grad_by_freq
        kernels = _kernels(table.weight) if plain and not (ids.is_floating_point() or ids.is_complex()) else None
        # (the kernel gives a negative id a row of zeros, which would pass for a token's: it goes behind the table)
        x = table(ids) if kernels is None else kernels.embedding(torch.where(ids < 0, table.num_embeddings, ids.long()), table.weight)
        x, branch = add_norm(x, None, self.embedding_ln)[1], None
        for blk in self.blocks:
            if _as_built(blk, Block):
                x, branch = blk.stages(x, branch, mask)
            else:
                x, branch = blk(x if branch is None else x + branch, mask), None
        return self.output_layer(add_norm(x, branch, self.output_ln, _rounds(x, self.output_layer))[1])


def _losses(logits):
    """The same where there is nothing to fall back on."""
    kernels = _kernels(logits)
    assert kernels is not None, "this step is for the package's torch flavour (KERAS_BACKEND=torch) and logits in 16 or 32 bits on the GPU"
    return kernels


def _logits(model, ids, autocast_dtype):
    """The model's logits for every token but the first of each text."""
    dev = ids.device.type
    with torch.autocast(dev, dtype=autocast_dtype, enabled=autocast_dtype is not None):
        return model(ids[:, :-1])


def _update(optimizer, loss):
    loss.backward()
    optimizer.step()
    return loss.detach()


def train_step(model, optimizer, ids, autocast_dtype=None):
    """One next-token cross-entropy step: forward, backward, optimizer update.  Returns the loss."""
    optimizer.zero_grad(set_to_none=True)
    logits, target = _logits(model, ids, autocast_dtype), ids[:, 1:]
    kernels = _kernels(logits)
    if kernels is not None:
        if logits.dim() != 3 or logits.shape[:-1] != target.shape:
            logits, target = logits.reshape(-1, logits.shape[-1]), target.reshape(-1)
        return _update(optimizer, kernels.cross_entropy(logits, target.long()))
    return _update(optimizer, F.cross_entropy(logits.float().reshape(-1, logits.shape[-1]), target.reshape(-1)))


class Optimizers(torch.optim.Optimizer):
    """Several optimizers, of a model's parameters each a part, as one: groups and state are theirs, one behind the other, and so they are saved and loaded.  A group is added
    to one of them."""

    def __init__(self, *optimizers):
        self.optimizers = optimizers
        params = [p for group in self.param_groups for p in group["params"]]
        assert len({id(p) for p in params}) == len(params), "a parameter belongs to one of the optimizers"
        super().__init__(self.param_groups, {})

    # (the base class sets both once and adds the groups that are there already)
    @property
    def param_groups(self):
        return [group for optimizer in self.optimizers for group in optimizer.param_groups]

    @param_groups.setter
    def param_groups(self, groups):
        pass

    @property
    def state(self):
        return {p: state for optimizer in self.optimizers for p, state in optimizer.state.items()}

    @state.setter
    def state(self, state):
        pass

    def add_param_group(self, param_group):
        assert any(param_group is group for group in self.param_groups), "a group is added to one of the optimizers"

    def __getstate__(self):
        return dict(optimizers=self.optimizers, defaults=self.defaults)

    def zero_grad(self, set_to_none=True):
        for optimizer in self.optimizers:
            optimizer.zero_grad(set_to_none=set_to_none)

    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for optimizer in self.optimizers:
            optimizer.step()
        return loss

    def state_dict(self):
        state, groups, first = {}, [], 0
        for optimizer in self.optimizers:
            d = optimizer.state_dict()
            state.update({first + i: s for i, s in d["state"].items()})
            groups += [dict(group, params=[first + i for i in group["params"]]) for group in d["param_groups"]]
            first += sum(len(group["params"]) for group in d["param_groups"])
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, state_dict):
        groups = list(state_dict["param_groups"])
        assert [len(group["params"]) for group in groups] == [len(group["params"]) for group in self.param_groups], "saved from other groups of parameters"
        for optimizer in self.optimizers:
            mine, groups = groups[:len(optimizer.param_groups)], groups[len(optimizer.param_groups):]
            ids = {i for group in mine for i in group["params"]}
            optimizer.load_state_dict({"state": {i: s for i, s in state_dict["state"].items() if i in ids}, "param_groups": mine})


def muon_and_adamw(model, lr=0.02, weight_decay=0.0, adamw_lr=1e-4, adamw=None, **options):
    """The package's Muon for the weight matrices of the model's layers and its AdamW for the rest (embedding, norms, biases, mixes, output layer), as one
    optimizer for the steps here.  options as of rwkv_kernel.Muon, adamw: a dict of what AdamW takes beside them (moment_bits, betas, max_grad_norm: of AdamW's
    gradients alone, which Muon's steps do not depend on the size of).  skip_nonfinite is refused: Muon takes every step, and the model's would be half a step."""
    from rwkv_kernel import AdamW, Muon

    adamw = dict(dict(lr=adamw_lr, weight_decay=weight_decay), **(adamw or {}))
    assert not adamw.get("skip_nonfinite"), "Muon leaves no step out: skip_nonfinite would leave out AdamW's half of one"
    matrices = [m.weight for m in model.blocks.modules() if isinstance(m, nn.Linear)]
    others = {id(p) for p in matrices}
    others = [p for p in model.parameters() if id(p) not in others]
    return Optimizers(Muon(matrices, lr=lr, weight_decay=weight_decay, **options), AdamW(others, **adamw))


# Fine-tuning steps on the operator package's losses (its torch flavour, on the GPU).  Texts are ids (B, T+1); mask (B, T) says which of
# their tokens from the second on count (a prompt's and the padding's do not).

@torch.no_grad()
def token_logprobs(model, ids, mask, autocast_dtype=None, temperature=1.0):
    """Log probabilities (B, T) of the texts' tokens: what a reference or a sampling model makes of them."""
    logits = _logits(model, ids, autocast_dtype)
    return _losses(logits).token_logprobs(logits, ids[:, 1:], mask, temperature=temperature)


def preference_step(model, optimizer, ids, mask, ref_logps, autocast_dtype=None, **options):
    """One step on pairs of texts, the chosen ones and then as many rejected ones.  ref_logps (B): sums of the reference model's token_logprobs; options
    as of rwkv_kernel.preference_loss.  Returns the loss."""
    optimizer.zero_grad(set_to_none=True)
    logits = _logits(model, ids, autocast_dtype)
    return _update(optimizer, _losses(logits).preference_loss(logits, ids[:, 1:], mask, ref_logps=ref_logps, **options)[0])


def policy_step(model, optimizer, ids, mask, old_logps, advantages, autocast_dtype=None, **options):
    """One step on sampled texts: old_logps (B, T) are the sampling model's token_logprobs, advantages (B,) or (B, T); options as of
    rwkv_kernel.policy_loss.  Returns the loss."""
    optimizer.zero_grad(set_to_none=True)
    logits = _logits(model, ids, autocast_dtype)
    return _update(optimizer, _losses(logits).policy_loss(logits, ids[:, 1:], mask, old_logps, advantages, **options)[0])


# the layer shape of configuration 4: RWKV6-1.6B (24 layers, d_model 2048, 32 heads of 64, FFN 7168)
CONFIG4 = dict(num_layers=24, vocabulary_size=65536, hidden_size=2048, decomposer_size=32, head_size=64, expand_size=7168)
