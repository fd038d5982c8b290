"""What a training step does behind the model's last layer, as cases that can be timed and compared.

    cross_entropy    the next-token loss of a training step and its gradient by the logits
    token_logprobs   log probabilities of the tokens that stand there: a reference model's pass (forward alone), or with a gradient
    preference_loss  paired log ratios of chosen and rejected texts against a reference model, and the gradient by the logits
    policy_loss      clipped probability ratios with a KL term against a reference model, and the gradient by the logits
    adamw_step       the optimizer's step over all parameters, moments in 32 bits or in 8, gradients clipped by their common norm

Every case is one call (and its backward pass) of ``rwkv_kernel``'s functions of these names.  Sizes: the vocabulary of 65536 and the
layers (width 2048, feed-forward 7168, mixers of rank 32) are this repository's benchmark model, and what lies around them.

The module is imported with the repository's root as the working folder.
"""
import math
import os
import sys

import torch

own = False                 # the framework's kernels, or the same operators in elementary operations

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
LOSSES = ("cross_entropy", "token_logprobs", "preference_loss", "policy_loss")
LOSS_SCALE = {"bf16": 1.0, "f16": 4096.0, "f32": 1.0}   # what a training in half precision multiplies its loss by
BETA = 0.1                  # of the preference loss
CLIP, KL = 0.2, 0.04        # of the policy loss
LR, BETAS, EPS, DECAY = 1e-3, (0.9, 0.99), 1e-8, 0.01
BLOCK = 256                 # elements that share a scale where moments are held in 8 bits
U32 = 0xFFFFFFFF


def _loss(op, B, T, V, dtype="bf16", fill=1.0, grad=True, temperature=1.0):
    """`fill`: the shortest text's share of T; lengths are spread evenly from there to T."""
    return {"op": op, "B": B, "T": T, "V": V, "dtype": dtype, "fill": fill, "grad": grad, "temperature": temperature}


def _adamw(layers, C, E, V, dtype="f32", bits=32, master=False, clip=0.0):
    """Parameters of `layers` layers of width C with feed-forward E, and embedding and head of V tokens (0: none)."""
    return {"op": "adamw_step", "layers": layers, "C": C, "E": E, "V": V, "dtype": dtype, "bits": bits, "master": master, "clip": clip}


def listed():
    named = {
        # the training step of the benchmark's model: batch 8, 1024 tokens
        "cross_entropy_model": _loss("cross_entropy", 8, 1024, 65536),
        # a small model in full precision, texts of different lengths
        "cross_entropy_small": _loss("cross_entropy", 4, 200, 8000, dtype="f32", fill=0.3),
        # scoring the last tokens of one text: few rows, latency alone
        "logprobs_few": _loss("token_logprobs", 1, 17, 65536, grad=False),
        # a reference model's pass over a batch of texts of different lengths
        "logprobs_reference": _loss("token_logprobs", 16, 512, 65536, fill=0.5, grad=False),
        # log probabilities with a gradient, half precision, a vocabulary that nothing divides
        "logprobs_odd": _loss("token_logprobs", 4, 333, 50277, dtype="f16", fill=0.7, temperature=0.8),
        # one pair of texts
        "preference_pair": _loss("preference_loss", 2, 777, 65536, fill=0.6),
        # a batch of eight pairs: the largest logits
        "preference_batch": _loss("preference_loss", 16, 1024, 65536, fill=0.5),
        # a small model's step on sampled texts, full precision
        "policy_small": _loss("policy_loss", 4, 64, 32000, dtype="f32", fill=0.2),
        # a batch of sampled texts of the benchmark's model
        "policy_batch": _loss("policy_loss", 8, 1024, 65536, fill=0.4),
        # one small layer: latency, many tensors of a few hundred elements
        "adamw_small": _adamw(1, 256, 896, 0),
        # layers, embedding and head of the benchmark's model in full precision, gradients clipped: the largest case
        "adamw_model": _adamw(4, 2048, 7168, 65536, clip=1.0),
        # the same in bf16 with moments in 8 bits, as where memory is short
        "adamw_model_8bit": _adamw(4, 2048, 7168, 65536, dtype="bf16", bits=8, clip=1.0),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cross_entropy", "token_logprobs", "preference_loss", "policy_loss", "adamw_step", "adamw_step"])
    if op == "adamw_step":
        dtype = rng.choice(["f32", "bf16", "f16"])
        C = _log_int(rng, 100, 2000)
        return _adamw(rng.randint(1, 4), C, 3 * C + rng.randint(0, C), rng.choice([0, _log_int(rng, 1000, 65536)]), dtype=dtype,
                      bits=rng.choice([32, 8]), master=dtype != "f32" and rng.random() < 0.5, clip=rng.choice([0.0, 1.0]))
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    V = rng.choice([65536, 50277, _log_int(rng, 1000, 160000)])
    rows = _log_int(rng, 2, min(20000, 2 ** 29 // V))
    B = min(rows, 2 * rng.randint(1, 8))
    B += B % 2
    return _loss(op, B, max(1, rows // B), V, dtype=dtype, fill=rng.choice([1.0, 0.6, 0.25]),
                 grad=op != "token_logprobs" or rng.random() < 0.5, temperature=rng.choice([1.0, 0.7]) if op in ("token_logprobs", "policy_loss") else 1.0)


def _lengths(case):
    """Counted tokens of each text, longest first."""
    B, T = case["B"], case["T"]
    return [max(1, round(T * (1.0 - (1.0 - case["fill"]) * b / max(1, B - 1)))) for b in range(B)]


def _shapes(case):
    """The parameters of the benchmark's model (24 tensors and more to a layer), at this case's sizes."""
    C, E, V, R, W = case["C"], case["E"], case["V"], 32, 64
    mixers = [(R, C), (C, R), (C,)] * 5
    layer = mixers + [(W, C), (C, W), (C,)] + [(C, C)] * 5 + [(C,)] * 8 + [(E, C), (C, E), (C, C)] + [(C,)] * 2
    return ([(V, C), (C,), (C,)] if V else []) + layer * case["layers"] + ([(C,), (C,), (V, C)] if V else [])


def _views(flat, shapes, unit):
    """A tensor of each shape in one buffer, each on a multiple of `unit` elements."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at:at + n].view(s))
        at += (n + unit - 1) // unit * unit
    return out


def _room(shapes, unit):
    return sum((math.prod(s) + unit - 1) // unit * unit for s in shapes)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = {"case": case}

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    if case["op"] == "adamw_step":
        # weights, gradients and moments as in the middle of a training: every tensor has gradients of a size of its own
        shapes = _shapes(case)
        n = _room(shapes, BLOCK)
        size = torch.exp(normal(n // BLOCK)) * 1e-2
        spread = lambda x: (x.view(-1, BLOCK) * size[:, None]).view(-1)  # noqa: E731
        # (the moments first, the largest temporaries with them)
        m, r = spread(normal(n, std=0.3)), spread(normal(n).abs() * 0.5 + 0.5)
        if case["bits"] == 8:
            # what a step before this one left: float8 values under one scale for each 256 elements
            scales = []
            for name, x in (("m", m), ("v", r)):
                s = x.view(-1, BLOCK).abs().amax(1) / 448.0
                state[name] = (x.view(-1, BLOCK) / s[:, None]).to(torch.float8_e4m3fn).view(-1)
                scales.append(s)
            state["scales"] = torch.stack(scales, 1).contiguous()
            state["scale_list"] = list(state["scales"].split([(math.prod(s) + BLOCK - 1) // BLOCK for s in shapes]))
        else:
            state["m"], state["v"] = m, r * r
        p = normal(n, std=0.05)
        if case["master"]:
            state["master"] = p
            state["master_list"] = _views(p, shapes, BLOCK)
        state["p"], state["g"] = p.to(dt), spread(normal(n)).to(dt)
        # (what lies between two tensors belongs to none of them)
        for name in ("p", "g", "m", "v"):
            state[name + "_list"] = _views(state[name], shapes, BLOCK)
        state["step"] = torch.full((), 1000, dtype=torch.int64, device=dev)
        state["seed"] = seed & U32
        return state
    B, T, V = case["B"], case["T"], case["V"]
    order = torch.randperm(B, generator=g, device=dev)
    lengths = torch.tensor(_lengths(case), device=dev)[order]
    state["mask"] = torch.arange(T, device=dev)[None, :] < lengths[:, None]
    state["ids"] = torch.randint(0, V, (B, T), generator=g, device=dev)
    # logits of a trained model: the token that stands there is among the likely ones
    x = normal(B, T, V, std=2.0)
    x.scatter_add_(2, state["ids"][..., None], normal(B, T, 1) + 9.0)
    state["logits"] = x.to(dt)
    del x
    if case["op"] in ("preference_loss", "policy_loss"):
        lp = state["logits"].float().mul_(1.0 / case["temperature"])
        lp = (lp.gather(2, state["ids"][..., None])[..., 0] - lp.logsumexp(2))
    if case["op"] == "preference_loss":
        # the reference model's log probability of each text
        state["ref"] = (lp * state["mask"]).sum(1) + normal(B, std=5.0)
    if case["op"] == "policy_loss":
        # the sampling model was this one a few steps ago.  (No ratio within 1e-3 of where the clipping begins: there the gradient jumps.)
        d = normal(B, T, std=0.12)
        d = torch.where(((d.exp() - 1.0).abs() - CLIP).abs() < 1e-3, torch.zeros_like(d), d)
        state["old"], state["ref"] = lp - d, lp + normal(B, T, std=0.2)
        state["advantages"] = normal(B)
    if case["op"] == "token_logprobs" and case["grad"]:
        state["gout"] = normal(B, T) * state["mask"]
    state["scale"] = torch.full((), LOSS_SCALE[case["dtype"]], device=dev)
    state["logits"].requires_grad_(case["grad"])
    return state


# ---- the framework's kernels ----

def _run_own(s):
    path = os.path.join(os.getcwd(), "star-rwkv6_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    os.environ.setdefault("KERAS_BACKEND", "torch")
    import rwkv_kernel

    c = s["case"]
    if c["op"] == "adamw_step":
        norm = rwkv_kernel.adamw_step(
            s["p_list"], s["g_list"], s["m_list"], s["v_list"], s["step"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY,
            scales=s.get("scale_list"), masters=s.get("master_list"), max_grad_norm=c["clip"] or None, seed=s["seed"])
        return _updated(s, norm)
    x, ids, mask = s["logits"], s["ids"], s["mask"]
    if c["op"] == "token_logprobs":
        lp = rwkv_kernel.token_logprobs(x, ids, mask, temperature=c["temperature"])
        return [lp, *torch.autograd.grad(lp, x, s["gout"])] if c["grad"] else [lp]
    if c["op"] == "cross_entropy":
        out = [rwkv_kernel.cross_entropy(x, ids, mask)]
    elif c["op"] == "preference_loss":
        out = list(rwkv_kernel.preference_loss(x, ids, mask, ref_logps=s["ref"], beta=BETA))
    else:
        out = list(rwkv_kernel.policy_loss(x, ids, mask, s["old"], s["advantages"], ref_logps=s["ref"], clip_low=CLIP, clip_high=CLIP,
                                           kl_weight=KL, temperature=c["temperature"]))
    return [*out, *torch.autograd.grad(out[0], x, s["scale"])]


def _updated(s, norm):
    return {"p": s["p"], "m": s["m"], "v": s["v"], "scales": s.get("scales"), "master": s.get("master"), "norm": norm}


# ---- the plain forms ----

def _softmax(s):
    """exp(x - lse), and log probabilities of the tokens that stand there, zero where none counts; rows that do not count are not looked at."""
    x = s["logits"].detach().float() * (1.0 / s["case"]["temperature"])
    x = torch.where(s["mask"][..., None], x, torch.zeros_like(x))
    top = x.amax(2, keepdim=True)
    x = x - top
    lp = x.gather(2, s["ids"][..., None])[..., 0].double()
    x = torch.exp(x)
    total = x.sum(2, keepdim=True)
    lp = torch.where(s["mask"], lp - torch.log(total.double())[..., 0], torch.zeros_like(lp))
    return x / total, lp


def _by_logits(s, p, coef):
    """The gradient by the logits: coef * (1 at the token that stands there - p)."""
    coef = coef.float() * s["mask"] * (1.0 / s["case"]["temperature"])
    p = p * -coef[..., None]
    p.scatter_add_(2, s["ids"][..., None], coef[..., None])
    return p.to(s["logits"].dtype)


def _run_loss(s):
    c, mask = s["case"], s["mask"]
    p, lp = _softmax(s)
    if c["op"] == "token_logprobs":
        return [lp.float(), _by_logits(s, p, s["gout"])] if c["grad"] else [lp.float()]
    count = mask.sum().double()
    if c["op"] == "cross_entropy":
        return [(-lp.sum() / count).float(), _by_logits(s, p, -s["scale"] / count * mask)]
    if c["op"] == "preference_loss":
        P = c["B"] // 2
        text = lp.sum(1)
        d = BETA * ((text[:P] - text[P:]) - (s["ref"][:P].double() - s["ref"][P:].double()))
        loss = (torch.log1p(torch.exp(-d.abs())) + torch.clamp(-d, min=0.0)).sum() / P
        by_text = s["scale"] * -BETA / (1.0 + torch.exp(d)) / P
        return [loss.float(), text.float(), _by_logits(s, p, torch.cat([by_text, -by_text])[:, None] * mask)]
    A = s["advantages"].double()[:, None]
    ratio = torch.exp(lp - s["old"].double())
    free, held = ratio * A, torch.clamp(ratio, 1.0 - CLIP, 1.0 + CLIP) * A
    e = s["ref"].double() - lp
    kl = torch.exp(e) - e - 1.0
    loss = ((KL * kl - torch.minimum(free, held)) * mask).sum() / count
    coef = (KL * (1.0 - torch.exp(e)) - torch.where(free <= held, free, torch.zeros_like(free))) / count
    stats = torch.stack([(kl * mask).sum(), ((free > held) & mask).sum().double()]) / count
    return [loss.float(), lp.float(), stats.float(), _by_logits(s, p, s["scale"] * coef * mask)]


def _mix(x):
    x = (x ^ (x >> 16)) * 0xBB67AE85 & U32
    x = (x ^ (x >> 15)) * 0x9E3779B9 & U32
    return x ^ (x >> 16)


def _to_float8(x, random, positive):
    """The float8 (4 exponent bits, 3 mantissa bits) below or above x, above with the probability that keeps the mean; at most 448.
    In fp32's own bits: 2^-120 brings the exponents together, below the smallest normal number too."""
    bits = (x.abs() * 2.0 ** -120).view(torch.int32).long()
    code = torch.clamp((bits + (random << 4)) >> 20, max=0x7E)
    if positive:   # a denominator is never rounded to zero
        code = torch.where((code == 0) & (x > 0), torch.ones_like(code), code)
    return (code | ((x < 0).long() << 7)).to(torch.uint8).view(torch.float8_e4m3fn)


def _rows(x):
    return torch.cat([x, x.new_zeros(-x.numel() % BLOCK)]).view(-1, BLOCK)


def _adamw_one(s, j, scale, c1, c2):
    """One tensor's step, in place."""
    c, (b1, b2) = s["case"], BETAS
    p, g = s["master_list" if c["master"] else "p_list"][j], s["g_list"][j].float() * scale
    m, v = s["m_list"][j], s["v_list"][j]
    if c["bits"] == 8:
        sc = s["scale_list"][j]
        m0 = (_rows(m.view(-1).float()) * sc[:, :1]).view(-1)[:m.numel()].view(m.shape)
        r0 = (_rows(v.view(-1).float()) * sc[:, 1:]).view(-1)[:v.numel()].view(v.shape)
        v0 = r0 * r0
    else:
        m0, v0 = m, v
    m1, v1 = m0 * b1 + g * (1.0 - b1), v0 * b2 + g * g * (1.0 - b2)
    r1 = torch.sqrt(v1)
    new = p.float() * (1.0 - LR * DECAY) - (m1 * (LR / c1)) / (r1 * (1.0 / torch.sqrt(c2)) + EPS)
    p.copy_(new)
    if c["master"]:
        s["p_list"][j].copy_(new)
    if c["bits"] == 8:
        key = _mix((s["seed"] * 0x9E3779B9 + s["step"] * 0xBB67AE85 + j) & U32)
        h = _rows(_mix((torch.arange(m.numel(), device=m.device) * 0x9E3779B9 + key) & U32))
        m1, r1 = _rows(m1.reshape(-1)), _rows(r1.reshape(-1))
        top = torch.stack([m1.abs().amax(1), r1.amax(1)], 1).clamp(min=2.0 ** -100)
        sc.copy_(top * (1.0 / 448.0))
        m.view(-1).copy_(_to_float8(m1 * (448.0 / top[:, :1]), h & 0xFFFF, False).view(-1)[:m.numel()])
        v.view(-1).copy_(_to_float8(r1 * (448.0 / top[:, 1:]), h >> 16, True).view(-1)[:v.numel()])
    else:
        m.copy_(m1)
        v.copy_(v1)


def _run_adamw(s):
    c = s["case"]
    s["step"] += 1
    t = s["step"].double()
    c1, c2 = ((1.0 - torch.pow(b, t)) for b in BETAS)
    norm, scale = None, 1.0
    if c["clip"]:
        norm = torch.sqrt(torch.stack([g.double().square().sum() for g in s["g_list"]]).sum()).float()
        scale = (c["clip"] / torch.clamp(norm.double(), min=c["clip"])).float()
    [_adamw_one(s, j, scale, c1.float(), c2.float()) for j in range(len(s["p_list"]))]
    return _updated(s, norm)


def run(state):
    if own:
        return _run_own(state)
    return _run_adamw(state) if state["case"]["op"] == "adamw_step" else _run_loss(state)


# ---- what a pass cannot do without ----

def work(case):
    if case["op"] == "adamw_step":
        n, es = sum(math.prod(s) for s in _shapes(case)), DTYPES[case["dtype"]].itemsize
        moments = 4.0 if case["bits"] == 8 else 16.0   # two of them, read and written
        # weights and gradients read, weights written, and the weights in fp32 behind them read and written
        return {"bytes": n * ((2 * es if case["master"] else 3 * es) + moments + (8 if case["master"] else 0)), "flops": 16.0 * n}
    rows, V, es = sum(_lengths(case)), case["V"], DTYPES[case["dtype"]].itemsize
    # the logits of the rows that count, read once, and the gradient of all rows, written once
    read, written = rows * V * es, case["B"] * case["T"] * V * es if case["grad"] else 0
    return {"bytes": float(read + written + case["B"] * case["T"] * 16), "flops": (4.0 + (4.0 if case["grad"] else 0.0)) * rows * V}


# ---- 64 bits ----

def _exact_loss(s):
    c, mask, ids = s["case"], s["mask"], s["ids"]
    x = s["logits"].detach().double().requires_grad_(c["grad"])
    logits = x.masked_fill(~mask[..., None], 0.0) / c["temperature"]
    lp = -torch.nn.functional.cross_entropy(logits.view(-1, c["V"]), ids.view(-1), reduction="none").view(mask.shape)
    lp = lp.masked_fill(~mask, 0.0)
    if c["op"] == "token_logprobs":
        return [lp.detach(), *torch.autograd.grad(lp, x, s["gout"].double())] if c["grad"] else [lp]
    if c["op"] == "cross_entropy":
        out = [-lp[mask].mean()]
    elif c["op"] == "preference_loss":
        chosen, rejected = lp.sum(1).chunk(2)
        ref_chosen, ref_rejected = s["ref"].double().chunk(2)
        out = [-torch.nn.functional.logsigmoid(BETA * (chosen - ref_chosen - rejected + ref_rejected)).mean(), lp.sum(1)]
    else:
        ratio, A = (lp - s["old"].double()).exp()[mask], s["advantages"].double()[:, None].expand(mask.shape)[mask]
        gap = (s["ref"].double() - lp)[mask]
        kl = torch.expm1(gap) - gap
        beyond = torch.where(A > 0, ratio > 1 + CLIP, ratio < 1 - CLIP)
        term = torch.where(beyond, torch.where(A > 0, 1.0 + CLIP, 1.0 - CLIP) * A, ratio * A)
        out = [(KL * kl - term).mean(), lp, torch.stack([kl.mean(), beyond.double().mean()])]
    grad = torch.autograd.grad(out[0], x, s["scale"].double())
    return [o.detach() for o in out] + [grad[0]]


def _exact_adamw(s):
    c, (b1, b2) = s["case"], BETAS
    used = torch.zeros(s["p"].numel(), dtype=torch.bool, device=s["p"].device)
    for view in _views(used, [g.shape for g in s["g_list"]], BLOCK):
        view.fill_(True)
    g, p = s["g"].double(), s["master" if c["master"] else "p"].double()
    norm = (g * used).norm() if c["clip"] else None
    if c["clip"] and float(norm) > c["clip"]:
        g = g * (c["clip"] / norm)
    m, v = s["m"].double(), s["v"].double()
    if c["bits"] == 8:
        wide = s["scales"].double().repeat_interleave(BLOCK, 0)
        m, v = m * wide[:, 0], (v * wide[:, 1]).square()
    t = 1001
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g.square()
    new = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    new = torch.where(used, new, p)
    out = {"p": new, "m": None, "v": None, "scales": None, "master": new if c["master"] else None, "norm": norm}
    if c["master"]:
        out["p"] = torch.where(used, new, s["p"].double())
    if c["bits"] == 8:
        # which of its two neighbours a moment is rounded to is drawn: the scales are what there is in 64 bits
        top = torch.stack([(m * used).view(-1, BLOCK).abs().amax(1), (v.sqrt() * used).view(-1, BLOCK).amax(1)], 1)
        out["scales"] = top.clamp(min=2.0 ** -100) / 448.0
    else:
        out["m"], out["v"] = torch.where(used, m, s["m"].double()), torch.where(used, v, s["v"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(s) if case["op"] == "adamw_step" else _exact_loss(s)
