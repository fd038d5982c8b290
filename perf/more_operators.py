"""What a training step does before, between and after the layers' own operators, as cases that can be timed and compared.

    embedding      rows of a table by token, and the table's gradient
    layer_norm     the norm over a token's channels, with the residual addition before it or without, and its gradients
    orthogonalize  matrices brought near to the nearest matrix with orthonormal rows or columns, by Newton-Schulz products
    muon_step      the optimizer's step on weight matrices: momentum, orthogonalized updates, weight decay

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
LN_EPS = 1e-5
STEPS, COEFFICIENTS, NS_EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def _embedding(B, T, V, C, dtype="f32", out="same", grad=True, fill=1.0, scale=1.0):
    """`dtype`: the table's.  `fill`: the shortest text's share of T, padding behind it."""
    return {"op": "embedding", "B": B, "T": T, "V": V, "C": C, "dtype": dtype, "out": dtype if out == "same" else out, "grad": grad, "fill": fill,
            "scale": scale}


def _norm(rows, C, dtype="f32", branch="same", add=True, affine=True, grad=True):
    """`dtype`: the residual stream's; `branch`: what is added to it and what comes out for the next layer."""
    return {"op": "layer_norm", "rows": rows, "C": C, "dtype": dtype, "branch": dtype if branch == "same" else branch, "add": add, "affine": affine,
            "grad": grad}


def _matrices(op, shapes, dtype="f32", master=False, nesterov=True):
    """`shapes`: "count x rows x columns", several with spaces between them."""
    return {"op": op, "shapes": shapes, "dtype": dtype, "master": master, "nesterov": nesterov}


def _layers(n):
    """The matrices of n layers of the benchmark's model."""
    return "%dx32x2048 %dx2048x32 %dx64x2048 %dx2048x64 %dx2048x2048 %dx7168x2048 %dx2048x7168" % (5 * n, 5 * n, n, n, 6 * n, n, n)


def listed():
    named = {
        # one token of one text is generated: latency alone
        "embedding_token": _embedding(1, 1, 65536, 2048, dtype="bf16", grad=False),
        # the training step of the benchmark's model: batch 8, 1024 tokens, the table in full precision
        "embedding_model": _embedding(8, 1024, 65536, 2048),
        # half precision, texts of different lengths, sizes that nothing divides, scaled rows
        "embedding_odd": _embedding(5, 333, 50277, 777, dtype="f16", fill=0.4, scale=math.sqrt(777.0)),
        # the token before the next layer: latency alone, no gradient
        "norm_token": _norm(1, 2048, dtype="f32", branch="bf16", grad=False),
        # between two stages of a layer of the benchmark's model, a stream in full precision with branches in bf16
        "norm_model": _norm(8192, 2048, dtype="f32", branch="bf16"),
        # a stream in half precision, a width that nothing divides, no addition
        "norm_odd": _norm(1665, 777, dtype="f16", add=False),
        # longer and wider, everything in bf16
        "norm_wide": _norm(32768, 4096, dtype="bf16"),
        # the low-rank mixers of one layer: small matrices, latency
        "orthogonalize_mixers": _matrices("orthogonalize", "5x32x2048 5x2048x32", dtype="bf16"),
        # one matrix that nothing divides
        "orthogonalize_odd": _matrices("orthogonalize", "1x777x1311"),
        # one projection
        "orthogonalize_square": _matrices("orthogonalize", "1x2048x2048", dtype="bf16"),
        # the matrices of a small model
        "muon_small": _matrices("muon_step", "24x256x256 4x896x256 4x256x896"),
        # the matrices of two layers of the benchmark's model, weights in bf16 with masters: the largest case
        "muon_model": _matrices("muon_step", _layers(2), dtype="bf16", master=True),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["embedding", "layer_norm", "orthogonalize", "muon_step"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    narrow = rng.choice(["same", "bf16", "f16"]) if dtype == "f32" else "same"
    if op == "embedding":
        V, C = rng.choice([65536, _log_int(rng, 100, 160000)]), _log_int(rng, 32, 4096)
        N = _log_int(rng, 1, min(20000, 2 ** 26 // C))
        B = min(N, rng.randint(1, 16))
        while V * C > 2 ** 28:
            V //= 2
        return _embedding(B, N // B, V, C, dtype=dtype, out=narrow, grad=rng.random() < 0.7, fill=rng.choice([1.0, 0.5]), scale=rng.choice([1.0, math.sqrt(C)]))
    if op == "layer_norm":
        C = _log_int(rng, 32, 8192)
        return _norm(_log_int(rng, 1, min(65536, 2 ** 27 // C)), C, dtype=dtype, branch=narrow, add=rng.random() < 0.6, affine=rng.random() < 0.8,
                     grad=rng.random() < 0.7)
    shapes = []
    for _ in range(rng.randint(1, 3)):
        m, n = _log_int(rng, 16, 2500), _log_int(rng, 16, 2500)
        shapes.append("%dx%dx%d" % (rng.randint(1, max(1, min(8, 2 ** 23 // (m * n)))), m, n))
    return _matrices(op, " ".join(shapes), dtype=dtype, master=op == "muon_step" and dtype != "f32" and rng.random() < 0.5, nesterov=rng.random() < 0.7)


def _lengths(case):
    B, T = case["B"], case["T"]
    return [max(1, round(T * (1.0 - (1.0 - case["fill"]) * b / max(1, B - 1)))) for b in range(B)]


def _shapes(case):
    out = []
    for part in case["shapes"].split():
        count, rows, columns = (int(x) for x in part.split("x"))
        out += [(rows, columns)] * count
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    state = {"case": case}

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=dev) * std

    if case["op"] == "embedding":
        B, T, V, C = case["B"], case["T"], case["V"], case["C"]
        # tokens as in a text: some common ones, many rare ones, the k-th most common with a probability like 1 / k
        rank = torch.exp(torch.rand(B, T, generator=g, device=dev, dtype=torch.float64) * math.log(V)).long().clamp(1, V) - 1
        ids = torch.randperm(V, generator=g, device=dev)[rank]
        lengths = torch.tensor(_lengths(case), device=dev)[torch.randperm(B, generator=g, device=dev)]
        state["ids"] = torch.where(torch.arange(T, device=dev)[None, :] < lengths[:, None], ids, torch.full_like(ids, -1))
        state["weight"] = normal(V, C, std=0.02).to(dt).requires_grad_(case["grad"])
        if case["grad"]:
            state["gout"] = normal(B, T, C, std=1e-2).to(DTYPES[case["out"]])
        return state
    if case["op"] == "layer_norm":
        rows, C, branch = case["rows"], case["C"], DTYPES[case["branch"]]
        # the stream of a trained model: a mean, a few channels larger than the others
        size = torch.exp(normal(C, std=0.5))
        state["x"] = (normal(rows, C) * size + 0.3).to(dt).requires_grad_(case["grad"])
        if case["add"]:
            state["add"] = normal(rows, C, std=0.5).to(branch).requires_grad_(case["grad"])
        if case["affine"]:
            state["weight"] = (1.0 + normal(C, std=0.2)).requires_grad_(case["grad"])
            state["bias"] = normal(C, std=0.2).requires_grad_(case["grad"])
        if case["grad"]:
            state["gy"] = normal(rows, C, std=1e-2).to(branch)
            if case["add"]:
                state["gtotal"] = normal(rows, C, std=1e-2).to(dt)
        return state

    def update(m, n):
        # a gradient: a few strong directions, and what is left of many weak ones
        r = min(m, n, 16)
        strong = (normal(m, r) * torch.exp(-torch.arange(r, device=dev) / 4.0)) @ normal(r, n)
        return (strong + normal(m, n, std=0.3)) * 1e-3

    shapes = _shapes(case)
    state["grads"] = [update(m, n).to(dt) for m, n in shapes]
    if case["op"] == "muon_step":
        # weights and momenta in buffers of their own, one matrix right behind the other
        flat = {"momenta": torch.cat([update(m, n).view(-1) * 0.3 for m, n in shapes]),
                "params": torch.cat([normal(m, n, std=0.5 / math.sqrt(n)).view(-1) for m, n in shapes])}
        flat["masters"] = flat["params"] if case["master"] else None
        flat["params"] = flat["params"].to(dt)
        state["flat"] = flat
        for name, x in flat.items():
            state[name] = x if x is None else [v.view(shape) for v, shape in zip(x.split([math.prod(shape) for shape in shapes]), shapes)]
    return state


# ---- the framework's kernels ----

def _run_own(s):
    path = os.path.join(os.getcwd(), "star-rwkv6_amd")
    if path not in sys.path:
        sys.path.insert(1, path)
    os.environ.setdefault("KERAS_BACKEND", "torch")
    import rwkv_kernel

    c = s["case"]
    if c["op"] == "embedding":
        out = rwkv_kernel.embedding(s["ids"], s["weight"], scale=c["scale"], dtype=DTYPES[c["out"]])
        return [out.detach(), *torch.autograd.grad(out, s["weight"], s["gout"])] if c["grad"] else [out]
    if c["op"] == "layer_norm":
        out = rwkv_kernel.layer_norm(s["x"], s.get("weight"), s.get("bias"), eps=LN_EPS, add=s.get("add"), dtype=DTYPES[c["branch"]])
        out = list(out) if c["add"] else [out]
        if not c["grad"]:
            return out
        leaves = [s[name] for name in ("x", "add", "weight", "bias") if name in s]
        arriving = [s[name] for name in ("gy", "gtotal") if name in s]
        return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, arriving))
    if c["op"] == "orthogonalize":
        return rwkv_kernel.orthogonalize(s["grads"], steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS)
    rwkv_kernel.muon_step(s["params"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, nesterov=c["nesterov"], weight_decay=DECAY, scale="shape",
                          steps=STEPS, coefficients=COEFFICIENTS, eps=NS_EPS, masters=s["masters"])
    return s["flat"]


# ---- the plain forms ----

def _run_embedding(s):
    c, ids, w = s["case"], s["ids"].view(-1), s["weight"].detach()
    held = ids >= 0
    rows = w[ids.clamp(min=0)].float() * c["scale"]
    out = [torch.where(held[:, None], rows, torch.zeros_like(rows)).to(DTYPES[c["out"]]).view(*s["ids"].shape, -1)]
    if c["grad"]:
        total = torch.zeros(w.shape, device=w.device)
        total.index_add_(0, ids.clamp(min=0), s["gout"].view(len(ids), -1).float() * held[:, None])
        out.append((total * c["scale"]).to(w.dtype))
    return out


def _run_norm(s):
    c, x = s["case"], s["x"].detach()
    total = x.float()
    if c["add"]:
        total = total + s["add"].detach().float()
    total = total.to(x.dtype)        # what the next layers and the backward pass see
    wide = total.float()
    mean = wide.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((wide - mean).square().mean(1, keepdim=True) + LN_EPS)
    xh = (wide - mean) * rstd
    y = xh * s["weight"].detach() + s["bias"].detach() if c["affine"] else xh
    out = [y.to(DTYPES[c["branch"]])] + ([total] if c["add"] else [])
    if not c["grad"]:
        return out
    g = s["gy"].float()
    gw = g * s["weight"].detach() if c["affine"] else g
    gx = rstd * (gw - gw.mean(1, keepdim=True) - xh * (gw * xh).mean(1, keepdim=True))
    if c["add"]:
        gx = gx + s["gtotal"].float()
    out.append(gx.to(x.dtype))
    if c["add"]:
        out.append(gx.to(s["add"].dtype))
    return out + ([(g * xh).sum(0), g.sum(0)] if c["affine"] else [])


def _newton_schulz(x):
    """Of a stack of matrices of one shape, in 32 bits."""
    x = x / (torch.sqrt(x.double().square().sum((1, 2), keepdim=True)) + NS_EPS).float()
    tall = x.shape[1] > x.shape[2]
    if tall:
        x = x.mT.contiguous()
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        gram = torch.bmm(x, x.mT.contiguous())
        x = a * x + torch.bmm(b * gram + c * torch.bmm(gram, gram), x)
    return x.mT if tall else x


def _by_shape(matrices):
    groups = {}
    for i, x in enumerate(matrices):
        groups.setdefault(x.shape, []).append(i)
    return groups.values()


def _run_matrices(s):
    c = s["case"]
    if c["op"] == "orthogonalize":
        updates = [g.float() for g in s["grads"]]
    else:
        updates = []
        for g, buf in zip(s["grads"], s["momenta"]):
            buf.mul_(MOMENTUM).add_(g.float() * (1.0 - MOMENTUM))
            updates.append(g.float() * (1.0 - MOMENTUM) + buf * MOMENTUM if c["nesterov"] else buf)
    out = [None] * len(updates)
    for group in _by_shape(updates):
        for i, o in zip(group, _newton_schulz(torch.stack([updates[i] for i in group])).unbind()):
            out[i] = o
    if c["op"] == "orthogonalize":
        return [o.to(g.dtype) for o, g in zip(out, s["grads"])]
    weights = s["masters"] or s["params"]
    for w, p, o in zip(weights, s["params"], out):
        new = w.float() * (1.0 - LR * DECAY) - o * (LR * math.sqrt(max(1.0, o.shape[0] / o.shape[1])))
        w.copy_(new)
        p.copy_(new)
    return s["flat"]


def run(state):
    if own:
        return _run_own(state)
    return {"embedding": _run_embedding, "layer_norm": _run_norm}.get(state["case"]["op"], _run_matrices)(state)


# ---- what a pass cannot do without ----

def work(case):
    es = DTYPES[case["dtype"]].itemsize
    if case["op"] == "embedding":
        B, T, V, C, out = case["B"], case["T"], case["V"], case["C"], DTYPES[case["out"]].itemsize
        n = sum(_lengths(case))
        # of n tokens with probabilities like 1 / k, about this many different ones
        kinds = sum(1.0 - math.exp(n * math.log1p(-1.0 / (k * math.log(V + 1.0)))) for k in range(2, V + 1)) + 1.0 if n > 1 else 1.0
        read, written = 8 * B * T + kinds * C * es, B * T * C * out
        if case["grad"]:
            read, written = read + n * C * out, written + V * C * es
        return {"bytes": float(read + written), "flops": float(n * C * (2 if case["grad"] else 1))}
    if case["op"] == "layer_norm":
        n, branch, add = case["rows"] * case["C"], DTYPES[case["branch"]].itemsize, case["add"]
        # forward: the stream and what is added to it read, the output and the new stream written; backward: the stream and the arriving
        # gradients read, the gradients of the two written (one serves for both where they have one type)
        forward = es + branch + (branch + es if add else 0)
        backward = es + branch + es + (es + (branch if branch != es else 0) if add else 0)
        return {"bytes": float(n * (forward + (backward if case["grad"] else 0))), "flops": n * (8.0 + (14.0 if case["grad"] else 0.0))}
    flops = total = 0
    for shape in _shapes(case):
        m, n = min(shape), max(shape)
        # X X^T and the square of it are symmetric: half of either
        flops += STEPS * (m * (m + 1) * n + m * (m + 1) * m + 2 * m * m * n)
        total += m * n
    # an update read and its orthogonalized form written; or gradient read, momentum and weights read and written
    each = 2 * es if case["op"] == "orthogonalize" else es + 8 + ((8 + es) if case["master"] else 2 * es)
    return {"bytes": float(total * each), "flops": float(flops)}


# ---- 64 bits ----

def _exact_norm(s):
    c = s["case"]
    leaves = {name: s[name].detach().double().requires_grad_(c["grad"]) for name in ("x", "add", "weight", "bias") if name in s}
    total = leaves["x"]
    if c["add"]:
        # (rounded to the stream's type, which a gradient passes by)
        added = total + leaves["add"]
        total = added + (added.detach().to(s["x"].dtype).double() - added.detach())
    centred = total - total.mean(1, keepdim=True)
    y = centred * (centred.pow(2).mean(1, keepdim=True) + LN_EPS).rsqrt()
    if c["affine"]:
        y = torch.addcmul(leaves["bias"], y, leaves["weight"])
    out = [y] + ([total] if c["add"] else [])
    if not c["grad"]:
        return out
    grads = torch.autograd.grad(out, list(leaves.values()), [s[name].double() for name in ("gy", "gtotal") if name in s])
    return [o.detach() for o in out] + list(grads)


def _exact_embedding(s):
    c, ids, w = s["case"], s["ids"], s["weight"].detach()
    held = ids >= 0
    out = torch.zeros(*ids.shape, c["C"], dtype=torch.float64, device=w.device)
    out[held] = w[ids[held]].double() * c["scale"]
    if not c["grad"]:
        return [out]
    grad = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
    grad.index_put_((ids[held],), s["gout"][held].double(), accumulate=True)
    return [out, grad.mul_(c["scale"])]


def _exact_orthogonal(u):
    x = u / (u.norm() + NS_EPS)
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        if x.shape[0] <= x.shape[1]:
            gram = x @ x.T
            x = a * x + b * (gram @ x) + c * (gram @ (gram @ x))
        else:
            gram = x.T @ x
            x = a * x + b * (x @ gram) + c * ((x @ gram) @ gram)
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "embedding":
        return _exact_embedding(s)
    if case["op"] == "layer_norm":
        return _exact_norm(s)
    grads = [g.double() for g in s["grads"]]
    if case["op"] == "orthogonalize":
        return [_exact_orthogonal(g) for g in grads]
    momenta = [torch.lerp(buf.double(), g, 1.0 - MOMENTUM) for buf, g in zip(s["momenta"], grads)]
    updates = [torch.lerp(g, buf, MOMENTUM) for g, buf in zip(grads, momenta)] if case["nesterov"] else momenta
    weights = []
    for w, u in zip(s["masters"] or s["params"], updates):
        weights.append(w.double() * (1.0 - LR * DECAY) - LR * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 * _exact_orthogonal(u))
    weights = torch.cat([w.reshape(-1) for w in weights])
    return {"momenta": torch.cat([buf.reshape(-1) for buf in momenta]), "params": weights, "masters": weights if case["master"] else None}
