"""Measured cases of the vocabulary and gradient-norm operators.

Three operators that stand at the two ends and in the tail of a training step against a large vocabulary:

* ``embedding``  rows of one table by token, times a scale; the table's gradient is the sum of the rows' gradients per token;
* ``xent``       softmax cross entropy of ``x . W^T + b`` over the vocabulary, with the gradients of ``x``, ``W`` and ``b``;
* ``clip``       the norm over many gradient tensors together, and the gradients scaled down to a bound.

``run`` computes them with elementary torch operations in 32 bits (``own = False``) or through ``phc_gnn_amd`` (``own = True``).
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_BYTES = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORE = -100


def listed():
    return [
        # ---- embedding: one token of a decoding step; the node types of a molecule batch (few rows, each met very often); a ragged
        # fp16 batch with padding; the largest table ----
        {"name": "emb_one_token", "op": "embedding", "dtype": "bf16", "n": 1, "v": 50000, "d": 1024, "scale": 32.0, "pad": -1, "train": False},
        {"name": "emb_node_types", "op": "embedding", "dtype": "f32", "n": 13568, "v": 119, "d": 128, "scale": 1.0, "pad": -1, "train": True},
        {"name": "emb_ragged", "op": "embedding", "dtype": "f16", "n": 4099, "v": 32003, "d": 257, "scale": 16.0, "pad": 0, "train": True},
        {"name": "emb_large", "op": "embedding", "dtype": "bf16", "n": 131072, "v": 131072, "d": 2048, "scale": 45.25, "pad": -1, "train": True},
        # ---- xent: the log-likelihood of a few tokens; a masked-node step of the fp32 models against a fragment vocabulary; an ordinary
        # 16-bit training step; odd sizes with a weight for each token; the largest step ----
        {"name": "xent_score_few", "op": "xent", "dtype": "bf16", "n": 5, "v": 32000, "d": 512, "bias": False, "reduction": "none", "train": False, "ignored": 0.0},
        {"name": "xent_fragments", "op": "xent", "dtype": "f32", "n": 13568, "v": 5000, "d": 256, "bias": True, "reduction": "mean", "train": True, "ignored": 0.85},
        {"name": "xent_step", "op": "xent", "dtype": "bf16", "n": 4096, "v": 32000, "d": 1024, "bias": False, "reduction": "mean", "train": True, "ignored": 0.05},
        {"name": "xent_weighted_odd", "op": "xent", "dtype": "f16", "n": 1021, "v": 30011, "d": 770, "bias": True, "reduction": "none", "train": True, "ignored": 0.1},
        {"name": "xent_large", "op": "xent", "dtype": "bf16", "n": 8192, "v": 131072, "d": 2048, "bias": False, "reduction": "mean", "train": True, "ignored": 0.0},
        # ---- clip: the parameters of a four-layer PHM model (norm below the bound, as in most steps); 16-bit gradients clipped into
        # 32-bit ones for the optimizer; the gradients of a large model ----
        {"name": "clip_phm_model", "op": "clip", "dtype": "f32", "layers": 4, "width": 128, "vocab": 119, "to": "inplace", "norm": 2.0, "bound": 4.0},
        {"name": "clip_mixed", "op": "clip", "dtype": "bf16", "layers": 12, "width": 768, "vocab": 32000, "to": "f32", "norm": 2.0, "bound": 0.25},
        {"name": "clip_large", "op": "clip", "dtype": "f32", "layers": 24, "width": 1280, "vocab": 50000, "to": "f32", "norm": 2.0, "bound": 0.25},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["embedding", "xent", "xent", "clip"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "embedding":
        while True:
            n, v, d = _log_int(rng, 1, 131072), _log_int(rng, 50, 131072), _log_int(rng, 32, 4096)
            if rng.random() < 0.6:
                d = max(32, d // 8 * 8)
            if (n + v) * d * _BYTES[dtype] <= 262144 * 2048 * 2:
                break
        return {"op": op, "dtype": dtype, "n": n, "v": v, "d": d, "scale": rng.choice([1.0, 0.5, math.sqrt(d)]),
                "pad": rng.choice([-1, 0, v - 1]), "train": rng.random() < 0.75}
    if op == "xent":
        while True:
            n, v, d = _log_int(rng, 1, 16384), _log_int(rng, 1000, 131072), _log_int(rng, 64, 4096)
            if rng.random() < 0.6:
                d = d // 8 * 8
            # (a product in 32 bits costs several times one in 16)
            if n * v * d * (8 if dtype == "f32" else 1) <= 8192 * 131072 * 2048:
                break
        return {"op": op, "dtype": dtype, "n": n, "v": v, "d": d, "bias": rng.random() < 0.5,
                "reduction": rng.choice(["mean", "mean", "sum", "none"]), "train": rng.random() < 0.75, "ignored": rng.choice([0.0, 0.1, 0.85])}
    layers, width, vocab = rng.randint(1, 24), _log_int(rng, 64, 1280), _log_int(rng, 28, 50000)
    to = rng.choice(["inplace", "same", "f32"])
    return {"op": op, "dtype": dtype, "layers": layers, "width": width, "vocab": vocab, "to": to,
            "norm": rng.choice([2.0, 2.0, 1.0, math.inf]), "bound": 4.0 if to == "inplace" else rng.choice([0.25, 4.0])}


def _clip_shapes(case):
    """A table, then per layer four square maps, a widening and a narrowing one, their biases, two norms and small rule tensors."""
    w, out = case["width"], [(case["vocab"], case["width"])]
    for _ in range(case["layers"]):
        out += [(w, w)] * 4 + [(4 * w, w), (w, 4 * w), (4 * w,), (w,), (w,), (w,), (w,), (4, 4, 4), (1,)]
    return out


def _clip_out_dtype(case):
    return torch.float32 if case["to"] == "f32" else _DTYPES[case["dtype"]]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "clip":
        shapes = _clip_shapes(case)
        size = sum(math.prod(s) for s in shapes)
        size_of = [math.prod(s) for s in shapes]
        if case["to"] == "inplace":
            # gradients that live in one flat buffer, as a data-parallel step keeps them
            state["flat"] = torch.empty(size, dtype=dt, device=dev)
            grads = [t.view(s) for t, s in zip(state["flat"].split(size_of), shapes)]
        else:
            grads = [torch.empty(s, dtype=dt, device=dev) for s in shapes]
        for i, t in enumerate(grads):
            t.copy_(torch.randn(t.shape, generator=g, device=dev) * (0.005 + 0.001 * (i % 7)))
        state["grads"] = grads
        # the bound as a share of the norm to expect: 0.25 clips, 4 does not (in place it never does: a pass leaves its input as it is)
        state["max_norm"] = case["bound"] * {2.0: 0.008 * math.sqrt(size), 1.0: 0.0064 * size, math.inf: 0.04}[case["norm"]]
        if case["to"] == "inplace":
            params = []
            for t in grads:
                p = torch.nn.Parameter(torch.empty_like(t))
                p.grad = t
                params.append(p)
            state["params"] = params
        else:
            # the optimizer's own flat gradient buffer
            state["flat"] = torch.empty(size, dtype=_clip_out_dtype(case), device=dev)
            state["out"] = [t.view(s) for t, s in zip(state["flat"].split(size_of), shapes)]
        return state
    n, v, d = case["n"], case["v"], case["d"]
    # token frequencies fall with the token's number, as in a sorted vocabulary
    u = torch.rand(n, generator=g, device=dev, dtype=torch.float64)
    tokens = ((float(v + 1) ** u).long() - 1).clamp_(0, v - 1)
    if case["op"] == "embedding":
        state["tokens"] = tokens
        state["weight"] = (torch.randn(v, d, generator=g, device=dev) * 0.02).to(dt).requires_grad_(case["train"])
        if case["train"]:
            state["dy"] = torch.randn(n, d, generator=g, device=dev).mul_(0.125).to(dt)
        return state
    w = torch.randn(v, d, generator=g, device=dev) * (2.0 / math.sqrt(d))
    x = torch.randn(n, d, generator=g, device=dev)
    # some tokens are predicted well already: their row leans towards the target's
    x.add_(w[tokens] * (2.0 * torch.rand(n, 1, generator=g, device=dev)))
    if case["ignored"] > 0:
        tokens = torch.where(torch.rand(n, generator=g, device=dev) < case["ignored"], torch.full_like(tokens, _IGNORE), tokens)
        tokens[0] = v - 1                      # one token at least is not ignored
    state["target"] = tokens
    state["x"] = x.to(dt).requires_grad_(case["train"])
    state["weight"] = w.to(dt).requires_grad_(case["train"])
    state["bias"] = (torch.randn(v, generator=g, device=dev) * 0.5).to(dt).requires_grad_(case["train"]) if case["bias"] else None
    if case["train"]:
        state["upstream"] = torch.rand(n, generator=g, device=dev) if case["reduction"] == "none" else torch.ones((), device=dev)
    return state


# ---- the framework's operators ----------------------------------------------------------------------------------------------------
def _run_own(state):
    case = state["case"]
    if case["op"] == "clip":
        from phc_gnn_amd import optim
        if case["to"] == "inplace":
            norm = optim.clip_grad_norm_(state["params"], state["max_norm"], norm_type=case["norm"])
            return [norm, state["flat"]]
        norm, _ = optim.clip_grads(state["grads"], state["max_norm"], norm_type=case["norm"], out=state["out"])
        return [norm, state["flat"]]
    from phc_gnn_amd import ops
    if case["op"] == "embedding":
        w = state["weight"]
        y = ops.embedding(state["tokens"], w, scale=case["scale"], padding_idx=None if case["pad"] < 0 else case["pad"])
        if not case["train"]:
            return [y]
        (dw,) = torch.autograd.grad(y, [w], state["dy"])
        return [y.detach(), dw]
    leaves = [t for t in (state["x"], state["weight"], state["bias"]) if t is not None]
    loss = ops.linear_cross_entropy(state["x"], state["weight"], state["target"], bias=state["bias"], ignore_index=_IGNORE,
                                    reduction=case["reduction"])
    if not case["train"]:
        return [loss]
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves, state["upstream"]))


# ---- plain form: elementary operations in 32 bits ------------------------------------------------------------------------------------
def _run_plain(state):
    case = state["case"]
    if case["op"] == "clip":
        parts = []
        for t in state["grads"]:
            f = t.float()
            parts.append((f * f).sum() if case["norm"] == 2.0 else (f.abs().sum() if case["norm"] == 1.0 else f.abs().max()))
        parts = torch.stack(parts)
        norm = torch.sqrt(parts.sum()) if case["norm"] == 2.0 else (parts.sum() if case["norm"] == 1.0 else parts.max())
        coef = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
        if case["to"] == "inplace":
            for t in state["grads"]:
                t.copy_(t.float() * coef)
            return [norm, state["flat"]]
        for t, o in zip(state["grads"], state["out"]):
            o.copy_(t.float() * coef)
        return [norm, state["flat"]]
    if case["op"] == "embedding":
        tokens, w = state["tokens"], state["weight"].detach()
        y = (w[tokens].float() * case["scale"]).to(w.dtype)
        if not case["train"]:
            return [y]
        dw = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
        dw.index_add_(0, tokens, state["dy"].float())
        dw *= case["scale"]
        if case["pad"] >= 0:
            dw[case["pad"]] = 0.0
        return [y, dw.to(w.dtype)]
    x, w, t = state["x"].detach(), state["weight"].detach(), state["target"]
    xf, wf = x.float(), w.float()
    logits = xf @ wf.t()
    if state["bias"] is not None:
        logits += state["bias"].detach().float()
    valid = t != _IGNORE
    at = torch.where(valid, t, torch.zeros_like(t))
    top = logits.max(dim=1, keepdim=True).values
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    losses = (torch.log(total) + top - logits.gather(1, at[:, None]))[:, 0]
    losses = torch.where(valid, losses, torch.zeros_like(losses))
    count = valid.sum().float()
    loss = losses if case["reduction"] == "none" else (losses.sum() if case["reduction"] == "sum" else losses.sum() / count)
    if not case["train"]:
        return [loss]
    g = state["upstream"] if case["reduction"] == "none" else (torch.ones_like(losses) if case["reduction"] == "sum" else torch.ones_like(losses) / count)
    g = torch.where(valid, g, torch.zeros_like(g))
    dl = e.div_(total)
    dl[torch.arange(len(t), device=t.device), at] -= 1.0
    dl *= g[:, None]
    out = [loss, (dl @ wf).to(x.dtype), (dl.t() @ xf).to(w.dtype)]
    if state["bias"] is not None:
        out.append(dl.sum(dim=0).to(w.dtype))
    return out


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------
def _exact_xent(case, s):
    """Tokens in pieces, from the definition: p = softmax(x W^T + b), loss_i = -log p_{i,t_i}, and the chain rule."""
    w = s["weight"].detach().double()
    b = None if s["bias"] is None else s["bias"].detach().double()
    t = s["target"]
    n, v = t.shape[0], w.shape[0]
    kept = (t != _IGNORE).double()
    if case["reduction"] == "mean":
        weight_of = kept / kept.sum()
    else:
        weight_of = kept.clone()
    up = weight_of * s["upstream"].double() if case["train"] else None
    dw = torch.zeros_like(w) if case["train"] else None
    db = torch.zeros(v, dtype=torch.float64, device=w.device)
    dx, losses = [], []
    piece = max(1, min(n, (1 << 28) // v))
    for i in range(0, n, piece):
        xi = s["x"].detach()[i:i + piece].double()
        z = xi @ w.t()
        if b is not None:
            z = z + b
        logp = z - torch.logsumexp(z, dim=1, keepdim=True)
        del z
        hit = (torch.arange(v, device=w.device)[None, :] == t[i:i + piece, None])
        losses.append(-(logp.masked_fill(~hit, 0.0)).sum(dim=1))
        if case["train"]:
            dz = (logp.exp() - hit.double()) * up[i:i + piece, None]
            dx.append(dz @ w)
            dw += dz.t() @ xi
            db += dz.sum(dim=0)
    losses = torch.cat(losses) * kept
    loss = losses if case["reduction"] == "none" else (losses * weight_of).sum()
    if not case["train"]:
        return [loss]
    return [loss, torch.cat(dx), dw] + ([db] if b is not None else [])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        flat = [t.double() for t in s["grads"]]
        if case["norm"] == math.inf:
            norm = torch.stack([t.abs().amax() for t in flat]).amax()
        else:
            norm = torch.stack([t.abs().pow(case["norm"]).sum() for t in flat]).sum().pow(1.0 / case["norm"])
        coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
        return [norm, torch.cat([t.flatten() for t in flat]) * coef]
    if case["op"] == "embedding":
        w = s["weight"].detach()
        y = torch.index_select(w, 0, s["tokens"]).double() * case["scale"]
        if not case["train"]:
            return [y]
        # tokens in sorted order, one running sum per run
        order = torch.argsort(s["tokens"], stable=True)
        dw = torch.zeros(w.shape, dtype=torch.float64, device=w.device)
        for i in range(0, len(order), 16384):
            rows = order[i:i + 16384]
            dw.index_put_((s["tokens"][rows],), s["dy"][rows].double() * case["scale"], accumulate=True)
        if case["pad"] >= 0:
            dw[case["pad"]].zero_()
        return [y, dw]
    return _exact_xent(case, s)


def work(case):
    s = _BYTES[case["dtype"]]
    if case["op"] == "clip":
        size = sum(math.prod(t) for t in _clip_shapes(case))
        written = 0 if case["to"] == "inplace" else size * (4 if case["to"] == "f32" else s)
        return {"bytes": size * s + written + 4, "flops": 2 * size + (0 if case["to"] == "inplace" else size)}
    n, v, d = case["n"], case["v"], case["d"]
    if case["op"] == "embedding":
        rows = min(n, v)
        forward = 8 * n + rows * d * s + n * d * s
        return {"bytes": forward + (n * d * s + v * d * s if case["train"] else 0), "flops": n * d * (2 if case["train"] else 1)}
    reads = (n + v) * d * s + 8 * n + (v * s if case["bias"] else 0)
    out = 4 * (n if case["reduction"] == "none" else 1)
    if not case["train"]:
        return {"bytes": reads + out, "flops": 2 * n * v * d}
    return {"bytes": 2 * reads - 8 * n + out, "flops": 6 * n * v * d}
