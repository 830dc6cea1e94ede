"""Timed cases of the model operators: layer norm, causal attention over packed sequences, top-k distillation.

These are what runs between the hooked Linear modules of a collection step: the norms and the attention of the
model's forward and backward pass, and the loss on its logits.  A case with `train` true is a training step's
share (forward, then the gradients from a given output gradient); without it, the forward pass alone.

`run` computes a case either in its plain form (elementary torch operations in 32 bits, rounded once at the
end) or, with `own` set, through the package's entry points.  `exact` is the definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


# ---- the cases ------------------------------------------------------------------------------------------------

def listed() -> list[dict]:
    return [
        # a document of a single token, forward only: nothing but latency
        dict(name="norm-one-token", op="norm", rows=1, d=768, dtype="bfloat16", train=False),
        # one 4096-token batch of the 768-wide model, norms trained (the Trainer callback's use)
        dict(name="norm-768-train", op="norm", rows=4096, d=768, dtype="bfloat16", train=True),
        # odd sizes in full precision: rows that start on no vector boundary
        dict(name="norm-odd-fp32", op="norm", rows=1531, d=1001, dtype="float32", train=True),
        # a large token batch of the 4096-wide decoder
        dict(name="norm-4096-train", op="norm", rows=32768, d=4096, dtype="bfloat16", train=True),
        # many short documents packed into one batch (instruction data), forward only
        dict(name="attention-short-docs", op="attention", layout="packed", lengths=_spread(48, 1, 96, 7), heads=12,
             kv_heads=12, head_dim=64, dtype="bfloat16", train=False),
        # the collection benchmark's batch: 4 documents of 1024 tokens, 12 heads of 64, q/k/v views of one projection
        dict(name="attention-12x64-train", op="attention", layout="batch", lengths="1024 1024 1024 1024", heads=12,
             kv_heads=12, head_dim=64, dtype="bfloat16", train=True),
        # documents of very different lengths packed without padding, 16 heads of 64
        dict(name="attention-packed-train", op="attention", layout="packed", lengths=_lognormal(24, 11), heads=16,
             kv_heads=16, head_dim=64, dtype="float16", train=True),
        # the decoder with grouped heads: 32 query heads on 8 key/value heads of 128
        dict(name="attention-grouped-train", op="attention", layout="batch", lengths="4096 4096", heads=32, kv_heads=8,
             head_dim=128, dtype="bfloat16", train=True),
        # one long document through the same decoder, forward only
        dict(name="attention-long", op="attention", layout="packed", lengths="16384", heads=32, kv_heads=8,
             head_dim=128, dtype="bfloat16", train=False),
        # a handful of supervised tokens, vocabulary of odd size, full precision
        dict(name="distill-few-fp32", op="distill", rows=3, vocab=50257, k=8, temperature=2.0, dtype="float32",
             train=True),
        # the collection benchmark's logits against 64 teacher entries a token
        dict(name="distill-50k-train", op="distill", rows=4096, vocab=50304, k=64, temperature=1.0, dtype="bfloat16",
             train=True),
        # the decoder's vocabulary, a ragged number of supervised tokens
        dict(name="distill-128k-train", op="distill", rows=2047, vocab=128256, k=32, temperature=1.0,
             dtype="bfloat16", train=True),
    ]


def _text(lengths: list[int]) -> str:
    return " ".join(map(str, lengths))


def _lengths(case: dict) -> list[int]:
    return [int(v) for v in case["lengths"].split()]


def _spread(n: int, lo: int, hi: int, step: int) -> str:
    return _text([lo + (i * step * 5) % (hi - lo + 1) for i in range(n)])


def _lognormal(n: int, seed: int) -> str:
    """Document lengths as a text corpus has them: lognormal around 400 tokens, 16 to 2048."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.exp(6.0 + torch.randn(n, generator=gen, dtype=torch.float64))
    return _text([int(v) for v in x.round().clamp(16, 2048)])


def _log_uniform(rng, lo: float, hi: float) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["norm", "attention", "attention", "distill"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    train = rng.random() < 0.7
    if op == "norm":
        d = _log_uniform(rng, 32, 8192)
        rows = _log_uniform(rng, 1, min(32768, (1 << (27 if dtype != "float32" else 26)) // d))
        return dict(op=op, rows=rows, d=d, dtype=dtype, train=train)
    if op == "distill":
        vocab = _log_uniform(rng, 1000, 131072)
        rows = _log_uniform(rng, 1, min(4096, (1 << 26) // vocab))
        return dict(op=op, rows=rows, vocab=vocab, k=_log_uniform(rng, 1, 128),
                    temperature=rng.choice([1.0, 2.0, 0.7]), dtype=dtype, train=True)
    head_dim = rng.choice([32, 64, 64, 80, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4])
    layout = rng.choice(["packed", "batch"])
    longest = _log_uniform(rng, 1, 4096 if dtype != "float32" else 1024)
    n = max(1, min(32, _log_uniform(rng, 1, 16384) // longest))
    lengths = [rng.randint(max(1, longest // 8), longest) for _ in range(n)]
    return dict(op=op, layout=layout, lengths=_text(lengths), heads=heads, kv_heads=kv_heads, head_dim=head_dim,
                dtype=dtype, train=train)


def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["d"]
        if not case["train"]:
            return {"bytes": 2 * n * size + 2 * case["d"] * size, "flops": 8 * n}
        return {"bytes": 4 * n * size + 4 * case["d"] * size, "flops": 22 * n}
    if case["op"] == "distill":
        n = case["rows"] * case["vocab"]
        entries = case["rows"] * case["k"] * 8
        if not case["train"]:
            return {"bytes": n * size + entries + 4 * case["rows"], "flops": 4 * n}
        return {"bytes": 2 * n * size + entries + 8 * case["rows"], "flops": 8 * n}
    lengths = _lengths(case)
    tokens = sum(lengths)
    pairs = sum(l * (l + 1) // 2 for l in lengths) * case["heads"]
    q, kv = tokens * case["heads"] * case["head_dim"], tokens * case["kv_heads"] * case["head_dim"]
    if not case["train"]:
        return {"bytes": (2 * q + 2 * kv) * size, "flops": 4 * pairs * case["head_dim"]}
    return {"bytes": (4 * q + 4 * kv) * size, "flops": 14 * pairs * case["head_dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------

def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["train"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    state = {"op": case["op"], "train": train}
    if case["op"] == "norm":
        rows, d = case["rows"], case["d"]
        # a residual stream: a common offset and a few loud features
        x = randn(rows, d) * (1 + 4 * (torch.rand(d, generator=gen, device=dev) > 0.98)) + 0.3
        state.update(x=x.to(dtype), weight=(1 + 0.2 * randn(d)).to(dtype), bias=(0.1 * randn(d)).to(dtype), eps=1e-5)
        if train:
            state["grad"] = randn(rows, d).to(dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
        return state
    if case["op"] == "distill":
        rows, vocab, k = case["rows"], case["vocab"], case["k"]
        logits = 2.5 * randn(rows, vocab)
        # the teacher agrees with the student up to noise; its highest entries are what was kept
        noisy = logits + randn(rows, vocab)
        top = torch.topk(noisy, k, dim=1)
        state.update(logits=logits.to(dtype), ids=top.indices.contiguous(), teacher=top.values.to(dtype).contiguous(),
                     temperature=case["temperature"])
        if train:
            state["logits"].requires_grad_()
            state["grad"] = torch.rand(rows, generator=gen, device=dev) + 0.5
        return state
    lengths, heads, kv_heads, dim = _lengths(case), case["heads"], case["kv_heads"], case["head_dim"]
    state.update(lengths=lengths, layout=case["layout"], scale=dim ** -0.5)
    if case["layout"] == "packed":
        lead = (sum(lengths),)
        ends = torch.tensor([0] + lengths).cumsum(0)
        state["cu_seqlens"] = ends.to(torch.int32).to(dev)
    else:
        lead = (len(lengths), max(lengths))
        state["device_lengths"] = torch.tensor(lengths, dtype=torch.int32, device=dev)
    # queries, keys and values are views of one projection's output, as a model has them
    if heads == kv_heads:
        qkv = (1.2 * randn(*lead, heads, 3 * dim)).to(dtype)
        q, k, v = qkv.split(dim, dim=-1)
    else:
        q = (1.2 * randn(*lead, heads, dim)).to(dtype)
        k, v = (1.2 * randn(*lead, kv_heads, 2 * dim)).to(dtype).split(dim, dim=-1)
    state.update(q=q.detach(), k=k.detach(), v=v.detach())
    if train:
        state["grad"] = randn(*lead, heads, dim).to(dtype)
        for name in ("q", "k", "v"):
            state[name].requires_grad_()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------

def run(state: dict):
    return _run_own(state) if own else _PLAIN[state["op"]](state)


def _run_own(state: dict):
    import bergson_amd as B

    if state["op"] == "norm":
        leaves = (state["x"], state["weight"], state["bias"])
        out = B.layer_norm(*leaves, eps=state["eps"])
    elif state["op"] == "distill":
        leaves = (state["logits"],)
        out = B.topk_distillation(state["logits"], state["ids"], state["teacher"], temperature=state["temperature"])
    else:
        leaves = (state["q"], state["k"], state["v"])
        if state["layout"] == "packed":
            out = B.causal_attention(*leaves, cu_seqlens=state["cu_seqlens"], scale=state["scale"])
        else:
            out = B.causal_attention(*leaves, lengths=state["device_lengths"], scale=state["scale"])
    if not state["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, leaves, state["grad"]))


def _plain_norm(state: dict):
    with torch.no_grad():
        x = state["x"]
        wide, weight, bias = x.float(), state["weight"].float(), state["bias"].float()
        centred = wide - wide.mean(1, keepdim=True)
        rstd = 1.0 / (centred.square().mean(1, keepdim=True) + state["eps"]).sqrt()
        unit = centred * rstd
        out = (unit * weight + bias).to(x.dtype)
        if not state["train"]:
            return out
        grad = state["grad"].float()
        inner = grad * weight
        dx = rstd * (inner - inner.mean(1, keepdim=True) - unit * (inner * unit).mean(1, keepdim=True))
        return out, dx.to(x.dtype), (grad * unit).sum(0).to(x.dtype), grad.sum(0).to(x.dtype)


def _plain_distill(state: dict):
    with torch.no_grad():
        logits, ids, tau = state["logits"], state["ids"], state["temperature"]
        z = logits.float() / tau
        z = z - z.amax(1, keepdim=True)
        exps = z.exp()
        total = exps.sum(1, keepdim=True)
        t = state["teacher"].float() / tau
        t = t - t.amax(1, keepdim=True)
        log_p = t - t.exp().sum(1, keepdim=True).log()
        p = log_p.exp()
        log_q = z.gather(1, ids) - total.log()
        losses = tau * tau * (p * (log_p - log_q)).sum(1)
        if not state["train"]:
            return losses
        dz = exps / total
        dz.scatter_add_(1, ids, -p)
        dz *= (tau * state["grad"]).unsqueeze(1)
        return losses, dz.to(logits.dtype)


def _sequences(state: dict):
    """Index of every sequence's rows in the leading dimension(s)."""
    start = 0
    for n, length in enumerate(state["lengths"]):
        if state["layout"] == "packed":
            yield slice(start, start + length)
            start += length
        else:
            yield (n, slice(0, length))


def _plain_attention(state: dict):
    with torch.no_grad():
        q, k, v = state["q"], state["k"], state["v"]
        heads, kv_heads, scale, train = q.shape[-2], k.shape[-2], state["scale"], state["train"]
        group = heads // kv_heads
        out = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        grads = [torch.zeros(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v)] if train else []
        for rows in _sequences(state):
            length = q[rows].shape[0]
            # as many key/value heads at a time as keep the score matrices at a few GB
            step = max(1, min(kv_heads, (1 << 29) // max(1, length * length * group)))
            future = torch.ones(length, length, dtype=torch.bool, device=q.device).triu(1)
            for h in range(0, kv_heads, step):
                kv = slice(h, min(h + step, kv_heads))
                qh = slice(kv.start * group, kv.stop * group)
                qs = q[rows][:, qh].float().transpose(0, 1).unflatten(0, (-1, group)).flatten(1, 2)  # [kv, group * len, D]
                ks = k[rows][:, kv].float().transpose(0, 1).contiguous()
                vs = v[rows][:, kv].float().transpose(0, 1).contiguous()
                s = (qs @ ks.transpose(1, 2).contiguous()).mul_(scale).unflatten(1, (group, length))
                s.masked_fill_(future, float("-inf"))
                s -= s.amax(3, keepdim=True)
                s.exp_()
                s /= s.sum(3, keepdim=True)
                p = s.flatten(1, 2)
                o = p @ vs

                def place(t, width):  # [kv, group * len, D] -> [len, heads, D]
                    return t.unflatten(1, (width, length)).flatten(0, 1).transpose(0, 1)

                out[rows][:, qh] = place(o, group).to(q.dtype)
                if not train:
                    continue
                do = state["grad"][rows][:, qh].float().transpose(0, 1).unflatten(0, (-1, group)).flatten(1, 2)
                dv = p.transpose(1, 2).contiguous() @ do
                dp = do @ vs.transpose(1, 2).contiguous()
                dp -= (do * o).sum(2, keepdim=True)
                dp *= p
                ds = dp.mul_(scale)
                grads[0][rows][:, qh] = place(ds @ ks, group).to(q.dtype)
                grads[1][rows][:, kv] = place(ds.transpose(1, 2).contiguous() @ qs, 1).to(q.dtype)
                grads[2][rows][:, kv] = place(dv, 1).to(q.dtype)
        return (out, *grads) if train else out


_PLAIN = {"norm": _plain_norm, "distill": _plain_distill, "attention": _plain_attention}


# ---- the definition in 64 bits --------------------------------------------------------------------------------

def exact(case: dict, seed: int):
    state = prepare(case, seed)
    leaves = {name: t.detach().double() for name, t in state.items()
              if isinstance(t, torch.Tensor) and t.is_floating_point()}
    if case["op"] == "norm":
        return _exact_norm(leaves, state)
    if case["op"] == "distill":
        return _exact_distill(leaves, state)
    return _exact_attention(leaves, state)


def _exact_norm(t: dict, state: dict):
    names = ("x", "weight", "bias")
    for name in names:
        t[name].requires_grad_(state["train"])
    var, mean = torch.var_mean(t["x"], dim=-1, correction=0, keepdim=True)
    out = (t["x"] - mean) / torch.sqrt(var + state["eps"]) * t["weight"] + t["bias"]
    if not state["train"]:
        return out
    return (out.detach(), *torch.autograd.grad(out, [t[name] for name in names], t["grad"]))


def _exact_distill(t: dict, state: dict):
    tau = state["temperature"]
    z = t["logits"].requires_grad_(state["train"])
    log_q = torch.log_softmax(z / tau, dim=-1)
    log_p = torch.log_softmax(t["teacher"] / tau, dim=-1)
    losses = tau ** 2 * (log_p.exp() * (log_p - torch.take_along_dim(log_q, state["ids"], 1))).sum(-1)
    if not state["train"]:
        return losses
    return losses.detach(), torch.autograd.grad(losses, z, t["grad"])[0]


def _exact_attention(t: dict, state: dict):
    """Head by head: softmax over the allowed positions, gradients by automatic differentiation."""
    q, k, v = t["q"], t["k"], t["v"]
    group = q.shape[-2] // k.shape[-2]
    result = [torch.zeros_like(x) for x in ((q, q, k, v) if state["train"] else (q,))]
    for rows in _sequences(state):
        length = q[rows].shape[0]
        allowed = torch.arange(length, device=q.device)
        allowed = allowed[:, None] >= allowed[None, :]
        for h in range(q.shape[-2]):
            parts = [x[rows][:, i].contiguous().requires_grad_(state["train"]) for x, i in
                     ((q, h), (k, h // group), (v, h // group))]
            scores = torch.where(allowed, parts[0] @ parts[1].T * state["scale"], -math.inf)
            out = torch.softmax(scores, dim=1) @ parts[2]
            result[0][rows][:, h] = out.detach()
            if state["train"]:
                dq, dk, dv = torch.autograd.grad(out, parts, t["grad"][rows][:, h])
                result[1][rows][:, h] = dq
                result[2][rows][:, h // group] += dk
                result[3][rows][:, h // group] += dv
    return tuple(result) if state["train"] else result[0]
