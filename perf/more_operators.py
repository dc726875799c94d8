"""The operators of policy training and serving of adapters over quantized weights, for timing.

Three kinds of call, over the sizes, bit widths and group sizes they are used with:

* ``logp``  log probabilities of given tokens through a quantized vocabulary head, the entropy
            and the likeliest tokens; or, of a training step, the same without the likeliest
            tokens and the gradient of the hidden states;
* ``lora``  a quantized projection with low-rank adapters of many requests beside it, or its
            gradients (the input's and the adapters');
* ``clip``  the norm over many gradients and the gradients clipped to it.

Weights follow the distributions of the repository's benchmark: 4-bit scales uniform in
[0.002, 0.02] with biases near -8 scale; 8-bit scales uniform in [1e-4, 2e-3] with biases
-128 scale.  The weights of every product are the bf16 values that ``ops.dequantize`` gives.
"""
import math

import torch

own = False

DEV = "cuda"


def listed():
    return [
        # One decoded token with its 20 likeliest alternatives: the latency of reading the head once.
        dict(name="logp_m1_top20", kind="logp", M=1, V=32000, K=2048, bits=4, group=64, k=1, top=20,
             T=1.0, step=False),
        # Scoring a prompt chunk of odd length over a large vocabulary, groups of 128, 5 alternatives.
        dict(name="logp_m509_top5", kind="logp", M=509, V=151936, K=2048, bits=4, group=128, k=1,
             top=5, T=1.0, step=False),
        # Scoring a long batch through an 8B-sized head, four candidate answers a position.
        dict(name="logp_m2048_top20", kind="logp", M=2048, V=128256, K=4096, bits=4, group=64, k=4,
             top=20, T=1.0, step=False),
        # A small policy step on an 8-bit checkpoint with an odd vocabulary.
        dict(name="logp_step_m37", kind="logp", M=37, V=50257, K=1024, bits=8, group=64, k=1, top=0,
             T=1.0, step=True),
        # A policy step over a batch of sampled answers, sampled at a temperature of 0.7.
        dict(name="logp_step_m1000", kind="logp", M=1000, V=128256, K=4096, bits=4, group=64, k=1,
             top=0, T=0.7, step=True),
        # One token of one request through a square projection: latency.
        dict(name="lora_m1", kind="lora", M=1, N=4096, K=4096, E=8, r=16, bits=4, group=64, grad=False),
        # A decode batch of many requests, each with its own adapter or none, through a gate projection.
        dict(name="lora_m48_e32", kind="lora", M=48, N=14336, K=4096, E=32, r=16, bits=4, group=64,
             grad=False),
        # A prompt batch of several requests with adapters of a high rank.
        dict(name="lora_m2048_r64", kind="lora", M=2048, N=14336, K=4096, E=8, r=64, bits=4, group=64,
             grad=False),
        # A short fine-tuning batch, small rank, 8 bits, a key projection.
        dict(name="lora_step_m509", kind="lora", M=509, N=1024, K=4096, E=1, r=8, bits=8, group=64,
             grad=True),
        # A training batch of one adapter through a gate projection.
        dict(name="lora_step_m2048", kind="lora", M=2048, N=14336, K=4096, E=1, r=32, bits=4, group=64,
             grad=True),
        # The adapters' gradients of one small layer: launch latency.
        dict(name="clip_layer", kind="clip", layers=1, D=2048, I=5632, kv=256, r=8, bf16=False,
             max_norm=1.0),
        # The adapters' gradients of a whole 8B-sized model.
        dict(name="clip_model", kind="clip", layers=32, D=4096, I=14336, kv=1024, r=32, bf16=False,
             max_norm=1.0),
    ]


def _logint(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    return max(lo, _logint(rng, lo, hi) // step * step)


def _seconds(case):
    """A rough estimate of a pass, to keep drawn cases below the largest listed one."""
    w = work(case)
    return w["bytes"] / 4e12 + w["flops"] / 1e15


def draw(rng):
    most = max(_seconds(c) for c in listed())
    while True:
        kind = rng.choice(("logp", "logp", "lora", "lora", "clip"))
        bits = rng.choice((4, 4, 8))
        group = rng.choice((64, 64, 32, 128))
        K = _width(rng, 512, 8192, rng.choice((256, 256, 128)))
        if kind == "logp":
            step = rng.random() < 0.4
            c = dict(kind=kind, M=_logint(rng, 1, 2048), V=_logint(rng, 1000, 152000), K=K, bits=bits,
                     group=group, k=rng.choice((1, 1, rng.randint(2, 16))),
                     top=0 if step else rng.choice((0, 1, rng.randint(2, 64))),
                     T=rng.choice((1.0, 1.0, round(rng.uniform(0.5, 1.5), 2))), step=step)
        elif kind == "lora":
            c = dict(kind=kind, M=_logint(rng, 1, 4096), N=_width(rng, 256, 16384, 8), K=K,
                     E=rng.choice((1, 4, 16, 64)), r=rng.choice((8, 16, 32, 64, 128)), bits=bits,
                     group=group, grad=rng.random() < 0.5)
        else:
            D = _width(rng, 512, 8192, 64)
            c = dict(kind=kind, layers=_logint(rng, 1, 48), D=D, I=_width(rng, D, 4 * D, 8),
                     kv=_width(rng, 64, D, 64), r=rng.choice((4, 8, 16, 32, 64)),
                     bf16=rng.random() < 0.4, max_norm=round(rng.uniform(0.2, 2.0), 2))
        if _seconds(c) <= most:
            return c


# ---- inputs -------------------------------------------------------------------


def _packed(gen, N, K, bits, group):
    """A random quantized weight [N, K]: (words, scales, biases)."""
    w = torch.randint(-2**31, 2**31, (N, K * bits // 32), dtype=torch.int32, device=DEV,
                      generator=gen)
    lo, hi, mid = (0.002, 0.02, 8) if bits == 4 else (1e-4, 2e-3, 128)
    s = torch.empty(N, K // group, device=DEV).uniform_(lo, hi, generator=gen).bfloat16()
    b = -mid * s.float()
    if bits == 4:
        b += torch.empty_like(b).normal_(0.0, 1e-3, generator=gen)
    return w, s, b.bfloat16()


def _normal(gen, *shape):
    return torch.empty(*shape, device=DEV).normal_(generator=gen)


def _uniform(gen, *shape):
    return torch.empty(*shape, device=DEV).uniform_(generator=gen)


def _ints(gen, n, *shape):
    return torch.randint(0, n, shape, device=DEV, generator=gen)


def _adapter_ids(gen, M, E):
    """An adapter for each row, one row or run in ten without: rows of their own in a decode
    batch, runs of a request's rows in a longer one; one adapter takes all rows."""
    if E == 1:
        return torch.zeros(M, dtype=torch.int32, device=DEV)
    if M <= 64:
        run = torch.arange(M, device=DEV)
    else:
        # About two runs an adapter, of uneven lengths.
        starts = (_uniform(gen, M) < 2 * E / M).long()
        run = starts.cumsum(0)
    pick = _ints(gen, E, M)
    pick = torch.where(_uniform(gen, M) < 0.1, torch.full_like(pick, -1), pick)
    return pick[run.clamp(max=M - 1)].int()


def _clip_shapes(c):
    """Shapes of the adapters of a transformer's layers: q, k, v, o, gate, up and down."""
    D, I, kv, r = c["D"], c["I"], c["kv"], c["r"]
    layer = []
    for n, k in ((D, D), (kv, D), (kv, D), (D, D), (I, D), (I, D), (D, I)):
        layer += [(r, k), (n, r)]
    return layer * c["layers"]


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    p = {"case": dict(c)}
    if c["kind"] == "logp":
        M, V, K, k = c["M"], c["V"], c["K"], c["k"]
        p["w"] = _packed(gen, V, K, c["bits"], c["group"])
        likely = _ints(gen, V, M)
        # Hidden states that lean towards a token by as much as a trained model's do: from not
        # at all to a clear favourite.
        rows = _weights(c, tuple(t[likely] for t in p["w"]))
        p["h"] = (_normal(gen, M, K) + rows * 1.5 * _uniform(gen, M, 1)).bfloat16()
        # The given tokens of a row differ; the first is the likely one, one in twenty is absent.
        at = torch.arange(k, device=DEV)
        ids = (likely[:, None] + at * (1 + _ints(gen, V // k, M, 1))) % V
        p["ids"] = torch.where(_uniform(gen, M, k) < 0.05, torch.full_like(ids, -1), ids).int()
        # Advantages and the entropy bonus, in the mean over the tokens.
        p["da"] = _normal(gen, M, k) / M
        p["dent"] = torch.full((M,), -0.01 / M, device=DEV)
    elif c["kind"] == "lora":
        M, N, K, E, r = c["M"], c["N"], c["K"], c["E"], c["r"]
        p["w"] = _packed(gen, N, K, c["bits"], c["group"])
        p["x"] = _normal(gen, M, K).bfloat16()
        p["a"] = (_normal(gen, E, r, K) / math.sqrt(K)).bfloat16()
        p["b"] = (_normal(gen, E, N, r) * 0.5 / math.sqrt(r)).bfloat16()
        p["adapters"] = _adapter_ids(gen, M, E)
        p["scales"] = 0.5 + 1.5 * _uniform(gen, E)
        if c["grad"]:
            p["dy"] = (_normal(gen, M, N) / M).bfloat16()
    else:
        t = torch.bfloat16 if c["bf16"] else torch.float32
        shapes = _clip_shapes(c)
        p["grads"] = [(_normal(gen, *s) * (1e-3 * (1 + i % 7))).to(t) for i, s in enumerate(shapes)]
        # The clipped ones go to one buffer, as an optimizer over a flat state takes them.
        p["flat"] = torch.empty(sum(a * b for a, b in shapes), dtype=t, device=DEV)
        parts = p["flat"].split([a * b for a, b in shapes])
        p["outs"] = [v.view(s) for v, s in zip(parts, shapes)]
    return p


# ---- the operators' plain forms -------------------------------------------------


def _weights(c, w):
    """The values of packed weights, as ops.dequantize defines them: the product and the sum
    each rounded to bf16; float32."""
    words, s, b = w
    bits, group = c["bits"], c["group"]
    at = torch.arange(0, 32, bits, device=DEV, dtype=torch.int32)
    q = ((words.unsqueeze(-1) >> at) & ((1 << bits) - 1)).reshape(*s.shape, group).float()
    v = (q * s.float().unsqueeze(-1)).bfloat16().float() + b.float().unsqueeze(-1)
    return v.bfloat16().float().reshape(*words.shape[:-1], -1)


def _plain_top(c, h, W, logits, n):
    """The n largest logits of each row and their tokens: candidates by the 32-bit logits, ordered
    by 64-bit ones, equal ones to the lower token."""
    m = min(n + 16, c["V"])
    cand = logits.topk(m, dim=-1).indices.sort(dim=-1).values
    exact = torch.empty(cand.shape, dtype=torch.float64, device=DEV)
    for r in range(0, c["M"], 128):
        rows = W[cand[r:r + 128]].double()
        exact[r:r + 128] = (rows * h[r:r + 128, None, :].double()).sum(-1) / c["T"]
    order = torch.sort(exact, dim=-1, descending=True, stable=True).indices[:, :n]
    return cand.gather(1, order), exact.gather(1, order)


def _plain_logp(c, p):
    W, h, T = _weights(c, p["w"]), p["h"].float(), c["T"]
    logits = (h @ W.T) / T
    best = logits.amax(-1, keepdim=True)
    low = logits - best
    e = low.exp()
    z = e.sum(-1, keepdim=True)
    lz = z.log()
    ids = p["ids"].long()
    there = ids >= 0
    at = ids.clamp(min=0)
    logp = torch.where(there, low.gather(1, at) - lz, torch.zeros_like(lz))
    prob = e / z
    entropy = lz[:, 0] - (prob * low).sum(-1)
    out = {"logp": logp, "entropy": entropy, "lse": best[:, 0] + lz[:, 0]}
    if c["top"]:
        top, value = _plain_top(c, h, W, logits, c["top"])
        out["top_ids"] = top.int()
        out["top_logp"] = (value - best.double() - lz.double()).float()
    if c["step"]:
        a = torch.where(there, p["da"], torch.zeros_like(p["da"]))
        d = (low - lz + entropy[:, None]) * p["dent"][:, None] + a.sum(-1, keepdim=True)
        d *= -prob
        d.scatter_add_(1, at, a)
        out["dh"] = ((d @ W) / T).bfloat16()
    return out


def _plain_lora(c, p):
    W, x, ad = _weights(c, p["w"]), p["x"].float(), p["adapters"]
    a, b, s = p["a"].float(), p["b"].float(), p["scales"]
    if not c["grad"]:
        y = x @ W.T
        for e in range(c["E"]):
            rows = (ad == e).nonzero()[:, 0]
            y[rows] += s[e] * ((x[rows] @ a[e].T) @ b[e].T)
        return y.bfloat16()
    dy = p["dy"].float()
    dx = dy @ W
    da, db = torch.zeros_like(a), torch.zeros_like(b)
    for e in range(c["E"]):
        rows = (ad == e).nonzero()[:, 0]
        t = x[rows] @ a[e].T
        dt = s[e] * (dy[rows] @ b[e])
        dx[rows] += dt @ a[e]
        da[e] = dt.T @ x[rows]
        db[e] = s[e] * (dy[rows].T @ t)
    return {"dx": dx.bfloat16(), "da": da, "db": db}


def _plain_clip(c, p):
    total = torch.zeros((), dtype=torch.float64, device=DEV)
    for g in p["grads"]:
        total += (g.double() * g.double()).sum()
    norm = total.sqrt()
    factor = (c["max_norm"] / norm).clamp(max=1.0).float()
    for g, out in zip(p["grads"], p["outs"]):
        out.copy_(g.float() * factor)
    return {"norm": norm.float(), "clipped": p["flat"]}


# ---- one pass -------------------------------------------------------------------


def _own(c, p):
    from fastmlx_amd import ops

    if c["kind"] == "logp":
        form = dict(temperature=c["T"], group_size=c["group"], bits=c["bits"])
        r = ops.head_logprobs(p["h"], *p["w"], p["ids"], top=c["top"], **form)
        out = dict(zip(("logp", "entropy", "lse", "top_ids", "top_logp"), r))
        if c["step"]:
            out["dh"] = ops.head_logprobs_grad(p["h"], *p["w"], p["ids"], *r[:3], p["da"],
                                               grad_entropy=p["dent"], **form)
        return out
    if c["kind"] == "lora":
        lora = (p["a"], p["b"], p["adapters"], p["scales"])
        if not c["grad"]:
            return ops.quantized_matmul_lora(p["x"], *p["w"], *lora, c["group"], c["bits"])
        r = ops.quantized_matmul_lora_grad(p["dy"], p["x"], *p["w"], *lora, c["group"], c["bits"])
        return dict(zip(("dx", "da", "db"), r))
    _, norm = ops.clip_grad_norm(p["grads"], c["max_norm"], outs=p["outs"])
    return {"norm": norm, "clipped": p["flat"]}


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return {"logp": _plain_logp, "lora": _plain_lora, "clip": _plain_clip}[c["kind"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------


def _weight_bytes(N, K, bits, group):
    return N * K * bits // 8 + N * (K // group) * 4


def work(case):
    c = case
    if c["kind"] == "logp":
        M, V, K = c["M"], c["V"], c["K"]
        b = _weight_bytes(V, K, c["bits"], c["group"]) + 2 * M * K + M * (8 + 8 * c["k"] + 8 * c["top"])
        f = 2 * M * V * K
        if c["step"]:
            b += 2 * M * K + M * (4 + 4 * c["k"])
            f *= 2
    elif c["kind"] == "lora":
        M, N, K, E, r = c["M"], c["N"], c["K"], c["E"], c["r"]
        used = min(M, E) * 2 * r * (K + N)  # the adapters that M rows name, at most
        b = _weight_bytes(N, K, c["bits"], c["group"]) + 2 * M * (K + N) + used
        f = 2 * M * N * K + 2 * M * r * (K + N)
        if c["grad"]:
            b += 2 * M * K + 4 * E * r * (K + N)
            f += 2 * M * r * (2 * K + N)
    else:
        n = sum(a * b for a, b in _clip_shapes(c))
        # A gradient is read for the norm and once more to be scaled.
        b = n * (2 if c["bf16"] else 4) * 3
        f = 3 * n
    return {"bytes": float(b), "flops": float(f)}


# ---- the same in 64 bits --------------------------------------------------------


def _exact_weights(c, words, s, b):
    """Packed weights as their definition has it, value by value of a word: float64."""
    bits = c["bits"]
    s = s.double().repeat_interleave(c["group"], -1)
    b = b.double().repeat_interleave(c["group"], -1)
    v = torch.empty_like(s)
    per = 32 // bits
    for i in range(per):
        q = (words.long() >> (bits * i)) % (1 << bits)
        v[..., i::per] = ((q * s[..., i::per]).bfloat16().double() + b[..., i::per]).bfloat16()
    return v


def _exact_logp(c, p):
    W = _exact_weights(c, *p["w"])
    logits = p["h"].double() @ W.T / c["T"]
    lse = torch.logsumexp(logits, -1)
    logp = logits - lse[:, None]
    ids = p["ids"].long()
    on = (ids >= 0).double()
    prob = logp.exp()
    entropy = torch.special.entr(prob).sum(-1)
    out = {"logp": on * logp.gather(1, ids.clamp(min=0)), "entropy": entropy, "lse": lse}
    if c["top"]:
        out["top_ids"] = None
        out["top_logp"] = logp.topk(c["top"], dim=-1).values
    if c["step"]:
        a = p["da"].double() * on
        d = torch.zeros_like(logp).scatter_add_(1, ids.clamp(min=0), a)
        d -= prob * a.sum(-1, keepdim=True)
        d -= prob * (logp + entropy[:, None]) * p["dent"].double()[:, None]
        out["dh"] = d @ W / c["T"]
    return out


def _exact_lora(c, p):
    W = _exact_weights(c, *p["w"])
    x, ad = p["x"].double(), p["adapters"].long()
    E, r, K, N = c["E"], c["r"], c["K"], c["N"]
    # Every adapter's weight beside W, over the rows that name it.
    dx = da = db = y = None
    if c["grad"]:
        dy = p["dy"].double()
        dx = dy @ W
        da = torch.zeros(E, r, K, dtype=torch.float64, device=DEV)
        db = torch.zeros(E, N, r, dtype=torch.float64, device=DEV)
    else:
        y = x @ W.T
    for e in set(ad.tolist()) - {-1}:
        on = (ad == e).double()[:, None]
        A, B, s = p["a"][e].double(), p["b"][e].double(), p["scales"][e].double()
        delta = s * (B @ A)
        if y is not None:
            y += (on * x) @ delta.T
            continue
        dx += (on * dy) @ delta
        dw = (on * dy).T @ x  # the gradient of the adapter's whole weight
        da[e] = s * (B.T @ dw)
        db[e] = s * (dw @ A.T)
    return y if y is not None else {"dx": dx, "da": da, "db": db}


def _exact_clip(c, p):
    norm = torch.sqrt(sum(torch.dot(g.double().flatten(), g.double().flatten()) for g in p["grads"]))
    factor = torch.clamp(c["max_norm"] / norm, max=1.0)
    return {"norm": norm, "clipped": torch.cat([g.double().flatten() * factor for g in p["grads"]])}


def exact(case, seed):
    if case["kind"] == "lora" and case["E"] > 16 and case["M"] > 512:
        return None  # a whole product in 64 bits for every adapter
    p = prepare(case, seed)
    return {"logp": _exact_logp, "lora": _exact_lora, "clip": _exact_clip}[case["kind"]](case, p)
