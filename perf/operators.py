"""The operators of training and scoring over quantized weights, for timing.

Four kinds of call, over the sizes, bit widths and group sizes they are used with:

* ``ce``      the cross entropy of a quantized vocabulary head, the loss alone (scoring text)
              or the loss and the gradient of the hidden states (a training step);
* ``distill`` the divergence from a teacher's top logits through the same head;
* ``rows``    a mixture-of-experts layer's token rows sorted by expert and summed back with
              the router's weights, forward and backward;
* ``grad``    the input gradient of a quantized product, of one matrix or of expert runs.

Weights follow the distributions of the repository's benchmark: 4-bit scales uniform in
[0.002, 0.02] with biases near -8 scale; 8-bit scales uniform in [1e-4, 2e-3] with biases
-128 scale.  The weights of every product are the bf16 values that ``ops.dequantize`` gives.
"""
import math

import torch

own = False

DEV = "cuda"
IGNORE = -100


def listed():
    return [
        # The log-likelihood of one token: the latency of a call that reads the head once.
        dict(name="ce_score_m1", kind="ce", M=1, V=32000, K=2048, bits=4, group=64, grad=False),
        # Scoring a prompt chunk of odd length over a large vocabulary, groups of 128.
        dict(name="ce_score_m509", kind="ce", M=509, V=151936, K=2048, bits=4, group=128,
             grad=False),
        # A small fine-tuning batch on an 8-bit checkpoint with an odd vocabulary.
        dict(name="ce_step_m37", kind="ce", M=37, V=50257, K=1024, bits=8, group=64, grad=True),
        # A full training batch through an 8B-sized head.
        dict(name="ce_step_m2048", kind="ce", M=2048, V=128256, K=4096, bits=4, group=64,
             grad=True),
        # Distillation of a short answer, few teacher entries, groups of 32.
        dict(name="distill_m16_k20", kind="distill", M=16, V=32000, K=2560, k=20, bits=4, group=32,
             grad=True),
        # Distillation of a batch of sequences with the most teacher entries.
        dict(name="distill_m1000_k64", kind="distill", M=1000, V=128256, K=4096, k=64, bits=4,
             group=64, grad=True),
        # The rows of one short sequence through a many-expert layer: launch latency.
        dict(name="rows_t16", kind="rows", T=16, E=512, k=10, D=2048, wbf16=True),
        # An odd batch with float weights.
        dict(name="rows_t1021", kind="rows", T=1021, E=64, k=6, D=2048, wbf16=False),
        # A training batch through a wide expert layer with skewed expert popularity.
        dict(name="rows_t8192", kind="rows", T=8192, E=256, k=8, D=7168, wbf16=True),
        # The gradient of a small batch through an attention projection.
        dict(name="grad_m13", kind="grad", M=13, N=4096, K=4096, E=0, bits=4, group=64),
        # A training batch through a gate projection.
        dict(name="grad_m2048", kind="grad", M=2048, N=14336, K=4096, E=0, bits=4, group=64),
        # A training batch through the up projections of a mixture of experts, 8 bits.
        dict(name="grad_experts_8bit", kind="grad", M=8192, N=512, K=2048, E=64, bits=8, group=64),
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
        kind = rng.choice(("ce", "ce", "distill", "rows", "grad", "grad"))
        bits = rng.choice((4, 4, 8))
        group = rng.choice((64, 64, 32, 128))
        # Model widths are multiples of 256 almost always, of the group in any case.
        K = _width(rng, 512, 8192, rng.choice((256, 256, 128)))
        if kind in ("ce", "distill"):
            c = dict(kind=kind, M=_logint(rng, 1, 2048), V=_logint(rng, 1000, 152000), K=K,
                     bits=bits, group=group, grad=rng.random() < 0.6)
            if kind == "distill":
                c["k"] = _logint(rng, 1, 64)
                c["grad"] = True
        elif kind == "rows":
            E = rng.choice((8, 64, 128, 256, 512))
            c = dict(kind=kind, T=_logint(rng, 1, 8192), E=E, k=rng.randint(1, min(E, 10)),
                     D=_width(rng, 512, 7168, rng.choice((256, 64))), wbf16=rng.random() < 0.5)
        elif rng.random() < 0.5:
            c = dict(kind=kind, M=_logint(rng, 1, 4096), N=_logint(rng, 256, 28672), K=K, E=0,
                     bits=bits, group=group)
        else:
            c = dict(kind=kind, M=_logint(rng, 1, 16384), N=_width(rng, 128, 2048, 64), K=K,
                     E=rng.choice((4, 16, 64, 128)), bits=bits, group=group)
        if _seconds(c) <= most:
            return c


# ---- inputs -------------------------------------------------------------------


def _packed(gen, lead, K, bits, group):
    """A random quantized weight [*lead, K]: (words, scales, biases)."""
    w = torch.randint(-2**31, 2**31, (*lead, K * bits // 32), dtype=torch.int32, device=DEV,
                      generator=gen)
    lo, hi, mid = (0.002, 0.02, 8) if bits == 4 else (1e-4, 2e-3, 128)
    s = torch.empty(*lead, K // group, device=DEV).uniform_(lo, hi, generator=gen).bfloat16()
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


def _hidden(c, gen, w, likely):
    """Hidden states that lean towards their likely next token by as much as a trained
    model's do: from not at all to a clear favourite."""
    M, K = c["M"], c["K"]
    rows = _weights(c, tuple(t[likely] for t in w))
    return (_normal(gen, M, K) + rows * 1.5 * _uniform(gen, M, 1)).bfloat16()


def _popular(gen, T, E, k):
    """k distinct experts a token, their popularity as Zipf(1.1) over shuffled ids: the top
    k of log-popularity plus Gumbel noise."""
    rank = torch.randperm(E, device=DEV, generator=gen).float() + 1
    u = _uniform(gen, T, E).clamp_(1e-6, 1 - 1e-6)
    return (-1.1 * rank.log() - (-u.log()).log()).topk(k, dim=-1).indices.int()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(seed)
    p = {"case": dict(c)}
    if c["kind"] in ("ce", "distill"):
        M, V = c["M"], c["V"]
        p["w"] = _packed(gen, (V,), c["K"], c["bits"], c["group"])
        p["scale"] = _uniform(gen, M) / M  # the weight of each token in the mean
        if c["kind"] == "ce":
            likely = _ints(gen, V, M)
            # One token in twenty is padding.
            p["targets"] = torch.where(_uniform(gen, M) < 0.05, torch.full_like(likely, IGNORE),
                                       likely).int()
        else:
            # The ids of a row differ: a start, and a step that does not come round.
            k = c["k"]
            at = torch.arange(k, device=DEV)
            ids = (_ints(gen, V, M, 1) + at * (1 + _ints(gen, V // k, M, 1))) % V
            likely = ids[:, 0]
            p["ids"] = ids.int()
            p["teacher"] = (4 * _normal(gen, M, k)).sort(dim=-1, descending=True).values.bfloat16()
        p["h"] = _hidden(c, gen, p["w"], likely)
    elif c["kind"] == "rows":
        T, k, D = c["T"], c["k"], c["D"]
        p["x"] = _normal(gen, T, D).bfloat16()
        p["inds"] = _popular(gen, T, c["E"], k)
        w = torch.softmax(_normal(gen, T, k), -1)
        p["weights"] = w.bfloat16() if c["wbf16"] else w
        # What the experts return and what comes back from the layers above.
        p["y"] = _normal(gen, T * k, D).bfloat16()
        p["dout"] = (_normal(gen, T, D) / D).bfloat16()
        p["dxs"] = (_normal(gen, T * k, D) / D).bfloat16()
    else:
        M, E = c["M"], c["E"]
        p["dy"] = (_normal(gen, M, c["N"]) / M).bfloat16()
        p["w"] = _packed(gen, (E, c["N"]) if E else (c["N"],), c["K"], c["bits"], c["group"])
        if E:
            e = _popular(gen, M, E, 1).flatten().long()
            count = torch.bincount(e, minlength=E)
            p["offsets"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).int()
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


def _plain_ce(c, p):
    W, h = _weights(c, p["w"]), p["h"].float()
    logits = h @ W.T
    top = logits.amax(-1, keepdim=True)
    lse = (logits - top).exp().sum(-1).log() + top[:, 0]
    y = p["targets"].long()
    kept = y != IGNORE
    at = torch.where(kept, y, torch.zeros_like(y))[:, None]
    loss = torch.where(kept, lse - logits.gather(1, at)[:, 0], torch.zeros_like(lse))
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        d = (logits - lse[:, None]).exp()
        d.scatter_add_(1, at, torch.full_like(lse, -1.0)[:, None])
        d *= torch.where(kept, p["scale"], torch.zeros_like(lse))[:, None]
        out["dh"] = (d @ W).bfloat16()
    return out


def _temperature(c):
    return 2.0


def _plain_distill(c, p):
    W, h, T = _weights(c, p["w"]), p["h"].float(), _temperature(c)
    logits = (h @ W.T) / T
    top = logits.amax(-1, keepdim=True)
    lse = (logits - top).exp().sum(-1).log() + top[:, 0]
    ids = p["ids"].long()
    t = p["teacher"].float() / T
    t = t - t.amax(-1, keepdim=True)
    logq = t - t.exp().sum(-1, keepdim=True).log()
    q = logq.exp()
    loss = T * T * (q * (logq - logits.gather(1, ids) + lse[:, None])).sum(-1)
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        d = (logits - lse[:, None]).exp()
        d.scatter_add_(1, ids, -q)
        d *= T * p["scale"][:, None]
        out["dh"] = (d @ W).bfloat16()
    return out


def _plain_rows(c, p):
    T, k = c["T"], c["k"]
    flat = p["inds"].flatten().long()
    order = torch.argsort(flat, stable=True)
    pos = torch.empty_like(order)
    pos[order] = torch.arange(T * k, device=DEV)
    count = torch.zeros(c["E"], dtype=torch.long, device=DEV)
    count.index_add_(0, flat, torch.ones_like(flat))
    offsets = torch.cat([count.new_zeros(1), count.cumsum(0)])
    xs = p["x"][order // k]
    w = p["weights"].float()
    y = p["y"].float()[pos].view(T, k, -1)
    out = (y * w[..., None]).sum(1).bfloat16()
    dout = p["dout"].float()
    dy = torch.empty_like(p["y"])
    dy[pos] = (dout[:, None, :] * w[..., None]).bfloat16().view(T * k, -1)
    dw = (y * dout[:, None, :]).sum(-1).to(p["weights"].dtype)
    dx = p["dxs"].float()[pos].view(T, k, -1).sum(1).bfloat16()
    return {"xs": xs, "order": order.int(), "pos": pos.int().view(T, k), "offsets": offsets.int(),
            "out": out, "dy": dy, "dweights": dw, "dx": dx}


def _plain_grad(c, p):
    dy = p["dy"].float()
    if not c["E"]:
        return (dy @ _weights(c, p["w"])).bfloat16()
    W = _weights(c, p["w"])
    ends = p["offsets"].tolist()
    runs = dy.split([b - a for a, b in zip(ends, ends[1:])])
    return torch.cat([run @ mat for run, mat in zip(runs, W)]).bfloat16()


# ---- one pass -------------------------------------------------------------------


def _own(c, p):
    from fastmlx_amd import ops

    if c["kind"] == "ce":
        r = ops.head_cross_entropy(p["h"], *p["w"], p["targets"], ignore_index=IGNORE,
                                   grad=c["grad"], grad_loss=p["scale"] if c["grad"] else None,
                                   group_size=c["group"], bits=c["bits"])
        return dict(zip(("loss", "lse", "dh"), r))
    if c["kind"] == "distill":
        r = ops.head_distill(p["h"], *p["w"], p["ids"], p["teacher"], temperature=_temperature(c),
                             grad=c["grad"], grad_loss=p["scale"] if c["grad"] else None,
                             group_size=c["group"], bits=c["bits"])
        return dict(zip(("loss", "lse", "dh"), r))
    if c["kind"] == "rows":
        xs, order, pos, offsets = ops.moe_sort(p["x"], p["inds"], c["E"])
        out = ops.moe_unsort(p["y"], pos, p["weights"])
        dy, dw = ops.moe_unsort_grad(p["dout"], p["y"], pos, p["weights"])
        dx = ops.moe_sort_grad(p["dxs"], pos)
        return {"xs": xs, "order": order, "pos": pos, "offsets": offsets, "out": out, "dy": dy,
                "dweights": dw, "dx": dx}
    if c["E"]:
        return ops.gather_qmm_grad(p["dy"], *p["w"], p["offsets"], c["group"], c["bits"])
    return ops.quantized_matmul_grad(p["dy"], *p["w"], c["group"], c["bits"])


def run(state):
    c = state["case"]
    if own:
        return _own(c, state)
    return {"ce": _plain_ce, "distill": _plain_distill, "rows": _plain_rows,
            "grad": _plain_grad}[c["kind"]](c, state)


# ---- what a pass cannot do without ----------------------------------------------


def _weight_bytes(N, K, bits, group):
    return N * K * bits // 8 + N * (K // group) * 4


def work(case):
    c = case
    if c["kind"] in ("ce", "distill"):
        M, V, K = c["M"], c["V"], c["K"]
        products = 2 if c["grad"] else 1
        per_row = 4 if c["kind"] == "ce" else 6 * c["k"]
        b = _weight_bytes(V, K, c["bits"], c["group"]) + products * 2 * M * K + M * (12 + per_row)
        f = products * 2 * M * V * K
    elif c["kind"] == "rows":
        T, k, D = c["T"], c["k"], c["D"]
        S = T * k
        # x, y, dout and dxs read once; xs, out, dy and dx written once.
        b = 2 * D * (4 * T + 4 * S) + S * (12 + 2 * (2 if c["wbf16"] else 4)) + 4 * c["E"]
        f = 6 * S * D
    else:
        M, N, K = c["M"], c["N"], c["K"]
        matrices = 1
        if c["E"]:
            # Distinct experts under Zipf(1.1), independent draws.
            pop = [r ** -1.1 for r in range(1, c["E"] + 1)]
            matrices = sum(1 - (1 - q / sum(pop)) ** M for q in pop)
        b = matrices * _weight_bytes(N, K, c["bits"], c["group"]) + 2 * M * (N + K)
        f = 2 * M * N * K
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


def _exact_head(c, p):
    W = _exact_weights(c, *p["w"])
    T = _temperature(c) if c["kind"] == "distill" else 1.0
    logp = torch.log_softmax(p["h"].double() @ W.T / T, -1)
    M = c["M"]
    q = torch.zeros_like(logp)
    if c["kind"] == "ce":
        keep = (p["targets"] != IGNORE).double()
        ids = p["targets"].long().clamp(min=0)[:, None]
        wanted = keep[:, None]
    else:
        keep = torch.ones(M, dtype=torch.float64, device=DEV)
        ids = p["ids"].long()
        wanted = torch.softmax(p["teacher"].double() / T, -1)
    loss = T * T * (torch.special.entr(wanted).neg() - wanted * logp.gather(1, ids)).sum(-1)
    # The sum of exponentials again, from the likeliest token's logit.
    v = logp.argmax(-1)
    best = (p["h"].double() * W[v]).sum(-1) / T
    lse = best - logp.gather(1, v[:, None])[:, 0]
    out = {"loss": loss, "lse": lse}
    if c["grad"]:
        q.scatter_add_(1, ids, wanted)
        d = (logp.exp() * keep[:, None] - q) * (T * p["scale"].double())[:, None]
        out["dh"] = d @ W
    return out


def _exact_rows(c, p):
    T, k, D = c["T"], c["k"], c["D"]
    order = sorted(range(T * k), key=p["inds"].flatten().tolist().__getitem__)
    order = torch.tensor(order, device=DEV)
    token = order // k
    w = p["weights"].double().flatten()[order][:, None]
    y, dout = p["y"].double(), p["dout"].double()
    zero = torch.zeros(T, D, dtype=torch.float64, device=DEV)
    dw = torch.empty(T * k, dtype=torch.float64, device=DEV)
    dw[order] = (y * dout[token]).sum(-1)
    return {"xs": p["x"].double()[token], "order": None, "pos": None, "offsets": None,
            "out": zero.index_add(0, token, w * y), "dy": w * dout[token],
            "dweights": dw.view(T, k), "dx": zero.index_add(0, token, p["dxs"].double())}


def _exact_grad(c, p):
    dy = p["dy"].double()
    if not c["E"]:
        return dy @ _exact_weights(c, *p["w"])
    ends = p["offsets"].tolist()
    parts = [dy[lo:hi] @ _exact_weights(c, *(t[e] for t in p["w"]))
             for e, (lo, hi) in enumerate(zip(ends, ends[1:]))]
    return torch.cat(parts)


def exact(case, seed):
    p = prepare(case, seed)
    return {"ce": _exact_head, "distill": _exact_head, "rows": _exact_rows,
            "grad": _exact_grad}[case["kind"]](case, p)
