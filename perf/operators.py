"""The operators of a decode step whose weights are picked per row, as measurable cases.

* `route`: the router of a mixture-of-experts layer, from its logits to the chosen experts and their weights.
* `experts`: the layer's experts for a few tokens: two products with a gated activation between them, summed over a token's experts.
* `lora`: low-rank adapters of many requests at once, added to what a shared projection has made.

`run` calls `triton_shared_amd.ops` where `own` is set, and else computes the same from elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ITEM = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}


def listed():
    return [
        # one token of an interactive session, 8 of 128 experts: latency is what counts
        dict(name="route_one", kind="route", tokens=1, experts=128, top=8, dtype="bf16", scoring="softmax", bias=False),
        # a prompt's tokens; scores by sigmoid, chosen with a balancing bias
        dict(name="route_prompt", kind="route", tokens=16384, experts=256, top=8, dtype="fp32", scoring="sigmoid", bias=True),
        # one token through 8 small experts of 128
        dict(name="experts_one", kind="experts", tokens=1, experts=128, top=8, hidden=2048, inner=768, dtype="bf16", weights="bf16", order="in", activation="silu", gated=True),
        # four sessions on eight large experts, weights as the tiled product keeps them (outputs contiguous)
        dict(name="experts_wide", kind="experts", tokens=4, experts=8, top=2, hidden=4096, inner=8192, dtype="fp16", weights="fp16", order="out", activation="silu", gated=True),
        # sessions in a batch, int8 weights with a scale per output column
        dict(name="experts_int8", kind="experts", tokens=24, experts=16, top=2, hidden=4096, inner=4096, dtype="fp16", weights="int8", order="out", activation="silu", gated=True),
        # an odd number of tokens, sizes in no tile's multiples, no gate
        dict(name="experts_odd", kind="experts", tokens=13, experts=10, top=3, hidden=1432, inner=2004, dtype="bf16", weights="bf16", order="out", activation="gelu_tanh", gated=False),
        # a full decode batch: nearly every expert is picked, by a few tokens each
        dict(name="experts_batch", kind="experts", tokens=256, experts=64, top=6, hidden=4096, inner=1536, dtype="bf16", weights="bf16", order="in", activation="silu", gated=True),
        # one session with an adapter
        dict(name="lora_one", kind="lora", tokens=1, inputs=4096, outputs=4096, rank=16, adapters=8, runs=1, dtype="bf16", plain=0.0),
        # a decode batch, nearly every session with an adapter of its own
        dict(name="lora_decode", kind="lora", tokens=64, inputs=4096, outputs=8192, rank=16, adapters=64, runs=1, dtype="fp16", plain=0.1),
        # odd sizes, ranks below a tile, sessions without an adapter among them
        dict(name="lora_odd", kind="lora", tokens=37, inputs=1333, outputs=2050, rank=12, adapters=5, runs=1, dtype="bf16", plain=0.4),
        # prompts of several requests one after another
        dict(name="lora_prompts", kind="lora", tokens=8192, inputs=4096, outputs=4096, rank=64, adapters=16, runs=700, dtype="bf16", plain=0.1),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of these ranges; sizes over their logarithm, odd ones among them."""
    most = max((work(c)["bytes"] for c in listed()))
    while True:
        kind = rng.choice(["route", "experts", "experts", "lora"])
        if kind == "route":
            experts = _log(rng, 8, 512)
            c = dict(kind=kind, tokens=_log(rng, 1, 16384), experts=experts, top=rng.randint(1, min(10, experts)), dtype=rng.choice(["fp32", "bf16", "fp16"]),
                     scoring=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5)
        elif kind == "experts":
            experts = _log(rng, 4, 128)
            step = rng.choice([1, 8, 64])
            dtype = rng.choice(["bf16", "fp16"])
            c = dict(kind=kind, tokens=_log(rng, 1, 256), experts=experts, top=rng.randint(1, min(8, experts)), hidden=-(-_log(rng, 512, 6144) // step) * step,
                     inner=-(-_log(rng, 256, 8192) // step) * step, dtype=dtype, weights=rng.choice([dtype, dtype, "int8"]), order=rng.choice(["in", "out"]),
                     activation=rng.choice(["silu", "gelu_tanh", "relu"]), gated=rng.random() < 0.75)
            # (the whole table of weights, as the plain form widens it)
            if experts * c["hidden"] * c["inner"] * (3 if c["gated"] else 2) > 64 * 3 * 4096 * 1536:
                continue
        else:
            step = rng.choice([1, 8, 64])
            tokens = _log(rng, 1, 8192)
            c = dict(kind=kind, tokens=tokens, inputs=-(-_log(rng, 512, 8192) // step) * step, outputs=-(-_log(rng, 512, 8192) // step) * step,
                     rank=rng.choice([4, 8, 16, 16, 24, 32, 64, 128]), adapters=_log(rng, 1, 64), runs=1 if tokens <= 128 else tokens // rng.randint(2, 16),
                     dtype=rng.choice(["bf16", "fp16"]), plain=rng.choice([0.0, 0.1, 0.5]))
            if tokens * c["rank"] * c["adapters"] > 8192 * 64 * 16:
                continue
        if work(c)["bytes"] <= most:
            return c


def _distinct(choices, share, times):
    """How many of `choices` are expected to be picked at least once, each with probability `share` at each of `times`."""
    return choices * (1.0 - (1.0 - share) ** times)


def work(case):
    if case["kind"] == "route":
        n = case["tokens"] * case["experts"]
        return {"bytes": n * ITEM[case["dtype"]] + 8 * case["tokens"] * case["top"] + (4 * case["experts"] if case["bias"] else 0), "flops": 4 * n}
    if case["kind"] == "experts":
        t, k, e, h, i = (case[x] for x in ("tokens", "top", "experts", "hidden", "inner"))
        cols = (2 if case["gated"] else 1) * i
        scales = 4 * (cols + h) if case["weights"] == "int8" else 0
        return {"bytes": _distinct(e, k / e, t) * ((cols * h + i * h) * ITEM[case["weights"]] + scales) + 2 * t * h * ITEM[case["dtype"]] + 8 * t * k,
                "flops": 2 * t * k * (cols * h + i * h)}
    t, kin, n, r = (case[x] for x in ("tokens", "inputs", "outputs", "rank"))
    rows = t * (1.0 - case["plain"])
    used = _distinct(case["adapters"], 1.0 / case["adapters"], rows / case["runs"])
    return {"bytes": 2 * (rows * kin + 2 * t * n + used * r * (kin + n)) + 4 * t, "flops": 2 * rows * r * (kin + n)}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        t = torch.empty(*shape, dtype=dtype, device="cuda")
        return t.normal_(0.0, scale, generator=g)

    s = dict(case)
    dt = DTYPES[case["dtype"]]
    if case["kind"] == "route":
        t, e = case["tokens"], case["experts"]
        s.update(logits=normal(t, e, scale=2.0, dtype=dt), bias=normal(e, scale=0.05) if case["bias"] else None)
    elif case["kind"] == "experts":
        t, k, e, h, i = (case[x] for x in ("tokens", "top", "experts", "hidden", "inner"))
        cols = (2 if case["gated"] else 1) * i

        def table(inputs, outputs):
            shape = (e, inputs, outputs) if case["order"] == "out" else (e, outputs, inputs)
            if case["weights"] == "int8":
                w = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8, device="cuda")
                scales = torch.empty(e, outputs, device="cuda").uniform_(0.8, 1.2, generator=g) * (inputs ** -0.5 / 73.0)
            else:
                w, scales = normal(*shape, scale=inputs ** -0.5, dtype=DTYPES[case["weights"]]), None
            return (w if case["order"] == "out" else w.transpose(1, 2)), scales

        w_up, s_up = table(h, cols)
        w_down, s_down = table(i, h)
        chosen = torch.rand(t, e, generator=g, device="cuda").topk(k, dim=1)
        shares = torch.softmax(chosen.values * 3.0, dim=1)
        s.update(x=normal(t, h, dtype=dt), ids=chosen.indices.int(), shares=shares, w_up=w_up, w_down=w_down, s_up=s_up, s_down=s_down)
    else:
        t, kin, n, r, count = (case[x] for x in ("tokens", "inputs", "outputs", "rank", "adapters"))
        # runs of rows of one request, each with an adapter or without
        requests = -(-t // case["runs"])
        ids = torch.randint(0, count, (requests,), generator=g, dtype=torch.int32, device="cuda")
        ids = torch.where(torch.rand(requests, generator=g, device="cuda") < case["plain"], torch.full_like(ids, -1), ids)
        s.update(base=normal(t, n, dtype=dt), x=normal(t, kin, dtype=dt), a=normal(count, r, kin, scale=kin ** -0.5, dtype=dt), b=normal(count, n, r, scale=r ** -0.5, dtype=dt),
                 ids=ids.repeat_interleave(case["runs"])[:t].contiguous(), scales=torch.empty(count, device="cuda").uniform_(0.5, 2.0, generator=g))
    return s


def _route_plain(s):
    # in 64 bits: a score next to the last chosen one decides which expert it is
    logits = s["logits"].double()
    scores = torch.sigmoid(logits) if s["scoring"] == "sigmoid" else torch.softmax(logits, dim=1)
    by = scores + s["bias"].double() if s["bias"] is not None else logits
    ids = torch.sort(by, dim=1, descending=True, stable=True).indices[:, :s["top"]]
    chosen = torch.gather(scores, 1, ids)
    return ids.int(), (chosen / chosen.sum(dim=1, keepdim=True)).float()


def _activate(name, v):
    if name == "silu":
        return v / (1.0 + torch.exp(-v))
    if name == "relu":
        return torch.clamp(v, min=0.0)
    return 0.5 * v * (1.0 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _experts_plain(s):
    x, ids, shares = s["x"].float(), s["ids"].long(), s["shares"]
    t, k = ids.shape
    w_up, w_down, s_up, s_down = s["w_up"], s["w_down"], s["s_up"], s["s_down"]
    few = t * k < s["experts"]
    if few:  # the picked experts' weights, one product per token and expert
        flat = ids.reshape(-1)
        w_up, w_down = w_up[flat], w_down[flat]
        s_up, s_down = (None, None) if s_up is None else (s_up[flat], s_down[flat])
        rows = x.repeat_interleave(k, dim=0)[:, None, :]
    else:  # every token through every expert, weighted by what it picked
        rows = x[None].expand(w_up.shape[0], -1, -1)
    v = torch.bmm(rows, w_up.float().contiguous())
    if s_up is not None:
        v = v * s_up[:, None, :]
    i = s["inner"]
    v = _activate(s["activation"], v[..., :i]) * v[..., i:] if s["gated"] else _activate(s["activation"], v)
    v = torch.bmm(v, w_down.float().contiguous())
    if s_down is not None:
        v = v * s_down[:, None, :]
    if few:
        y = (v.reshape(t, k, -1) * shares[:, :, None]).sum(dim=1)
    else:
        picked = torch.zeros(t, w_up.shape[0], device=x.device).scatter_add_(1, ids, shares)
        y = (v * picked.t()[:, :, None]).sum(dim=0)
    return y.to(s["x"].dtype)


def _lora_plain(s):
    a, b, x, ids = s["a"].float(), s["b"].float(), s["x"].float(), s["ids"]
    count, r, kin = a.shape
    v = (x @ a.reshape(count * r, kin).t()).reshape(-1, count, r)  # every adapter's, then the row's own
    mine = torch.where(ids[:, None] == torch.arange(count, device=ids.device)[None], s["scales"][None], 0.0)
    v = (v * mine[:, :, None]).reshape(-1, count * r)
    return (s["base"].float() + v @ b.transpose(1, 2).reshape(count * r, -1)).to(s["base"].dtype)


def run(s):
    """One pass through an operator, and its outputs."""
    if s["kind"] == "route":
        if own:
            from triton_shared_amd import ops
            ids, weights = ops.moe_route(s["logits"], s["top"], scoring=s["scoring"], bias=s["bias"])
        else:
            ids, weights = _route_plain(s)
        return {"ids": ids, "weights": weights}
    if s["kind"] == "experts":
        if own:
            from triton_shared_amd import ops
            return ops.moe_experts(s["x"], s["ids"], s["shares"], s["w_up"], s["w_down"], s_up=s["s_up"], s_down=s["s_down"], activation=s["activation"], gated=s["gated"])
        return _experts_plain(s)
    if own:
        from triton_shared_amd import ops
        return ops.lora_add(s["base"], s["x"], s["a"], s["b"], s["ids"], scales=s["scales"])
    return _lora_plain(s)


def exact(case, seed):
    """The same outputs from the definitions in 64 bits, a row or an expert at a time."""
    s = prepare(case, seed)
    if case["kind"] == "route":
        logits = s["logits"].double().cpu().numpy()
        if case["scoring"] == "sigmoid":
            scores = 1.0 / (1.0 + np.exp(-logits))
        else:
            scores = np.exp(logits - logits.max(axis=1, keepdims=True))
            scores /= scores.sum(axis=1, keepdims=True)
        by = scores + s["bias"].double().cpu().numpy() if case["bias"] else logits
        ids = np.argsort(-by, axis=1, kind="stable")[:, :case["top"]]
        got = np.take_along_axis(scores, ids, axis=1)
        return {"ids": ids.astype(np.int32), "weights": got / got.sum(axis=1, keepdims=True)}
    if case["kind"] == "experts":
        x, i = s["x"].double(), case["inner"]
        y = torch.zeros(case["tokens"], case["hidden"], dtype=torch.float64, device="cuda")
        for e in range(case["experts"]):
            rows, slots = torch.nonzero(s["ids"] == e, as_tuple=True)
            if not len(rows):
                continue
            v = x[rows] @ s["w_up"][e].double()
            v = v if s["s_up"] is None else v * s["s_up"][e].double()
            gate = v[:, :i] if case["gated"] else v
            if case["activation"] == "silu":
                act = gate * torch.special.expit(gate)
            elif case["activation"] == "relu":
                act = torch.where(gate > 0, gate, torch.zeros_like(gate))
            else:
                act = gate * torch.special.expit(2.0 * math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate ** 3))
            v = (act * v[:, i:] if case["gated"] else act) @ s["w_down"][e].double()
            v = v if s["s_down"] is None else v * s["s_down"][e].double()
            y.index_add_(0, rows, v * s["shares"][rows, slots].double()[:, None])
        return y
    y = s["base"].double()
    for n in range(case["adapters"]):
        rows = torch.nonzero(s["ids"] == n)[:, 0]
        if len(rows):
            y[rows] += s["scales"][n].double() * ((s["x"][rows].double() @ s["a"][n].double().t()) @ s["b"][n].double().t())
    return y
