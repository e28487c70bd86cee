"""The attention part of a decode step over a cache held in 4 bits, as measurable cases.

* `slots`: block tables and slot maps of a batch, built on the GPU from its requests' lengths and a stack of free pages.
* `rope`: norms of queries and keys for each head, and the rotation by position, in one pass over both.
* `cache`: keys and values put into a paged cache of 4 bits, and read back as the values that it then holds.
* `attend`: attention over that cache: single tokens, a few tokens, prompts behind what is cached already.

`run` calls `triton_shared_amd.ops` where `own` is set, and else computes the same from elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a decode step of 64 requests: a token each, a page more for some
        dict(name="slots_step", kind="slots", requests=64, low=1, high=8192, fresh="one", most=1, page=16, spare=0),
        # prompts of a full batch, among them requests that decode; rows padded to what a graph was captured for
        dict(name="slots_prompts", kind="slots", requests=211, low=1, high=6000, fresh="some", most=160, page=64, spare=100),
        # one token of an interactive session: latency is what counts
        dict(name="rope_one", kind="rope", tokens=1, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16", interleaved=False, norm=True),
        # a prompt's tokens
        dict(name="rope_prompt", kind="rope", tokens=8192, heads=32, kv_heads=8, dim=128, rotary=128, dtype="bf16", interleaved=False, norm=True),
        # an odd number of tokens and heads, half of each head rotated, in neighbouring pairs
        dict(name="rope_odd", kind="rope", tokens=617, heads=15, kv_heads=5, dim=80, rotary=40, dtype="fp16", interleaved=True, norm=True),
        # a decode batch's keys and values
        dict(name="cache_step", kind="cache", tokens=64, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a prompt's
        dict(name="cache_prompt", kind="cache", tokens=16384, kv_heads=8, dim=128, page=64, dtype="fp16"),
        # one session
        dict(name="attend_one", kind="attend", requests=1, low=4000, high=4000, fresh=1, heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16"),
        # a decode batch of ragged lengths
        dict(name="attend_decode", kind="attend", requests=64, low=100, high=8192, fresh=1, heads=32, kv_heads=8, dim=128, page=16, window=0, dtype="bf16"),
        # two long documents
        dict(name="attend_long", kind="attend", requests=2, low=110000, high=131072, fresh=1, heads=64, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
        # drafted tokens of an odd number of requests, some with nothing cached before; five queries a key, a window
        dict(name="attend_odd", kind="attend", requests=13, low=5, high=3000, fresh=5, heads=15, kv_heads=3, dim=96, page=32, window=1000, dtype="fp16"),
        # a piece of a prompt behind what is cached already
        dict(name="attend_prompt", kind="attend", requests=4, low=2048, high=5000, fresh=1024, heads=32, kv_heads=8, dim=128, page=64, window=0, dtype="bf16"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of these ranges; sizes over their logarithm, odd ones among them."""
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["kind"], {"bytes": 0, "flops": 0})
        for x in w:
            m[x] = max(m[x], w[x])
    while True:
        kind = rng.choice(["slots", "rope", "cache", "attend", "attend"])
        dtype = rng.choice(["bf16", "fp16"])
        if kind == "slots":
            c = dict(kind=kind, requests=_log(rng, 1, 512), low=1, high=_log(rng, 8, 8192), fresh=rng.choice(["one", "some"]), most=_log(rng, 2, 512), page=rng.choice([16, 32, 48, 64, 128]),
                     spare=rng.choice([0, 0, 7, 100]))
        elif kind == "rope":
            kv_heads, dim = rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 80, 96, 128, 128, 192, 256])
            c = dict(kind=kind, tokens=_log(rng, 1, 8192), heads=kv_heads * rng.randint(1, 8), kv_heads=kv_heads, dim=dim, rotary=dim // rng.choice([1, 1, 2]), dtype=dtype,
                     interleaved=rng.random() < 0.4, norm=rng.random() < 0.8)
        elif kind == "cache":
            c = dict(kind=kind, tokens=_log(rng, 1, 16384), kv_heads=rng.choice([1, 2, 3, 4, 8]), dim=rng.choice([64, 96, 128, 128, 192, 256]), page=rng.choice([16, 32, 48, 64, 128]), dtype=dtype)
        else:
            kv_heads, high = rng.choice([1, 2, 3, 4, 8]), _log(rng, 16, 131072)
            c = dict(kind=kind, requests=_log(rng, 1, 64), low=max(1, high // rng.choice([1, 2, 16, 100])), high=high, fresh=rng.choice([1, 1, 1, rng.randint(2, 8), _log(rng, 16, 1024)]),
                     heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 8, 16]), kv_heads=kv_heads, dim=rng.choice([64, 96, 128, 128, 192, 256]), page=rng.choice([16, 32, 48, 64, 128]),
                     window=rng.choice([0, 0, 0, _log(rng, 64, 4096)]), dtype=dtype)
        if all(work(c)[x] <= most[kind][x] for x in most[kind]):
            return c


def _spread(i, low, high):
    """The i'th of many numbers of [low, high] that are dense over their logarithm there."""
    at = (i * 0.6180339887498949 + 0.37) % 1.0
    return min(high, max(low, int(round(low * (high / low) ** at))))


def _lengths(case):
    """(tokens in the cache after the step, how many of them are new) of each request."""
    many = range(case["requests"])
    lengths = [_spread(i, case["low"], case["high"]) for i in many]
    if case["kind"] == "attend":
        lengths = [max(n, case["fresh"]) if i != 1 else min(n, case["fresh"]) for i, n in enumerate(lengths)]  # (one request begins here)
        return lengths, [min(n, case["fresh"]) for n in lengths]
    fresh = [1 if case["fresh"] == "one" or i % 3 else _spread(i * 7 + 1, 1, case["most"]) for i in many]
    return lengths, [min(n, f) for n, f in zip(lengths, fresh)]


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    if case["kind"] == "slots":
        lengths, fresh = _lengths(case)
        taken = sum(_pages(n, case["page"]) - _pages(n - f, case["page"]) for n, f in zip(lengths, fresh))
        rows = sum(fresh) + case["spare"]
        return {"bytes": 8 * len(lengths) + 8 * taken + 4 * len(lengths) + 12 * rows + 4 * (len(lengths) + 1) + 8, "flops": 2 * rows}
    if case["kind"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        return {"bytes": 4 * n + case["tokens"] * (4 * case["rotary"] + 4) + (4 * case["dim"] if case["norm"] else 0), "flops": 8 * n}
    if case["kind"] == "cache":
        n = 2 * case["tokens"] * case["kv_heads"]
        return {"bytes": n * (2 * case["dim"] + 2 * (case["dim"] // 2 + 4) + 2 * case["dim"]) + 8 * case["tokens"], "flops": 6 * n * case["dim"]}
    lengths, fresh = _lengths(case)
    window = case["window"] or 1 << 60
    seen = sum(min(n, window + f - 1) for n, f in zip(lengths, fresh))
    pairs = sum(sum(min(p + 1, window) for p in range(n - f, n)) for n, f in zip(lengths, fresh))
    return {"bytes": seen * case["kv_heads"] * (case["dim"] + 8) + 4 * sum(fresh) * case["heads"] * case["dim"] + 4 * seen // case["page"], "flops": 4 * case["dim"] * case["heads"] * pairs}


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape, scale=1.0, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, scale, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _tables(case, g, spare=0):
    """lengths, fresh and their tensors, how many pages there are, a table of random pages for what is cached after the step, and the other pages."""
    lengths, fresh = _lengths(case)
    each = [_pages(n, case["page"]) for n in lengths]
    pages = sum(each) + spare
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lengths), max(each) + 1), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(each):
        table[b, :n] = order[at:at + n]
        at += n
    return lengths, fresh, pages, table, order[at:]


def _keys_and_values(case, tokens, g):
    """Keys whose channels have levels of their own, as a projection with a bias makes them, and values."""
    dt = DTYPES[case["dtype"]]
    level = _normal(g, 1, case["kv_heads"], case["dim"])
    both = _normal(g, tokens, 2 * case["kv_heads"], case["dim"], dtype=dt)
    both[:, :case["kv_heads"]] += level.to(dt)
    return both[:, :case["kv_heads"]], both[:, case["kv_heads"]:]


def _inputs(case, seed):
    """The inputs that both forms share."""
    g = _generator(seed)
    s = dict(case)
    if case["kind"] == "slots":
        lengths, fresh, pages, table, others = _tables(case, g, spare=50)
        # what the step takes is on the stack of free pages still
        free = torch.cat([others] + [table[b, _pages(n - f, case["page"]):_pages(n, case["page"])] for b, (n, f) in enumerate(zip(lengths, fresh))])
        for b, (n, f) in enumerate(zip(lengths, fresh)):
            table[b, _pages(n - f, case["page"]):] = -1
        s.update(table=table, lengths=_ints(lengths), fresh=_ints(fresh), free=free[torch.randperm(len(free), generator=g, device="cuda")].contiguous(), count=_ints([len(free)]),
                 rows=sum(fresh) + case["spare"])
    elif case["kind"] == "rope":
        t, h, kv, d = (case[x] for x in ("tokens", "heads", "kv_heads", "dim"))
        qkv = _normal(g, t, h + 2 * kv, d, dtype=DTYPES[case["dtype"]])
        far = 40000
        angles = torch.arange(far, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, case["rotary"], 2, dtype=torch.float64, device="cuda") / case["rotary"])
        weights = [(1.0 + _normal(g, d, scale=0.2)).to(qkv.dtype) if case["norm"] else None for _ in range(2)]
        s.update(q=qkv[:, :h], k=qkv[:, h:h + kv], positions=torch.randint(0, far, (t,), generator=g, dtype=torch.int32, device="cuda"), cos_sin=torch.cat([angles.cos(), angles.sin()], 1).float(),
                 w_q=weights[0], w_k=weights[1], eps=1e-6)
    elif case["kind"] == "cache":
        k, v = _keys_and_values(case, case["tokens"], g)
        pages = _pages(case["tokens"], case["page"]) + 9
        slots = torch.randperm(pages, generator=g, device="cuda")[torch.arange(case["tokens"], device="cuda") // case["page"]] * case["page"] + torch.arange(case["tokens"], device="cuda") % case["page"]
        slots[torch.rand(case["tokens"], generator=g, device="cuda") < 0.02] = -1  # padding
        s.update(k=k, v=v, slots=slots.int(), pages=pages)
    else:
        lengths, fresh, pages, table, _ = _tables(case, g, spare=3)
        s.update(q=_normal(g, sum(fresh), case["heads"], case["dim"], scale=1.5, dtype=DTYPES[case["dtype"]]), table=table, lengths=_ints(lengths),
                 starts=_ints([sum(fresh[:b]) for b in range(len(fresh) + 1)]), pages=pages, host_lengths=lengths, host_fresh=fresh, longest=max(lengths))
        s["k"], s["v"] = _keys_and_values(case, pages * case["page"], g)  # what its slots are to hold
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["kind"] in ("cache", "attend"):
        dt, kv, d = DTYPES[case["dtype"]], case["kv_heads"], case["dim"]
        if own:
            from triton_shared_amd import ops
            s["cache"] = ops.kv4_cache(s["pages"], kv, d, page=case["page"], dtype=dt, device="cuda")
        else:
            slots = s["pages"] * case["page"] + 1  # (the last for what has none)
            s["cache"] = [(torch.zeros(slots, kv, d // 2, dtype=torch.uint8, device="cuda"), torch.zeros(slots, kv, 2, dtype=dt, device="cuda")) for _ in range(2)]
    if case["kind"] == "attend":
        k, v = s.pop("k"), s.pop("v")
        for at in range(0, len(k), 65536):
            part = slice(at, min(at + 65536, len(k)))
            slots = torch.arange(part.start, part.stop, dtype=torch.int32, device="cuda")
            if own:
                ops.kv4_write(s["cache"], k[part], v[part], slots)
            else:
                for kept, x in zip(s["cache"], (k, v)):
                    _write_plain(kept, x[part], slots.long())
    return s


def _slots_plain(s):
    table, page = s["table"], s["page"]
    lengths, fresh = s["lengths"].long(), s["fresh"].long()
    past = lengths - fresh
    ends = torch.cumsum(fresh, 0)
    starts = torch.cat([torch.zeros_like(ends[:1]), ends])
    before, after = (past + page - 1) // page, (lengths + page - 1) // page
    first = torch.cumsum(after - before, 0) - (after - before)
    columns = torch.arange(table.shape[1], device="cuda")[None]
    at = s["count"].long() - 1 - (first[:, None] + columns - before[:, None])
    new = (columns >= before[:, None]) & (columns < after[:, None])
    table.copy_(torch.where(new, torch.where(at >= 0, s["free"][at.clamp(0, len(s["free"]) - 1)], -1), table))
    rows = torch.arange(s["rows"], device="cuda")
    requests = (rows[:, None] >= ends[None]).sum(dim=1)
    real = requests < len(ends)
    r = requests.clamp(max=len(ends) - 1)
    positions = past[r] + rows - starts[r]
    pages = table[r, (positions // page).clamp(0, table.shape[1] - 1)].long()
    slots = torch.where(real & (pages >= 0), pages * page + positions % page, -1)
    left = (s["count"] - (after - before).sum()).clamp(min=0)
    return {"table": table, "slots": slots.int(), "positions": torch.where(real, positions, -1).int(), "requests": torch.where(real, requests, -1).int(), "starts": starts.int(), "left": left.int()}


def _rope_plain(s, x, w):
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt((y * y).mean(dim=2, keepdim=True) + s["eps"]) * w.float()
    r = s["rotary"]
    at = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin = at[..., :r // 2], at[..., r // 2:]
    if s["interleaved"]:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=3).flatten(2)
    else:
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=2)
    return torch.cat([turned, y[..., r:]], dim=2).to(x.dtype)


def _write_plain(kept, x, slots):
    codes, pairs = kept
    low, high = x.amin(dim=2), x.amax(dim=2)
    step = ((high.float() - low.float()) / 15.0).to(x.dtype)
    # in 64 bits: next to a border between two codes 32 may lose which side it is
    code = torch.ceil((x.double() - low.double()[..., None]) / step.double()[..., None] - 0.5).clamp(0, 15)
    code = torch.where(step[..., None] > 0, code, 0.0).to(torch.uint8)
    codes[slots] = code[..., 0::2] | code[..., 1::2] << 4
    pairs[slots] = torch.stack([step, low], dim=2)


def _read_plain(kept, slots):
    codes, pairs = kept[0][slots], kept[1][slots].float()
    code = torch.stack([codes & 15, codes >> 4], dim=3).flatten(2).float()
    return code * pairs[..., 0:1] + pairs[..., 1:2]


def _cache_plain(s):
    there = s["slots"] >= 0
    slots = torch.where(there, s["slots"], s["pages"] * s["page"]).long()
    out = []
    for kept, x in zip(s["cache"], (s["k"], s["v"])):
        _write_plain(kept, x, slots)
        out.append(torch.where(there[:, None, None], _read_plain(kept, slots), 0.0).to(x.dtype))
    return out


def _attend_plain(s):
    q, page, kv = s["q"], s["page"], s["kv_heads"]
    out = torch.empty_like(q)
    group, scale, at = s["heads"] // kv, s["dim"] ** -0.5, 0
    for b, (n, f) in enumerate(zip(s["host_lengths"], s["host_fresh"])):
        first = max(0, n - f + 1 - s["window"]) if s["window"] else 0  # what none of its rows sees is left out
        seen = torch.arange(first, n, device="cuda")
        slots = s["table"][b].long()[seen // page] * page + seen % page
        k, v = (_read_plain(kept, slots).transpose(0, 1).contiguous() for kept in s["cache"])
        rows = q[at:at + f].float().reshape(f, kv, group, -1).transpose(0, 1).reshape(kv, f * group, -1)
        scores = torch.matmul(rows, k.transpose(1, 2).contiguous()) * scale
        where = torch.arange(n - f, n, device="cuda").repeat_interleave(group)[:, None]
        hidden = seen[None] > where
        if s["window"]:
            hidden = hidden | (seen[None] <= where - s["window"])
        scores = scores.masked_fill(hidden[None], float("-inf"))
        weights = torch.exp(scores - scores.amax(dim=2, keepdim=True))
        y = torch.matmul(weights, v) / weights.sum(dim=2, keepdim=True)
        out[at:at + f] = y.reshape(kv, f, group, -1).transpose(0, 1).reshape(f, s["heads"], -1).to(q.dtype)
        at += f
    return out


def run(s):
    """One pass through an operator (`cache`: through the two that write and read), and its outputs."""
    if own:
        from triton_shared_amd import ops
    if s["kind"] == "slots":
        if not own:
            return _slots_plain(s)
        slots, positions, requests, starts, left = ops.page_slots(s["table"], s["lengths"], s["fresh"], s["free"], s["count"], s["page"], s["rows"])
        return {"table": s["table"], "slots": slots, "positions": positions, "requests": requests, "starts": starts, "left": left}
    if s["kind"] == "rope":
        if own:
            q, k = ops.qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], s["w_q"], s["w_k"], eps=s["eps"], interleaved=s["interleaved"])
        else:
            q, k = _rope_plain(s, s["q"], s["w_q"]), _rope_plain(s, s["k"], s["w_k"])
        return {"q": q, "k": k}
    if s["kind"] == "cache":
        if own:
            ops.kv4_write(s["cache"], s["k"], s["v"], s["slots"])
            k, v = ops.kv4_read(s["cache"], s["slots"], s["dim"])
        else:
            k, v = _cache_plain(s)
        return {"k": k, "v": v}
    if own:
        return ops.kv4_attention(s["q"], s["cache"], s["table"], s["lengths"], s["starts"], window=s["window"] or None, longest=s["longest"])
    return _attend_plain(s)


def _held(x):
    """The values that 4 bits hold of x, by the borders between codes, in 64 bits."""
    wide = x.double()
    low, high = wide.min(dim=-1, keepdim=True).values, wide.max(dim=-1, keepdim=True).values
    step = ((high.float() - low.float()) / torch.tensor(15.0, device=x.device)).to(x.dtype).double()  # (the format's: in 32 bits, then in the type)
    code = torch.zeros_like(wide)
    for border in range(15):
        code += (wide - low > (border + 0.5) * step).double()
    return code * step + low


def exact(case, seed):
    """The same outputs from the definitions in 64 bits: a request, a token or a head at a time."""
    s = _inputs(case, seed)
    if case["kind"] == "slots":
        table, free, page = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy(), case["page"]
        left, total = int(s["count"][0]), 0
        slots, positions, requests = (np.full(s["rows"], -1, np.int32) for _ in range(3))
        starts = [0]
        for b, (n, f) in enumerate(zip(*_lengths(case))):
            for p in range(n - f, n):
                if p % page == 0:
                    left -= 1
                    table[b, p // page] = free[left]
                slots[total], positions[total], requests[total] = table[b, p // page] * page + p % page, p, b
                total += 1
            starts.append(total)
        return {"table": table, "slots": slots, "positions": positions, "requests": requests, "starts": np.array(starts, np.int32), "left": np.array([left], np.int32)}
    if case["kind"] == "rope":
        out, half = {}, case["rotary"] // 2
        at = s["cos_sin"].double()[s["positions"].long()]
        turn = torch.complex(at[:, :half], at[:, half:])[:, None]
        first = torch.arange(half, device="cuda") * (2 if case["interleaved"] else 1)
        second = first + (1 if case["interleaved"] else half)
        for name in ("q", "k"):
            y = s[name].double()
            if case["norm"]:
                y = y / torch.sqrt(y.pow(2).sum(dim=2, keepdim=True) / case["dim"] + s["eps"]) * s["w_" + name].double()
            z = torch.complex(y[..., first], y[..., second]) * turn
            y = y.clone()
            y[..., first], y[..., second] = z.real, z.imag
            out[name] = y
        return out
    if case["kind"] == "cache":
        there = (s["slots"] >= 0).double()[:, None, None]
        return {"k": _held(s["k"]) * there, "v": _held(s["v"]) * there}
    kv, page, window = case["kv_heads"], case["page"], case["window"]
    group, out = case["heads"] // kv, []
    for b, (n, f) in enumerate(zip(s["host_lengths"], s["host_fresh"])):
        first = max(0, n - f + 1 - window) if window else 0
        j = torch.arange(first, n, device="cuda")
        slots = s["table"][b].long()[j // page] * page + j % page
        i = torch.arange(n - f, n, device="cuda")
        seen = j[None] <= i[:, None]
        if window:
            seen &= j[None] > i[:, None] - window
        q = s["q"][s["starts"][b]:s["starts"][b + 1]].double()
        y = torch.empty(f, case["heads"], case["dim"], dtype=torch.float64, device="cuda")
        for g in range(kv):
            k, v = _held(s["k"][slots, g]), _held(s["v"][slots, g])
            for h in range(g * group, (g + 1) * group):
                score = (q[:, h] @ k.t()) / math.sqrt(case["dim"])
                y[:, h] = torch.softmax(torch.where(seen, score, -math.inf), dim=1) @ v
        out.append(y)
    return torch.cat(out)
