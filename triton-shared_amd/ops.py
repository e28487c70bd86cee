"""Operators of a decode step beside its shared projections.  Those whose weights are picked per row of activations:

    ids, weights = ops.moe_route(logits, 8)                                  # the router, from its logits
    y = ops.moe_experts(x, ids, weights, w_up, w_down)                       # the experts of a few tokens
    q = ops.lora_add(q, x, a, b, adapter_of_row, scales=scales, out=q)       # adapters of many requests, after the projection

and its attention over a paged cache held in 4 bits:

    cache = ops.kv4_cache(pages, kv_heads, dim, page=16)                                                       # once, of each layer
    slots, positions, owners, starts, left = ops.page_slots(table, lengths, fresh, free, count, 16, rows)      # once a step, for all layers
    q, k = ops.qk_norm_rope(q, k, positions, cos_sin, w_q, w_k)
    ops.kv4_write(cache, k, v, slots)
    y = ops.kv4_attention(q, cache, table, lengths, starts)                                                    # (kv4_read: what slots hold, as values)

They are hand-written kernels behind the C ABI (include/tts_hip.h: tts_moe_route, tts_moe_experts, tts_lora_add, tts_page_slots, tts_qk_norm_rope,
tts_kv4_write, tts_kv4_read, tts_kv4_attention), for code that calls them beside its Triton kernels: on the current stream of their tensors' device,
asynchronous, capturable into a graph.
Wrong arguments raise ValueError or TypeError, what is not implemented NotImplementedError, failing HIP calls RuntimeError.
They have no derivatives: tensors that require gradients are refused where gradients are recorded, and those with a forward-mode tangent anywhere.
"""
import ctypes
import math
import operator

import torch
from torch.autograd import forward_ad

from . import _native

_DTYPES = {torch.float32: _native.DTYPE_F32, torch.float16: _native.DTYPE_F16, torch.bfloat16: _native.DTYPE_BF16, torch.int8: _native.DTYPE_I8, torch.int32: _native.DTYPE_I32}
_SCORING = {"softmax": 0, "sigmoid": 1}
_ACTIVATION = {"silu": 0, "gelu_tanh": 1, "relu": 2}


def _describe(name, t, device):
    """The tts_tensor of an argument (None: a null pointer)."""
    if t is None:
        return None
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a {type(t).__name__}, not a tensor")
    if t.device != device:
        raise TypeError(f"{name} lives on device '{t.device}', not on '{device}'" if t.is_cuda else f"{name} lives on device '{t.device}'; this backend needs GPU memory")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} is {t.dtype}")
    if t.dim() > 3:
        raise ValueError(f"{name} has {t.dim()} dimensions")
    if t.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(f"{name} requires a gradient, and this operator has no backward pass: call it under torch.no_grad()")
    if forward_ad.unpack_dual(t).tangent is not None:
        raise NotImplementedError(f"{name} has a forward-mode tangent, which this operator does not carry on")
    d = _native.TtsTensor(t.data_ptr(), _DTYPES[t.dtype], t.dim())
    d.shape[:t.dim()] = t.shape
    d.stride[:t.dim()] = t.stride()
    return d


_fast = None


def _native_calls():
    """The launch extension's functions of the names below (csrc/launch_module.cpp), which take the ordinary calls; False without it."""
    global _fast
    module, lib = _native.launch_module(), _native.lib()
    if module is None:
        _fast = False
    else:
        address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
        entries = (lib.tts_moe_route, lib.tts_moe_experts_workspace, lib.tts_moe_experts, lib.tts_lora_add_workspace, lib.tts_lora_add, lib.tts_page_slots, lib.tts_qk_norm_rope,
                   lib.tts_kv4_write, lib.tts_kv4_read, lib.tts_kv4_attention_workspace, lib.tts_kv4_attention)
        module.setup_ops(*map(address, entries), torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch.is_grad_enabled, *_DTYPES, torch.Tensor, torch.nn.Parameter,
                         _native._raise)
        _fast = module
    return _fast


def _ordinary():
    """The launch extension's calls, or False: without it, and inside a level of forward-mode derivatives, since it does not look for tangents."""
    fast = _native_calls() if _fast is None else _fast
    return fast if getattr(forward_ad, "_current_level", 0) < 0 else False


def _device_of(name, t):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} is a {type(t).__name__}, not a tensor")
    if not t.is_cuda:
        raise TypeError(f"{name} lives on device '{t.device}'; this backend needs GPU memory")
    return t.device


def _choice(name, value, table):
    if value not in table:
        raise ValueError(f"{name} is {value!r}, not one of {', '.join(map(repr, table))}")
    return table[value]


def _written(out):
    """`out`, of which autograd knows now that it has changed: a backward pass that has saved it raises."""
    torch.autograd.graph.increment_version(out)
    return out


def _whole(name, value):
    """An integer argument, which C's conversion would cut to 32 bits."""
    value = operator.index(value)
    if not -2 ** 31 <= value < 2 ** 31:
        raise ValueError(f"{name} is {value}")
    return value


def _call(entry, device, *args):
    with torch.cuda.device(device):
        status = entry(*args, torch.cuda.current_stream(device).cuda_stream)
    if status != _native.TTS_OK:
        _native._raise(status)


def _workspace(entry, device, *args):
    size = ctypes.c_size_t()
    status = entry(*args, ctypes.byref(size))
    if status != _native.TTS_OK:
        _native._raise(status)
    return torch.empty(size.value, dtype=torch.uint8, device=device)


def moe_route(logits, k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    """The router of a mixture-of-experts layer: (ids int32 [T, k], weights float32 [T, k]) from logits [T, E].

    With s the softmax or the sigmoid of a row, ids are the experts of the k largest s + bias (without a bias: the k largest logits),
    largest first, ties to the lowest expert; weights are scale * s, over the sum of the chosen s if `renormalize` (right also
    where 32 bits hold none of them; under e^-745 s counts as 0).  Logits of -inf are never chosen: where fewer
    than k others are left, ids are -1 and weights 0.  A row that holds a NaN gets weights of NaN, as does the softmax of
    one that holds +inf.
    """
    fast = _ordinary()
    if fast:
        made = fast.moe_route(logits, k, _SCORING.get(scoring), bias, renormalize, scale)
        if made is not None:
            return made
    device = _device_of("logits", logits)
    if logits.dim() != 2:
        raise ValueError(f"logits have {logits.dim()} dimensions, not 2")
    if k < 1 or k > logits.shape[1]:
        raise ValueError(f"k is {k}" if k < 1 else f"k is {k}, and there are {logits.shape[1]} experts")
    ids = torch.empty(logits.shape[0], k, dtype=torch.int32, device=device)
    weights = torch.empty(logits.shape[0], k, dtype=torch.float32, device=device)
    _call(_native.lib().tts_moe_route, device, _describe("logits", logits, device), _describe("bias", bias, device), _choice("scoring", scoring, _SCORING), bool(renormalize),
          float(scale), _describe("ids", ids, device), _describe("weights", weights, device))
    return ids, weights


def moe_experts(x, ids, weights, w_up, w_down, s_up=None, s_down=None, activation="silu", gated=True, out=None):
    """The experts of a mixture-of-experts layer for a few tokens (T * k <= 4096):

        out[t] = sum over j of weights[t, j] * (h w_down[e]),   h = f(x[t] w_up[e][:, :I]) * (x[t] w_up[e][:, I:]),   e = ids[t, j]

    x [T, H] in float16 or bfloat16, ids [T, k] int32 and weights [T, k] float32 as `moe_route` gives them, w_up [E, H, 2 I] (not `gated`: [E, H, I],
    and h = f(x[t] w_up[e])), w_down [E, I, O].  Weights are of x's type, or int8 with float32 scales per output column: s_up [E, 2 I], s_down [E, O].
    Either dimension of a matrix may be the contiguous one: pass `w.transpose(1, 2)` of weights stored as [E, outputs, inputs].
    An id outside [0, E) contributes nothing.  `out` may be x.
    """
    fast = _ordinary()
    if fast:
        made = fast.moe_experts(x, ids, weights, w_up, w_down, s_up, s_down, _ACTIVATION.get(activation), gated, out)
        if made is not None:
            return made if out is None else _written(out)
    device = _device_of("x", x)
    act = _choice("activation", activation, _ACTIVATION)
    dx, di, du, dd = _describe("x", x, device), _describe("ids", ids, device), _describe("w_up", w_up, device), _describe("w_down", w_down, device)
    work = _workspace(_native.lib().tts_moe_experts_workspace, device, dx, di, du, dd, bool(gated))
    given, out = out, torch.empty(x.shape[0], w_down.shape[2], dtype=x.dtype, device=device) if out is None else out
    _call(_native.lib().tts_moe_experts, device, dx, di, _describe("weights", weights, device), du, _describe("s_up", s_up, device), dd, _describe("s_down", s_down, device), act,
          bool(gated), _describe("out", out, device), work.data_ptr(), work.numel())
    return out if given is None else _written(out)


def lora_add(base, x, a, b, ids, scales=None, out=None):
    """Low-rank adapters of many requests, added to what a shared projection made of the same rows:

        out[t] = base[t] + scales[d] * (x[t] a[d]^T) b[d]^T,   d = ids[t];   out[t] = base[t] where d is not in [0, n)

    base [T, N], x [T, K], a [n, r, K], b [n, N, r] (as nn.Linear stores such weights), all float16 or all bfloat16; ids [T] int32, scales [n] float32
    or None for 1; T up to 2097120.  `out` may be base itself, for an update in place.  A prompt's rows next to each other share the reading of their adapter.
    """
    fast = _ordinary()
    if fast:
        made = fast.lora_add(base, x, a, b, ids, scales, out)
        if made is not None:
            return made if out is None else _written(out)
    device = _device_of("base", base)
    db, dx, da, dl = _describe("base", base, device), _describe("x", x, device), _describe("a", a, device), _describe("b", b, device)
    work = _workspace(_native.lib().tts_lora_add_workspace, device, dx, dl)
    given, out = out, torch.empty_like(base, memory_format=torch.contiguous_format) if out is None else out
    _call(_native.lib().tts_lora_add, device, db, dx, da, dl, _describe("ids", ids, device), _describe("scales", scales, device), _describe("out", out, device), work.data_ptr(),
          work.numel())
    return out if given is None else _written(out)


def page_slots(table, lengths, fresh, free, count, page, rows):
    """Block tables and slot maps of a step, from its requests' lengths: (slots [rows], positions [rows], owners [rows], starts [B + 1], left [1]), all int32.

    table [B, M] int32 holds the pages of each request in order (`page` tokens each); lengths [B] int32 the tokens it has after this step, fresh [B] int32 how many of them are new, its last ones.
    free [F] int32 is a stack of free pages, the first count[0] of it, the last of them the top.  Requests take the pages that they lack from the top, the first
    request first, and those are written into `table` (-1 where the stack has run out); `left` is what count is afterwards.  The step's rows are the new tokens of one request after another:
    request b's are starts[b] .. starts[b + 1] - 1, `owners` has the request of each, `positions` its position and `slots` its place in the cache, for `kv4_write`.  A row
    without a page has slot -1, and rows behind the last request's -1 in all three.  B up to 4096.
    """
    fast = _ordinary()
    if fast:
        made = fast.page_slots(table, lengths, fresh, free, count, page, rows)
        if made is not None:
            _written(table)
            return made
    device = _device_of("table", table)
    if table.dim() != 2:
        raise ValueError(f"table has {table.dim()} dimensions, not 2")
    page, rows = _whole("page", page), _whole("rows", rows)
    if rows < 0:
        raise ValueError(f"rows is {rows}")
    sizes = (rows, rows, rows, table.shape[0] + 1, 1)
    made = torch.empty(sum(sizes), dtype=torch.int32, device=device).split_with_sizes(sizes)
    _call(_native.lib().tts_page_slots, device, *(_describe(n, t, device) for n, t in (("table", table), ("lengths", lengths), ("fresh", fresh), ("free", free), ("count", count))), page,
          *(_describe(n, t, device) for n, t in zip(("slots", "positions", "owners", "starts", "left"), made)))
    _written(table)
    return made


def qk_norm_rope(q, k, positions, cos_sin, w_q=None, w_k=None, eps=1e-6, interleaved=False, out=None):
    """Norms of queries and keys for each head, and the rotation by position, in one pass: (q, k) turned.

    q [T, Hq, D] and k [T, Hk, D] in float32, float16 or bfloat16 (D even, up to 512), views of one projection's rows as well.  Of each head y = x / sqrt(mean(x^2) + eps) * w, with w_q and
    w_k [D] of its type or float32 (without them y = x); then pairs (a, b) of its first R elements become (a cos - b sin, b cos + a sin): elements n and n + R / 2, or 2 n and
    2 n + 1 if `interleaved`.  cos_sin [P, R] float32 has the cosines of a position's R / 2 angles, then their sines; positions [T] int32.  Rows whose position is not in [0, P) are padding:
    zeros in what is returned, or, in an `out` that is given, as they were.  `out` is a pair (q, k) and may be q and k themselves.
    """
    fast = _ordinary()
    given = out is not None
    q_out, k_out = out if given else (None, None)
    if given and (q_out is None or k_out is None):
        raise ValueError("out is a pair of tensors")
    if fast:
        made = fast.qk_norm_rope(q, k, positions, cos_sin, w_q, w_k, eps, interleaved, q_out, k_out)
        if made is not None:
            return (_written(q_out), _written(k_out)) if given else made
    device = _device_of("q", q)
    dq, dk = _describe("q", q, device), _describe("k", k, device)
    if not given:
        q_out, k_out = torch.empty_like(q, memory_format=torch.contiguous_format), torch.empty_like(k, memory_format=torch.contiguous_format)
    _call(_native.lib().tts_qk_norm_rope, device, dq, dk, _describe("positions", positions, device), _describe("cos_sin", cos_sin, device), _describe("w_q", w_q, device),
          _describe("w_k", w_k, device), float(eps), bool(interleaved), not given, _describe("q_out", q_out, device), _describe("k_out", k_out, device))
    return (_written(q_out), _written(k_out)) if given else (q_out, k_out)


def kv4_cache(pages, heads, dim, page=16, dtype=torch.bfloat16, device="cuda"):
    """An empty cache of 4 bits for one layer: [pages, heads, page * (dim + 8) / 2] of `dtype` (float16 or bfloat16, the type of its keys and values), whose inner layout the operators know.

    `dim` is a multiple of 32 up to 256, `page` (the tokens of a page) a multiple of 16.  What it takes is dim + 8 bytes for a token's key and value of each head.
    """
    if dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"dtype is {dtype}, not float16 or bfloat16")
    if dim % 32 or not 32 <= dim <= 256:
        raise NotImplementedError(f"heads of {dim} elements, not a multiple of 32 up to 256")
    if page % 16 or page < 16:
        raise NotImplementedError(f"pages of {page} tokens, not a multiple of 16")
    return torch.zeros(pages, heads, page * (dim + 8) // 2, dtype=dtype, device=device)


def kv4_write(cache, k, v, slots):
    """Puts keys and values k, v [T, Hk, D] of the cache's type into its slots [T] int32 and returns the cache; rows whose slot is not in it (-1: padding) are left out.

    Of each head of a token, and of key and value each: an element x is held as code * step + lowest, step = (highest - lowest) / 15 rounded to the type, code the number of borders (n + 1/2) * step
    that x - lowest is above.  What is not finite makes the head NaN.  The slots in the cache are distinct (as `page_slots` gives them).
    """
    fast = _ordinary()
    if fast and fast.kv4_write(cache, k, v, slots) is not None:
        return _written(cache)
    device = _device_of("cache", cache)
    _call(_native.lib().tts_kv4_write, device, _describe("cache", cache, device), _describe("k", k, device), _describe("v", v, device), _describe("slots", slots, device))
    return _written(cache)


def kv4_read(cache, slots, dim):
    """The keys and values [T, Hk, dim] that slots [T] int32 of a cache hold, as values of its type; zeros for a slot that is not in it."""
    fast = _ordinary()
    if fast:
        made = fast.kv4_read(cache, slots, dim)
        if made is not None:
            return made
    device = _device_of("cache", cache)
    if cache.dim() != 3:
        raise ValueError(f"cache has {cache.dim()} dimensions, not 3")
    ds = _describe("slots", slots, device)
    if slots.dim() != 1:
        raise ValueError(f"slots have {slots.dim()} dimensions, not 1")
    k, v = (torch.empty(slots.shape[0], cache.shape[1], _whole("dim", dim), dtype=cache.dtype, device=device) for _ in range(2))
    _call(_native.lib().tts_kv4_read, device, _describe("cache", cache, device), ds, _describe("k", k, device), _describe("v", v, device))
    return k, v


def kv4_attention(q, cache, table, lengths, starts, scale=None, window=None, longest=None, out=None):
    """Attention of a step's rows over the cache:

        out[t, h] = sum over j of softmax_j(scale * q[t, h] . k_j) v_j

    q [T, Hq, D] of the cache's type, Hq a multiple of its heads: head h reads the cache's head h // (Hq // Hk).  Rows starts[b] .. starts[b + 1] - 1 are the last tokens of request b, which has
    lengths[b] tokens in the pages table[b] (table [B, M], lengths [B], starts [B + 1], all int32, as `page_slots` leaves them); the row at position i sees the tokens j <= i, with a
    `window` those of i - window < j.  scale is D ** -0.5 unless it is given.  A row that sees nothing is zeros; rows of no request are zeros too, or as they were in an `out` that is given (it may be q).
    `longest`, a length that no request passes, lets short requests in a wide table do with fewer workgroups.  A table's row has places for less than 2^30 tokens.
    """
    if window is not None and _whole("window", window) < 1:
        raise ValueError(f"window is {window}")
    if longest is not None and _whole("longest", longest) < 1:
        raise ValueError(f"longest is {longest}")
    fast = _ordinary()
    if fast:
        made = fast.kv4_attention(q, cache, table, lengths, starts, scale, window or 0, longest or 0, out)
        if made is not None:
            return made if out is None else _written(out)
    device = _device_of("q", q)
    dq, dc, dt = _describe("q", q, device), _describe("cache", cache, device), _describe("table", table, device)
    work = _workspace(_native.lib().tts_kv4_attention_workspace, device, dq, dc, dt, window or 0, longest or 0)
    given, out = out, torch.empty_like(q, memory_format=torch.contiguous_format) if out is None else out
    _call(_native.lib().tts_kv4_attention, device, dq, dc, dt, _describe("lengths", lengths, device), _describe("starts", starts, device), float(1.0 / math.sqrt(q.shape[2]) if scale is None else scale),
          window or 0, longest or 0, given is None, _describe("out", out, device), work.data_ptr(), work.numel())
    return out if given is None else _written(out)
