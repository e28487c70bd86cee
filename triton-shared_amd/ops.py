"""Operators whose weights are picked per row of activations: what a decode step does beside its shared projections.

    ids, weights = ops.moe_route(logits, 8)                                  # the router, from its logits
    y = ops.moe_experts(x, ids, weights, w_up, w_down)                       # the experts of a few tokens
    q = ops.lora_add(q, x, a, b, adapter_of_row, scales=scales, out=q)       # adapters of many requests, after the projection

They are hand-written kernels behind the C ABI (include/tts_hip.h: tts_moe_route, tts_moe_experts, tts_lora_add), for code that
calls them beside its Triton kernels: on the current stream of their tensors' device, asynchronous, capturable into a graph.
Wrong arguments raise ValueError or TypeError, what is not implemented NotImplementedError, failing HIP calls RuntimeError.
They have no derivatives: tensors that require gradients are refused where gradients are recorded, and those with a forward-mode tangent anywhere.
"""
import ctypes

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
    """The launch extension's own moe_route, moe_experts and lora_add (csrc/launch_module.cpp), which take the ordinary calls; False without it."""
    global _fast
    module, lib = _native.launch_module(), _native.lib()
    if module is None:
        _fast = False
    else:
        address = lambda f: ctypes.cast(f, ctypes.c_void_p).value  # noqa: E731
        module.setup_ops(address(lib.tts_moe_route), address(lib.tts_moe_experts_workspace), address(lib.tts_moe_experts), address(lib.tts_lora_add_workspace), address(lib.tts_lora_add),
                         torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream, torch.is_grad_enabled, *_DTYPES, torch.Tensor, torch.nn.Parameter, _native._raise)
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
