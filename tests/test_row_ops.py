"""The operators whose weights are picked per row (triton_shared_amd.ops; tts_moe_route, tts_moe_experts, tts_lora_add): against
their formulas in 64 bits, at the sizes, ids and values where they can go wrong; what they refuse (no GPU needed); and a decode step of
all of them together."""
import ctypes
import itertools

import numpy as np
import pytest
import torch

import triton_shared_amd as tsa
from triton_shared_amd import ops

N = tsa._native
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of fp32


def half(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def smallest(dtype):
    return torch.finfo(TYPES[dtype]).smallest_normal * torch.finfo(TYPES[dtype]).eps  # a step below the normal numbers


def gpu(*shape, seed=0, scale=1.0, dtype="fp32"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g).to(TYPES[dtype])


# ---------------------------------------------------------------------------------------------------------------- refusals, on the CPU
FAKE = 1 << 20  # an address that a refused call never uses


def tensor(dtype, *shape, stride=None, ptr=FAKE):
    t = N.TtsTensor(ptr, dtype, len(shape))
    if stride is None:
        stride = [int(np.prod(shape[d + 1:])) for d in range(len(shape))]
    t.shape[:len(shape)] = list(shape)
    t.stride[:len(shape)] = list(stride)
    return t


F32, F16, BF16, I8, I32 = N.DTYPE_F32, N.DTYPE_F16, N.DTYPE_BF16, N.DTYPE_I8, N.DTYPE_I32
FAR = [FAKE + (i << 32) for i in range(16)]


def route_args(**kw):
    a = dict(logits=tensor(BF16, 4, 16, ptr=FAR[0]), bias=None, scoring=0, renormalize=1, scale=1.0, ids=tensor(I32, 4, 2, ptr=FAR[1]), weights=tensor(F32, 4, 2, ptr=FAR[2]), stream=None)
    return list((a | kw).values())


def experts_args(**kw):
    a = dict(x=tensor(BF16, 4, 64, ptr=FAR[0]), ids=tensor(I32, 4, 2, ptr=FAR[1]), weights=tensor(F32, 4, 2, ptr=FAR[2]), w_up=tensor(BF16, 8, 64, 96, ptr=FAR[3]), s_up=None,
             w_down=tensor(BF16, 8, 48, 64, ptr=FAR[4]), s_down=None, activation=0, gated=1, out=tensor(BF16, 4, 64, ptr=FAR[5]), work=FAR[6], bytes=1 << 30, stream=None)
    return list((a | kw).values())


def lora_args(**kw):
    a = dict(base=tensor(F16, 4, 96, ptr=FAR[0]), x=tensor(F16, 4, 64, ptr=FAR[1]), a=tensor(F16, 3, 16, 64, ptr=FAR[2]), b=tensor(F16, 3, 96, 16, ptr=FAR[3]), ids=tensor(I32, 4, ptr=FAR[4]),
             scales=None, out=tensor(F16, 4, 96, ptr=FAR[5]), work=FAR[6], bytes=1 << 30, stream=None)
    return list((a | kw).values())


REFUSALS = [
    ("tts_moe_route", route_args, dict(logits=None), N.TTS_INVALID, "logits is missing"),
    ("tts_moe_route", route_args, dict(logits=tensor(I32, 4, 16)), N.TTS_INVALID, "logits are i32"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 4, 16, stride=(1, 4))), N.TTS_INVALID, "stride 4, not 1"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 64)), N.TTS_INVALID, "1 dimensions, not 2"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 4, 2000)), N.TTS_UNSUPPORTED, "2000 experts"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 4, 1)), N.TTS_INVALID, "2 of 1 experts"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 4, 16, ptr=0)), N.TTS_INVALID, "null pointer"),
    ("tts_moe_route", route_args, dict(logits=tensor(BF16, 4, 16, ptr=FAKE + 1)), N.TTS_INVALID, "not aligned"),
    ("tts_moe_route", route_args, dict(scoring=2), N.TTS_INVALID, "scoring 2"),
    ("tts_moe_route", route_args, dict(bias=tensor(F32, 15)), N.TTS_INVALID, "bias: dimension 0 is 15"),
    ("tts_moe_route", route_args, dict(bias=tensor(BF16, 16)), N.TTS_INVALID, "bias is bf16, not f32"),
    ("tts_moe_route", route_args, dict(ids=tensor(I32, 4, 0)), N.TTS_INVALID, "empty"),
    ("tts_moe_route", route_args, dict(ids=tensor(I32, 4, 2, stride=(1, 1))), N.TTS_INVALID, "rows overlap"),
    ("tts_moe_route", route_args, dict(ids=tensor(I32, 4, 2, ptr=FAR[2])), N.TTS_INVALID, "ids shares memory with weights"),
    ("tts_moe_route", route_args, dict(weights=tensor(F32, 4, 2, ptr=FAR[0] + 64)), N.TTS_INVALID, "weights shares memory with logits"),
    ("tts_moe_route", route_args, dict(logits=tensor(F32, 4, 100), ids=tensor(I32, 4, 65), weights=tensor(F32, 4, 65)), N.TTS_UNSUPPORTED, "65 experts of a token"),
    ("tts_moe_experts", experts_args, dict(x=tensor(F32, 4, 64)), N.TTS_UNSUPPORTED, "takes f16 and bf16"),
    ("tts_moe_experts", experts_args, dict(x=tensor(BF16, 4, 64, stride=(128, 2))), N.TTS_INVALID, "x: its last dimension"),
    ("tts_moe_experts", experts_args, dict(x=tensor(BF16, 4, 72)), N.TTS_INVALID, "w_up: dimension 1 is 64"),
    ("tts_moe_experts", experts_args, dict(ids=tensor(I32, 5, 2)), N.TTS_INVALID, "ids: dimension 0 is 5"),
    ("tts_moe_experts", experts_args, dict(ids=tensor(F32, 4, 2)), N.TTS_INVALID, "ids is f32, not i32"),
    ("tts_moe_experts", experts_args, dict(weights=tensor(F32, 4, 3)), N.TTS_INVALID, "weights: dimension 1 is 3"),
    ("tts_moe_experts", experts_args, dict(weights=tensor(BF16, 4, 2)), N.TTS_INVALID, "weights is bf16"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(F16, 8, 64, 96)), N.TTS_INVALID, "w_up is f16, not i8 or x's type"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(BF16, 8, 64, 95)), N.TTS_INVALID, "two halves"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(BF16, 8, 64, 96, stride=(64 * 192, 192, 2))), N.TTS_INVALID, "neither its inputs"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(BF16, 8, 64, 96, stride=(1 << 40, 1, 1 << 30))), N.TTS_UNSUPPORTED, "past 4 GiB"),
    ("tts_moe_experts", experts_args, dict(w_down=tensor(BF16, 7, 48, 64)), N.TTS_INVALID, "w_down: dimension 0 is 7"),
    ("tts_moe_experts", experts_args, dict(w_down=tensor(BF16, 8, 96, 64)), N.TTS_INVALID, "w_down: dimension 1 is 96"),
    ("tts_moe_experts", experts_args, dict(w_down=tensor(I8, 8, 48, 64)), N.TTS_INVALID, "w_down is i8, not bf16"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(BF16, 8, 64, 8), w_down=tensor(BF16, 8, 4, 64)), N.TTS_UNSUPPORTED, "narrower than 8"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(I8, 8, 64, 24), w_down=tensor(I8, 8, 12, 64)), N.TTS_UNSUPPORTED, "narrower than 16"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(BF16, 8, 64, 1 << 26, stride=(64, 1, 1)), w_down=tensor(BF16, 8, 1 << 25, 64)), N.TTS_UNSUPPORTED, "wider than 16777216"),
    ("tts_moe_experts", experts_args, dict(s_up=tensor(F32, 8, 96)), N.TTS_INVALID, "scales belong to i8"),
    ("tts_moe_experts", experts_args, dict(w_up=tensor(I8, 8, 64, 96), w_down=tensor(I8, 8, 48, 64)), N.TTS_INVALID, "s_up is missing"),
    ("tts_moe_experts", experts_args, dict(activation=3), N.TTS_INVALID, "activation 3"),
    ("tts_moe_experts", experts_args, dict(out=tensor(F16, 4, 64)), N.TTS_INVALID, "out is f16, not bf16"),
    ("tts_moe_experts", experts_args, dict(out=tensor(BF16, 4, 64, stride=(0, 1))), N.TTS_INVALID, "rows overlap"),
    ("tts_moe_experts", experts_args, dict(out=tensor(BF16, 4, 64, ptr=FAR[4] + 256)), N.TTS_INVALID, "out shares memory with w_down"),
    ("tts_moe_experts", experts_args, dict(bytes=16), N.TTS_INVALID, "the workspace has 16 bytes"),
    ("tts_moe_experts", experts_args, dict(work=None), N.TTS_INVALID, "workspace is a null pointer"),
    ("tts_moe_experts", experts_args, dict(work=FAR[6] + 16), N.TTS_INVALID, "256 bytes"),
    ("tts_moe_experts", experts_args, dict(x=tensor(BF16, 2049, 64), ids=tensor(I32, 2049, 2), weights=tensor(F32, 2049, 2), out=tensor(BF16, 2049, 64)), N.TTS_UNSUPPORTED, "more than 4096 in all"),
    ("tts_lora_add", lora_args, dict(x=tensor(F32, 4, 64)), N.TTS_UNSUPPORTED, "takes f16 and bf16"),
    ("tts_lora_add", lora_args, dict(base=tensor(BF16, 4, 96)), N.TTS_INVALID, "base is bf16, not f16"),
    ("tts_lora_add", lora_args, dict(base=tensor(F16, 4, 95)), N.TTS_INVALID, "base: dimension 1 is 95"),
    ("tts_lora_add", lora_args, dict(a=tensor(F16, 3, 64, 16)), N.TTS_INVALID, "a: dimension 1 is 64"),
    ("tts_lora_add", lora_args, dict(a=tensor(F16, 3, 16, 64, stride=(1024, 1, 16))), N.TTS_INVALID, "a: its last dimension"),
    ("tts_lora_add", lora_args, dict(b=tensor(F16, 3, 96, 16, stride=(1536, 1, 96))), N.TTS_INVALID, "b: its last dimension"),
    ("tts_lora_add", lora_args, dict(a=tensor(F16, 3, 2000, 64), b=tensor(F16, 3, 96, 2000)), N.TTS_UNSUPPORTED, "a rank of 2000"),
    ("tts_lora_add", lora_args, dict(a=tensor(F16, 3, 0, 64), b=tensor(F16, 3, 96, 0)), N.TTS_INVALID, "empty"),
    ("tts_lora_add", lora_args, dict(ids=tensor(I32, 3)), N.TTS_INVALID, "ids: dimension 0 is 3"),
    ("tts_lora_add", lora_args, dict(scales=tensor(F16, 3)), N.TTS_INVALID, "scales is f16"),
    ("tts_lora_add", lora_args, dict(out=tensor(F16, 4, 96, ptr=FAR[0] + 2)), N.TTS_INVALID, "out shares memory with base"),
    ("tts_lora_add", lora_args, dict(out=tensor(F16, 4, 96, ptr=FAR[1] + 64)), N.TTS_INVALID, "out shares memory with x"),
    ("tts_lora_add", lora_args, dict(bytes=0), N.TTS_INVALID, "the workspace has 0 bytes"),
]


@pytest.mark.parametrize("entry,args,change,status,says", REFUSALS, ids=[f"{r[0][4:]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refused_calls(entry, args, change, status, says):
    assert getattr(N.lib(), entry)(*args(**change)) == status
    assert says in N.lib().tts_last_error().decode()


def test_experts_of_more_workgroups_than_a_launch_has_are_refused():
    # tables of one matrix for all experts: 4096 slots in groups of their own, 2^24 columns
    size, L = ctypes.c_size_t(), N.lib()
    wide = dict(x=tensor(BF16, 4096, 8), ids=tensor(I32, 4096, 1))
    up = tensor(BF16, 4096, 8, 1 << 24, stride=(0, 1 << 24, 1))
    down = tensor(BF16, 4096, 1 << 24, 8, stride=(0, 8, 1))
    assert L.tts_moe_experts_workspace(wide["x"], wide["ids"], up, down, 0, ctypes.byref(size)) == N.TTS_UNSUPPORTED
    assert "more workgroups" in L.tts_last_error().decode()
    up, down = tensor(BF16, 4096, 8, 8, stride=(0, 8, 1)), tensor(BF16, 4096, 8, 1 << 24, stride=(0, 1 << 24, 1))
    assert L.tts_moe_experts_workspace(wide["x"], wide["ids"], up, down, 0, ctypes.byref(size)) == N.TTS_UNSUPPORTED
    few = dict(x=tensor(BF16, 64, 8), ids=tensor(I32, 64, 1))
    assert L.tts_moe_experts_workspace(few["x"], few["ids"], up, down, 0, ctypes.byref(size)) == N.TTS_OK


def test_calls_for_no_tokens_do_nothing():
    L = N.lib()
    assert L.tts_moe_route(*route_args(logits=tensor(BF16, 0, 16, ptr=0), ids=tensor(I32, 0, 2, ptr=0), weights=tensor(F32, 0, 2, ptr=0))) == 0
    assert L.tts_moe_experts(*experts_args(x=tensor(BF16, 0, 64, ptr=0), ids=tensor(I32, 0, 2, ptr=0), weights=tensor(F32, 0, 2, ptr=0), out=tensor(BF16, 0, 64, ptr=0), work=None, bytes=0)) == 0
    assert L.tts_lora_add(*lora_args(base=tensor(F16, 0, 96, ptr=0), x=tensor(F16, 0, 64, ptr=0), ids=tensor(I32, 0, ptr=0), out=tensor(F16, 0, 96, ptr=0), work=None, bytes=0)) == 0


def test_adapters_of_more_rows_than_a_grid_has_are_refused():
    size, L = ctypes.c_size_t(), N.lib()
    assert L.tts_lora_add_workspace(tensor(BF16, 2097120, 64), tensor(BF16, 8, 64, 16), ctypes.byref(size)) == N.TTS_OK
    assert L.tts_lora_add_workspace(tensor(BF16, 2097121, 64), tensor(BF16, 8, 64, 16), ctypes.byref(size)) == N.TTS_UNSUPPORTED
    assert "2097121 rows" in L.tts_last_error().decode()


def test_columns_of_one_buffer_are_told_apart():
    # out and x side by side in rows of one buffer do not overlap; moved by one element they do
    x = tensor(F16, 4, 64, stride=(256, 1), ptr=FAR[1] + 2 * 96)
    for out, fine in ((tensor(F16, 4, 96, stride=(256, 1), ptr=FAR[1]), True), (tensor(F16, 4, 96, stride=(256, 1), ptr=FAR[1] + 2), False),
                      (tensor(F16, 4, 96, stride=(256, 1), ptr=FAR[1] + 2 * 160), True), (tensor(F16, 4, 96, stride=(256, 1), ptr=FAR[1] + 2 * 257), False)):
        # (the workspace is refused next)
        N.lib().tts_lora_add(*lora_args(x=x, out=out, bytes=0))
        assert ("workspace" in N.lib().tts_last_error().decode()) == fine


def test_python_arguments_are_checked_without_a_gpu():
    cpu = torch.zeros(4, 16)
    with pytest.raises(TypeError, match="GPU memory"):
        ops.moe_route(cpu, 2)
    with pytest.raises(TypeError, match="GPU memory"):
        ops.moe_experts(cpu, cpu, cpu, cpu, cpu)
    with pytest.raises(TypeError, match="not a tensor"):
        ops.lora_add([1.0], cpu, cpu, cpu, cpu)


def test_workspaces_hold_what_the_kernels_put_there():
    size = ctypes.c_size_t()
    L = N.lib()
    assert L.tts_moe_experts_workspace(tensor(BF16, 5, 64), tensor(I32, 5, 3), tensor(BF16, 8, 64, 200), tensor(BF16, 8, 100, 40), 1, ctypes.byref(size)) == 0
    assert size.value >= 15 * 104 * 4 + 15 * 40 * 4
    assert L.tts_lora_add_workspace(tensor(BF16, 5, 64), tensor(BF16, 8, 64, 12), ctypes.byref(size)) == 0
    assert size.value >= 5 * 16 * 4


# ---------------------------------------------------------------------------------------------------------------- the router
def route_exact(logits, k, scoring, bias, renormalize, scale):
    """ids and weights of the definition, a row at a time in 64 bits."""
    rows = logits.double().cpu().numpy()
    add = None if bias is None else bias.double().cpu().numpy()
    ids, weights = np.full((len(rows), k), -1, np.int32), np.zeros((len(rows), k))
    for t, l in enumerate(rows):
        with np.errstate(all="ignore"):
            most = np.nanmax(l) if not np.isnan(l).all() else np.nan
            e = np.exp(l - most)
            s = 1.0 / (1.0 + np.exp(-l)) if scoring == "sigmoid" else e / np.nansum(e)
            c = l if add is None else s + add  # (both scores rise with the logit)
        able = [i for i in range(len(l)) if l[i] > -np.inf and c[i] > -np.inf]
        chosen = sorted(able, key=lambda i: (-c[i], i))[:k]
        if not chosen:
            continue
        with np.errstate(all="ignore"):
            w = np.where(s[chosen] == 0, 0.0, s[chosen] / (s[chosen].sum() if renormalize else 1.0) * scale)
        ids[t, :len(chosen)] = chosen
        weights[t, :len(chosen)] = np.nan if np.isnan(l).any() else w
    return ids, weights


def check_route(logits, k, scoring="softmax", bias=None, renormalize=True, scale=1.0):
    ids, weights = ops.moe_route(logits, k, scoring=scoring, bias=bias, renormalize=renormalize, scale=scale)
    want, exact = route_exact(logits, k, scoring, bias, renormalize, scale)
    assert np.array_equal(ids.cpu().numpy(), want)
    got = weights.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(exact))
    # the difference from the maximum (half a step of up to 2 |l|), the exponential (2 steps), a sum of up to E of them (E / 2 halves at
    # most, log2 E for the tree plus E / lanes in turn: 64 covers 1024 experts), a division or two and the scale
    lo = np.nan_to_num(np.abs(logits.double().cpu().numpy()), posinf=0.0).max(initial=0.0) if logits.numel() else 0.0
    lim = U * (2 * min(lo, 200.0) + 64 + 12)
    fine = ~np.isnan(exact)
    assert np.all(np.abs(got - exact)[fine] <= lim * np.abs(exact)[fine] + 2.0 ** -126)


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,experts,k,dtype", [(1, 128, 8, "bf16"), (1, 1, 1, "fp32"), (3, 8, 2, "fp16"), (5, 60, 4, "bf16"), (37, 64, 64, "fp32"), (19, 65, 6, "fp32"), (130, 129, 8, "fp32"),
                                                    (33, 256, 9, "bf16"), (7, 257, 10, "fp32"), (6, 512, 8, "fp16"), (9, 1000, 33, "fp32"), (4, 1024, 64, "bf16"), (2050, 16, 1, "fp32")])
@pytest.mark.parametrize("scoring,bias,renormalize", [("softmax", False, True), ("softmax", False, False), ("softmax", True, True), ("sigmoid", False, True), ("sigmoid", True, False)])
def test_route(tokens, experts, k, dtype, scoring, bias, renormalize):
    logits = gpu(tokens, experts, seed=tokens + experts, scale=2.0, dtype=dtype)
    check_route(logits, k, scoring, gpu(experts, seed=5, scale=0.1) if bias else None, renormalize, 1.0 if renormalize else 2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [24, 200, 700])
def test_route_ties_masks_and_nan(experts, scoring, bias):
    logits = gpu(12, experts, seed=3, scale=2.0, dtype="bf16").float()
    logits[0] = 0.5                                # all the same
    logits[1] = float("-inf")                      # a mask that leaves nothing
    logits[2, 3:] = float("-inf")                  # ... fewer than k
    logits[3, ::2] = float("-inf")
    logits[4, 7] = float("nan")
    logits[5] = float("nan")
    logits[6] = torch.finfo(torch.float32).min     # a mask of the type's lowest value
    logits[6, 5] = 1.0
    logits[7] = torch.finfo(torch.float32).min
    logits[8] *= 40.0                              # scores that run into 0 and 1
    logits[9] = torch.where(torch.arange(experts, device="cuda") % 3 == 0, 1.0, 0.25)
    add = (torch.arange(experts, device="cuda") % 4).float() * 0.25 if bias else None
    check_route(logits, 6, scoring, add)


@pytest.mark.gpu
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("experts", [40, 250, 600])
def test_route_scores_that_32_bits_cannot_tell_apart(scoring, experts):
    # biases that bring the scores to the same value but for some 2^-30 of it, rising with the expert in half of the rows' experts
    logits = gpu(1, experts, seed=11, scale=1.5)
    l = logits[0].double()
    s = torch.sigmoid(l) if scoring == "sigmoid" else torch.softmax(l, 0)
    bias = (1.5 - s).float()                # rounded: s + bias is 1.5 but for half a step of it
    check_route(logits, 9, scoring, bias)
    many = logits.repeat(70, 1)
    many[::3, 5] += 0.75                    # some rows have one that stands out
    check_route(many, 9, scoring, bias)
    check_route(many, 9, scoring, torch.full_like(bias, 1e6))
    bias[3] = float("inf")                  # always chosen
    bias[4], bias[6] = float("-inf"), float("nan")
    many[:, 7] = float("-inf")
    check_route(many, 1, scoring, bias)
    check_route(many, 4, scoring, bias)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("experts", [24, 200, 700])
@pytest.mark.parametrize("bias", [False, True])
def test_route_sigmoids_below_32_bits_keep_their_ratio(bias, experts, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(experts)
    logits = torch.empty(9, experts, device="cuda").uniform_(-200.0, -90.0, generator=g)
    for i, l in enumerate((-20.0, -86.0, -100.0, -103.0, -110.0, -600.0)):  # two of them, one apart, and others far below
        logits[i] = -690.0
        logits[i, 3], logits[i, 11] = l, l - 1.0
    logits[6, 4] = 2.0                              # one that is not small
    logits[7] = torch.finfo(TYPES[dtype]).min       # a mask that leaves nothing: no weights
    logits[8] = 0.25 - (torch.arange(experts, device="cuda") % 7).float()
    logits = logits.to(TYPES[dtype])
    add = (torch.arange(experts, device="cuda") % 5 == 3).float() if bias else None  # (3 among them, and others of lower scores)
    check_route(logits, 2, "sigmoid", add)
    check_route(logits, 6, "sigmoid", add, scale=2.5)
    check_route(logits, 6, "sigmoid", add, renormalize=False)


@pytest.mark.gpu
@pytest.mark.parametrize("experts", [24, 200, 700])
def test_route_a_bias_that_chooses_far_below_the_largest_logit(experts):
    logits = gpu(5, experts, seed=experts, scale=2.0)
    logits[0, 1] = 95.0
    logits[1, 1], logits[2, 1] = 120.0, 400.0
    logits[3, 1] = 1e30                             # ... so far that nothing of the others is left
    add = torch.where(torch.arange(experts, device="cuda") % 2 == 0, 4.0, 0.0)
    check_route(logits, 8, "softmax", add)
    check_route(logits, 8, "softmax", add, renormalize=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("experts", [24, 200, 700])
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("bias,renormalize", [(False, True), (False, False), (True, True), (True, False)])
def test_route_infinite_logits(bias, renormalize, scoring, experts, dtype):
    # softmax of a row with one is NaN: NaN weights, of the experts that the limit of ever larger logits picks
    logits = gpu(7, experts, seed=experts + 1, scale=2.0, dtype=dtype)
    inf = float("inf")
    logits[0, 5] = inf
    logits[1, 5], logits[1, 20], logits[1, 7] = inf, inf, -inf
    logits[2] = inf
    logits[3], logits[3, 9] = -inf, inf
    logits[4, 6], logits[4, 9], logits[4, 2] = torch.finfo(TYPES[dtype]).max, inf, torch.finfo(TYPES[dtype]).min
    logits[5, 6], logits[5, 9] = float("nan"), inf
    add = (torch.arange(experts, device="cuda") % 4).float() * 0.25 if bias else None
    ids, weights = (t.cpu().numpy() for t in ops.moe_route(logits, 4, scoring=scoring, bias=add, renormalize=renormalize))
    for t, l in enumerate(logits.double().cpu().numpy()):
        if scoring == "sigmoid":
            with np.errstate(all="ignore"):
                s = 1.0 / (1.0 + np.exp(-l))
        elif np.isposinf(l).any():
            s = np.isposinf(l) / np.isposinf(l).sum()
        else:
            s = np.exp(l - l.max()) / np.exp(l - l.max()).sum()
        c = s + add.double().cpu().numpy() if bias else l
        chosen = sorted((i for i in range(experts) if l[i] > -np.inf), key=lambda i: (-c[i], i))[:4]
        assert list(ids[t]) == chosen + [-1] * (4 - len(chosen)), f"row {t}"
        if np.isnan(l).any() or (scoring == "softmax" and np.isposinf(l).any()):
            assert np.isnan(weights[t, :len(chosen)]).all() and not weights[t, len(chosen):].any(), f"row {t}"
        else:
            w = s[chosen] / (s[chosen].sum() if renormalize else 1.0)
            # arguments of an exponential up to 13 (or one past 88, whose exponential is below 2^-126), and as in check_route
            assert np.all(np.abs(weights[t, :len(chosen)] - w) <= U * (2 * 13 + 64 + 12) * w + 2.0 ** -126), f"row {t}"


@pytest.mark.gpu
def test_route_of_columns_of_a_wider_buffer():
    wide = gpu(21, 300, seed=8, dtype="bf16")
    check_route(wide[:, 7:107], 5)
    check_route(wide[:, :40], 5, "sigmoid")
    a = ops.moe_route(wide[:, 7:107], 5)
    b = ops.moe_route(wide[:, 7:107].contiguous(), 5)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.gpu
def test_route_of_more_tokens_than_one_grid():
    # 16 lanes a token: 2^28 of them are 2^32 lanes, more than a launch may have
    tokens = 2 ** 28 + 19
    logits = torch.zeros(tokens, 1, dtype=torch.bfloat16, device="cuda")
    logits[-1] = float("-inf")
    logits[2 ** 27 + 3] = float("nan")      # (a NaN is never chosen)
    ids, weights = ops.moe_route(logits, 1)
    for t in (2 ** 27 + 3, -1):
        assert int(ids[t]) == -1 and float(weights[t]) == 0.0
        ids[t], weights[t] = 0, 1.0
    assert not ids.any() and bool((weights == 1.0).all())


# ---------------------------------------------------------------------------------------------------------------- the experts
def activation_exact(name, v):
    if name == "silu":
        return v * torch.special.expit(v)
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    return v * torch.special.expit(2.0 * (2.0 / np.pi) ** 0.5 * (v + 0.044715 * v ** 3))


def experts_exact(x, ids, weights, w_up, w_down, s_up, s_down, activation, gated):
    """The layer in 64 bits, and how far 32-bit sums in any order, the 16-bit parts of h and the final rounding can take it."""
    T, k = ids.shape
    inner, outputs = w_down.shape[1], w_down.shape[2]
    H = x.shape[1]
    dtype = "bf16" if x.dtype == torch.bfloat16 else "fp16"
    part = 2.0 ** -15 if dtype == "bf16" else 2.0 ** -20  # of h's two parts together, with a factor of two to spare
    y, err = torch.zeros(T, outputs, dtype=torch.float64, device="cuda"), torch.zeros(T, outputs, dtype=torch.float64, device="cuda")
    for t, j in itertools.product(range(T), range(k)):
        e = int(ids[t, j])
        if not 0 <= e < w_up.shape[0]:
            continue
        row, up, down = x[t].double(), w_up[e].double(), w_down[e].double()
        if s_up is not None:
            up, down = up * s_up[e].double(), down * s_down[e].double()
        v, dv = row @ up, (H + 2) * U * (row.abs() @ up.abs())
        # the slopes of the activations are at most 1.13; a few roundings of their own: 16, and of what is exponentiated
        g, dg = v[:inner], dv[:inner]
        f = activation_exact(activation, g)
        df = 1.13 * dg + (16 + 4 * g.abs()) * U * f.abs() + 2.0 ** -120
        h, dh = (f * v[inner:], df * v[inner:].abs() + f.abs() * dv[inner:] + df * dv[inner:]) if gated else (f, df)
        dh = dh + (part + U) * h.abs() + 2.0 ** -30 * h.abs().max() * part
        w = abs(float(weights[t, j]))
        y[t] += float(weights[t, j]) * (h @ down)
        err[t] += w * (dh @ down.abs() + (2 * inner + k + 4) * U * (h.abs() @ down.abs()))
    return y, err + half(dtype) * (y.abs() + err) + smallest(dtype)


def make_experts(T, k, E, H, I, O, dtype="bf16", weights=None, order_up="in", order_down="in", gated=True, seed=0):
    def table(inputs, outputs, order, s):
        shape = (E, outputs, inputs) if order == "in" else (E, inputs, outputs)
        if weights == "int8":
            g = torch.Generator(device="cuda")
            g.manual_seed(s)
            w, sc = torch.randint(-128, 128, shape, generator=g, dtype=torch.int8, device="cuda"), gpu(E, outputs, seed=s + 1).abs() * inputs ** -0.5 / 73 + 1e-5
        else:
            w, sc = gpu(*shape, seed=s, scale=inputs ** -0.5, dtype=dtype), None
        return (w.transpose(1, 2) if order == "in" else w), sc
    w_up, s_up = table(H, (2 if gated else 1) * I, order_up, seed + 10)
    w_down, s_down = table(I, O, order_down, seed + 20)
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 30)
    ids = torch.rand(T, E, generator=g, device="cuda").topk(k, dim=1).indices.int()
    shares = torch.rand(T, k, generator=g, device="cuda") / k
    return dict(x=gpu(T, H, seed=seed + 40, dtype=dtype), ids=ids, weights=shares, w_up=w_up, w_down=w_down, s_up=s_up, s_down=s_down, gated=gated)


def check_experts(a, activation="silu", out=None):
    got = ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"], s_up=a["s_up"], s_down=a["s_down"], activation=activation, gated=a["gated"], out=out)
    want, lim = experts_exact(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"], a["s_up"], a["s_down"], activation, a["gated"])
    off = (got.double() - want).abs()
    assert bool((off <= lim).all()), f"off by {(off / lim).max().item():.2f} of what is allowed"
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("order_up,order_down", [("in", "in"), ("out", "out"), ("in", "out"), ("out", "in")])
@pytest.mark.parametrize("dtype,weights", [("bf16", None), ("fp16", None), ("bf16", "int8"), ("fp16", "int8")])
@pytest.mark.parametrize("T,k,E,H,I,O,gated", [(1, 2, 8, 128, 64, 128, True), (3, 2, 4, 200, 72, 136, True), (17, 3, 5, 96, 160, 264, False), (5, 2, 6, 333, 75, 131, True), (2, 1, 3, 16, 16, 16, True),
                                               (40, 4, 4, 70, 129, 65, False)])
def test_experts(T, k, E, H, I, O, gated, dtype, weights, order_up, order_down):
    check_experts(make_experts(T, k, E, H, I, O, dtype, weights, order_up, order_down, gated, seed=T + I))


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["in", "out"])
def test_experts_of_the_narrowest_layer(order):
    check_experts(make_experts(2, 1, 3, 8, 8, 8, "bf16", None, order, order, True))
    check_experts(make_experts(3, 2, 3, 9, 11, 10, "fp16", None, order, order, False))


@pytest.mark.gpu
@pytest.mark.parametrize("T,k,E,H,I,O", [(1, 8, 32, 2048, 768, 2048), (16, 2, 4, 1024, 1536, 1032), (70, 2, 3, 512, 256, 520)])
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh", "relu"])
def test_experts_of_ordinary_sizes(T, k, E, H, I, O, activation):
    check_experts(make_experts(T, k, E, H, I, O, order_up="in", order_down="out"), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("I,O", [(2072, 64), (24, 4100)])
@pytest.mark.parametrize("dtype,weights,order", [("bf16", None, "in"), ("fp16", None, "out"), ("bf16", "int8", "in"), ("fp16", "int8", "out")])
def test_experts_with_several_slabs_per_workgroup(I, O, dtype, weights, order):
    a = make_experts(40, 2, 64, 40, I, O, dtype, weights, order, order)
    a["ids"][:35, 0] = 7                    # and an expert whose rows take several turns
    check_experts(a)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [256, 100])      # up to 64, and up to 32, rows of an expert at once
@pytest.mark.parametrize("H,I,O,gated", [(808, 520, 1032, True), (72, 1544, 72, True), (72, 72, 3112, True), (72, 1032, 72, False)])
@pytest.mark.parametrize("dtype,weights", [("bf16", None), ("fp16", None), ("bf16", "int8"), ("fp16", "int8")])
@pytest.mark.parametrize("order", ["in", "out"])
def test_experts_of_many_rows_in_wide_tiles(order, dtype, weights, H, I, O, gated, T):
    a = make_experts(T, 5, 64, H, I, O, dtype, weights, order, order, gated, seed=T)
    a["ids"][:70, 0] = 7                        # an expert whose rows take several turns
    got = ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"], s_up=a["s_up"], s_down=a["s_down"], gated=gated)
    rows = [0, 15, 16, 17, 31, 32, 33, 63, 64, 69, 70, T - 2, T - 1]
    part = {n: a[n][rows] for n in ("x", "ids", "weights")}
    want, lim = experts_exact(**part, w_up=a["w_up"], w_down=a["w_down"], s_up=a["s_up"], s_down=a["s_down"], activation="silu", gated=gated)
    off = (got[rows].double() - want).abs()
    assert bool((off <= lim).all()), f"off by {(off / lim).max().item():.2f} of what is allowed"
    # all rows, against calls of a few tokens
    for at in range(0, T, 50):
        few = [a[n][at:at + 50] for n in ("x", "ids", "weights")]
        again = ops.moe_experts(*few, a["w_up"], a["w_down"], s_up=a["s_up"], s_down=a["s_down"], gated=gated)
        # (both within `lim` of the same values, and no row's `lim` is twice the largest of the rows above: these are alike)
        assert bool(((got[at:at + 50].double() - again.double()).abs() <= 4 * lim.max()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts_ids_outside_repeated_and_one_for_all(dtype):
    a = make_experts(50, 3, 6, 128, 96, 128, dtype)
    a["ids"][0] = -1                        # a row with no expert: zeros
    a["ids"][1, 1] = 6
    a["ids"][2, 2] = -2 ** 31
    a["ids"][3, 0] = 2 ** 31 - 1
    a["ids"][4] = a["ids"][4, 0].clone()    # the same expert three times
    got = check_experts(a)
    assert not got[0].any()
    a["ids"][:] = 3                         # 150 rows of one expert
    check_experts(a)
    a["ids"][:] = -1
    assert not check_experts(a).any()


@pytest.mark.gpu
def test_experts_with_more_experts_than_slots_and_back():
    for T, E in ((3, 64), (3, 4), (1, 3), (2, 2), (40, 100), (50, 101)):  # (with more than 64 slots: found by all wavefronts together)
        a = make_experts(T, 2, E, 64, 64, 64)
        a["ids"][0, 1] = a["ids"][T - 1, 0]  # one expert in two rows
        check_experts(a)


@pytest.mark.gpu
def test_experts_fill_the_slots():
    a = make_experts(1024, 4, 16, 64, 32, 64)
    got = ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"])
    rows = [0, 1, 511, 777, 1023]
    part = a | {"x": a["x"][rows], "ids": a["ids"][rows], "weights": a["weights"][rows]}
    want, lim = experts_exact(*(part[n] for n in ("x", "ids", "weights", "w_up", "w_down", "s_up", "s_down")), "silu", True)
    assert bool(((got[rows].double() - want).abs() <= lim).all())


@pytest.mark.gpu
def test_experts_fp16_hidden_values_past_fp16():
    # h of a hundred thousands, weighted down again: the result fits fp16, h does not
    a = make_experts(4, 2, 3, 64, 64, 64, "fp16")
    a["x"] *= 300
    a["weights"] *= 1e-3
    check_experts(a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_experts_infinities_and_nan_stay_where_they_are(dtype):
    a = make_experts(20, 2, 5, 100, 76, 92, dtype)
    a["ids"][:, 0], a["ids"][:, 1] = 1, 2
    a["ids"][5] = torch.tensor([3, 4], dtype=torch.int32, device="cuda")
    want = ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"])
    a["x"][7, 3], a["x"][8, 99] = float("nan"), float("inf")
    a["w_up"][3, 50, 20] = float("inf")     # row 5's expert
    a["w_down"][0] = float("nan")           # nobody's
    got = ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"])
    others = [t for t in range(20) if t not in (5, 7, 8)]
    assert torch.equal(got[others], want[others])
    assert got[7].isnan().all() and not got[8].isfinite().any() and not got[5].isfinite().any()


@pytest.mark.gpu
def test_experts_strided_in_place_and_a_whole_buffer_behind():
    a = make_experts(9, 2, 4, 96, 64, 96)
    want = check_experts(a)
    wide = torch.full((12, 160), 7.0, dtype=torch.bfloat16, device="cuda")
    wide[:9, 32:128] = a["x"]
    x = wide[:9, 32:128]
    ids = torch.full((9, 5), 99, dtype=torch.int32, device="cuda")
    ids[:, 1:3] = a["ids"]
    shares = torch.zeros(9, 7, device="cuda")
    shares[:, 4:6] = a["weights"]
    out = ops.moe_experts(x, ids[:, 1:3], shares[:, 4:6], a["w_up"], a["w_down"], out=x)   # out is x
    assert out is x and torch.equal(x, want)
    wide[:9, 32:128] = 7.0
    assert bool((wide == 7.0).all())        # nothing beside it was touched


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["in", "out"])
def test_experts_past_32_bits(order):
    # the second expert begins 2^31 elements behind the first
    H, I, far = 64, 64, 2 ** 31 + 8
    a = make_experts(3, 2, 2, H, I, H, weights="int8", order_up=order, order_down=order)
    big = torch.zeros(far + H * 2 * I, dtype=torch.int8, device="cuda")
    for name in ("w_up", "w_down"):
        w = a[name]
        shape, inner = w.shape, w.stride()[1:]
        view = torch.as_strided(big, shape, (far, *inner))
        view.copy_(w)
        b = a | {name: view}
        assert torch.equal(check_experts(b), check_experts(a))


# ---------------------------------------------------------------------------------------------------------------- the adapters
def lora_exact(base, x, a, b, ids, scales):
    dtype = "bf16" if x.dtype == torch.bfloat16 else "fp16"
    part = 2.0 ** -15 if dtype == "bf16" else 2.0 ** -20
    y, err = base.double(), torch.zeros(base.shape, dtype=torch.float64, device="cuda")
    K, r = x.shape[1], a.shape[1]
    for n in range(a.shape[0]):
        rows = torch.nonzero(ids == n)[:, 0]
        if not len(rows):
            continue
        s = 1.0 if scales is None else float(scales[n])
        xd, ad, bd = x[rows].double(), a[n].double().t(), b[n].double().t()
        v, dv = s * (xd @ ad), abs(s) * (K + 40) * U * (xd.abs() @ ad.abs())
        dv = dv + (part + 2 * U) * v.abs() + 2.0 ** -30 * part * v.abs().amax(dim=1, keepdim=True)
        y[rows] += v @ bd
        err[rows] += dv @ bd.abs() + (2 * r + 4) * U * (v.abs() @ bd.abs() + y[rows].abs())
    return y, err + half(dtype) * (y.abs() + err) + smallest(dtype)


def make_lora(T, K, O, r, n, dtype="bf16", runs=1, plain=0.2, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    ids = torch.randint(0, n, (-(-T // runs),), generator=g, dtype=torch.int32, device="cuda")
    ids = torch.where(torch.rand(ids.shape, generator=g, device="cuda") < plain, torch.full_like(ids, -1), ids).repeat_interleave(runs)[:T].contiguous()
    return dict(base=gpu(T, O, seed=seed + 1, dtype=dtype), x=gpu(T, K, seed=seed + 2, dtype=dtype), a=gpu(n, r, K, seed=seed + 3, scale=K ** -0.5, dtype=dtype),
                b=gpu(n, O, r, seed=seed + 4, scale=r ** -0.5, dtype=dtype), ids=ids, scales=gpu(n, seed=seed + 5) + 1.5)


def check_lora(a, **kw):
    base = a["base"].clone()
    want, lim = lora_exact(base, a["x"], a["a"], a["b"], a["ids"], a["scales"])
    got = ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"], scales=a["scales"], **kw)
    off = (got.double() - want).abs()
    assert bool((off <= lim).all()), f"off by {(off / lim).max().item():.2f} of what is allowed"
    alone = (a["ids"] < 0) | (a["ids"] >= a["a"].shape[0])
    assert torch.equal(got[alone].view(torch.int16), base[alone].view(torch.int16))
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,K,O,r,n,runs", [(1, 64, 96, 16, 3, 1), (1, 4096, 512, 8, 2, 1), (16, 128, 256, 16, 16, 1), (37, 333, 515, 12, 5, 1), (64, 1024, 768, 16, 64, 1), (130, 200, 300, 64, 7, 1),
                                            (5, 7, 3, 1, 2, 1), (3, 1, 1, 1, 1, 1), (33, 96, 130, 33, 4, 3), (20, 64, 80, 128, 3, 2), (9, 70, 264, 200, 2, 1), (4, 40, 40, 1024, 2, 1),
                                            (1100, 96, 130, 16, 6, 90), (1037, 130, 96, 24, 9, 1), (2048, 64, 512, 64, 3, 700), (1500, 257, 77, 130, 4, 333)])
def test_lora(T, K, O, r, n, runs, dtype):
    check_lora(make_lora(T, K, O, r, n, dtype, runs, seed=T + r))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("r", [2, 4, 7])
@pytest.mark.parametrize("T,O,runs", [(20, 4096, 1), (20, 515, 1), (1100, 1040, 90), (1100, 515, 1)])
def test_lora_of_ranks_below_an_octet(T, O, runs, r, dtype):
    check_lora(make_lora(T, 96, O, r, 5, dtype, runs, seed=T + O + r))


@pytest.mark.gpu
@pytest.mark.parametrize("T", [19, 1300])
def test_lora_ids_and_no_scales(T):
    a = make_lora(T, 96, 160, 16, 4, plain=0.0)
    a["ids"][1], a["ids"][2], a["ids"][3] = 4, -2 ** 31, 2 ** 31 - 1
    a["scales"] = None
    check_lora(a)
    a["ids"][:] = 2
    check_lora(a)
    a["ids"][:] = -1
    check_lora(a)
    spaced = torch.randint(0, 4, (T, 3), dtype=torch.int32, device="cuda")
    a["ids"] = spaced[:, 1]                 # a stride of 3
    check_lora(a)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [21, 1040])
def test_lora_in_place_in_columns_of_a_buffer(T):
    a = make_lora(T, 64, 96, 8, 3)
    want = check_lora(a)
    wide = torch.full((T, 256), 3.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 16:112], wide[:, 160:224] = a["base"], a["x"]
    y, x = wide[:, 16:112], wide[:, 160:224]
    assert ops.lora_add(y, x, a["a"], a["b"], a["ids"], scales=a["scales"], out=y) is y
    assert torch.equal(y, want) and torch.equal(x, a["x"])
    wide[:, 16:112], wide[:, 160:224] = 3.0, 3.0
    assert bool((wide == 3.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [32, 1088])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_lora_of_one_request_does_not_reach_another(T, dtype):
    a = make_lora(T, 100, 140, 20, 4, dtype, plain=0.1)
    a["ids"][3] = -1
    want = check_lora(a)
    a["a"][1, 3, 5] = float("inf")
    a["b"][2, 7] = float("nan")
    a["x"][(a["ids"] < 0).nonzero()[0, 0]] = float("nan")   # a row without an adapter
    got = ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"], scales=a["scales"])
    fine = (a["ids"] != 1) & (a["ids"] != 2)
    assert torch.equal(got[fine], want[fine])
    two = a["ids"] == 2
    assert got[two][:, 7].isnan().all() and torch.equal(got[two][:, 8:], want[two][:, 8:])
    assert not got[a["ids"] == 1].isfinite().any(dim=1).any()


@pytest.mark.gpu
def test_lora_fp16_inner_values_past_fp16():
    a = make_lora(6, 64, 64, 16, 3, "fp16")
    a["x"] *= 3000
    a["a"] *= 30
    a["b"] *= 1e-3
    check_lora(a)


@pytest.mark.gpu
def test_lora_past_32_bits():
    far = 2 ** 31 + 8
    a = make_lora(6, 64, 64, 8, 2, plain=0.0)
    want = check_lora(a)
    big = torch.zeros(far + 64 * 64, dtype=torch.bfloat16, device="cuda")
    for name in ("a", "b"):
        view = torch.as_strided(big, a[name].shape, (far, *a[name].stride()[1:]))
        view.copy_(a[name])
        assert torch.equal(check_lora(a | {name: view}), want)


# ---------------------------------------------------------------------------------------------------------------- how they are called
@pytest.mark.gpu
def test_gradients_are_refused_where_they_are_recorded():
    a = make_lora(4, 64, 64, 8, 2)
    a["a"].requires_grad_()
    with pytest.raises(NotImplementedError, match="no backward"):
        ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"])
    with torch.no_grad():
        ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"])
    logits = gpu(3, 8).requires_grad_()
    with pytest.raises(NotImplementedError, match="no backward"):
        ops.moe_route(logits, 2)


@pytest.mark.gpu
def test_forward_mode_derivatives_are_refused():
    from torch.autograd import forward_ad as fwd

    a, e, logits = make_lora(4, 64, 64, 8, 2), make_experts(2, 2, 3, 64, 64, 64), gpu(3, 8)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for under in (torch.enable_grad, torch.no_grad):  # (no_grad is of the backward mode)
            with under():
                with pytest.raises(NotImplementedError, match="logits has a forward-mode tangent"):
                    ops.moe_route(dual(logits), 2)
                with pytest.raises(NotImplementedError, match="weights has a forward-mode tangent"):
                    ops.moe_experts(e["x"], e["ids"], dual(e["weights"]), e["w_up"], e["w_down"])
                with pytest.raises(NotImplementedError, match="scales has a forward-mode tangent"):
                    ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"], scales=dual(a["scales"]))
                with pytest.raises(NotImplementedError, match="out has a forward-mode tangent"):
                    ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"], out=dual(torch.empty_like(a["base"])))
        inside = ops.moe_route(logits, 2)   # without one: as ever
    assert all(torch.equal(x, y) for x, y in zip(inside, ops.moe_route(logits, 2)))


@pytest.mark.gpu
@pytest.mark.parametrize("ordinary", [True, False])
def test_autograd_notices_that_out_was_written(ordinary, monkeypatch):
    if not ordinary:  # the calls that the launch extension leaves to Python
        monkeypatch.setattr(ops, "_fast", False)
    a, e = make_lora(4, 64, 64, 8, 2), make_experts(2, 2, 3, 64, 64, 64)
    for write in (lambda out: ops.lora_add(out, a["x"], a["a"], a["b"], a["ids"], out=out), lambda out: ops.moe_experts(e["x"], e["ids"], e["weights"], e["w_up"], e["w_down"], out=out[:2])):
        factor = torch.ones(64, device="cuda", requires_grad=True)
        saved = a["base"].clone()
        y = (saved * factor).sum()
        write(saved)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
    with torch.inference_mode():
        out = torch.empty_like(a["base"])
        assert ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"], out=out) is out
    version = a["base"]._version
    with pytest.raises(ValueError):         # a refused call has written nothing
        ops.lora_add(a["base"], a["x"], a["a"], a["b"], a["ids"].float(), out=a["base"])
    assert a["base"]._version == version


@pytest.mark.gpu
def test_python_arguments_are_checked():
    a = make_experts(2, 2, 3, 64, 64, 64)
    call = lambda **kw: ops.moe_experts(**({k: v for k, v in a.items()} | kw))  # noqa: E731
    with pytest.raises(ValueError, match="activation is 'tanh'"):
        call(activation="tanh")
    with pytest.raises(ValueError, match="int64"):
        call(ids=a["ids"].long())
    with pytest.raises(TypeError, match="GPU memory"):
        call(weights=a["weights"].cpu())
    with pytest.raises(NotImplementedError, match="f16 and bf16"):
        call(x=a["x"].float())
    with pytest.raises(ValueError, match="neither its inputs"):
        call(w_up=a["w_up"].repeat_interleave(2, dim=2)[:, :, ::2])
    with pytest.raises(ValueError, match="scoring"):
        ops.moe_route(gpu(2, 8), 2, scoring="tanh")
    with pytest.raises(ValueError, match="k is 0"):
        ops.moe_route(gpu(2, 8), 0)
    ids, weights = ops.moe_route(gpu(0, 8), 2)
    assert ids.shape == weights.shape == (0, 2)
    assert ops.moe_experts(a["x"][:0], a["ids"][:0], a["weights"][:0], a["w_up"], a["w_down"]).shape == (0, 64)


@pytest.mark.gpu
def test_route_refuses_more_choices_than_experts_before_it_allocates():
    logits = gpu(16384, 8)
    for k in (9, 10 ** 9, 10 ** 30):        # (a table of 10^9 choices would be 65 TB)
        with pytest.raises(ValueError, match=f"k is {k}"):
            ops.moe_route(logits, k)


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call():
    e, l = make_experts(24, 4, 8, 256, 192, 256), make_lora(70, 256, 256, 16, 9)
    first = None
    for _ in range(5):
        got = (ops.moe_experts(e["x"], e["ids"], e["weights"], e["w_up"], e["w_down"]), ops.lora_add(l["base"], l["x"], l["a"], l["b"], l["ids"], scales=l["scales"]))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


@pytest.mark.gpu
def test_two_streams_at_once():
    e = [make_experts(24, 4, 8, 256, 192, 256, seed=s) for s in (1, 2)]
    want = [check_experts(a) for a in e]
    streams = [torch.cuda.Stream() for _ in e]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, a in enumerate(e):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.moe_experts(a["x"], a["ids"], a["weights"], a["w_up"], a["w_down"]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


def decode_step(s):
    """Projection with adapters, router, experts and the residual: the projections are Triton programs of the same backend."""
    import triton
    from triton_shared_amd.examples import kernels as K

    def product(x, w, out):
        (m, k), n = x.shape, w.shape[1]
        K.matmul_tiles[(triton.cdiv(m, 128) * triton.cdiv(n, 128),)](x, w, out, m, n, k, k, 1, n, 1, n, 1, BM=128, BN=128, BK=64, GROUP_M=8)
        return out

    h = product(s["x"], s["w_proj"], s["h"])
    ops.lora_add(h, s["x"], s["a"], s["b"], s["adapter"], scales=s["scales"], out=h)
    logits = product(h, s["w_router"], s["logits"])
    s["picked"], s["shares"] = ops.moe_route(logits, 3)
    return ops.moe_experts(h, s["picked"], s["shares"], s["w_up"], s["w_down"])


def make_decode(T, seed):
    D, I, E = 256, 192, 16
    l, e = make_lora(T, D, D, 16, 5, seed=seed), make_experts(T, 3, E, D, I, D, seed=seed + 7)
    empty = lambda n: torch.empty(T, n, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    return dict(x=l["x"], w_proj=gpu(D, D, seed=1, scale=D ** -0.5, dtype="bf16"), h=empty(D), a=l["a"], b=l["b"], adapter=l["ids"], scales=l["scales"], w_router=gpu(D, E, seed=2, scale=D ** -0.5, dtype="bf16"),
                logits=empty(E), w_up=e["w_up"], w_down=e["w_down"])


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 13])
def test_a_decode_step_of_all_of_them(T):
    tsa.activate()
    s = make_decode(T, 3)
    y = decode_step(s)
    # each from what the one before it made, in 64 bits
    proj = (s["x"].double() @ s["w_proj"].double()).bfloat16()
    want, lim = lora_exact(proj, s["x"], s["a"], s["b"], s["adapter"], s["scales"])
    # (the projection's own rounding may fall to the other side: a whole step of it)
    assert bool(((s["h"].double() - want).abs() <= lim + 2 * half("bf16") * proj.double().abs()).all())
    ids, weights = route_exact(s["logits"], 3, "softmax", None, True, 1.0)
    assert np.array_equal(s["picked"].cpu().numpy(), ids) and np.allclose(s["shares"].cpu().numpy(), weights, rtol=1e-5)
    want, lim = experts_exact(s["h"], s["picked"], s["shares"], s["w_up"], s["w_down"], None, None, "silu", True)
    assert bool(((y.double() - want).abs() <= lim).all())


@pytest.mark.gpu
def test_a_decode_step_in_a_graph():
    tsa.activate()
    s, t = make_decode(7, 4), make_decode(7, 9)
    want = [decode_step(s).clone(), decode_step(t).clone()]
    inputs = [{k: s[k].clone() for k in ("x", "adapter")}, {k: t[k].clone() for k in ("x", "adapter")}]
    torch.cuda.synchronize()
    graphs = []
    for state in (s, t):  # two graphs, each with scratch memory of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = decode_step(state)
        graphs.append((g, y))
    for turn in range(4):
        for (g, y), state, first in zip(graphs, (s, t), (0, 1)):
            from_ = (turn + first) % 2  # other inputs into the same graph (the weights stay its own)
            state["x"].copy_(inputs[from_]["x"])
            state["adapter"].copy_(inputs[from_]["adapter"])
            g.replay()
            torch.cuda.synchronize()
            eager = decode_step(state)
            assert torch.equal(y, eager)
            if from_ == first:
                assert torch.equal(y, want[first])
