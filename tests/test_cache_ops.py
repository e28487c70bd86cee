"""The attention part of a decode step over a cache held in 4 bits (triton_shared_amd.ops; tts_page_slots, tts_qk_norm_rope, tts_kv4_write, tts_kv4_read,
tts_kv4_attention): against their formulas in 64 bits, at the sizes, pages, masks and values where they can go wrong; what they refuse (no GPU
needed); and steps of all of them together."""
import ctypes
import math

import numpy as np
import pytest
import torch

import triton_shared_amd as tsa
from triton_shared_amd import ops

N = tsa._native
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
U = 2.0 ** -24  # half a step of fp32
NAN, INF = float("nan"), float("inf")


def half(dtype):
    return torch.finfo(TYPES[dtype]).eps / 2


def smallest(dtype):
    return torch.finfo(TYPES[dtype]).smallest_normal * torch.finfo(TYPES[dtype]).eps  # a step below the normal numbers


def gpu(*shape, seed=0, scale=1.0, dtype="fp32"):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.empty(*shape, device="cuda").normal_(0.0, scale, generator=g).to(TYPES[dtype])


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------- refusals, on the CPU
FAR = [(1 << 20) + (i << 34) for i in range(16)]  # addresses that a refused call never uses


def tensor(dtype, *shape, stride=None, ptr=FAR[0]):
    t = N.TtsTensor(ptr, dtype, len(shape))
    if stride is None:
        stride = [int(np.prod(shape[d + 1:])) for d in range(len(shape))]
    t.shape[:len(shape)] = list(shape)
    t.stride[:len(shape)] = list(stride)
    return t


F32, F16, BF16, I8, I32 = N.DTYPE_F32, N.DTYPE_F16, N.DTYPE_BF16, N.DTYPE_I8, N.DTYPE_I32


def slots_args(**kw):
    a = dict(table=tensor(I32, 3, 8, ptr=FAR[0]), lengths=tensor(I32, 3, ptr=FAR[1]), fresh=tensor(I32, 3, ptr=FAR[2]), free=tensor(I32, 20, ptr=FAR[3]), count=tensor(I32, 1, ptr=FAR[4]), page=16,
             slots=tensor(I32, 5, ptr=FAR[5]), positions=tensor(I32, 5, ptr=FAR[6]), owners=tensor(I32, 5, ptr=FAR[7]), starts=tensor(I32, 4, ptr=FAR[8]), left=tensor(I32, 1, ptr=FAR[9]), stream=None)
    return list((a | kw).values())


def rope_args(**kw):
    a = dict(q=tensor(BF16, 5, 8, 64, ptr=FAR[0]), k=tensor(BF16, 5, 2, 64, ptr=FAR[1]), positions=tensor(I32, 5, ptr=FAR[2]), cos_sin=tensor(F32, 100, 64, ptr=FAR[3]), w_q=tensor(BF16, 64, ptr=FAR[4]),
             w_k=tensor(BF16, 64, ptr=FAR[5]), eps=1e-6, interleaved=0, clear=0, q_out=tensor(BF16, 5, 8, 64, ptr=FAR[6]), k_out=tensor(BF16, 5, 2, 64, ptr=FAR[7]), stream=None)
    return list((a | kw).values())


def cache_t(dtype=BF16, pages=10, heads=2, page=16, dim=64, ptr=FAR[0], **kw):
    return tensor(dtype, pages, heads, page * (dim + 8) // 2, ptr=ptr, **kw)


def write_args(**kw):
    a = dict(cache=cache_t(), k=tensor(BF16, 5, 2, 64, ptr=FAR[1]), v=tensor(BF16, 5, 2, 64, ptr=FAR[2]), slots=tensor(I32, 5, ptr=FAR[3]), stream=None)
    return list((a | kw).values())


def read_args(**kw):
    a = dict(cache=cache_t(), slots=tensor(I32, 5, ptr=FAR[3]), k=tensor(BF16, 5, 2, 64, ptr=FAR[1]), v=tensor(BF16, 5, 2, 64, ptr=FAR[2]), stream=None)
    return list((a | kw).values())


def attend_args(**kw):
    a = dict(q=tensor(BF16, 5, 8, 64, ptr=FAR[1]), cache=cache_t(), table=tensor(I32, 3, 4, ptr=FAR[2]), lengths=tensor(I32, 3, ptr=FAR[3]), starts=tensor(I32, 4, ptr=FAR[4]), scale=0.125, window=0, longest=0, clear=0,
             out=tensor(BF16, 5, 8, 64, ptr=FAR[5]), work=FAR[6], bytes=1 << 30, stream=None)
    return list((a | kw).values())


REFUSALS = [
    ("tts_page_slots", slots_args, dict(table=None), N.TTS_INVALID, "table is missing"),
    ("tts_page_slots", slots_args, dict(table=tensor(I32, 3, 8, stride=(1, 3))), N.TTS_INVALID, "stride 3, not 1"),
    ("tts_page_slots", slots_args, dict(table=tensor(I32, 3, 8, stride=(4, 1))), N.TTS_INVALID, "rows overlap"),
    ("tts_page_slots", slots_args, dict(table=tensor(I32, 5000, 8)), N.TTS_UNSUPPORTED, "5000 requests"),
    ("tts_page_slots", slots_args, dict(lengths=tensor(I32, 4, ptr=FAR[1])), N.TTS_INVALID, "lengths: dimension 0 is 4"),
    ("tts_page_slots", slots_args, dict(fresh=tensor(F32, 3, ptr=FAR[2])), N.TTS_INVALID, "fresh is f32, not i32"),
    ("tts_page_slots", slots_args, dict(count=tensor(I32, 2, ptr=FAR[4])), N.TTS_INVALID, "count: dimension 0 is 2"),
    ("tts_page_slots", slots_args, dict(page=0), N.TTS_INVALID, "a page of 0"),
    ("tts_page_slots", slots_args, dict(positions=tensor(I32, 6, ptr=FAR[6])), N.TTS_INVALID, "positions: dimension 0 is 6"),
    ("tts_page_slots", slots_args, dict(starts=tensor(I32, 3, ptr=FAR[8])), N.TTS_INVALID, "starts: dimension 0 is 3"),
    ("tts_page_slots", slots_args, dict(left=tensor(I32, 1, ptr=FAR[4])), N.TTS_INVALID, "left shares memory with count"),
    ("tts_page_slots", slots_args, dict(owners=tensor(I32, 5, ptr=FAR[5] + 16)), N.TTS_INVALID, "owners shares memory with slots"),
    ("tts_page_slots", slots_args, dict(free=tensor(I32, 20, ptr=0)), N.TTS_INVALID, "free is a null pointer"),
    ("tts_qk_norm_rope", rope_args, dict(q=tensor(I8, 5, 8, 64)), N.TTS_INVALID, "q is i8"),
    ("tts_qk_norm_rope", rope_args, dict(q=tensor(BF16, 5, 512)), N.TTS_INVALID, "2 dimensions, not 3"),
    ("tts_qk_norm_rope", rope_args, dict(q=tensor(BF16, 5, 8, 63)), N.TTS_INVALID, "63 elements, not an even"),
    ("tts_qk_norm_rope", rope_args, dict(q=tensor(BF16, 5, 8, 514)), N.TTS_UNSUPPORTED, "514 elements"),
    ("tts_qk_norm_rope", rope_args, dict(k=tensor(F16, 5, 2, 64, ptr=FAR[1])), N.TTS_INVALID, "k is f16, not bf16"),
    ("tts_qk_norm_rope", rope_args, dict(k=tensor(BF16, 5, 2, 64, stride=(256, 128, 2), ptr=FAR[1])), N.TTS_INVALID, "k: its last dimension"),
    ("tts_qk_norm_rope", rope_args, dict(cos_sin=tensor(F32, 100, 66, ptr=FAR[3])), N.TTS_INVALID, "cos_sin: dimension 1 is 66"),
    ("tts_qk_norm_rope", rope_args, dict(cos_sin=tensor(F32, 100, 33, ptr=FAR[3])), N.TTS_INVALID, "cos_sin: dimension 1 is 33"),
    ("tts_qk_norm_rope", rope_args, dict(cos_sin=tensor(BF16, 100, 64, ptr=FAR[3])), N.TTS_INVALID, "cos_sin is bf16"),
    ("tts_qk_norm_rope", rope_args, dict(w_k=None), N.TTS_INVALID, "w_k is missing"),
    ("tts_qk_norm_rope", rope_args, dict(w_q=tensor(F16, 64, ptr=FAR[4])), N.TTS_INVALID, "w_q is f16, not bf16"),
    ("tts_qk_norm_rope", rope_args, dict(w_k=tensor(F32, 64, ptr=FAR[5])), N.TTS_INVALID, "w_k is f32, not bf16"),
    ("tts_qk_norm_rope", rope_args, dict(eps=-1.0), N.TTS_INVALID, "eps"),
    ("tts_qk_norm_rope", rope_args, dict(eps=NAN), N.TTS_INVALID, "eps"),
    ("tts_qk_norm_rope", rope_args, dict(eps=1e39), N.TTS_INVALID, "eps"),
    ("tts_qk_norm_rope", rope_args, dict(q_out=tensor(BF16, 5, 8, 64, stride=(512, 32, 1), ptr=FAR[6])), N.TTS_INVALID, "q_out: its rows overlap"),
    ("tts_qk_norm_rope", rope_args, dict(q_out=tensor(BF16, 5, 8, 64, ptr=FAR[0] + 2)), N.TTS_INVALID, "q_out shares memory with q"),
    ("tts_qk_norm_rope", rope_args, dict(k_out=tensor(BF16, 5, 2, 64, ptr=FAR[0])), N.TTS_INVALID, "k_out shares memory with q"),
    ("tts_qk_norm_rope", rope_args, dict(k_out=tensor(BF16, 5, 2, 64, ptr=FAR[3])), N.TTS_INVALID, "k_out shares memory with cos_sin"),
    ("tts_kv4_write", write_args, dict(cache=tensor(F32, 10, 2, 576)), N.TTS_UNSUPPORTED, "takes f16 and bf16"),
    ("tts_kv4_write", write_args, dict(cache=tensor(BF16, 10, 2, 577)), N.TTS_INVALID, "not a number of tokens times 36"),
    ("tts_kv4_write", write_args, dict(cache=cache_t(page=24)), N.TTS_UNSUPPORTED, "pages of 24"),
    ("tts_kv4_write", write_args, dict(cache=tensor(BF16, 10, 2, 576, stride=(1160, 580, 1))), N.TTS_INVALID, "multiples of 16 bytes"),
    ("tts_kv4_write", write_args, dict(cache=cache_t(ptr=FAR[0] + 8)), N.TTS_INVALID, "multiples of 16 bytes"),
    ("tts_kv4_write", write_args, dict(cache=tensor(BF16, 10, 2, 576, stride=(576, 0, 1))), N.TTS_INVALID, "rows overlap"),
    ("tts_kv4_write", write_args, dict(cache=cache_t(pages=1 << 28)), N.TTS_UNSUPPORTED, "more than 32 bits number"),
    ("tts_kv4_write", write_args, dict(cache=cache_t(pages=0)), N.TTS_INVALID, "cache is empty"),
    ("tts_kv4_write", write_args, dict(k=tensor(BF16, 5, 2, 40, ptr=FAR[1])), N.TTS_UNSUPPORTED, "heads of 40"),
    ("tts_kv4_write", write_args, dict(k=tensor(BF16, 5, 3, 64, ptr=FAR[1])), N.TTS_INVALID, "k: dimension 1 is 3"),
    ("tts_kv4_write", write_args, dict(v=tensor(F16, 5, 2, 64, ptr=FAR[2])), N.TTS_INVALID, "v is f16"),
    ("tts_kv4_write", write_args, dict(slots=tensor(I32, 6, ptr=FAR[3])), N.TTS_INVALID, "slots: dimension 0 is 6"),
    ("tts_kv4_write", write_args, dict(slots=tensor(I32, 5, stride=(2,), ptr=FAR[3])), N.TTS_INVALID, "stride 2"),
    ("tts_kv4_write", write_args, dict(v=tensor(BF16, 5, 2, 64, ptr=FAR[0] + 128)), N.TTS_INVALID, "cache shares memory with v"),
    ("tts_kv4_read", read_args, dict(k=tensor(BF16, 5, 2, 64, ptr=FAR[2] + 4)), N.TTS_INVALID, "k shares memory with v"),
    ("tts_kv4_read", read_args, dict(v=tensor(BF16, 5, 2, 64, stride=(0, 64, 1), ptr=FAR[2])), N.TTS_INVALID, "v: its rows overlap"),
    ("tts_kv4_attention", attend_args, dict(q=tensor(F16, 5, 8, 64, ptr=FAR[1])), N.TTS_INVALID, "q is f16, not bf16"),
    ("tts_kv4_attention", attend_args, dict(q=tensor(BF16, 5, 7, 64, ptr=FAR[1])), N.TTS_INVALID, "7 heads, not a multiple"),
    ("tts_kv4_attention", attend_args, dict(q=tensor(BF16, 5, 8, 288, ptr=FAR[1])), N.TTS_UNSUPPORTED, "heads of 288"),
    ("tts_kv4_attention", attend_args, dict(lengths=tensor(I32, 4, ptr=FAR[3])), N.TTS_INVALID, "lengths: dimension 0 is 4"),
    ("tts_kv4_attention", attend_args, dict(starts=tensor(I32, 3, ptr=FAR[4])), N.TTS_INVALID, "starts: dimension 0 is 3"),
    ("tts_kv4_attention", attend_args, dict(table=tensor(I32, 3, 4, stride=(1, 3), ptr=FAR[2])), N.TTS_INVALID, "table: its last dimension"),
    ("tts_kv4_attention", attend_args, dict(window=-1), N.TTS_INVALID, "window is -1"),
    ("tts_kv4_attention", attend_args, dict(longest=-1), N.TTS_INVALID, "longest is -1"),
    ("tts_kv4_attention", attend_args, dict(scale=INF), N.TTS_INVALID, "scale"),
    ("tts_kv4_attention", attend_args, dict(scale=-1e39), N.TTS_INVALID, "scale"),
    ("tts_kv4_attention", attend_args, dict(out=tensor(BF16, 5, 8, 64, ptr=FAR[1] + 2)), N.TTS_INVALID, "out shares memory with q"),
    ("tts_kv4_attention", attend_args, dict(out=tensor(BF16, 5, 8, 64, ptr=FAR[0] + 128)), N.TTS_INVALID, "out shares memory with cache"),
    ("tts_kv4_attention", attend_args, dict(table=tensor(I32, 3, 1000, ptr=FAR[2]), bytes=16), N.TTS_INVALID, "the workspace has 16 bytes"),
    ("tts_kv4_attention", attend_args, dict(table=tensor(I32, 3, 1000, ptr=FAR[2]), work=None), N.TTS_INVALID, "workspace is a null pointer"),
    ("tts_kv4_attention", attend_args, dict(q=tensor(BF16, 1 << 24, 8, 64, ptr=FAR[1])), N.TTS_UNSUPPORTED, "16777216 rows of 8 heads"),
    ("tts_kv4_attention", attend_args, dict(q=tensor(BF16, 4097, 4095, 32, ptr=FAR[1]), cache=cache_t(heads=4095, dim=32), table=tensor(I32, 4097, 4, ptr=FAR[2]), lengths=tensor(I32, 4097, ptr=FAR[3]),
                                            starts=tensor(I32, 4098, ptr=FAR[4]), out=tensor(BF16, 4097, 4095, 32, ptr=FAR[5])), N.TTS_UNSUPPORTED, "4097 requests of 4095 heads"),   # 2^24 - 1 workgroups and 8
]


@pytest.mark.parametrize("entry,args,change,status,says", REFUSALS, ids=[f"{r[0][4:]}-{i}" for i, r in enumerate(REFUSALS)])
def test_refused_calls(entry, args, change, status, says):
    assert getattr(N.lib(), entry)(*args(**change)) == status
    assert says in N.lib().tts_last_error().decode()


def test_calls_for_no_rows_do_nothing():
    L = N.lib()
    none = dict(ptr=0)
    assert L.tts_qk_norm_rope(*rope_args(q=tensor(BF16, 0, 8, 64, **none), k=tensor(BF16, 0, 2, 64, **none), positions=tensor(I32, 0, **none), q_out=tensor(BF16, 0, 8, 64, **none), k_out=tensor(BF16, 0, 2, 64, **none))) == 0
    assert L.tts_kv4_write(*write_args(k=tensor(BF16, 0, 2, 64, **none), v=tensor(BF16, 0, 2, 64, **none), slots=tensor(I32, 0, **none))) == 0
    assert L.tts_kv4_read(*read_args(k=tensor(BF16, 0, 2, 64, **none), v=tensor(BF16, 0, 2, 64, **none), slots=tensor(I32, 0, **none))) == 0
    assert L.tts_kv4_attention(*attend_args(q=tensor(BF16, 0, 8, 64, **none), out=tensor(BF16, 0, 8, 64, **none))) == 0
    assert L.tts_kv4_attention(*attend_args(table=tensor(I32, 0, 4, **none), lengths=tensor(I32, 0, **none), starts=tensor(I32, 1))) == 0


def test_columns_of_a_projection_are_told_apart():
    # q and k, columns of the same rows, are turned where they are
    rows = dict(stride=(12 * 64, 64, 1))
    q, k = tensor(BF16, 5, 8, 64, **rows), tensor(BF16, 5, 2, 64, ptr=FAR[0] + 8 * 128, **rows)
    far = tensor(BF16, 5, 2, 64, ptr=FAR[0] + 7 * 128, **rows)
    for k_out, says in ((k, "eps"), (far, "k_out shares memory with k")):
        # (a refusal that comes after those of shared memory does not exist: a wrong eps comes before)
        status = N.lib().tts_qk_norm_rope(*rope_args(q=q, k=k, q_out=q, k_out=k_out, eps=-1.0 if says == "eps" else 1e-6))
        assert status == N.TTS_INVALID and says in N.lib().tts_last_error().decode()


def test_workspaces_hold_the_slices():
    size = ctypes.c_size_t()
    q, cache = tensor(BF16, 4, 8, 64, ptr=FAR[1]), cache_t()
    assert N.lib().tts_kv4_attention_workspace(q, cache, tensor(I32, 4, 1000, ptr=FAR[2]), 0, 0, ctypes.byref(size)) == 0
    long = size.value
    assert long >= 4 * 8 * 2 * 66 * 4
    assert N.lib().tts_kv4_attention_workspace(q, cache, tensor(I32, 4, 1000, ptr=FAR[2]), 0, 100, ctypes.byref(size)) == 0 and size.value == 0   # short ones need none
    assert N.lib().tts_kv4_attention_workspace(q, cache, tensor(I32, 4, 1000, ptr=FAR[2]), 20, 0, ctypes.byref(size)) == 0 and size.value == 0    # nor does a narrow window
    assert N.lib().tts_kv4_attention_workspace(q, cache, tensor(I32, 4, 1000, ptr=FAR[2]), 0, 1 << 40, ctypes.byref(size)) == 0 and size.value == long


def test_strides_of_single_pages_and_heads_say_nothing():
    L, size = N.lib(), ctypes.c_size_t()
    for heads, pages, stride, status in ((1, 10, (576, 1, 1), 0), (2, 1, (1, 576, 1), 0), (1, 1, (5, 3, 1), 0), (2, 10, (1152, 577, 1), N.TTS_INVALID), (1, 10, (577, 1, 1), N.TTS_INVALID)):
        cache = tensor(BF16, pages, heads, 576, stride=stride)
        assert L.tts_kv4_attention_workspace(tensor(BF16, 4, 8, 64, ptr=FAR[1]), cache, tensor(I32, 4, 4, ptr=FAR[2]), 0, 0, ctypes.byref(size)) == status


def test_python_arguments_are_checked_without_a_gpu():
    cpu = torch.zeros(4, 16, dtype=torch.int32)
    with pytest.raises(TypeError, match="GPU memory"):
        ops.page_slots(cpu, cpu, cpu, cpu, cpu, 16, 4)
    with pytest.raises(TypeError, match="GPU memory"):
        ops.qk_norm_rope(cpu, cpu, cpu, cpu)
    with pytest.raises(TypeError, match="not a tensor"):
        ops.kv4_write([1.0], cpu, cpu, cpu)
    with pytest.raises(ValueError, match="window is 0"):
        ops.kv4_attention(cpu, cpu, cpu, cpu, cpu, window=0)
    with pytest.raises(ValueError, match="longest is 0"):
        ops.kv4_attention(cpu, cpu, cpu, cpu, cpu, longest=0)
    with pytest.raises(NotImplementedError, match="pages of 8"):
        ops.kv4_cache(4, 2, 64, page=8, device="cpu")
    with pytest.raises(NotImplementedError, match="heads of 80"):
        ops.kv4_cache(4, 2, 80, device="cpu")
    with pytest.raises(ValueError, match="float32"):
        ops.kv4_cache(4, 2, 64, dtype=torch.float32, device="cpu")
    assert ops.kv4_cache(4, 2, 64, page=32, device="cpu").shape == (4, 2, 32 * 36)


# ---------------------------------------------------------------------------------------------------------------- slots
def slots_exact(table, lengths, fresh, free, count, page, rows):
    """The definition, a token at a time."""
    table, free = table.cpu().numpy().astype(np.int64).copy(), free.cpu().numpy()
    B, M = table.shape
    left = min(max(int(count[0]), 0), len(free))
    slots, positions, owners, starts = [], [], [], [0]
    for b in range(B):
        n = max(int(lengths[b]), 0)
        past = n - min(max(int(fresh[b]), 0), n)
        for j in range(min(-(-past // page), M), min(-(-n // page), M)):
            left -= 1
            table[b, j] = free[left] if left >= 0 else -1
        for p in range(past, n):
            at = table[b, p // page] if p // page < M else -1
            slot = at * page + p % page
            slots.append(slot if at >= 0 and slot < 2 ** 31 else -1)
            positions.append(p)
            owners.append(b)
        starts.append(len(slots))
    fill = lambda x: np.array((x + [-1] * rows)[:rows], np.int32)  # noqa: E731
    return table.astype(np.int32), fill(slots), fill(positions), fill(owners), np.array(starts, np.int32), np.array([max(left, 0)], np.int32)


def check_slots(table, lengths, fresh, free, count, page, rows):
    want = slots_exact(table, lengths, fresh, free, count, page, rows)
    got = (table, *ops.page_slots(table, lengths, fresh, free, count, page, rows))
    for name, x, y in zip(("table", "slots", "positions", "owners", "starts", "left"), got, want):
        assert np.array_equal(x.cpu().numpy(), y), name
    return got[1:]


def make_slots(lengths, fresh, page, columns=None, spare=10, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    each = [-(-n // page) for n in lengths]
    columns = max(each, default=0) + 2 if columns is None else columns
    order = torch.randperm(sum(each) + spare, generator=g, device="cuda").int()
    table = torch.full((len(lengths), columns), -7, dtype=torch.int32, device="cuda")
    at = 0
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        have = min(-(-(n - min(f, n)) // page), columns)
        table[b, :have] = order[at:at + have]
        at += have
    return table, ints(lengths), ints(fresh), order[at:].contiguous(), ints([len(order) - at])


@pytest.mark.gpu
@pytest.mark.parametrize("page", [1, 16, 48, 100])
@pytest.mark.parametrize("lengths,fresh", [([1], [1]), ([0], [0]), ([5, 0, 17], [5, 0, 1]), ([100, 16, 17, 33], [1, 1, 1, 1]), ([160, 96, 7], [160, 0, 7]), ([300, 1, 299, 48], [37, 1, 100, 48])])
def test_slots(lengths, fresh, page):
    check_slots(*make_slots(lengths, fresh, page), page, sum(fresh))
    check_slots(*make_slots(lengths, fresh, page, seed=1), page, sum(fresh) + 13)   # padded
    check_slots(*make_slots(lengths, fresh, page, seed=2), page, sum(fresh) // 2)   # fewer rows than there are tokens
    check_slots(*make_slots(lengths, fresh, page, seed=3, spare=0), page, sum(fresh))


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [63, 64, 257, 1000, 4096])
def test_slots_of_many_requests(requests):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, 200, requests)
    fresh = np.minimum(rng.integers(0, 20, requests) * (rng.random(requests) < 0.7), lengths)
    check_slots(*make_slots(lengths.tolist(), fresh.tolist(), 16), 16, int(fresh.sum()) + 5)


@pytest.mark.gpu
def test_slots_where_the_stack_runs_out():
    table, lengths, fresh, free, count = make_slots([40, 33, 64, 5], [40, 1, 64, 5], 16, spare=0)
    for n in (0, 1, 5, len(free), len(free) + 100, -3):
        check_slots(table.clone(), lengths, fresh, free, ints([n]), 16, 110)
    check_slots(table.clone(), lengths, fresh, free[:4].contiguous(), ints([9]), 16, 110)
    check_slots(table.clone(), lengths, fresh, free[:0], ints([9]), 16, 110)


@pytest.mark.gpu
def test_slots_of_tables_too_narrow_and_odd_numbers():
    for columns in (0, 1, 2, 3):
        check_slots(*make_slots([40, 70, 16, 17], [40, 30, 1, 17], 16, columns=columns), 16, 90)
    table, _, _, free, count = make_slots([40, 30], [40, 30], 16)
    check_slots(table.clone(), ints([-5, 30]), ints([3, 40]), free, count, 16, 40)       # negative lengths, more new tokens than tokens
    check_slots(table.clone(), ints([20, 30]), ints([-2, 30]), free, count, 16, 40)
    check_slots(table.clone(), ints([20, 30]), ints([20, 30]), free + 2 ** 30, count, 16, 60)  # slots past 32 bits: none
    wide = torch.full((2, 64), -7, dtype=torch.int32, device="cuda")[:, 8:16]                # a table inside a larger one
    check_slots(wide, ints([20, 30]), ints([20, 30]), free, count, 16, 60)


@pytest.mark.gpu
def test_slots_of_no_requests():
    none = ints([])
    got = check_slots(torch.empty(0, 4, dtype=torch.int32, device="cuda"), none, none, ints([3, 4]), ints([2]), 16, 3)
    assert got[3].tolist() == [0] and got[4].tolist() == [2]


@pytest.mark.gpu
def test_slots_behind_2_31_rows():
    big = 2 ** 31 - 1
    table = torch.arange(6, dtype=torch.int32, device="cuda").reshape(3, 2)
    slots, positions, owners, starts, left = ops.page_slots(table, ints([big, big, 5]), ints([big, big, 5]), ints(list(range(50))), ints([50]), 1 << 28, 20)
    assert starts.tolist() == [0, big, big, big] and owners.tolist() == [0] * 20 and positions.tolist() == list(range(20))
    assert left.tolist() == [45] and table.tolist() == [[49, 48], [47, 46], [45, 5]]


# ---------------------------------------------------------------------------------------------------------------- norms and the rotation
def turns(places, rotary, seed=0):
    angles = torch.arange(places, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary) + seed
    return torch.cat([angles.cos(), angles.sin()], 1).float()


def rope_exact(x, positions, cos_sin, w, eps, interleaved):
    """The definition in 64 bits and how far 32 bits and one rounding may be off."""
    dtype = {v: k for k, v in TYPES.items()}[x.dtype]
    y, D, R = x.double(), x.shape[2], cos_sin.shape[1]
    slip = 0.0
    if w is not None:
        y = y / torch.sqrt((y * y).mean(dim=2, keepdim=True) + eps) * w.double()
        slip = (D / 2 + 10) * U  # the sum of D squares (half of it in the root), the mean, eps, root, quotient, two products
    real = (positions >= 0) & (positions < cos_sin.shape[0])
    at = cos_sin.double()[torch.where(real, positions, 0).long()][:, None]
    cos, sin = at[..., :R // 2], at[..., R // 2:]
    first = torch.arange(R // 2, device="cuda") * (2 if interleaved else 1)
    second = first + (1 if interleaved else R // 2)
    a, b = y[..., first], y[..., second]
    size = y.abs()
    out = y.clone()
    out[..., first], out[..., second] = a * cos - b * sin, b * cos + a * sin
    size[..., first], size[..., second] = (a * cos).abs() + (b * sin).abs(), (b * cos).abs() + (a * sin).abs()
    err = (slip + 3 * U) * size
    return out, err + half(dtype) * (out.abs() + err) + smallest(dtype), real


def check_rope(q, k, positions, cos_sin, w_q=None, w_k=None, eps=1e-6, interleaved=False, out=None):
    wants = [rope_exact(x, positions, cos_sin, w, eps, interleaved) for x, w in ((q, w_q), (k, w_k))]
    before = None if out is None else [o.clone() for o in out]
    got = ops.qk_norm_rope(q, k, positions, cos_sin, w_q, w_k, eps=eps, interleaved=interleaved, out=out)
    for i, (y, (want, lim, real)) in enumerate(zip(got, wants)):
        off = (y.double() - want).abs()[real]
        assert bool((off <= lim[real]).all()), f"off by {(off / lim[real]).max().item():.2f} of what is allowed"
        others = y[~real]
        assert torch.equal(others, torch.zeros_like(others) if out is None else before[i][~real])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,D,R", [(1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (3, 5, 1, 64, 64), (7, 4, 2, 96, 48), (5, 3, 3, 80, 40), (33, 6, 2, 80, 80), (9, 2, 1, 6, 4), (4, 3, 1, 50, 20), (2, 2, 1, 256, 64),
                                         (5, 7, 1, 192, 192), (3, 2, 2, 512, 512), (2, 2, 1, 510, 256), (70, 15, 5, 128, 32), (13, 40, 8, 128, 128), (2, 1, 4, 144, 16), (5, 3, 1, 72, 24), (3, 2, 2, 200, 104), (2, 1, 1, 504, 8)])
def test_rope(T, Hq, Hk, D, R, interleaved, dtype):
    q, k = gpu(T, Hq, D, seed=1, scale=3.0, dtype=dtype), gpu(T, Hk, D, seed=2, scale=0.2, dtype=dtype)
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    positions = torch.randint(0, 500, (T,), generator=g, dtype=torch.int32, device="cuda")
    w = [1.0 + gpu(D, seed=s, scale=0.3) for s in (3, 4)]
    cos_sin = turns(500, R)
    check_rope(q, k, positions, cos_sin, *(x.to(q.dtype) for x in w), interleaved=interleaved)
    check_rope(q, k, positions, cos_sin, *w, eps=0.5, interleaved=interleaved)
    check_rope(q, k, positions, cos_sin, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 50])
def test_rope_of_padding_in_place_and_strides(D):
    T, Hq, Hk = 21, 6, 2
    qkv = gpu(T, Hq + 2 * Hk, D + 3, seed=1, dtype="bf16")[..., :D]
    positions, cos_sin = ints(list(range(T - 4)) + [-1, 100, 2 ** 31 - 1, -2 ** 31]), turns(100, D)
    w = [gpu(D, seed=s, dtype="bf16") for s in (5, 6)]
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hk], qkv[:, Hq + Hk:]
    want = check_rope(q, k, positions, cos_sin, *w)
    others = [gpu(Hq, T, D, seed=9, dtype="bf16").transpose(0, 1), gpu(T, Hk, D, seed=10, dtype="bf16")]    # heads before tokens
    got = check_rope(q, k, positions, cos_sin, *w, out=others)
    assert all(x is y for x, y in zip(got, others))
    real = slice(0, T - 4)
    assert all(torch.equal(x[real], y[real]) for x, y in zip(got, want))
    before = v.clone()
    q0 = q.clone()
    got = check_rope(q, k, positions, cos_sin, *w, out=(q, k))
    assert got[0] is q and torch.equal(q[real], want[0][real]) and torch.equal(k[real], want[1][real]) and torch.equal(v, before) and torch.equal(q[T - 4:], q0[T - 4:])
    # rows of a table further apart than they are wide
    wide = gpu(100, D + 10, seed=3)
    wide[:, 4:4 + D] = cos_sin
    again = ops.qk_norm_rope(q, k, positions, wide[:, 4:4 + D], *w)
    assert all(torch.equal(x, y) for x, y in zip(again, ops.qk_norm_rope(q, k, positions, cos_sin, *w)))


@pytest.mark.gpu
def test_rope_zeros_infinities_and_no_places():
    q, k = gpu(6, 3, 64, dtype="bf16"), gpu(6, 1, 64, seed=1, dtype="bf16")
    w = [torch.ones(64, device="cuda")] * 2
    cos_sin, positions = turns(10, 64), ints([0, 1, 2, 3, 4, 5])
    q[0] = 0.0
    clean = ops.qk_norm_rope(q, k, positions, cos_sin, *w)
    assert bool((clean[0][0] == 0).all())
    with_eps_0 = ops.qk_norm_rope(q, k, positions, cos_sin, *w, eps=0.0)
    assert bool(with_eps_0[0][0].isnan().all()) and torch.equal(with_eps_0[1], clean[1])    # 0 / 0, as the formula gives
    q[2, 1, 5], q[3, 0, 7] = NAN, INF
    got = ops.qk_norm_rope(q, k, positions, cos_sin, *w)
    assert got[0][2, 1].isnan().all() and bool(got[0][3, 0].isnan().any())
    got[0][2, 1], got[0][3, 0] = clean[0][2, 1], clean[0][3, 0]
    assert all(torch.equal(x, y) for x, y in zip(got, clean))                               # nothing of it elsewhere
    none = torch.empty(0, 64, device="cuda")
    assert all(bool((x == 0).all()) for x in ops.qk_norm_rope(q, k, positions, none, *w))   # no position is in the table
    outs = [torch.full_like(x, 3.0) for x in (q, k)]
    ops.qk_norm_rope(q, k, positions, none, *w, out=outs)
    assert all(bool((x == 3.0).all()) for x in outs)


# ---------------------------------------------------------------------------------------------------------------- the cache
def held(x):
    """code, step and lowest value [.., 1] of the heads of x, in 64 bits, by the borders of the definition."""
    wide = x.double()
    low, high = wide.min(dim=-1, keepdim=True).values, wide.max(dim=-1, keepdim=True).values
    step = ((high.float() - low.float()) / torch.tensor(15.0, device=x.device)).to(x.dtype).double()
    code = torch.zeros_like(wide)
    for n in range(15):
        code += ((wide - low > (n + 0.5) * step) & (step > 0)).double()
    bad = ~(x.float().isfinite().all(dim=-1, keepdim=True) & (high.float() - low.float()).isfinite())
    return code, torch.where(bad, NAN, step), torch.where(bad, NAN, low)


def held_values(x):
    code, step, low = held(x)
    return (code * step + low).float().to(x.dtype)


def same(x, y):
    return torch.equal(x.isnan(), y.isnan()) and torch.equal(torch.nan_to_num(x.float(), nan=0.0), torch.nan_to_num(y.float(), nan=0.0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H,D,page", [(1, 1, 32, 16), (5, 2, 64, 16), (37, 3, 96, 48), (130, 8, 128, 64), (9, 1, 160, 32), (21, 5, 192, 16), (6, 2, 224, 112), (33, 4, 256, 128)])
def test_cache(T, H, D, page, dtype):
    pages = -(-T // page) + 3
    cache = ops.kv4_cache(pages, H, D, page=page, dtype=TYPES[dtype])
    g = torch.Generator(device="cuda")
    g.manual_seed(T)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:T].int()
    k, v = gpu(T, H, D, seed=1, dtype=dtype) + gpu(1, H, D, seed=3, dtype=dtype), gpu(T, H, D, seed=2, scale=0.01, dtype=dtype)
    assert ops.kv4_write(cache, k, v, slots) is cache
    got = ops.kv4_read(cache, slots, D)
    assert same(got[0], held_values(k)) and same(got[1], held_values(v))
    # half a step of what it was, the step's own rounding, which 15 of it add up, and the value's rounding to the type
    for y, x in zip(got, (k, v)):
        _, step, low = held(x)
        assert bool(((y.double() - x.double()).abs() <= step * (0.5 + 16 * half(dtype)) + half(dtype) * x.double().abs() * 2).all())
    everything = ops.kv4_read(cache, torch.arange(pages * page, dtype=torch.int32, device="cuda"), D)
    others = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    others[slots.long()] = False
    assert all(bool((x[others] == 0).all()) for x in everything)      # nothing else was written
    again = cache.clone()
    more = torch.randperm(T, generator=g, device="cuda")[: T // 2 + 1]
    ops.kv4_write(again, v[more], k[more], slots[more])               # over what was there
    got = ops.kv4_read(again, slots, D)
    mixed_k, mixed_v = held_values(k), held_values(v)
    mixed_k[more], mixed_v[more] = held_values(v)[more], held_values(k)[more]
    assert same(got[0], mixed_k) and same(got[1], mixed_v)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_cache_borders_and_odd_values(dtype):
    D, lowest = 64, torch.finfo(TYPES[dtype]).min
    x = gpu(20, 1, D, seed=1, dtype=dtype)
    x[0] = 0.0
    x[1] = -2.5                                                         # all the same
    x[2, 0] = torch.arange(D, device="cuda").to(x.dtype) / 4            # a step of 1.05, rounded
    x[3, 0] = (torch.arange(D, device="cuda") % 31).to(x.dtype) / 2     # a step of 1: every other one lies on a border
    x[4, 0] = x[3, 0] - 8.0
    x[5, 0, 3] = NAN
    x[6, 0, 9] = INF
    x[7, 0, 63] = -INF
    x[8] *= smallest(dtype) * 4                                         # below the normal numbers
    x[9] = 0.0
    x[9, 0, 5] = smallest(dtype)                                        # a step that rounds to 0
    x[10] = -0.0
    x[11, 0, 1] = lowest                                                # far apart
    x[12, 0, 1], x[12, 0, 2] = lowest, -lowest                          # bf16: a range past 32 bits
    x[13, 0] = torch.where(torch.arange(D, device="cuda") % 2 == 0, 3.0, -3.0).to(x.dtype)
    x[13, 0, ::5] = 2.0 ** -20                                          # 27 bits between it and -3
    x[14] = x[14] * 1e-4 + 100.0
    if dtype == "bf16":
        x[15] *= 1e-38
        x[16] *= 1e37
    slots = torch.arange(20, dtype=torch.int32, device="cuda")
    cache = ops.kv4_cache(2, 1, D, dtype=TYPES[dtype])
    ops.kv4_write(cache, x, -x, slots)
    k, v = ops.kv4_read(cache, slots, D)
    assert same(k, held_values(x)) and same(v, held_values(-x))
    # (fp16's largest is held as -65504 + 15 * 8736 = 65536, since 131008 / 15 = 8733.9 is rounded to 8736: an infinity as a value of the type, but no NaN)
    assert bool(k[5].isnan().all() and k[6].isnan().all() and k[7].isnan().all()) and (dtype == "fp16") == (not bool(k[12].isnan().any()))


@pytest.mark.gpu
def test_cache_slots_that_are_not_there():
    cache = ops.kv4_cache(3, 2, 64)
    k, v = gpu(8, 2, 64, seed=1, dtype="bf16"), gpu(8, 2, 64, seed=2, dtype="bf16")
    slots = ints([5, -1, 47, 48, -2 ** 31, 2 ** 31 - 1, 0, 1000])
    guard = torch.zeros(5, 2, 576, dtype=torch.bfloat16, device="cuda")
    ops.kv4_write(guard[1:4], k, v, slots)
    assert bool((guard[0] == 0).all() and (guard[4] == 0).all())
    ops.kv4_write(cache, k, v, slots)
    assert torch.equal(cache.view(torch.int16), guard[1:4].view(torch.int16))
    got = ops.kv4_read(cache, slots, 64)
    real = [0, 2, 6]
    for y, x in zip(got, (k, v)):
        want = torch.zeros_like(x)
        want[real] = held_values(x)[real]
        assert same(y, want)


@pytest.mark.gpu
def test_cache_of_layers_strides_and_past_32_bits():
    D, H, page = 96, 3, 16
    layers = torch.zeros(4, 2, H, page * (D + 8) // 2, dtype=torch.float16, device="cuda")   # a page's layers next to each other
    qkv = gpu(30, 11, D + 1, seed=1, dtype="fp16")[..., 1:]
    k, v = qkv[:, 4:7], qkv[:, 7:10].transpose(0, 1).contiguous().transpose(0, 1)
    slots = torch.arange(30, dtype=torch.int32, device="cuda") * 2
    ops.kv4_write(layers[:, 1], k, v, slots)
    assert bool((layers[:, 0] == 0).all())
    got = ops.kv4_read(layers[:, 1], slots, D)
    assert same(got[0], held_values(k)) and same(got[1], held_values(v))
    far = 2 ** 31 + 8
    big = torch.zeros(2 * far, dtype=torch.float16, device="cuda")
    for strides in ((far, layers.shape[3], 1), (layers.shape[3], far // 2 // 8 * 8, 1)):
        cache = torch.as_strided(big, (2, H, layers.shape[3]), strides)
        ops.kv4_write(cache, k[:16], v[:16], slots[:16])
        got = ops.kv4_read(cache, slots[:16], D)
        assert same(got[0], held_values(k[:16])) and same(got[1], held_values(v[:16]))


# ---------------------------------------------------------------------------------------------------------------- the attention
def make_attend(lengths, fresh, Hq, Hk, D, page=16, dtype="bf16", seed=0, columns=None, q_scale=1.5):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    each = [-(-n // page) for n in lengths]
    pages = sum(each) + 2
    order = torch.randperm(pages, generator=g, device="cuda").int()
    table = torch.full((len(lengths), (max(each, default=0) + 1) if columns is None else columns), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(each):
        n = min(n, table.shape[1])
        table[b, :n] = order[at:at + n]
        at += n
    a = dict(q=gpu(sum(fresh), Hq, D, seed=seed + 1, scale=q_scale, dtype=dtype), table=table, lengths=ints(lengths), starts=ints(np.concatenate([[0], np.cumsum(fresh)]).tolist()))
    a["k"] = gpu(pages * page, Hk, D, seed=seed + 2, dtype=dtype) + gpu(1, Hk, D, seed=seed + 3, dtype=dtype)
    a["v"] = gpu(pages * page, Hk, D, seed=seed + 4, dtype=dtype)
    return fill(a, page)


def fill(a, page):
    """The cache of a's keys and values; what no request has in it is left as memory may be: NaN."""
    dt = a["q"].dtype
    cache = ops.kv4_cache(len(a["k"]) // page, a["k"].shape[1], a["q"].shape[2], page=page, dtype=dt)
    cache.view(torch.int16).fill_(-1)
    used = torch.full((len(a["k"]),), False, device="cuda")
    for b, n in enumerate(a["lengths"].tolist()):
        j = torch.arange(min(n, a["table"].shape[1] * page), device="cuda")
        at = a["table"][b].long()[j // page]
        used[(at * page + j % page)[(at >= 0) & (at < len(cache))]] = True
    ops.kv4_write(cache, a["k"], a["v"], torch.where(used, torch.arange(len(used), device="cuda"), -1).int())
    return a | dict(cache=cache, page=page)


def attend_exact(a, scale, window):
    """out by its definition in 64 bits, how far the kernel may be off, and the rows that have a request."""
    q, page, dtype = a["q"], a["page"], {v: k for k, v in TYPES.items()}[a["q"].dtype]
    T, Hq, D = q.shape
    Hk = a["k"].shape[1]
    group = Hq // Hk
    out, lim = torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda"), torch.zeros(T, Hq, D, dtype=torch.float64, device="cuda")
    real = torch.zeros(T, dtype=torch.bool, device="cuda")
    starts = a["starts"].tolist()
    for b, n in enumerate(a["lengths"].tolist()):
        first, f = starts[b], starts[b + 1] - starts[b]
        if f == 0:
            continue
        real[first:first + f] = True
        places = min(n, a["table"].shape[1] * page)
        j = torch.arange(max(places, 1), device="cuda")
        at = a["table"][b].long()[(j // page).clamp(max=max(a["table"].shape[1] - 1, 0))] if a["table"].shape[1] else torch.full_like(j, -1)
        there = (at >= 0) & (at < len(a["k"]) // page) & (j < places)
        slots = torch.where(there, at * page + j % page, 0)
        i = torch.arange(n - f, n, device="cuda")
        seen = there[None] & (j[None] <= i[:, None])
        if window:
            seen &= j[None] > i[:, None] - window
        for g in range(Hk):
            ck, sk, lk = held(a["k"][slots, g])
            cv, sv, lv = held(a["v"][slots, g])
            for h in range(g * group, (g + 1) * group):
                x = q[first:first + f, h].double()
                z = (x @ (ck * sk + lk).t()) * scale
                size = (x.abs() @ ck.t() * sk.t().abs() + x.abs().sum(dim=1, keepdim=True) * lk.t().abs()) * abs(scale)
                # the score: D products and as many sums of each part, of which a sum may be cut where it is not rounded, four factors, and q: fp16's last place below its normal
                # numbers, 2^-24, of which half is lost, times 16 for half of the elements, where the largest is 2^13 at least: 2^-34 of that
                off = (2 * D + 20) * U * size + 2.0 ** -34 * x.abs().amax(dim=1, keepdim=True) * (ck.sum(dim=1)[None] * sk.t().abs()) * abs(scale)
                z = torch.where(seen, z, -INF)
                most = z.amax(dim=1, keepdim=True)
                most = torch.where(most == -INF, 0.0, most)
                e = torch.where(seen, torch.exp(z - most), 0.0)
                total = e.sum(dim=1, keepdim=True)
                # the exponential: of a difference that is rounded, of a power of two within two steps
                slip = torch.where(seen, off + 4 * U * (torch.where(seen, z, 0.0).abs() + most.abs()) + 6 * U, 0.0)
                w = e / total.clamp(min=1e-300)
                count = seen.sum(dim=1, keepdim=True).double()
                # the sums: of as many tokens as a lane has, and joining them; the statistics' error, and that of each weight
                per = torch.where(seen, slip + (count / 4 + 64) * 2 * U, 0.0)
                value, big, codes = cv * sv + lv, (cv * sv).abs() + lv.abs(), (cv * sv).abs()
                if bool(value.isfinite().all() and w.isfinite().all()):
                    y = w @ value
                    err = (w * (2 * per + (w * per).sum(dim=1, keepdim=True))) @ big + 2.0 ** -11 * (w @ codes)
                    largest = torch.where(seen, sv.abs().t(), 0.0).amax(dim=1, keepdim=True)
                    err = err + 15 * count * 2.0 ** -34 * largest / total.clamp(min=1e-300)
                else:
                    y = torch.zeros(f, D, dtype=torch.float64, device="cuda")
                    err = torch.zeros_like(y)
                    for r in range(f):  # (a NaN that a row does not see stays out of it)
                        s = seen[r]
                        if not bool(s.any()):
                            continue
                        wr, pr = w[r, s], per[r, s]
                        y[r] = wr @ value[s]
                        err[r] = (wr * (2 * pr + (wr * pr).sum())) @ big[s] + 2.0 ** -11 * (wr @ codes[s])
                        err[r] += 15 * count[r] * 2.0 ** -34 * sv[s].abs().max() / total[r]
                out[first:first + f, h], lim[first:first + f, h] = y, err + half(dtype) * (y.abs() + err) + smallest(dtype)
    return out, lim, real


def check_attend(a, scale=None, window=None, longest=None, out=None, q=None):
    want, lim, real = attend_exact(a, a["q"].shape[2] ** -0.5 if scale is None else scale, window)
    before = None if out is None else out.clone()
    got = ops.kv4_attention(a["q"] if q is None else q, a["cache"], a["table"], a["lengths"], a["starts"], scale=scale, window=window, longest=longest, out=out)
    nan = want.isnan()
    assert torch.equal(got.isnan() & real[:, None, None], nan & real[:, None, None])
    off = torch.where(nan, 0.0, (got.double() - want).abs())[real]
    allowed = torch.where(nan, 1.0, lim)[real]
    assert bool((off <= allowed).all()), f"off by {(off / allowed).max().item():.2f} of what is allowed"
    others = got[~real]
    assert torch.equal(others, torch.zeros_like(others) if out is None else before[~real])
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("lengths,fresh,Hq,Hk,D,page", [
    ([1], [1], 1, 1, 32, 16), ([1, 17, 64, 65], [1, 1, 1, 1], 8, 2, 64, 16), ([300], [1], 4, 4, 96, 48), ([1000, 255, 257, 3], [1, 1, 1, 1], 32, 8, 128, 16), ([70, 700], [1, 1], 5, 1, 160, 32),
    ([129, 64], [1, 1], 6, 2, 192, 16), ([80, 500], [1, 1], 4, 2, 224, 112), ([333, 5], [1, 1], 16, 1, 256, 64),
    ([2500], [1], 24, 1, 128, 16), ([90, 33], [1, 1], 17, 1, 64, 16),                          # more than 16 queries a key
    ([7, 90, 300, 5], [5, 3, 6, 5], 15, 3, 96, 32), ([40, 0, 20], [7, 0, 1], 12, 4, 64, 16),   # a few tokens each
    ([200, 500], [60, 90], 4, 2, 128, 16), ([150, 333], [100, 333], 8, 2, 64, 48), ([700, 130, 90], [200, 130, 1], 4, 1, 256, 64), ([300, 300], [150, 20], 6, 2, 192, 16),  # prompts
])
def test_attend(lengths, fresh, Hq, Hk, D, page, dtype):
    a = make_attend(lengths, fresh, Hq, Hk, D, page, dtype, seed=sum(lengths))
    check_attend(a, longest=max(lengths))
    check_attend(a, window=37)


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,fresh,Hq,Hk,D,page", [([9000, 30, 5000], [1, 1, 1], 8, 2, 128, 16), ([6000], [3], 16, 2, 64, 64), ([4100, 4000], [70, 5], 4, 2, 96, 32), ([3500], [200], 2, 1, 128, 16)])
def test_attend_in_slices(lengths, fresh, Hq, Hk, D, page):
    a = make_attend(lengths, fresh, Hq, Hk, D, page, seed=7)
    first = check_attend(a)
    # however the tokens are dealt: a table with many places, a longest that is too short
    wide = a | dict(table=torch.nn.functional.pad(a["table"], (0, 3000), value=-1))
    for longest in (None, 100, max(lengths), 2 ** 31 - 1):
        got = check_attend(wide, longest=longest)
        assert bool(((got.double() - first.double()).abs() <= 2 * (2.0 ** -8 * first.double().abs() + 0.01)).all())
    check_attend(wide, window=300)


@pytest.mark.gpu
@pytest.mark.parametrize("requests,Hq,Hk", [(64, 4, 2), (65, 4, 2), (200, 4, 1), (130, 24, 2)])
def test_attend_many_requests(requests, Hq, Hk):
    rng = np.random.default_rng(requests)
    lengths = rng.integers(0, 90, requests)
    lengths[[3, requests - 2]] = 3500, 1300                                       # in slices, beside short ones
    fresh = np.minimum(rng.integers(0, 4, requests), lengths)
    a = make_attend(lengths.tolist(), fresh.tolist(), Hq, Hk, 64, 16, seed=requests)
    check_attend(a)
    check_attend(a, longest=1000)                                                 # ... in none
    check_attend(a, window=40)


@pytest.mark.gpu
def test_attend_more_than_16_blocks_of_a_wavefront():
    check_attend(make_attend([5000, 4200] + [10] * 14, [1] * 16, 64, 64, 32, 16, seed=1))


@pytest.mark.gpu
def test_attend_windows_that_see_everything():
    a = make_attend([3, 300], [5, 40], 4, 2, 64)
    want = check_attend(a)
    for window in (301, 2 ** 30, 2 ** 31 - 1):
        assert torch.equal(check_attend(a, window=window), want)


# (what a window leaves of a length near 2^31 begins where 32 bits end)
@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk,fresh,longest", [(4, 2, 1, None), (4, 2, 6, None), (64, 64, 1, 100), (64, 64, 130, None)])
def test_attend_windows_of_lengths_far_past_the_table(Hq, Hk, fresh, longest):
    a = make_attend([640, 704, 1296, 656], [fresh] * 4, Hq, Hk, 64)
    a["lengths"] = ints([2 ** 31 - 1, 2 ** 31 - 90, 1296, 2 ** 31 - 400])
    for window in (1, 17, 65, 300, 2 ** 30, 2 ** 31 - 1):
        check_attend(a, window=window, longest=longest)


# Calls of many short requests: wavefronts with heads of their own (also where `longest` is not true)
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attend_many_short_requests(D, dtype):
    a = make_attend([70, 300, 1, 0, 129, 64, 17, 1090], [1, 1, 1, 0, 3, 2, 1, 1], 64, 64, D, 16, dtype, seed=D)
    check_attend(a, longest=100)
    check_attend(a, longest=100, window=65)


@pytest.mark.gpu
@pytest.mark.parametrize("requests,Hq,Hk,fresh", [(60, 20, 5, 1), (40, 48, 6, 3), (60, 35, 7, 2), (80, 4, 4, 4)])
def test_attend_many_short_requests_of_shared_heads(requests, Hq, Hk, fresh):
    rng = np.random.default_rng(requests + Hk)
    lengths = rng.integers(0, 130, requests)
    new = np.minimum(rng.integers(0, fresh + 1, requests), lengths)
    a = make_attend(lengths.tolist(), new.tolist(), Hq, Hk, 64, 16, seed=requests)
    check_attend(a, longest=60)
    padded = a | dict(q=torch.cat([a["q"], gpu(6, Hq, 64, seed=50, dtype="bf16")]))
    check_attend(padded, longest=60)
    check_attend(padded, longest=60, out=torch.full_like(padded["q"], 5.0))
    a["table"][::3, 1:3], a["table"][1::7, 0] = -1, len(a["cache"])
    check_attend(a, longest=60)
    v = a["v"].clone()
    v[::5, 1] = NAN
    check_attend(fill(a | dict(v=v), 16), longest=60)


# Calls of many rows in many workgroups: wavefronts with rows of their own
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attend_many_rows(D, dtype):
    a = make_attend([250, 391, 171], [240, 391, 150], 64, 64, D, 48, dtype, seed=D)
    check_attend(a)
    check_attend(a, window=65)


@pytest.mark.gpu
def test_attend_many_rows_of_shared_heads_and_what_is_not_there():
    a = make_attend([260, 30, 401, 64, 0], [220, 30, 130, 5, 0], 192, 32, 64, 16, seed=3)
    want = check_attend(a)
    check_attend(a, window=1)
    check_attend(a, window=130)
    T = len(a["q"])
    wide = gpu(T + 9, 200, 65, seed=4, dtype="bf16")
    q = wide[:T, 3:195, 1:]
    q.copy_(a["q"])
    padded = a | dict(q=wide[:, 3:195, 1:])
    assert torch.equal(check_attend(padded)[:T], want)
    before = wide.clone()
    assert torch.equal(check_attend(padded, out=padded["q"])[:T], want)          # in place, rows behind the last request as they were
    wide[:T, 3:195, 1:] = before[:T, 3:195, 1:]
    assert torch.equal(wide, before)
    a["table"][0, 2], a["table"][2, 7], a["table"][2, 20] = -1, len(a["cache"]), 2 ** 31 - 1
    check_attend(a)
    k, v = a["k"].clone(), a["v"].clone()
    v[int(a["table"][0, 15]) * 16 + 5, 3] = NAN                                   # position 245 of the first request, a head of the cache
    k[int(a["table"][2, 19]) * 16 + 3, 7, 5] = -INF
    check_attend(fill(a | dict(k=k, v=v), 16))
    check_attend(fill(a | dict(k=k, v=v), 16), window=100)
    long = make_attend([1500, 300], [130, 300], 96, 96, 64, 16, seed=5)
    check_attend(long | dict(table=torch.nn.functional.pad(long["table"], (0, 500), value=-1)))


@pytest.mark.gpu
def test_attend_rows_that_see_nothing_and_padding():
    a = make_attend([3, 40, 0, 20], [5, 2, 2, 1], 8, 2, 64)     # more rows than tokens: the first have no position
    got = check_attend(a)
    assert bool((got[:2] == 0).all() and (got[7:9] == 0).all())
    padded = a | dict(q=torch.cat([a["q"], gpu(6, 8, 64, seed=50, dtype="bf16")]))
    assert bool((check_attend(padded)[10:] == 0).all())
    check_attend(padded, out=torch.full_like(padded["q"], 5.0))  # left as they were
    late = padded | dict(starts=padded["starts"] + 3)            # rows before the first request
    check_attend(late)
    check_attend(late, out=torch.full_like(padded["q"], 5.0))
    nobody = a | dict(lengths=a["lengths"] * 0)
    assert bool((check_attend(nobody) == 0).all())
    none = ops.kv4_attention(a["q"], a["cache"], a["table"][:0], a["lengths"][:0], ints([0]))
    assert bool((none == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fresh", [1, 4, 120])
def test_attend_pages_that_are_not_there(fresh):
    lengths = [200, 130, 150]
    a = make_attend(lengths, [fresh] * 3, 4, 2, 64)
    a["table"][0, 0], a["table"][0, 3], a["table"][1, 8], a["table"][2, :] = -1, len(a["cache"]), 2 ** 31 - 1, -2 ** 31
    got = check_attend(a)
    assert bool((got[2 * fresh:] == 0).all())
    narrow = make_attend(lengths, [fresh] * 3, 4, 2, 64, columns=5)    # lengths past the table
    check_attend(narrow)
    check_attend(narrow, window=100)
    check_attend(make_attend([20, 30], [2, 2], 4, 2, 64, columns=0))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 1000])
@pytest.mark.parametrize("fresh", [1, 6, 130])
def test_attend_windows(window, fresh):
    check_attend(make_attend([300, 131, 900], [fresh] * 3, 4, 2, 64, seed=window), window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("fresh", [1, 5, 140])
def test_attend_nan_reaches_the_rows_that_see_it(fresh):
    a = make_attend([400, 150], [fresh, fresh], 4, 2, 64)
    k, v = a["k"].clone(), a["v"].clone()
    slot = lambda b, j: int(a["table"][b, j // 16]) * 16 + j % 16  # noqa: E731
    v[slot(0, 398), 0] = NAN            # seen by the last two rows of its request, through one head of the cache
    k[slot(1, 149), 1, 3] = INF         # ... by the last row
    check_attend(fill(a | dict(k=k, v=v), 16))
    check_attend(fill(a | dict(k=k, v=v), 16), window=2)
    q = a["q"].clone()
    q[0, 0, 5], q[1, 1, 6] = NAN, INF
    check_attend(a | dict(q=q))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("fresh", [1, 100])
def test_attend_odd_values(dtype, fresh):
    a = make_attend([500, 130], [fresh, fresh], 4, 2, 64, dtype=dtype, q_scale=6.0)     # few tokens that count
    check_attend(a)
    check_attend(a, scale=3.0)
    check_attend(a, scale=0.0)
    check_attend(a, scale=-0.25)
    check_attend(a | dict(q=a["q"] * 0))
    check_attend(a | dict(q=a["q"] * 1e-6), scale=1e4)
    v = a["v"].clone()
    v[::3] *= 1e-4                      # steps of values far from each other
    v[1::3] *= 50.0
    v[2::7] = 1.25                      # ... of none
    check_attend(fill(a | dict(v=v), 16))
    check_attend(fill(a | dict(v=v * 0 + 2), 16))
    k = a["k"] * 0 + 1                  # every score the same
    check_attend(fill(a | dict(k=k), 16))
    if dtype == "bf16":
        check_attend(fill(a | dict(v=a["v"] * 1e30), 16))
        check_attend(fill(a | dict(v=a["v"] * 1e-30), 16))
        check_attend(fill(a | dict(k=a["k"] * 1e20, q=a["q"] * 1e-20), 16))


@pytest.mark.gpu
@pytest.mark.parametrize("fresh", [1, 70])
def test_attend_strides_and_in_place(fresh):
    a = make_attend([300, 100, 9], [fresh, fresh, 3], 6, 2, 96, page=32)
    want = check_attend(a)
    T = len(a["q"])
    qkv = gpu(T, 10, 97, seed=4, dtype="bf16")
    q = qkv[:, 2:8, 1:]
    q.copy_(a["q"])
    before = qkv.clone()
    y = gpu(6, T, 96, seed=5, dtype="bf16").transpose(0, 1)
    assert check_attend(a, q=q, out=y) is y and torch.equal(y, want)
    assert ops.kv4_attention(q, a["cache"], a["table"], a["lengths"], a["starts"], out=q) is q and torch.equal(q, want)
    q.copy_(a["q"])
    assert torch.equal(qkv, before)     # nothing beside it was touched
    wide = torch.full((3, 40), 77, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + a["table"].shape[1]] = a["table"]
    assert torch.equal(check_attend(a | dict(table=wide[:, 5:5 + a["table"].shape[1]])), want)
    layers = torch.zeros(len(a["cache"]), 3, *a["cache"].shape[1:], dtype=torch.bfloat16, device="cuda")
    layers[:, 1] = a["cache"]
    assert torch.equal(check_attend(a | dict(cache=layers[:, 1])), want)


@pytest.mark.gpu
@pytest.mark.parametrize("fresh", [1, 70])
def test_attend_past_32_bits(fresh):
    a = make_attend([40, 100], [fresh if fresh == 1 else 30, fresh], 4, 2, 64, page=112)
    want = check_attend(a)
    size, far = a["cache"].shape[2], 2 ** 31 + 8
    big = torch.zeros(3 * far + 2 * size, dtype=torch.bfloat16, device="cuda")
    cache = torch.as_strided(big, a["cache"].shape, (far, size, 1))
    cache.copy_(a["cache"])
    assert torch.equal(check_attend(a | dict(cache=cache)), want)


# ---------------------------------------------------------------------------------------------------------------- how they are called
@pytest.mark.gpu
@pytest.mark.parametrize("ordinary", [True, False])
def test_python_calls_both_ways(ordinary, monkeypatch):
    a = make_attend([30, 60], [1, 1], 4, 2, 64)
    s = make_slots([30, 61], [30, 1], 16)
    q, k = gpu(2, 4, 64, dtype="bf16"), gpu(2, 2, 64, seed=1, dtype="bf16")
    calls = [lambda: ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"], a["starts"], window=40, longest=64), lambda: ops.qk_norm_rope(q, k, ints([3, 4]), turns(9, 64)),
             lambda: ops.kv4_read(a["cache"], ints([1, 2, 3]), 64), lambda: ops.page_slots(*s, 16, 40), lambda: ops.kv4_write(a["cache"].clone(), k, k, ints([0, 7]))]
    want = [c() for c in calls]
    if not ordinary:  # the calls that the launch extension leaves to Python
        monkeypatch.setattr(ops, "_fast", False)
    flat = lambda x: x if isinstance(x, tuple) else (x,)  # noqa: E731
    for c, w in zip(calls, want):
        assert all(torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x, y.view(torch.int16) if y.dtype == torch.bfloat16 else y) for x, y in zip(flat(c()), flat(w)))
    for wrong, error, says in [(lambda: ops.kv4_attention(a["q"].float(), a["cache"], a["table"], a["lengths"], a["starts"]), ValueError, "q is f32, not bf16"),
                               (lambda: ops.kv4_attention(a["q"], a["cache"], a["table"].long(), a["lengths"], a["starts"]), ValueError, "int64"),
                               (lambda: ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"].cpu(), a["starts"]), TypeError, "GPU memory"),
                               (lambda: ops.page_slots(s[0], s[1], s[2], s[3], s[4], 0, 4), ValueError, "a page of 0"),
                               (lambda: ops.page_slots(s[0], s[1], s[2], s[3], s[4], 2 ** 32 + 16, 4), ValueError, "page is"),
                               (lambda: ops.kv4_read(a["cache"], ints([1]), 40), NotImplementedError, "heads of 40"),
                               (lambda: ops.kv4_read(a["cache"], ints([1]), 2 ** 33), ValueError, "dim is"),
                               (lambda: ops.kv4_write(a["cache"], k.half(), k, ints([0, 1])), ValueError, "k is f16"),
                               (lambda: ops.qk_norm_rope(q, k, ints([0, 1]), turns(9, 64), out=(q, None)), ValueError, "pair"),
                               (lambda: ops.qk_norm_rope(q, k, ints([0, 1]), turns(9, 64), k[0, 0]), ValueError, "w_k is missing"),
                               (lambda: ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"], a["starts"], window=2 ** 40), ValueError, "window is")]:
        with pytest.raises(error, match=says):
            wrong()


@pytest.mark.gpu
def test_gradients_and_tangents_are_refused():
    from torch.autograd import forward_ad as fwd

    a = make_attend([30, 60], [1, 1], 4, 2, 64)
    q, k = gpu(2, 4, 64, dtype="bf16"), gpu(2, 2, 64, seed=1, dtype="bf16")
    calls = [lambda x: ops.kv4_attention(x, a["cache"], a["table"], a["lengths"], a["starts"]), lambda x: ops.qk_norm_rope(x, k, ints([3, 4]), turns(9, 64)),
             lambda x: ops.kv4_write(a["cache"], k, x[:, :2], ints([0, 7]))]
    for call in calls:
        with pytest.raises(NotImplementedError, match="no backward"):
            call(q.clone().requires_grad_())
        with torch.no_grad():
            call(q.clone().requires_grad_())
        with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode tangent"):
            call(fwd.make_dual(q, torch.ones_like(q)))


@pytest.mark.gpu
@pytest.mark.parametrize("ordinary", [True, False])
def test_autograd_notices_what_was_written(ordinary, monkeypatch):
    if not ordinary:
        monkeypatch.setattr(ops, "_fast", False)
    a = make_attend([30, 60], [1, 1], 4, 2, 64)
    q, k = gpu(2, 4, 64, dtype="bf16"), gpu(2, 2, 64, seed=1, dtype="bf16")
    s = make_slots([30, 61], [30, 1], 16)
    for x, write in ((q, lambda: ops.qk_norm_rope(q, k, ints([3, 4]), turns(9, 64), out=(q, k))), (k, lambda: ops.qk_norm_rope(q, k, ints([3, 4]), turns(9, 64), out=(q, k))),
                     (q, lambda: ops.kv4_attention(q, a["cache"], a["table"], a["lengths"], a["starts"], out=q)), (a["cache"], lambda: ops.kv4_write(a["cache"], k, k, ints([0, 7]))),
                     (s[0], lambda: ops.page_slots(*s, 16, 40))):
        version = x._version
        write()
        assert x._version > version


@pytest.mark.gpu
def test_two_streams_at_once():
    a = [make_attend([3000, 700], [1, 1], 8, 2, 128, seed=s) for s in (1, 2)]
    want = [ops.kv4_attention(x["q"], x["cache"], x["table"], x["lengths"], x["starts"]) for x in a]
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, x in enumerate(a):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.kv4_attention(x["q"], x["cache"], x["table"], x["lengths"], x["starts"]))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i in (0, 1) for y in got[i])


class Session:
    """A batch of requests that grows: what a serving loop keeps, and one step of all operators for it."""

    def __init__(self, requests, pages, Hq=8, Hk=2, D=64, page=16, seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.Hq, self.Hk, self.D, self.page = Hq, Hk, D, page
        self.table = torch.full((requests, 12), -1, dtype=torch.int32, device="cuda")
        self.free, self.count = torch.randperm(pages, generator=g, device="cuda").int(), ints([pages])
        self.cache = ops.kv4_cache(pages, Hk, D, page=page)
        self.cos_sin, self.w = turns(200, D), [1.0 + gpu(D, seed=seed + s, scale=0.2) for s in (1, 2)]
        self.lengths = torch.zeros(requests, dtype=torch.int32, device="cuda")

    def step(self, qkv, fresh):
        lengths = self.lengths + fresh
        slots, positions, owners, starts, left = ops.page_slots(self.table, lengths, fresh, self.free, self.count, self.page, len(qkv))
        q, k, v = qkv[:, :self.Hq], qkv[:, self.Hq:self.Hq + self.Hk], qkv[:, self.Hq + self.Hk:]
        q, k = ops.qk_norm_rope(q, k, positions, self.cos_sin, *self.w)
        ops.kv4_write(self.cache, k, v, slots)
        y = ops.kv4_attention(q, self.cache, self.table, lengths, starts)
        self.lengths.copy_(lengths)
        self.count.copy_(left)
        return y, q, k, v, slots, positions, owners, starts


@pytest.mark.gpu
def test_steps_of_a_growing_batch():
    # prompts, then a token each, then a few each: what the steps before have written is there, and attention is that of the whole sequences
    s = Session(3, 40)
    kept = [[torch.empty(0, 2, 64, dtype=torch.bfloat16, device="cuda")] * 2 for _ in range(3)]
    for n, fresh in enumerate([[30, 0, 70], [1, 20, 1], [1, 1, 1], [4, 3, 0], [1, 1, 1], [16, 16, 16]]):
        rows = sum(fresh) + n
        y, q, k, v, slots, positions, owners, starts = s.step(gpu(rows, 12, 64, seed=n, dtype="bf16"), ints(fresh))
        lengths = s.lengths.tolist()
        used = s.table[s.table >= 0]
        assert len(used.unique()) == len(used) == sum(-(-m // 16) for m in lengths) and int(s.count[0]) == 40 - len(used)
        pad = slice(sum(fresh), rows)
        assert bool((y[pad] == 0).all() and (q[pad] == 0).all() and (slots[pad] == -1).all() and (owners[pad] == -1).all())
        at, parts = starts.tolist(), []
        for b in range(3):
            own = slice(at[b], at[b + 1])
            assert owners[own].tolist() == [b] * fresh[b] and positions[own].tolist() == list(range(lengths[b] - fresh[b], lengths[b]))
            kept[b] = [torch.cat([old, new[own]]) for old, new in zip(kept[b], (k, v))]
            parts.append(kept[b])
        # the same from sequences that lie one behind another
        each = [-(-m // 16) for m in lengths]
        pages = torch.split(torch.arange(sum(each), dtype=torch.int32, device="cuda"), each)
        table = torch.full((3, max(each)), -1, dtype=torch.int32, device="cuda")
        for b in range(3):
            table[b, :each[b]] = pages[b]
        whole = [torch.cat([torch.nn.functional.pad(p[i], (0, 0, 0, 0, 0, each[b] * 16 - lengths[b])) for b, p in enumerate(parts)]) for i in (0, 1)]
        a = dict(q=q, table=table, lengths=s.lengths.clone(), starts=starts, k=whole[0], v=whole[1], page=16)
        want, lim, real = attend_exact(a, 0.125, None)
        assert bool(((y.double() - want).abs() <= lim)[real].all())
        stored = ops.kv4_read(s.cache, slots, 64)
        assert same(stored[0][:pad.start], held_values(k[:pad.start])) and same(stored[1][:pad.start], held_values(v[:pad.start]))


@pytest.mark.gpu
def test_steps_in_graphs():
    sessions, rows = [Session(4, 60, seed=s) for s in (0, 5)], 40
    plain = [Session(4, 60, seed=s) for s in (0, 5)]
    qkv, fresh = [gpu(rows, 12, 64, seed=9, dtype="bf16") for _ in sessions], [ints([0] * 4) for _ in sessions]
    for s, x, f in zip(sessions, qkv, fresh):  # (a step of nothing: what is loaded lazily is)
        s.step(x, f)
    torch.cuda.synchronize()
    graphs = []
    for s, x, f in zip(sessions, qkv, fresh):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            made = s.step(x, f)
        graphs.append((g, made))
    for n, new in enumerate([[9, 0, 20, 5], [1, 1, 1, 1], [0, 33, 1, 1], [1, 1, 1, 1], [2, 0, 5, 7]]):
        for i, (g, made) in enumerate(graphs):
            x = gpu(rows, 12, 64, seed=20 * n + i, dtype="bf16")
            qkv[i].copy_(x)
            fresh[i].copy_(ints(new))
            g.replay()
            torch.cuda.synchronize()
            eager = plain[i].step(x, ints(new))
            assert all(torch.equal(a, b) for a, b in zip(made, eager))
            assert torch.equal(sessions[i].cache.view(torch.int16), plain[i].cache.view(torch.int16)) and torch.equal(sessions[i].table, plain[i].table)
            assert torch.equal(sessions[i].count, plain[i].count) and torch.equal(sessions[i].lengths, plain[i].lengths)


@pytest.mark.gpu
def test_results_do_not_change_from_call_to_call():
    a = make_attend([2000, 300, 77], [1, 1, 1], 8, 2, 128)
    b = make_attend([400, 300], [150, 120], 8, 2, 128)
    c, d = make_attend([250, 391, 171], [240, 391, 150], 64, 64, 64), make_attend([70, 300, 1, 129] * 3, [1] * 12, 64, 64, 64)
    for x in (a, b, c, d):
        call = lambda: ops.kv4_attention(x["q"], x["cache"], x["table"], x["lengths"], x["starts"], longest=100 if x is d else None)  # noqa: E731, B023
        first = call()
        for _ in range(5):
            assert torch.equal(call(), first)


# A step with more new tokens than rows: those that have one are where `page_slots` says, and see nothing behind themselves (never written, the others are NaN here)
@pytest.mark.gpu
@pytest.mark.parametrize("lengths,fresh,rows,Hq,Hk,longest", [
    ([5], [5], 3, 4, 2, None), ([40, 90, 33], [1, 7, 2], 4, 8, 2, None), ([40, 90, 33], [1, 7, 2], 8, 8, 2, None),
    ([9000, 30], [40, 1], 17, 8, 2, None),                                                           # in slices
    ([70, 300, 1, 129], [3, 5, 1, 4], 7, 64, 64, 60),                                                # wavefronts with heads of their own
    ([250, 391, 171], [240, 391, 150], 500, 64, 64, None), ([250, 391], [240, 391], 301, 192, 32, None),  # ... with rows of their own
])
def test_attend_of_fewer_rows_than_new_tokens(lengths, fresh, rows, Hq, Hk, longest):
    a = make_attend(lengths, fresh, Hq, Hk, 64, seed=rows)
    table = a["table"].clone()
    taken = [a["table"][b, c].item() for b, (n, f) in enumerate(zip(lengths, fresh)) for c in range(-(-(n - f) // 16), -(-n // 16))]
    slots, positions, _, starts, _ = ops.page_slots(table, a["lengths"], ints(fresh), ints(taken[::-1]), ints([len(taken)]), 16, rows)
    assert torch.equal(table, a["table"]) and torch.equal(starts, a["starts"])
    at, want_at = starts.tolist(), []
    for n, f, first in zip(lengths, fresh, at):
        want_at += list(range(n - f, n))
    assert positions.tolist() == want_at[:rows]
    k, v = a["k"].clone(), a["v"].clone()
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        for j in range(n - f + min(max(rows - at[b], 0), f), n):
            k[int(table[b, j // 16]) * 16 + j % 16], v[int(table[b, j // 16]) * 16 + j % 16] = NAN, NAN
    kept = fill(a | dict(k=k, v=v), 16)
    assert bool((slots >= 0).all())
    for window in (None, 1, 20):
        want, lim, _ = attend_exact(a, 0.125, window)
        got = ops.kv4_attention(a["q"][:rows], kept["cache"], table, a["lengths"], starts, window=window, longest=longest)
        assert bool(((got.double() - want[:rows]).abs() <= lim[:rows]).all())


@pytest.mark.gpu
def test_steps_with_more_new_tokens_than_rows():
    # all of a step's operators: the first rows of a step that has them all
    fresh = [30, 1, 70]
    whole, cut = Session(3, 40), Session(3, 40)
    for n, rows in enumerate([101, 100, 60, 31, 30, 7]):
        x = gpu(101, 12, 64, seed=n, dtype="bf16")
        for s in (whole, cut):
            s.table.fill_(-1), s.lengths.zero_(), s.count.fill_(40)
        want, got = whole.step(x, ints(fresh)), cut.step(x[:rows], ints(fresh))
        for a, b in zip(want[1:7], got[1:7]):
            assert torch.equal(a[:rows], b)
        # (each within half a step of bf16 and 2^-11 of the codes' part of what is exact, and that is less than 15 steps, some 6)
        assert bool(((got[0].double() - want[0][:rows].double()).abs() <= 2.0 ** -6 * want[0][:rows].double().abs() + 0.02).all())


# Calls of each kind: tiles of 4, of 8 and of 16 rows, slices, wavefronts with heads and with rows of their own
KINDS = {"4": ([300, 1, 70], [1, 1, 1], 8, 2, None), "8": ([300, 1, 70], [1, 1, 1], 16, 2, None), "16": ([300, 40], [40, 40], 8, 2, None), "slices": ([6000, 1], [1, 1], 8, 2, None),
         "heads": ([70, 300, 1, 0, 129, 64, 17, 1090], [1, 1, 1, 0, 3, 2, 1, 1], 64, 64, 100), "rows": ([250, 391, 171], [240, 391, 150], 64, 64, None)}


# Scores past 2^24, the largest of 32 bits between which whole numbers lie: those that are the same count the same ...
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("D,size", [(128, 4000.0), (64, 8000.0), (32, 60000.0)])
def test_attend_large_scores_that_are_the_same(D, size, dtype, kind):
    lengths, fresh, Hq, Hk, longest = KINDS[kind]
    a = make_attend(lengths, fresh, Hq, Hk, D, 16, dtype, seed=D)
    sign = torch.where(torch.arange(len(a["q"]) * Hq, device="cuda") % 3 == 0, -1.0, 1.0).reshape(-1, Hq, 1)
    a = fill(a | dict(k=torch.full_like(a["k"], size), q=(torch.full_like(a["q"], size) * sign).to(a["q"].dtype)), 16)
    for window in (None, 30):
        want, lim, _ = attend_exact(a, 0.0, window)  # (by the same scores without them)
        got = ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"], a["starts"], window=window, longest=longest)
        assert bool(((got.double() - want).abs() <= lim).all())


# ... and of others the largest alone: a key's elements are one number of -32 to 32 and three times that, and scores its products with 2^23 and more
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_attend_large_scores_of_which_one_counts(sign, dtype, kind):
    lengths, fresh, Hq, Hk, longest = KINDS[kind]
    a = make_attend(lengths, fresh, Hq, Hk, 64, 16, dtype, seed=3)
    level = (torch.arange(len(a["k"]), device="cuda") * 7 % 32 + 1).to(a["k"].dtype)
    level[::2] *= -1
    each = 1 + 2 * (torch.arange(64, device="cuda") % 2).to(level.dtype)  # (three times as much, within 2^-8 as it is held: no other order)
    a = fill(a | dict(k=(level[:, None, None] * each).expand_as(a["k"]).contiguous(), q=torch.full_like(a["q"], 32768.0 * sign)), 16)
    got = ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"], a["starts"], scale=4.0, longest=longest)
    assert bool(got.isfinite().all())
    code, step, low = held(a["v"])
    v, at = code * step + low, a["starts"].tolist()
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        j = torch.arange(n, device="cuda")
        slots = a["table"][b].long()[j // 16] * 16 + j % 16
        z = level[slots].double() * sign
        for r in range(f):
            seen = slots[:n - f + r + 1]
            chosen = seen[z[:n - f + r + 1] == z[:n - f + r + 1].max()]
            want = v[chosen].mean(dim=0).repeat_interleave(Hq // Hk, dim=0)
            # the values in 32 bits; weights that are the same, of which each may be off by 2^-11 of 15 steps; sums of as many; the rounding
            lim = 2.0 ** -11 * 15 * step[chosen].amax() + 2.0 ** -16 * v[chosen].abs().amax() + half(dtype) * want.abs()
            assert bool(((got[at[b] + r].double() - want).abs() <= lim).all())


# Elements of q near the end of bf16, with keys that make ordinary scores of them; scales at both ends of 32 bits
@pytest.mark.gpu
@pytest.mark.parametrize("kind", list(KINDS))
@pytest.mark.parametrize("q_scale,k_scale,scale", [(1e36, 1e-36, None), (2.0 ** 124, 2.0 ** -124, None), (2.0 ** 100, 2.0 ** -100, 0.3), (1e-20, 1e-6, 1e26), (2.0 ** -100, 1.0, 2.0 ** 100), (1.0, 1e-30, 1e30), (1e30, 1e8, 1e-38),
                                                   (1.0, 1e20, 1e-41), (1e-36, 1e36, None)])
def test_attend_rows_and_scales_near_the_ends(q_scale, k_scale, scale, kind):
    lengths, fresh, Hq, Hk, longest = KINDS[kind]
    a = make_attend(lengths, fresh, Hq, Hk, 64, seed=5)
    a = fill(a | dict(q=(a["q"].float().clamp(-5, 5) * q_scale).bfloat16(), k=(a["k"].float() * k_scale).bfloat16()), 16)
    assert bool(a["q"].isfinite().all() and a["k"].isfinite().all())
    check_attend(a, scale=scale, longest=longest)
    # rows of all sizes side by side
    mixed = a["q"].clone()
    mixed[:, ::3] = (mixed[:, ::3].float() / q_scale).bfloat16()
    check_attend(a | dict(q=mixed), scale=scale, longest=longest)


@pytest.mark.gpu
def test_attend_rows_whose_sum_is_not_finite():
    a = make_attend([30, 70], [1, 40], 4, 2, 128, seed=5)
    q = a["q"].abs().clamp(0.5, 1.0) * 2.0 ** 127  # 32 bits hold no sum of four
    check_attend(fill(a | dict(q=q, k=a["k"] * 2.0 ** -120), 16))


# (no GPU needed: tokens that a row of the table has places for and that the kernel would leave out)
@pytest.mark.parametrize("columns,page,longest,refused", [((1 << 26) - 1, 16, 0, False), (1 << 26, 16, 0, True), (1 << 26, 16, 1000, True), ((1 << 14) - 1, 1 << 16, 0, False), (1 << 14, 1 << 16, 0, True), (1 << 30, 16, 0, True)])
def test_tables_with_places_for_2_30_tokens_are_refused(columns, page, longest, refused):
    bytes_ = ctypes.c_size_t()
    status = N.lib().tts_kv4_attention_workspace(tensor(BF16, 1, 8, 32, ptr=FAR[1]), cache_t(pages=10, page=page, dim=32), tensor(I32, 1, columns, ptr=FAR[2]), 0, longest, ctypes.byref(bytes_))
    assert status == (N.TTS_UNSUPPORTED if refused else N.TTS_OK)
    if refused:
        assert f"places for {columns * page} tokens" in N.lib().tts_last_error().decode()


# Values of a token that most rows do not see, far larger than theirs, or none: rows that do not see it are what they are without it, bit by bit
@pytest.mark.gpu
@pytest.mark.parametrize("lengths,fresh,Hq,Hk,longest", [([300, 40], [40, 40], 8, 2, None), ([9, 130], [5, 3], 8, 2, None), ([200, 70], [3, 2], 6, 3, None), ([6000, 2000], [3, 3], 16, 2, None), ([3500, 90], [200, 90], 2, 1, None),
                                                         ([70, 300, 1, 0, 129, 64, 17, 1090], [1, 1, 1, 0, 3, 2, 1, 3], 64, 64, 100), ([250, 391, 171], [240, 391, 150], 64, 64, None), ([260, 401], [220, 130], 192, 32, None)])
@pytest.mark.parametrize("dtype,window", [("bf16", None), ("bf16", 2), ("bf16", 70), ("fp16", None), ("fp16", 70)])
def test_attend_of_large_values_that_rows_do_not_see(lengths, fresh, Hq, Hk, longest, dtype, window):
    a = make_attend(lengths, fresh, Hq, Hk, 64, 16, dtype, seed=sum(lengths))
    if dtype == "fp16":
        a = fill(a | dict(v=a["v"] * 2.0 ** -12), 16)
    plain = check_attend(a, window=window, longest=longest)
    starts = a["starts"].tolist()
    for size, back in [(1e10, 1), (1e10, 2), (2.0 ** 24, 65), (2.0 ** 120, 1), (NAN, 1), (INF, 65)]:  # the last token, or one that some rows no longer see
        if dtype == "fp16":
            size = min(size, 2.0 ** 24)
        v, sees = a["v"].clone(), torch.zeros(len(a["q"]), dtype=torch.bool, device="cuda")
        for b, (n, f) in enumerate(zip(lengths, fresh)):
            j = n - back
            if j < 0:
                continue
            slot = int(a["table"][b, j // 16]) * 16 + j % 16
            v[slot] = (v[slot].float() * size).to(v.dtype)
            i = torch.arange(n - f, n, device="cuda")
            sees[starts[b]:starts[b + 1]] = (i >= j) & ((i - j < window) if window else True)
        x = fill(a | dict(v=v), 16)
        if size == 1e10 or (dtype == "fp16" and back == 2):
            got = check_attend(x, window=window, longest=longest)
        else:
            got = ops.kv4_attention(x["q"], x["cache"], x["table"], x["lengths"], x["starts"], window=window, longest=longest)
        assert torch.equal(got[~sees].view(torch.int16), plain[~sees].view(torch.int16))
        assert size == size or bool(got[sees].isnan().all())


def codes_part(a, scale, window):
    """What the codes' part of the values, code times step, comes to in each row: what the rounding of the weights is of."""
    out, starts, group = torch.zeros(a["q"].shape, dtype=torch.float64, device="cuda"), a["starts"].tolist(), a["q"].shape[1] // a["k"].shape[1]
    for b, n in enumerate(a["lengths"].tolist()):
        j = torch.arange(n, device="cuda")
        slots, i = a["table"][b].long()[j // a["page"]] * a["page"] + j % a["page"], torch.arange(n - starts[b + 1] + starts[b], n, device="cuda")
        seen = (j[None] <= i[:, None]) & ((j[None] > i[:, None] - window) if window else True)
        for h in range(a["q"].shape[1]):
            code, step, low = held(a["k"][slots, h // group])
            z = a["q"][starts[b]:starts[b + 1], h].double() @ (code * step + low).t() * scale
            code, step, _ = held(a["v"][slots, h // group])
            out[starts[b]:starts[b + 1], h] = torch.softmax(torch.where(seen, z, -INF), dim=1) @ (code * step)
    return out


# The weights of an fp16 cache are the sum of two 16-bit numbers, and within 2^-22 (one of them: 2^-11).  Tokens by twos have the same key and opposite values, of which nothing is left but what 4 bits make
# of them, while the codes' parts of both add up to 15 steps; rows see few, so that the bounds of sums and scores are small beside 2^-12 of that
@pytest.mark.gpu
@pytest.mark.parametrize("D", [32, 64])
@pytest.mark.parametrize("lengths,fresh,Hq,Hk,longest,window", [([4, 6, 8, 12] * 12, [1] * 48, 32, 8, None, None), ([4, 6, 8, 12] * 12, [1] * 48, 32, 4, None, None), ([4, 6, 8, 12] * 12, [4, 1, 5, 12] * 12, 16, 2, None, None),
                                                                ([300, 800, 20], [3, 1, 20], 4, 2, None, 8), ([4, 8, 300, 6] * 8, [1] * 32, 16, 4, 16, 8), ([250, 390, 170], [240, 390, 150], 64, 64, None, 6)])
def test_attend_fp16_weights_in_two_parts(lengths, fresh, Hq, Hk, longest, window, D):
    a = make_attend(lengths, fresh, Hq, Hk, D, 16, "fp16", seed=D, q_scale=0.1)
    k, v = a["k"].clone(), a["v"].clone()
    k[1::2], v[1::2] = k[::2], -v[::2]
    a = fill(a | dict(k=k, v=v), 16)
    scale = D ** -0.5
    want, lim, real = attend_exact(a, scale, window)
    one, two = 2.0 ** -11, 2.0 ** -21
    lim = lim - (one - two) * (1 + half("fp16")) * codes_part(a, scale, window)
    got = ops.kv4_attention(a["q"], a["cache"], a["table"], a["lengths"], a["starts"], window=window, longest=longest)
    off = (got.double() - want).abs()[real]
    assert bool((off <= lim[real]).all()), f"off by {(off / lim[real]).max().item():.2f} of what is allowed"


# Prompts beside single tokens: in one call, and in two with the rows, lengths, tables and starts of each
@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hk", [(8, 2), (64, 32)])
def test_attend_prompts_and_single_tokens_in_one_call_and_in_two(Hq, Hk):
    lengths, fresh = [700, 300, 5000, 40, 1, 2200], [700, 130, 1, 1, 1, 1]
    a = make_attend(lengths, fresh, Hq, Hk, 64, seed=Hq)
    check_attend(a)
    prompts, singles = slice(0, 2), slice(2, 6)
    for part in (prompts, singles):
        first, behind = sum(fresh[:part.start]), sum(fresh[:part.stop])
        x = a | dict(q=a["q"][first:behind], table=a["table"][part], lengths=a["lengths"][part], starts=a["starts"][part.start:part.stop + 1] - first)
        check_attend(x, longest=max(lengths[part]))
