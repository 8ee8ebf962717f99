"""Penalties, biases and masks on logits, against 64 bits.

A touched logit goes through at most four roundings to fp32, each at most 2^-24
of its result, all of which are at most the sum of the sizes of what is added;
then one to its type. A logit that nothing touches keeps its bits.
"""

from __future__ import annotations

import pytest
import torch

from kernelo_b200.kernels.logits import adjust_logits
from kernelo_b200.kernels.softmax import softmax

pytestmark = pytest.mark.gpu

UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
DTYPES = tuple(UNIT)


def make(rows, vocab, dtype, device, *, history=50, biases=5, masks=None, seed=0, prompts=True):
    gen = torch.Generator().manual_seed(seed)
    a = {"logits": (torch.randn(rows, vocab, generator=gen) * 4).to(dtype)}
    if history:
        a["tokens"] = (torch.rand(rows, history, generator=gen).pow(3) * vocab).int().clamp(max=vocab - 1)
        a["token_lens"] = torch.randint(0, history + 1, (rows,), generator=gen, dtype=torch.int32)
        if prompts:
            a["prompt_lens"] = (a["token_lens"] * torch.rand(rows, generator=gen)).int()
        a["repetition"] = torch.rand(rows, generator=gen) + 0.75
        a["frequency"], a["presence"] = (torch.rand(rows, generator=gen) - 0.25 for _ in range(2))
    if biases:
        a["bias_tokens"] = torch.randint(-2, vocab, (rows, biases), generator=gen, dtype=torch.int32)
        a["bias_values"] = torch.randn(rows, biases, generator=gen) * 5
    if masks:
        a["allowed"] = torch.randint(-2 ** 31, 2 ** 31, (masks, -(-vocab // 32)), generator=gen).int()
        a["allowed_rows"] = torch.randint(-1, masks + 1, (rows,), generator=gen, dtype=torch.int32)
    return {n: t.to(device) for n, t in a.items()}


def plain(a):
    """The definition, row by row and token by token in 64 bits; the sizes of its terms; which tokens are touched."""
    a = {n: t.cpu() for n, t in a.items()}
    want, size = a["logits"].double(), a["logits"].double().abs()
    touched = torch.zeros(want.shape, dtype=torch.bool)
    rows, vocab = want.shape
    for r in range(rows):
        if "tokens" in a:
            n = min(max(int(a["token_lens"][r]), 0), a["tokens"].shape[1])
            prompt = int(a["prompt_lens"][r]) if "prompt_lens" in a else 0
            seen, count = set(), {}
            for i, v in enumerate(a["tokens"][r, :n].tolist()):
                if 0 <= v < vocab:
                    seen.add(v)
                    count[v] = count.get(v, 0) + (i >= prompt)
            for v in seen:
                x = float(want[r, v])
                by = float(a["repetition"][r]) if "repetition" in a else 1.0
                x = x / by if x > 0 else x * by
                less = (float(a["frequency"][r]) * count[v] if "frequency" in a else 0.0,
                        float(a["presence"][r]) if "presence" in a else 0.0) if count[v] else (0.0, 0.0)
                size[r, v] += abs(x) + abs(less[0]) + abs(less[1])
                want[r, v], touched[r, v] = x - less[0] - less[1], True
        if "bias_tokens" in a:
            for v, b in dict(zip(a["bias_tokens"][r].tolist(), a["bias_values"][r].tolist())).items():
                if 0 <= v < vocab:
                    want[r, v] += b
                    size[r, v] += abs(b)
                    touched[r, v] = True
        which = -1
        if "allowed" in a:
            which = int(a["allowed_rows"][r]) if "allowed_rows" in a else r
            if 0 <= which < a["allowed"].shape[0]:
                bits = (a["allowed"][which].long()[:, None] >> torch.arange(32)) & 1
                off = bits.flatten()[:vocab] == 0
                want[r, off], size[r, off], touched[r, off] = -torch.inf, 0.0, True
    return want, size, touched


def check(got, a):
    want, size, touched = plain(a)
    dtype, had = a["logits"].dtype, a["logits"].cpu()
    got = got.cpu()
    assert got.dtype == dtype and got.shape == had.shape
    same = (got == had) | (got.isnan() & had.isnan())
    assert same[~touched].all()
    off = 2.0 ** -22 * size
    off = off + UNIT[dtype] * (want.abs() + off) + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133)
    inf = want.isinf()
    assert torch.equal(got.double()[inf], want[inf])
    assert ((got.double() - want).abs() <= off)[touched & ~inf].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 7), (2, 31), (2, 33), (5, 1000), (3, 4097), (2, 8192), (2, 8200),
                                        (7, 32001), (40, 8195), (300, 130)])
def test_sizes(rows, vocab, dtype, device):
    a = make(rows, vocab, dtype, device, masks=rows)
    before = a["logits"].clone()
    check(adjust_logits(**a), a)
    assert torch.equal(a["logits"], before)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("have", ["history", "biases", "masks", "history biases", "history masks", "biases masks", ""])
def test_parts(have, dtype, device):
    kinds = {n: 9 if n in have else 0 for n in ("history", "biases", "masks")}
    a = make(9, 2049, dtype, device, **kinds)
    check(adjust_logits(**a), a)


@pytest.mark.parametrize("without", [("repetition",), ("frequency", "presence"), ("prompt_lens",), ("presence",),
                                     ("repetition", "frequency", "presence"), ("allowed_rows",)])
def test_factors_left_out(without, device):
    a = make(6, 500, torch.float32, device, masks=6)
    a = {n: t for n, t in a.items() if n not in without}
    check(adjust_logits(**a), a)


@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place_and_odd_strides(dtype, device):
    a = make(5, 1003, dtype, device, masks=3)
    want = adjust_logits(**a)
    for room, skip, out_room, out_skip in ((1003, 0, 1003, 0), (1009, 3, 1009, 3), (1016, 1, 1010, 2), (1016, 8, 1016, 0)):
        src = torch.zeros(5, room + skip, device=device, dtype=dtype)
        dst = torch.full((5, out_room + out_skip), 7.0, device=device, dtype=dtype)
        view, out = src[:, skip:skip + 1003], dst[:, out_skip:out_skip + 1003]
        view.copy_(a["logits"])
        rest = a | {"logits": view}
        assert adjust_logits(**rest, out=out) is out and torch.equal(out, want)
        assert (dst[:, :out_skip] == 7).all() and (dst[:, out_skip + 1003:] == 7).all()
        assert adjust_logits(**rest, out=view) is view and torch.equal(view, want)
        assert not src[:, :skip].any() and not src[:, skip + 1003:].any()
    # a history, biases and masks in wider buffers, and one history for all rows
    wide = torch.full((5, 80), 2 ** 31 - 1, dtype=torch.int32, device=device)
    wide[:, 11:61] = a["tokens"]
    masks = torch.zeros(3, 40, dtype=torch.int32, device=device)
    masks[:, 5:5 + a["allowed"].shape[1]] = a["allowed"]
    rest = a | {"tokens": wide[:, 11:61], "allowed": masks[:, 5:5 + a["allowed"].shape[1]]}
    assert torch.equal(adjust_logits(**rest), want)
    rest = a | {"tokens": a["tokens"][:1].expand(5, -1), "token_lens": a["token_lens"][:1].expand(5).contiguous()}
    check(adjust_logits(**rest), rest)


def test_what_lies_outside_is_ignored(device):
    """Ids outside the vocabulary, lengths outside the history, masks that are none of them; nothing past a length is read."""
    a = make(6, 300, torch.bfloat16, device, masks=2)
    gen = torch.Generator().manual_seed(1)
    bad = torch.tensor([-1, 300, 2 ** 31 - 1, -2 ** 31, 299, 0], dtype=torch.int32)
    a["tokens"] = bad[torch.randint(0, 6, (6, 50), generator=gen)].to(device)
    a["token_lens"] = torch.tensor([-5, 0, 1, 50, 51, 2 ** 31 - 1], dtype=torch.int32, device=device)
    a["prompt_lens"] = torch.tensor([3, -1, 0, 2 ** 31 - 1, -2 ** 31, 25], dtype=torch.int32, device=device)
    a["bias_tokens"] = bad[torch.randint(0, 6, (6, 5), generator=gen)].to(device)
    a["allowed_rows"] = torch.tensor([0, 1, 2, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=device)
    check(adjust_logits(**a), a)


@pytest.mark.parametrize("biases", [1, 2, 31, 32, 33, 512, 513, 1500, 16384])
def test_lists_of_biases_with_tokens_listed_twice(biases, device):
    a = make(6, 9001, torch.bfloat16, device, masks=6, biases=biases)
    gen = torch.Generator().manual_seed(5)
    few = torch.randint(-1, 9001, (max(1, biases // 3),), generator=gen, dtype=torch.int32)
    a["bias_tokens"] = few[torch.randint(0, few.numel(), (6, biases), generator=gen)].to(device)
    a["tokens"][:, ::2] = a["bias_tokens"][:, :1].clamp(min=0)
    check(adjust_logits(**a), a)
    view = a["logits"].clone()
    assert torch.equal(adjust_logits(**(a | {"logits": view}), out=view), adjust_logits(**a))


def test_a_token_listed_many_times(device):
    """Counts do not depend on an order, and of several biases the last one counts."""
    a = make(4, 9000, torch.float32, device, history=20000, biases=700)
    a["tokens"][0], a["tokens"][1, ::2] = 17, 8999
    a["token_lens"][:] = 20000
    a["prompt_lens"] = torch.tensor([0, 10000, 20000, 19999], dtype=torch.int32, device=device)
    a["bias_tokens"][0], a["bias_tokens"][1, 10:] = 17, 3
    a["frequency"].fill_(0.01)
    first = adjust_logits(**a)
    check(first, a)
    for _ in range(3):
        assert torch.equal(adjust_logits(**a), first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_and_masks_that_leave_nothing(dtype, device):
    a = make(4, 70, dtype, device, history=40, masks=4)
    low = torch.finfo(dtype).min
    a["tokens"][:] = torch.arange(40, dtype=torch.int32, device=device)
    a["token_lens"][:], a["prompt_lens"][:] = 40, 20
    a["allowed_rows"] = torch.tensor([0, 1, 2, -1], dtype=torch.int32, device=device)
    a["bias_tokens"][:] = -1
    a["allowed"][0], a["allowed"][1], a["allowed"][2] = 0, -1, 0
    a["allowed"][2, 1] = -(1 << 31)  # token 63 alone
    a["logits"][:, ::5], a["logits"][:, 1::5], a["logits"][:, 2::5] = torch.inf, -torch.inf, torch.nan
    a["logits"][:, 3::5] = low
    got = adjust_logits(**a)
    assert (got[0] == -torch.inf).all()
    assert (got[2, :63] == -torch.inf).all() and (got[2, 64:] == -torch.inf).all()
    for r in (1, 3):
        assert (got[r, ::5] == torch.inf).all() and (got[r, 1::5] == -torch.inf).all() and got[r, 2::5].isnan().all()
        assert torch.equal(got[r, 43::5], a["logits"][r, 43::5])
    assert (got[2, 63] == a["logits"][2, 63]) and low == a["logits"][2, 63]
    # probabilities of a row with one token left
    p = softmax(got[2:3].where(got[2:3] != low, torch.zeros_like(got[2:3])))
    assert p[0, 63] == 1 and p.sum() == 1


def test_large_rows_past_32_bit_offsets(device):
    """Rows that begin beyond 2^31 elements."""
    if torch.cuda.get_device_properties(device).total_memory < 40 << 30:
        pytest.skip("needs 12 GB")
    rows, vocab = 3, 1000
    big = torch.empty(2 * (1 << 30) + 5000, dtype=torch.bfloat16, device=device)
    logits = big.as_strided((rows, vocab), (1 << 30, 1))
    a = make(rows, vocab, torch.bfloat16, device, masks=rows)
    logits.copy_(a["logits"])
    assert torch.equal(adjust_logits(**(a | {"logits": logits}), out=logits), adjust_logits(**a))


def test_captured_replayed_and_on_another_stream(device):
    a = make(20, 5000, torch.bfloat16, device, masks=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        adjust_logits(**a)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = softmax(adjust_logits(**a))
    for seed in (1, 2):
        for n, t in make(20, 5000, torch.bfloat16, device, masks=4, seed=seed).items():
            a[n].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            eager = adjust_logits(**a)
        side.synchronize()
        check(eager, a)
        assert torch.equal(out, softmax(eager))


def test_empty(device):
    a = make(4, 100, torch.float16, device, masks=4)
    none = {n: t[:0] for n, t in a.items() if n != "allowed"} | {"allowed": a["allowed"]}
    assert adjust_logits(**none).shape == (0, 100)
    a = make(4, 100, torch.float16, device, masks=4)
    a["tokens"], a["bias_tokens"], a["bias_values"] = a["tokens"][:, :0], a["bias_tokens"][:, :0], a["bias_values"][:, :0]
    check(adjust_logits(**a), a)
    assert adjust_logits(a["logits"][:, :0]).shape == (4, 0)


def test_refusals(device):
    a = make(4, 100, torch.float16, device, masks=4)
    logits = a["logits"]
    for change, message in ((dict(logits=logits[0]), "rows, vocabulary"), (dict(logits=logits.t()), "contiguous"),
                            (dict(tokens=None), "go together"), (dict(token_lens=None), "go together"),
                            (dict(tokens=None, token_lens=None), "penalties need"), (dict(tokens=a["tokens"].long()), "tokens must be"),
                            (dict(tokens=a["tokens"][:3]), "tokens must have shape"), (dict(bias_values=None), "go together"),
                            (dict(bias_values=a["bias_values"].half()), "bias_values must be"),
                            (dict(bias_values=a["bias_values"][:, :4]), "one shape"), (dict(allowed=None), "allowed_rows needs"),
                            (dict(allowed=a["allowed"][:, :3]), "3 words for 100 tokens"),
                            (dict(allowed=a["allowed"][:3], allowed_rows=None), "allowed must have shape"),
                            (dict(repetition=a["repetition"].cpu()), "repetition must be on"),
                            (dict(frequency=a["frequency"][:, None]), "frequency must have shape"),
                            (dict(tokens=a["tokens"].t().contiguous().t()), "tokens must have contiguous"),
                            (dict(out=logits[:, :50]), "out must be"), (dict(out=logits.float()), "out must be"),
                            (dict(out=torch.zeros(1, 100, device=device).half().expand(4, 100)), "overlaps itself"),
                            (dict(out=logits.t().contiguous().t()), "contiguous rows")):
        with pytest.raises(ValueError, match=message):
            adjust_logits(**(a | change))
    long = {"bias_tokens": torch.zeros(4, 16385, dtype=torch.int32, device=device), "bias_values": torch.zeros(4, 16385, device=device)}
    with pytest.raises(ValueError, match="16384 biases"):
        adjust_logits(**(a | long))
    buf = torch.zeros(8, 100, device=device, dtype=torch.float16)
    with pytest.raises(ValueError, match="shares memory with logits"):
        adjust_logits(buf[:4], out=buf[1:5])
    with pytest.raises(ValueError, match="overlaps itself"):
        one = buf[:1].expand(4, 100)
        adjust_logits(one, out=one)
