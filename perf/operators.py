"""What the serving operators are measured on: prompt attention, attention for
drafted tokens over a paged cache, rotary positions with the cache write, and
block tables with slot maps built from request lengths.

Each case is a dict of plain values. ``prepare`` makes what a serving loop has
in hand before the call, ``run`` makes one call: through this package where
``own`` is true, in elementary torch operations in fp32 otherwise.
"""

from __future__ import annotations

import functools
import importlib
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one long prompt at the 4096-hidden block's geometry with four query heads to a key head
        _prefill("prefill_one_8192", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=1, longest=8192),
        # a batch of prompts packed without padding, odd lengths, some continuing a cached prefix
        _prefill("prefill_packed_ragged", dtype="fp16", heads=32, kv_heads=8, dim=128, seqs=9, longest=1021,
                 prefix=509, ragged=7, lse=True),
        # short prompts on a small block (256 hidden, 8 heads): the call's latency
        _prefill("prefill_small", dtype="fp16", heads=8, kv_heads=8, dim=32, seqs=4, longest=160, ragged=3),
        # ordinary decoding: one new token for each request of a ragged batch
        _tree("decode_batch_64", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=64, longest=4096, nodes=1,
              block=16, ragged=5),
        # speculative decoding: 16 drafted tokens for each request, as trees
        _tree("tree_16x16", dtype="fp16", heads=32, kv_heads=8, dim=128, seqs=16, longest=8192, nodes=16, block=32,
              ragged=11, lse=True),
        # one request with a very long cache: the work has to be split along the cache
        _tree("decode_long_131072", dtype="bf16", heads=32, kv_heads=8, dim=128, seqs=1, longest=131072, nodes=1,
              block=16),
        # one request, a short cache, a small block: the call's latency
        _tree("decode_one_short", dtype="fp16", heads=8, kv_heads=8, dim=32, seqs=1, longest=100, nodes=1, block=16),
        # a prompt's rotary positions, its keys and values written to the cache
        _rotary("rotary_prompt_8192", dtype="bf16", heads=32, kv_heads=8, dim=128, rot=128, tokens=8192, cache=True,
                keep=True),
        # one decoding step's, adjacent pairs, half of each head rotated
        _rotary("rotary_decode_64", dtype="fp16", heads=32, kv_heads=8, dim=128, rot=64, tokens=64,
                interleaved=True, cache=True),
        # the gradient's direction over a training sequence, every head its own keys
        _rotary("rotary_gradient_2048", dtype="fp32", heads=32, kv_heads=32, dim=128, rot=128, tokens=2048,
                inverse=True),
        # one decoding step's block tables and slots
        _slots("slots_decode_64", seqs=64, context=4096, new=1, block=16),
        # many requests with prompts of different lengths at once
        _slots("slots_prompts_512", seqs=512, context=2048, new=131, block=16, ragged=13),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("prefill", "tree", "rotary", "slots"))
    kv_heads = rng.choice((1, 2, 4, 8))
    heads = kv_heads * rng.choice((1, 2, 4, 5) if kv_heads == 8 else (1, 2, 4, 7, 8))
    dim = rng.choice((32, 64, 80, 112, 128, 128))
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
    ragged = rng.randrange(1, 1 << 20)
    if op == "prefill":
        seqs = log_int(1, 32)
        # rows of all requests together: the square is what the plain form holds
        causal = rng.random() < 0.8
        most = min(8192, int(math.sqrt(32 * 8192 * 8192 / heads / (1 if causal else 2)))) if dtype != "fp32" else 2048
        longest = max(1, min(log_int(1, 8192), 2 * most // (seqs + 1) - 1, 8192))
        prefix = rng.choice((0, 0, log_int(1, 512)))
        prefix = max(0, min(prefix, most // seqs - longest))
        return _prefill(None, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, longest=longest,
                        prefix=prefix, ragged=ragged, causal=causal, lse=rng.random() < 0.5)
    if op == "tree":
        seqs = log_int(1, 128)
        nodes = rng.choice((1, 1, log_int(1, 64)))
        longest = log_int(1, max(1, min(131072, 262144 // seqs, (1 << 28) // (seqs * heads * nodes))))
        if dtype == "fp32":
            longest = min(longest, 16384)
        return _tree(None, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs, longest=longest,
                     nodes=nodes, block=rng.choice((8, 16, 32, 64)), ragged=ragged, lse=rng.random() < 0.5)
    if op == "rotary":
        cache = rng.random() < 0.6
        return _rotary(None, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim,
                       rot=rng.choice((dim, dim, dim // 2)), tokens=log_int(1, 8192),
                       interleaved=rng.random() < 0.5, inverse=not cache and rng.random() < 0.5, cache=cache,
                       keep=cache and rng.random() < 0.5)
    seqs = log_int(1, 1024)
    new = rng.choice((1, log_int(1, max(1, 65536 // seqs))))
    return _slots(None, seqs=seqs, context=log_int(1, 32768), new=new, block=rng.choice((8, 16, 32, 64)),
                  ragged=ragged)


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _prefill(name, *, dtype, heads, kv_heads, dim, seqs, longest, prefix=0, ragged=0, causal=True, lse=False):
    return _named(name, dict(op="prefill", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs,
                             longest=longest, prefix=prefix, ragged=ragged, causal=causal, lse=lse))


def _tree(name, *, dtype, heads, kv_heads, dim, seqs, longest, nodes, block, ragged=0, lse=False):
    return _named(name, dict(op="tree", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, seqs=seqs,
                             longest=longest, nodes=nodes, block=block, ragged=ragged, lse=lse))


def _rotary(name, *, dtype, heads, kv_heads, dim, rot, tokens, interleaved=False, inverse=False, cache=False,
            keep=False):
    return _named(name, dict(op="rotary", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                             tokens=tokens, interleaved=interleaved, inverse=inverse, cache=cache, keep=keep))


def _slots(name, *, seqs, context, new, block, ragged=0):
    return _named(name, dict(op="slots", seqs=seqs, context=context, new=new, block=block, ragged=ragged))


def _lengths(case, most, salt, least=1):
    """One length per request, from the case alone: all `most`, or ragged with the first one `most`."""
    if not case["ragged"]:
        return [most] * case["seqs"]
    rng = random.Random(case["ragged"] * 8 + salt)
    return [most] + [rng.randint(min(least, most), most) for _ in range(case["seqs"] - 1)]


def _prompt_lengths(case):
    q = _lengths(case, case["longest"], 0)
    before = _lengths(case, case["prefix"], 1, 0) if case["prefix"] else [0] * case["seqs"]
    return q, [a + b for a, b in zip(q, before)]


def _tree_lengths(case):
    """Cached tokens and drafted nodes of every request (together at most `longest` + `nodes`)."""
    return _lengths(case, case["longest"], 0, 0), _lengths(case, case["nodes"], 1)


def _slot_lengths(case):
    return _lengths(case, case["context"], 0, 0), _lengths(case, case["new"], 1, 0)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    return {"prefill": _prepare_prefill, "tree": _prepare_tree, "rotary": _prepare_rotary,
            "slots": _prepare_slots}[case["op"]](case, seed)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype, gain=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * gain).to(dtype)


def _offsets(lengths):
    return torch.tensor(np.concatenate([[0], np.cumsum(lengths)]), dtype=torch.int32, device="cuda")


def _prepare_prefill(case, seed):
    gen, dtype = _generator(seed), _DTYPES[case["dtype"]]
    lens_q, lens_k = _prompt_lengths(case)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    # queries a little larger than keys: some rows of the softmax are peaked, as trained heads' are
    return {"case": case, "q": _randn(gen, (sum(lens_q), heads, dim), dtype, 2.0),
            "k": _randn(gen, (sum(lens_k), kv_heads, dim), dtype),
            "v": _randn(gen, (sum(lens_k), kv_heads, dim), dtype),
            "cu_q": _offsets(lens_q), "cu_k": _offsets(lens_k)}


def _prepare_tree(case, seed):
    gen, dtype, rng = _generator(seed), _DTYPES[case["dtype"]], np.random.default_rng(seed)
    context, nodes = _tree_lengths(case)
    block, kv_heads, dim = case["block"], case["kv_heads"], case["dim"]
    blocks = [-(-(c + n) // block) for c, n in zip(context, nodes)]
    total = sum(blocks)
    order = rng.permutation(total + 3)  # pages in no order, a few of them nobody's
    table = np.full((case["seqs"], max(blocks)), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(blocks):
        table[r, :n] = order[at:at + n]
        at += n
    masks = []
    for n in nodes:  # a tree: each node sees itself and its ancestors
        seen = np.zeros(n, dtype=np.uint64)
        for i in range(n):
            seen[i] = np.uint64(1) << np.uint64(i)
            if i:
                seen[i] |= seen[rng.integers(max(0, i - 6), i)]
        masks.append(seen)
    cu = _offsets(nodes)
    return {"case": case, "q": _randn(gen, (sum(nodes), case["heads"], dim), dtype, 2.0),
            "k_cache": _randn(gen, (total + 3, kv_heads, block, dim), dtype),
            "v_cache": _randn(gen, (total + 3, kv_heads, block, dim), dtype),
            "table": torch.from_numpy(table).cuda(),
            "context": torch.tensor(context, dtype=torch.int32, device="cuda"),
            "cu_q": None if case["nodes"] == 1 else cu,
            "mask": None if case["nodes"] == 1 else
            torch.from_numpy(np.concatenate(masks).view(np.int64)).cuda().view(-1, 1)}


def _prepare_rotary(case, seed):
    gen, dtype, rng = _generator(seed), _DTYPES[case["dtype"]], np.random.default_rng(seed)
    tokens, heads, kv_heads, dim, rot = (case[n] for n in ("tokens", "heads", "kv_heads", "dim", "rot"))
    most = 16384
    angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    state = {"case": case, "q": _randn(gen, (tokens, heads, dim), dtype),
             "k": _randn(gen, (tokens, kv_heads, dim), dtype), "v": _randn(gen, (tokens, kv_heads, dim), dtype),
             "table": torch.cat([angle.cos(), angle.sin()], 1).float(),
             "positions": torch.from_numpy(rng.integers(0, most, tokens).astype(np.int32)).cuda()}
    if case["cache"]:
        block = 16
        blocks = -(-tokens // block) + 2
        shape = (blocks, kv_heads, block, dim)
        state["k_cache"], state["v_cache"] = _randn(gen, shape, dtype), _randn(gen, shape, dtype)
        page = rng.permutation(blocks)[np.arange(tokens) // block]
        state["slots"] = torch.from_numpy(page * block + np.arange(tokens) % block).cuda()
    return state


def _prepare_slots(case, seed):
    rng, block = np.random.default_rng(seed), case["block"]
    context, new = (np.array(n) for n in _slot_lengths(case))
    held, after = -(-context // block), -(-(context + new) // block)
    total = int(after.sum())
    order = rng.permutation(total + 5)
    table = np.full((case["seqs"], max(1, int(after.max())) + 2), -1, dtype=np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = order[at:at + n]
        at += n
    to = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    return {"case": case, "context": to(context), "new": to(new), "table": torch.from_numpy(table).cuda(),
            "free": torch.from_numpy(order[at:].astype(np.int32)).cuda(),
            "most": int(new.sum()) + 7}  # a little room: a captured step's buffers are sized for its largest


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


@functools.lru_cache(maxsize=None)
def _package(name):
    return importlib.import_module("kernelo_b200.kernels." + name)


def _own_prefill(s):
    c = s["case"]
    return _package("attention").prefill_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=c["causal"],
                                                   return_lse=c["lse"])


def _own_tree(s):
    return _package("attention").tree_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["context"],
                                                s["cu_q"], s["mask"], return_lse=s["case"]["lse"])


def _own_rotary(s):
    c, rotary = s["case"], _package("rotary")
    if not c["cache"]:
        return rotary.rotary(s["q"], s["k"], s["positions"], s["table"], interleaved=c["interleaved"],
                             inverse=c["inverse"])
    k_out = torch.empty_like(s["k"]) if c["keep"] else None
    q_out = rotary.rotary_to_cache(s["q"], s["k"], s["v"], s["positions"], s["table"], s["k_cache"], s["v_cache"],
                                   s["slots"], interleaved=c["interleaved"], k_out=k_out)
    return q_out, k_out, s["k_cache"], s["v_cache"]


def _own_slots(s):
    got = _package("paged").build_slots(s["context"], s["new"], s["table"], s["free"], block_size=s["case"]["block"],
                                        max_tokens=s["most"])
    return got.cu_new, got.positions, got.slots, got.blocks_taken, got.dropped, s["table"]


def _softmax_parts(scores, allowed):
    """(weights, sums, log-sum-exp) of masked scores; a row with nothing left has weights and sums of zero."""
    scores.masked_fill_(~allowed, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    weights = scores.sub_(top).exp_()
    sums = weights.sum(-1, keepdim=True)
    return weights, sums, (top + sums.log()).squeeze(-1)


def _plain_prefill(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    (rows, heads, dim), (keys, kv_heads, _) = q.shape, k.shape
    group, cu_q, cu_k = heads // kv_heads, s["cu_q"].long(), s["cu_k"].long()
    at_q, at_k = torch.arange(rows, device=q.device), torch.arange(keys, device=q.device)
    seq_q = torch.searchsorted(cu_q[1:], at_q, right=True)
    seq_k = torch.searchsorted(cu_k[1:], at_k, right=True)
    allowed = seq_q[:, None] == seq_k[None, :]
    if c["causal"]:
        # the last query of a request sees its last key
        pos_q = at_q - cu_q[seq_q + 1] + cu_k[seq_q + 1] - cu_k[seq_q]
        pos_k = at_k - cu_k[seq_k]
        allowed &= pos_k[None, :] <= pos_q[:, None]
    qf = q.float().view(rows, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * rows, dim)
    scores = torch.matmul(qf, k.float().permute(1, 2, 0)).mul_(dim ** -0.5).view(kv_heads, group, rows, keys)
    weights, sums, lse = _softmax_parts(scores, allowed)
    out = torch.matmul(weights.view(kv_heads, group * rows, keys), v.float().transpose(0, 1))
    out = out.view(kv_heads, group, rows, dim) / torch.where(sums > 0, sums, torch.ones_like(sums))
    out = out.permute(2, 0, 1, 3).reshape(rows, heads, dim).to(q.dtype)
    return (out, lse.view(heads, rows).t().contiguous()) if c["lse"] else out


def _plain_tree(s):
    c, q, table, context = s["case"], s["q"], s["table"], s["context"].long()
    (rows, heads, dim), (_, kv_heads, block, _) = q.shape, s["k_cache"].shape
    seqs, group, device = table.shape[0], heads // kv_heads, q.device
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(seqs + 1, device=device)
    nodes, most = cu[1:] - cu[:-1], c["nodes"]
    pages = table.long().clamp(min=0)
    keys = table.shape[1] * block
    k = s["k_cache"][pages].transpose(1, 2).reshape(seqs, kv_heads, keys, dim).float()
    v = s["v_cache"][pages].transpose(1, 2).reshape(seqs, kv_heads, keys, dim).float()
    at = torch.arange(keys, device=device)
    length = (context + nodes)[:, None]
    v = v.masked_fill_((at >= length)[:, None, :, None], 0.0)  # what lies past the end of a request is anything
    node = torch.arange(most, device=device)
    place = (cu[:-1, None] + node).clamp(max=rows - 1)  # [seqs, most]
    qf = q[place].float().view(seqs, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4)
    scores = torch.matmul(qf.reshape(seqs, kv_heads, group * most, dim), k.transpose(-1, -2)).mul_(dim ** -0.5)
    drafted = at - context[:, None]  # [seqs, keys]: the node that a key belongs to
    if s["mask"] is None:
        sees = (drafted[:, None, :] >= 0) & (drafted[:, None, :] <= node[:, None])
    else:
        bits = s["mask"][place, 0]
        sees = (drafted[:, None, :] >= 0) & (((bits[:, :, None] >> drafted.clamp(0, 63)[:, None, :]) & 1) == 1)
    allowed = ((drafted < 0)[:, None, :] | sees) & (at < length)[:, None, :]
    weights, sums, lse = _softmax_parts(scores.view(seqs, kv_heads, group, most, keys), allowed[:, None, None])
    out = torch.matmul(weights.view(seqs, kv_heads, group * most, keys), v).view(seqs, kv_heads, group, most, dim)
    out = out / torch.where(sums > 0, sums, torch.ones_like(sums))
    owner = torch.searchsorted(cu[1:], torch.arange(rows, device=device), right=True)
    mine = torch.arange(rows, device=device) - cu[owner]
    out = out.permute(0, 3, 1, 2, 4)[owner, mine].reshape(rows, heads, dim).to(q.dtype)
    return (out, lse.permute(0, 3, 1, 2)[owner, mine].reshape(rows, heads)) if c["lse"] else out


def _turn(x, cos, sin, rot, interleaved):
    xf = x.float()
    if interleaved:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, xf[..., rot:]], -1).to(x.dtype)


def _plain_rotary(s):
    c = s["case"]
    rows = s["table"][s["positions"].long()][:, None]
    cos, sin = rows[..., :c["rot"] // 2], rows[..., c["rot"] // 2:]
    sin = -sin if c["inverse"] else sin
    q, k = (_turn(s[n], cos, sin, c["rot"], c["interleaved"]) for n in ("q", "k"))
    if not c["cache"]:
        return q, k
    block = s["k_cache"].shape[2]
    page, at = s["slots"] // block, s["slots"] % block
    s["k_cache"][page, :, at] = k
    s["v_cache"][page, :, at] = s["v"]
    return q, k if c["keep"] else None, s["k_cache"], s["v_cache"]


def _plain_slots(s):
    block, table, free, most = s["case"]["block"], s["table"], s["free"], s["most"]
    context, new, device = s["context"].long(), s["new"].long(), s["context"].device
    zero = torch.zeros(1, dtype=torch.long, device=device)
    cu = torch.cat([zero, new.cumsum(0)])
    held = (context + block - 1) // block
    after = (context + new + block - 1) // block
    base = torch.cat([zero, (after - held).cumsum(0)])
    column = torch.arange(table.shape[1], device=device)
    taken = base[:-1, None] + column - held[:, None]
    fresh = (column >= held[:, None]) & (column < after[:, None])
    given = torch.where(taken < free.numel(), free[taken.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, given, table))
    token = torch.arange(most, device=device)
    owner = torch.searchsorted(cu[1:], token, right=True).clamp(max=new.numel() - 1)
    valid = token < cu[-1]
    position = torch.where(valid, context[owner] + token - cu[owner], 0)
    page = table[owner, (position // block).clamp(max=table.shape[1] - 1)].long()
    good = valid & (page >= 0) & (position // block < table.shape[1])
    slots = torch.where(good, page * block + position % block, -1)
    dropped = (cu[-1:] - good.sum()).int()
    return cu.int(), position.int(), slots, base[-1:].int(), dropped, table


_OWN = {"prefill": _own_prefill, "tree": _own_tree, "rotary": _own_rotary, "slots": _own_slots}
_PLAIN = {"prefill": _plain_prefill, "tree": _plain_tree, "rotary": _plain_rotary, "slots": _plain_slots}


# ------------------------------------------------------------------ work
def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}.get(case.get("dtype"), 0)
    if case["op"] == "prefill":
        lens_q, lens_k = _prompt_lengths(case)
        pairs = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(lens_q, lens_k))
        rows, keys = sum(lens_q), sum(lens_k)
        return {"bytes": size * case["dim"] * 2 * (rows * case["heads"] + keys * case["kv_heads"])
                + (4 * rows * case["heads"] if case["lse"] else 0),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "tree":
        context, nodes = _tree_lengths(case)
        rows, keys = sum(nodes), sum(context) + sum(nodes)
        pairs = sum(n * (c + (n + 1) / 2) for c, n in zip(context, nodes))
        return {"bytes": size * case["dim"] * 2 * (rows * case["heads"] + keys * case["kv_heads"])
                + (4 * rows * case["heads"] if case["lse"] else 0),
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "rotary":
        row, tokens = size * case["dim"], case["tokens"]
        copies = 4 + case["keep"] if case["cache"] else 2  # k and v read, both written to the cache, k' kept too
        return {"bytes": tokens * row * (2 * case["heads"] + case["kv_heads"] * copies) + tokens * (4 * case["rot"] + 4 + 8 * case["cache"]),
                "flops": 3 * tokens * case["rot"] * (case["heads"] + case["kv_heads"])}
    context, new = _slot_lengths(case)
    block, tokens = case["block"], sum(new)
    pages = sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(context, new))
    partly = sum(1 for c, n in zip(context, new) if n and c % block)
    return {"bytes": 8 * case["seqs"] + 4 * (case["seqs"] + 1) + 12 * (tokens + 7) + 8 * pages + 4 * partly + 8,
            "flops": 0}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] == "slots":
        return None
    s = prepare(case, seed)
    return {"prefill": _exact_prefill, "tree": _exact_tree, "rotary": _exact_rotary}[case["op"]](case, s)


def _exact_head(q, k, v, seen):
    """One head's output and log-sum-exp, from the sums over what each row sees."""
    scores = (q.double() @ k.double().T) / math.sqrt(q.shape[1])
    scores = torch.where(seen, scores, -math.inf)
    lse = torch.logsumexp(scores, 1)
    weights = torch.where(seen, torch.exp(scores - torch.where(lse > -math.inf, lse, 0.0)[:, None]), 0.0)
    return weights @ v.double(), lse


def _exact_prefill(case, s):
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    q0 = k0 = 0
    for n, m in zip(*_prompt_lengths(case)):
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        if case["causal"]:
            seen = seen.tril(m - n)
        for h in range(case["heads"]):
            kh = h // (case["heads"] // case["kv_heads"])
            out[q0:q0 + n, h], lse[q0:q0 + n, h] = _exact_head(
                s["q"][q0:q0 + n, h], s["k"][k0:k0 + m, kh], s["v"][k0:k0 + m, kh], seen)
        q0, k0 = q0 + n, k0 + m
    return (out, lse) if case["lse"] else out


def _exact_tree(case, s):
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for r, (c, n) in enumerate(zip(*_tree_lengths(case))):
        place = torch.arange(c + n, device="cuda")
        page, row = s["table"][r].long()[place // case["block"]], place % case["block"]
        k, v = s["k_cache"][page, :, row], s["v_cache"][page, :, row]
        seen = torch.ones(n, c + n, dtype=torch.bool, device="cuda")
        if s["mask"] is not None:
            words = s["mask"][at:at + n, 0].tolist()
            seen[:, c:] = torch.tensor([[bool(w >> j & 1) for j in range(n)] for w in words], device="cuda")
        for h in range(case["heads"]):
            kh = h // (case["heads"] // case["kv_heads"])
            out[at:at + n, h], lse[at:at + n, h] = _exact_head(s["q"][at:at + n, h], k[:, kh], v[:, kh], seen)
        at += n
    return (out, lse) if case["lse"] else out


def _exact_rotary(case, s):
    rot, half = case["rot"], case["rot"] // 2
    row = s["table"].double()[s["positions"].long()]
    unit = torch.complex(row[:, :half], -row[:, half:] if case["inverse"] else row[:, half:])[:, None]
    done = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, half),
                                                                                         slice(half, rot))
        z = torch.complex(x[..., first], x[..., second]) * unit
        y[..., first], y[..., second] = z.real, z.imag
        done.append(y)
    if not case["cache"]:
        return tuple(done)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    block = k_cache.shape[2]
    for t, slot in enumerate(s["slots"].tolist()):
        k_cache[slot // block, :, slot % block] = done[1][t]
        v_cache[slot // block, :, slot % block] = s["v"][t].double()
    return done[0], done[1] if case["keep"] else None, k_cache, v_cache
