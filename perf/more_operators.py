"""What the second set of serving operators is measured on: norms of each head of q
and k with the position rotation (and the cache write, and the gradient) in one
pass; penalties, biases and grammar masks on logits; and the pages of a cache
when requests fork, end, or are moved together.

Each case is a dict of plain values. ``prepare`` makes what a program has in hand
before the call, ``run`` makes one call: through this package where ``own`` is
true, in elementary torch operations in fp32 otherwise.
"""

from __future__ import annotations

import functools
import importlib
import math

import numpy as np
import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # a prompt at the 4096-hidden block's geometry: its keys go to the cache and, packed, to its own attention
        _norm("norm_rotary_prompt_8192", dtype="bf16", heads=32, kv_heads=8, dim=128, rot=128, tokens=8192, cache=True,
              keep=True),
        # one decoding step's tokens, adjacent pairs, half of each head turned: the call's latency
        _norm("norm_rotary_decode_64", dtype="fp16", heads=32, kv_heads=8, dim=128, rot=64, tokens=64,
              interleaved=True, cache=True),
        # the gradient over a training batch's tokens, both weights' among it
        _norm("norm_rotary_gradient_4096", dtype="bf16", heads=32, kv_heads=8, dim=128, rot=128, tokens=4096,
              gradient=True),
        # the small block's (256 hidden, 8 heads), an odd number of tokens
        _norm("norm_rotary_gradient_333", dtype="fp32", heads=8, kv_heads=8, dim=32, rot=32, tokens=333, gradient=True),
        # a full batch at the benchmark's vocabulary: every request penalised and biased, some under a grammar
        _logits("logits_batch_512", dtype="fp32", rows=512, vocab=32000, history=2048, biases=32, masks=64,
                penalties=True),
        # a few requests, an odd vocabulary, rows off the vector grid: the call's latency
        _logits("logits_few_7", dtype="bf16", rows=7, vocab=32001, history=700, biases=8, masks=7, penalties=True),
        # sixteen requests of a 16-layer model each answered four more ways
        _fork("fork_16_by_4", dtype="bf16", caches=32, kv_heads=8, block=16, dim=128, parents=16, each=4, longest=2048,
              ragged=3),
        # one request of one block answered four ways
        _fork("fork_one_by_4", dtype="fp16", caches=2, kv_heads=8, block=16, dim=128, parents=1, each=4, longest=700),
        # a server's batch ends: long requests, most of them forks that share their prompts' pages
        _release("release_256", requests=256, ended=192, longest=32768, block=16, group=4, ragged=5),
        # one request ends
        _release("release_one", requests=64, ended=1, longest=4096, block=16, group=1, ragged=7),
        # a pool of pages half free after hours of serving, an 8-layer model, moved together
        _compact("compact_4096", dtype="bf16", caches=16, kv_heads=8, block=16, dim=128, requests=32, longest=2048,
                 group=2, spare=1.0, ragged=9),
        # a single block's small pool
        _compact("compact_small", dtype="fp16", caches=2, kv_heads=2, block=16, dim=64, requests=4, longest=300, group=1,
                 spare=0.5, ragged=11),
    ]


def draw(rng):
    def log_int(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op = rng.choice(("norm", "norm", "logits", "logits", "fork", "release", "compact"))
    dtype = rng.choice(("fp16", "bf16", "bf16", "fp32"))
    ragged = rng.randrange(1, 1 << 20)
    dim = rng.choice((32, 64, 80, 96, 128, 128, 256))
    if op == "norm":
        kv_heads = rng.choice((1, 2, 4, 8))
        heads = kv_heads * rng.choice((1, 2, 4, 5, 8))
        gradient = rng.random() < 0.5
        cache = not gradient and rng.random() < 0.6
        # elements of a prompt or batch, at most those of the listed ones
        most = 4096 * 40 * 128 // ((heads + kv_heads) * dim * (2 if dtype == "fp32" else 1))
        return _norm(None, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, rot=rng.choice((dim, dim, dim // 2)),
                     tokens=log_int(1, max(1, min(8192, most))), interleaved=rng.random() < 0.5, gradient=gradient,
                     cache=cache, keep=cache and rng.random() < 0.5)
    if op == "logits":
        rows = log_int(1, 512)
        vocab = log_int(250, min(131072, 512 * 32000 // rows))
        return _logits(None, dtype=dtype, rows=rows, vocab=vocab, history=log_int(1, 4096 if rows > 64 else 32768),
                       biases=rng.choice((0, log_int(1, 64))), masks=rng.choice((0, rows, log_int(1, rows))),
                       penalties=rng.random() < 0.8)
    block, kv_heads = rng.choice((8, 16, 32, 64)), rng.choice((1, 2, 4, 8))
    if op == "fork":
        parents = log_int(1, 32)
        return _fork(None, dtype=dtype, caches=2 * log_int(1, 12), kv_heads=kv_heads, block=block, dim=min(dim, 128),
                     parents=parents, each=rng.randint(1, 8 if parents <= 8 else 2), longest=log_int(1, 1024), ragged=ragged)
    group = rng.choice((1, 2, 4, 7))
    if op == "release":
        requests = log_int(1, 256)
        return _release(None, requests=requests, ended=rng.randint(1, requests), longest=log_int(1, 16384), block=block,
                        group=group, ragged=ragged)
    return _compact(None, dtype=dtype, caches=2 * log_int(1, 8), kv_heads=kv_heads, block=block, dim=min(dim, 64),
                    requests=log_int(1, 32), longest=log_int(1, 1024), group=group, spare=rng.choice((0.1, 0.5, 1.0)),
                    ragged=ragged)


def _named(name, case):
    return case if name is None else {"name": name, **case}


def _norm(name, *, dtype, heads, kv_heads, dim, rot, tokens, interleaved=False, cache=False, keep=False, gradient=False):
    return _named(name, dict(op="norm", dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, tokens=tokens,
                             interleaved=interleaved, cache=cache, keep=keep, gradient=gradient))


def _logits(name, *, dtype, rows, vocab, history, biases, masks, penalties):
    return _named(name, dict(op="logits", dtype=dtype, rows=rows, vocab=vocab, history=history, biases=biases,
                             masks=masks, penalties=penalties))


def _fork(name, *, dtype, caches, kv_heads, block, dim, parents, each, longest, ragged=0):
    return _named(name, dict(op="fork", dtype=dtype, caches=caches, kv_heads=kv_heads, block=block, dim=dim,
                             parents=parents, each=each, longest=longest, ragged=ragged))


def _release(name, *, requests, ended, longest, block, group, ragged=0):
    return _named(name, dict(op="release", requests=requests, ended=ended, longest=longest, block=block, group=group,
                             ragged=ragged))


def _compact(name, *, dtype, caches, kv_heads, block, dim, requests, longest, group, spare, ragged=0):
    return _named(name, dict(op="compact", dtype=dtype, caches=caches, kv_heads=kv_heads, block=block, dim=dim,
                             requests=requests, longest=longest, group=group, spare=spare, ragged=ragged))


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    return {"norm": _prepare_norm, "logits": _prepare_logits, "fork": _prepare_fork, "release": _prepare_release,
            "compact": _prepare_compact}[case["op"]](case, seed)


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(gen, shape, dtype, gain=1.0, mean=0.0):
    return (torch.randn(shape, generator=gen, device="cuda") * gain + mean).to(dtype)


def _prepare_norm(case, seed):
    gen, dtype, rng = _generator(seed), _DTYPES[case["dtype"]], np.random.default_rng(seed)
    tokens, heads, kv_heads, dim, rot = (case[n] for n in ("tokens", "heads", "kv_heads", "dim", "rot"))
    most = 16384
    angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    # a projection's output before its norm: heads and tokens of different sizes
    state = {"case": case, "q": _randn(gen, (tokens, heads, dim), dtype, 2.5),
             "k": _randn(gen, (tokens, kv_heads, dim), dtype, 0.4),
             "q_weight": _randn(gen, (dim,), dtype, 0.1, 1.0), "k_weight": _randn(gen, (dim,), dtype, 0.1, 1.0),
             "table": torch.cat([angle.cos(), angle.sin()], 1).float(),
             "positions": torch.from_numpy(rng.integers(0, most, tokens).astype(np.int32)).cuda()}
    if case["gradient"]:
        state["dq"], state["dk"] = (_randn(gen, state[n].shape, dtype) for n in ("q", "k"))
    if case["cache"]:
        block = 16
        blocks = -(-tokens // block) + 2
        shape = (blocks, kv_heads, block, dim)
        state["v"] = _randn(gen, (tokens, kv_heads, dim), dtype)
        state["k_cache"], state["v_cache"] = _randn(gen, shape, dtype), _randn(gen, shape, dtype)
        page = rng.permutation(blocks)[np.arange(tokens) // block]
        state["slots"] = torch.from_numpy(page * block + np.arange(tokens) % block).cuda()
    return state


def _prepare_logits(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    rows, vocab, most = case["rows"], case["vocab"], case["history"]
    state = {"case": case, "logits": _randn(gen, (rows, vocab), _DTYPES[case["dtype"]], 4.0), "tokens": None,
             "lens": None, "prompts": None, "repetition": None, "frequency": None, "presence": None,
             "bias_tokens": None, "bias_values": None, "allowed": None, "allowed_rows": None}
    if case["penalties"]:
        # text repeats its frequent tokens: ids crowd towards the first ones
        ids = (torch.rand((rows, most), generator=gen, device="cuda").pow_(4) * vocab).int().clamp_(max=vocab - 1)
        lens = rng.integers(0, most + 1, rows)
        state["tokens"] = ids
        state["lens"] = torch.from_numpy(lens.astype(np.int32)).cuda()
        state["prompts"] = torch.from_numpy((lens * rng.random(rows)).astype(np.int32)).cuda()
        for n, low, wide in (("repetition", 1.0, 0.5), ("frequency", 0.0, 0.5), ("presence", 0.0, 1.0)):
            state[n] = torch.rand(rows, generator=gen, device="cuda") * wide + low
    if case["biases"]:
        at = rng.integers(0, vocab, (rows, case["biases"]))
        at[rng.random(at.shape) < 0.2] = -1  # rows have different numbers of biases
        state["bias_tokens"] = torch.from_numpy(at.astype(np.int32)).cuda()
        state["bias_values"] = _randn(gen, at.shape, torch.float32, 5.0)
    if case["masks"]:
        words = -(-vocab // 32)
        state["allowed"] = torch.from_numpy(rng.integers(0, 1 << 32, (case["masks"], words), dtype=np.uint32)
                                            .view(np.int32)).cuda()
        which = rng.integers(0, case["masks"], rows)
        if case["masks"] < rows:
            which[rng.random(rows) < 0.7] = -1  # not every request has a grammar
        state["allowed_rows"] = torch.from_numpy(which.astype(np.int32)).cuda()
    return state


def _holding(case, requests, group):
    """Lengths, and how many of its first pages each request shares with the first of its `group`: from the case alone."""
    lens = _lengths(case, requests)
    first = np.arange(requests) // group * group
    share = np.random.default_rng(case["ragged"] + 1).random(requests)
    common = (np.minimum(lens, lens[first]) * share).astype(np.int64) // case["block"]
    common[first == np.arange(requests)] = 0
    return lens, first, common


def _table(case, requests, group, rng, spare):
    """Lengths, a block table, counts of further holders, and the free pages: of each `group` requests the later ones
    are forks of the first at some point, and share its whole pages up to there."""
    lens, first, common = _holding(case, requests, group)
    cols = -(-lens // case["block"])
    column = np.arange(int(cols.max()) + 2)
    fresh = (column >= common[:, None]) & (column < cols[:, None])
    total = int(fresh.sum())
    order = rng.permutation(total + max(3, int(total * spare)))
    table = np.full(fresh.shape, -1, dtype=np.int32)
    table[fresh] = order[:total]
    table = np.where(column < common[:, None], table[first], table)
    shared = np.maximum(np.bincount(table[table >= 0], minlength=order.size) - 1, 0)
    return lens, table, shared, order[total:]


def _lengths(case, requests):
    """One length per request, from the case alone: all `longest`, or ragged with the first one `longest`."""
    if not case["ragged"]:
        return np.full(requests, case["longest"], dtype=np.int64)
    lens = np.random.default_rng(case["ragged"]).integers(0, case["longest"] + 1, requests)
    lens[0] = case["longest"]
    return lens


def _ints(values):
    return torch.from_numpy(np.ascontiguousarray(values, dtype=np.int32)).cuda()


def _caches(case, gen, pages):
    """Every layer's keys and values, one after another in one allocation."""
    shape = (case["caches"], pages, case["kv_heads"], case["block"], case["dim"])
    return torch.empty(shape, dtype=_DTYPES[case["dtype"]], device="cuda").normal_(generator=gen)


def _prepare_fork(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    parents, each = case["parents"], case["each"]
    lens, table, shared, free = _table(case, parents, 1, rng, 0.0)
    free = np.concatenate([free, shared.size + rng.permutation(parents * each)])
    shared = np.concatenate([shared, np.zeros(parents * each, dtype=np.int64)])
    rows = rng.permutation(parents * (1 + each))  # requests lie in no order
    whole = np.full((rows.size, table.shape[1]), -1, dtype=np.int32)
    whole[rows[:parents]] = table
    context = np.zeros(rows.size)
    context[rows[:parents]] = lens
    return {"case": case, "caches": _caches(case, gen, shared.size), "table": _ints(whole), "context": _ints(context),
            "shared": _ints(shared), "free": _ints(free), "parents": _ints(np.repeat(rows[:parents], each)),
            "children": _ints(rows[parents:])}


def _prepare_release(case, seed):
    rng = np.random.default_rng(seed)
    lens, table, shared, _ = _table(case, case["requests"], case["group"], rng, 0.0)
    return {"case": case, "table": _ints(table), "context": _ints(lens), "shared": _ints(shared),
            "ended": _ints(_ended(case))}


def _ended(case):
    return np.random.default_rng(case["ragged"] + 2).permutation(case["requests"])[:case["ended"]]


def _prepare_compact(case, seed):
    gen, rng = _generator(seed), np.random.default_rng(seed)
    lens, table, shared, _ = _table(case, case["requests"], case["group"], rng, case["spare"])
    return {"case": case, "caches": _caches(case, gen, shared.size), "table": _ints(table), "context": _ints(lens),
            "shared": _ints(shared)}


# ------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    return (_OWN if own else _PLAIN)[op](state)


@functools.lru_cache(maxsize=None)
def _package(name):
    return importlib.import_module("kernelo_b200.kernels." + name)


def _own_norm(s):
    c, rotary = s["case"], _package("rotary")
    if c["gradient"]:
        return rotary.norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], s["positions"], s["table"], s["q_weight"],
                                           s["k_weight"], eps=_EPS, interleaved=c["interleaved"])
    if not c["cache"]:
        return rotary.norm_rotary(s["q"], s["k"], s["positions"], s["table"], s["q_weight"], s["k_weight"], eps=_EPS,
                                  interleaved=c["interleaved"])
    k_out = torch.empty_like(s["k"]) if c["keep"] else None
    q_out = rotary.norm_rotary_to_cache(s["q"], s["k"], s["v"], s["positions"], s["table"], s["q_weight"], s["k_weight"],
                                        s["k_cache"], s["v_cache"], s["slots"], eps=_EPS, interleaved=c["interleaved"],
                                        k_out=k_out)
    return q_out, k_out, s["k_cache"], s["v_cache"]


def _own_logits(s):
    return _package("logits").adjust_logits(
        s["logits"], tokens=s["tokens"], token_lens=s["lens"], prompt_lens=s["prompts"], repetition=s["repetition"],
        frequency=s["frequency"], presence=s["presence"], bias_tokens=s["bias_tokens"], bias_values=s["bias_values"],
        allowed=s["allowed"], allowed_rows=s["allowed_rows"])


def _own_fork(s):
    shared = s["shared"].clone()  # so that the state can be passed again
    got = _package("paged").fork_requests(s["caches"].unbind(0), s["table"], s["context"], shared, s["free"],
                                          s["parents"], s["children"])
    return s["caches"], s["table"], s["context"], shared, got.blocks_taken, got.dropped


def _own_release(s):
    table, context, shared = (s[n].clone() for n in ("table", "context", "shared"))
    got = _package("paged").release_requests(table, context, shared, s["ended"], block_size=s["case"]["block"])
    return table, context, shared, got.pages, got.count


def _own_compact(s):
    # the pages that move stay readable where they were: with the table as it was, the state can be passed again
    table, shared = (s[n].clone() for n in ("table", "shared"))
    got = _package("paged").compact_pages(s["caches"].unbind(0), table, s["context"], shared)
    return s["caches"], table, shared, got.renamed, got.live


def _turn(xf, cos, sin, rot, interleaved):
    if interleaved:
        a, b = xf[..., 0:rot:2], xf[..., 1:rot:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = xf[..., :rot // 2], xf[..., rot // 2:rot]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([turned, xf[..., rot:]], -1)


def _plain_norm(s):
    c = s["case"]
    rows = s["table"][s["positions"].long()][:, None]
    cos, sin = rows[..., :c["rot"] // 2], rows[..., c["rot"] // 2:]

    def forward(x, weight):
        xf = x.float()
        xf = xf * torch.rsqrt(xf.square().mean(-1, keepdim=True) + _EPS) * weight.float()
        return _turn(xf, cos, sin, c["rot"], c["interleaved"]).to(x.dtype)

    def backward(dy, x, weight):
        xf = x.float()
        inv = torch.rsqrt(xf.square().mean(-1, keepdim=True) + _EPS)
        unit, g = xf * inv, _turn(dy.float(), cos, -sin, c["rot"], c["interleaved"])
        gw = g * weight.float()
        dx = inv * (gw - unit * (gw * unit).mean(-1, keepdim=True))
        return dx.to(x.dtype), (g * unit).sum((0, 1))

    if c["gradient"]:
        dq, dq_weight = backward(s["dq"], s["q"], s["q_weight"])
        dk, dk_weight = backward(s["dk"], s["k"], s["k_weight"])
        return dq, dk, dq_weight, dk_weight
    q, k = forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])
    if not c["cache"]:
        return q, k
    block = s["k_cache"].shape[2]
    page, at = s["slots"] // block, s["slots"] % block
    s["k_cache"][page, :, at] = k
    s["v_cache"][page, :, at] = s["v"]
    return q, k if c["keep"] else None, s["k_cache"], s["v_cache"]


def _plain_logits(s):
    logits = s["logits"]
    rows, vocab = logits.shape
    device, x = logits.device, logits.float()
    if s["tokens"] is not None:
        ids, place = s["tokens"].long(), torch.arange(s["tokens"].shape[1], device=device)
        held = place < s["lens"][:, None]
        answered = held & (place >= s["prompts"][:, None])
        count = x.new_zeros(rows, vocab, dtype=torch.int32).scatter_add_(1, ids, answered.int())
        seen = x.new_zeros(rows, vocab, dtype=torch.int32).scatter_add_(1, ids, held.int()) > 0
        by = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / by, x * by), x)
        x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_tokens"] is not None:
        # of a token that is listed twice the last value counts
        at, place = s["bias_tokens"].long(), torch.arange(s["bias_tokens"].shape[1], device=device)
        to = torch.where(at >= 0, at, vocab)
        last = torch.full((rows, vocab + 1), -1, device=device).scatter_reduce_(1, to, place.expand(rows, -1), "amax")[:, :vocab]
        x = x + torch.where(last >= 0, s["bias_values"].gather(1, last.clamp(min=0)), 0.0)
    if s["allowed"] is not None:
        bits = s["allowed"][s["allowed_rows"].long().clamp(min=0)][:, :, None] >> torch.arange(32, device=device, dtype=torch.int32)
        may = ((bits & 1) == 1).flatten(1)[:, :vocab] | (s["allowed_rows"] < 0)[:, None]
        x = torch.where(may, x, -math.inf)
    return x.to(logits.dtype)


def _plain_fork(s):
    caches, table, context, free = s["caches"], s["table"], s["context"], s["free"]
    block, parents, children = caches.shape[3], s["parents"].long(), s["children"].long()
    lens = context[parents]
    full, tail = lens // block, lens % block
    needs = tail > 0
    rank = needs.cumsum(0) - needs.long()
    got = needs & (rank < free.numel())
    page = torch.where(got, free[rank.clamp(max=free.numel() - 1)], -1)  # (the list is longer than what is taken)
    column, rows = torch.arange(table.shape[1], device=table.device), table[parents]
    common = column < full[:, None]
    shared = s["shared"].index_add(0, rows.clamp(min=0).flatten(), common.int().flatten())
    ours = (column == full[:, None]) & needs[:, None]
    table[children] = torch.where(common, rows, torch.where(ours, page[:, None], -1))
    context[children] = lens
    source = rows.gather(1, full[:, None].long())[:, 0].clamp(min=0).long()
    target = torch.where(got, page, free[-1]).long()
    copied = ((torch.arange(block, device=table.device) < tail[:, None]) & got[:, None])[None, :, None, :, None]
    caches[:, target] = torch.where(copied, caches[:, source], caches[:, target])
    taken = needs.sum(dtype=torch.int32)[None]
    return caches, table, context, shared, taken, taken - got.sum(dtype=torch.int32)


def _plain_release(s):
    table, context, shared, ended = s["table"], s["context"], s["shared"], s["ended"].long()
    block, (_, cols) = s["case"]["block"], s["table"].shape
    rows = table[ended]
    held = (torch.arange(cols, device=table.device) < ((context[ended] + block - 1) // block)[:, None]) & (rows >= 0)
    page, held, place = rows.clamp(min=0).flatten().long(), held.flatten(), torch.arange(rows.numel(), device=table.device)
    left = shared.index_add(0, page, -held.int())
    free = left < 0
    # a page goes where the first of its holders in the list has it
    first = torch.full((shared.numel(),), rows.numel(), device=table.device)
    first = first.scatter_reduce_(0, page, torch.where(held, place, rows.numel()), "amin")
    listed_ = held & free[page] & (first[page] == place)
    rank = listed_.cumsum(0) - 1
    pages = torch.full((rows.numel() + 1,), -1, dtype=torch.int32, device=table.device)
    pages[torch.where(listed_, rank, rows.numel())] = torch.where(listed_, rows.flatten(), -1)
    return (table.index_fill(0, ended, -1), context.index_fill(0, ended, 0), torch.where(free, 0, left), pages[:-1],
            listed_.sum(dtype=torch.int32)[None])


def _plain_compact(s):
    caches, table, context, shared = s["caches"], s["table"], s["context"], s["shared"]
    pages, block = caches.shape[1], caches.shape[3]
    held = (torch.arange(table.shape[1], device=table.device) < ((context + block - 1) // block)[:, None]) & (table >= 0)
    live = torch.zeros(pages, dtype=torch.int32, device=table.device)
    live = live.index_add(0, table.clamp(min=0).flatten(), held.int().flatten()) > 0
    count, page = live.sum(), torch.arange(pages, device=table.device)
    mover, hole = live & (page >= count), ~live & (page < count)
    # the i-th page behind the live ones' number goes to the i-th hole before it
    holes = torch.zeros(pages + 1, dtype=torch.int64, device=table.device)
    holes[torch.where(hole, hole.cumsum(0) - 1, pages)] = page
    renamed = torch.where(mover, holes[(mover.cumsum(0) - 1).clamp(min=0)], torch.where(live, page, -1))
    new_table = torch.where(held, renamed[table.clamp(min=0).long()].int(), table)
    new_shared = torch.zeros(pages + 1, dtype=torch.int32, device=table.device)
    new_shared[torch.where(live, renamed, pages)] = shared
    moving = torch.nonzero(mover).flatten()
    caches[:, renamed[moving]] = caches[:, moving]
    return caches, new_table, new_shared[:-1], renamed.int(), count.int()[None]


_OWN = {"norm": _own_norm, "logits": _own_logits, "fork": _own_fork, "release": _own_release, "compact": _own_compact}
_PLAIN = {"norm": _plain_norm, "logits": _plain_logits, "fork": _plain_fork, "release": _plain_release,
          "compact": _plain_compact}


# ------------------------------------------------------------------ work
def work(case):
    size = {"fp16": 2, "bf16": 2, "fp32": 4}.get(case.get("dtype"), 0)
    if case["op"] == "norm":
        row, tokens, heads, kv_heads, rot = size * case["dim"], case["tokens"], case["heads"], case["kv_heads"], case["rot"]
        angles = tokens * (4 * rot + 4)
        if case["gradient"]:  # x and dy read, dx written, the weights and their gradients
            return {"bytes": tokens * row * 3 * (heads + kv_heads) + angles + 2 * case["dim"] * (size + 4),
                    "flops": tokens * (heads + kv_heads) * (11 * case["dim"] + 3 * rot)}
        copies = 4 + case["keep"] if case["cache"] else 2  # k and v read, both written to the cache, k' kept too
        return {"bytes": tokens * row * (2 * heads + kv_heads * copies) + angles + 8 * tokens * case["cache"] + 2 * row,
                "flops": tokens * (heads + kv_heads) * (4 * case["dim"] + 3 * rot)}
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        total = 2 * rows * vocab * size + 8 * rows * case["biases"]
        if case["penalties"]:
            total += rows * (2 * case["history"] + 20)  # histories are half as long on average
        if case["masks"]:
            total += case["masks"] * (-(-vocab // 32)) * 4 + 4 * rows
        return {"bytes": total, "flops": rows * vocab}
    block = case["block"]
    if case["op"] == "fork":
        lens, each = _lengths(case, case["parents"]), case["each"]
        token = case["caches"] * case["kv_heads"] * case["dim"] * size
        tails, columns = int((lens % block).sum()), int((-(-lens // block)).sum())
        # a parent's last page read once, written for each child; its row likewise, and counts of its whole pages
        return {"bytes": tails * token * (1 + each) + 4 * columns * (1 + each) + 8 * int((lens // block).sum()), "flops": 0}
    lens, _, common = _holding(case, case["requests"], case["group"])
    columns = -(-lens // block)
    if case["op"] == "release":
        # each held page's number read and cleared, its count read and written; the list of those that go back, at most
        return {"bytes": 16 * int(columns[_ended(case)].sum()) + 12 * case["ended"] + 4, "flops": 0}
    live = int((columns - common).sum())
    free = max(3, int(live * case["spare"]))
    # as many pages move as lie behind the live ones' number, on average; every row is read, and written where they do
    page = case["caches"] * case["kv_heads"] * block * case["dim"] * size
    return {"bytes": int(live * free / (live + free) * (2 * page + 8)) + 4 * int(columns.sum()) + 8 * (live + free), "flops": 0}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] not in ("norm", "logits"):  # pages are numbered, and their contents copied
        return None
    return {"norm": _exact_norm, "logits": _exact_logits}[case["op"]](case, prepare(case, seed))


def _exact_norm(case, s):
    rot, half = case["rot"], case["rot"] // 2
    row = s["table"].double()[s["positions"].long()]
    unit = torch.complex(row[:, :half], row[:, half:])[:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, half), slice(half, rot))

    def turned(x, by):
        y, z = x.clone(), torch.complex(x[..., first], x[..., second]) * by
        y[..., first], y[..., second] = z.real, z.imag
        return y

    done = []
    for name in ("q", "k"):
        x, weight = s[name].double(), s[name + "_weight"].double()
        size = torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / case["dim"] + _EPS)
        if not case["gradient"]:
            done.append(turned(x / size * weight, unit))
            continue
        # y_i = R (w x_i / size): dx = J^T R^T dy with J = diag(w) (1 / size - x x^T / (dim size^3))
        back = turned(s["d" + name].double(), unit.conj())
        along = torch.einsum("thd,thd->th", back * weight, x)[..., None]
        done.append(back * weight / size - x * along / (case["dim"] * size ** 3))
        done.append(torch.einsum("thd,thd->d", back, x / size))
    if case["gradient"]:
        return done[0], done[2], done[1], done[3]
    if not case["cache"]:
        return tuple(done)
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    block = k_cache.shape[2]
    for t, slot in enumerate(s["slots"].tolist()):
        k_cache[slot // block, :, slot % block] = done[1][t]
        v_cache[slot // block, :, slot % block] = s["v"][t].double()
    return done[0], done[1] if case["keep"] else None, k_cache, v_cache


def _exact_logits(case, s):
    out = s["logits"].double()
    vocab = case["vocab"]
    for r in range(case["rows"]):
        x = out[r]
        if case["penalties"]:
            n, prompt = int(s["lens"][r]), int(s["prompts"][r])
            ids = s["tokens"][r, :n].long()
            met = torch.unique(ids)
            by = s["repetition"][r].double()
            x[met] = torch.where(x[met] > 0, x[met] / by, x[met] * by)
            met, times = torch.unique(ids[prompt:], return_counts=True)
            x[met] -= s["frequency"][r].double() * times + s["presence"][r].double()
        if case["biases"]:
            values = dict(zip(s["bias_tokens"][r].tolist(), s["bias_values"][r].tolist()))
            values.pop(-1, None)
            at = torch.tensor(list(values), dtype=torch.long, device="cuda")
            x[at] += torch.tensor(list(values.values()), dtype=torch.float64, device="cuda")
        if case["masks"] and int(s["allowed_rows"][r]) >= 0:
            words = s["allowed"][int(s["allowed_rows"][r])].cpu().numpy()
            bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]
            x[torch.from_numpy(bits == 0).cuda()] = -math.inf
    return out
