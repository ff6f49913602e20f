"""The serving operators next to the S+LR linears, as cases that can be timed:

* ``attend``    one new token per row attends over a paged key-value cache
* ``append``    new tokens' keys and values go into their pages
* ``advance``   rows fork, end and grow: page tables, shared pages and copies
* ``compact``   live pages move to the lowest page numbers
* ``logprobs``  log probabilities of given tokens, entropy and top choices

``run`` computes them in elementary torch operations, or (``own``) through
``s_salaad_b200.kvcache.PagedCache`` and ``s_salaad_b200.ops.token_logprobs``.

A cache is two tensors.  ``pool`` [layers, 2, pages, kv_heads, page_size,
head_dim] holds keys (0) and values (1).  ``state`` (int32) is a header
{pages short, rows over capacity, pages copied, pages in use}, then lens
[rows], refs [pages] (table entries that name a page; 0 = free) and the page
table [rows, width] (-1 = unused).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
ESIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
HEADER = 4


# ------------------------------------------------------------- cases --

def listed():
    return [
        # one user, a short chat with the 60M-parameter model of the benchmark (8 heads of 64)
        dict(name="attend_one_short", op="attend", dtype="bf16", rows=1, heads=8, kv_heads=8, dim=64, page=16,
             low=203, high=203),
        # a served batch with shared key heads, chats of every age, some rows empty
        dict(name="attend_batch", op="attend", dtype="bf16", rows=48, heads=32, kv_heads=8, dim=128, page=16,
             low=0, high=6007),
        # two users with book-length contexts: few rows, all the length
        dict(name="attend_long", op="attend", dtype="fp16", rows=2, heads=32, kv_heads=8, dim=128, page=64,
             low=98765, high=131071),
        # the fp32 parity path: the 7B-shaped model's 32 unshared heads
        dict(name="attend_fp32", op="attend", dtype="fp32", rows=8, heads=32, kv_heads=32, dim=128, page=16,
             low=1, high=2050),
        # a decode step of a batch
        dict(name="append_step", op="append", dtype="bf16", rows=64, kv_heads=8, dim=128, page=16, low=0, high=4000,
             new=0),
        # ragged prompts of a batch, packed, with unused rows behind the last
        dict(name="append_prompts", op="append", dtype="fp16", rows=24, kv_heads=8, dim=128, page=32, low=0, high=777,
             new=1999),
        # beam search: each prompt's row becomes 4, last pages are copied
        dict(name="fork_beams", op="advance", dtype="bf16", layers=8, kv_heads=8, dim=64, page=16, rows=32, width=64,
             pages=2048, low=17, high=600, fanout=4),
        # a large server's step: rows end, move up and grow by a token; 16k pages
        dict(name="grow_server", op="advance", dtype="bf16", layers=4, kv_heads=8, dim=128, page=16, rows=250,
             width=512, pages=16001, low=1, high=1900, fanout=1),
        # a small model's cache after some requests left
        dict(name="compact_small", op="compact", dtype="fp32", layers=2, kv_heads=8, dim=64, page=16, rows=16,
             width=32, pages=300, low=5, high=300),
        # a large pool, three fifths live
        dict(name="compact_large", op="compact", dtype="bf16", layers=8, kv_heads=8, dim=128, page=16, rows=100,
             width=128, pages=6000, low=1, high=1000),
        # scores of a decode step's choices
        dict(name="logprobs_step", op="logprobs", dtype="fp32", rows=8, vocab=32000, top=8),
        # scores of a prompt under a model with a large vocabulary
        dict(name="logprobs_prompt", op="logprobs", dtype="bf16", rows=2048, vocab=151936, top=20),
    ]


def _log(rng, lo, hi):
    return int(min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "append", "advance", "compact", "logprobs", "logprobs"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 160000)
        rows = _log(rng, 1, 2048)
        if dtype == "fp32":
            rows = max(1, rows // 2)
        return dict(op=op, dtype=dtype, rows=rows, vocab=vocab, top=rng.choice([0, 1, 5, 8, 20, 32]))
    kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256])
    page = rng.choice([16, 16, 32, 64])
    e = ESIZE[dtype]
    if op in ("attend", "append"):
        budget = 200_000_000 // (kv_heads * dim * e)  # tokens in all
        rows = _log(rng, 1, 256)
        high = _log(rng, 1, max(1, min(131072, budget // rows)))
        low = high if rows == 1 else rng.choice([0, 1, max(1, high // 2), high])
        if op == "attend":
            return dict(op=op, dtype=dtype, rows=rows, heads=kv_heads * rng.choice([1, 1, 2, 3, 4, 8, 16]),
                        kv_heads=kv_heads, dim=dim, page=page, low=min(low, high), high=high)
        new = rng.choice([0, _log(rng, 1, max(1, min(4096, budget // rows)))])
        return dict(op=op, dtype=dtype, rows=rows, kv_heads=kv_heads, dim=dim, page=page, low=min(low, high),
                    high=high, new=new)
    layers = rng.choice([1, 2, 4, 6])
    rows = _log(rng, 4, 200)
    high = _log(rng, 2, 2000)
    fanout = rng.choice([1, 2, 4]) if op == "advance" else 1
    held = rows * (high // page + 2)
    per_page = layers * 2 * kv_heads * page * dim * e
    while held * 2 * per_page > 3_000_000_000 and rows > 4:
        rows = max(4, rows // 2)
        held = rows * (high // page + 2)
    while held * 2 * per_page > 3_000_000_000 and high > 2:
        high = max(2, high // 2)
        held = rows * (high // page + 2)
    case = dict(op=op, dtype=dtype, layers=layers, kv_heads=kv_heads, dim=dim, page=page, rows=rows,
                width=high // page + rng.choice([2, 5, 40]), pages=held + rng.randrange(3, held + 4),
                low=rng.choice([1, high]), high=high)
    if op == "advance":
        case["fanout"] = fanout
    return case


# ------------------------------------------------------------ inputs --

def _spread(low, high, n):
    """n whole numbers from low to high, evenly spread."""
    return np.array([low + (high - low) * i // max(1, n - 1) for i in range(n)], dtype=np.int64)


def _held(case):
    """Tokens in each row before the call, in the order before shuffling."""
    return _spread(case["low"], case["high"], max(1, case["rows"] // case.get("fanout", 1)))


def _tables(lens, rows, width, pages, page, rng):
    """State of a cache whose rows hold `lens` tokens, their pages anywhere in the pool."""
    state = np.zeros(HEADER + rows + pages + rows * width, np.int32)
    table = np.full((rows, width), -1, np.int32)
    ids = rng.permutation(pages)
    at = 0
    refs = np.zeros(pages, np.int32)
    for r, n in enumerate(lens):
        c = -(-int(n) // page)
        table[r, :c] = ids[at:at + c]
        refs[ids[at:at + c]] = 1
        at += c
    state[3] = at
    state[HEADER:HEADER + len(lens)] = lens
    state[HEADER + rows:HEADER + rows + pages] = refs
    state[HEADER + rows + pages:] = table.reshape(-1)
    return state


def _views(state, rows, pages):
    a, b = HEADER + rows, HEADER + rows + pages
    return state[:HEADER], state[HEADER:a], state[a:b], state[b:].view(rows, -1)


def _normal(shape, dtype, gen, scale=1.0):
    t = torch.empty(shape, dtype=dtype, device="cuda")
    return t.normal_(0.0, scale, generator=gen)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.Generator(np.random.PCG64(seed))
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] == "logprobs":
        n, v = case["rows"], case["vocab"]
        s["logits"] = _normal((n, v), dtype, gen, 2.5)
        targets = rng.integers(0, v, n)
        targets[rng.random(n) < 0.05] = -100  # padding
        s["targets"] = torch.from_numpy(targets).cuda()
        return s
    page, kvh, dim = case["page"], case["kv_heads"], case["dim"]
    lens = rng.permutation(_held(case))
    layers = case.get("layers", 1)
    rows = case["rows"]
    if case["op"] == "append":
        new = np.minimum(1, lens) if case["new"] == 0 else rng.permutation(_spread(1, case["new"], rows))
        if case["new"]:
            lens = lens + new
        tokens = rows if case["new"] == 0 else int(new.sum()) + 5
        s["cu"] = None if case["new"] == 0 else torch.from_numpy(
            np.concatenate([[0], np.cumsum(new)]).astype(np.int32)).cuda()
        s["k"] = _normal((tokens, kvh, dim), dtype, gen)
        s["v"] = _normal((tokens, kvh, dim), dtype, gen)
    if case["op"] in ("attend", "append"):
        width = max(1, -(-int(lens.max()) // page))
        pages = int(lens.sum()) // page + rows + 3
    else:
        width, pages = case["width"], case["pages"]
    s["width"], s["pages"] = width, pages
    s["pool"] = _normal((layers, 2, pages, kvh, page, dim), dtype, gen)
    s["state"] = torch.from_numpy(_tables(lens, rows, width, pages, page, rng)).cuda()
    if case["op"] == "attend":
        s["q"] = _normal((rows, case["heads"], dim), dtype, gen, 2.0)
        s["scale"] = dim ** -0.5
    if case["op"] == "advance":
        if case["fanout"] > 1:
            parents = np.minimum(np.arange(rows) // case["fanout"], len(lens) - 1)
        else:
            parents = rng.permutation(rows)
            parents[rng.random(rows) < 0.1] = -1
        s["parents"] = torch.from_numpy(parents.astype(np.int32)).cuda()
    if case["op"] in ("advance", "compact"):
        s["before"] = s["state"].clone()
    if own:
        from s_salaad_b200.kvcache import PagedCache

        s["cache"] = PagedCache(num_layers=layers, num_pages=pages, kv_heads=kvh, head_dim=dim, page_size=page,
                                max_seqs=rows, max_pages=width, dtype=dtype, device="cuda", pool=s["pool"],
                                state=s["state"])
    return s


# --------------------------------------------------------- plain forms --

def _attend_plain(s):
    rows, kvh, dim, page = s["rows"], s["kv_heads"], s["dim"], s["page"]
    _, lens, _, table = _views(s["state"], rows, s["pages"])
    at = table.clamp(min=0).long()
    span = table.shape[1] * page
    k = s["pool"][0, 0][at].permute(0, 2, 1, 3, 4).reshape(rows, kvh, span, dim).float()
    q = s["q"].float().view(rows, kvh, -1, dim)
    seen = (torch.arange(span, device="cuda") < lens[:, None])[:, None, None]
    score = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    score = torch.where(seen, score, float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    v = s["pool"][0, 1][at].permute(0, 2, 1, 3, 4).reshape(rows, kvh, span, dim).float()
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    lse = (top + torch.log(total)).view(rows, -1)
    return {"out": out.view(rows, -1, dim).to(s["q"].dtype), "lse": lse}


def _append_plain(s):
    rows, page = s["rows"], s["page"]
    _, lens, _, table = _views(s["state"], rows, s["pages"])
    token = torch.arange(s["k"].shape[0], device="cuda")
    if s["cu"] is None:
        row, pos = token, lens.long() - 1
        pick = pos >= 0
    else:
        cu = s["cu"].long()
        row = torch.searchsorted(cu, token, right=True) - 1
        pick = row < rows
        row = row.clamp(max=rows - 1)
        pos = lens.long()[row] - (cu[row + 1] - token)
    row, pos = row[pick], pos[pick]
    at = table[row, pos // page].long()
    s["pool"][0, 0][at, :, pos % page] = s["k"][pick]
    s["pool"][0, 1][at, :, pos % page] = s["v"][pick]
    return {"pool": s["pool"]}


def _ceil(a, b):
    return torch.div(a + (b - 1), b, rounding_mode="floor")


def _advance_plain(s):
    rows, pages, page, width = s["rows"], s["pages"], s["page"], s["width"]
    s["state"].copy_(s["before"])
    head, lens, refs, table = _views(s["state"], rows, pages)
    kept = s["parents"] >= 0
    pick = s["parents"].clamp(min=0).long()
    t = torch.where(kept[:, None], table[pick], -1).long()
    low = torch.where(kept, lens[pick], 0).long()
    n = (low > 0).long()  # every row that holds tokens grows by one
    used = torch.zeros(pages + 1, dtype=torch.long, device="cuda")
    used = used.scatter_add(0, torch.where(t >= 0, t, pages).view(-1), torch.ones_like(t).view(-1))[:pages]
    have, want = _ceil(low, page), _ceil(low + n, page)
    row = torch.arange(rows, device="cuda")
    last = t.gather(1, (have - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    shared = (n > 0) & (low % page > 0) & (used[last] > 1)
    bin_ = torch.where(shared, last, pages)
    growers = torch.zeros(pages + 1, dtype=torch.long, device="cuda").scatter_add(0, bin_, torch.ones_like(bin_))
    first = torch.full((pages + 1,), rows, device="cuda").scatter_reduce(0, bin_, row, "amin")
    copy = shared & ~((growers[last] == used[last]) & (first[last] == row))
    need = (want - have) + copy.long()
    free = used == 0
    over = (want > width) & (n > 0)
    fits = (need.sum() <= free.sum()) & ~over.any()
    short = (need.sum() - free.sum()).clamp(min=0)
    copy, want = copy & fits, torch.where(fits, want, have)
    start = torch.cumsum(need, 0) - need
    ids = torch.arange(pages, device="cuda")
    ranks = torch.where(free, torch.cumsum(free.long(), 0) - 1, pages)
    order = torch.zeros(pages + 1, dtype=torch.long, device="cuda").scatter(0, ranks, ids)
    col = torch.arange(width, device="cuda")[None]
    fresh = (col >= have[:, None]) & (col < want[:, None])
    nth = (start + copy.long())[:, None] + col - have[:, None]
    t2 = torch.where(fresh, order[nth.clamp(0, pages)], t)
    own_copy = order[start.clamp(0, pages)]
    t2 = torch.where(copy[:, None] & (col == (have - 1)[:, None]), own_copy[:, None], t2)
    src, dst = last[copy], own_copy[copy]
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    used = torch.zeros(pages + 1, dtype=torch.long, device="cuda")
    used = used.scatter_add(0, torch.where(t2 >= 0, t2, pages).view(-1), torch.ones_like(t2).view(-1))[:pages]
    table.copy_(t2)
    refs.copy_(used)
    lens.copy_(torch.where(fits, low + n, low))
    head.copy_(torch.stack([short, over.sum(), copy.sum(), (used > 0).sum()]))
    return {"state": s["state"], "pool": s["pool"]}


def _compact_plain(s):
    rows, pages = s["rows"], s["pages"]
    s["state"].copy_(s["before"])
    head, _, refs, table = _views(s["state"], rows, pages)
    ids = torch.arange(pages, device="cuda")
    live = refs > 0
    n = live.sum()
    src, dst = ids[live & (ids >= n)], ids[~live & (ids < n)]
    to = ids.clone()
    to[src] = dst
    s["pool"][:, :, dst] = s["pool"][:, :, src]
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()].int(), -1))
    refs[dst] = refs[src]
    refs[src] = 0
    head.copy_(torch.stack([n * 0, n * 0, n * 0 + src.shape[0], n]))
    return {"state": s["state"], "pool": s["pool"]}


def _logprobs_plain(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    lse = top + torch.log(total)
    entropy = torch.log(total)[:, 0] - (e * (x - top)).sum(-1) / total[:, 0]
    del e
    t = s["targets"]
    lp = torch.where(t < 0, 0.0, (x.gather(1, t.clamp(min=0)[:, None]) - lse)[:, 0])
    out = {"logprob": lp, "entropy": entropy}
    if s["top"]:
        bits = (x + 0.0).view(torch.int32)
        key = torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF).long() << 32
        key += torch.arange(x.shape[1] - 1, -1, -1, device="cuda")  # ties go to the lowest index
        at = (x.shape[1] - 1) - (torch.topk(key, s["top"], -1).values & 0xFFFFFFFF)
        out["top_ids"], out["top_logprobs"] = at, x.gather(1, at) - lse
    return out


_PLAIN = {"attend": _attend_plain, "append": _append_plain, "advance": _advance_plain, "compact": _compact_plain,
          "logprobs": _logprobs_plain}


def _own(s):
    op = s["op"]
    if op == "logprobs":
        from s_salaad_b200.ops import token_logprobs

        r = token_logprobs(s["logits"], s["targets"], top=s["top"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if s["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    cache = s["cache"]
    if op == "attend":
        out, lse = cache.attend(0, s["q"], scale=s["scale"], return_lse=True)
        return {"out": out, "lse": lse}
    if op == "append":
        cache.append(0, s["k"], s["v"], cu_tokens=s["cu"])
        return {"pool": s["pool"]}
    s["state"].copy_(s["before"])
    if op == "advance":
        cache.advance(1, parents=s["parents"])
    else:
        cache.compact()
    return {"state": s["state"], "pool": s["pool"]}


def run(state):
    return _own(state) if own else _PLAIN[state["op"]](state)


# ----------------------------------------------------------------- work --

def _copied(case):
    """Pages that an advance by one token has to copy (fanout > 1: all children of a row whose last page is partly
    filled but one)."""
    f, page = case["fanout"], case["page"]
    if f == 1:
        return 0
    held = _held(case)
    extra = case["rows"] - f * len(held)  # rows left over follow the last prompt; its place is shuffled
    return sum((f - 1) + (extra / len(held)) for n in held if n % page)


def work(case):
    e = ESIZE[case["dtype"]]
    if case["op"] == "logprobs":
        n, v, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": n * v * e + n * (8 + 8 + 12 * k), "flops": 5 * n * v}
    page, kvh, dim, rows = case["page"], case["kv_heads"], case["dim"], case["rows"]
    held = _held(case)
    token = 2 * kvh * dim * e
    pages = sum(-(-int(n) // page) for n in held)
    if case["op"] == "attend":
        total, h = int(held.sum()), case["heads"]
        return {"bytes": total * token + rows * h * (2 * dim * e + 4) + 4 * (rows + pages),
                "flops": 4 * total * h * dim}
    if case["op"] == "append":
        n = int(np.minimum(1, held).sum()) if case["new"] == 0 else int(_spread(1, case["new"], rows).sum())
        return {"bytes": 2 * n * token + 8 * rows, "flops": 0}
    book = 4 * (rows + case["pages"])
    per_page = case["layers"] * page * token
    if case["op"] == "advance":
        return {"bytes": int(2 * book + 4 * rows + 4 * pages * (1 + case["fanout"]) + 2 * per_page * _copied(case)),
                "flops": 0}
    moved = pages * (case["pages"] - pages) // case["pages"]  # live pages above the live count, on average
    return {"bytes": 2 * book + 8 * pages + 2 * per_page * moved, "flops": 0}


# ------------------------------------------------------- in 64 bits --

def exact(case, seed):
    if case["op"] not in ("attend", "logprobs"):
        return None  # whole numbers and copies: nothing is rounded
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        lp, ent, val = [], [], []
        for a in range(0, case["rows"], 256):
            x = s["logits"][a:a + 256].double()
            z = torch.logsumexp(x, -1)
            t = s["targets"][a:a + 256]
            lp.append(torch.where(t < 0, 0.0, x.gather(1, t.clamp(min=0)[:, None])[:, 0] - z))
            logp = x - z[:, None]
            ent.append(-(logp.exp() * logp).sum(-1))
            if case["top"]:
                val.append(logp.topk(case["top"], -1).values)
        out = {"logprob": torch.cat(lp), "entropy": torch.cat(ent)}
        if case["top"]:
            out["top_ids"], out["top_logprobs"] = None, torch.cat(val)
        return out
    _, lens, _, table = _views(s["state"], case["rows"], s["pages"])
    kvh, dim = case["kv_heads"], case["dim"]
    outs, lses = [], []
    for r, n in enumerate(lens.tolist()):
        q = s["q"][r].double().view(kvh, -1, dim)
        if n == 0:
            outs.append(torch.zeros(case["heads"], dim, dtype=torch.double, device="cuda"))
            lses.append(torch.full((case["heads"],), float("-inf"), dtype=torch.double, device="cuda"))
            continue
        at = table[r, :-(-n // case["page"])].long()
        k, v = (s["pool"][0, i, at].double().transpose(0, 1).reshape(kvh, -1, dim)[:, :n] for i in (0, 1))
        score = s["scale"] * torch.einsum("hgd,htd->hgt", q, k)
        outs.append(torch.einsum("hgt,htd->hgd", torch.softmax(score, -1), v).reshape(-1, dim))
        lses.append(torch.logsumexp(score, -1).reshape(-1))
    return {"out": torch.stack(outs), "lse": torch.stack(lses)}
