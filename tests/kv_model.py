"""A plain model of the paged cache's book-keeping and attention, for tests.

:class:`Book` restates the rules of ``slr_kv_advance`` / ``slr_kv_compact``
row by row in Python; :func:`attention` is the definition in 64 bits with an
error bound that follows from the arithmetic of a correct kernel.
"""
from __future__ import annotations

import numpy as np
import torch

HEADER = 4


class Book:
    """Header, lens, refs and table as Python lists (same rules, no GPU)."""

    def __init__(self, rows: int, pages: int, width: int, page: int):
        self.rows, self.pages, self.width, self.page = rows, pages, width, page
        self.header = [0, 0, 0, 0]
        self.lens = [0] * rows
        self.table = [[-1] * width for _ in range(rows)]

    def refs(self) -> list[int]:
        n = [0] * self.pages
        for row in self.table:
            for p in row:
                if p >= 0:
                    n[p] += 1
        return n

    def state(self) -> list[int]:
        return self.header + self.lens + self.refs() + [p for row in self.table for p in row]

    def _pages(self, n: int) -> int:
        return -(-n // self.page)

    def advance(self, n_new, parents=None) -> list[tuple[int, int]]:
        """Applies a step; returns the page copies (src, dst)."""
        if parents is not None:
            old_t, old_l = [list(r) for r in self.table], list(self.lens)
            for i, p in enumerate(parents):
                self.table[i] = list(old_t[p]) if p >= 0 else [-1] * self.width
                self.lens[i] = old_l[p] if p >= 0 else 0
        grow = [0] * self.rows
        for i in range(self.rows):
            n = n_new if isinstance(n_new, int) else n_new[i]
            if n < 0:
                self.lens[i] = max(0, self.lens[i] + n)
                for c in range(self._pages(self.lens[i]), self.width):
                    self.table[i][c] = -1
            elif n > 0 and (self.lens[i] > 0 or not isinstance(n_new, int)):
                grow[i] = n
        refs = self.refs()
        sharers: dict[int, list[int]] = {}
        for i in range(self.rows):
            if grow[i] and self.lens[i] % self.page:
                last = self.table[i][self.lens[i] // self.page]
                if refs[last] > 1:
                    sharers.setdefault(last, []).append(i)
        copy = {i for p, s in sharers.items() for i in (s[1:] if len(s) == refs[p] else s)}
        need = [self._pages(self.lens[i] + grow[i]) - self._pages(self.lens[i]) + (i in copy) for i in range(self.rows)]
        free = [p for p in range(self.pages) if refs[p] == 0]
        over = sum(self.lens[i] + grow[i] > self.width * self.page for i in range(self.rows))
        live = self.pages - len(free)
        if over or sum(need) > len(free):
            self.header = [max(0, sum(need) - len(free)), over, 0, live]
            return []
        pairs, at = [], 0
        for i in range(self.rows):
            mine = free[at:at + need[i]]
            at += need[i]
            c = self._pages(self.lens[i])
            if i in copy:
                pairs.append((self.table[i][c - 1], mine[0]))
                self.table[i][c - 1] = mine[0]
                mine = mine[1:]
            self.table[i][c:c + len(mine)] = mine
            self.lens[i] += grow[i]
        self.header = [0, 0, len(pairs), live + at]
        return pairs

    def compact(self) -> list[tuple[int, int]]:
        refs = self.refs()
        n = sum(r > 0 for r in refs)
        src = [p for p in range(n, self.pages) if refs[p]]
        dst = [p for p in range(n) if not refs[p]]
        to = dict(zip(src, dst))
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        self.header = [0, 0, len(src), n]
        return list(zip(src, dst))


def attention(q, k, v, scale):
    """q [heads, dim], k and v [kv_heads, T, dim] (any dtype): (out, lse) in
    64 bits and elementwise bounds of a kernel with fp32 sums whose
    probabilities keep 16 bits, before the output's rounding.

    A score of D products summed in fp32 is off by at most (D + 4) 2^-24
    scale Σ|q k|; that is also the relative error of its exponential, to
    which exp2 and its argument add 2^-20 and 16-bit probabilities 2^-16; T
    additions add T 2^-24.  Numerator and denominator each carry that.
    """
    heads, dim = q.shape
    kvh, T, _ = k.shape
    q, k, v = q.double().reshape(kvh, -1, dim), k.double(), v.double()
    if T == 0:
        z = torch.zeros(heads, dim, dtype=torch.double, device=q.device)
        return z, torch.full((heads,), float("-inf"), dtype=torch.double, device=q.device), z, z[:, 0]
    s = scale * torch.einsum("hgd,htd->hgt", q, k)
    mag = abs(scale) * torch.einsum("hgd,htd->hgt", q.abs(), k.abs()).amax(-1)
    p = torch.softmax(s, -1)
    eps = (dim + 4) * 2.0 ** -24 * mag + 2.0 ** -20 + T * 2.0 ** -24
    o = torch.einsum("hgt,htd->hgd", p, v)
    spread = torch.einsum("hgt,htd->hgd", p, v.abs())
    lse = torch.logsumexp(s, -1)
    return (o.reshape(heads, dim), lse.reshape(heads), (spread * (2 * eps + 2.0 ** -16)[..., None]).reshape(heads, dim),
            (eps + lse.abs() * 2.0 ** -21).reshape(heads))


def filled_cache(lens, *, kv_heads, dim, page, width=None, layers=1, dtype=torch.bfloat16, device="cuda", seed=0,
                 garbage=float("nan"), layout="heads", extra=3):
    """A PagedCache whose rows hold `lens` random tokens in scattered pages;
    every slot that holds no token is `garbage`.  Returns (cache, keys, values)
    with the contiguous tokens [layer][row] -> [kv_heads, T, dim]."""
    from s_salaad_b200.kvcache import PagedCache

    rng = np.random.Generator(np.random.PCG64(seed))
    rows = len(lens)
    width = width or max(1, max(-(-n // page) for n in lens))
    used = sum(-(-n // page) for n in lens)
    pages = used + extra
    if layout == "heads":
        pool = torch.full((layers, 2, pages, kv_heads, page, dim), garbage, dtype=dtype, device=device)
    else:  # slots before heads, keys and values of a page side by side
        pool = torch.full((pages, layers, 2, page, kv_heads, dim), garbage, dtype=dtype,
                          device=device).permute(1, 2, 0, 4, 3, 5)
    cache = PagedCache(num_layers=layers, num_pages=pages, kv_heads=kv_heads, head_dim=dim, page_size=page,
                       max_seqs=rows, max_pages=width, dtype=dtype, device=device, pool=pool)
    ids = rng.permutation(pages)[:used]
    table = np.full((rows, width), -1, np.int32)
    at = 0
    for r, n in enumerate(lens):
        c = -(-n // page)
        table[r, :c] = ids[at:at + c]
        at += c
    refs = np.zeros(pages, np.int32)
    refs[ids] = 1
    cache.page_table.copy_(torch.from_numpy(table))
    cache.refs.copy_(torch.from_numpy(refs))
    cache.lens.copy_(torch.tensor(list(lens), dtype=torch.int32))
    cache.header[3] = used
    gen = torch.Generator(device="cpu").manual_seed(seed + 1)
    keys, values = [], []
    for layer in range(layers):
        ks, vs = [], []
        for r, n in enumerate(lens):
            kv = torch.randn(2, kv_heads, n, dim, generator=gen).to(dtype).to(device)
            for t in range(0, n, page):
                e = min(n, t + page)
                pool[layer, :, int(table[r, t // page]), :, :e - t] = kv[:, :, t:e]
            ks.append(kv[0])
            vs.append(kv[1])
        keys.append(ks)
        values.append(vs)
    return cache, keys, values
