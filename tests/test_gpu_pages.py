"""PagedCache.advance, compact and copy_pages: the state is compared word for
word with a row-by-row model (kv_model.Book), the pool bit for bit."""
from __future__ import annotations

import random

import pytest
import torch

from kv_model import Book, attention
from s_salaad_b200.kvcache import PagedCache

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _pair(rows, pages, width, page=16, layers=2, kv_heads=2, dim=8, dtype=BF16):
    cache = PagedCache(num_layers=layers, num_pages=pages, kv_heads=kv_heads, head_dim=dim, page_size=page,
                       max_seqs=rows, max_pages=width, dtype=dtype)
    cache.pool.copy_(torch.arange(pages, device="cuda").view(1, 1, pages, 1, 1, 1) % 251)
    return cache, Book(rows, pages, width, page)


def _vec(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _same(cache, book):
    got, want = cache.state.tolist(), book.state()
    if got != want:
        a, b = 4 + book.rows, 4 + book.rows + book.pages
        assert got[:4] == want[:4]
        assert got[4:a] == want[4:a]
        assert got[a:b] == want[a:b]
        assert got[b:] == want[b:]


def _step(cache, book, n_new, parents=None):
    pool = cache.pool.clone()
    pairs = book.advance(n_new, parents)
    cache.advance(n_new if isinstance(n_new, int) else _vec(n_new), None if parents is None else _vec(parents))
    _same(cache, book)
    for s, d in pairs:
        pool[:, :, d] = pool[:, :, s]
    assert torch.equal(cache.pool, pool)
    return pairs


def test_grow_fork_copy_rollback_end(cuda):
    cache, book = _pair(4, 20, 4)
    _step(cache, book, [20, 16, 0, 1])
    _step(cache, book, 1)
    assert _step(cache, book, 0, [0, 0, 0, 1]) == []          # fork without growth shares everything
    assert len(_step(cache, book, 1)) == 2                    # three rows share page 1 and all grow: the lowest keeps it
    _step(cache, book, 0, [0, 0, 2, 3])
    assert len(_step(cache, book, [0, 1, 1, 1])) == 1         # row 0 stays: row 1 copies
    _step(cache, book, [-3, -100, 0, -17])
    _step(cache, book, 1)                                     # the emptied row stays empty
    _step(cache, book, 0, [-1, 3, -1, 2])
    _step(cache, book, [5, 0, 40, -1])
    _step(cache, book, 0, [-1] * 4)
    assert not bool(cache.refs.any()) and bool((cache.page_table == -1).all())
    cache.check()


def test_growth_is_all_or_nothing(cuda):
    cache, book = _pair(3, 5, 4)
    _step(cache, book, [30, 16, 1])
    _step(cache, book, [0, 1, 0], [0, 1, 2])
    before = cache.state.clone()
    _step(cache, book, [3, 16, 16])                           # three pages short
    with pytest.raises(RuntimeError, match="3 pages missing"):
        cache.check()
    assert torch.equal(before[4:], cache.state[4:])
    _step(cache, book, [40, 0, 0])                            # past 4 pages
    with pytest.raises(RuntimeError, match="1 rows past"):
        cache.check()
    _step(cache, book, 1, [0, -1, 2])                         # room again: the ended row's pages are free
    cache.check()


@pytest.mark.parametrize("rows,pages,width", [(1, 3, 2), (7, 40, 6), (33, 300, 9), (200, 9000, 70),
                                              (512, 6000, 512), (513, 6000, 20), (40, 3000, 513),
                                              (700, 5000, 12)])
def test_random_steps(cuda, rows, pages, width):
    """Random forks, ends, rollbacks, growth and compactions."""
    rng = random.Random(rows)
    cache, book = _pair(rows, pages, width, layers=1, kv_heads=1)
    for i in range(12):
        parents = None
        if i % 3 == 1:
            parents = [rng.choice([-1] + [rng.randrange(rows)] * 4) for _ in range(rows)]
        kind = rng.randrange(4)
        if kind == 0:
            n_new = rng.choice([0, 1, 1, 3, -1])
        else:
            n_new = [rng.choice([0, 1, 1, 2, 15, 17, 40, -1, -20]) if rng.random() < 0.7 else 0 for _ in range(rows)]
        _step(cache, book, n_new, parents)
        if i % 4 == 3:
            pool = cache.pool.clone()
            pairs = book.compact()
            cache.compact()
            _same(cache, book)
            for s, d in pairs:
                pool[:, :, d] = pool[:, :, s]
            assert torch.equal(cache.pool, pool)


def test_long_rows_grow_at_once(cuda):
    cache, book = _pair(3, 30000, 12000, layers=1, kv_heads=1)
    _step(cache, book, [11000 * 16, 5, 12000 * 16])
    _step(cache, book, [1, 16, -100000])
    _step(cache, book, 1, [2, 0, 2])
    _step(cache, book, 0, [2, -1, -1])
    book.compact()
    cache.compact()
    _same(cache, book)


def test_bad_parents_and_state_are_reported(cuda):
    cache, book = _pair(3, 10, 3)
    _step(cache, book, [5, 6, 7])
    cache.advance(0, _vec([2, 3, 1]))                          # row 3 does not exist: row 1 ends
    with pytest.raises(ValueError, match="out of range"):
        cache.check()
    assert cache.lens.tolist() == [7, 0, 6]
    cache.page_table[0, 0] = 10
    cache.advance(1)
    with pytest.raises(ValueError, match="out of range"):
        cache.check()


@pytest.mark.parametrize("dtype,kv_heads,dim,page", [(BF16, 2, 64, 16), (F32, 1, 8, 16), (F16, 3, 40, 48)])
def test_copy_pages(cuda, dtype, kv_heads, dim, page):
    cache = PagedCache(num_layers=3, num_pages=50, kv_heads=kv_heads, head_dim=dim, page_size=page, max_seqs=1,
                       max_pages=1, dtype=dtype)
    cache.pool.copy_(torch.randn(cache.pool.shape, device="cuda"))
    want = cache.pool.clone()
    src, dst = [3, 49, 3, 7], [0, 20, 48, 7]
    cache.copy_pages(_vec(src), _vec(dst))
    for s, d in zip(src, dst):
        want[:, :, d] = want[:, :, s]
    assert torch.equal(cache.pool, want)
    cache.copy_pages(_vec([]), _vec([]))
    cache.check()
    # 1 -> 2 and 2 -> 4 clash, 5 -> 6 twice, 50 and -1 do not exist; 8 -> 9 is fine
    cache.copy_pages(_vec([1, 2, 5, 5, 50, 0, 8]), _vec([2, 4, 6, 6, 10, -1, 9]))
    want[:, :, 9] = want[:, :, 8]
    assert torch.equal(cache.pool, want)
    with pytest.raises(ValueError, match="out of range"):
        cache.check()
    cache.check()


def test_pages_of_another_layout_are_copied(cuda):
    pool = torch.randn(30, 2, 2, 16, 3, 8, device="cuda").permute(1, 2, 0, 4, 3, 5)
    cache = PagedCache(num_layers=2, num_pages=30, kv_heads=3, head_dim=8, page_size=16, max_seqs=2, max_pages=3,
                       dtype=F32, pool=pool)
    cache.advance(_vec([20, 0]))
    cache.advance(0, _vec([0, 0]))
    want = pool.clone()
    cache.advance(1)
    assert cache.page_table.tolist() == [[0, 1, -1], [0, 2, -1]]
    want[:, :, 2] = want[:, :, 1]
    assert torch.equal(pool, want)


def test_refusals(cuda):
    cache, _ = _pair(3, 10, 3)
    with pytest.raises(TypeError, match="parents must be int32"):
        cache.advance(1, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match=r"parents must be \[3\]"):
        cache.advance(1, _vec([0, 1]))
    with pytest.raises(ValueError, match=r"n_new must be \[3\]"):
        cache.advance(torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ValueError, match="n_new out of range"):
        cache.advance(1 << 31)
    with pytest.raises(ValueError, match=r"dst must be \[2\]"):
        cache.copy_pages(_vec([0, 1]), _vec([2]))
    assert not bool(cache.state[:7].any())


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_run_of_them_together_eager_and_replayed(cuda, dtype):
    """Prompts, decode steps with forks and ends, a compaction: attention sees
    each row's own history, eagerly and from one captured step."""
    rows, kvh, heads, dim, page = 6, 2, 4, 64, 16
    cache = PagedCache(num_layers=2, num_pages=60, kv_heads=kvh, head_dim=dim, page_size=page, max_seqs=rows,
                       max_pages=8, dtype=dtype)
    cache.pool.fill_(float("nan"))
    gen = torch.Generator(device="cpu").manual_seed(0)
    new = [17, 1, 0, 40, 0, 0]
    hist = [[[torch.empty(0, kvh, dim, dtype=dtype, device="cuda") for _ in range(rows)] for _ in "kv"] for _ in "01"]
    cache.advance(_vec(new))
    cu = _vec([0, 17, 18, 18, 58, 58, 58])
    for layer in range(2):
        kv = torch.randn(2, 58, kvh, dim, generator=gen).to(dtype).cuda()
        cache.append(layer, kv[0], kv[1], cu)
        for i in range(2):
            for r in range(rows):
                hist[layer][i][r] = kv[i, int(cu[r]):int(cu[r + 1])]
    parents = torch.zeros(rows, dtype=torch.int32, device="cuda")
    k, v, q = (torch.zeros(2, rows, h, dim, dtype=dtype, device="cuda") for h in (kvh, kvh, heads))
    outs = [None, None]

    def step():
        cache.advance(1, parents)
        for layer in range(2):
            cache.append(layer, k[layer], v[layer])
            outs[layer] = cache.attend(layer, q[layer])

    plan = [[0, 0, 1, 3, 3, -1], [0, 1, 2, 3, 4, 5], [4, 4, 4, 0, -1, 1], [0, 1, 2, 3, 4, 5], [5, 0, 3, -1, -1, 5]]
    graph = None
    for i, p in enumerate(plan * 2):
        parents.copy_(_vec(p))
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=gen))
        if i == 3:  # the graph's first run is its capture's replay: advance must not run twice
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        if graph is None:
            step()
        else:
            graph.replay()
        if i == 6:
            cache.compact()
            for layer in range(2):
                outs[layer].copy_(cache.attend(layer, q[layer]))
        cache.check()
        half = torch.finfo(dtype).eps / 2
        for layer in range(2):
            for j, new_tok in enumerate((k, v)):
                old = hist[layer][j]
                hist[layer][j] = [torch.cat([old[a], new_tok[layer, r:r + 1]]) if a >= 0 and len(old[a]) else old[a][:0]
                                  if a >= 0 else old[0][:0] for r, a in enumerate(p)]
            for r in range(rows):
                kk, vv = (hist[layer][j][r].transpose(0, 1) for j in range(2))
                o, _, tol, _ = attention(q[layer, r], kk, vv, dim ** -0.5)
                assert bool(((outs[layer][r].double() - o).abs() <= tol + o.abs() * half + 1e-9).all()), (i, layer, r)
