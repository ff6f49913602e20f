"""PagedCache.attend and PagedCache.append against 64 bits.

The bound of each element follows from the kernel's arithmetic
(kv_model.attention) plus half a step of the output type.
"""
from __future__ import annotations

import pytest
import torch

from kv_model import attention, filled_cache
from s_salaad_b200.kvcache import PagedCache

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _check(cache, keys, values, q, scale, layer=0, out=None):
    got, lse = cache.attend(layer, q, scale=scale, out=out, return_lse=True)
    half = torch.finfo(cache.dtype).eps / 2
    for r in range(q.shape[0]):
        o, z, tol, ztol = attention(q[r], keys[layer][r], values[layer][r],
                                    cache.head_dim ** -0.5 if scale is None else scale)
        bound = tol + o.abs() * half + torch.finfo(cache.dtype).tiny
        err = (got[r].double() - o).abs()
        assert bool((err <= bound).all()), (r, float((err - bound).max()), float(err.max()))
        if keys[layer][r].shape[1] == 0:
            assert bool((lse[r] == float("-inf")).all()) and bool((got[r] == 0).all())
        else:
            assert bool(((lse[r].double() - z).abs() <= ztol).all()), (r, float((lse[r].double() - z).abs().max()))
    cache.check()
    return got, lse


def _q(rows, heads, dim, dtype, seed=7, scale=1.0):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(rows, heads, dim, generator=g) * scale).to(dtype).cuda()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 4, 64), (8, 2, 128), (1, 1, 8), (9, 3, 80), (17, 1, 96),
                                                (6, 2, 256), (40, 2, 128), (5, 1, 40)])
def test_shapes(cuda, dtype, heads, kv_heads, dim):
    lens = [0, 1, 15, 16, 17, 33, 64, 65, 200, 0, 511]
    cache, k, v = filled_cache(lens, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype)
    _check(cache, k, v, _q(len(lens), heads, dim, dtype), None)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("layout", ["heads", "slots"])
def test_page_sizes_and_layouts(cuda, dtype, page, layout):
    lens = [page - 1, page, page + 1, 3 * page + 5, 700]
    cache, k, v = filled_cache(lens, kv_heads=2, dim=64, page=page, dtype=dtype, layers=2, layout=layout)
    for layer in (0, 1):
        _check(cache, k, v, _q(5, 6, 64, dtype), 0.2, layer=layer)


@pytest.mark.parametrize("dtype,rows,length,heads,kv_heads", [
    (BF16, 1, 20011, 8, 1), (F16, 2, 9000, 4, 4), (F32, 1, 5003, 4, 1), (BF16, 3, 4097, 32, 8)])
def test_few_rows_are_split_and_joined(cuda, dtype, rows, length, heads, kv_heads):
    lens = [length - 1000 * r for r in range(rows)]
    cache, k, v = filled_cache(lens, kv_heads=kv_heads, dim=128, page=32, dtype=dtype)
    q = _q(rows, heads, 128, dtype)
    a = _check(cache, k, v, q, None)
    b = cache.attend(0, q, return_lse=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])  # whatever the timing


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_ragged_rows(cuda, dtype):
    lens = [(r * 37) % 300 if r % 5 else 0 for r in range(700)]
    cache, k, v = filled_cache(lens, kv_heads=2, dim=64, page=16, dtype=dtype)
    _check(cache, k, v, _q(700, 2, 64, dtype), None)


def test_most_rows(cuda):
    """As many rows as a cache takes, nearly all empty."""
    lens = [0] * 2048
    lens[0], lens[1023], lens[2047] = 5, 100, 333
    cache, k, v = filled_cache(lens, kv_heads=1, dim=256, page=16, dtype=BF16)
    got, _ = cache.attend(0, _q(2048, 2, 256, BF16), return_lse=True)
    for r in (0, 1023, 2047):
        o, _, tol, _ = attention(_q(2048, 2, 256, BF16)[r], k[0][r], v[0][r], 256 ** -0.5)
        assert bool(((got[r].double() - o).abs() <= tol + o.abs() * 2.0 ** -8).all())
    got[[0, 1023, 2047]] = 0
    assert not bool(got.any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,heads,kv_heads", [(64, 8, 8), (128, 32, 8), (256, 20, 1), (40, 3, 3)])
@pytest.mark.parametrize("width", [None, 30, 900, 5000])
def test_few_short_rows(cuda, dtype, dim, heads, kv_heads, width):
    """Short rows with a short table (one launch) and with a long one (split and joined)."""
    lens = [3, 0, 17, 64, 130]
    cache, k, v = filled_cache(lens, kv_heads=kv_heads, dim=dim, page=16, dtype=dtype, width=width)
    _check(cache, k, v, _q(5, heads, dim, dtype), None)


def test_workspace_too_small_is_refused(cuda):
    import ctypes

    from s_salaad_b200 import _lib

    cache, _, _ = filled_cache([20], kv_heads=1, dim=64, page=16, width=100000)
    q, out = _q(1, 1, 64, BF16), torch.empty(1, 1, 64, dtype=BF16, device="cuda")
    lib, ref = _lib.load(), ctypes.byref(cache.struct)
    need = lib.slr_kv_attend_workspace_size(ref, 1, 1)
    assert need > 0 and lib.slr_kv_attend_workspace_size(ref, 2, 1) == 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for ptr, size in ((None, 0), (None, need), (ws.data_ptr(), need - 1)):
        rc = lib.slr_kv_attend(ref, 0, q.data_ptr(), 64, 64, out.data_ptr(), 64, 64, None, 1, 1, 1.0, ptr, size, None)
        assert rc == _lib.SLR_ERR_WORKSPACE and "workspace" in _lib.last_error()


def test_fewer_rows_than_the_cache_holds(cuda):
    lens = [40, 50, 60]
    cache, k, v = filled_cache(lens, kv_heads=2, dim=64, page=16)
    _check(cache, k, v, _q(2, 4, 64, BF16), None)
    assert cache.attend(0, _q(2, 4, 64, BF16)[:0]).shape == (0, 4, 64)


def test_strides_and_alignment_of_q_and_out(cuda):
    cache, k, v = filled_cache([37, 90], kv_heads=2, dim=64, page=16)
    base = _q(2, 4, 64, BF16)
    wide = torch.zeros(2, 5, 67, dtype=BF16, device="cuda")
    q = wide[:, 1:, 3:]
    q.copy_(base)
    out = torch.zeros(4, 2, 65, dtype=BF16, device="cuda").transpose(0, 1)[..., 1:]
    _check(cache, k, v, q, None, out=out)
    assert torch.equal(out, cache.attend(0, base))


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales(cuda, scale, dtype):
    cache, k, v = filled_cache([1, 30, 333], kv_heads=2, dim=64, page=16, dtype=dtype)
    _check(cache, k, v, _q(3, 4, 64, dtype), scale)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_growing_scores(cuda, dtype):
    """Scores that rise along the row move the running maximum at every tile."""
    cache, k, v = filled_cache([500], kv_heads=1, dim=64, page=16, dtype=dtype)
    ramp = torch.linspace(-1, 1, 500, device="cuda").to(dtype)
    k[0][0].copy_(ramp[None, :, None].expand(1, 500, 64))
    for t in range(0, 500, 16):
        e = min(500, t + 16)
        cache.pool[0, 0, int(cache.page_table[0, t // 16]), :, :e - t] = k[0][0][:, t:e]
    _check(cache, k, v, torch.full((1, 2, 64), 4.0, dtype=dtype, device="cuda"), None)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_infinities_and_nan(cuda, dtype):
    """A -inf score has weight 0, a row of them is empty; NaN and +inf scores give NaN."""
    dim = 64
    cache, k, v = filled_cache([100, 100, 100, 100, 2000], kv_heads=1, dim=dim, page=16, dtype=dtype)
    q = torch.zeros(5, 1, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0

    def put(row, t, x):
        page = int(cache.page_table[row, t // 16])
        cache.pool[0, 0, page, 0, t % 16] = 0
        cache.pool[0, 0, page, 0, t % 16, 0] = x

    for t in range(100):
        put(0, t, float("-inf"))
        put(1, t, float("-inf") if t != 41 else 0.0)
        put(2, t, 0.0 if t != 70 else float("inf"))
        put(3, t, 0.0 if t != 99 else float("nan"))
    for t in range(2000):
        put(4, t, float("-inf") if t < 1500 else 0.0)
    got, lse = cache.attend(0, q, scale=1.0, return_lse=True)
    assert not bool(got[0].any()) and bool((lse[0] == float("-inf")).all())
    assert torch.equal(got[1, 0], v[0][1][0, 41]) and float(lse[1]) == 0.0
    assert bool(torch.isnan(got[2:4]).all()) and bool(torch.isnan(lse[2:4]).all())
    want = v[0][4][0, 1500:].double().mean(0)
    spread = v[0][4][0, 1500:].double().abs().mean(0)
    half = torch.finfo(dtype).eps / 2
    # weights of exactly 1: only the sums and the output's rounding are inexact
    assert bool(((got[4, 0].double() - want).abs() <= want.abs() * half + spread * 2000 * 2.0 ** -24 + 1e-9).all())


def test_bad_pages_and_lengths_are_left_out_and_reported(cuda):
    cache, k, v = filled_cache([40, 40, 40, 40], kv_heads=1, dim=64, page=16, garbage=0.0)
    q = _q(4, 2, 64, BF16)
    cache.check()
    cache.page_table[0, 1] = cache.num_pages      # past the pool
    cache.page_table[1, 2] = -7
    cache.lens[2] = -5                            # as empty
    cache.lens[3] = 1 << 30                       # as the row's capacity
    got, lse = cache.attend(0, q, return_lse=True)
    with pytest.raises(ValueError, match="out of range"):
        cache.check()
    cache.check()  # reading it cleared it
    keep0 = torch.cat([k[0][0][:, :16], k[0][0][:, 32:]], 1), torch.cat([v[0][0][:, :16], v[0][0][:, 32:]], 1)
    for r, (kk, vv) in enumerate([keep0, (k[0][1][:, :32], v[0][1][:, :32])]):
        o, _, tol, _ = attention(q[r], kk, vv, 64 ** -0.5)
        assert bool(((got[r].double() - o).abs() <= tol + o.abs() * 2.0 ** -8).all())
    assert not bool(got[2].any())
    full = torch.zeros(1, 48, 64, device="cuda", dtype=BF16)
    kk, vv = full.clone(), full.clone()
    kk[:, :40], vv[:, :40] = k[0][3], v[0][3]
    o, _, tol, _ = attention(q[3], kk, vv, 64 ** -0.5)
    assert bool(((got[3].double() - o).abs() <= tol + o.abs() * 2.0 ** -8).all())


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 bytes and 2^31 elements: the last pages."""
    pages, kvh, page, dim = 140000, 2, 64, 128
    pool = torch.empty(1, 2, pages, kvh, page, dim, dtype=BF16, device="cuda")  # 9.2 GB
    cache = PagedCache(num_layers=1, num_pages=pages, kv_heads=kvh, head_dim=dim, page_size=page, max_seqs=1,
                       max_pages=4, dtype=BF16, pool=pool)
    cache.page_table[0, :3] = torch.tensor([pages - 1, 3, pages - 2], device="cuda", dtype=torch.int32)
    cache.refs[[pages - 1, 3, pages - 2]] = 1
    n = 150
    cache.lens[0] = n
    k, v = (_q(n, kvh, dim, BF16, seed=s) for s in (1, 2))
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    cache.append(0, k, v, cu)
    q = _q(1, 4, dim, BF16)
    _check(cache, [[k.transpose(0, 1)]], [[v.transpose(0, 1)]], q, None)
    del pool, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("kv_heads,dim,page", [(2, 64, 16), (3, 40, 32), (1, 8, 16), (8, 128, 48)])
@pytest.mark.parametrize("aligned", [True, False])
def test_append_packed_prompts(cuda, dtype, kv_heads, dim, page, aligned):
    had, new = [0, 5, 0, 100, 31, 7], [3, 0, 0, 77, 1, page * 2]
    lens = [a + b for a, b in zip(had, new)]
    cache, keys, values = filled_cache(lens, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype, layers=2,
                                       garbage=-1.0)
    before = cache.pool.clone()
    g = torch.Generator(device="cpu").manual_seed(3)
    n = sum(new) + 4  # four tokens of padding
    x = torch.randn(2, n, kv_heads, dim + (0 if aligned else 1), generator=g).to(dtype).cuda()
    k, v = x[0, ..., :dim], x[1, ..., -dim:]
    cu = torch.tensor([0] + [sum(new[:i + 1]) for i in range(len(new))], dtype=torch.int32, device="cuda")
    cache.append(1, k, v, cu)
    cache.check()
    want = before.clone()
    at = 0
    for r in range(len(lens)):
        for t in range(had[r], lens[r]):
            p = int(cache.page_table[r, t // page])
            want[1, 0, p, :, t % page], want[1, 1, p, :, t % page] = k[at], v[at]
            at += 1
    assert torch.equal(cache.pool, want)


def test_append_one_token_per_row(cuda):
    lens = [1, 0, 16, 17, 0]
    cache, _, _ = filled_cache(lens, kv_heads=2, dim=64, page=16, garbage=-1.0)
    before = cache.pool.clone()
    k, v = _q(4, 2, 64, BF16, seed=1), _q(4, 2, 64, BF16, seed=2)  # the last row gets none
    cache.append(0, k, v)
    want = before.clone()
    for r in (0, 2, 3):
        t = lens[r] - 1
        p = int(cache.page_table[r, t // 16])
        want[0, 0, p, :, t % 16], want[0, 1, p, :, t % 16] = k[r], v[r]
    assert torch.equal(cache.pool, want)
    cache.check()


def test_append_reports_what_has_no_place(cuda):
    cache, _, _ = filled_cache([10, 20], kv_heads=1, dim=64, page=16, garbage=0.0)
    before = cache.pool.clone()
    k = _q(12, 1, 64, BF16)
    cache.append(0, k[:12], k[:12], torch.tensor([0, 12, 12], dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="out of range"):
        cache.check()  # 12 tokens cannot be the last of 10: the first two are left out
    p = int(cache.page_table[0, 0])
    before[0, :, p, 0, :10] = k[2:12, 0]
    assert torch.equal(cache.pool, before)
    cache.page_table[1, 1] = cache.num_pages
    cache.append(0, k[:2], k[:2])
    with pytest.raises(ValueError, match="out of range"):
        cache.check()


def test_two_streams_and_a_graph(cuda):
    """Calls of two caches on two streams at once, and replays of a captured
    call while the lengths change."""
    a = filled_cache([900, 31], kv_heads=2, dim=128, page=16, seed=1)
    b = filled_cache([77, 1200], kv_heads=2, dim=128, page=16, seed=2)
    qa, qb = _q(2, 8, 128, BF16, 1), _q(2, 8, 128, BF16, 2)
    want_a, want_b = a[0].attend(0, qa), b[0].attend(0, qb)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got_a, got_b = [], []
    for _ in range(20):
        with torch.cuda.stream(s1):
            got_a.append(a[0].attend(0, qa))
        with torch.cuda.stream(s2):
            got_b.append(b[0].attend(0, qb))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want_a) for g in got_a) and all(torch.equal(g, want_b) for g in got_b)
    cache, k, v = a
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = cache.attend(0, qa, return_lse=True)
    for lens in ([900, 31], [1, 0], [640, 16], [900, 1]):
        cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        o, z = out.clone(), lse.clone()
        e, f = cache.attend(0, qa, return_lse=True)
        assert torch.equal(o, e) and torch.equal(z, f)
        for r in range(2):
            if lens[r]:
                x, _, tol, _ = attention(qa[r], k[0][r][:, :lens[r]], v[0][r][:, :lens[r]], 128 ** -0.5)
                assert bool(((o[r].double() - x).abs() <= tol + x.abs() * 2.0 ** -8).all())
            else:
                assert not bool(o[r].any())


def test_output_in_place_of_q(cuda):
    """q is read before its row's output is written, in one launch and split."""
    for width in (None, 5000):
        cache, k, v = filled_cache([300, 5, 0, 77], kv_heads=2, dim=64, page=16, width=width)
        q = _q(4, 6, 64, BF16)
        want = cache.attend(0, q)
        got = q.clone()
        assert cache.attend(0, got, out=got) is got and torch.equal(got, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_one_q_for_all_rows_and_heads(cuda, dtype):
    cache, k, v = filled_cache([300, 5, 40], kv_heads=2, dim=64, page=16, dtype=dtype)
    q = _q(1, 1, 64, dtype).expand(3, 4, 64)
    assert torch.equal(cache.attend(0, q), cache.attend(0, q.contiguous()))
    _check(cache, k, v, q, None)


def test_refusals(cuda):
    cache, _, _ = filled_cache([10, 20], kv_heads=2, dim=64, page=16)
    q = _q(2, 4, 64, BF16)
    with pytest.raises(TypeError, match="q must be"):
        cache.attend(0, q.float())
    with pytest.raises(ValueError, match="multiple of 2 heads"):
        cache.attend(0, q[:, :3])
    with pytest.raises(ValueError, match="at most 2 rows"):
        cache.attend(0, _q(3, 4, 64, BF16))
    with pytest.raises(ValueError, match=r"\[tokens, heads, 64\]"):
        cache.attend(0, q[..., :32])
    with pytest.raises(ValueError, match="unit stride"):
        cache.attend(0, _q(2, 64, 4, BF16).transpose(1, 2))
    with pytest.raises(ValueError, match="layer out of range"):
        cache.attend(1, q)
    with pytest.raises(ValueError, match="scale must be finite"):
        cache.attend(0, q, scale=float("nan"))
    with pytest.raises(ValueError, match="on cuda:0"):
        cache.attend(0, q.cpu())
    with pytest.raises(ValueError, match="out must be"):
        cache.attend(0, q, out=torch.empty(2, 2, 64, dtype=BF16, device="cuda"))
    with pytest.raises(ValueError, match="no backward"):
        cache.attend(0, q.clone().requires_grad_())
    with torch.no_grad():
        cache.attend(0, q.clone().requires_grad_())
    for out in (q[:1].clone().expand(2, 4, 64), q[:, :1].clone().expand(2, 4, 64)):
        with pytest.raises(ValueError, match="overlaps itself"):
            cache.attend(0, q, out=out)
    kv = q[:, :2]
    with pytest.raises(ValueError, match="k and v must be"):
        cache.append(0, q, q)
    with pytest.raises(ValueError, match="k and v must be"):
        cache.append(0, kv, kv[:1])
    with pytest.raises(ValueError, match="tokens out of range"):
        cache.append(0, _q(3, 2, 64, BF16), _q(3, 2, 64, BF16))
    with pytest.raises(TypeError, match="cu_tokens must be int32"):
        cache.append(0, kv, kv, torch.zeros(3, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match=r"cu_tokens must be \[3\]"):
        cache.append(0, kv, kv, torch.zeros(2, dtype=torch.int32, device="cuda"))
    pool = torch.zeros(1, 2, 4, 2, 16, 64, dtype=BF16, device="cuda")
    kw = dict(num_layers=1, num_pages=4, kv_heads=2, head_dim=64, page_size=16, max_seqs=2, max_pages=2)
    with pytest.raises(TypeError, match="pool must be"):
        PagedCache(**kw, dtype=F16, pool=pool)
    with pytest.raises(ValueError, match="pool must be"):
        PagedCache(**kw, pool=pool[:, :, :3])
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache(**kw, pool=torch.zeros(1, 2, 4, 2, 32, 64, dtype=BF16, device="cuda")[:, :, :, :, :16])
    with pytest.raises(ValueError, match="on cuda:1"):
        PagedCache(**kw, pool=pool, device="cuda:1")
    with pytest.raises(ValueError, match="state must be"):
        PagedCache(**kw, pool=pool, state=torch.zeros(3, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
