"""ops.token_logprobs against 64 bits.

Bounds: x - lse carries the rounding of its last subtraction and of lse
(2^-23 of |x| + |lse|), exp2's and the sums' relative error (2^-20 + vocab
2^-24, less by far for tree sums); the entropy, a weighted mean of t = x - max,
carries the same relative error of mean |t| on top.
"""
from __future__ import annotations

import pytest
import torch

from s_salaad_b200 import _lib
from s_salaad_b200.ops import token_logprobs

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = float("inf")


def _logits(rows, vocab, dtype, seed=0, scale=2.5):
    g = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(rows, vocab, generator=g) * scale).to(dtype).cuda()


def _order(x, top):
    """Greatest first, ties by lower index, -0 = +0, NaN as -inf."""
    v = torch.nan_to_num(x.double(), nan=-INF, posinf=INF, neginf=-INF) + 0.0
    return torch.sort(v, dim=-1, descending=True, stable=True).indices[..., :top]


def _check(x, targets, top):
    r = token_logprobs(x, targets, top=top)
    d = x.double()
    lse = torch.logsumexp(d, -1)
    rel = 2.0 ** -20 + x.shape[-1] * 2.0 ** -24
    p = torch.exp(d - lse[:, None])
    logp = torch.where(p > 0, d - lse[:, None], 0.0)
    ent = -(p * logp).sum(-1)
    mean_t = (p * torch.where(p > 0, (d.amax(-1, keepdim=True) - d).abs(), 0.0)).sum(-1)
    assert bool(((r.entropy.double() - ent).abs() <= rel * (2 * mean_t + 1) + ent * 2.0 ** -22).all())
    if targets is not None:
        t = targets.clamp(min=0)[:, None]
        want = torch.where(targets < 0, 0.0, (d.gather(1, t) - lse[:, None])[:, 0])
        tol = rel + 2.0 ** -22 * (d.gather(1, t)[:, 0].abs() + lse.abs())
        ok = (r.logprob.double() - want).abs() <= tol
        assert bool((ok | (r.logprob.double() == want)).all())
    if top:
        ids = _order(x, top)
        assert torch.equal(r.top_ids, ids)
        want = d.gather(1, ids) - lse[:, None]
        tol = rel + 2.0 ** -22 * (d.gather(1, ids).abs() + lse.abs()[:, None])
        ok = ((r.top_logprobs.double() - want).abs() <= tol) | (r.top_logprobs.double() == want)
        assert bool(ok.all())
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


def _targets(rows, vocab, seed=1):
    g = torch.Generator(device="cpu").manual_seed(seed)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[::5] = -100
    return t.cuda()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 7, 7), (5, 32, 32), (2, 97, 5), (4, 1001, 32), (1, 32000, 8),
                                            (9, 32000, 0), (2, 151936, 20), (700, 4099, 4), (1300, 515, 32)])
def test_shapes(cuda, dtype, rows, vocab, top):
    _check(_logits(rows, vocab, dtype), _targets(rows, vocab), top)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shift", [0, 1, 3, 7])
def test_unaligned_rows(cuda, dtype, shift):
    wide = _logits(6, 5003 + shift, dtype)
    _check(wide[:, shift:], _targets(6, 5003), 16)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("rows", [2, 900])
def test_ties_go_to_the_lowest_index(cuda, dtype, rows):
    vocab = 9001
    g = torch.Generator(device="cpu").manual_seed(2)
    x = torch.randint(-2, 3, (rows, vocab), generator=g).to(dtype).cuda()
    x[0] = 1.0
    x[1, ::2] = -0.0
    x[1, 1::2] = 0.0
    _check(x, _targets(rows, vocab), 32)


@pytest.mark.parametrize("rows", [1, 900])
def test_sorted_and_clustered_rows(cuda, rows):
    """The best tokens side by side, rising and falling: many in one thread's
    vectors, and more ties at the top than the candidate buffer holds."""
    vocab = 40000
    up = torch.arange(vocab, device="cuda", dtype=F32).expand(rows, vocab) * 1e-3
    _check(up, None, 32)
    _check(up.flip(-1).contiguous(), None, 32)
    x = torch.zeros(rows, vocab, dtype=BF16, device="cuda")
    x[:, 1000:1040] = 5.0
    _check(x, None, 32)
    # each thread's first vector holds its greatest value, the others nearly as much
    y = torch.full((rows, vocab), 1.0, device="cuda")
    y[:, -30000:] += torch.linspace(0, 1e-3, 30000, device="cuda")
    y[:, 0:4] = 3.0
    _check(y, None, 32)


def test_masked_vocabulary(cuda):
    for dtype in (BF16, F32):
        x = _logits(6, 3001, dtype)
        x[:, 100:2900] = -INF
        x[1] = -INF
        x[1, 77] = 2.0            # one token left: probability 1
        x[2, :] = torch.finfo(dtype).min
        x[3, :] = torch.finfo(dtype).min
        x[3, 5] = 0.0
        t = torch.tensor([500, 77, 3, 4, 5, -1], device="cuda")
        r = token_logprobs(x, t, top=8)
        assert float(r.logprob[0]) == -INF and float(r.logprob[1]) == 0.0 and float(r.entropy[1]) == 0.0
        assert r.top_ids[1].tolist() == [77, 0, 1, 2, 3, 4, 5, 6]
        assert r.top_logprobs[1, 1:].tolist() == [-INF] * 7
        n = torch.tensor(float((x[2] != -INF).sum())).log()
        assert abs(float(r.entropy[2]) - float(n)) < 1e-4 and abs(float(r.logprob[2]) + float(n)) < 1e-4
        assert float(r.entropy[3]) == 0.0 and not bool(torch.isnan(r.logprob).any())
        assert float(r.logprob[5]) == 0.0
        _check(x[[0, 4, 5]], t[[4, 4, 4]], 32)


def test_rows_without_a_distribution_give_nan(cuda):
    for rows in (4, 700):
        x = _logits(rows, 2000, BF16)
        x[0] = -INF
        x[1, 5] = INF
        x[2, 1999] = float("nan")
        t = torch.full((rows,), 7, device="cuda")
        r = token_logprobs(x, t, top=3)
        assert bool(torch.isnan(r.logprob[:3]).all() and torch.isnan(r.entropy[:3]).all()
                    and torch.isnan(r.top_logprobs[:3]).all())
        assert r.top_ids[0].tolist() == [0, 1, 2] and int(r.top_ids[1, 0]) == 5
        assert torch.equal(r.top_ids, _order(x, 3))
        assert not bool(torch.isnan(r.logprob[3:]).any())
        t[:] = -1
        assert not bool(token_logprobs(x, t).logprob.any())


def test_target_past_the_vocabulary_is_reported(cuda):
    import ctypes

    lib = _lib.load()
    x = _logits(3, 50, F32)
    r = token_logprobs(x, torch.tensor([0, 50, 2 ** 40], device="cuda"))
    assert bool(torch.isnan(r.logprob[1:]).all()) and not bool(torch.isnan(r.logprob[0]))
    st = ctypes.c_int(-1)
    _lib.check(lib.slr_device_status(ctypes.byref(st)))
    assert st.value == _lib.SLR_ERR_BAD_INDEX
    _lib.check(lib.slr_device_status(ctypes.byref(st)))
    assert st.value == _lib.SLR_OK


def test_leading_dimensions_strides_and_graph(cuda):
    x = _logits(12, 999, BF16).view(3, 4, 999)
    t = _targets(12, 999).view(3, 4)
    a, b = token_logprobs(x, t, top=4), token_logprobs(x.view(12, 999), t.view(12), top=4)
    for u, v in zip(a, b):
        assert u.shape[:2] == (3, 4) and torch.equal(u.view(v.shape), v)
    c = token_logprobs(x.transpose(0, 1), t.transpose(0, 1), top=4, entropy=False)
    # Row i * 999 elements starts at another 16-byte offset than before, so its sums are taken in another order: each
    # side is within rel + 2^-22 (|x| + |lse|) of 64 bits (module comment), with |x| and |lse| below 20 here.
    tol = 2 * (2.0 ** -20 + 999 * 2.0 ** -24 + 2.0 ** -22 * 40)
    assert c.entropy is None and bool(((c.logprob - a.logprob.transpose(0, 1)).abs() <= tol).all())
    assert torch.equal(c.top_ids, a.top_ids.transpose(0, 1))
    z = token_logprobs(x[:0], t[:0], top=2)
    assert z.logprob.shape == (0, 4) and z.top_ids.shape == (0, 4, 2)
    one = token_logprobs(x[0, 0], t[0, 0], top=2)
    assert one.logprob.shape == () and torch.equal(one.top_ids, a.top_ids[0, 0, :2])
    step = token_logprobs(x[:, -1], top=1)  # rows 4 x vocab apart
    assert torch.equal(step.top_ids, a.top_ids[:, -1, :1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = token_logprobs(x, t, top=4)
    x.copy_(_logits(12, 999, BF16, seed=9).view(3, 4, 999))
    graph.replay()
    for u, v in zip(r, token_logprobs(x, t, top=4)):
        assert torch.equal(u, v)


def test_refusals(cuda):
    x = _logits(3, 50, F32)
    t = torch.zeros(3, dtype=torch.int64, device="cuda")
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x, top=33)
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x[:, :5].contiguous(), top=6)
    with pytest.raises(TypeError, match="int64"):
        token_logprobs(x, t.int())
    with pytest.raises(ValueError, match="targets must be"):
        token_logprobs(x, t[:2])
    with pytest.raises(ValueError, match="targets must be"):
        token_logprobs(x, t.cpu())
    with pytest.raises(TypeError, match="float32/float16/bfloat16"):
        token_logprobs(x.double())
    with pytest.raises(ValueError, match="no backward"):
        token_logprobs(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="CUDA tensor"):
        token_logprobs(x.cpu())
