"""PagedCache.attend where the weights' own arithmetic shows: far apart, close
together, and scores of any size."""
from __future__ import annotations

import pytest
import torch

import test_gpu_attend as attend_tests
from kv_model import attention, filled_cache

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _put(cache, layer, kv, row, tokens):
    """tokens [kv_heads, T, dim] as the keys (kv = 0) or values (1) of a row."""
    page, n = cache.page_size, tokens.shape[1]
    for t in range(0, n, page):
        e = min(n, t + page)
        cache.pool[layer, kv, int(cache.page_table[row, t // page]), :, :e - t] = tokens[:, t:e]


@pytest.mark.parametrize("width,length", [(None, 300), (500, 6000)])
@pytest.mark.parametrize("powers", [20, 24, 26])
@pytest.mark.parametrize("first", [True, False])
def test_one_dominating_token_in_fp16(cuda, width, length, powers, first):
    """One token (a sink) has nearly all the weight and the value 0, the others
    2^-20 to 2^-26 of it and large values: the output is theirs alone.

    Bound: kv_model.attention's, and fp16's fixed step for small weights, which
    are held to within 2^-32 of the greatest."""
    dim = 64
    cache, _, _ = filled_cache([length] * 3, kv_heads=1, dim=dim, page=16, dtype=F16, width=width)
    q = torch.zeros(3, 2, dim, dtype=F16, device="cuda")
    q[:, 0, 0], q[:, 1, 0] = 1.0, 0.5
    at = 0 if first else length // 3
    g = torch.Generator(device="cpu").manual_seed(powers)
    keys, values = [], []
    for r in range(3):
        k, v = torch.zeros(1, length, dim), torch.rand(1, length, dim, generator=g) * 3e4 + 2e4
        k[0, :, 0] = -powers * 0.6931 + torch.rand(length, generator=g) * 0.05 * r
        k[0, at], v[0, at] = 0.0, 0.0
        k, v = k.to(F16).cuda(), v.to(F16).cuda()
        _put(cache, 0, 0, r, k)
        _put(cache, 0, 1, r, v)
        keys.append(k)
        values.append(v)
    got = cache.attend(0, q, scale=1.0)
    for r in range(3):
        o, _, tol, _ = attention(q[r], keys[r], values[r], 1.0)
        s = torch.einsum("hd,td->ht", q[r].double(), keys[r][0].double())
        total = torch.exp(s - s.amax(-1, keepdim=True)).sum(-1, keepdim=True)
        step = 2.0 ** -32 * values[r][0].double().sum(0) / total
        bound = tol + o.abs() * 2.0 ** -11 + step + 2.0 ** -25
        err = (got[r].double() - o).abs()
        assert bool((err <= bound).all()), (r, float((err / o.abs()).max()), float((bound / o.abs()).max()))
    cache.check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_weights_that_nearly_cancel(cuda, dtype):
    """Two tokens with values 1 and -1 whose scores a and a + 2^-16 are exact in
    fp32: the output is the difference of their weights, which 16-bit weights
    lose.

    Bound: each weight's relative error is that of the score times log2 e (two
    roundings, |x| < 1.3: 2^-23) and of exp2 (2^-22): below 2^-21, the same for
    the denominator; then half a step of the output."""
    rows, dim = 128, 64
    cache, _, _ = filled_cache([3] * rows, kv_heads=1, dim=dim, page=16, dtype=dtype)
    a = (-torch.arange(1, rows + 1).double() / 144).to(BF16 if dtype == F32 else dtype)
    q = torch.zeros(rows, 1, dim, dtype=dtype, device="cuda")
    q[:, :, :2] = 1.0
    spread, want = torch.empty(rows).double(), torch.empty(rows).double()
    for r in range(rows):
        k, v = torch.zeros(1, 3, dim), torch.zeros(1, 3, dim)
        k[0, 1:, 0] = float(a[r])
        k[0, 1, 1] = 2.0 ** -16
        v[0, 1], v[0, 2] = 1.0, -1.0
        _put(cache, 0, 0, r, k.to(dtype).cuda())
        _put(cache, 0, 1, r, v.to(dtype).cuda())
        s = torch.stack([a[r].double() * 0, a[r].double() + 2.0 ** -16, a[r].double()])
        p = torch.softmax(s, 0)
        want[r], spread[r] = p[1] - p[2], p[1] + p[2]
    got = cache.attend(0, q, scale=1.0)[:, 0].double().cpu()
    bound = want.abs() * torch.finfo(dtype).eps / 2 + spread * 2.0 ** -20
    err = (got - want[:, None]).abs().amax(-1)
    assert bool((err <= bound).all()), float((err / bound).max())
    assert bool((got == got[:, :1]).all())  # all columns have the same values
    cache.check()


@pytest.mark.parametrize("dtype,size", [(BF16, 1e5), (BF16, 1e18), (F16, 3e3), (F16, 6e4), (F32, 1e5), (F32, 1e18)])
@pytest.mark.parametrize("width", [None, 3000])
@pytest.mark.parametrize("sign", [1, -1])
def test_scores_of_any_size(cuda, dtype, size, width, sign):
    """Finite scores as far from zero as the types allow: the greatest takes
    the whole weight; equal ones share it."""
    dim, n = 64, 70
    cache, _, values = filled_cache([n] * 4, kv_heads=1, dim=dim, page=16, dtype=dtype, width=width)
    q = torch.zeros(4, 2, dim, dtype=dtype, device="cuda")
    q[:, :, 0] = size * torch.tensor([1.0, 0.731], device="cuda")
    for r, at in enumerate((0, 41, 69, None)):
        k = torch.zeros(1, n, dim)
        k[0, :, 0] = sign * size * (0.613 if at is None or sign > 0 else 0.95)
        if at is not None:
            k[0, at, 0] = sign * size * (0.913 if sign > 0 else 0.517)
        _put(cache, 0, 0, r, k.to(dtype).cuda())
    got, lse = cache.attend(0, q, scale=0.77, return_lse=True)
    for r, at in enumerate((0, 41, 69)):
        assert torch.equal(got[r], values[0][r][0, at].expand(2, dim)), r
    v = values[0][3][0].double()
    # equal weights: the sums (relative 2^-16 + n 2^-24 at most) and the output's rounding
    bound = v.mean(0).abs() * torch.finfo(dtype).eps / 2 + v.abs().mean(0) * 2.0 ** -15
    assert bool(((got[3].double() - v.mean(0)).abs() <= bound).all())
    k0 = torch.stack([cache.pool[0, 0, int(cache.page_table[r, (at or 0) // 16]), 0, (at or 0) % 16, 0].double()
                      for r, at in enumerate((0, 41, 69, None))])
    top = 0.77 * q[:, :, 0].double() * k0[:, None]
    top[3] += torch.log(torch.tensor(float(n)))
    assert bool(((lse.double() - top).abs() <= top.abs() * 2.0 ** -21).all())
    cache.check()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("base", [0.0, 300.0, 2000.0, 3e4])
@pytest.mark.parametrize("rise", [1.0, 5.0, 8.0, 13.0, 16.0])
def test_rising_scores_far_from_zero(cuda, dtype, base, rise):
    """Scores of about 60000 base (10^7 to 10^9) that rise by a few powers of
    two from token to token, down to one step of fp32.  With equal values the
    output is that value whatever the weights are: half a step of the type and
    2^-20 for the two sums, which add the same weights."""
    dim, n = 64, 200
    cache, _, _ = filled_cache([n, n], kv_heads=1, dim=dim, page=16, dtype=dtype)
    q = torch.zeros(2, 2, dim, dtype=dtype, device="cuda")
    q[:, 0, 0], q[:, 1, 0] = 6e4, -6e4
    q[:, :, 1] = 1.0
    k = torch.zeros(1, n, dim)
    k[0, :, 0] = base
    k[0, :, 1] = torch.arange(n) * rise
    for r in range(2):
        _put(cache, 0, 0, r, (k if r == 0 else k.flip(1)).to(dtype).cuda())
        _put(cache, 0, 1, r, torch.full((1, n, dim), 3.0, dtype=dtype, device="cuda"))
    got, lse = cache.attend(0, q, scale=0.6931472, return_lse=True)
    assert bool(((got.double() - 3.0).abs() <= 3.0 * (torch.finfo(dtype).eps / 2 + 2.0 ** -20)).all())
    assert bool(torch.isfinite(lse).all())
    cache.check()


def test_scales_growing_scores_and_infinities_in_fp16(cuda):
    """What test_gpu_attend has in bf16 and fp32, with its bounds."""
    attend_tests.test_growing_scores(cuda, F16)
    attend_tests.test_infinities_and_nan(cuda, F16)
    for scale in (-0.3, 0.0, 3.0):
        attend_tests.test_scales(cuda, scale, F16)
    attend_tests.test_one_q_for_all_rows_and_heads(cuda, F16)
    attend_tests.test_many_ragged_rows(cuda, F16)
    for width in (None, 30, 900, 5000):
        attend_tests.test_few_short_rows(cuda, F16, 256, 20, 1, width)
