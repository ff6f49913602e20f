"""PagedCache.attend where the weights' own arithmetic shows: scores of any
size."""
from __future__ import annotations

import pytest
import torch

from kv_model import filled_cache

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _put(cache, layer, kv, row, tokens):
    """tokens [kv_heads, T, dim] as the keys (kv = 0) or values (1) of a row."""
    page, n = cache.page_size, tokens.shape[1]
    for t in range(0, n, page):
        e = min(n, t + page)
        cache.pool[layer, kv, int(cache.page_table[row, t // page]), :, :e - t] = tokens[:, t:e]


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
