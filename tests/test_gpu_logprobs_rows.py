"""ops.token_logprobs on rows without numbers and on rows far from zero."""
from __future__ import annotations

import pytest
import torch

from s_salaad_b200.ops import token_logprobs

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF, NAN = float("inf"), float("nan")


def _rows_of_nan(vocab, dtype):
    """One row of each kind: NaN alone; NaN and -inf; NaN with fewer finite
    logits than are asked for; NaN before, and behind, a normal half; one
    finite logit at either end; NaN at the places of whole 16-byte vectors."""
    g = torch.Generator(device="cpu").manual_seed(vocab)
    x = torch.full((8, vocab), NAN)
    x[1, ::2] = -INF
    at = torch.randperm(vocab, generator=g)[:5]
    x[2, at] = torch.randn(5, generator=g)
    half = torch.randn(vocab, generator=g) * 2.5
    x[3, vocab // 2:] = half[vocab // 2:]
    x[4, :vocab // 2] = half[:vocab // 2]
    x[5, 0] = -3.0
    x[6, -1] = -3.0
    x[7, torch.arange(vocab) // 8 % 3 == 0] = 1.0
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("vocab", [97, 32000, 32768, 65536, 151936])
@pytest.mark.parametrize("copies", [1, 100])
@pytest.mark.parametrize("top", [1, 20, 32])
def test_best_tokens_of_rows_with_nan(cuda, dtype, vocab, copies, top):
    """NaN ranks with -inf and equal values by lower index, in few rows (several
    blocks each) and in many; the ids are tokens."""
    kinds = _rows_of_nan(vocab, dtype)
    key = torch.nan_to_num(kinds.double(), nan=-INF, neginf=-INF)
    want = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :top]
    r = token_logprobs(kinds.cuda().repeat(copies, 1), top=top)
    assert torch.equal(r.top_ids.cpu(), want.repeat(copies, 1))
    assert bool(torch.isnan(r.entropy).all()) and bool(torch.isnan(r.top_logprobs).all())


@pytest.mark.parametrize("dtype,shift", [(F32, 3e3), (F32, 1e6), (F32, -1e6), (F16, 3e4)])
@pytest.mark.parametrize("rows,vocab", [(5, 1001), (700, 1001), (3, 32000)])
def test_logits_far_from_zero(cuda, dtype, shift, rows, vocab):
    """A number added to all logits of a row changes nothing: the error goes by
    the distance from the greatest logit, not by the logits' own size.

    Bounds: the sums' relative error (2^-20 + vocab 2^-24) and the rounding of
    x - max, of its product with log2 e and of the last subtraction (2^-22 of
    |x - max| + log vocab)."""
    g = torch.Generator(device="cpu").manual_seed(int(abs(shift)) + rows)
    x = (torch.randn(rows, vocab, generator=g) * 2.5 + shift).to(dtype).cuda()
    t = torch.randint(0, vocab, (rows,), generator=g).cuda()
    r = token_logprobs(x, t, top=5)
    d = x.double()
    d = d - d.amax(-1, keepdim=True)
    logp = d - torch.logsumexp(d, -1, keepdim=True)
    rel = 2.0 ** -20 + vocab * 2.0 ** -24
    tol = rel + 2.0 ** -22 * (d.abs() + torch.log(torch.tensor(float(vocab))))
    err = (r.logprob.double()[:, None] - logp.gather(1, t[:, None])).abs()
    assert bool((err <= tol.gather(1, t[:, None])).all()), float(err.max())
    err = (r.top_logprobs.double() - logp.gather(1, r.top_ids)).abs()
    assert bool((err <= tol.gather(1, r.top_ids)).all()), float(err.max())
    ent, mean = -(logp.exp() * logp).sum(-1), (logp.exp() * d.abs()).sum(-1)
    assert bool(((r.entropy.double() - ent).abs() <= rel * (2 * mean + 1) + ent * 2.0 ** -22).all())
