"""Calls of the serving operators that need no GPU: what the Python layer does
around the library, with the library replaced."""
from __future__ import annotations

import weakref

import pytest
import torch
from torch.autograd import forward_ad

from s_salaad_b200 import _lib, kvcache
from s_salaad_b200.kvcache import PagedCache


def _host_cache(lib, **over):
    """A cache whose tensors are on the host and whose library is `lib`."""
    c = PagedCache.__new__(PagedCache)
    c.device, c.dtype, c._index = torch.device("cpu"), torch.bfloat16, -1
    c.num_layers, c.num_pages, c.kv_heads, c.head_dim = 2, 8, 2, 64
    c.page_size, c.max_seqs, c.max_pages = 16, 4, 2
    c._attend_ws, c._ref, c._lib = {}, None, lib
    for k, v in over.items():
        setattr(c, k, v)
    return c


def test_the_workspace_lives_until_the_call_returns(monkeypatch):
    """The attention's scratch memory is not given back to the allocator, where
    another thread could take it, before its kernel has been launched."""
    made, seen = [], []
    empty = torch.empty

    def recording(*a, **kw):
        t = empty(*a, **kw)
        made.append((t.data_ptr(), weakref.ref(t)))
        return t

    class Lib:
        @staticmethod
        def slr_kv_attend_workspace_size(ref, rows, heads):
            return 4096

        @staticmethod
        def slr_kv_attend(*args):
            ws, size = args[12], args[13]
            seen.append((size, any(p == ws and r() is not None for p, r in made)))
            return _lib.SLR_OK

    monkeypatch.setattr(kvcache, "_switch", lambda index: -1)
    monkeypatch.setattr(kvcache, "_stream", lambda device: 0)
    monkeypatch.setattr(torch, "empty", recording)
    _host_cache(Lib).attend(0, torch.zeros(3, 4, 64, dtype=torch.bfloat16))
    assert seen == [(4096, True)]


class _Accepts:
    """A library that takes every call."""

    def __getattr__(self, name):
        return lambda *args: 0


def test_gradients_and_tangents_are_refused(monkeypatch):
    """An input that a derivative would be expected of, in either mode, is an
    error and not a result without one."""
    monkeypatch.setattr(kvcache, "_switch", lambda index: -1)
    monkeypatch.setattr(kvcache, "_stream", lambda device: 0)
    cache = _host_cache(_Accepts())
    q, kv = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        dq, dkv = forward_ad.make_dual(q, q), forward_ad.make_dual(kv, kv)
        for call in (lambda: cache.attend(0, dq), lambda: cache.attend(0, q, out=dq),
                     lambda: cache.append(0, dkv, kv), lambda: cache.append(0, kv, dkv),
                     lambda: cache.append(0, dkv[:, :, :], kv)):
            with pytest.raises(ValueError, match="no forward-mode derivative"):
                call()
        cache.attend(0, forward_ad.unpack_dual(dq).primal)
        cache.attend(0, q)
        cache.append(0, kv, kv)
        with torch.inference_mode():  # no derivatives here
            cache.attend(0, dq)
    for call in (lambda: cache.attend(0, q.clone().requires_grad_()), lambda: cache.append(0, kv, kv.clone().requires_grad_())):
        with pytest.raises(ValueError, match="no backward"):
            call()
        with torch.no_grad():
            call()


@pytest.mark.gpu
def test_tangents_and_a_pool_with_gradients_are_refused(cuda):
    from s_salaad_b200.ops import token_logprobs

    x = torch.randn(3, 50, device=cuda)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="no forward-mode derivative"):
            token_logprobs(forward_ad.make_dual(x, x), top=2)
        token_logprobs(x, top=2)
    pool = torch.zeros(1, 2, 4, 1, 16, 64, dtype=torch.bfloat16, device=cuda)
    kw = dict(num_layers=1, num_pages=4, kv_heads=1, head_dim=64, max_seqs=1, max_pages=1)
    with pytest.raises(ValueError, match="no backward"):
        PagedCache(**kw, pool=pool.clone().requires_grad_())
    PagedCache(**kw, pool=pool)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_score_takes_the_ids_that_the_model_takes(monkeypatch, dtype):
    """Embeddings index with int32 too; the targets are the next ids either way."""
    from types import SimpleNamespace

    from s_salaad_b200.inference import paged

    seen = {}

    def scores(logits, targets, *, top):
        seen["targets"] = targets
        return paged.TokenLogprobs(torch.zeros(2, 4), torch.zeros(2, 4), None, None)

    monkeypatch.setattr(paged, "token_logprobs", scores)
    ids = torch.tensor([[1, 2, 3, 0], [4, 5, 6, 7]], dtype=dtype)
    r = paged.score(lambda **kw: SimpleNamespace(logits=torch.zeros(2, 4, 9)), ids, ignore_id=0)
    assert r.logprob.shape == (2, 3)
    assert seen["targets"].dtype == torch.int64
    assert seen["targets"].tolist() == [[2, 3, -100, -100], [5, 6, 7, -100]]


def test_cache_for_model_takes_the_number_of_pages_as_given(monkeypatch):
    """0 pages are refused (by PagedCache), not replaced by the default."""
    from types import SimpleNamespace

    from s_salaad_b200.inference import paged

    made = []
    monkeypatch.setattr(paged, "PagedCache", lambda **kw: made.append(kw["num_pages"]))
    model = SimpleNamespace(config=SimpleNamespace(hidden_size=64, num_attention_heads=4, num_hidden_layers=1),
                            parameters=lambda: iter([torch.zeros(1)]))
    for pages in (None, 0, 7):
        paged.cache_for_model(model, 3, 40, num_pages=pages)
    assert made == [3 * (3 + 1), 0, 7]
