"""Calls of the serving operators that need no GPU: what the Python layer does
around the library, with the library replaced."""
from __future__ import annotations

import weakref

import torch

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
