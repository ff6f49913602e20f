"""Refusals of the serving operators that need no GPU: descriptors that the C
ABI rejects before anything is launched, and the Python checks."""
from __future__ import annotations

import ctypes

import pytest
import torch

from kv_model import Book
from s_salaad_b200 import _lib
from s_salaad_b200.kvcache import PagedCache
from s_salaad_b200.ops import token_logprobs


def _cache(**over):
    s = _lib.SlrKvCache()
    s.k, s.v, s.state = 1 << 20, 1 << 21, 1 << 22  # never dereferenced: every call here is refused on the host
    s.num_layers, s.num_pages, s.kv_heads, s.head_dim, s.page_size = 2, 10, 2, 64, 16
    s.max_rows, s.max_pages, s.dtype = 4, 3, _lib.SLR_BF16
    s.token_stride, s.head_stride, s.page_stride = 64, 16 * 64, 2 * 16 * 64
    s.layer_stride = 2 * 10 * s.page_stride
    for k, v in over.items():
        setattr(s, k, v)
    return s


def _advance(s, ws=256, size=1 << 20):
    return _lib.load().slr_kv_advance(ctypes.byref(s), None, None, 1, ws, size, None)


@pytest.mark.parametrize("over", [dict(head_dim=0), dict(head_dim=12), dict(head_dim=264), dict(page_size=8),
                                  dict(page_size=24), dict(page_size=2048), dict(num_layers=0), dict(num_pages=0),
                                  dict(kv_heads=0), dict(max_rows=0), dict(max_rows=2049), dict(max_pages=0),
                                  dict(max_pages=1 << 27), dict(k=None), dict(v=None), dict(state=None), dict(k=8),
                                  dict(layer_stride=4), dict(head_stride=2 * 16 * 64), dict(page_stride=64),
                                  dict(token_stride=-64)])
def test_bad_descriptors(over):
    s = _cache(**over)
    assert _advance(s) == _lib.SLR_ERR_INVALID_ARGUMENT
    assert "kv cache" in _lib.last_error()


def test_bad_arguments():
    lib = _lib.load()
    s = _cache()
    ref = ctypes.byref(s)
    need = lib.slr_kv_pages_workspace_size(ref)
    assert need > 0 and lib.slr_kv_pages_workspace_size(ctypes.byref(_cache(head_dim=7))) == 0
    assert lib.slr_kv_advance(None, None, None, 1, 256, need, None) == _lib.SLR_ERR_INVALID_ARGUMENT
    assert _advance(_cache(dtype=9)) == _lib.SLR_ERR_UNSUPPORTED_DTYPE
    for ws, size in ((None, need), (256, need - 1), (8, need)):
        assert _advance(s, ws, size) == _lib.SLR_ERR_WORKSPACE
        assert lib.slr_kv_compact(ref, ws, size, None) == _lib.SLR_ERR_WORKSPACE
    bad = _lib.SLR_ERR_INVALID_ARGUMENT
    assert lib.slr_kv_copy_pages(ref, None, None, 1, None) == bad
    assert lib.slr_kv_copy_pages(ref, 256, 256, -1, None) == bad
    assert lib.slr_kv_copy_pages(ref, None, None, 0, None) == _lib.SLR_OK
    for layer, tokens in ((-1, 1), (2, 1), (0, -1), (0, 5)):
        assert lib.slr_kv_append(ref, layer, 256, 128, 64, 256, 128, 64, tokens, None, None) == bad
    assert lib.slr_kv_append(ref, 0, None, 128, 64, 256, 128, 64, 1, None, None) == bad
    assert lib.slr_kv_append(ref, 0, 256, -1, 64, 256, 128, 64, 1, None, None) == bad
    assert lib.slr_kv_append(ref, 0, None, 128, 64, None, 128, 64, 0, None, None) == _lib.SLR_OK
    for layer, rows, heads, scale in ((2, 1, 4, 1.0), (0, 5, 4, 1.0), (0, -1, 4, 1.0), (0, 1, 3, 1.0), (0, 1, 0, 1.0),
                                      (0, 1, 8192, 1.0), (0, 1, 4, float("inf"))):
        assert lib.slr_kv_attend(ref, layer, 256, 1, 1, 256, 1, 1, None, rows, heads, scale, 256, need, None) == bad
    assert lib.slr_kv_attend(ref, 0, None, 1, 1, 256, 1, 1, None, 1, 4, 1.0, 256, need, None) == bad
    assert lib.slr_kv_attend(ref, 0, 256, 1, 1, 256, 1, 1, None, 1, 4, 1.0, 8, need, None) == _lib.SLR_ERR_WORKSPACE
    huge = ctypes.byref(_cache(max_rows=2048, max_pages=1 << 22))
    assert lib.slr_kv_attend(huge, 0, 256, 1, 1, 256, 1, 1, None, 1, 4, 1.0, 256, need,
                             None) == _lib.SLR_ERR_UNSUPPORTED


@pytest.mark.parametrize("rows,heads,row,head", [(2, 4, 0, 64), (1, 4, 256, 0), (2, 4, 256, 63), (2, 4, 255, 64),
                                                 (2, 2, 63, 1), (2, 4, 64, 127), (3, 4, 64, 191), (2, 4, 1 << 62, 1 << 62)])
def test_output_that_overlaps_itself(rows, heads, row, head):
    lib, s = _lib.load(), _cache()
    rc = lib.slr_kv_attend(ctypes.byref(s), 0, 256, 1, 1, 256, row, head, None, rows, heads, 1.0, 256, 1 << 20, None)
    assert rc == _lib.SLR_ERR_INVALID_ARGUMENT and "overlaps itself" in _lib.last_error()


def test_bad_logprob_arguments():
    lib = _lib.load()

    def call(stride=0, rows=2, vocab=50, dtype=_lib.SLR_F32, targets=256, lp=256, top=3, ids=256, val=256, x=256):
        return lib.slr_token_logprobs(x, stride, rows, vocab, dtype, targets, lp, None, top, ids, val, None)

    assert call(dtype=5) == _lib.SLR_ERR_UNSUPPORTED_DTYPE
    for over in (dict(rows=-1), dict(vocab=0), dict(vocab=1 << 31), dict(rows=(1 << 27) + 1), dict(stride=-1),
                 dict(top=-1), dict(top=33), dict(vocab=2), dict(targets=None), dict(lp=None), dict(ids=None),
                 dict(val=None), dict(x=None)):
        assert call(**over) == _lib.SLR_ERR_INVALID_ARGUMENT, over
    assert call(rows=0, x=None) == _lib.SLR_OK


def test_no_cpu_path():
    kw = dict(num_layers=1, num_pages=4, kv_heads=1, head_dim=64, max_seqs=1, max_pages=1)
    with pytest.raises(ValueError, match="CUDA"):
        PagedCache(**kw, device="cpu")
    for over in (dict(head_dim=60), dict(page_size=8), dict(max_seqs=0), dict(max_seqs=5000), dict(num_pages=2 ** 31)):
        with pytest.raises(ValueError):
            PagedCache(**{**kw, **over})
    with pytest.raises(TypeError):
        PagedCache(**kw, dtype=torch.float64)
    with pytest.raises(ValueError, match="CUDA tensor"):
        PagedCache(**kw, pool=torch.zeros(1, 2, 4, 1, 16, 64, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="CUDA tensor"):
        token_logprobs(torch.zeros(2, 5))


def test_the_model_of_the_rules():
    """The row-by-row model that the GPU tests compare with, on a case by hand."""
    b = Book(3, 8, 3, 16)
    assert b.advance([20, 3, 0]) == [] and b.lens == [20, 3, 0]
    assert b.table == [[0, 1, -1], [2, -1, -1], [-1, -1, -1]] and b.header == [0, 0, 0, 3]
    assert b.advance(0, [0, 0, 0]) == [] and b.refs()[:3] == [3, 3, 0]
    assert b.advance(1) == [(1, 2), (1, 3)]
    assert b.table == [[0, 1, -1], [0, 2, -1], [0, 3, -1]] and b.lens == [21] * 3
    assert b.advance(0, [-1, -1, 2]) == [] and b.header == [0, 0, 0, 2]
    assert b.compact() == [(3, 1)] and b.table[2] == [0, 1, -1]
    assert b.advance([0, 0, 100]) == [] and b.header == [0, 1, 0, 2] and b.lens[2] == 21
