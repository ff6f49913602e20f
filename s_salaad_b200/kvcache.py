"""A paged key-value cache on the GPU and the attention that reads it.

:class:`PagedCache` holds the keys and values of many sequences ("rows") in
pages, with lengths, page table and reference counts on the device: no call
waits for the host, and every call can be captured into a CUDA graph (the
lengths may differ from replay to replay).  One decode step is

* :meth:`PagedCache.advance` — rows fork, end, roll back or grow; shared
  pages are copied before they are written;
* per layer :meth:`PagedCache.append` (the new tokens' keys and values) and
  :meth:`PagedCache.attend` (one query token per row).

Calls on one cache belong on one stream at a time, in order (as for any tensor
that they update), but :meth:`PagedCache.attend` may run on several: it only
reads the cache, and its scratch memory comes from torch's allocator per call.
The reference keeps no cache (``ssalaad/inference/generate.py:12-26``
recomputes the prefix).
"""
from __future__ import annotations

import ctypes

import torch
from torch.autograd import forward_ad

from . import _lib
from .ops import _DeviceGuard, _no_graph, _require_cuda, _stream, _switch, slr_dtype

HEADER = _lib.SLR_KV_HEADER_WORDS


class PagedCache:
    """Keys and values of up to ``max_seqs`` rows in ``num_pages`` pages of
    ``page_size`` tokens (a multiple of 16), for ``num_layers`` layers of
    ``kv_heads`` heads of ``head_dim`` (a multiple of 8 up to 256); a row holds
    up to ``max_pages`` pages.

    ``pool`` [num_layers, 2, num_pages, kv_heads, page_size, head_dim] (keys at
    index 0, values at 1; ``dtype`` fp32, fp16 or bf16) and ``state`` may be
    given, else they are made (the pool uninitialised: slots that no token was
    written to are never read into a result).  In a given pool the block of a
    page must be contiguous, its heads before its slots or after them.

    ``state`` (int32) holds all book-keeping: ``state.clone()`` is a snapshot
    and ``state.copy_(snapshot)`` goes back to it (pages written since then keep
    their new contents).  :attr:`lens`, :attr:`refs`, :attr:`page_table` and
    :attr:`header` are views of it.
    """

    def __init__(self, *, num_layers: int, num_pages: int, kv_heads: int, head_dim: int, page_size: int = 16,
                 max_seqs: int, max_pages: int, dtype: torch.dtype = torch.bfloat16, device="cuda",
                 pool: torch.Tensor | None = None, state: torch.Tensor | None = None):
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError("PagedCache needs a CUDA device (s_salaad_b200 has no CPU path)")
        code = slr_dtype(dtype)
        sizes = dict(num_layers=num_layers, num_pages=num_pages, kv_heads=kv_heads, head_dim=head_dim,
                     page_size=page_size, max_seqs=max_seqs, max_pages=max_pages)
        for name, n in sizes.items():
            if not 1 <= int(n) < 2 ** 31:
                raise ValueError(f"{name} must be in [1, 2^31), got {n}")
        if head_dim % 8 or head_dim > 256:
            raise ValueError(f"head_dim must be a multiple of 8 up to 256, got {head_dim}")
        if page_size % 16 or page_size > 1024:
            raise ValueError(f"page_size must be a multiple of 16 up to 1024, got {page_size}")
        if max_seqs > _lib.SLR_KV_MAX_ROWS:
            raise ValueError(f"max_seqs must be at most {_lib.SLR_KV_MAX_ROWS}, got {max_seqs}")
        if max_pages * page_size >= 2 ** 31:
            raise ValueError("max_pages * page_size must be below 2^31")
        words = HEADER + max_seqs + num_pages + max_seqs * max_pages
        shape = (num_layers, 2, num_pages, kv_heads, page_size, head_dim)
        if pool is not None:
            _require_cuda("pool", pool)
            if pool.dtype != dtype:
                raise TypeError(f"pool must be {dtype}, got {pool.dtype}")
            if tuple(pool.shape) != shape:
                raise ValueError(f"pool must be {shape}, got {tuple(pool.shape)}")
            if head_dim > 1 and pool.stride(5) != 1:
                raise ValueError("pool must have unit stride in the last dimension")
            _no_graph("PagedCache (pool)", pool)
        if state is not None:
            _require_cuda("state", state)
            if state.dtype != torch.int32:
                raise TypeError(f"state must be int32, got {state.dtype}")
            if tuple(state.shape) != (words,) or not state.is_contiguous():
                raise ValueError(f"state must be a contiguous vector of {words} words")
        given = [t.device for t in (pool, state) if t is not None]
        if device.index is None:
            device = given[0] if given else torch.device("cuda", torch.cuda.current_device())
        if any(d != device for d in given):
            raise ValueError(f"pool and state must be on {device}")
        self.device, self.dtype = device, dtype
        self.num_layers, self.num_pages, self.kv_heads, self.head_dim = num_layers, num_pages, kv_heads, head_dim
        self.page_size, self.max_seqs, self.max_pages = page_size, max_seqs, max_pages
        self.pool = pool if pool is not None else torch.empty(shape, dtype=dtype, device=device)
        if state is None:
            state = torch.zeros(words, dtype=torch.int32, device=device)
            state[HEADER + max_seqs + num_pages:] = -1
        self.state = state
        a, b = HEADER + max_seqs, HEADER + max_seqs + num_pages
        self.header, self.lens, self.refs = state[:HEADER], state[HEADER:a], state[a:b]
        self.page_table = state[b:].view(max_seqs, max_pages)
        s = self.struct = _lib.SlrKvCache()
        # a dimension of size 1 has no stride of its own: torch may report any
        st = [self._stride(i) for i in range(6)]
        s.k = self.pool.data_ptr()
        s.v = self.pool.data_ptr() + st[1] * self.pool.element_size()
        s.state = state.data_ptr()
        s.layer_stride, s.page_stride, s.head_stride, s.token_stride = st[0], st[2], st[3], st[4]
        s.num_layers, s.num_pages, s.kv_heads, s.head_dim = num_layers, num_pages, kv_heads, head_dim
        s.page_size, s.max_rows, s.max_pages, s.dtype = page_size, max_seqs, max_pages, code
        self._ref = ctypes.byref(s)
        lib = self._lib = _lib.load()
        self._pages_ws = int(lib.slr_kv_pages_workspace_size(self._ref))
        if not self._pages_ws:
            raise ValueError(f"PagedCache: {_lib.last_error()}")
        # Scratch of the book-keeping: its calls change the state, so they are in order anyway.
        self._ws = torch.empty(self._pages_ws, dtype=torch.uint8, device=device)
        self._attend_ws: dict = {}
        self._index = device.index  # calls compare this number: cheaper than torch.device

    def _stride(self, i: int) -> int:
        """Stride of pool dimension i; of one of size 1, the packed one."""
        p = self.pool
        if p.shape[i] > 1 or i in (1, 5):
            return p.stride(i)
        if i == 3:  # one head: its slots are the whole block
            return self.page_size * self.head_dim
        if i in (0, 2):
            block = self.kv_heads * self.page_size * self.head_dim
            return max(p.stride(i), block) if i == 0 else block
        return p.stride(i)

    # ------------------------------------------------------ book-keeping --
    def _vector(self, name: str, t: torch.Tensor, n: int) -> torch.Tensor:
        """int32 [n] on the cache's device, contiguous."""
        if t.dtype is not torch.int32:
            raise TypeError(f"{name} must be int32, got {t.dtype}")
        if t.get_device() != self._index or t.dim() != 1 or t.shape[0] != n:
            raise ValueError(f"{name} must be [{n}] on {self.device}")
        return t if t.is_contiguous() else t.contiguous()

    def advance(self, n_new: int | torch.Tensor = 1, parents: torch.Tensor | None = None) -> None:
        """The book-keeping of one step, for all rows at once.

        With ``parents`` (int32 [max_seqs]) row i first becomes row
        ``parents[i]`` as it was before the call (negative: empty): the same
        parent several times forks it (its pages are shared), rows left out
        end and their pages are free.  Then row i grows by ``n_new[i]`` tokens
        (int32 [max_seqs]; negative: drops that many from its end), or with one
        number every row that holds tokens does.  New pages are the lowest free
        ones in row order; a row about to write into a shared last page gets a
        copy of it first.

        Growth is all or nothing: if pages are missing, or a row would pass
        ``max_pages``, no row grows and :meth:`check` raises.
        """
        n_all, n_ptr = 0, None
        if isinstance(n_new, torch.Tensor):
            n_new = self._vector("n_new", n_new, self.max_seqs)
            n_ptr = n_new.data_ptr()
        else:
            n_all = int(n_new)
            if not -2 ** 31 < n_all < 2 ** 31:
                raise ValueError(f"n_new out of range: {n_all}")
        if parents is not None:
            parents = self._vector("parents", parents, self.max_seqs)
        back = _switch(self._index)
        try:
            rc = self._lib.slr_kv_advance(self._ref, None if parents is None else parents.data_ptr(), n_ptr, n_all,
                                          self._ws.data_ptr(), self._pages_ws, _stream(self.device))
        finally:
            if back >= 0:
                torch.cuda.set_device(back)
        if rc:
            _lib.check(rc, "kv_advance")

    def compact(self) -> None:
        """Moves the live pages to the lowest numbers (order kept among the
        moved ones) and rewrites the table; the pages from ``header[3]`` on are
        free then."""
        back = _switch(self._index)
        try:
            rc = self._lib.slr_kv_compact(self._ref, self._ws.data_ptr(), self._pages_ws, _stream(self.device))
        finally:
            if back >= 0:
                torch.cuda.set_device(back)
        if rc:
            _lib.check(rc, "kv_compact")

    def resize(self, num_pages: int) -> None:
        """Moves the cache to a new pool of ``num_pages`` pages (more, or after
        rows have left fewer: the live pages are compacted first).  Waits for
        the GPU; raises ValueError if the live pages do not fit.  A pool or
        state given at construction, and graphs captured with this cache, are
        not used afterwards."""
        if not 1 <= int(num_pages) < 2 ** 31:
            raise ValueError(f"num_pages must be in [1, 2^31), got {num_pages}")
        self.compact()
        live = int(self.header[3])
        if live > num_pages:
            raise ValueError(f"{live} pages are in use, more than {num_pages}")
        new = PagedCache(num_layers=self.num_layers, num_pages=num_pages, kv_heads=self.kv_heads,
                         head_dim=self.head_dim, page_size=self.page_size, max_seqs=self.max_seqs,
                         max_pages=self.max_pages, dtype=self.dtype, device=self.device)
        new.pool[:, :, :live] = self.pool[:, :, :live]
        new.header.copy_(self.header)
        new.lens.copy_(self.lens)
        new.refs[:live] = self.refs[:live]
        new.page_table.copy_(self.page_table)
        self.__dict__.update(new.__dict__)

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Copies pages ``src[i]`` to ``dst[i]`` (int32) of every layer; the
        state is not touched.  Pairs that clash (a dst that is another pair's
        src or dst) or are out of range are left out and reported by
        :meth:`check`."""
        src = self._vector("src", src, src.shape[0] if src.dim() == 1 else -1)
        dst = self._vector("dst", dst, src.shape[0])
        with _DeviceGuard(self.device):
            rc = self._lib.slr_kv_copy_pages(self._ref, src.data_ptr(), dst.data_ptr(), src.shape[0],
                                             _stream(self.device))
        _lib.check(rc, "kv_copy_pages")

    def check(self) -> None:
        """Waits for the GPU and raises if the last :meth:`advance` could not
        grow (RuntimeError) or if a kernel met an index out of range since the
        last check on this device (ValueError)."""
        with _DeviceGuard(self.device):
            status = ctypes.c_int(0)
            _lib.check(self._lib.slr_device_status(ctypes.byref(status)), "device_status")
        if status.value == _lib.SLR_ERR_BAD_INDEX:
            raise ValueError("a page, length, row or token index was out of range")
        if status.value:
            raise RuntimeError(f"device status: {self._lib.slr_status_string(status.value).decode()}")
        short, over = self.header[:2].tolist()
        if short or over:
            raise RuntimeError(f"the cache could not grow: {short} pages missing, {over} rows past "
                               f"{self.max_pages} pages")

    # ---------------------------------------------------------- per layer --
    def _tokens(self, name: str, t: torch.Tensor) -> tuple:
        """(shape, strides) of [tokens, heads, head_dim] on the cache's device."""
        if t.dtype is not self.dtype:
            raise TypeError(f"{name} must be {self.dtype}, got {t.dtype}")
        if t.get_device() != self._index:
            raise ValueError(f"{name} must be on {self.device}, got {t.device}")
        shape, stride = t.shape, t.stride()
        if len(shape) != 3 or shape[2] != self.head_dim:
            raise ValueError(f"{name} must be [tokens, heads, {self.head_dim}], got {tuple(shape)}")
        if stride[2] != 1:
            raise ValueError(f"{name} must have unit stride in the last dimension")
        if t.requires_grad or forward_ad._current_level >= 0:  # (calls of a few microseconds)
            _no_graph(f"PagedCache ({name})", t)
        return shape, stride

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, cu_tokens: torch.Tensor | None = None) -> None:
        """Writes new tokens' keys and values [tokens, kv_heads, head_dim]
        into ``layer``, after :meth:`advance` made room (and gave the row its
        own copy of a shared last page): a row's tokens go to its last positions.  ``cu_tokens`` (int32 [max_seqs + 1]): row b's
        tokens are ``[cu[b], cu[b + 1])``, further ones are padding.  Without
        it token i is row i's, and empty rows are skipped."""
        shape, ks = self._tokens("k", k)
        v_shape, vs = self._tokens("v", v)
        if shape != v_shape or shape[1] != self.kv_heads:
            raise ValueError(f"k and v must be [tokens, {self.kv_heads}, {self.head_dim}]")
        cu = None
        if cu_tokens is not None:
            cu_tokens = self._vector("cu_tokens", cu_tokens, self.max_seqs + 1)
            cu = cu_tokens.data_ptr()
        back = _switch(self._index)
        try:
            rc = self._lib.slr_kv_append(self._ref, layer, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
                                         shape[0], cu, _stream(self.device))
        finally:
            if back >= 0:
                torch.cuda.set_device(back)
        if rc:
            _lib.check(rc, "kv_append")

    def attend(self, layer: int, q: torch.Tensor, *, scale: float | None = None, out: torch.Tensor | None = None,
               return_lse: bool = False):
        """``softmax(scale * q · Kᵀ) · V`` of one query token per row, q
        [rows, heads, head_dim] (rows <= max_seqs, heads a multiple of
        kv_heads, consecutive heads share a key head), over all tokens of each
        row; ``scale`` defaults to ``head_dim ** -0.5``.  Empty rows give zeros.
        ``out`` may be ``q`` itself, not a tensor that overlaps itself.
        Returns ``out``, or ``(out, lse)`` with the float32 log-sum-exp
        [rows, heads] (-inf for empty rows)."""
        shape, qs = self._tokens("q", q)
        rows, heads, dim = shape
        if rows > self.max_seqs or heads == 0 or heads % self.kv_heads:
            raise ValueError(f"q must have at most {self.max_seqs} rows and a multiple of {self.kv_heads} heads, "
                             f"got {tuple(shape)}")
        if out is None:
            out = torch.empty(rows, heads, dim, dtype=self.dtype, device=self.device)
            os = (heads * dim, dim)
        else:
            out_shape, os = self._tokens("out", out)
            if out_shape != shape:
                raise ValueError(f"out must be {tuple(shape)}, got {tuple(out_shape)}")
        lse = torch.empty(rows, heads, dtype=torch.float32, device=self.device) if return_lse else None
        back = _switch(self._index)
        try:
            need = self._attend_ws.get((rows, heads))
            if need is None:
                need = int(self._lib.slr_kv_attend_workspace_size(self._ref, rows, heads))
                if len(self._attend_ws) > 256:
                    self._attend_ws.clear()
                self._attend_ws[(rows, heads)] = need
            # held until the launch: a block given back before could go to another thread of this stream
            ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
            rc = self._lib.slr_kv_attend(
                self._ref, layer, q.data_ptr(), qs[0], qs[1], out.data_ptr(), os[0], os[1],
                lse.data_ptr() if return_lse else None, rows, heads, dim ** -0.5 if scale is None else scale,
                None if ws is None else ws.data_ptr(), need, _stream(self.device))
        finally:
            if back >= 0:
                torch.cuda.set_device(back)
        if rc:
            _lib.check(rc, "kv_attend")
        return (out, lse) if return_lse else out
