"""Generation and scoring on the paged key-value cache.

The reference decodes greedily and recomputes the prefix every step
(``ssalaad/inference/generate.py:12-26``).  Here the keys and values of every
sequence live in a :class:`~s_salaad_b200.kvcache.PagedCache`, the model's
attention layers append to it and read it through an attention function
registered with Hugging Face, and the tokens are chosen by
:func:`~s_salaad_b200.ops.token_logprobs`; no step waits for the GPU.  Several
threads may generate with one model at once on one stream: each has its own
cache, and their forwards take turns.  Other forwards of the model meanwhile use
its own attention (they take no turn: a compressed model's layers keep one
workspace each, so calls of one such model otherwise belong to one thread).

* :func:`generate_paged` — greedy decoding (``generate(..., paged=True)``);
* :func:`beam_search` — the ``beams`` most probable continuations found by beam
  search: hypotheses fork and end by page reference, only a shared last page is
  copied;
* :func:`score` — log probability of every token of given sequences.
"""
from __future__ import annotations

import contextlib
import sys
import threading

import torch

from ..kvcache import PagedCache
from ..ops import TokenLogprobs, token_logprobs

_active = threading.local()  # .cache, .cu_tokens, .turn: set while this thread runs a model on a cache
_switch_lock = threading.Lock()
_names: dict = {}  # a model's own attention -> the dispatched one
_switched: dict = {}  # id of a config -> its _Users, while there are any


def _paged_attention(module, query, key, value, attention_mask, scaling=None, **kwargs):
    """Hugging Face attention function: query [rows, heads, T, head_dim], key
    and value [rows, kv_heads, T, head_dim] of the T new tokens of each row."""
    if kwargs.get("sliding_window") is not None:
        raise ValueError("the paged cache has no sliding-window attention")
    if kwargs.get("softcap") is not None or kwargs.get("s_aux") is not None:
        raise ValueError("the paged cache has no attention with capped scores or sinks")
    cache, layer = _active.cache, module.layer_idx
    rows, heads, new, dim = query.shape
    if new == 1:
        cache.append(layer, key[:, :, 0], value[:, :, 0])
        return cache.attend(layer, query[:, :, 0], scale=scaling)[:, None], None
    # a prompt: attention among its own tokens, which start their rows
    k, v = (t.transpose(1, 2).reshape(rows * new, -1, dim) for t in (key, value))
    cache.append(layer, k, v, _active.cu_tokens)
    out = torch.nn.functional.scaled_dot_product_attention(query, key, value, is_causal=True, scale=scaling,
                                                           enable_gqa=heads != key.shape[1])
    return out.transpose(1, 2), None


def _dispatched(own: str) -> str:
    """The name of an attention that is the paged one in threads on a cache and
    the attention ``own`` in all others."""
    from transformers import AttentionInterface, AttentionMaskInterface

    if own in _names:
        return _names[own]
    name = f"slr_paged_{len(_names)}"

    def attention(module, *args, **kwargs):
        if getattr(_active, "cache", None) is not None:
            return _paged_attention(module, *args, **kwargs)
        known = AttentionInterface()
        run = known[own] if own in known else sys.modules[type(module).__module__].eager_attention_forward
        return run(module, *args, **kwargs)

    def mask(*args, **kwargs):
        known = AttentionMaskInterface()
        if getattr(_active, "cache", None) is not None or own not in known:
            return None
        return known[own](*args, **kwargs)

    AttentionInterface.register(name, attention)
    AttentionMaskInterface.register(name, mask)
    _names[own] = name
    return name


class _Users:
    """The threads that have one model on caches."""

    def __init__(self, model):
        self.model, self.own, self.threads = model, model.config._attn_implementation, 0
        # Held over a forward: compressed layers keep one workspace each, which
        # launches of two forwards in turn would share.  (A hook may generate, too.)
        self.turn = threading.RLock()


@contextlib.contextmanager
def _on_cache(model, cache: PagedCache):
    """Within the block the model's attention layers use the cache, in this
    thread: the model's attention is switched to a dispatched one by the first
    thread that enters and back by the last that leaves."""
    kinds = set(getattr(model.config, "layer_types", None) or ()) - {"full_attention", "sliding_attention"}
    if kinds:  # layers that keep a state of their own between tokens (a sliding window is refused where it is met)
        raise ValueError(f"the paged cache holds attention layers only, the model has {sorted(kinds)}")
    key = id(model.config)
    with _switch_lock:
        users = _switched.get(key)
        if users is None:
            users = _Users(model)
            model.set_attn_implementation(_dispatched(users.own))
            _switched[key] = users
        users.threads += 1
    outer = dict(_active.__dict__)
    _active.cache, _active.cu_tokens, _active.turn = cache, None, users.turn
    try:
        yield
    finally:
        _active.__dict__.clear()
        _active.__dict__.update(outer)
        with _switch_lock:
            users.threads -= 1
            if not users.threads:
                del _switched[key]
                users.model.set_attn_implementation(users.own)


def cache_for_model(model, max_seqs: int, max_tokens: int, *, page_size: int = 16, num_pages: int | None = None) -> PagedCache:
    """An empty cache of the model's layers, key heads and dtype for
    ``max_seqs`` sequences of up to ``max_tokens`` tokens; by default with pages
    for all of them at once, plus one each for a copy of a shared page."""
    c = model.config
    dim = getattr(c, "head_dim", None) or c.hidden_size // c.num_attention_heads
    width = -(-max_tokens // page_size)
    p = next(model.parameters())
    if num_pages is None:
        num_pages = max_seqs * (width + 1)
    return PagedCache(num_layers=c.num_hidden_layers, num_pages=num_pages,
                      kv_heads=getattr(c, "num_key_value_heads", None) or c.num_attention_heads, head_dim=dim,
                      page_size=page_size, max_seqs=max_seqs, max_pages=width, dtype=p.dtype, device=p.device)


def _prefill(model, cache: PagedCache, input_ids: torch.Tensor) -> torch.Tensor:
    """Runs prompts [batch, T] into the cache's first rows; logits of their
    last positions [batch, vocab]."""
    batch, new = input_ids.shape
    n_new = torch.zeros(cache.max_seqs, dtype=torch.int32, device=cache.device)
    n_new[:batch] = new
    cache.advance(n_new)
    cu = torch.zeros(cache.max_seqs + 1, dtype=torch.int32, device=cache.device)
    cu[1:] = torch.cumsum(n_new, 0)
    _active.cu_tokens = cu
    with _active.turn:
        return model(input_ids=input_ids, use_cache=False, logits_to_keep=1).logits[:, -1]


def _decode(model, cache: PagedCache, tokens: torch.Tensor) -> torch.Tensor:
    """One step: tokens [rows] are the last of rows that advance() has just
    grown by one; their logits [rows, vocab]."""
    positions = (cache.lens[:tokens.shape[0]] - 1).long()[:, None]
    with _active.turn:
        return model(input_ids=tokens[:, None], position_ids=positions, use_cache=False).logits[:, -1]


@torch.inference_mode()
def generate_paged(model, input_ids: torch.Tensor, max_new_tokens: int, *, page_size: int = 16) -> torch.Tensor:
    """:func:`~s_salaad_b200.inference.generate` on a paged cache (same
    arguments, result and errors; equal greatest logits: the lowest token).
    Every step's logits are looked at, and an error is raised once, after the
    last step: until then the step only notes it on the GPU."""
    from .generate import _check_request

    _check_request(model, input_ids, max_new_tokens)
    if max_new_tokens == 0:
        return input_ids
    batch, prompt = input_ids.shape
    cache = cache_for_model(model, batch, prompt + max_new_tokens, page_size=page_size)
    chosen, finite = [], []
    with _on_cache(model, cache):
        logits = _prefill(model, cache, input_ids)
        for step in range(max_new_tokens):
            if step:
                cache.advance(1)
                logits = _decode(model, cache, chosen[-1])
            finite.append(torch.isfinite(logits).all())
            chosen.append(token_logprobs(logits, top=1, entropy=False).top_ids[:, 0])
    if not torch.stack(finite).all():
        raise FloatingPointError("Non-finite inference logits.")
    cache.check()
    return torch.cat([input_ids, torch.stack(chosen, dim=1)], dim=1)


@torch.inference_mode()
def beam_search(model, input_ids: torch.Tensor, max_new_tokens: int, beams: int, *,
                page_size: int = 16) -> tuple[torch.Tensor, torch.Tensor]:
    """Beam search with ``beams`` (1 to 32) hypotheses per prompt of
    ``input_ids`` [batch, prompt]: (sequences [batch, beams, prompt +
    max_new_tokens], scores [batch, beams]), the score of a sequence being the
    sum of its new tokens' log probabilities, best first.  -inf logits are
    tokens of probability 0; FloatingPointError if the logits of a kept
    hypothesis held a NaN or +inf, or fewer than ``beams`` continuations have a
    probability above 0."""
    from .generate import _check_request

    _check_request(model, input_ids, max_new_tokens)
    if max_new_tokens == 0:
        raise ValueError("beam search needs at least one new token.")
    vocab = model.config.vocab_size
    if not 1 <= beams <= min(32, vocab):
        raise ValueError("beams must be between 1 and min(32, vocabulary).")
    batch, prompt = input_ids.shape
    cache = cache_for_model(model, batch * beams, prompt + max_new_tokens, page_size=page_size)
    dev = cache.device
    with _on_cache(model, cache):
        best = token_logprobs(_prefill(model, cache, input_ids), top=beams, entropy=False)
        scores, tokens = best.top_logprobs, best.top_ids  # [batch, beams]
        sequences = torch.cat([input_ids[:, None].expand(batch, beams, prompt), tokens[..., None]], dim=2)
        first_row = torch.arange(batch, device=dev)[:, None] * beams
        parents = torch.arange(batch, device=dev)[:, None].expand(batch, beams)  # the prompts' rows
        for _ in range(max_new_tokens - 1):
            cache.advance(1, parents=parents.reshape(-1).to(torch.int32))
            best = token_logprobs(_decode(model, cache, tokens.reshape(-1)), top=beams, entropy=False)
            total = scores.reshape(batch, beams, 1) + best.top_logprobs.view(batch, beams, beams)
            scores, at = total.view(batch, -1).topk(beams, dim=1)
            tokens = best.top_ids.view(batch, -1).gather(1, at)
            parent = at // beams
            parents = first_row + parent
            kept = sequences.gather(1, parent[..., None].expand(batch, beams, sequences.shape[2]))
            sequences = torch.cat([kept, tokens[..., None]], dim=2)
    if not torch.isfinite(scores).all():
        raise FloatingPointError("Non-finite inference logits.")
    cache.check()
    return sequences, scores


@torch.inference_mode()
def score(model, input_ids: torch.Tensor, *, top: int = 0, ignore_id: int | None = None) -> TokenLogprobs:
    """Log probability of every token of ``input_ids`` [batch, length] given
    the ones before it, entropy, and the ``top`` likeliest tokens in its place:
    tensors [batch, length - 1] (and [..., top]) for the tokens from the second
    on.  Targets equal to ``ignore_id`` (padding) get log probability 0."""
    if input_ids.ndim != 2 or input_ids.shape[1] < 2:
        raise ValueError("Expected a batch of at least two input token IDs each.")
    logits = model(input_ids=input_ids, use_cache=False).logits
    # the last position predicts nothing: scoring it too keeps the rows packed
    targets = torch.full_like(input_ids, -100, dtype=torch.int64)
    targets[:, :-1] = input_ids[:, 1:]
    if ignore_id is not None:
        targets.masked_fill_(targets == ignore_id, -100)
    r = token_logprobs(logits, targets, top=top)
    return TokenLogprobs(*(None if t is None else t[:, :-1] for t in r))
