"""Scores of beam search against the same sequences on caches of their own."""
from __future__ import annotations

import pytest
import torch

from s_salaad_b200 import workloads
from s_salaad_b200.inference import beam_search, cache_for_model
from s_salaad_b200.inference.paged import _active, _decode, _on_cache
from s_salaad_b200.ops import token_logprobs


def _model(dtype):
    from s_salaad_b200.efficient import build_model_from_config

    cfg = dict(workloads.LLAMA_60M, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, vocab_size=97, max_position_embeddings=128, model_type="llama")
    torch.manual_seed(0)
    model = build_model_from_config(cfg, attn_implementation="sdpa").eval()
    with torch.no_grad():  # spread the logits: the initialisation leaves them nearly equal
        model.lm_head.weight.mul_(20.0)
    return model.to(device="cuda", dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("prompt,beams,new", [(21, 4, 30), (16, 3, 40), (1, 5, 34)])
def test_forked_pages_hold_what_rows_of_their_own_would(cuda, dtype, prompt, beams, new):
    """The same operators without forks, moves, ends and page copies: every
    hypothesis in a row of its own from the prompt on, its tokens given.

    Bound: both take the same roundings but for the order of sums, which can
    flip the rounding of a logit: one step of the type at the greatest logit
    for each token, independent over the tokens."""
    model = _model(dtype)
    g = torch.Generator().manual_seed(prompt)
    ids = torch.randint(0, 97, (2, prompt), generator=g).to(cuda)
    seqs, scores = beam_search(model, ids, new, beams)
    rows = 2 * beams
    flat = seqs.view(rows, -1)
    with torch.inference_mode():
        cache = cache_for_model(model, rows, prompt + new)
        total, most = torch.zeros(rows, device=cuda), torch.zeros((), device=cuda)
        with _on_cache(model, cache):
            logits = torch.empty(rows, 97, dtype=dtype, device=cuda)
            for j in range(beams):  # the prompts as beam search takes them, two at a time, into rows j and beams + j
                n_new = torch.zeros(rows, dtype=torch.int32, device=cuda)
                n_new[j::beams] = prompt
                cache.advance(n_new)
                _active.cu_tokens = torch.cat([n_new[:1] * 0, torch.cumsum(n_new, 0)]).int()
                if prompt > 1:
                    logits[j::beams] = model(input_ids=ids, use_cache=False, logits_to_keep=1).logits[:, -1]
            if prompt == 1:  # a prompt of one token is appended as row i's
                logits = model(input_ids=flat[:, :1], use_cache=False, logits_to_keep=1).logits[:, -1]
            for t in range(prompt, prompt + new):
                if t > prompt:
                    cache.advance(1)
                    logits = _decode(model, cache, flat[:, t - 1])
                total += token_logprobs(logits, flat[:, t]).logprob
                most = torch.maximum(most, logits.abs().max().float())
        cache.check()
    assert int(cache.refs.max()) == 1  # nothing was shared
    bound = new ** 0.5 * torch.finfo(dtype).eps * float(most)
    assert bound < 0.1 * float(scores.abs().min())
    assert bool(((scores.view(-1) - total).abs() <= bound).all()), (float((scores.view(-1) - total).abs().max()), bound)
