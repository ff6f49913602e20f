"""What paged generation does with logits that are not finite."""
from __future__ import annotations

import pytest
import torch

from s_salaad_b200 import workloads
from s_salaad_b200.inference import beam_search, generate

F32, BF16 = torch.float32, torch.bfloat16


def _model(vocab, dtype=F32, device="cuda"):
    from s_salaad_b200.efficient import build_model_from_config

    cfg = dict(workloads.LLAMA_60M, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, vocab_size=vocab, max_position_embeddings=128, model_type="llama")
    torch.manual_seed(0)
    return build_model_from_config(cfg, attn_implementation="sdpa").eval().to(device=device, dtype=dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("-inf"), float("inf"), float("nan")])
@pytest.mark.parametrize("step", [0, 2, 4])
def test_one_logit_that_is_not_finite_raises_as_without_pages(cuda, bad, step):
    """At the first, a middle or the last of 5 steps, in one row of two."""
    model, calls = _model(97), []

    def spoil(module, args, output):
        if len(calls) == step:
            output = output.clone()
            output[1, -1, 7] = bad
        calls.append(0)
        return output

    hook = model.lm_head.register_forward_hook(spoil)
    ids = torch.tensor([[1, 2, 3], [4, 5, 6]], device=cuda)
    for paged in (False, True):
        calls.clear()
        with pytest.raises(FloatingPointError, match="Non-finite inference logits"):
            generate(model, ids, 5, paged=paged)
    assert model.config._attn_implementation == "sdpa"
    hook.remove()
    assert torch.equal(generate(model, ids, 5, paged=True)[:, :3], ids)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_model_of_nan_raises_at_a_large_vocabulary(cuda, dtype):
    """Tokens chosen on the way there exist (the embedding is indexed with them)."""
    model = _model(32768, dtype)
    with torch.no_grad():
        model.lm_head.weight.fill_(float("nan"))
    ids = torch.tensor([[1, 2, 3]], device=cuda)
    for call in (lambda: generate(model, ids, 4, paged=True), lambda: beam_search(model, ids, 4, 3)):
        with pytest.raises(FloatingPointError, match="Non-finite inference logits"):
            call()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_beam_search_over_a_masked_vocabulary(cuda):
    """-inf logits are tokens that are never taken, and no error; without
    enough other continuations it is one."""
    model, most = _model(97), 90

    def mask(module, args, output):
        output = output.clone()
        output[..., :most] = float("-inf")
        return output

    model.lm_head.register_forward_hook(mask)
    ids = torch.tensor([[95, 2, 3]], device=cuda)
    seqs, scores = beam_search(model, ids, 4, 7)
    assert bool((seqs[0, :, 3:] >= 90).all()) and bool(torch.isfinite(scores).all())
    most = 95  # 2 tokens: 2 continuations of one token, 4 of two
    with pytest.raises(FloatingPointError, match="Non-finite"):
        beam_search(model, ids, 1, 4)
    seqs, scores = beam_search(model, ids, 2, 4)
    assert sorted(s[3:] for s in seqs[0].tolist()) == [[95, 95], [95, 96], [96, 95], [96, 96]]
