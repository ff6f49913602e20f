"""Generation, beam search and scoring on the paged cache (s_salaad_b200.inference).

The paged attention and the model's own round differently, so tokens are not
compared one by one: every chosen token is checked against a full forward of
the sequence it belongs to, with the 16-bit tolerance of the cached loop's
test (2e-2 of the logits' RMS + 5 % of their range) or, in fp32, 1e-4 of it.
"""
from __future__ import annotations

import pytest
import torch

from s_salaad_b200 import workloads
from s_salaad_b200.inference import beam_search, cache_for_model, generate, generate_paged, score

F32, BF16 = torch.float32, torch.bfloat16


def _tiny(dtype=F32, device="cpu", model_type="llama", kv_heads=2):
    from s_salaad_b200.efficient import build_model_from_config

    cfg = dict(workloads.LLAMA_60M, hidden_size=64, intermediate_size=128, num_hidden_layers=2,
               num_attention_heads=4, num_key_value_heads=kv_heads, vocab_size=97, max_position_embeddings=128,
               model_type=model_type)
    if model_type == "qwen3":
        cfg["head_dim"] = 32
    torch.manual_seed(0)
    model = build_model_from_config(cfg, attn_implementation="sdpa").eval()
    with torch.no_grad():  # spread the logits: the initialisation leaves them nearly equal
        model.lm_head.weight.mul_(20.0)
    return model.to(device=device, dtype=dtype)


def test_cpu_model_is_refused():
    model = _tiny()
    ids = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="CUDA device"):
        generate(model, ids, 2, paged=True)
    assert model.config._attn_implementation == "sdpa"


def test_request_errors():
    model = _tiny()
    ids = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="nonempty batch"):
        generate_paged(model, ids[0], 2)
    with pytest.raises(ValueError, match="context length"):
        generate_paged(model, ids, 200)
    assert torch.equal(generate_paged(model, ids, 0), ids)
    with pytest.raises(ValueError, match="at least one new token"):
        beam_search(model, ids, 0, 2)
    with pytest.raises(ValueError, match="beams must be"):
        beam_search(model, ids, 2, 33)
    with pytest.raises(ValueError, match="at least two"):
        score(model, ids[:, :1])


def test_other_attention_is_refused():
    from s_salaad_b200.inference.paged import _on_cache, _paged_attention

    for over in (dict(sliding_window=8), dict(softcap=30.0), dict(s_aux=torch.zeros(4))):
        with pytest.raises(ValueError, match="the paged cache has no"):
            _paged_attention(None, None, None, None, None, **over)
    model = _tiny(model_type="qwen3")
    model.config.layer_types = ["full_attention", "linear_attention"]
    with pytest.raises(ValueError, match="linear_attention"):
        with _on_cache(model, None):
            pass
    assert model.config._attn_implementation == "sdpa"


def _tolerance(logits, dtype):
    rms, most = float(logits.pow(2).mean().sqrt()), float(logits.abs().max())
    return 1e-4 * most if dtype == F32 else 2e-2 * rms + 0.05 * most


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("model_type,kv_heads", [("llama", 4), ("llama", 1), ("qwen3", 2)])
@pytest.mark.parametrize("prompt", [1, 5, 40])
def test_greedy_tokens_are_the_full_forwards(cuda, dtype, model_type, kv_heads, prompt):
    model = _tiny(dtype, cuda, model_type, kv_heads)
    g = torch.Generator().manual_seed(prompt)
    ids = torch.randint(0, 97, (3, prompt), generator=g).to(cuda)
    out = generate(model, ids, 40, paged=True)
    assert out.shape == (3, prompt + 40) and torch.equal(out[:, :prompt], ids)
    assert model.config._attn_implementation == "sdpa"
    with torch.inference_mode():
        logits = model(input_ids=out[:, :-1], use_cache=False).logits.float()[:, prompt - 1:]
    picked = logits.gather(2, out[:, prompt:, None])[..., 0]
    assert bool((logits.amax(-1) - picked <= _tolerance(logits, dtype)).all())


@pytest.mark.gpu
def test_compressed_model_in_fp32_agrees_with_the_cached_loop(cuda, tmp_path):
    """Where the best logit leads by more than the tolerance, both loops choose it."""
    from s_salaad_b200.efficient import build_efficient_model

    path = tmp_path / "cfg2.pt"
    workloads.compressed_bundle(path, n_layers=2)
    model, config, _ = build_efficient_model(path, device=cuda, dtype=F32)
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, config["vocab_size"], (2, 16), generator=g).to(cuda)
    out = generate(model, ids, 24, paged=True)
    with torch.inference_mode():
        logits = model(input_ids=out[:, :-1], use_cache=False).logits[:, 15:]
    top = logits.topk(2, dim=-1)
    clear = top.values[..., 0] - top.values[..., 1] > _tolerance(logits, F32)
    assert bool(clear.any()) and torch.equal(out[:, 16:][clear], top.indices[..., 0][clear])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_search(cuda, dtype):
    model = _tiny(dtype, cuda)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 97, (2, 21), generator=g).to(cuda)
    seqs, scores = beam_search(model, ids, 30, 4)
    assert seqs.shape == (2, 4, 51) and scores.shape == (2, 4)
    assert torch.equal(seqs[:, :, :21], ids[:, None].expand(2, 4, 21))
    assert bool((scores[:, :-1] >= scores[:, 1:]).all())
    flat = seqs.view(8, 51)
    assert len({tuple(s.tolist()) for s in flat}) == 8  # hypotheses differ
    with torch.inference_mode():
        logits = model(input_ids=flat[:, :-1], use_cache=False).logits.double()[:, 20:]
    lp = torch.log_softmax(logits, -1).gather(2, flat[:, 21:, None]).sum((1, 2)).view(2, 4)
    # 30 log probabilities, each off by at most twice the logits' tolerance
    assert bool(((scores - lp).abs() <= 60 * _tolerance(logits, dtype)).all())
    one, s1 = beam_search(model, ids, 30, 1)
    greedy = generate_paged(model, ids, 30)
    assert torch.equal(one[:, 0], greedy)
    if dtype == F32:  # the best of four is not worse than greedy by more than rounding
        assert bool((scores[:, 0] >= s1[:, 0] - 60 * _tolerance(logits, dtype)).all())


@pytest.mark.gpu
def test_beam_search_against_a_plain_one(cuda):
    """fp32, small enough to enumerate: the same hypotheses as recomputing every prefix."""
    model = _tiny(F32, cuda)
    ids = torch.tensor([[3, 14, 15, 92, 6]], device=cuda)
    seqs, scores = beam_search(model, ids, 12, 3)
    hyps = [(0.0, ids[0])]
    with torch.inference_mode():
        for _ in range(12):
            grown = []
            for s, h in hyps:
                lp = torch.log_softmax(model(input_ids=h[None], use_cache=False).logits[0, -1].double(), -1)
                top = lp.topk(3)
                grown += [(s + float(v), torch.cat([h, i[None]])) for v, i in zip(top.values, top.indices)]
            hyps = sorted(grown, key=lambda t: -t[0])[:3]
    for j, (s, h) in enumerate(hyps):
        assert abs(s - float(scores[0, j])) < 1e-2
        assert torch.equal(seqs[0, j], h)


@pytest.mark.gpu
def test_score(cuda):
    model = _tiny(F32, cuda)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(1, 97, (3, 17), generator=g).to(cuda)
    ids[1, 12:] = 0
    r = score(model, ids, top=5, ignore_id=0)
    with torch.inference_mode():
        logp = torch.log_softmax(model(input_ids=ids, use_cache=False).logits.double(), -1)[:, :-1]
    want = logp.gather(2, ids[:, 1:, None])[..., 0]
    want[1, 11:] = 0.0
    assert r.logprob.shape == (3, 16) and r.top_ids.shape == (3, 16, 5)
    assert bool(((r.logprob - want).abs() < 1e-4).all())
    assert bool(((r.entropy + (logp.exp() * logp).sum(-1)).abs() < 1e-4).all())
    assert torch.equal(r.top_ids, logp.topk(5, -1).indices)


@pytest.mark.gpu
def test_non_finite_logits_raise(cuda):
    model = _tiny(F32, cuda)
    with torch.no_grad():
        model.lm_head.weight.fill_(float("nan"))
    ids = torch.zeros(1, 4, dtype=torch.long, device=cuda)
    with pytest.raises(FloatingPointError, match="Non-finite"):
        generate(model, ids, 2, paged=True)
    with pytest.raises(FloatingPointError, match="Non-finite"):
        beam_search(model, ids, 2, 2)
    assert model.config._attn_implementation == "sdpa"


@pytest.mark.gpu
def test_sliding_window_is_refused(cuda):
    model = _tiny(F32, cuda, "qwen3")
    for layer in model.model.layers:
        layer.self_attn.sliding_window = 8
    with pytest.raises(ValueError, match="sliding-window"):
        generate(model, torch.zeros(1, 4, dtype=torch.long, device=cuda), 2, paged=True)
    assert model.config._attn_implementation == "sdpa"


@pytest.mark.gpu
def test_first_calls_of_a_process_can_be_captured(cuda):
    """The operators' first use on a device, inside a graph capture."""
    import subprocess
    import sys

    from conftest import REPO

    code = """
import torch
from s_salaad_b200.kvcache import PagedCache
from s_salaad_b200.ops import token_logprobs
cache = PagedCache(num_layers=1, num_pages=40, kv_heads=2, head_dim=64, max_seqs=3, max_pages=10)
long = PagedCache(num_layers=1, num_pages=40, kv_heads=2, head_dim=64, max_seqs=3, max_pages=5000)
k, q = torch.ones(3, 2, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 4, 64, dtype=torch.bfloat16, device="cuda")
x, t = torch.zeros(3, 1000, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
n = torch.tensor([1, 0, 17], dtype=torch.int32, device="cuda")
outs = []
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    for c in (cache, long):
        c.advance(n)
        c.append(0, k, k)
        outs.append(c.attend(0, q))
        c.compact()
    outs.append(token_logprobs(x, t, top=3))
for _ in range(3):
    g.replay()
torch.cuda.synchronize()
for c in (cache, long):
    assert c.lens.tolist() == [3, 0, 51], c.lens
    c.check()
assert not outs[0][1].any() and not outs[1][1].any()
assert outs[2].top_ids.tolist() == [[0, 1, 2]] * 3
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=REPO, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


@pytest.mark.gpu
def test_cache_resize_keeps_the_rows(cuda):
    model = _tiny(F32, cuda)
    cache = cache_for_model(model, 4, 100)
    assert (cache.num_layers, cache.kv_heads, cache.head_dim, cache.max_pages) == (2, 2, 16, 7)
    k = torch.randn(4 * 50, 2, 16, device=cuda)
    cache.advance(torch.full((4,), 50, dtype=torch.int32, device=cuda))
    cu = torch.arange(0, 201, 50, dtype=torch.int32, device=cuda)
    for layer in range(2):
        cache.append(layer, k + layer, k - layer, cu)
    q = torch.randn(4, 4, 16, device=cuda)
    cache.advance(0, torch.tensor([-1, 3, -1, 1], dtype=torch.int32, device=cuda))
    want = [cache.attend(layer, q) for layer in range(2)]
    with pytest.raises(ValueError, match="8 pages are in use"):
        cache.resize(7)
    cache.resize(8)
    assert cache.pool.shape[2] == 8 and int(cache.header[3]) == 8
    assert all(torch.equal(w, cache.attend(layer, q)) for layer, w in enumerate(want))
    cache.advance(1)
    assert cache.lens.tolist() == [0, 51, 0, 51]
    cache.check()
    cache.resize(40)
    cache.advance(torch.tensor([30, 0, 0, 20], dtype=torch.int32, device=cuda))
    cache.check()
    assert cache.lens.tolist() == [30, 51, 0, 71]
