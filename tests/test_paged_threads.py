"""One model used by several threads, some of them on a paged cache.

The cache is a plain one on the host, so no GPU is needed: what is tested is
which attention each thread's forward reaches.
"""
from __future__ import annotations

import threading

import pytest
import torch

from s_salaad_b200 import workloads
from s_salaad_b200.inference.paged import _decode, _on_cache, _prefill


class HostCache:
    """The part of PagedCache that a model's forward calls, on the host."""

    device = torch.device("cpu")

    def __init__(self, rows):
        self.max_seqs, self.lens = rows, torch.zeros(rows, dtype=torch.int32)
        self.kv = {}

    def advance(self, n_new):
        self.lens += n_new

    def append(self, layer, k, v, cu_tokens=None):
        for r in range(self.max_seqs):
            a, b = (r, r + 1) if cu_tokens is None else (int(cu_tokens[r]), int(cu_tokens[r + 1]))
            old = self.kv.get((layer, r), (k[:0], v[:0]))
            self.kv[layer, r] = torch.cat([old[0], k[a:b]]), torch.cat([old[1], v[a:b]])
            assert len(self.kv[layer, r][0]) == int(self.lens[r])

    def attend(self, layer, q, *, scale):
        out = torch.empty_like(q)
        for r in range(self.max_seqs):
            k, v = (t.repeat_interleave(q.shape[1] // t.shape[1], 1) for t in self.kv[layer, r])
            p = torch.softmax(torch.einsum("hd,thd->ht", q[r], k) * scale, -1)
            out[r] = torch.einsum("ht,thd->hd", p, v)
        return out


def _model(attn):
    from s_salaad_b200.efficient import build_model_from_config

    cfg = dict(workloads.LLAMA_60M, hidden_size=64, intermediate_size=128, num_hidden_layers=2, num_attention_heads=4,
               num_key_value_heads=2, vocab_size=97, max_position_embeddings=64, model_type="llama")
    torch.manual_seed(0)
    model = build_model_from_config(cfg, attn_implementation=attn).eval()
    with torch.no_grad():
        model.lm_head.weight.mul_(20.0)
    return model


class Steps:
    """A thread on a cache of its own that takes a step whenever it is told to."""

    def __init__(self, model, ids):
        self.model, self.ids, self.logits, self.error = model, ids, [], None
        self.go, self.done = threading.Semaphore(0), threading.Semaphore(0)
        self.thread = threading.Thread(target=self._run, daemon=True)
        self.thread.start()

    def _run(self):
        with torch.inference_mode():
            self.go.acquire()
            try:
                cache = HostCache(self.ids.shape[0])
                with _on_cache(self.model, cache):
                    self.logits.append(_prefill(self.model, cache, self.ids[:, :3]))
                    for t in range(3, self.ids.shape[1]):
                        self.done.release()
                        self.go.acquire()
                        cache.advance(1)
                        self.logits.append(_decode(self.model, cache, self.ids[:, t]))
            except BaseException as e:  # noqa: BLE001 (handed to the test)
                self.error = e
            self.done.release()

    def step(self):
        self.go.release()
        assert self.done.acquire(timeout=60)
        if self.error is not None:
            raise self.error


@pytest.mark.parametrize("attn", ["sdpa", "eager"])
@pytest.mark.parametrize("order", ["ab-first-ends-first", "ab-last-ends-first"])
def test_threads_that_generate_with_one_model(attn, order):
    """Whoever ends first, the others go on with their own caches; forwards of
    threads without one use the model's own attention, padding included."""
    model = _model(attn)
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 97, (2, 2, 7), generator=g)
    plain = torch.randint(0, 97, (2, 6), generator=g)
    mask = torch.tensor([[0, 0, 1, 1, 1, 1], [1] * 6])

    def own():
        with torch.inference_mode():
            return (model(input_ids=plain, attention_mask=mask, use_cache=False).logits[mask.bool()],
                    model(input_ids=plain, use_cache=False).logits)

    before = own()
    with torch.inference_mode():
        full = [model(input_ids=i, use_cache=False).logits for i in ids]
    short, long = Steps(model, ids[0, :, :5]), Steps(model, ids[1])
    first, second = (short, long) if order == "ab-first-ends-first" else (long, short)
    first.step()
    second.step()
    for a, b in zip(before, own()):
        assert torch.equal(a, b)
    long.step()
    short.step()
    short.step()  # ends
    assert not short.thread.join(60) and not short.thread.is_alive()
    for a, b in zip(before, own()):
        assert torch.equal(a, b)
    for _ in range(3):
        long.step()
    long.thread.join(60)
    for user, want, n in ((short, full[0], 5), (long, full[1], 7)):
        assert len(user.logits) == n - 2
        for j, got in enumerate(user.logits):
            # fp32 on both sides, sums in another order
            assert bool(((got - want[:, 2 + j]).abs() <= 1e-4 * want.abs().max()).all()), j
    assert model.config._attn_implementation == attn
    for a, b in zip(before, own()):
        assert torch.equal(a, b)


def test_an_error_in_one_thread_leaves_the_others(monkeypatch):
    model = _model("sdpa")
    ids = torch.arange(10).view(2, 5)
    with torch.inference_mode():
        want = model(input_ids=ids, use_cache=False).logits
    user = Steps(model, ids)
    user.step()
    with pytest.raises(ZeroDivisionError):
        with _on_cache(model, HostCache(1)):
            raise ZeroDivisionError
    user.step()
    user.step()
    assert bool(((user.logits[2] - want[:, 4]).abs() <= 1e-4 * want.abs().max()).all())
    assert model.config._attn_implementation == "sdpa"


def test_a_forward_hook_that_generates():
    """A generation inside a forward on a cache: the inner one has its own
    cache, and the outer one goes on with its own."""
    model = _model("sdpa")
    ids, other = torch.arange(10).view(2, 5), torch.arange(50, 58).view(2, 4)
    got = {}

    def inner(module, args):
        if "inner" not in got:
            got["inner"] = None
            cache = HostCache(2)
            with _on_cache(model, cache):
                got["inner"] = _prefill(model, cache, other)

    with torch.inference_mode():
        want, want_inner = (model(input_ids=i, use_cache=False).logits[:, -1] for i in (ids, other))
        hook = model.model.layers[1].register_forward_pre_hook(inner)
        done = threading.Event()

        def outer():
            with torch.inference_mode():
                cache = HostCache(2)
                with _on_cache(model, cache):
                    _prefill(model, cache, ids[:, :4])
                    cache.advance(1)
                    got["outer"] = _decode(model, cache, ids[:, 4])
            done.set()

        threading.Thread(target=outer, daemon=True).start()
        assert done.wait(60)
    hook.remove()
    for a, b in ((got["inner"], want_inner), (got["outer"], want)):
        assert bool(((a - b).abs() <= 1e-4 * b.abs().max()).all())
    assert model.config._attn_implementation == "sdpa"


@pytest.mark.gpu
def test_threads_with_a_compressed_model(cuda, tmp_path):
    """Each thread gets what it gets alone, bit by bit (the layers' kernels do
    not depend on timing), although the layers' workspaces are shared."""
    from s_salaad_b200.efficient import build_efficient_model
    from s_salaad_b200.inference import beam_search, generate

    path = tmp_path / "cfg2.pt"
    workloads.compressed_bundle(path, n_layers=2)
    model, config, _ = build_efficient_model(path, device=cuda, dtype=torch.bfloat16)
    own = model.config._attn_implementation
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, config["vocab_size"], (1 + i % 3, 5 + 9 * i), generator=g).to(cuda) for i in range(4)]

    def run(i):
        if i == 3:
            return beam_search(model, prompts[i], 20, 2)[0]
        return generate(model, prompts[i], 20 + 5 * i, paged=True)

    alone = [run(i) for i in range(4)]
    got, errors = [[] for _ in range(4)], []

    def work(i):
        try:
            for _ in range(3):
                got[i].append(run(i))
        except BaseException as e:  # noqa: BLE001 (handed to the test)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,), daemon=True) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(300)
    assert not errors, errors
    for i in range(4):
        assert len(got[i]) == 3 and all(torch.equal(x, alone[i]) for x in got[i]), i
    assert model.config._attn_implementation == own
