"""Paged cache of the Llama runtime on CPU: page accounting, and the same tokens as with the contiguous cache."""
import pytest
import torch

from rustorch_b200.llm import LlamaConfig, LlamaRuntime, PagedKVCache, Sampler, SamplingConfig, apply_min_p_to_probs
from serving_reference import draw_token


def _runtime(**kw):
    cfg = LlamaConfig(vocab_size=97, n_layer=2, n_embd=64, n_head=4, n_head_kv=2, n_ff=96, context_length=64, **kw)
    return LlamaRuntime.random_init(cfg, device="cpu", seed=3, std=0.2)


@pytest.mark.parametrize("kw", [dict(), dict(rope_interleaved=False), dict(rope_scaling={"rope_type": "linear", "factor": 4.0})])
@pytest.mark.parametrize("page", [1, 5, 64])
def test_paged_cache_gives_the_same_logits_and_tokens(kw, page):
    rt = _runtime(**kw)
    prompt = torch.randint(0, 97, (3, 11), generator=torch.Generator().manual_seed(0))
    plain, paged = rt.new_cache(3, 32), rt.new_paged_cache(3, 32, page=page)
    a, b = rt.prefill(prompt, plain), rt.prefill(prompt, paged)
    assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)          # angles in 64 bits there, in 32 here; the rest is 32-bit arithmetic
    for _ in range(4):
        tok = a.argmax(-1)
        a, b = rt.decode_step(tok, plain), rt.decode_step(tok, paged)
        assert torch.allclose(a, b, rtol=1e-4, atol=1e-4)
    assert paged.lengths == plain.lengths == [15] * 3 and paged.seq_len(1) == 15
    assert [len(p) for p in paged.pages] == [(15 + page - 1) // page] * 3
    out, _ = rt.generate(prompt, 5, cache=rt.new_paged_cache(3, 32, page=page))
    assert torch.equal(out, rt.generate(prompt, 5)[0])


def test_pages_are_shared_and_given_back():
    c = PagedKVCache(1, 3, 2, max_len=40, head_dim=8, device="cpu", dtype=torch.float32, page=4, n_pages=12)
    assert c.nbytes() == 2 * 12 * 2 * 4 * 8 * 4
    c.reserve(0, 9)
    c.reserve(1, 4)
    c.reserve(0, 5)                                            # has them already
    assert len(c.pages[0]) == 3 and len(c.pages[1]) == 1 and len(c.free) == 8
    assert c.block_table[0].tolist()[:4] == c.pages[0] + [-1] and len({*c.pages[0], *c.pages[1]}) == 4
    with pytest.raises(RuntimeError, match="full"):
        c.reserve(2, 36)
    assert c.pages[2] == [] and len(c.free) == 8
    with pytest.raises(ValueError):
        c.reserve(2, 41)
    c.release(0)
    c.reserve(2, 36)
    assert len(c.free) == 2 and c.block_table[0].tolist() == [-1] * 10
    c.clear()
    assert sorted(c.free) == list(range(12)) and c.lengths == [0, 0, 0]
    for bad in (dict(page=0), dict(max_len=0)):
        with pytest.raises(ValueError):
            PagedKVCache(1, 1, 1, **{**dict(max_len=4, head_dim=8, device="cpu"), **bad})


def test_freed_pages_serve_another_sequence():
    """A sequence that took over released pages sees only its own tokens."""
    rt = _runtime()
    g = torch.Generator().manual_seed(1)
    first, second = torch.randint(0, 97, (1, 20), generator=g), torch.randint(0, 97, (1, 9), generator=g)
    cache = rt.new_paged_cache(1, 32, page=4, n_pages=6)
    rt.prefill(first, cache)
    cache.release(0)
    assert torch.allclose(rt.prefill(second, cache), rt.prefill(second, rt.new_cache(1, 32)), rtol=1e-4, atol=1e-4)


def test_min_p_and_draw():
    probs = torch.tensor([[0.5, 0.3, 0.15, 0.05]])
    assert torch.allclose(apply_min_p_to_probs(probs, 0.2), torch.tensor([[0.5, 0.3, 0.15, 0.0]]) / 0.95)
    assert apply_min_p_to_probs(probs, 0.0) is probs
    with pytest.raises(ValueError):
        SamplingConfig(min_p=1.5).validate()
    g = torch.Generator().manual_seed(2)
    logits, u = torch.randn(6, 50, generator=g) * 2, torch.rand(6, generator=g)
    s = Sampler(SamplingConfig(temperature=0.8, top_k=20, top_p=0.9, min_p=0.05, repetition_penalty=1.3))
    tok = s.draw(logits, u)
    assert tok.tolist() == [draw_token(logits[r], float(u[r]), 0.8, 20, 0.9, 0.05) for r in range(6)]
    again = s.draw(logits, u)
    penalised = logits.clone()
    for r in range(6):
        x = float(logits[r, tok[r]])
        penalised[r, tok[r]] = x / 1.3 if x > 0 else x * 1.3
    assert again.tolist() == [draw_token(penalised[r], float(u[r]), 0.8, 20, 0.9, 0.05) for r in range(6)]
    assert s.history.shape == (6, 2)
    torch.manual_seed(0)
    counts = torch.bincount(torch.stack([Sampler(SamplingConfig(min_p=0.25))(torch.log(probs)) for _ in range(200)]).flatten(), minlength=4)
    assert counts[3] == 0 and counts[:3].min() > 0
