"""The Llama runtime on the paged cache and with tokens drawn on the device."""
import pytest
import torch

from conftest import rel_err

pytestmark = pytest.mark.gpu


def _runtime(**kw):
    from rustorch_b200.llm import LlamaConfig, LlamaRuntime
    cfg = LlamaConfig(**{**dict(vocab_size=1000, n_layer=3, n_embd=512, n_head=8, n_head_kv=2, n_ff=1024, context_length=512), **kw})
    return LlamaRuntime.random_init(cfg, device="cuda", seed=5, std=0.05)


@pytest.mark.parametrize("kw,T", [(dict(), 100), (dict(), 7), (dict(rope_interleaved=False, n_head=4, n_head_kv=4), 64),
                                  (dict(rope_scaling={"rope_type": "linear", "factor": 2.0}), 33), (dict(n_embd=384, n_head=4, n_head_kv=1, n_ff=512), 20)])
def test_paged_and_contiguous_caches_agree(kw, T):
    """Prompt (flash attention over 16 tokens and more, paged attention below) and decode steps, fed the same tokens."""
    rt = _runtime(**kw)
    prompt = torch.randint(0, 1000, (3, T), generator=torch.Generator().manual_seed(0))
    plain, paged = rt.new_cache(3, 160), rt.new_paged_cache(3, 160, page=16)
    a, b = rt.prefill(prompt, plain), rt.prefill(prompt, paged)
    assert rel_err(b, a) < 2e-2                                # fp16 activations: the tolerance of the runtime's other tests is 3e-2
    for _ in range(5):
        tok = a.argmax(-1)
        a, b = rt.decode_step(tok, plain), rt.decode_step(tok, paged)
        assert rel_err(b, a) < 2e-2
    for li in range(3):
        at = torch.arange(T + 5, device="cuda")
        for s in range(3):
            k = paged.k[li][paged.block_table[s].long()[at // 16], :, at % 16].transpose(0, 1)
            assert rel_err(k, plain.k[li][s, :, : T + 5]) < 2e-2


@pytest.mark.parametrize("paged", [False, True])
def test_graph_decode_draws_the_tokens_of_the_eager_loop(paged):
    """Greedy and sampled: the replayed graph gives what prefill, a step at a time and Sampler.draw give (the contiguous cache's
    attention splits its keys by the bound it is given, so the steps get the graph's)."""
    from rustorch_b200.llm import Sampler, SamplingConfig
    rt = _runtime()
    prompt = torch.randint(0, 1000, (4, 24), generator=torch.Generator().manual_seed(1))
    new = 12
    u = torch.rand(new, 4, generator=torch.Generator().manual_seed(2))
    make = (lambda: rt.new_paged_cache(4, 64, page=16)) if paged else (lambda: rt.new_cache(4, 64))
    for cfg in (None, SamplingConfig(temperature=0.9, top_k=100, top_p=0.95, min_p=0.01), SamplingConfig(temperature=1.2)):
        got, _ = rt.generate_graph(prompt, new, cache=make(), sampling=cfg, uniform=None if cfg is None else u)
        cache, sampler = make(), Sampler(cfg)
        logits, toks = rt.prefill(prompt, cache), []
        for i in range(new):
            toks.append(logits.argmax(-1) if cfg is None else sampler.draw(logits, u[i].cuda()))
            if i + 1 < new:
                if paged:
                    cache.reserve(0, 24 + new), cache.reserve(1, 24 + new), cache.reserve(2, 24 + new), cache.reserve(3, 24 + new)
                at = torch.full((4,), 24 + i, device="cuda")
                logits = rt.forward_tokens(toks[-1], at, torch.arange(4, device="cuda"), cache, max_kv=cache.max_len)
        assert torch.equal(got[:, 24:], torch.stack(toks, 1))
    seeded = SamplingConfig(temperature=1.0, seed=11)
    first, _ = rt.generate_graph(prompt, new, cache=make(), sampling=seeded)
    assert torch.equal(first, rt.generate_graph(prompt, new, cache=make(), sampling=seeded)[0])
    assert rt.generate_graph(prompt, 1, cache=make(), sampling=seeded)[0].shape == (4, 25)
    with pytest.raises(ValueError):
        rt.generate_graph(prompt, new, sampling=SamplingConfig(repetition_penalty=1.2))
    with pytest.raises(ValueError):
        rt.generate_graph(prompt, new, sampling=SamplingConfig(), uniform=u[:3])


def test_sequences_of_different_ages_share_a_pool():
    """A batch whose sequences grow, end and are replaced keeps each sequence's logits."""
    rt = _runtime()
    g = torch.Generator().manual_seed(3)
    cache = rt.new_paged_cache(3, 128, page=8, n_pages=20)
    prompts = [torch.randint(0, 1000, (n,), generator=g) for n in (50, 9, 30)]

    def feed(b, tokens, start):
        cache.reserve(b, start + len(tokens))
        pos = torch.arange(start, start + len(tokens), device="cuda")
        out = rt.forward_tokens(tokens.cuda(), pos, torch.full_like(pos, b), cache, last_only=torch.tensor([len(tokens) - 1], device="cuda"))
        cache.lengths[b] = start + len(tokens)
        return out
    for b, p in enumerate(prompts):
        feed(b, p[: len(p) // 2], 0)
    cache.release(1)
    prompts[1] = torch.randint(0, 1000, (40,), generator=g)
    feed(1, prompts[1][:20], 0)
    for b, p in enumerate(prompts):
        out = feed(b, p[cache.lengths[b]:], cache.lengths[b])
        alone = rt.prefill(p.view(1, -1), rt.new_cache(1, 128))
        assert rel_err(out, alone) < 2e-2
