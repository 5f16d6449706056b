"""Captured decoding at its limits: a cache that just fits, numbers that run out, sequences that the batch does not cover."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _runtime(**kw):
    from rustorch_b200.llm import LlamaConfig, LlamaRuntime
    cfg = LlamaConfig(**{**dict(vocab_size=1000, n_layer=3, n_embd=512, n_head=8, n_head_kv=2, n_ff=1024, context_length=512), **kw})
    return LlamaRuntime.random_init(cfg, device="cuda", seed=5, std=0.05)


def _prompt(rows, n):
    return torch.randint(0, 1000, (rows, n), generator=torch.Generator().manual_seed(rows * n))


@pytest.mark.parametrize("new", [1, 9])
def test_graph_generation_fits_a_cache_without_a_place_for_the_last_token(new):
    """The last token is returned, never appended: T + new - 1 positions are enough, as for the eager loop."""
    from rustorch_b200 import _native
    rt, prompt = _runtime(), _prompt(3, 24)
    tight = rt.new_paged_cache(3, 24 + new - 1, page=1, n_pages=3 * (24 + new - 1))
    got, _ = rt.generate_graph(prompt, new, cache=tight)
    _native.check_status()
    assert torch.equal(got, rt.generate_graph(prompt, new, cache=rt.new_paged_cache(3, 128))[0])
    assert tight.lengths == [24 + new - 1] * 3 and tight.free == []


def test_replays_beyond_the_numbers_use_the_last_row():
    """Four rows of numbers, seven replays: the last ones draw by the fourth row and stay in its place of the output."""
    from rustorch_b200 import _native
    from rustorch_b200.llm import SamplingConfig
    rt, prompt = _runtime(), _prompt(2, 5)
    cfg, u = SamplingConfig(temperature=1.1, top_p=0.95), torch.rand(4, 2, generator=torch.Generator().manual_seed(1))

    def decode(numbers, replays):
        cache = rt.new_paged_cache(2, 64, page=8)
        cache.reserve(0, 20), cache.reserve(1, 20)
        g = rt.capture_decode_graph(cache, 2, cfg, numbers)
        logits = rt.prefill(prompt, cache)
        g.tok.copy_(logits.argmax(-1)), g.pos.fill_(5), g.step.zero_()
        for _ in range(replays):
            g.graph.replay()
        torch.cuda.synchronize()
        _native.check_status()
        return g.out.cpu(), g.tok.cpu(), int(g.step)
    out, tok, step = decode(u, 7)
    long_out, long_tok, _ = decode(torch.cat([u, u[3:].expand(3, -1)]), 7)       # the same numbers, spelled out
    assert step == 3 and torch.equal(out[:, :3], long_out[:, :3]) and torch.equal(tok, long_tok)
    assert torch.equal(out[:, 3], long_out[:, 6]) and int(out[:, 4:].abs().sum()) == 0
    exact, _, _ = decode(u, 4)
    assert torch.equal(exact[:, :4], long_out[:, :4])
