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
