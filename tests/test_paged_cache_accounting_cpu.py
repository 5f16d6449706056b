"""Paged cache of the Llama runtime: lengths and pages when calls cover some of the sequences, when sequences end and when the pool is tight."""
import pytest
import torch

from rustorch_b200.llm import LlamaConfig, LlamaRuntime


def _runtime(**kw):
    cfg = LlamaConfig(vocab_size=97, n_layer=2, n_embd=64, n_head=4, n_head_kv=2, n_ff=96, context_length=64, **kw)
    return LlamaRuntime.random_init(cfg, device="cpu", seed=3, std=0.2)


def _prompt(rows, n, seed=0):
    return torch.randint(0, 97, (rows, n), generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("paged", [False, True])
def test_a_prompt_of_fewer_rows_keeps_the_other_sequences(paged):
    rt = _runtime()
    cache = rt.new_paged_cache(4, 32, page=4) if paged else rt.new_cache(4, 32)
    first, second = _prompt(4, 9), _prompt(2, 6, seed=1)
    rt.prefill(first, cache)
    rt.prefill(second, cache)
    assert cache.lengths == [6, 6, 9, 9] and cache.seq_len(3) == 9
    tok = torch.tensor([1, 2, 3, 4])
    out = rt.decode_step(tok, cache)
    assert cache.lengths == [7, 7, 10, 10]
    alone = rt.new_cache(4, 32)
    rt.prefill(first, alone)
    assert torch.allclose(out[2:], rt.decode_step(tok, alone)[2:], rtol=1e-4, atol=1e-4)
    fresh = rt.new_cache(2, 32)
    rt.prefill(second, fresh)
    assert torch.allclose(out[:2], rt.decode_step(tok[:2], fresh), rtol=1e-4, atol=1e-4)
    rt.decode_step(tok[:2], cache)                             # a step of the first two
    assert cache.lengths == [8, 8, 10, 10]
    if paged:
        cache.release(3)
        assert cache.lengths[3] == 0 and cache.pages[3] == []
        cache.reserve(3, 5)
    cache.clear()
    assert cache.lengths == [0] * 4
    if paged:
        assert sorted(cache.free) == list(range(cache.n_pages)) and bool((cache.block_table == -1).all())


def test_clear_gives_back_pages_of_sequences_that_no_call_covered():
    rt = _runtime()
    cache = rt.new_paged_cache(4, 32, page=4)
    cache.reserve(3, 20)
    rt.prefill(_prompt(2, 9), cache)
    cache.clear()
    assert sorted(cache.free) == list(range(32))
    cache.release(3)
    assert cache.lengths == [0] * 4
