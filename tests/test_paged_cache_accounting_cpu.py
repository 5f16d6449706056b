"""Paged cache of the Llama runtime: lengths and pages when calls cover some of the sequences, when sequences end and when the pool is tight."""
import pytest
import torch

from rustorch_b200.llm import LlamaConfig, LlamaRuntime, SamplingConfig


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


def test_a_released_sequence_sits_out_until_it_is_reserved_again():
    rt = _runtime()
    prompt, tok = _prompt(4, 9), torch.tensor([5, 6, 7, 8])
    cache, plain = rt.new_paged_cache(4, 32, page=3, n_pages=17), rt.new_cache(4, 32)
    rt.prefill(prompt, cache), rt.prefill(prompt, plain)
    cache.release(1)
    before = [k.clone() for k in cache.k]
    taken = [list(p) for p in cache.pages]
    for step in range(3):                                      # a pool that the others need for themselves
        out, want = rt.decode_step(tok, cache), rt.decode_step(tok, plain)
        assert torch.allclose(out[[0, 2, 3]], want[[0, 2, 3]], rtol=1e-4, atol=1e-4) and bool(torch.isfinite(out).all())
        assert cache.lengths == [10 + step, 0, 10 + step, 10 + step] and cache.pages[1] == []
    for k, old in zip(cache.k, before):                        # nothing was written to pages that nobody holds
        for page in cache.free:
            assert torch.equal(k[page], old[page])
    assert cache.pages[0][:3] == taken[0] and len(cache.free) == 17 - 3 * 4
    # its place is taken by another sequence, fed by hand
    new = _prompt(1, 5, seed=2)[0]
    cache.reserve(1, 5)
    pos = torch.arange(5)
    rt.forward_tokens(new, pos, torch.full_like(pos, 1), cache)
    cache.lengths[1] = 5
    out = rt.decode_step(tok, cache)
    fresh = rt.new_cache(1, 32)
    rt.prefill(new[None], fresh)
    assert torch.allclose(out[1], rt.decode_step(tok[1:2], fresh)[0], rtol=1e-4, atol=1e-4)
    assert cache.lengths == [13, 6, 13, 13]


def test_a_released_batch_is_filled_by_the_next_prompt_and_a_cleared_one_starts_anew():
    rt = _runtime()
    prompt, tok = _prompt(2, 7), torch.tensor([5, 6])
    cache = rt.new_paged_cache(2, 32, page=4)
    for _ in range(2):
        rt.prefill(prompt, cache)
        assert rt.decode_step(tok, cache).shape == (2, 97) and cache.lengths == [8, 8]
        cache.release(0), cache.release(1)
    assert rt.decode_step(tok, cache).shape == (2, 97) and cache.lengths == [0, 0] and len(cache.free) == cache.n_pages
    cache.clear()                                              # like a new cache, whose sequences start at position 0 with their first step
    plain = rt.new_cache(2, 32)
    for _ in range(2):
        assert torch.allclose(rt.decode_step(tok, cache), rt.decode_step(tok, plain), rtol=1e-4, atol=1e-4)
    assert cache.lengths == [2, 2]


def test_captured_sampling_without_numbers_is_refused():
    rt = _runtime()
    for bad in (None, torch.zeros(0, 2), torch.zeros(3, 4), torch.zeros(2)):
        with pytest.raises(ValueError, match="random numbers"):
            rt.capture_decode_graph(rt.new_paged_cache(2, 32), 2, SamplingConfig(), bad)
