"""The Llama runtime's table of rotation frequencies is made once."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 2.0}])
def test_one_table_serves_all_layers_and_steps(scaling):
    from rustorch_b200.llm import LlamaConfig, LlamaRuntime
    cfg = LlamaConfig(vocab_size=100, n_layer=2, n_embd=128, n_head=2, n_head_kv=1, n_ff=256, context_length=64, rope_scaling=scaling)
    rt = LlamaRuntime.random_init(cfg, device="cuda", seed=1, std=0.05)
    table = rt._inv_freq(64, rt.device)
    want = 10000.0 ** (-torch.arange(32, dtype=torch.float64) * 2.0 / 64) / (2.0 if scaling else 1.0)
    assert table.is_cuda and torch.allclose(table.double().cpu(), want, rtol=1e-5)
    for device in ("cuda", rt.device, table.device, torch.device("cuda", torch.cuda.current_device())):
        assert rt._inv_freq(64, device) is table
    calls = []
    build = rt._build_inv_freq
    rt._build_inv_freq = lambda *a: calls.append(a) or build(*a)
    rt.prefill(torch.zeros(1, 8, dtype=torch.long), rt.new_paged_cache(1, 32))
    assert not calls and rt._inv_freq(64, "cuda") is table


def test_a_table_made_inside_a_capture_is_not_kept():
    """Its memory belongs to the graph and holds nothing before the first replay."""
    from rustorch_b200.llm import LlamaConfig, LlamaRuntime
    cfg = LlamaConfig(vocab_size=100, n_layer=1, n_embd=128, n_head=2, n_head_kv=1, n_ff=256, context_length=64)
    rt = LlamaRuntime.random_init(cfg, device="cuda", seed=1, std=0.05)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = rt._inv_freq(64, "cuda")
    eager = rt._inv_freq(64, "cuda")
    assert eager is not inside and rt._inv_freq(64, "cuda") is eager
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inside, eager) and float(eager[0]) == 1.0
