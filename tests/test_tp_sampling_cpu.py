"""Sampled decoding on tensor-parallel ranks (gloo, two processes): every rank draws by the same numbers."""
import json
import os
import socket
import subprocess
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

WORKER = """
import json, sys
import torch
import torch.distributed as dist
from datetime import timedelta
from rustorch_b200.llm import LlamaConfig, LlamaRuntime, Sampler, SamplingConfig
dist.init_process_group("gloo", timeout=timedelta(seconds=60))
rank = dist.get_rank()
cfg = LlamaConfig(vocab_size=97, n_layer=2, n_embd=64, n_head=4, n_head_kv=2, n_ff=128, context_length=64)
rt = LlamaRuntime.random_init(cfg, device="cpu", tp_rank=rank, tp_world=2, tp_group=dist.group.WORLD, seed=3, std=0.2)
torch.manual_seed(100 + rank)                       # processes whose generators stand at different places
out = {"unseeded": rt._numbers(SamplingConfig(), 6, 3).tolist(), "seeded": rt._numbers(SamplingConfig(seed=4), 6, 3).tolist()}
mine = torch.full((6, 3), 0.25 * (rank + 1), dtype=torch.float64)
given = rt._numbers(SamplingConfig(), 6, 3, mine)
out["given"], out["mine"] = given.tolist(), mine.tolist()
u = rt._shared_numbers(torch.rand(6, 3))
prompt = torch.randint(0, 97, (3, 9), generator=torch.Generator().manual_seed(0))
cache, sampler, toks = rt.new_paged_cache(3, 32, page=4), Sampler(SamplingConfig(temperature=1.5)), []
logits = rt.prefill(prompt, cache)
for i in range(6):
    toks.append(sampler.draw(logits, u[i]))
    logits = rt.decode_step(toks[-1], cache)
out["tokens"] = torch.stack(toks, 1).tolist()
json.dump(out, open(sys.argv[1], "w"))
dist.destroy_process_group()
"""


def test_tensor_parallel_ranks_draw_by_the_first_ranks_numbers(tmp_path):
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    procs = []
    for r in range(2):
        env = dict(os.environ, MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), RANK=str(r), WORLD_SIZE="2", OMP_NUM_THREADS="1")
        procs.append(subprocess.Popen([sys.executable, "-c", WORKER, str(tmp_path / f"{r}.json")], env=env, cwd=ROOT, stdout=subprocess.PIPE,
                                      stderr=subprocess.STDOUT, text=True))
    outs = [p.communicate(timeout=180)[0] for p in procs]
    for p, o in zip(procs, outs):
        assert p.returncode == 0, o[-3000:]
    a, b = (json.load(open(tmp_path / f"{r}.json")) for r in range(2))
    for key in ("unseeded", "seeded", "given", "tokens"):
        assert a[key] == b[key], key
    assert a["unseeded"] == torch.rand(6, 3, generator=torch.Generator().manual_seed(100)).tolist()
    assert a["seeded"] == torch.rand(6, 3, generator=torch.Generator().manual_seed(4)).tolist()
    assert a["given"] == [[0.25] * 3] * 6 and b["mine"] == [[0.5] * 3] * 6       # the caller's own tensor stays
