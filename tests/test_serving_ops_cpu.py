"""Paged cache and sampling operators on CPU tensors against their 64-bit definitions, and what they refuse."""
import pytest
import torch

from rustorch_b200.error import IndexOutOfBounds
from rustorch_b200.ops.paged import paged_append, paged_attention
from rustorch_b200.ops.sampling import sample_tokens
from serving_reference import attend, draw_token, paged_cache, rotate


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot,norm", [(16, False), (8, True), (0, True)])
def test_append_rotates_and_places_rows(interleaved, rot, norm):
    g = torch.Generator().manual_seed(0)
    n, H, hkv, D, page = 5, 4, 2, 16, 3
    q, k, v = (torch.randn(n, h, D, generator=g) for h in (H, hkv, hkv))
    table = torch.tensor([[4, 1, -1], [0, 3, 5]], dtype=torch.int32)
    kp, vp = torch.zeros(6, hkv, page, D), torch.zeros(6, hkv, page, D)
    pos = torch.tensor([0, 5, 8, 2, 1], dtype=torch.int32)
    seq = torch.tensor([0, 0, 1, -1, 1], dtype=torch.int32)
    inv = torch.rand(rot // 2, generator=g)
    w = torch.rand(D, generator=g) + 0.5 if norm else None
    out = paged_append(q, k, v, kp, vp, table, pos, seq, inv, interleaved=interleaved, q_norm=w, k_norm=w, eps=1e-5)
    want_q, want_k = rotate(q, pos, inv, interleaved, w, 1e-5), rotate(k, pos, inv, interleaved, w, 1e-5)
    want_q[3] = 0.0
    assert (out - want_q).abs().max() < 2e-6 * 8
    written = torch.zeros(6, page, dtype=torch.bool)
    for t, (pg, row) in {0: (4, 0), 1: (1, 2), 2: (5, 2), 4: (0, 1)}.items():
        assert (kp[pg, :, row] - want_k[t]).abs().max() < 2e-6 * 8 and torch.equal(vp[pg, :, row], v[t])
        written[pg, row] = True
    assert kp.transpose(1, 2)[~written].abs().max() == 0 and vp.transpose(1, 2)[~written].abs().max() == 0


@pytest.mark.parametrize("window,softcap", [(0, 0.0), (5, 0.0), (0, 3.0), (1, 2.0)])
def test_attention_against_64_bits(window, softcap):
    g = torch.Generator().manual_seed(1)
    lengths = [0, 1, 7, 23]
    kp, vp, table = paged_cache(lengths, 2, 4, 16, torch.float32, "cpu", g)
    seq = torch.tensor([0, 1, 2, 3, 3, -1], dtype=torch.int32)
    kv_len = torch.tensor([0, 1, 7, 22, 23, 4], dtype=torch.int32)
    q = torch.randn(6, 6, 16, generator=g)
    out = paged_attention(q, kp, vp, table, kv_len, seq, window=window, softcap=softcap)
    want, tol = attend(q, kp, vp, table, kv_len, seq, 0.25, window, softcap)
    assert ((out.double() - want).abs() <= tol).all()
    assert out[0].abs().max() == 0 and out[5].abs().max() == 0


@pytest.mark.parametrize("temperature,top_k,top_p,min_p", [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (0.7, 5, 1.0, 0.0), (1.3, 0, 0.6, 0.0),
                                                           (1.0, 0, 1.0, 0.2), (0.9, 20, 0.8, 0.01)])
def test_sampling_against_the_definition(temperature, top_k, top_p, min_p):
    g = torch.Generator().manual_seed(2)
    logits = (torch.randn(40, 61, generator=g) * 2).half().float()
    logits[3] = 0.5                                                              # all equal
    logits[4, 10:] = -float("inf")
    logits[5, ::2] = float("nan")
    logits[6] = -float("inf")
    u = torch.rand(40, generator=g)
    u[7], u[8] = 0.0, 1.0
    got = sample_tokens(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got.tolist() == [draw_token(logits[r], float(u[r]), temperature, top_k, top_p, min_p) for r in range(40)]
    rows = sample_tokens(logits, u, temperature=torch.full((40,), temperature), top_k=torch.full((40,), top_k, dtype=torch.int32),
                         top_p=top_p, min_p=min_p)
    assert torch.equal(rows, got)                                                # one setting for all, or the same for every row


def test_bad_indices_raise():
    kp, vp = torch.zeros(2, 1, 4, 8), torch.zeros(2, 1, 4, 8)
    table = torch.tensor([[1, -1]], dtype=torch.int32)
    one = lambda x: torch.tensor([x], dtype=torch.int32)                         # noqa: E731
    q = torch.zeros(1, 1, 8)
    for pos, seq in ((4, 0), (8, 0), (-1, 0), (0, 1), (0, -2)):
        with pytest.raises(IndexOutOfBounds):
            paged_append(q, q, q, kp, vp, table, one(pos), one(seq), torch.zeros(4))
    for length, seq in ((5, 0), (9, 0), (-1, 0), (1, 1), (1, -2)):
        with pytest.raises(IndexOutOfBounds):
            paged_attention(q, kp, vp, table, one(length), one(seq))


def test_refusals():
    kp, vp = torch.zeros(2, 2, 4, 8), torch.zeros(2, 2, 4, 8)
    table = torch.zeros(1, 2, dtype=torch.int32)
    i1 = torch.zeros(1, dtype=torch.int32)
    q, k = torch.zeros(1, 4, 8), torch.zeros(1, 2, 8)
    for kw in (dict(q=torch.zeros(1, 3, 8)), dict(q=torch.zeros(1, 4, 16)), dict(kv_len=i1.long()), dict(block_table=table.long()),
               dict(seq=torch.zeros(2, dtype=torch.int32)), dict(v_pages=vp[:1]), dict(window=-1), dict(softcap=-1.0), dict(scale=float("nan"))):
        with pytest.raises(RuntimeError):
            paged_attention(**{**dict(q=q, k_pages=kp, v_pages=vp, block_table=table, kv_len=i1, seq=i1), **kw})
    for kw in (dict(k=torch.zeros(1, 4, 8)), dict(v=torch.zeros(1, 2, 4)), dict(pos=i1.long()), dict(inv_freq=torch.zeros(5)), dict(seq=i1.long())):
        with pytest.raises(RuntimeError):
            paged_append(**{**dict(q=q, k=k, v=k, k_pages=kp, v_pages=vp, block_table=table, pos=i1, seq=i1, inv_freq=torch.zeros(4)), **kw})
    with pytest.raises(ValueError):
        paged_attention(q.clone().requires_grad_(), kp, vp, table, i1, i1)
    with pytest.raises(ValueError):
        paged_append(q, k.clone().requires_grad_(), k, kp, vp, table, i1, i1, torch.zeros(4))
    logits, u = torch.zeros(2, 5), torch.zeros(2)
    for kw in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.5),
               dict(min_p=-0.1), dict(min_p=1.1), dict(uniform=torch.zeros(3)), dict(uniform=torch.zeros(2, dtype=torch.int32)),
               dict(temperature=torch.zeros(3)), dict(top_k=torch.zeros(2)), dict(logits=torch.zeros(5)), dict(logits=torch.zeros(2, 0))):
        with pytest.raises(RuntimeError):
            sample_tokens(**{**dict(logits=logits, uniform=u), **kw})
