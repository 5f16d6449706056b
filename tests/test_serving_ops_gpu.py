"""Paged cache append, paged attention and token sampling kernels against their 64-bit definitions."""
import math
import os
import subprocess
import sys

import pytest
import torch

from serving_reference import attend, draw_token, half_step, paged_cache, rotate, rotate_tolerance

pytestmark = pytest.mark.gpu


def _ops():
    from rustorch_b200.ops import paged, sampling
    return paged.paged_append, paged.paged_attention, sampling.sample_tokens


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _check(out, want, tol, what=""):
    bad = (out.double().cpu() - want).abs() > tol
    assert not bool(bad.any()) and bool(torch.isfinite(out).all()), (what, int(bad.sum()), bad.nonzero()[:3].tolist())


# -------------------------------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,hkv,D,rot,page,interleaved,norm", [
    (32, 8, 128, 128, 16, False, True), (4, 4, 64, 64, 32, True, False), (12, 12, 64, 32, 24, False, False), (14, 2, 80, 80, 24, True, True),
    (3, 1, 96, 96, 1, False, True), (2, 2, 256, 64, 64, False, True), (5, 5, 40, 24, 7, False, False), (1, 1, 36, 36, 5, True, True),
    (2, 1, 192, 192, 128, True, True), (2, 1, 31, 30, 8, False, True), (4, 2, 32, 0, 16, False, True), (1, 1, 512, 512, 16, False, True)])
def test_append_against_64_bits(dtype, H, hkv, D, rot, page, interleaved, norm):
    append, _, _ = _ops()
    g = torch.Generator().manual_seed(D)
    start, new = [0, 131000, 5], [9, 3, 1]
    max_pages = 131072 // page + 1
    n, n_pages = sum(new), 30
    table = torch.full((3, max_pages), -1, dtype=torch.int32)
    order, used = torch.randperm(n_pages, generator=g), 0
    for s in range(3):
        for p in range(start[s] // page, (start[s] + new[s] - 1) // page + 1):
            table[s, p] = order[used]
            used += 1
    pos = torch.cat([torch.arange(a, a + m) for a, m in zip(start, new)]).to(torch.int32)
    seq = torch.arange(3, dtype=torch.int32).repeat_interleave(torch.tensor(new))
    perm = torch.randperm(n, generator=g)
    pos, seq = pos[perm], seq[perm]
    qkv = torch.randn(n, (H + 2 * hkv) * D, generator=g).to(dtype)
    q, k, v = (x.reshape(n, -1, D) for x in qkv.split([H * D, hkv * D, hkv * D], 1))
    inv = (10000.0 ** (-torch.arange(rot // 2).double() * 2 / max(1, rot))).float()
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype) if norm else None for _ in range(2)]
    kp, vp = (torch.randn(n_pages, hkv, page, D, generator=g).to(dtype) for _ in range(2))
    want_q, want_k = rotate(q, pos, inv, interleaved, w[0], 1e-5), rotate(k, pos, inv, interleaved, w[1], 1e-5)
    dev = [x.cuda() if x is not None else None for x in (qkv, kp, vp, table, pos, seq, inv, *w)]
    qkv_d, kp_d, vp_d = dev[:3]
    views = [x.unflatten(1, (-1, D)) for x in qkv_d.split([H * D, hkv * D, hkv * D], 1)]         # strided, as a projection leaves them
    k_out = torch.empty(n, hkv, D, dtype=dtype, device="cuda")
    out = append(*views, kp_d, vp_d, *dev[3:7], interleaved=interleaved, q_norm=dev[7], k_norm=dev[8], eps=1e-5, k_out=k_out)
    _check(out, want_q, rotate_tolerance(want_q, dtype), "q")
    _check(k_out, want_k, rotate_tolerance(want_k, dtype), "k_out")
    for t in range(n):
        pg, row = int(table[seq[t], pos[t] // page]), int(pos[t]) % page
        assert torch.equal(kp_d[pg, :, row], k_out[t]) and torch.equal(vp_d[pg, :, row].cpu(), v[t])
        kp[pg, :, row], vp[pg, :, row] = kp_d[pg, :, row].cpu(), vp_d[pg, :, row].cpu()
    assert torch.equal(kp_d.cpu(), kp) and torch.equal(vp_d.cpu(), vp)                           # no other row was touched
    assert torch.equal(qkv_d.cpu(), qkv)
    # in place, and again: the same bits
    again = append(*views, kp_d, vp_d, *dev[3:7], interleaved=interleaved, q_norm=dev[7], k_norm=dev[8], eps=1e-5, q_out=views[0], k_out=views[1])
    assert again.data_ptr() == views[0].data_ptr() and torch.equal(again, out) and torch.equal(views[1], k_out) and torch.equal(kp_d.cpu(), kp)


def test_append_strides_and_alignment():
    """Rows at odd offsets, transposed heads, pages laid out row by row, expanded inputs: the values do not depend on the layout."""
    append, _, _ = _ops()
    g = torch.Generator().manual_seed(3)
    n, H, hkv, D, page = 6, 4, 2, 64, 8
    pos, table, inv = _i32([0, 1, 2, 3, 8, 9]), _i32([[2, 0, 1]]), torch.rand(32, generator=g).cuda()
    seq = _i32([0] * 6)
    q, k, v = (torch.randn(n, h, D, generator=g).half().cuda() for h in (H, hkv, hkv))
    kp, vp = torch.zeros(3, hkv, page, D, dtype=torch.half, device="cuda"), torch.zeros(3, hkv, page, D, dtype=torch.half, device="cuda")
    out = append(q, k, v, kp, vp, table, pos, seq, inv)

    def odd(x):
        y = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")[1:].view(x.shape)
        return y.copy_(x)
    for qq, kk, vv in ((odd(q), odd(k), odd(v)), tuple(x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))):
        pool = torch.zeros(3, page, 2, hkv, D, dtype=torch.half, device="cuda").permute(2, 0, 3, 1, 4)
        assert torch.equal(append(qq, kk, vv, pool[0], pool[1], table, pos, seq, inv, q_out=odd(q)), out)
        assert torch.equal(pool[0], kp) and torch.equal(pool[1], vp)
    one = k[:, :1].expand(-1, hkv, -1)
    append(q, one, one, kp, vp, table, pos, seq, inv)
    assert torch.equal(kp[:, 0], kp[:, 1]) and torch.equal(vp[2, 1, 3], k[3, 0])


# ----------------------------------------------------------------------------------------------------------- attention
LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 777]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,hkv,D,page,window,softcap", [
    (8, 2, 128, 16, 0, 0.0), (4, 4, 64, 32, 0, 0.0), (14, 2, 80, 24, 100, 30.0), (16, 1, 128, 64, 0, 0.0), (17, 1, 64, 16, 64, 0.0),
    (3, 3, 96, 1, 0, 5.0), (40, 1, 32, 8, 1, 0.0), (2, 1, 256, 128, 33, 0.0), (5, 1, 192, 5, 0, 0.0), (6, 2, 8, 1000, 0, 0.0), (7, 7, 248, 16, 17, 2.0)])
def test_attention_against_64_bits(dtype, H, hkv, D, page, window, softcap):
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(D + H)
    kp, vp, table = paged_cache(LENGTHS, hkv, page, D, dtype, "cuda", g)
    q = torch.randn(len(LENGTHS), H, D, generator=g).to(dtype).cuda()
    out = attention(q, kp, vp, table, _i32(LENGTHS), window=window, softcap=softcap)
    want, tol = attend(q, kp, vp, table, LENGTHS, None, 1 / math.sqrt(D), window, softcap)
    _check(out, want, tol)
    assert float(out[0].abs().max()) == 0.0
    assert torch.equal(out, attention(q, kp, vp, table, _i32(LENGTHS), window=window, softcap=softcap))      # the same bits again


@pytest.mark.parametrize("length,H,hkv,D", [(40001, 4, 1, 128), (9000, 8, 8, 64), (70000, 2, 2, 64), (20003, 16, 1, 256)])
def test_attention_over_one_long_sequence(length, H, hkv, D):
    """The length is the only axis to split: a scale that makes single keys matter, one of them at each end."""
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(length)
    kp, vp, table = paged_cache([length], hkv, 64, D, torch.bfloat16, "cuda", g)
    q = torch.randn(1, H, D, generator=g).bfloat16().cuda()
    for at in (0, length - 1, length // 2):
        kp[table[0, at // 64].long(), :, at % 64] = q[0, ::H // hkv]
    want, tol = attend(q, kp, vp, table, [length], None, 1 / math.sqrt(D))
    _check(attention(q, kp, vp, table, _i32([length])), want, tol)


def test_attention_many_tokens_of_few_sequences():
    """1100 tokens (prompt pieces, padded ones among them) of three sequences, in any order; every one sees its own length."""
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(4)
    lengths = [300, 41, 650]
    kp, vp, table = paged_cache(lengths, 2, 16, 64, torch.float16, "cuda", g, layout="row")
    seq = torch.randint(-1, 3, (1100,), generator=g, dtype=torch.int32)
    kv_len = torch.tensor([int(torch.randint(0, lengths[max(0, int(s))] + 1, (1,), generator=g)) for s in seq], dtype=torch.int32)
    qkv = torch.randn(1100, 6, 64, generator=g).half().cuda()
    q = qkv[:, 1:5]                                                              # strided
    out = torch.full((1100, 4, 64), float("nan"), dtype=torch.half, device="cuda")
    assert attention(q, kp, vp, table, kv_len.cuda(), seq.cuda(), scale=0.2, out=out) is out
    want, tol = attend(q, kp, vp, table, kv_len, seq, 0.2)
    _check(out, want, tol)
    # a transposed output and queries at an odd address: the same bits
    other = torch.empty(4, 1100, 64, dtype=torch.half, device="cuda").transpose(0, 1)
    q_odd = torch.empty(q.numel() + 1, dtype=torch.half, device="cuda")[1:].view(q.shape).copy_(q)
    assert torch.equal(attention(q_odd, kp, vp, table, kv_len.cuda(), seq.cuda(), scale=0.2, out=other), out)


def test_attention_extreme_scores():
    """Scores far apart (one key takes all), all equal (the mean of V), and a negative scale."""
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(5)
    kp, vp, table = paged_cache([500], 1, 16, 64, torch.float16, "cuda", g)
    q = torch.randn(1, 2, 64, generator=g).half().cuda()
    for scale in (1000.0, 0.0, -0.5):
        want, tol = attend(q, kp, vp, table, [500], None, scale)
        _check(attention(q, kp, vp, table, _i32([500]), scale=scale), want, tol, scale)
    kp[table[0, :31].long()] = 60000.0                                           # dot products near the largest 32-bit powers of two, all equal
    out = attention(q.abs() * 0 + 60000.0, kp, vp, table, _i32([500]), scale=1.0)
    want = vp[table[0, :31].long()].transpose(1, 2).reshape(-1, 64).double().mean(0)      # 496 keys share it: the last four score far below
    assert ((out[0].double() - want).abs() <= (half_step(torch.float16) + 600 * 2.0 ** -24) * 4 + half_step(torch.float16) * want.abs()).all()


@pytest.mark.parametrize("softcap", [1e5, 1e30])
def test_attention_cap_far_above_the_scores(softcap):
    """cap tanh(x / cap) - x is x^3 / (3 cap^2), nothing here: the tolerance is that of uncapped scores, whose ``(D + 4) 2^-24`` of
    the products' sizes covers the eight roundings of the capped form."""
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(8)
    kp, vp, table = paged_cache([700], 2, 16, 64, torch.float16, "cuda", g)
    q = torch.randn(1, 4, 64, generator=g).half().cuda()
    want, tol = attend(q, kp, vp, table, [700], None, 0.5)
    _check(attention(q, kp, vp, table, _i32([700]), scale=0.5, softcap=softcap), want, tol)


def test_attention_writes_over_its_queries():
    _, attention, _ = _ops()
    g = torch.Generator().manual_seed(9)
    kp, vp, table = paged_cache([3000, 5, 0], 2, 16, 128, torch.bfloat16, "cuda", g)
    q = torch.randn(3, 40, 128, generator=g).bfloat16().cuda()
    want = attention(q, kp, vp, table, _i32([3000, 5, 0]))
    assert attention(q, kp, vp, table, _i32([3000, 5, 0]), out=q) is q and torch.equal(q, want)


# ------------------------------------------------------------------------------------------------------------ sampling
def _logits(rows, vocab, dtype, gen):
    x = torch.randn(rows, vocab, generator=gen) * 2
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 20), generator=gen), 4 + 3 * torch.rand(rows, 20, generator=gen))
    x = x.to(dtype)
    if rows > 6:
        x[1] = 0.25                                                              # all equal
        x[2, vocab // 3:] = -float("inf")
        x[3, ::2] = float("nan")
        x[4] = -float("inf")
        x[5, ::7] = float("inf")
        x[6] = torch.where(torch.arange(vocab) % 3 == 0, 0.0, -0.0).to(dtype)    # equal numbers of two signs
    return x


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 300, 4097, 32000])
@pytest.mark.parametrize("temperature,top_k,top_p,min_p", [
    (1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.0), (0.7, 50, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 40, 0.9, 0.02), (5.0, 2000, 0.99, 0.0),
    (0.01, 3, 0.3, 0.5), (1.0, 1, 1.0, 1.0)])
def test_sampling_against_the_definition(dtype, vocab, temperature, top_k, top_p, min_p):
    _, _, sample = _ops()
    rows = 12 if vocab > 5000 else 40
    g = torch.Generator().manual_seed(vocab)
    x, u = _logits(rows, vocab, dtype, g), torch.rand(rows, generator=g)
    u[7], u[8] = 0.0, 1.0 - 2.0 ** -24
    want = [draw_token(x[r], float(u[r]), temperature, top_k, top_p, min_p) for r in range(rows)]
    got = sample(x.cuda(), u.cuda(), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    assert got.dtype == torch.int64 and got.tolist() == want
    every = {k: torch.full((rows,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device="cuda")
             for k, v in dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).items()}
    assert torch.equal(sample(x.cuda(), u.cuda(), **every), got)                 # one setting for all, or the same for every row


@pytest.mark.parametrize("rows,vocab,dtype", [(1, 128256, torch.float32), (3, 262144, torch.bfloat16), (4, 50257, torch.bfloat16), (200, 1000, torch.float32)])
def test_sampling_rows_with_their_own_settings(rows, vocab, dtype):
    _, _, sample = _ops()
    g = torch.Generator().manual_seed(rows)
    x, u = _logits(rows, vocab, dtype, g), torch.rand(rows, generator=g, dtype=torch.float64)
    pick = lambda v, t: torch.tensor(v, dtype=t)[torch.randint(0, len(v), (rows,), generator=g)]             # noqa: E731
    t, k = pick([0.0, 0.5, 1.0, 2.0, -1.0], torch.float32), pick([0, 1, 30, 500, vocab, vocab + 7, -3], torch.int32)
    p, m = pick([1.0, 0.9, 0.2, 1e-9, 0.0, 2.0], torch.float32), pick([0.0, 0.1, 1.0, 3.0], torch.float32)
    wide = torch.full((rows, vocab + 3), 99.0, dtype=dtype)                      # rows are a slice of a padded matrix
    wide[:, 1:vocab + 1] = x
    got = sample(wide.cuda()[:, 1:vocab + 1], u.cuda(), temperature=t.cuda(), top_k=k.cuda(), top_p=p.cuda(), min_p=m.cuda())
    want = [draw_token(x[r], float(u[r]), float(t[r]), int(k[r]), max(1e-300, float(p[r])), float(m[r])) for r in range(rows)]
    assert got.tolist() == want


@pytest.mark.parametrize("temperature", [1e-45, 1e-6, 1e30, 3e38])
@pytest.mark.parametrize("top_k,top_p,min_p", [(0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.7, 0.0), (900, 0.5, 0.3)])
def test_sampling_extreme_temperatures(temperature, top_k, top_p, min_p):
    _, _, sample = _ops()
    g = torch.Generator().manual_seed(4)
    x, u = _logits(9, 2000, torch.float32, g), torch.rand(9, generator=g)
    want = [draw_token(x[r], float(u[r]), temperature, top_k, top_p, min_p) for r in range(9)]
    assert sample(x.cuda(), u.cuda(), temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).tolist() == want


def test_sampling_many_near_ties():
    """Logits that lie within a few steps of the finest histogram, and an all-but-equal row over its list's length."""
    _, _, sample = _ops()
    g = torch.Generator().manual_seed(5)
    x = torch.randn(6, 30000, generator=g) * 1e-4 + torch.tensor([0.0, 1.0, -3.0, 100.0, 1e-3, 7.0])[:, None]
    u = torch.rand(6, generator=g)
    for kw in (dict(top_k=15000), dict(top_p=0.5), dict(top_k=20000, top_p=0.3), dict(min_p=0.9999)):
        want = [draw_token(x[r], float(u[r]), 1.0, kw.get("top_k", 0), kw.get("top_p", 1.0), kw.get("min_p", 0.0)) for r in range(6)]
        assert sample(x.cuda(), u.cuda(), **kw).tolist() == want, kw


def test_sampling_frequencies():
    """Evenly spaced numbers give every token its share: counts differ from rows * p by one at most."""
    _, _, sample = _ops()
    rows, vocab = 4096, 50
    x = torch.randn(vocab, generator=torch.Generator().manual_seed(6))
    u = (torch.arange(rows) + 0.5) / rows
    got = sample(x.cuda().expand(rows, vocab), u.cuda(), temperature=0.9)
    share = torch.softmax(x.double() / 0.9, -1) * rows
    assert ((torch.bincount(got.cpu(), minlength=vocab) - share).abs() <= 1.0 + 1e-9).all()
    assert (got[1:] >= got[:-1]).all()


def test_sampling_numbers_outside_the_unit_interval():
    _, _, sample = _ops()
    x = torch.zeros(5, 9, device="cuda")
    x[:, 8] = -float("inf")
    u = torch.tensor([-1.0, 1.0, 7.0, float("nan"), float("inf")], device="cuda")
    assert sample(x, u).tolist() == [0, 7, 7, 0, 7]
    assert sample(x, u.double()).tolist() == [0, 7, 7, 0, 7]


# -------------------------------------------------------------------------------------------------- together, refusals
def _decode_state(device="cuda", dtype=torch.float16, seed=7):
    g = torch.Generator().manual_seed(seed)
    B, H, hkv, D, page, V = 5, 8, 2, 64, 16, 1000
    lengths = [40, 0, 100, 16, 31]
    kp, vp, table = paged_cache([n + 4 for n in lengths], hkv, page, D, dtype, device, g)
    head = (torch.randn(H * D, V, generator=g) * 0.1).to(dtype).to(device)
    qkv = torch.randn(B, (H + 2 * hkv) * D, generator=g).to(dtype).to(device)
    return dict(H=H, hkv=hkv, D=D, kp=kp, vp=vp, table=table, head=head, qkv=qkv, pos=torch.tensor(lengths, dtype=torch.int32, device=device),
                inv=(10000.0 ** (-torch.arange(D // 2).double() * 2 / D)).float().to(device), u=torch.rand(B, generator=g).to(device))


def _decode(s, ops):
    """One decode step of a model with one layer: append, attend, project, draw."""
    append, attention, sample = ops
    q, k, v = (x.unflatten(1, (-1, s["D"])) for x in s["qkv"].split([s["H"] * s["D"], s["hkv"] * s["D"], s["hkv"] * s["D"]], 1))
    q = append(q, k, v, s["kp"], s["vp"], s["table"], s["pos"], None, s["inv"])
    att = attention(q, s["kp"], s["vp"], s["table"], s["pos"] + 1)
    return att, sample((att.flatten(1) @ s["head"]).float(), s["u"], temperature=0.8, top_k=50, top_p=0.9)


def test_decode_step_eager_captured_and_on_another_stream():
    """The three operators in a row; captured and replayed on new inputs; two captured graphs running at once; a side stream."""
    ops = _ops()
    s = _decode_state()
    att, tok = _decode(s, ops)
    q, k = (x.unflatten(1, (-1, 64)) for x in (s["qkv"][:, :512], s["qkv"][:, 512:640]))
    want_k = rotate(k.cpu(), s["pos"].cpu(), s["inv"].cpu(), False, None, 0.0)
    at = s["pos"].long()
    got_k = s["kp"][s["table"][torch.arange(5, device="cuda"), at // 16].long(), :, at % 16]
    _check(got_k, want_k, rotate_tolerance(want_k, torch.float16))
    rq = ops[0](q, k, k, s["kp"].clone(), s["vp"].clone(), s["table"], s["pos"], None, s["inv"])
    want, tol = attend(rq, s["kp"], s["vp"], s["table"], (s["pos"] + 1).cpu(), None, 0.125)
    _check(att, want, tol)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        att2, tok2 = _decode(s, ops)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(att, att2) and torch.equal(tok, tok2)

    states = [_decode_state(seed=8), _decode_state(seed=9)]
    expect = [_decode(_decode_state(seed=n), ops) for n in (8, 9)]
    graphs, outs = [], []
    for st in states:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(_decode(st, ops))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for st, graph in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    for (a, t), (wa, wt) in zip(outs, expect):
        assert torch.equal(a, wa) and torch.equal(t, wt)
    # a replay on other inputs of the same graph
    for st, src in zip(states, (9, 8)):
        new = _decode_state(seed=src)
        for key in ("qkv", "kp", "vp", "table", "pos", "u", "head"):
            st[key].copy_(new[key])
    for graph in graphs:
        graph.replay()
    for (a, t), (wa, wt) in zip(outs, reversed(expect)):
        assert torch.equal(a, wa) and torch.equal(t, wt)


def test_captured_and_eager_calls_at_once():
    """Long sequences, so that the length is split: a graph replays on one stream while eager calls run on two others."""
    _, attention, _ = _ops()
    sets = []
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        kp, vp, table = paged_cache([9000, 3000], 1, 16, 64, torch.float16, "cuda", g)
        q = torch.randn(2, 2, 64, generator=g).half().cuda()
        sets.append((q, kp, vp, table, _i32([9000, 3000])))
    want = [attention(*s) for s in sets]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = attention(*sets[0])
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(30):
        with torch.cuda.stream(streams[0]):
            graph.replay()
        for i in (0, 1):
            with torch.cuda.stream(streams[i + 1]):
                got[i].append(attention(*sets[i + 1]))
    torch.cuda.synchronize()
    assert torch.equal(captured, want[0])
    assert all(torch.equal(x, want[1]) for x in got[0]) and all(torch.equal(x, want[2]) for x in got[1])


def test_first_call_of_a_process_inside_a_capture():
    """Nothing has to run before a capture: what the kernels allocate once per process is allocated there."""
    code = """
import torch
from rustorch_b200 import _native
from rustorch_b200.ops.paged import paged_append, paged_attention
from rustorch_b200.ops.sampling import sample_tokens
x = torch.randn(1, 2, 64, device="cuda").half()
kp, vp = torch.zeros(2, 2, 16, 64, device="cuda").half(), torch.zeros(2, 2, 16, 64, device="cuda").half()
i = torch.zeros(1, dtype=torch.int32, device="cuda")
table, inv, u, one = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(32, device="cuda"), torch.full((1,), 0.5, device="cuda"), i + 1
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    q = paged_append(x, x, x, kp, vp, table, i, i, inv)
    out = paged_attention(q, kp, vp, table, one, i)
    tok = sample_tokens(out.flatten(1), u, temperature=0.0)
g.replay()
torch.cuda.synchronize()
_native.check_status()
assert torch.equal(out, x) and int(tok) == int(x.argmax())
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-800:]


def test_empty_calls():
    append, attention, sample = _ops()
    kp = torch.zeros(1, 2, 16, 64, dtype=torch.half, device="cuda")
    q, none, table = torch.empty(0, 4, 64, dtype=torch.half, device="cuda"), _i32([]), torch.zeros(0, 0, dtype=torch.int32, device="cuda")
    assert append(q, q[:, :2], q[:, :2], kp, kp.clone(), table, none, none, torch.zeros(32, device="cuda")).shape == (0, 4, 64)
    assert attention(q, kp, kp, table, none, none).shape == (0, 4, 64)
    assert sample(torch.empty(0, 9, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)
    no_pages = torch.empty(0, 2, 16, 64, dtype=torch.half, device="cuda")        # a cache that has no page yet
    assert float(attention(q.new_ones(1, 4, 64), no_pages, no_pages, torch.zeros(1, 0, dtype=torch.int32, device="cuda"), _i32([0])).abs().max()) == 0.0


def test_indices_out_of_range_are_reported_and_skipped():
    from rustorch_b200 import _native
    from rustorch_b200.error import IndexOutOfBounds
    append, attention, _ = _ops()
    kp = torch.zeros(2, 1, 16, 64, dtype=torch.half, device="cuda")
    vp = torch.zeros_like(kp)
    table = _i32([[1, -1, 2]])
    x = torch.ones(1, 1, 64, dtype=torch.half, device="cuda")
    inv = torch.ones(32, device="cuda")
    for pos, seq in ((16, 0), (32, 0), (48, 0), (-1, 0), (0, 1), (0, -2), (2 ** 31 - 1, 0)):
        out = append(x, x, x, kp, vp, table, _i32([pos]), _i32([seq]), inv)
        with pytest.raises(IndexOutOfBounds):
            _native.check_status()
        assert float(kp.abs().max()) == 0.0 and float(vp.abs().max()) == 0.0 and float(out.abs().max()) == 0.0
    for length, seq in ((17, 0), (40, 0), (49, 0), (-1, 0), (1, 1), (1, -2), (2 ** 31 - 1, 0)):
        out = attention(x, kp, vp, table, _i32([length]), _i32([seq]))
        with pytest.raises(IndexOutOfBounds):
            _native.check_status()
        assert bool(torch.isfinite(out).all())
    assert float(append(x, x, x, kp, vp, table, _i32([5]), _i32([-1]), inv).abs().max()) == 0.0 and float(kp.abs().max()) == 0.0
    append(x, x, x, kp, vp, table, _i32([5]), _i32([0]), inv)
    _native.check_status()
    assert float(kp[1, 0, 5].abs().max()) > 0.0


def test_refusals_on_the_device():
    append, attention, sample = _ops()
    kp = torch.zeros(2, 2, 4, 64, dtype=torch.half, device="cuda")
    table, i1 = _i32([[0, 1]]), _i32([1])
    q, k = torch.zeros(1, 4, 64, dtype=torch.half, device="cuda"), torch.zeros(1, 2, 64, dtype=torch.half, device="cuda")
    good = dict(q=q, k_pages=kp, v_pages=kp, block_table=table, kv_len=i1, seq=i1 * 0)
    attention(**good)
    odd = torch.zeros(kp.numel() + 1, dtype=torch.half, device="cuda")[1:].view(kp.shape)
    for kw in (dict(q=q.float()), dict(q=q.bfloat16()), dict(q=q[:, :3]), dict(q=q[0]), dict(q=q.cpu()), dict(kv_len=i1.long()), dict(kv_len=i1.cpu()),
               dict(seq=_i32([0, 0])), dict(block_table=table.long()), dict(block_table=table[0]), dict(k_pages=odd, v_pages=odd),
               dict(v_pages=kp.transpose(1, 2).contiguous().transpose(1, 2)), dict(k_pages=kp[:1]), dict(window=-1), dict(softcap=-1.0),
               dict(softcap=float("inf")), dict(softcap=1e-9), dict(scale=float("nan")), dict(scale=1e31), dict(out=torch.zeros(1, 4, 64, device="cuda")), dict(out=k),
               dict(out=q[:, :1].expand(-1, 4, -1)), dict(q=torch.zeros(1, 4, 60, dtype=torch.half, device="cuda")),
               dict(q=torch.zeros(1, 4, 320, dtype=torch.half, device="cuda"), k_pages=torch.zeros(2, 2, 4, 320, dtype=torch.half, device="cuda"),
                    v_pages=torch.zeros(2, 2, 4, 320, dtype=torch.half, device="cuda"))):
        with pytest.raises(RuntimeError):
            attention(**{**good, **kw})
    good = dict(q=q, k=k, v=k, k_pages=kp, v_pages=kp.clone(), block_table=table, pos=i1, seq=i1 * 0, inv_freq=torch.zeros(32, device="cuda"))
    append(**good)
    for kw in (dict(q=q.float()), dict(k=q), dict(v=k.bfloat16()), dict(pos=i1.long()), dict(seq=i1.cpu()), dict(inv_freq=torch.zeros(33, device="cuda")),
               dict(inv_freq=torch.zeros(32, device="cuda").double()), dict(q_norm=torch.ones(32, dtype=torch.half, device="cuda")),
               dict(k_norm=torch.ones(64, device="cuda")), dict(eps=-1.0), dict(q_out=k), dict(q_out=q[:, :1].expand(-1, 4, -1)), dict(k_out=q),
               dict(k_pages=kp[:1].expand(2, -1, -1, -1), v_pages=kp[:1].expand(2, -1, -1, -1))):
        with pytest.raises(RuntimeError):
            append(**{**good, **kw})
    x, u = torch.zeros(2, 9, device="cuda"), torch.zeros(2, device="cuda")
    for kw in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.t()), dict(uniform=u.half()), dict(uniform=u[:1]), dict(uniform=u.cpu()),
               dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=1e39), dict(top_k=-1), dict(top_p=0.0), dict(top_p=1.1),
               dict(min_p=2.0),
               dict(temperature=u.double()), dict(top_k=u), dict(top_p=u[:1]), dict(min_p=u.cpu()),
               dict(logits=torch.zeros(2, 262145, device="cuda"))):
        with pytest.raises(RuntimeError):
            sample(**{**dict(logits=x, uniform=u), **kw})
