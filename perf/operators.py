"""Measured cases of the token-serving operators: appending rotated keys and values to a paged cache, attention of new
tokens over that cache, and drawing the next token from given random numbers.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits, in 64 where positions are far or a
value may lie next to a border), or, where ``own`` is true, through the entry points of ``rustorch_b200.ops``.
"""
import functools
import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------------------------- cases
def _append(name, dtype, n_seq, new, start, heads, kv_heads, dim, rot, page, interleaved, norm):
    return dict(name=name, op="append", dtype=dtype, n_seq=n_seq, new=new, start=start, heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                page=page, interleaved=interleaved, norm=norm)


def _attend(name, dtype, n_seq, new, min_len, max_len, heads, kv_heads, dim, page, window=0, softcap=0.0):
    return dict(name=name, op="attend", dtype=dtype, n_seq=n_seq, new=new, min_len=min_len, max_len=max_len, heads=heads, kv_heads=kv_heads,
                dim=dim, page=page, window=window, softcap=softcap)


def _sample(name, dtype, rows, vocab, temperature, top_k, top_p, min_p, mixed=False):
    return dict(name=name, op="sample", dtype=dtype, rows=rows, vocab=vocab, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                mixed=mixed)


def listed():
    return [
        # one new token of one conversation (32 heads of 128, adjacent pairs as GGUF weights rotate): latency alone
        _append("append 1 token", "fp16", 1, 1, 41, 32, 32, 128, 128, 16, True, False),
        # four prompts at once on a grouped-query model whose queries and keys are normalised per head
        _append("append 8192 tokens", "bf16", 4, 2048, 0, 32, 8, 128, 128, 64, False, True),
        # pieces of 37 prompts late in a long context: 64-wide heads of which half rotate, pages of 24
        _append("append 777 tokens, odd", "fp16", 37, 21, 100003, 12, 12, 64, 32, 24, False, False),
        # a chat's first answers: one sequence, few keys, as many key heads as query heads
        _attend("attend 1 x 77", "fp16", 1, 1, 77, 77, 32, 32, 128, 16),
        # one user with a long document: the cache's length is the only axis to split
        _attend("attend 1 x 131071", "bf16", 1, 1, 131071, 131071, 32, 8, 128, 64),
        # a server's batch: 64 sequences of very different ages
        _attend("attend 64 ragged", "fp16", 64, 1, 1, 8192, 32, 8, 128, 16),
        # a small decoder of 12 heads of 64 in a large batch, up to its whole context
        _attend("attend 96 x 12 heads", "bf16", 96, 1, 5, 1024, 12, 12, 64, 32),
        # three proposed tokens a sequence, seven queries a key head, 80 wide, a window and capped scores; one sequence is new and empty
        _attend("attend window, cap", "bf16", 29, 3, 0, 2500, 14, 2, 80, 24, 1000, 30.0),
        # the next token of one conversation, with the usual filters
        _sample("sample 1 x 32000", "fp32", 1, 32000, 0.8, 50, 0.9, 0.0),
        # a server's batch with a nucleus and a floor under the probabilities
        _sample("sample 256 x 128256", "fp32", 256, 128256, 0.9, 0, 0.95, 0.01),
        # draws from the whole distribution: an odd vocabulary in 16 bits, where many logits tie
        _sample("sample 64 x 50257", "bf16", 64, 50257, 1.0, 0, 1.0, 0.0),
        # requests with settings of their own, greedy ones among them
        _sample("sample 37 mixed", "fp16", 37, 32000, 1.0, 0, 1.0, 0.0, True),
    ]


def draw(rng):
    def spread(lo, hi):
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    op = rng.choice(("append", "attend", "sample"))
    if op == "sample":
        vocab = spread(300, 128256)
        rows = spread(1, max(1, min(256, 33_000_000 // vocab)))
        mixed = rng.random() < 0.3
        c = _sample("", rng.choice(("fp32", "fp32", "bf16", "fp16")), rows, vocab, round(rng.uniform(0.3, 1.5), 2), rng.choice((0, 0, spread(1, 2000))),
                    rng.choice((1.0, round(rng.uniform(0.3, 0.99), 2))), rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 3))), mixed)
    else:
        kv_heads = rng.choice((1, 2, 3, 4, 8, 12))
        heads = kv_heads * rng.choice((1, 2, 4, 5, 7, 8))
        dim = rng.choice((32, 64, 80, 96, 128, 128, 192, 256))
        page = rng.choice((8, 16, 16, 24, 32, 64, 128))
        dtype = rng.choice(("fp16", "bf16"))
        if op == "append":
            new = spread(1, 2048)
            n_seq = spread(1, max(1, 8192 * 12288 // (new * dim * (heads + 2 * kv_heads) * 2)))
            rot = rng.choice((dim, dim, dim // 2))
            c = _append("", dtype, min(n_seq, 256), new, rng.choice((0, spread(1, 120000))), heads, kv_heads, dim, rot, page, rng.random() < 0.5,
                        rng.random() < 0.5)
        else:
            length = spread(1, 131072)
            new = rng.choice((1, 1, 1, 2, 4))
            n_seq = spread(1, max(1, min(128, 64 * 8192 * 8 * 128 // (length * new * kv_heads * dim * 3))))
            c = _attend("", dtype, n_seq, new, rng.choice((0, 1, length)), length, heads, kv_heads, dim, page, rng.choice((0, 0, spread(1, 4096))),
                        rng.choice((0.0, 0.0, 20.0, 50.0)))
    del c["name"]
    return c


def _lengths(case):
    """Cache lengths of the sequences, the longest last: few old ones, many young ones."""
    n, lo, hi = case["n_seq"], case["min_len"], case["max_len"]
    return [lo + int((hi - lo) * ((i + 1) / n) ** 2) if n > 1 else hi for i in range(n)]


def _visible(case):
    """(keys that each sequence's tokens read in all, keys summed over the tokens)."""
    distinct = total = 0
    for length in _lengths(case):
        lens = [max(0, length - j) for j in range(case["new"])]
        lows = [max(0, x - case["window"]) if case["window"] else 0 for x in lens]
        distinct += max(0, lens[0] - lows[-1])
        total += sum(x - y for x, y in zip(lens, lows))
    return distinct, total


def work(case):
    if case["op"] == "append":
        n, h, hkv, d = case["n_seq"] * case["new"], case["heads"], case["kv_heads"], case["dim"]
        return {"bytes": 2 * d * n * (2 * h + 4 * hkv) + 8 * n + 2 * case["rot"],
                "flops": n * (h + hkv) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    if case["op"] == "attend":
        distinct, total = _visible(case)
        n = case["n_seq"] * case["new"]
        return {"bytes": 4 * case["kv_heads"] * case["dim"] * distinct + 4 * n * case["heads"] * case["dim"] + 8 * n,
                "flops": 4 * case["heads"] * case["dim"] * total}
    size = 4 if case["dtype"] == "fp32" else 2
    return {"bytes": case["rows"] * (case["vocab"] * size + 12), "flops": 4 * case["rows"] * case["vocab"]}


# --------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device=dev, generator=g, dtype=torch.float32)

    if case["op"] == "sample":
        b, v = case["rows"], case["vocab"]
        # a bulk of unlikely tokens and a few dozen that stand out, as a language model's logits do
        logits = randn(b, v) * 2.0
        top = torch.randint(0, v, (b, 40), device=dev, generator=g)
        logits.scatter_add_(1, top, 4.0 + 3.0 * torch.rand(b, 40, device=dev, generator=g))
        st = dict(logits=logits.to(dt), uniform=torch.rand(b, device=dev, generator=g))
        if case["mixed"]:
            def pick(values, dtype):
                return torch.tensor(values, device=dev, dtype=dtype)[torch.randint(0, len(values), (b,), device=dev, generator=g)]
            st.update(temperature=pick([0.0, 0.7, 1.0, 1.3], torch.float32), top_k=pick([0, 1, 40, 200, v], torch.int32),
                      top_p=pick([1.0, 0.9, 0.5], torch.float32), min_p=pick([0.0, 0.05], torch.float32))
        else:
            st.update({k: case[k] for k in ("temperature", "top_k", "top_p", "min_p")})
        return dict(case=case, **st)

    page, hkv, d, new, n_seq = case["page"], case["kv_heads"], case["dim"], case["new"], case["n_seq"]
    if case["op"] == "append":
        first, last = case["start"] // page, (case["start"] + new - 1) // page          # only pages that are written exist
        per = last - first + 1
        n_pages = n_seq * per + 3
        table = torch.full((n_seq, last + 1), -1, device=dev, dtype=torch.int32)
        table[:, first:] = torch.randperm(n_pages, device=dev, generator=g)[: n_seq * per].view(n_seq, per).to(torch.int32)
        lengths = None
    else:
        lengths = torch.tensor(_lengths(case))[torch.randperm(n_seq, generator=torch.Generator().manual_seed(seed))]
        need = (lengths + page - 1) // page
        ends = need.cumsum(0)
        n_pages = int(ends[-1]) + 3
        table = torch.full((n_seq, max(1, int(need.max()))), -1, dtype=torch.int32)
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed + 1)).to(torch.int32)
        table[torch.arange(table.shape[1])[None] < need[:, None]] = order[: int(ends[-1])]
        table = table.to(dev)
    k_pages = randn(n_pages, hkv, page, d).to(dt)
    v_pages = randn(n_pages, hkv, page, d).to(dt)
    seq = torch.arange(n_seq, device=dev, dtype=torch.int32).repeat_interleave(new)
    st = dict(case=case, k_pages=k_pages, v_pages=v_pages, table=table, seq=seq)
    n, h = n_seq * new, case["heads"]
    if case["op"] == "attend":
        back = torch.arange(new - 1, -1, -1)
        st["kv_len"] = (lengths[:, None] - back[None]).clamp_min(0).reshape(-1).to(dev, torch.int32)
        st["q"] = randn(n, h, d).to(dt)
        return st
    # q | k | v are slices of one projection's output, as a model has them
    qkv = randn(n, (h + 2 * hkv) * d).to(dt)
    st["q"] = qkv[:, : h * d].view(n, h, d)
    st["k"] = qkv[:, h * d: (h + hkv) * d].view(n, hkv, d)
    st["v"] = qkv[:, (h + hkv) * d:].view(n, hkv, d)
    st["pos"] = (case["start"] + torch.arange(new, device=dev)).to(torch.int32).repeat(n_seq)
    st["inv_freq"] = (500000.0 ** (-torch.arange(case["rot"] // 2, dtype=torch.float64) * 2.0 / case["rot"])).float().to(dev)
    st["q_norm"] = (1.0 + 0.1 * randn(d)).to(dt) if case["norm"] else None
    st["k_norm"] = (1.0 + 0.1 * randn(d)).to(dt) if case["norm"] else None
    return st


# ------------------------------------------------------------------------------------------------------------ operators
@functools.lru_cache(None)
def _framework():
    from rustorch_b200.ops import paged, sampling
    return paged.paged_append, paged.paged_attention, sampling.sample_tokens


def run(st):
    c = st["case"]
    if c["op"] == "append":
        if own:
            q = _framework()[0](st["q"], st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["pos"], st["seq"], st["inv_freq"],
                                interleaved=c["interleaved"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=1e-6)
        else:
            q = _plain_append(st, c)
        return dict(q=q, k_pages=st["k_pages"], v_pages=st["v_pages"])
    if c["op"] == "attend":
        if own:
            return _framework()[1](st["q"], st["k_pages"], st["v_pages"], st["table"], st["kv_len"], st["seq"], window=c["window"],
                                   softcap=c["softcap"])
        return _plain_attend(st, c)
    if own:
        return _framework()[2](st["logits"], st["uniform"], temperature=st["temperature"], top_k=st["top_k"], top_p=st["top_p"],
                               min_p=st["min_p"])
    return _plain_sample(st)


def _plain_append(st, c):
    rot = c["rot"]
    ang = st["pos"].double()[:, None, None] * st["inv_freq"].double()
    cs, sn = ang.cos().float(), ang.sin().float()

    def turn(x, w):
        xf = x.float()
        if w is not None:
            xf = xf * torch.rsqrt((xf * xf).mean(-1, keepdim=True) + 1e-6) * w.float()
        head, rest = xf[..., :rot], xf[..., rot:]
        if c["interleaved"]:
            a, b = head[..., 0::2], head[..., 1::2]
            head = torch.stack([a * cs - b * sn, a * sn + b * cs], -1).flatten(-2)
        else:
            a, b = head[..., : rot // 2], head[..., rot // 2:]
            head = torch.cat([a * cs - b * sn, a * sn + b * cs], -1)
        return torch.cat([head, rest], -1).to(x.dtype)

    pos = st["pos"].long()
    page = st["table"][st["seq"].long(), pos // c["page"]].long()
    st["k_pages"][page, :, pos % c["page"]] = turn(st["k"], st["k_norm"])
    st["v_pages"][page, :, pos % c["page"]] = st["v"]
    return turn(st["q"], st["q_norm"])


def _plain_attend(st, c):
    n, hkv, d = st["q"].shape[0], c["kv_heads"], c["dim"]
    pages = st["table"].long().clamp_min(0)
    length = pages.shape[1] * c["page"]
    k = st["k_pages"][pages].float().transpose(1, 2).reshape(-1, 1, hkv, length, d)               # [n_seq, 1, Hkv, L, D]
    v = st["v_pages"][pages].float().transpose(1, 2).reshape(-1, 1, hkv, length, d)
    q = st["q"].float().view(c["n_seq"], c["new"], hkv, -1, d)                                    # the tokens come by sequence
    s = (q @ k.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    if c["softcap"]:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    at = torch.arange(length, device=s.device)
    end = st["kv_len"].long().view(c["n_seq"], c["new"], 1)
    seen = at < end
    if c["window"]:
        seen = seen & (at >= end - c["window"])
    seen = seen[:, :, None, None]
    s = s.masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    out = (p @ v) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.reshape(n, -1, d).to(st["q"].dtype)


def _plain_sample(st):
    logits = st["logits"].double()
    b, v = logits.shape
    dev = logits.device

    def column(x):
        return torch.as_tensor(x, device=dev).double().expand(b)[:, None]
    temp, top_k, top_p, min_p = (column(st[k]) for k in ("temperature", "top_k", "top_p", "min_p"))
    sorted_l, order = logits.sort(dim=-1, descending=True, stable=True)                               # equal logits: lowest index first
    greedy = temp == 0
    w = torch.exp((sorted_l - sorted_l[:, :1]) / torch.where(greedy, 1.0, temp))
    keep = (top_k <= 0) | (torch.arange(v, device=dev)[None] < top_k)
    w = torch.where(keep, w, 0.0)
    cum = w.cumsum(-1)
    keep = keep & ((top_p >= 1) | (cum - w < top_p * cum[:, -1:])) & (w >= min_p)
    mass = torch.zeros_like(w).scatter_(-1, order, torch.where(keep, w, 0.0)).cumsum(-1)
    last = torch.where(torch.zeros_like(keep).scatter_(-1, order, keep), torch.arange(v, device=dev)[None], -1).amax(-1, keepdim=True)
    token = torch.searchsorted(mass, st["uniform"].double()[:, None] * mass[:, -1:], right=True)
    return torch.where(greedy, order[:, :1], torch.minimum(token, last)).squeeze(1)


# ------------------------------------------------------------------------------------------------ definitions in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "append":
        half = case["rot"] // 2
        phase = torch.exp(1j * (st["pos"].double()[:, None] * st["inv_freq"].double()))[:, None]  # [n, 1, rot / 2]

        def turn(x, w):
            y = x.double()
            if w is not None:
                y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / case["dim"] + 1e-6) * w.double()
            even, odd = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["interleaved"] else (slice(0, half), slice(half, 2 * half))
            z = torch.complex(y[..., even], y[..., odd]) * phase
            y[..., even], y[..., odd] = z.real, z.imag
            return y
        k_pages, v_pages = st["k_pages"].double(), st["v_pages"].double()
        k = turn(st["k"], st["k_norm"])
        tables, page = st["table"].tolist(), case["page"]
        for s in range(case["n_seq"]):
            at, end, row = case["start"], case["start"] + case["new"], s * case["new"]
            while at < end:                                                                       # one page at a time
                m = min(end, (at // page + 1) * page) - at
                p = tables[s][at // page]
                k_pages[p, :, at % page: at % page + m] = k[row: row + m].transpose(0, 1)
                v_pages[p, :, at % page: at % page + m] = st["v"][row: row + m].double().transpose(0, 1)
                at, row = at + m, row + m
        return dict(q=turn(st["q"], st["q_norm"]), k_pages=k_pages, v_pages=v_pages)
    if case["op"] == "attend":
        q, group = st["q"].double(), case["heads"] // case["kv_heads"]
        out = torch.zeros_like(q)
        for t, (length, s) in enumerate(zip(st["kv_len"].tolist(), st["seq"].tolist())):
            low = max(0, length - case["window"]) if case["window"] else 0
            if length <= low:
                continue
            at = torch.arange(low, length, device=q.device)
            page = st["table"][s].long()[at // case["page"]]
            k = st["k_pages"][page, :, at % case["page"]].double()                                # [keys, Hkv, D]
            v = st["v_pages"][page, :, at % case["page"]].double()
            for h in range(case["kv_heads"]):
                x = q[t, h * group: (h + 1) * group] @ k[:, h].T / math.sqrt(case["dim"])
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                out[t, h * group: (h + 1) * group] = torch.softmax(x, -1) @ v[:, h]
        return out
    logits, u = st["logits"].double().cpu().numpy(), st["uniform"].double().cpu().numpy()
    b, v = logits.shape
    temp, top_k, top_p, min_p = (np.broadcast_to(st[k].double().cpu().numpy() if torch.is_tensor(st[k]) else float(st[k]), (b,))
                                 for k in ("temperature", "top_k", "top_p", "min_p"))
    tokens = np.zeros(b, np.int64)
    for i in range(b):
        x = logits[i]
        best = int(np.argmax(x))
        if temp[i] == 0:
            tokens[i] = best
            continue
        x = np.exp((x - x[best]) / temp[i])
        ranked = np.lexsort((np.arange(v), -logits[i]))[: int(top_k[i]) if top_k[i] > 0 else v]
        if top_p[i] < 1:
            before = np.concatenate([[0.0], np.cumsum(x[ranked])])
            ranked = ranked[: int(np.count_nonzero(before[:-1] < top_p[i] * before[-1]))]
        kept = np.sort(ranked[x[ranked] >= min_p[i]])
        mass = np.cumsum(x[kept])
        tokens[i] = kept[min(len(kept) - 1, int(np.count_nonzero(mass <= u[i] * mass[-1])))]
    return torch.from_numpy(tokens)
