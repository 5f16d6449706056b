"""64-bit definitions of the paged-cache and sampling operators, and inputs for their tests."""
import math

import torch


def half_step(dtype) -> float:
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def rotate(x, pos, inv_freq, interleaved, weight, eps):
    """RMSNorm (when ``weight`` is given) and rotation of ``x [n, heads, D]`` in 64 bits."""
    y = x.double().clone()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
    half = inv_freq.numel()
    for t in range(x.shape[0]):
        for i in range(half):
            angle = int(pos[t]) * float(inv_freq[i])
            ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            a, b = y[t, :, ia].clone(), y[t, :, ib].clone()
            y[t, :, ia] = a * math.cos(angle) - b * math.sin(angle)
            y[t, :, ib] = a * math.sin(angle) + b * math.cos(angle)
    return y


def rotate_tolerance(ref, dtype):
    """One rounding to ``dtype`` (subnormals: half of the smallest step), and 32-bit arithmetic before it: norm, weight, two
    products and functions of one angle are below 16 roundings of 2^-24 on values no larger than the head's largest pair."""
    smallest = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    return half_step(dtype) * ref.abs() + smallest + 16 * 2.0 ** -24 * 1.5 * ref.abs().amax(-1, keepdim=True)


def attend(q, k_pages, v_pages, table, kv_len, seq, scale, window=0, softcap=0.0):
    """Attention in 64 bits and the tolerance of a 16-bit kernel's answer, both ``[n, H, D]``."""
    n, H, D = q.shape
    hkv, page = k_pages.shape[1:3]
    out, tol = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    q, k_pages, v_pages, table = q.cpu(), k_pages.cpu(), v_pages.cpu(), table.cpu()
    unit = half_step(q.dtype)
    for t in range(n):
        s, length = t if seq is None else int(seq[t]), int(kv_len[t])
        low = max(0, length - window) if window else 0
        if s < 0 or length <= low:
            continue
        at = torch.arange(low, length)
        pages = table[s, at // page].long()
        for h in range(H):
            k, v = (x[pages, h // (H // hkv), at % page].double() for x in (k_pages, v_pages))
            x = (k @ q[t, h].double()) * scale
            off = (k.abs() @ q[t, h].double().abs()).max() * abs(scale) * (D + 4) * 2.0 ** -24
            if softcap:
                x, off = softcap * torch.tanh(x / softcap), off + softcap * 2.0 ** -21
            p = torch.softmax(x, -1)
            out[t, h] = p @ v
            mean = p @ v.abs()
            # the result's rounding; the weights' rounding to the value type; scores off by `off` in numerator and denominator; sums
            tol[t, h] = unit * out[t, h].abs() + mean * (unit + 2 * float(off) + (at.numel() ** 0.5 + 64) * 2.0 ** -23)
            if q.dtype == torch.float16:
                tol[t, h] += 2.0 ** -25                                          # half of the smallest fp16 step
    return out, tol


def draw_token(logits, u, temperature, top_k, top_p, min_p):
    """Token of one row of logits (any dtype) in 64 bits, by settings that are 32-bit numbers."""
    temperature, top_p, min_p = torch.tensor([temperature, top_p, min_p], dtype=torch.float32).tolist()
    l = [float(x) for x in logits.double()]
    l = [-math.inf if x != x else x for x in l]
    best = max(l)
    if best == -math.inf:
        return -1
    order = sorted(range(len(l)), key=lambda i: (-l[i], i))
    if not temperature > 0:
        return order[0]
    w = [1.0 if x == best else 0.0 if x == -math.inf else math.exp(max(-1000.0, (x - best) / temperature)) for x in l]
    w = [0.0 if x < 2.0 ** -46 else x for x in w]                                # the operator's resolution, part of its definition
    if top_k > 0:
        order = order[:top_k]
    if top_p < 1:
        mass, run, kept = math.fsum(w[i] for i in order), 0.0, []
        for i in order:
            if kept and run >= top_p * mass:
                break
            kept.append(i)
            run += w[i]
        order = kept
    kept = sorted(i for i in order if w[i] >= min(1.0, min_p))
    target = min(max(u, 0.0), 1.0 - 2.0 ** -53) * math.fsum(w[i] for i in kept)
    run = 0.0
    for i in kept:
        run += w[i]
        if run > target:
            return i
    return [i for i in kept if w[i] > 0][-1]


def paged_cache(lengths, hkv, page, D, dtype, device, gen, spare=3, layout="head"):
    """Pages with random contents in random order; rows behind each length, and spare pages, hold NaN or infinity."""
    need = [(n + page - 1) // page for n in lengths]
    n_pages = sum(need) + spare
    shape = (n_pages, hkv, page, D) if layout == "head" else (n_pages, page, hkv, D)
    k, v = (torch.randn(shape, generator=gen).to(dtype) for _ in range(2))
    if layout == "row":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    order = torch.randperm(n_pages, generator=gen).to(torch.int32)
    table = torch.full((len(lengths), max(1, max(need)) + 1), -1, dtype=torch.int32)
    used = 0
    for s, m in enumerate(need):
        table[s, :m] = order[used: used + m]
        used += m
        if lengths[s] % page:
            k[table[s, m - 1].long(), :, lengths[s] % page:] = float("nan")
            v[table[s, m - 1].long(), :, lengths[s] % page:] = float("inf")
    k[order[used:].long()] = float("nan")
    v[order[used:].long()] = float("nan")
    if layout == "row":                                                          # keep the strides on the device
        return k.transpose(1, 2).to(device).transpose(1, 2), v.transpose(1, 2).to(device).transpose(1, 2), table.to(device)
    return k.to(device), v.to(device), table.to(device)
