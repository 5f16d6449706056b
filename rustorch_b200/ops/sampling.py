"""Drawing the next token on the device from given random numbers (csrc/llm/sample_tokens.cu).

The reference's ``sample_token`` is a placeholder (example-cli/src/model/sampling.rs:8-300 returns ``vocab / 2``).
"""
from __future__ import annotations

import math
from typing import Union

import torch

from .. import _native

Setting = Union[float, int, torch.Tensor]


def sample_tokens(logits: torch.Tensor, uniform: torch.Tensor, *, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0) -> torch.Tensor:
    """One token for each row of ``logits [rows, vocab]`` (fp32, fp16 or bf16, up to 262144 tokens): int64 ``[rows]``.

    ``uniform``: fp32 or fp64 ``[rows]``, numbers in ``[0, 1)`` (others are moved to the nearest of these, NaN to 0).  With weights
    ``w = exp((l - max l) / temperature)`` and tokens ordered by logit (equal ones by index), ``top_k > 0`` keeps the first ``top_k``,
    ``top_p < 1`` of those the shortest prefix that holds ``top_p`` of their weight (one token at least), ``min_p`` what has at
    least ``min_p`` times the largest weight.  The token is the first one, in the vocabulary's order, at which the running sum
    of the kept weights exceeds ``uniform`` times their sum; it follows from the inputs alone, whatever the batch.

    Each setting is a number or a tensor with one value a row (int32 for ``top_k``, fp32 for the others; numbers are rounded to
    fp32, so both forms draw alike).  Temperature 0 takes the most likely token (lowest index of equals).  Logits of minus infinity and NaN are never drawn; a row that has no
    other gives -1.  Tokens of less than 1.4e-14 times the largest weight count as impossible.
    """
    scalars, rows = [], []
    for x in (temperature, top_k, top_p, min_p):
        tensor = isinstance(x, torch.Tensor)
        scalars.append(None if tensor else x)
        rows.append(x if tensor else None)
    t, k, p, m = scalars
    args = (logits, uniform, 1.0 if t is None else t, 0 if k is None else k, 1.0 if p is None else p, 0.0 if m is None else m,
            rows[0], rows[1], rows[2], rows[3])
    if logits.device.type == "cpu":
        return _sample_cpu(*args)
    return _native.load(required=True).sample_tokens(*args)


def _sample_cpu(logits, uniform, temperature, top_k, top_p, min_p, temperature_rows, top_k_rows, top_p_rows, min_p_rows):
    if logits.dim() != 2 or not 1 <= logits.shape[1] <= 262144 or not logits.is_floating_point():
        raise RuntimeError("sample_tokens: logits must be floating [rows, vocab] with 1 to 262144 tokens")
    rows, vocab = logits.shape
    for name, x, dtypes in (("uniform", uniform, (torch.float32, torch.float64)), ("temperature", temperature_rows, (torch.float32,)),
                            ("top_k", top_k_rows, (torch.int32,)), ("top_p", top_p_rows, (torch.float32,)), ("min_p", min_p_rows, (torch.float32,))):
        if x is not None and (x.dtype not in dtypes or x.shape != (rows,)):
            raise RuntimeError(f"sample_tokens: {name} must be one {' or '.join(map(str, dtypes))} a row")
    if not 0 <= temperature <= torch.finfo(torch.float32).max or top_k < 0 or not 0 < top_p <= 1 or not 0 <= min_p <= 1:
        raise RuntimeError("sample_tokens: temperature and top_k must not be negative, top_p in (0, 1], min_p in [0, 1]")
    temperature, top_p, min_p = torch.tensor([temperature, top_p, min_p], dtype=torch.float32).tolist()
    out = torch.empty(rows, dtype=torch.int64)
    for r in range(rows):
        l = logits[r].double().nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf)
        best = float(l.max())
        T = temperature if temperature_rows is None else float(temperature_rows[r])
        if best == -math.inf:
            out[r] = -1
            continue
        first = int((l == best).nonzero()[0])
        if not T > 0:
            out[r] = first
            continue
        w = torch.where(l == best, 1.0, torch.where(l == -math.inf, 0.0, torch.exp((l - best) / T)))
        w = torch.where(w < 2.0 ** -46, 0.0, w)
        order = torch.sort(l, descending=True, stable=True).indices
        k = top_k if top_k_rows is None else int(top_k_rows[r])
        order = order[:k] if 0 < k < vocab else order
        p = top_p if top_p_rows is None else float(top_p_rows[r])
        if p < 1:
            run = w[order].cumsum(0)
            order = order[: max(1, int((run - w[order] < p * run[-1]).sum()))]
        m = min(1.0, min_p if min_p_rows is None else float(min_p_rows[r]))
        kept = order[w[order] >= m].sort().values
        u = float(uniform[r])
        u = min(max(u, 0.0), 1.0) if u == u else 0.0
        run = w[kept].cumsum(0)
        at = int(torch.searchsorted(run, u * run[-1], right=True))
        if at >= len(kept):                                        # u = 1 (or a product that rounds up to the sum): the last possible token
            at = int((w[kept] > 0).nonzero()[-1])
        out[r] = kept[at]
    return out
