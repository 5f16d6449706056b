"""Paged attention on inputs whose answer is known to the last digits: what a rounding of weights or a lost key would change shows."""
import math

import pytest
import torch

from serving_reference import half_step

pytestmark = pytest.mark.gpu


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(keys, values, page, dtype):
    """One sequence's keys and values ``[n, D]`` as a cache of one head whose pages lie in reverse order."""
    n, D = keys.shape
    per = (n + page - 1) // page
    pages = torch.zeros(2, per * page, D)
    pages[0, :n], pages[1, :n] = keys, values
    k, v = pages.view(2, per, 1, page, D).flip(1).to(dtype).cuda()
    return k, v, torch.arange(per - 1, -1, -1, dtype=torch.int32, device="cuda")[None]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("s", [1.375, 2.0, 2.5, 4.25, 5.1875])
@pytest.mark.parametrize("heads,D", [(1, 64), (16, 128), (3, 256)])
def test_weights_keep_more_digits_than_the_values(dtype, s, heads, D):
    """One key of value 1 and about e^s keys of value -1 whose scores lie s below it: the two groups cancel, and what is left is off by
    half the relative error of the small weight.  A weight rounded once to 16 bits is off by more than the tolerance here."""
    n = round(math.exp(s))
    keys, values = torch.zeros(n + 1, D), -torch.ones(n + 1, D)
    keys[:, 0] = -s                                                              # exact in both types, as the product with 1 is
    keys[n // 2, 0], values[n // 2] = 0.0, 1.0
    w = math.exp(-s)
    want = (1 - n * w) / (1 + n * w)
    # the result's rounding; two roundings of a weight and a 32-bit exponential (2^-22 of it); scores of 32 bits, taken to base 2 and
    # subtracted, off by three half steps of 16; sums and one division
    unit = half_step(dtype)
    tol = unit * abs(want) + unit ** 2 + 2.0 ** -22 + 3 * 16 * 2.0 ** -24 + (n + 8) * 2.0 ** -24
    once = float(torch.tensor(16 * w).to(dtype)) / 16                            # the weight beside 16 for the largest, rounded once
    assert abs((1 - n * once) / (1 + n * w) - want) > 1.5 * tol
    from rustorch_b200.ops.paged import paged_attention
    q = torch.zeros(1, heads, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    out = paged_attention(q, *_pages(keys, values, 16, dtype), _i32([n + 1]), scale=1.0)
    assert float((out.double() - want).abs().max()) <= tol
