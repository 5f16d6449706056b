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


@pytest.mark.parametrize("n,heads,D,block", [(20003, 4, 128, 0), (20003, 16, 128, 0), (9001, 1, 64, 0), (40001, 8, 256, 0), (20003, 4, 128, 128), (9001, 1, 64, 48),
                                             (12345, 9, 192, 64)])
def test_every_key_of_a_split_sequence_counts_once(n, heads, D, block):
    """Key j holds 1 in place j mod D of its value and 0 elsewhere, its weight is 2^s with s = 0, 1 or 2 by blocks of keys (or 0
    everywhere): place d of the answer is the weight of the keys d, d + D, ... in the whole.  One key more or less moves a place by more
    than the tolerance, wherever the shares of the length are cut."""
    dtype = torch.float16
    at = torch.arange(n)
    s = at // block * 7 % 3 if block else torch.zeros(n, dtype=torch.long)
    keys, values = torch.zeros(n, D), torch.zeros(n, D)
    keys[:, 0], values[at, at % D] = s.float(), 1.0
    from rustorch_b200.ops.paged import paged_attention
    q = torch.zeros(1, heads, D, dtype=dtype, device="cuda")
    q[:, :, 0] = 1.0
    cache = _pages(keys, values, 64, dtype)
    for length in (n, n - 1, n - 65):
        weight = 2.0 ** s[:length].double()
        want = torch.zeros(D, dtype=torch.float64).index_add_(0, at[:length] % D, weight) / weight.sum()
        # the result's rounding (half of the smallest step below the normal numbers); weights whose scores are off by four roundings of
        # 2; 32-bit sums of equal signs: at most as many adds as there are units of 64 keys, and 64 within a unit; one division
        tol = half_step(dtype) * want + 2.0 ** -25 + want * (8 * 2.0 ** -24 + (n / 64 + 64) * 2.0 ** -24)
        assert float((weight.min() / weight.sum() / tol).min()) > 4.0
        out = paged_attention(q, *cache, _i32([length]), scale=math.log(2.0))
        assert bool(((out.double().cpu() - want).abs() <= tol).all()), length


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n,heads,D", [(500, 2, 64), (7001, 8, 128), (3000, 20, 64)])
def test_scores_a_thousand_apart(dtype, n, heads, D):
    """Small whole numbers: dot products are exact, the scale of 1000 puts unlike scores 1000 apart, and the answer is the mean of the
    values of the keys that share the largest."""
    from rustorch_b200.ops.paged import paged_attention
    g = torch.Generator().manual_seed(n)
    keys, values = torch.randint(-2, 3, (n, D), generator=g).float(), torch.randint(-64, 65, (n, D), generator=g).float() / 64
    q = torch.randint(-2, 3, (1, heads, D), generator=g).to(dtype)
    out = paged_attention(q.cuda(), *_pages(keys, values, 16, dtype), _i32([n]), scale=1000.0).double().cpu()
    dots = q[0].double() @ keys.double().t()
    for h in range(heads):
        top = dots[h] == dots[h].max()
        want = values[top].double().mean(0)
        # equal weights of 2^4 and sums of multiples of 1/64 are exact: the division and the result's rounding are left
        assert bool(((out[0, h] - want).abs() <= (half_step(dtype) + 2 * 2.0 ** -24) * want.abs()).all()), h


@pytest.mark.parametrize("seed", range(4))
def test_every_key_of_a_ragged_batch_counts_once(seed):
    """As above with equal weights: items of many lengths, several kv heads and tokens of one sequence share the grid's CTAs."""
    from rustorch_b200.ops.paged import paged_attention
    g = torch.Generator().manual_seed(seed)
    page, hkv, D = (16, 1, 24, 64)[seed], (1, 3, 2, 4)[seed], (128, 64, 256, 32)[seed]
    heads = hkv * (1, 5, 9, 2)[seed]
    lengths = [int(2 ** (torch.rand((), generator=g) * 12)) for _ in range(20)] + [0, 9000 >> seed]
    seq = torch.randint(0, len(lengths), (30,), generator=g, dtype=torch.int32)
    kv_len = torch.tensor([int(torch.randint(0, lengths[s] + 1, (1,), generator=g)) for s in seq.tolist()], dtype=torch.int32)
    need = [(n + page - 1) // page for n in lengths]
    order = torch.randperm(sum(need), generator=g).to(torch.int32)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int32)
    kp = torch.zeros(sum(need), hkv, page, D, dtype=torch.float16)
    vp = torch.zeros_like(kp)
    used = 0
    for s, n in enumerate(lengths):
        table[s, : need[s]] = order[used: used + need[s]]
        used += need[s]
        at = torch.arange(n)
        for h in range(hkv):                                                     # head h marks its keys one place further
            vp[table[s, at // page].long(), h, at % page, (at + h) % D] = 1.0
    q = torch.zeros(30, heads, D, dtype=torch.float16, device="cuda")
    out = paged_attention(q, kp.cuda(), vp.cuda(), table.cuda(), kv_len.cuda(), seq.cuda()).double().cpu()
    for t, n in enumerate(kv_len.tolist()):
        for h in range(heads):
            marks = (torch.arange(n) + h // (heads // hkv)) % D
            want = torch.bincount(marks, minlength=D).double() / max(1, n)
            # sums of equal weights are exact: the division and the result's rounding are left
            assert bool(((out[t, h] - want).abs() <= want * (half_step(torch.float16) + 2 * 2.0 ** -24) + 2.0 ** -25).all()), (t, h)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, 0.1])
@pytest.mark.parametrize("heads,D", [(1, 64), (12, 128), (2, 256)])
def test_infinite_values_stay_infinite(dtype, scale, heads, D):
    """Keys of a few different weights (equal ones with scale 0); some values of one sign are infinite: so is the answer in their place,
    and finite everywhere else.  NaN and infinities of both signs give NaN."""
    from rustorch_b200.ops.paged import paged_attention
    g = torch.Generator().manual_seed(D)
    n = 3000
    keys, values = torch.randn(n, D, generator=g), torch.randn(n, D, generator=g)
    at = torch.randint(0, n, (D,), generator=g)
    for d in range(D):
        if d % 4:
            values[at[d], d] = (float("inf"), -float("inf"), float("nan"))[d % 4 - 1]
        if d % 8 == 5:
            values[(at[d] + 100) % n, d] = -float("inf")
    q = torch.randn(1, heads, D, generator=g).to(dtype)
    out = paged_attention(q.cuda(), *_pages(keys, values, 16, dtype), _i32([n]), scale=scale).float().cpu()[0]
    for d in range(D):
        want = ("finite", "inf", "-inf", "nan")[d % 4] if d % 8 != 5 else "nan"
        got = out[:, d]
        assert bool({"finite": torch.isfinite(got), "inf": got == float("inf"), "-inf": got == -float("inf"), "nan": torch.isnan(got)}[want].all()), (d, want)


@pytest.mark.parametrize("power,softcap", [(24, 1e30), (24, 0.0), (24, 2.0), (0, 1e-6), (0, 1e30)])
def test_large_keys_small_scale_and_a_far_cap(power, softcap):
    """Keys and queries of 2^power, a scale of 2^(-2 power): scores are small whole numbers whatever the cap's distance, although scale /
    cap alone is below the 32-bit numbers."""
    from rustorch_b200.ops.paged import paged_attention
    n, D = 200, 64
    s = torch.arange(n) % 4
    keys, values = torch.zeros(n, D), torch.zeros(n, D)
    keys[:, 0], values[torch.arange(n), s] = s * 2.0 ** power, 1.0
    q = torch.zeros(1, 3, D, dtype=torch.bfloat16, device="cuda")
    q[:, :, 0] = 2.0 ** power
    score = s.double() if softcap == 0 or softcap == 1e30 else softcap * torch.tanh(s.double() / softcap)
    want = torch.zeros(D, dtype=torch.float64).index_add_(0, s, torch.softmax(score, 0))
    out = paged_attention(q, *_pages(keys, values, 16, torch.bfloat16), _i32([n]), scale=2.0 ** (-2 * power), softcap=softcap)
    # the result's rounding; two parts of a weight (2^-16 of it); scores below 4 in eight 32-bit roundings and a tanh to 2^-21 of the cap
    tol = want * (half_step(torch.bfloat16) + 2 * 2.0 ** -16 + 2 * 4 * (8 * 2.0 ** -24 + 2.0 ** -21)) + 2.0 ** -30
    assert bool(((out.double().cpu() - want).abs() <= tol).all())
