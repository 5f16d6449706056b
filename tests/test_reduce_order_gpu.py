"""Full reductions: sums of a training step's row losses repeat bit for bit, maxima and minima are exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 31, 257, 1025, 8192, 32768, 32769, 100003])
def test_sums_repeat_and_extremes_are_exact(n, dtype):
    from rustorch_b200.ops import kernels as K
    x = torch.randn(n, generator=torch.Generator().manual_seed(n)).to(dtype).cuda()
    wide = x.double()
    assert float(K.reduce_all(x, "max")) == float(x.max()) and float(K.reduce_all(x, "min")) == float(x.min())
    for mode, want, size in (("sum", wide.sum(), wide.abs().sum()), ("sumsq", wide.square().sum(), wide.square().sum())):
        got = [float(K.reduce_all(x, mode)) for _ in range(10)]
        assert abs(got[0] - float(want)) <= (n ** 0.5 + 40) * 2.0 ** -24 * float(size)
        assert n > 32768 or len(set(got)) == 1
