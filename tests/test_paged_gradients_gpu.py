"""The paged-cache kernels refuse every input that asks for a gradient, as the CPU forms do."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_inputs_that_ask_for_gradients_are_refused():
    from rustorch_b200.ops.paged import paged_append, paged_attention
    from test_paged_gradients_cpu import _append_args, _attention_args
    for op, args in ((paged_append, _append_args), (paged_attention, _attention_args)):
        def make():
            return {k: (t.half() if t.is_floating_point() and k != "inv_freq" else t).cuda() for k, t in args().items()}
        for name in [k for k, t in make().items() if t.is_floating_point()]:
            kw = make()
            kw[name].requires_grad_()
            with pytest.raises(ValueError, match="no backward pass"):
                op(**kw)
            with torch.no_grad():
                op(**kw)
        assert not op(**make()).requires_grad
