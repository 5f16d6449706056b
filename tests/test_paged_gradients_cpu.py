"""The paged-cache operators have no backward pass: every input that the formulas depend on is refused while it asks for a gradient."""
import pytest
import torch

from rustorch_b200.ops.paged import paged_append, paged_attention


def _append_args():
    i = torch.zeros(1, dtype=torch.int32)
    q, k = torch.ones(1, 2, 8), torch.ones(1, 1, 8)
    return dict(q=q, k=k, v=k.clone(), k_pages=torch.zeros(1, 1, 4, 8), v_pages=torch.zeros(1, 1, 4, 8), block_table=i.view(1, 1), pos=i, seq=i,
                inv_freq=torch.ones(4), q_norm=torch.ones(8), k_norm=torch.ones(8), q_out=torch.zeros(1, 2, 8), k_out=torch.zeros(1, 1, 8))


def _attention_args():
    i = torch.zeros(1, dtype=torch.int32)
    return dict(q=torch.ones(1, 2, 8), k_pages=torch.ones(1, 1, 4, 8), v_pages=torch.ones(1, 1, 4, 8), block_table=i.view(1, 1), kv_len=i + 2, seq=i,
                out=torch.zeros(1, 2, 8))


@pytest.mark.parametrize("op,args", [(paged_append, _append_args), (paged_attention, _attention_args)])
def test_inputs_that_ask_for_gradients_are_refused(op, args):
    floating = [k for k, t in args().items() if t.is_floating_point()]
    for name in floating:
        kw = args()
        kw[name].requires_grad_()
        with pytest.raises(ValueError, match="no backward pass"):
            op(**kw)
        with torch.no_grad():
            op(**kw)
    got = op(**args())
    assert not got.requires_grad
