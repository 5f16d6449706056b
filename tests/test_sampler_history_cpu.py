"""Repetition penalty over a history that holds -1, the token of a row that had none to draw."""
import pytest
import torch

from rustorch_b200.llm import Sampler, SamplingConfig, apply_repetition_penalty


def _penalised(logits, history, penalty):
    out = logits.clone()
    for r, row in enumerate(history.tolist()):
        for t in {x for x in row if x >= 0}:
            out[r, t] = out[r, t] / penalty if out[r, t] > 0 else out[r, t] * penalty
    return out


@pytest.mark.parametrize("history", [[[-1], [2]], [[0, -1, 3], [-1, -1, -1]], [[-1, 0, 0], [4, 4, -1]], [[1, 2], [3, 0]]])
def test_penalty_passes_over_missing_tokens(history):
    logits = torch.randn(2, 6, generator=torch.Generator().manual_seed(0))
    logits[0, 0], logits[1, 0] = 1.5, -1.5
    h = torch.tensor(history)
    assert torch.equal(apply_repetition_penalty(logits, h, 1.3), _penalised(logits, h, 1.3))
    assert torch.equal(apply_repetition_penalty(logits[0], h[0], 1.3), _penalised(logits[:1], h[:1], 1.3)[0])


def test_draw_goes_on_after_a_row_without_a_token():
    logits = torch.randn(3, 8, generator=torch.Generator().manual_seed(1))
    logits[1] = -float("inf")
    u = torch.rand(3, generator=torch.Generator().manual_seed(2))
    s = Sampler(SamplingConfig(repetition_penalty=1.4))
    first = s.draw(logits, u)
    assert int(first[1]) == -1
    second = s.draw(logits, u)
    plain = Sampler(SamplingConfig())
    assert torch.equal(second, plain.draw(_penalised(logits, first[:, None], 1.4), u)) and int(second[1]) == -1
    assert s.history.tolist() == torch.stack([first, second], 1).tolist()
