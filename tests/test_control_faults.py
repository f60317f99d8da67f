"""Options that change logits, at the edges of what they take (no GPU)."""
import numpy as np
import pytest
import torch

from tffinfer_b200.sampling import LogitControls, Sampler, SamplingParams


class _Ops:
    """Keeps what the sampler gives the kernels."""
    def __init__(self):
        self.controls = []

    def control_logits(self, logits, out, controls):
        self.controls.append(controls)

    def argmax(self, logits, out):
        out.copy_(logits.argmax(1).int())


def test_a_repetition_penalty_beside_a_bias_needs_no_prompt_length():
    """How many of a request's tokens are the prompt matters to the penalties of generated tokens and to a grammar alone."""
    ops = _Ops()
    params = [SamplingParams(repetition_penalty=1.5), SamplingParams(logit_bias=((1, 1.0),))]
    Sampler(ops, "cpu").sample(torch.zeros(2, 4), params, [0, 1], [0, 0], [[2, 3], []])
    c = ops.controls[0]
    assert c.history.tolist() == [2, 3] and c.history_len.tolist() == [2, 0] and c.settings[0].tolist() == [1.5, 0.0, 0.0]
    # without the request's tokens there is nothing to penalise, as in a step without biases
    Sampler(ops, "cpu").sample(torch.zeros(2, 4), params, [0, 1], [0, 0])
    assert ops.controls[1].history_len.tolist() == [0, 0]
    for p in (SamplingParams(repetition_penalty=1.5, presence_penalty=0.1), SamplingParams(token_mask=lambda made: None)):
        with pytest.raises(ValueError, match="needs the requests' tokens"):
            Sampler(ops, "cpu").sample(torch.zeros(2, 4), [p, params[1]], [0, 1], [0, 0], [[2, 3], []])


@pytest.mark.parametrize("penalty", [1e39, float("inf"), float("nan"), 1e-46, 0.0, -1.0])
def test_repetition_penalties_that_float32_does_not_hold(penalty):
    """An infinite one makes a logit of 0 NaN, one that rounds to 0 every positive logit infinite."""
    with pytest.raises(ValueError, match="repetition_penalty"):
        SamplingParams(repetition_penalty=penalty)


@pytest.mark.parametrize("penalty", [1.0, 3e38, 2e-45, 0.5])
def test_repetition_penalties_that_float32_holds(penalty):
    assert SamplingParams(repetition_penalty=penalty).repetition_penalty == penalty
