"""The command line's options that change logits (no GPU)."""
import math

import pytest

from tffinfer_b200.cli import build_parser, sampling_params
from tffinfer_b200.sampling import SamplingParams


def params(*argv):
    return sampling_params(build_parser().parse_args(["model", *argv]))


def test_options_reach_the_sampling_params():
    p = params("--n-predict", "5", "--repetition-penalty", "1.2", "--frequency-penalty", "0.5", "--presence-penalty", "-0.25", "--logit-bias", "7:1.5",
               "--logit-bias", "9:-inf", "--eos", "3")
    assert (p.repetition_penalty, p.frequency_penalty, p.presence_penalty) == (1.2, 0.5, -0.25)
    assert p.logit_bias == ((7, 1.5), (9, -math.inf)) and p.max_new_tokens == 5 and p.eos_token_ids == (3,) and p.is_greedy


def test_what_was_there_means_what_it_meant():
    assert params() == SamplingParams(max_new_tokens=64) and params("--temperature", "0.7", "--top-k", "5") == SamplingParams.make(
        temperature=0.7, top_k=5, max_new_tokens=64)
    assert params("--sample-type", "greedy", "--temperature", "0.7").is_greedy and not params("--sample-type", "random").is_greedy


@pytest.mark.parametrize("text", ["7", "7:", ":1", "a:1", "7:b", "7:1:2"])
def test_biases_that_are_none(text):
    with pytest.raises(SystemExit):
        build_parser().parse_args(["model", "--logit-bias", text])


@pytest.mark.parametrize("argv", [("--logit-bias", "-1:2"), ("--logit-bias", "1:inf"), ("--frequency-penalty", "nan"), ("--repetition-penalty", "1e39")])
def test_values_that_are_refused(argv):
    with pytest.raises(ValueError):
        params(*[argv[0] + "=" + argv[1]])
