"""The kernel trace counts the control of logits and the operators of drafted trees."""
import math

import pytest
import torch

from helpers import make_model_dir, PAGE_SIZE
from tffinfer_b200.config import EngineConfig
from tffinfer_b200.engine import Engine
from tffinfer_b200.kernels import trace
from tffinfer_b200.kernels.library import CudaKernels
from tffinfer_b200.sampling import SamplingParams

CALLS = ("control_logits", "attention_tree", "accept_tree", "keep_path")


def test_the_calls_are_traced():
    for name in CALLS:
        assert name in trace.TRACED and callable(getattr(CudaKernels, name))


@pytest.mark.gpu
def test_a_traced_generation_shows_the_control_of_logits(tmp_path):
    eng = Engine(make_model_dir(tmp_path, "B"), EngineConfig(dtype="float32", page_size=PAGE_SIZE["B"], max_cache_tokens=256, use_cuda_graphs=False))
    with trace.KernelTrace(eng.runner.ops) as t:
        eng.generate([[1, 2, 3]], SamplingParams(max_new_tokens=5, logit_bias=((4, 1.0), (7, -math.inf))))
    calls = {name: n for name, n, _ in t.summary()}
    assert calls["control_logits"] == 5
    torch.cuda.synchronize()
