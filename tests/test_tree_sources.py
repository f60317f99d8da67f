"""The library that an engine builds for its model holds the kernels of a step over drafted trees, where the model's mixers take one (no GPU)."""
import os

import pytest

import tffinfer_b200.models  # noqa: F401  registers the architectures
import tffinfer_b200.parts  # noqa: F401  registers the parts
from helpers import tiny_config
from tffinfer_b200 import get_architecture
from tffinfer_b200.csrc import build
from tffinfer_b200.kernels import library
from tffinfer_b200.parts.attention import GatedSinkAttention
from tffinfer_b200.parts.model import Model

ENTRY_POINTS = {"tff_attention_tree", "tff_attention_tree_tc", "tff_attention_tree_splits", "tff_accept_tree", "tff_keep_path", "tff_control_logits"}


def entry_points(files):
    out = set()
    for source in build.chosen_sources(files):
        with open(os.path.join(build.CSRC_DIR, source)) as f:
            out |= {name for name, _, _ in library.function_signatures(f.read())}
    return out


@pytest.mark.parametrize("name", ["A", "D"])
def test_a_model_of_plain_attention(name):
    cfg = tiny_config(name)
    model = Model(get_architecture(cfg.architecture).describe(cfg))
    assert ENTRY_POINTS <= entry_points(model.kernel_files())


@pytest.mark.parametrize("kw", [dict(), dict(qk_norm="head", qk_norm_eps=1e-6)])
def test_a_gated_mixer(kw):
    assert ENTRY_POINTS <= entry_points(GatedSinkAttention(64, 4, 2, 16, **kw).kernel_files())
