"""Controls of logits and draws at the edges of what they take."""
import numpy as np
import pytest
import torch

import plain_tree as plain
from tffinfer_b200.kernels.library import CudaKernels
from tffinfer_b200.sampling import LogitControls

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return CudaKernels()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def test_histories_that_are_none(ops):
    """Requests without tokens of their own, whatever their history's start says: ahead of the array, behind it, far outside; an empty array."""
    V, starts = 700, [-1, -3, 5, 7, 8, 9, 1 << 30, -(1 << 31), (1 << 31) - 1, 0, 3, 2]
    B = len(starts)
    logits = torch.randn(B, V, generator=torch.Generator().manual_seed(1)) * 4
    held = [1, 2, 3, 3, 699, 2, 1]
    # (a start inside the array with no tokens, or behind its end with some; a request without penalties; one with tokens, the last)
    lens = [4, 0, 0, 6, 1, 0, 9, 9, 9, 0, -5, 5]
    settings = [(1.5, 0.5, 0.25)] * B
    settings[3] = (1.0, 0.0, 0.0)
    for history in (held, []):
        seen = [history[2:7] if b == B - 1 else [] for b in range(B)]
        for first in range(4):                         # (the array's place within 16 bytes)
            store = i32([0] * first + history)
            c = LogitControls(i32(range(B + 1)), torch.tensor(settings, device=DEV), store[first:], i32(starts), i32(lens), i32([0] * B))
            out = torch.empty(B, V, device=DEV)
            ops.control_logits(logits.to(DEV), out, c)
            want = plain.control(logits, [(1, s, h, 0, []) for s, h in zip(settings, seen)])
            # two roundings, of values no larger than |x| * 1.5 + 0.5 * 3 + 0.25
            assert ((out.cpu().double() - want).abs() <= 2 * 2.0 ** -24 * (1.5 * logits.abs().double() + 1.75)).all()
            assert torch.equal(out.cpu()[:-1], logits[:-1])
