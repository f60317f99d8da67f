"""Controls of logits and draws at the edges of what they take."""
import math

import numpy as np
import pytest
import torch

import plain_tree as plain
from tffinfer_b200.kernels.library import CudaKernels
from tffinfer_b200.sampling import LogitControls, Sampler, SamplingParams

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


@pytest.mark.parametrize("penalty", [1.05, 1.2, 1.3, 0.7, 3.0, 1e-30])
@pytest.mark.parametrize("V", [4001, 20000])
def test_a_repetition_penalty_beside_other_controls(ops, penalty, V):
    """A request's logits are the same, bit by bit, whether its neighbour has a bias or not."""
    gen = torch.Generator().manual_seed(V)
    rows = torch.randn(2, V, generator=gen) * 4
    rows[0, ::7] *= 1e-38                           # some whose quotients or products are subnormal
    seen = torch.randint(0, V, (1500,), generator=gen).tolist() + list(range(0, V, 49))
    one = SamplingParams(repetition_penalty=penalty)
    sampler = Sampler(ops, DEV)
    got = []
    for beside in (SamplingParams(), SamplingParams(logit_bias=((3, 1.5),)), SamplingParams(frequency_penalty=0.5)):
        logits = rows.to(DEV)
        drawn = sampler.sample(logits, [one, beside], [0, 1], [0, 0], [seen, [1, 2]], [0, 2])
        got.append((logits[0].cpu(), int(drawn[0])))
    want = rows[0].clone()
    at = torch.tensor(sorted(set(seen)))
    p = torch.tensor(penalty, dtype=torch.float32)
    want[at] = torch.where(want[at] > 0, want[at] / p, want[at] * p)
    for logits, drawn in got:
        assert torch.equal(logits.view(torch.int32), want.view(torch.int32)) and drawn == got[0][1]


@pytest.mark.parametrize("least,most", [(-126, 127), (-3, 3), (-40, -20), (20, 70)])
def test_quotients_are_rounded_once(ops, least, most):
    """Logits of every exponent and their special values, penalties of many: what a division in float32 gives, to the bit."""
    rng = np.random.default_rng(abs(most))
    R, V = 64, 4096
    bits = rng.integers(0, 1 << 32, (R, V), dtype=np.uint32)
    bits[R // 2:] = bits[R // 2:] & 0x7fffff | rng.integers(0x3a000000 >> 23, 0x44000000 >> 23, (R - R // 2, V), dtype=np.uint32) << 23    # 2^-11 to 2^9
    x = torch.from_numpy(bits.view(np.float32).copy())
    x[x.isnan()] = 1.5
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = math.inf, -math.inf, 0.0, -0.0
    penalties = torch.from_numpy((rng.uniform(1, 2, R) * 2.0 ** rng.integers(least, most + 1, R)).astype(np.float32))
    settings = torch.stack([penalties, penalties * 0, penalties * 0], 1)
    c = LogitControls(i32(range(R + 1)), settings.to(DEV), i32(range(V)), i32([0] * R), i32([V] * R), i32([0] * R))
    out = torch.empty(R, V, device=DEV)
    ops.control_logits(x.to(DEV), out, c)
    want = torch.where(x > 0, x / penalties[:, None], x * penalties[:, None])
    assert torch.equal(out.cpu().view(torch.int32), want.view(torch.int32))


@pytest.mark.parametrize("nodes,kind", [([257], "random"), ([300, 2, 700], "random"), ([513], "chain"), ([1, 260], "star"), ([256, 257], "chain"), ([1100], "random")], ids=str)
def test_trees_of_more_nodes_than_attention_takes(ops, nodes, kind):
    """Every row of a tree gets its path's penalties, however many nodes the tree has."""
    V, few, R = 333, 9, sum(nodes)
    rng = np.random.default_rng(R)
    logits = torch.randn(R, V, generator=torch.Generator().manual_seed(R)) * 4
    trees = [list(range(-1, n - 1)) if kind == "chain" else [-1] + [0] * (n - 1) if kind == "star" else plain.random_tree(rng, n, spread=40, padding=n // 8) for n in nodes]
    tokens = rng.integers(0, few, R)
    settings = [(1.25, 0.0625, 0.5)] * len(nodes)
    histories = [rng.integers(0, few, 20).tolist() for _ in nodes]
    requests = [(n, s, h, 5, []) for n, s, h in zip(nodes, settings, histories)]
    c = LogitControls(i32(np.concatenate([[0], np.cumsum(nodes)])), torch.tensor(settings, device=DEV), i32(np.concatenate(histories)),
                      i32(np.arange(len(nodes)) * 20), i32([20] * len(nodes)), i32([5] * len(nodes)),
                      parents=i32(np.concatenate(trees)), tokens=i32(tokens))
    out = torch.empty(R, V, device=DEV)
    ops.control_logits(logits.to(DEV), out, c)
    want = plain.control(logits, requests, trees, tokens)
    # three roundings, of values no larger than |x| * 1.25 + the penalties of all nodes and of the history
    tol = 3 * 2.0 ** -24 * (1.25 * logits.abs().double() + 0.0625 * (max(nodes) + 20) + 0.5)
    assert ((out.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("biases,masked,want", [
    ([(5, 3e38), (5, 3e38), (5, -math.inf)], False, -math.inf), ([(5, -math.inf), (5, 3e38), (5, 3e38)], False, -math.inf),
    ([(5, 3e38), (5, 3e38)], True, -math.inf), ([(5, 2.0), (5, -math.inf)], True, -math.inf), ([(5, 3e38), (5, -3e38)], False, 1.0),
    ([(5, 3e38), (5, 3e38)], False, math.inf)], ids=str)
def test_biases_of_one_token_that_add_up_beyond_float32(ops, biases, masked, want):
    logits = torch.ones(1, 64, device=DEV)
    mask = np.full((1, 2), -1, dtype=np.int32)
    mask[0, 0] = ~np.int32(1 << 5)
    c = LogitControls(i32([0, 1]), torch.tensor([[1.0, 0.0, 0.0]], device=DEV), i32([]), i32([0]), i32([0]), i32([0]), i32([0, len(biases)]),
                      i32([t for t, _ in biases]), torch.tensor([v for _, v in biases], device=DEV), i32(mask) if masked else None)
    out = torch.empty_like(logits)
    ops.control_logits(logits, out, c)
    assert float(out[0, 5]) == want and (out[0, :5] == 1).all() and (out[0, 6:] == 1).all()


def draws_in_the_middle(row, T=1.0):
    """(tokens, numbers): numbers that lie in the middle of the kept tokens' stretches, by sums in 64 bits."""
    e = torch.exp((row.double() - row.max()) / T)
    ends = torch.cumsum(e, 0) / e.sum()
    kept = torch.nonzero(e > 0.0)[:, 0]
    u = (ends - e / e.sum() / 2)[kept].float()
    wide = (e / e.sum())[kept] > 1e-5             # (narrower ones lie within the rounding of the sums)
    return kept[wide], u[wide]


@pytest.mark.parametrize("V", [500, 32768, 151936])
@pytest.mark.parametrize("allowed,k", [(1, 50), (3, 50), (49, 50), (50, 50), (51, 50), (200, 50)])
def test_top_k_of_rows_with_few_allowed_tokens(ops, V, allowed, k):
    gen = torch.Generator().manual_seed(V + allowed)
    row = torch.randn(V, generator=gen)
    keep = torch.randperm(V, generator=gen)[:allowed]
    banned = torch.full((V,), -math.inf)
    banned[keep] = row[keep]
    top = torch.full((V,), -math.inf)
    best = torch.topk(banned, min(k, allowed)).indices
    top[best] = banned[best]
    tokens, u = draws_in_the_middle(top)
    R = tokens.numel()
    out = torch.empty(R, dtype=torch.int32, device=DEV)
    one = torch.ones(R, device=DEV)
    ops.sample(banned.repeat(R, 1).to(DEV), one, u.to(DEV), out, top_k=i32([k] * R), top_p=one, min_p=one * 0)
    assert out.tolist() == tokens.tolist()


def test_top_k_where_most_allowed_tokens_lie_far_below(ops):
    """Fewer than k tokens above e^-32 of the largest; with the largest taken away, the cut is what it would be without it."""
    V, k = 4096, 4
    row = torch.full((V,), -math.inf)
    row[7], row[100], row[200], row[300], row[400], row[500] = 0.0, -40.0, -41.0, -42.0, -43.0, -44.0
    for T, cut in ((1.0, None), (20.0, 4)):         # at T = 20 all lie within e^-3: the cut is seen
        top = row.clone()
        if cut:
            top[400] = top[500] = -math.inf
        tokens, u = draws_in_the_middle(top, T)
        R = tokens.numel()
        out = torch.empty(R, dtype=torch.int32, device=DEV)
        one = torch.ones(R, device=DEV)
        ops.sample(row.repeat(R, 1).to(DEV), one * T, u.to(DEV), out, top_k=i32([k] * R), top_p=one, min_p=one * 0)
        assert out.tolist() == tokens.tolist()


def test_rows_that_allow_nothing_give_the_first_token(ops):
    logits = torch.full((3, 40000), -math.inf, device=DEV)
    out = torch.full((3,), 9, dtype=torch.int32, device=DEV)
    one = torch.ones(3, device=DEV)
    for filters in ({}, dict(top_k=i32([50] * 3), top_p=one, min_p=one * 0), dict(top_k=i32([0] * 3), top_p=one * 0.9, min_p=one * 0.1)):
        ops.sample(logits, one, one * 0.5, out, **filters)
        assert out.tolist() == [0, 0, 0]


def test_a_grammar_does_not_make_top_k_slow(ops):
    """A row with fewer allowed tokens than k takes no longer than one whose tokens are all allowed (twice as long, for the clock's noise)."""
    V, R = 151936, 8
    gen = torch.Generator().manual_seed(1)
    open_ = (torch.randn(R, V, generator=gen) * 4).to(DEV)
    held = torch.full((R, V), -math.inf, device=DEV)
    held[:, :20] = open_[:, :20]
    out = torch.empty(R, dtype=torch.int32, device=DEV)
    one = torch.ones(R, device=DEV)
    def best(logits):
        times = []
        for _ in range(12):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ops.sample(logits, one, one * 0.5, out, top_k=i32([50] * R), top_p=one, min_p=one * 0)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)
    for logits in (held, torch.full_like(held, -math.inf)):
        t, limit = best(logits), 2 * best(open_)
        assert t <= limit, (t, limit)


def test_masks_that_leave_many(ops):
    """More allowed tokens than the list of candidates takes, most of them far below the largest; either filter, and both."""
    V = 40000
    row = torch.full((V,), -math.inf)
    row[1000:13000] = -40.0
    row[500] = 0.0
    logits = row.repeat(3, 1).to(DEV)
    one = torch.ones(3, device=DEV)
    out = torch.empty(3, dtype=torch.int32, device=DEV)
    for top_p in (1.0, 0.9):
        ops.sample(logits, one, one * 0.5, out, top_k=i32([50, 20000, 0]), top_p=one * top_p, min_p=one * 0)
        assert out.tolist() == [500, 500, 500]


def test_an_infinite_logit_is_drawn(ops):
    V = 40000
    for rest in (-math.inf, 1.0):
        row = torch.full((V,), rest)
        row[123] = math.inf
        logits = row.repeat(2, 1).to(DEV)
        one = torch.ones(2, device=DEV)
        out = torch.empty(2, dtype=torch.int32, device=DEV)
        ops.sample(logits, one, one * 0.5, out)
        assert out.tolist() == [123, 123]
        for k, p in ((50, 1.0), (0, 0.9), (50, 0.9), (20000, 0.99)):
            ops.sample(logits, one, one * 0.5, out, top_k=i32([k] * 2), top_p=one * p, min_p=one * 0)
            assert out.tolist() == [123, 123]
