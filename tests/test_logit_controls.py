"""Sampling options that change logits, their packing for the kernel, and what the launchers of the drafted trees' kernels refuse (no GPU)."""
import ctypes
import math
import os

import numpy as np
import pytest
import torch

import plain_tree as plain
from tffinfer_b200.csrc import build
from tffinfer_b200.kernels import library
from tffinfer_b200.sampling import LogitControls, Sampler, SamplingParams, uniform_for


def test_options_and_what_they_need():
    p = SamplingParams()
    assert not p.controls_logits and not p.needs_token_values
    assert SamplingParams(repetition_penalty=1.2).needs_token_values and not SamplingParams(repetition_penalty=1.2).controls_logits
    for kw in (dict(frequency_penalty=0.1), dict(presence_penalty=-0.2), dict(token_mask=lambda t: None)):
        assert SamplingParams(**kw).controls_logits and SamplingParams(**kw).needs_token_values
    b = SamplingParams(logit_bias=((3, 1.0), (5, -math.inf)))
    assert b.controls_logits and not b.needs_token_values
    for kw in (dict(frequency_penalty=math.inf), dict(presence_penalty=math.nan), dict(logit_bias=((-1, 1.0),)), dict(logit_bias=((1, math.inf),)),
               dict(logit_bias=((1, math.nan),))):
        with pytest.raises(ValueError):
            SamplingParams(**kw)
    # the fields that were there keep their places
    assert SamplingParams("top_k", 0.5, 3, 0.9, 0.1, 1.1, 7, 20, (2,)) == SamplingParams(
        type="top_k", temperature=0.5, top_k=3, top_p=0.9, min_p=0.1, repetition_penalty=1.1, seed=7, max_new_tokens=20, eos_token_ids=(2,))


def test_controls_are_packed_as_they_are_given():
    V = 70
    mask = np.array([5, -1, 7], dtype=np.int32)
    params = [SamplingParams(repetition_penalty=1.5, frequency_penalty=0.25, presence_penalty=0.5),
              SamplingParams(logit_bias=((60, 2.0), (3, -1.0), (60, 0.5))), SamplingParams(token_mask=lambda made: mask if made == [9, 9] else None),
              SamplingParams(token_mask=lambda made: None)]
    c = LogitControls.of(params, [2, 0, 1, 0], [[4, 5, 6], [], [8, 9, 9], [1]], V, "cpu")
    assert c.problem(4, V) is None
    assert c.row_start.tolist() == [0, 1, 2, 3, 4] and c.history.tolist() == [4, 5, 6, 8, 9, 9, 1]
    assert c.history_start.tolist() == [0, 3, 3, 6] and c.history_len.tolist() == [3, 0, 3, 1] and c.prompt_len.tolist() == [2, 0, 1, 0]
    assert c.settings.tolist() == [[1.5, 0.25, 0.5], [1, 0, 0], [1, 0, 0], [1, 0, 0]]
    assert c.bias_start.tolist() == [0, 0, 3, 3, 3] and c.bias_tokens.tolist() == [3, 60, 60] and c.bias_values.tolist() == [-1.0, 0.5, 2.0]
    assert c.mask.tolist() == [[5, -1, 7]] and c.mask_row.tolist() == [-1, -1, 0, -1]
    bare = LogitControls.of(params[:1], [0], [[]], V, "cpu")
    assert bare.bias_start is None and bare.mask is None and bare.mask_row is None and bare.history.numel() == 0 and bare.problem(1, V) is None
    for bad in (np.zeros(2, np.int32), np.zeros(3, np.int64), np.zeros(3, np.float32), np.zeros((1, 3), np.int32)):
        with pytest.raises(ValueError):
            LogitControls.of([SamplingParams(token_mask=lambda made: bad)], [0], [[1]], V, "cpu")


def test_sizes_that_do_not_fit():
    i = lambda *n: torch.zeros(*n, dtype=torch.int32)
    good = dict(row_start=i(3), settings=torch.zeros(2, 3), history=i(5), history_start=i(2), history_len=i(2), prompt_len=i(2), bias_start=i(3),
                bias_tokens=i(4), bias_values=torch.zeros(4), mask=i(1, 4), mask_row=i(6), parents=i(6), tokens=i(6))
    assert LogitControls(**good).problem(6, 128) is None
    for bad in (dict(row_start=i(2)), dict(settings=torch.zeros(2, 2)), dict(history_start=i(3)), dict(history_len=i(1)), dict(prompt_len=i(1)),
                dict(bias_start=i(2)), dict(bias_start=None), dict(bias_tokens=None), dict(bias_values=torch.zeros(3)), dict(mask=i(4)), dict(mask=i(1, 3)),
                dict(mask=None), dict(mask_row=i(5)), dict(parents=i(5)), dict(tokens=i(5)), dict(parents=None), dict(tokens=None), dict(row_start=i(0))):
        assert LogitControls(**{**good, **bad}).problem(6, 128) is not None, bad


class _PlainOps:
    """control_logits and the draws as the sampler calls them, in plain torch."""
    def __init__(self):
        self.calls = []

    def control_logits(self, logits, out, c):
        requests = []
        for b in range(c.settings.shape[0]):
            first, n = int(c.history_start[b]), int(c.history_len[b])
            e = c.bias_start[b:b + 2].tolist() if c.bias_start is not None else (0, 0)
            requests.append((1, tuple(c.settings[b].tolist()), c.history[first:first + n].tolist(), int(c.prompt_len[b]),
                             list(zip(c.bias_tokens[e[0]:e[1]].tolist(), c.bias_values[e[0]:e[1]].tolist())) if c.bias_start is not None else []))
        V = logits.shape[1]
        masks = None
        if c.mask is not None:
            bits = np.unpackbits(c.mask.numpy().view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
            masks = [bits[m] if m >= 0 else None for m in c.mask_row.tolist()]
        self.calls.append("control_logits")
        out.copy_(plain.control(logits, requests, masks=masks).float())

    def repetition_penalty(self, logits, rows, tokens, penalty):
        self.calls.append("repetition_penalty")

    def argmax(self, logits, out):
        out.copy_(logits.argmax(1).int())


def test_the_sampler_controls_the_rows_whose_requests_ask_for_it():
    ops = _PlainOps()
    s = Sampler(ops, "cpu")
    logits = lambda: torch.tensor([[1.0, 2.0, 3.0, 2.9], [1.0, 2.0, 3.0, 2.9], [1.0, 2.0, 3.0, 2.9], [1.0, 2.0, 3.0, 2.9]])
    params = [SamplingParams(), SamplingParams(frequency_penalty=0.06), SamplingParams(logit_bias=((0, 5.0), (2, -math.inf))),
              SamplingParams(token_mask=lambda made: np.array([0b10], dtype=np.int32))]
    got = s.sample(logits(), params, [0, 1, 2, 3], [0, 0, 0, 0], [[2, 2], [2, 2, 2], [], [1]], [1, 1, 0, 1])
    assert got.tolist() == [2, 3, 0, 1] and ops.calls == ["control_logits"]
    # a token of the prompt alone is no repetition for the frequency penalty
    assert s.sample(logits()[:1], [params[1]], [0], [0], [[2, 2, 2]], [3]).tolist() == [2]
    ops.calls.clear()
    s.sample(logits()[:1], [SamplingParams(repetition_penalty=1.5)], [0], [0], [[2]])
    assert ops.calls == ["repetition_penalty"]           # a repetition penalty alone goes the way it went


def test_draws_that_lack_what_their_controls_need():
    s, logits = Sampler(_PlainOps(), "cpu"), torch.zeros(1, 4)
    for p in (SamplingParams(frequency_penalty=0.1), SamplingParams(presence_penalty=0.1), SamplingParams(token_mask=lambda made: None)):
        with pytest.raises(ValueError, match="needs the requests' tokens"):
            s.sample(logits, [p], [0], [0])
        with pytest.raises(ValueError, match="needs the requests' tokens"):
            s.sample(logits, [p], [0], [0], [[1]])
    s.sample(logits, [SamplingParams(logit_bias=((1, 1.0),))], [0], [0])      # a bias needs none


def test_options_that_float32_and_int32_do_not_hold():
    for kw in (dict(frequency_penalty=1e39), dict(presence_penalty=-1e39), dict(logit_bias=((0, 1e39),)), dict(logit_bias=((2**31, 1.0),)),
               dict(frequency_penalty=math.nan)):
        with pytest.raises(ValueError):
            SamplingParams(**kw)


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(build.library_path(build=True, verbose=False))
    library.declare_functions(lib)
    return lib


ONE = 16                                                  # an address that is never read: every call below is refused first


def test_launchers_refuse_what_they_cannot_take(lib):
    bad, unsupported = -1, -2
    def tree(**kw):
        a = dict(q=ONE, is_bf16=0, q_start=ONE, pos_start=ONE, parents=ONE, table=ONE, width=4, cache=ONE, pages=9, layers=1, layer=0, page=16, out=ONE, T=5, B=1, most=5,
                 nq=4, nkv=2, d=64, dv=64, dc=64, scale=0.1, window=0, softcap=0.0, sink=0, sink_val=None, gate=None, keep=0, splits=1, ws=None, stream=None)
        a.update(kw)
        return lib.tff_attention_tree(*a.values())
    for kw in (dict(q=None), dict(parents=None), dict(table=None), dict(cache=None), dict(out=None), dict(nq=3), dict(nkv=0), dict(d=0), dict(dc=32), dict(page=0),
               dict(softcap=-1.0), dict(keep=-1), dict(splits=0), dict(splits=2)):
        assert tree(**kw) == bad, kw
    for kw in (dict(d=520, dc=520, dv=520), dict(most=257), dict(B=65536)):
        assert tree(**kw) == unsupported, kw
    for kw in (dict(T=0), dict(B=0), dict(most=0)):
        assert tree(**kw) == 0

    def tc(**kw):
        a = dict(q=ONE, q_start=ONE, pos_start=ONE, parents=ONE, table=ONE, width=4, cache=ONE, pages=9, layers=1, layer=0, page=16, out=ONE, T=5, B=1, most=5, nq=4,
                 nkv=2, d=64, scale=0.1, window=0, softcap=0.0, sink=0, sink_val=None, gate=None, keep=0, least=4, extra=3, whole=0, ws=ONE, floats=1 << 40, stream=None)
        a.update(kw)
        return lib.tff_attention_tree_tc(*a.values())
    for kw in (dict(q=None), dict(parents=None), dict(nq=5), dict(softcap=-1.0), dict(keep=-2), dict(least=0), dict(extra=-1), dict(extra=65), dict(ws=None), dict(width=0)):
        assert tc(**kw) == bad, kw
    for kw in (dict(d=96), dict(page=12), dict(page=128), dict(pages=0), dict(scale=0.0), dict(scale=-1.0), dict(most=257), dict(nq=400, nkv=2), dict(q=24), dict(cache=8),
               dict(out=4), dict(ws=8), dict(pages=1 << 30)):
        assert tc(**kw) == unsupported, kw
    assert tc(T=0) == 0 and tc(B=0) == 0

    accept = lambda **kw: lib.tff_accept_tree(*{**dict(tokens=ONE, parents=ONE, drawn=ONE, q_start=ONE, T=3, B=1, path=ONE, emitted=ONE, count=ONE, width=4, stream=None), **kw}.values())
    for kw in (dict(tokens=None), dict(parents=None), dict(drawn=None), dict(q_start=None), dict(path=None), dict(emitted=None), dict(count=None), dict(width=0)):
        assert accept(**kw) == bad, kw
    assert accept(B=0) == 0

    keep = lambda **kw: lib.tff_keep_path(*{**dict(cache=ONE, pages=4, layers=1, planes=2, heads=2, page=16, row=128, page_bytes=8192, layer_bytes=8192, pos=ONE, table=ONE, width=4,
                                                   path=ONE, count=ONE, B=1, w=8, stream=None), **kw}.values())
    for kw in (dict(cache=None), dict(pages=0), dict(planes=0), dict(heads=0), dict(page=0), dict(row=0), dict(row=7), dict(pos=None), dict(table=None), dict(width=0), dict(path=None),
               dict(count=None), dict(B=65536)):
        assert keep(**kw) == bad, kw
    assert keep(B=0) == 0 and keep(w=1) == 0 and keep(layers=0) == 0

    def control(**kw):
        a = dict(logits=ONE, out=64, rows=2, vocab=40, B=2, row_start=ONE, settings=ONE, history=ONE, size=4, h_start=ONE, h_len=ONE, prompt=ONE, bias_start=None, bias_tokens=None,
                 bias_values=None, biases=0, mask=None, mask_rows=0, words=0, mask_row=None, parents=None, tokens=None, stream=None)
        a.update(kw)
        return lib.tff_control_logits(*a.values())
    for kw in (dict(logits=None), dict(out=None), dict(vocab=0), dict(B=65536), dict(row_start=None), dict(settings=None), dict(h_start=None), dict(h_len=None), dict(prompt=None),
               dict(mask=ONE, mask_rows=1, words=1), dict(parents=ONE), dict(parents=ONE, tokens=ONE, out=ONE), dict(bias_start=ONE, biases=3)):
        assert control(**kw) == bad, kw
    assert control(rows=0) == 0 and control(B=0) == 0


@pytest.mark.parametrize("requests,nodes,kv", [(1, 1, 1), (1, 256, 40960), (64, 8, 6000), (2, 13, 700), (65535, 1, 10), (30000, 3, 500)])
def test_shares_of_the_general_kernel(lib, requests, nodes, kv):
    for nq, nkv, dv, window in ((16, 8, 128, 0), (64, 8, 64, 512), (3, 1, 300, 0), (128, 1, 512, 4096)):
        s = lib.tff_attention_tree_splits(requests, nodes, kv, nq, nkv, dv, window, 0, 148)
        assert 1 <= s <= 32 and requests * s <= 65535
        keys = min(kv, window + nodes) if window else kv
        assert s == 1 or s <= keys // 64
    assert lib.tff_attention_tree_splits(0, 1, 1, 1, 1, 1, 0, 0, 148) == 1 and lib.tff_attention_tree_splits(1, 1, 1, 3, 2, 64, 0, 0, 148) == 1
