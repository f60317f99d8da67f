"""A grammar that fails ends its own request and no other's."""
import numpy as np
import pytest
import torch

import plain_tree as plain
from cpu_ops import CpuOps
from helpers import make_model_dir, tiny_config, PAGE_SIZE
from tffinfer_b200.config import EngineConfig
from tffinfer_b200.engine import Engine, ModelRunner
from tffinfer_b200.sampling import SamplingParams

BACKENDS = ["cpu_twins", pytest.param("cuda", marks=pytest.mark.gpu)]


class Ops(CpuOps):
    def control_logits(self, logits, out, c):
        requests = []
        for b in range(c.settings.shape[0]):
            first, n = int(c.history_start[b]), int(c.history_len[b])
            requests.append((1, tuple(c.settings[b].tolist()), c.history[first:first + n].tolist(), int(c.prompt_len[b]), []))
        masks = None
        if c.mask is not None:
            bits = np.unpackbits(c.mask.numpy().view(np.uint8), axis=1, bitorder="little")[:, :logits.shape[1]].astype(bool)
            masks = [bits[m] if m >= 0 else None for m in c.mask_row.tolist()]
        out.copy_(plain.control(logits, requests, masks=masks).float())


def _engine(tmp_path, backend, **kw):
    d = make_model_dir(tmp_path, "B")
    kw.update(max_cache_tokens=512, max_live_requests=6)
    if backend == "cpu_twins":
        return Engine(runner=ModelRunner(d, EngineConfig(dtype="float32", page_size=PAGE_SIZE["B"], device="cpu", **kw), ops=Ops()))
    return Engine(d, EngineConfig(dtype="float32", page_size=PAGE_SIZE["B"], **kw))


WORDS = -(-tiny_config("B").vocab_size // 32)


def _even(made):
    bits = np.zeros(WORDS * 32, dtype=bool)
    bits[len(made) % 2::2] = True
    return np.packbits(bits, bitorder="little").view(np.int32)


def _fails(how, when):
    def mask(made):
        if len(made) < when:
            return _even(made)
        if how == "raises":
            raise RuntimeError("no rule for this token")
        return {"size": np.zeros(WORDS + 1, np.int32), "type": np.zeros(WORDS, np.int64), "list": [0] * WORDS}[how]
    return mask


@pytest.mark.parametrize("backend", BACKENDS)
@pytest.mark.parametrize("async_steps", [False, True])
@pytest.mark.parametrize("how,when", [("raises", 0), ("raises", 3), ("size", 2), ("type", 1), ("list", 1)])
def test_a_grammar_that_fails_ends_its_request(tmp_path, backend, async_steps, how, when):
    eng = _engine(tmp_path, backend, async_steps=async_steps)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, tiny_config("B").vocab_size, n).tolist() for n in (9, 4, 21)]
    others = [SamplingParams(max_new_tokens=8), SamplingParams(max_new_tokens=8, token_mask=_even)]
    want = eng.generate(prompts[:2], others)
    free = [p.num_free for p in eng.scheduler.cache.pools]
    ids = [eng.add_request(p, sp, key=i) for i, (p, sp) in enumerate(zip(prompts, others + [SamplingParams(max_new_tokens=8, token_mask=_fails(how, when))]))]
    ends, steps = [], 0
    while eng.has_unfinished():
        ends += [o for o in eng.step() if o.finished]
        steps += 1
        assert steps < 100
    got = [eng.requests[i] for i in ids]
    assert [r.generated for r in got[:2]] == want and [r.finish_reason for r in got[:2]] == ["length"] * 2
    assert got[2].finish_reason == "bad_mask" and got[2].status == "finished" and len(got[2].generated) == when
    assert [(o.request_id, o.token, o.finish_reason) for o in ends if o.request_id == ids[2]] == [(ids[2], None, "bad_mask")]
    assert [t % 2 for t in got[2].generated] == [i % 2 for i in range(when)]
    assert [p.num_free for p in eng.scheduler.cache.pools] == free and not eng.scheduler.running
    assert eng.generate(prompts[:2], others) == want       # and the engine goes on


def test_a_grammar_is_not_asked_for_a_token_that_is_not_drawn(tmp_path):
    eng, asked = _engine(tmp_path, "cpu_twins"), []
    def mask(made):
        asked.append(len(made))
        return None
    assert eng.generate([[1, 2, 3]], SamplingParams(max_new_tokens=0, token_mask=mask)) == [[]] and asked == []
    assert len(eng.generate([[1, 2, 3]], SamplingParams(max_new_tokens=4, token_mask=mask))[0]) == 4 and asked == [0, 1, 2, 3]


@pytest.mark.parametrize("backend", BACKENDS)
def test_a_grammar_that_reuses_its_array(tmp_path, backend):
    """One grammar serves two requests from one array, which it fills anew at each call: each request has its own mask."""
    eng, shared = _engine(tmp_path, backend), np.zeros(WORDS, np.int32)
    def parity(odd):
        def mask(made):
            bits = np.zeros(WORDS * 32, dtype=bool)
            bits[odd::2] = True
            shared[:] = np.packbits(bits, bitorder="little").view(np.int32)
            return shared
        return mask
    got = eng.generate([[1, 2, 3], [4, 5]], [SamplingParams(max_new_tokens=5, token_mask=parity(0)), SamplingParams(max_new_tokens=5, token_mask=parity(1))])
    assert [[t % 2 for t in g] for g in got] == [[0] * 5, [1] * 5]


def test_a_mask_that_allows_nothing_is_none():
    """Bits behind the vocabulary are no tokens.  (The draw from such a row would be token 0, which the grammar does not allow.)"""
    from tffinfer_b200.sampling import mask_of
    for vocab in (1, 31, 32, 33, 64, 70):
        words = -(-vocab // 32)
        none = np.zeros(words * 32, dtype=bool)
        none[vocab:] = True
        for empty in (np.zeros(words, np.int32), np.packbits(none, bitorder="little").view(np.uint32)):
            with pytest.raises(ValueError, match="allows no token"):
                mask_of(SamplingParams(token_mask=lambda made: empty), [], vocab)
        for t in {0, vocab // 2, vocab - 1}:
            some = np.zeros(words * 32, dtype=bool)
            some[t] = True
            got = mask_of(SamplingParams(token_mask=lambda made: np.packbits(some, bitorder="little").view(np.int32)), [], vocab)
            assert got.view(np.uint32)[t // 32] == 1 << t % 32


@pytest.mark.parametrize("backend", BACKENDS)
def test_a_grammar_that_has_come_to_its_end(tmp_path, backend):
    """It ends its request: nothing is drawn against it."""
    eng = _engine(tmp_path, backend)
    i = eng.add_request([1, 2, 3], SamplingParams(max_new_tokens=9, token_mask=lambda made: _even(made) if len(made) < 4 else np.zeros(WORDS, np.int32)))
    while eng.has_unfinished():
        eng.step()
    assert eng.requests[i].finish_reason == "bad_mask" and [t % 2 for t in eng.requests[i].generated] == [0, 1, 0, 1]
