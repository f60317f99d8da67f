"""Steps over trees of drafted tokens: positions, slots and refusals (no GPU)."""
import numpy as np
import pytest
import torch

import plain_tree as plain
from cpu_ops import CpuOps
from helpers import make_model_dir, tiny_config, PAGE_SIZE
from tffinfer_b200.config import EngineConfig
from tffinfer_b200.engine import ModelRunner, StepEntry
from tffinfer_b200.engine.runner import RequestError
from tffinfer_b200.parts.attention import GatedSinkAttention, GQAttention, BiasedChunkAttention


class Ops(CpuOps):
    """The twins, with slots of their own for keys and values, and the attention of trees."""

    def qk_norm_rope_kv_write(self, qkv, q_out, q_w, k_w, eps, table, rot_dim, batch, block_table, kv_cache, kv_layer, page_size, nq, nkv, d, write_cache):
        call = lambda cache, where: CpuOps.qk_norm_rope_kv_write(self, qkv, q_out, q_w, k_w, eps, table, rot_dim, where, block_table, cache, kv_layer,
                                                                 page_size, nq, nkv, d, write_cache)
        if batch.cache_slots is None:
            return call(kv_cache, batch)
        # a row at a time, through a cache of its own: the twin writes where the positions say
        keys = []
        for t in range(qkv.shape[0]):
            one = type("One", (), dict(positions=batch.positions[t:t + 1], tok_req=batch.tok_req[t:t + 1]))
            aside, out = kv_cache.clone(), torch.empty_like(q_out[t:t + 1])
            CpuOps.qk_norm_rope_kv_write(self, qkv[t:t + 1], out, q_w, k_w, eps, table, rot_dim, one, block_table, aside, kv_layer, page_size, nq, nkv, d, True)
            q_out[t:t + 1] = out
            b, pos = int(batch.tok_req[t]), int(batch.positions[t])
            keys.append(aside[int(block_table[b, pos // page_size]), kv_layer, :, :, pos % page_size].clone())
        for t, kv in enumerate(keys):
            b, at = int(batch.tok_req[t]), int(batch.cache_slots[t])
            kv_cache[int(block_table[b, at // page_size]), kv_layer, :, :, at % page_size] = kv

    def attend(self, h, w_qkv, q_w, k_w, eps, table, rot_dim, batch, block_table, kv_cache, kv_layer, page_size, out, nq, nkv, d, scale, window, write_cache):
        if batch.parents is None:
            return CpuOps.attend(self, h, w_qkv, q_w, k_w, eps, table, rot_dim, batch, block_table, kv_cache, kv_layer, page_size, out, nq, nkv, d, scale,
                                 window, write_cache)
        q = torch.empty((h.shape[0], nq * d), dtype=out.dtype)
        self.qkv_project(h, w_qkv, q, q_w, k_w, eps, table, rot_dim, batch, block_table, kv_cache, kv_layer, page_size, nq, nkv, d, write_cache)
        start, ctx = batch.q_start.tolist(), batch.pos_start.tolist()
        keys, values = [], []
        for b in range(batch.num_requests):
            n = torch.arange(ctx[b] + start[b + 1] - start[b])
            pages = block_table[b].long()[n // page_size]
            keys.append(kv_cache[pages, kv_layer, 0, :, n % page_size])
            values.append(kv_cache[pages, kv_layer, 1, :, n % page_size])
        trees = [batch.parents[start[b]:start[b + 1]].tolist() for b in range(batch.num_requests)]
        o, _, _ = plain.attention(q.view(-1, nq, d), keys, values, ctx, trees, nq, scale, window=window)
        out.copy_(o.reshape(out.shape))


def runner(tmp_path, name="B", ops=None, **kw):
    d = make_model_dir(tmp_path, name)
    return d, ModelRunner(d, EngineConfig(dtype="float32", page_size=PAGE_SIZE[name], device="cpu", max_cache_tokens=512, max_live_requests=4, **kw),
                          ops=ops or Ops())


def test_positions_and_slots_of_nodes(tmp_path):
    _, run = runner(tmp_path)
    run.add_request("a"), run.add_request("b")
    run.step([StepEntry("a", [1, 2, 3]), StepEntry("b", [4] * 9)])
    trees = [[-1, 0, 0, 1, 2, -1, -2, 6, 7, 9, 4], [-1, 0, 1, 2, 1, 9, -7]]
    batch = run.make_batch([StepEntry("a", list(range(11)), range(11)), StepEntry("b", list(range(7)), [0])], parents=trees)
    assert batch.parents.tolist() == [-1, 0, 0, 1, 2, -1, -2, 6, 7, -2, 4, -1, 0, 1, 2, 1, -2, -2]
    # (nodes that are not there stand at the first position)
    assert batch.positions.tolist() == [3, 4, 4, 5, 5, 3, 3, 3, 3, 3, 6, 9, 10, 11, 12, 11, 9, 9]
    assert batch.cache_slots.tolist() == list(range(3, 14)) + list(range(9, 16))
    assert batch.positions.dtype == batch.parents.dtype == batch.cache_slots.dtype == torch.int32
    assert batch.graph_bucket is None and batch.logit_rows.tolist() == list(range(11)) + [11]


def test_parents_that_do_not_fit_take_no_pages(tmp_path):
    _, run = runner(tmp_path)
    run.add_request("a"), run.add_request("b")
    free = [p.num_free for p in run.cache.pools]
    entries = [StepEntry("a", [1, 2, 3]), StepEntry("b", [4, 5])]
    for parents in ([[-1, 0, 0]], [[-1, 0], [-1, 0]], [[-1, 0, 1], [-1, 0, 1]], []):
        with pytest.raises(RequestError, match="parents"):
            run.make_batch(entries, parents=parents)
    with pytest.raises(RequestError, match="at most 256 nodes"):
        run.make_batch([StepEntry("a", [1] * 257)], parents=[[-1] * 257])
    assert [p.num_free for p in run.cache.pools] == free
    batch = run.make_batch(entries)
    with pytest.raises(ValueError, match="a number for each"):
        batch.with_parents([[-1, 0, 0], [-1]])
    batch.graph_bucket = 2
    with pytest.raises(ValueError, match="captured"):
        batch.with_parents([[-1, 0, 0], [-1, 0]])


def test_mixers_that_take_no_trees(tmp_path):
    assert GQAttention(64, 4, 2, 16, qk_norm_eps=1e-6).takes_trees and GatedSinkAttention(64, 4, 2, 16).takes_trees
    assert GatedSinkAttention(64, 4, 2, 16, qk_norm="head", qk_norm_eps=1e-6).takes_trees
    for m in (GatedSinkAttention(64, 4, 2, 16, conv_taps=3), GatedSinkAttention(64, 4, 2, 16, qk_norm="whole", qk_norm_eps=1e-6),
              BiasedChunkAttention(64, 4, 2, 16, chunk=8)):
        assert not m.takes_trees
    _, run = runner(tmp_path)
    run.add_request("a")
    run.model.blocks[1].mixer.takes_trees = False
    with pytest.raises(RequestError, match="gqa_attention"):
        run.make_batch([StepEntry("a", [1, 2])], parents=[[-1, 0]])


@pytest.mark.parametrize("name", ["B", "C"])
def test_nodes_have_the_logits_of_their_paths(tmp_path, name):
    """Branching trees through the step function, behind contexts of unequal lengths."""
    from plain_qwen3 import PlainModel
    d, run = runner(tmp_path, name)
    pm, rng = PlainModel(d), np.random.default_rng(5)
    V = tiny_config(name).vocab_size
    prompts = {r: rng.integers(0, V, n).tolist() for r, n in (("a", 5), ("b", 37))}
    for r in prompts:
        run.add_request(r)
    run.step([StepEntry(r, p) for r, p in prompts.items()])
    trees = {"a": [-1, 0, 0, 1, 1, 2, 5], "b": [-1, 0, 1, 0, 3, 3]}
    tokens = {r: rng.integers(0, V, len(t)).tolist() for r, t in trees.items()}
    batch = run.make_batch([StepEntry(r, tokens[r], range(len(t))) for r, t in trees.items()], parents=list(trees.values()))
    logits, row = run.run_batch(batch), 0
    for r, tree in trees.items():
        for i in range(len(tree)):
            path = [tokens[r][j] for j in reversed(plain.chain(tree, i))]
            want = pm.logits(prompts[r] + path)[-1]
            assert (logits[row] - want).abs().max() <= 2e-5 * want.abs().max(), (r, i)
            row += 1
