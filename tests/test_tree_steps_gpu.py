"""Steps over trees of drafted tokens on the GPU: the kernels that write keys and values put siblings into slots of their own, whole models
give every node the logits of its path, and generation over trees gives what generation token by token gives."""
import numpy as np
import pytest
import torch

import plain_tipezen
import plain_tree as plain
from helpers import make_model_dir, tiny_config, PAGE_SIZE, PROMPT_LENS
from plain_qwen3 import PlainModel
from tffinfer_b200.config import EngineConfig, RotaryConfig, TipezenConfig, TipezenLayer
from tffinfer_b200.engine import Engine, ModelRunner, StepEntry
from tffinfer_b200.engine.batch import StepBatch
from tffinfer_b200.engine.runner import RequestError
from tffinfer_b200.kernels.library import CudaKernels, KernelError
from tffinfer_b200.sampling import LogitControls
from tffinfer_b200.weights.random_init import random_state_dict

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return CudaKernels()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def step_batch(ctx, counts):
    n, c = np.asarray(counts), np.asarray(ctx)
    start, req, order = np.concatenate([[0], np.cumsum(n)]), np.repeat(np.arange(len(n)), n), np.lexsort((-(c + n), n))
    T = int(start[-1])
    return StepBatch(num_tokens=T, num_requests=len(n), num_logit_rows=T, max_q_len=int(n.max()), max_kv_len=int((c + n).max()), token_ids=i32(np.zeros(T)),
                     positions=i32(c[req] + np.arange(T) - start[req]), tok_req=i32(req), q_start=i32(start), pos_start=i32(c), kv_len=i32(c + n),
                     slots=i32(np.arange(len(n))), logit_rows=i32(np.arange(T)), req_order=i32(order), h_q_lens=n, h_pos_start=c, h_sorted_q_lens=n[order],
                     h_sorted_kv_lens=(c + n)[order], real_requests=len(n), real_logit_rows=T)


TREES = [[-1, 0, 0, 1, 1, 2, 5, 3, 0], [-1, 0, -1, 2, 2], [-1]]
CTX, PAGE = [37, 5, 64], 16

# what writes keys and values: plain heads (of 128: the kernel of its own), heads normed one by one, heads as they are
WRITERS = [("plain", dict(nq=4, nkv=2, d=64)), ("plain", dict(nq=4, nkv=2, d=128)), ("plain", dict(nq=6, nkv=3, d=48)),
           ("heads", dict(nq=4, nkv=2, d=64)), ("heads", dict(nq=4, nkv=2, d=40, interleaved=True)), ("gated", dict(nq=4, nkv=2, d=64)),
           ("gated", dict(nq=4, nkv=2, d=24, dv=40, interleaved=True))]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("kind,kw", WRITERS, ids=lambda x: str(x))
def test_a_node_is_what_the_last_token_of_its_path_is(ops, dtype, kind, kw):
    """Through the whole mixer (product, norms, rotation, cache write, attention): a node against a step that brings its path alone."""
    nq, nkv, d, dv, W = kw["nq"], kw["nkv"], kw["d"], kw.get("dv", kw["d"]), 64
    gen = torch.Generator().manual_seed(d)
    rand = lambda *s: torch.randn(*s, generator=gen)
    cols = nq * d + nkv * d + nkv * dv + (nq if kind == "gated" else 0)
    w = (rand(-(-cols // 8) * 8, W) / W ** 0.5).to(dtype).to(DEV)
    rows = [rand(c + len(t), W).to(dtype).to(DEV) for c, t in zip(CTX, TREES)]           # the mixer's input: cached tokens, then nodes
    norm = (rand(d).to(DEV) + 2, rand(d).to(DEV) + 2)
    freq = (torch.exp(-torch.arange(d // 2) / 3.0).to(DEV), d // 2 // 4 * 4 * 2 if d % 8 == 0 else d // 2 * 2, 1.0, kw.get("interleaved", False))
    table = torch.empty(512, d // 2, 2, device=DEV)
    ops.rope_table(table, 1e4, d)
    pages = sum(-(-(c + 16) // PAGE) for c in CTX)
    bt, at = np.full((3, 6), -1), 0
    for b, c in enumerate(CTX):
        k = -(-(c + 16) // PAGE)
        bt[b, :k] = np.arange(at, at + k)[::-1]
        at += k
    bt = i32(bt)

    def run(batch, h, cache, bt):
        out = torch.empty(h.shape[0], nq * dv, dtype=dtype, device=DEV)
        if kind == "plain":
            ops.attend(h, w[:cols].contiguous(), *norm, 1e-6, table, d, batch, bt, cache, 1, PAGE, out, nq, nkv, d, d ** -0.5, 0, True)
        else:
            heads = dict(norm=norm, eps=1e-6, bias=None, values_are_keys=False) if kind == "heads" else None
            ops.attend_gated(h, w, freq, batch, bt, cache, 1, PAGE, out, nq, nkv, d, dv, d ** -0.5, 0, 5.0, True, 0, None, None,
                             nq * d + nkv * (d + dv) if kind == "gated" else -1, True, heads=heads)
        return out.float().cpu()

    cache = torch.full((2, pages + 1, 2, nkv, PAGE, max(d, dv)), float("nan"), dtype=dtype, device=DEV).permute(1, 0, 2, 3, 4, 5)
    run(step_batch([0, 0, 0], CTX), torch.cat([r[:c] for r, c in zip(rows, CTX)]), cache, bt)
    before, counts = cache.clone(), [len(t) for t in TREES]
    batch = step_batch(CTX, counts).with_parents(TREES)
    got = run(batch, torch.cat([r[c:] for r, c in zip(rows, CTX)]), cache, bt)
    row = 0
    for b, (c, tree) in enumerate(zip(CTX, TREES)):
        for i in range(len(tree)):
            path = list(reversed(plain.chain(tree, i)))
            own = before.clone()
            want = run(step_batch([c], [len(path)]), rows[b][[c + j for j in path]].contiguous(), own, bt[b:b + 1].contiguous())[-1]
            # the same products and roundings, other orders of the sums: 64 of them, and for bfloat16 the outputs' rounding and the weights'
            tol = (2.0 ** -17 if dtype == torch.float32 else 2.0 ** -6) * float(got.abs().max())
            assert (got[row] - want).abs().max() <= tol, (b, i)
            # the node's keys and values in its own slot, as the path's last token has them in its position's
            slot, pos = c + i, c + len(path) - 1
            mine, theirs = (x[int(bt[b, s // PAGE]), 1, :, :, s % PAGE] for x, s in ((cache, slot), (own, pos)))
            assert torch.equal(mine[0, :, :d], theirs[0, :, :d]) and torch.equal(mine[1, :, :dv], theirs[1, :, :dv]), (b, i)
            row += 1
    # the cached tokens' slots are as they were
    for b, c in enumerate(CTX):
        for s in range(c):
            p = int(bt[b, s // PAGE])
            assert torch.equal(cache[p, 1, :, :, s % PAGE].nan_to_num(9.0), before[p, 1, :, :, s % PAGE].nan_to_num(9.0))
    ops.check_errors()


def test_large_prompt_portions_as_trees_are_not_fused(ops):
    """A step of so many nodes that the projection would write keys and values in its own epilogue, which knows positions alone."""
    nq, nkv, d, W, n = 8, 2, 128, 256, 250
    gen = torch.Generator().manual_seed(2)
    rng = np.random.default_rng(2)
    w = (torch.randn((nq + 2 * nkv) * d, W, generator=gen) / 16).bfloat16().to(DEV)
    trees = [plain.random_tree(rng, n, spread=30) for _ in range(6)]
    h = torch.randn(6 * n, W, generator=gen).bfloat16().to(DEV)
    table = torch.empty(512, d // 2, 2, device=DEV)
    ops.rope_table(table, 1e4, d)
    bt = i32(np.arange(6 * 16).reshape(6, 16))
    cache = torch.zeros(6 * 16, 1, 2, nkv, 16, d, dtype=torch.bfloat16, device=DEV)
    out = torch.empty(6 * n, nq * d, dtype=torch.bfloat16, device=DEV)
    batch = step_batch([0] * 6, [n] * 6).with_parents(trees)
    ops.attend(h, w, None, None, 0.0, table, d, batch, bt, cache, 0, 16, out, nq, nkv, d, d ** -0.5, 0, True)
    v = (h.float() @ w[(nq + nkv) * d:].float().T).view(6, n, nkv, d)
    held = cache[bt.long()][:, :, 0, 1].permute(0, 1, 3, 2, 4).reshape(6, 256, nkv, d)[:, :n].float()
    assert (held - v).abs().max() <= 2.0 ** -8 * v.abs().max() + 1e-3          # every node's values lie in its own slot
    ops.check_errors()


def test_kernels_that_take_no_trees(ops):
    batch = step_batch([3], [2]).with_parents([[-1, 0]])
    e = lambda *s: torch.zeros(*s, device=DEV)
    cache, bt = e(2, 1, 2, 2, 16, 64), i32([[0]])
    for call in (lambda: ops.attention(e(2, 256), batch, bt, cache, 0, 16, e(2, 256), 4, 2, 64, 0.1, 0),
                 lambda: ops.attention_ext(e(2, 256), batch, bt, cache, 0, 16, e(2, 256), 4, 2, 64, 64, 0.1, 0),
                 lambda: ops.attend_gated(e(2, 64), e(512, 64), None, batch, bt, cache, 0, 16, e(2, 256), 4, 2, 64, 64, 0.1, 0, 0.0, False, 0, None, None, -1,
                                          True, pre=dict(taps=1, norm=None, eps=1e-6))):
        with pytest.raises(KernelError, match="trees"):
            call()
    batch.cache_slots = i32([3])
    with pytest.raises(KernelError, match="cache slots"):
        ops.attend(e(2, 64), e(512, 64), None, None, 0.0, None, 0, batch, bt, cache, 0, 16, e(2, 256), 4, 2, 64, 0.1, 0, True)


def check_paths(run, logits_of, prompts, V, seed, tol, most=24):
    """Prompts, then a step of branching trees: every node's logits; then the draws' path is kept, and the step behind it."""
    rng = np.random.default_rng(seed)
    for r in prompts:
        run.add_request(r)
    run.step([StepEntry(r, p) for r, p in prompts.items()])
    known = {r: list(p) for r, p in prompts.items()}
    for turn in range(2):
        trees = {r: plain.random_tree(rng, int(rng.integers(1, most)), spread=5, padding=2) for r in known}
        tokens = {r: rng.integers(0, V, len(t)).tolist() for r, t in trees.items()}
        batch = run.make_batch([StepEntry(r, tokens[r], range(len(t))) for r, t in trees.items()], parents=list(trees.values()))
        logits = run.run_batch(batch).float().cpu()
        row, drawn = 0, []
        for r, tree in trees.items():
            for i in range(len(tree)):
                path = [tokens[r][j] for j in reversed(plain.chain(tree, i))]
                if path:
                    want = logits_of(known[r] + path)
                    assert (logits[row] - want).abs().max() <= tol * want.abs().max(), (r, i)
                row += 1
            # "draws" that confirm a path down the tree: at every node the token of its last child, where it has one
            child = {p: i for i, p in enumerate(tree) if p >= 0 and plain.chain(tree, i)}
            drawn += [tokens[r][child[i]] if i in child else 0 for i in range(len(tree))]
        B = len(trees)
        path, emitted, count = torch.empty(B, 64, dtype=torch.int32, device=DEV), torch.empty(B, 64, dtype=torch.int32, device=DEV), i32([0] * B)
        run.ops.accept_tree(batch, batch.parents, i32(drawn), path, emitted, count)
        for cache, table in zip(run.kv_caches, batch.block_tables):
            run.ops.keep_path(cache, batch, table, run.ecfg.page_size, path, count)
        for r, p, e, n in zip(trees, path.tolist(), emitted.tolist(), count.tolist()):
            assert n >= 1
            known[r] += [tokens[r][j] for j in p[:n]]
            run.cache.commit(r, n)
    last = {r: int(rng.integers(0, V)) for r in known}
    logits = run.step([StepEntry(r, [t], [0]) for r, t in last.items()]).float().cpu()
    for row, r in enumerate(known):
        want = logits_of(known[r] + [last[r]])
        assert (logits[row] - want).abs().max() <= tol * want.abs().max(), r
    run.ops.check_errors()


@pytest.mark.parametrize("dtype,tol", [("float32", 2e-5), ("bfloat16", 4e-2)])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_models_of_plain_attention(tmp_path, name, dtype, tol):
    d = make_model_dir(tmp_path, name)
    run = ModelRunner(d, EngineConfig(dtype=dtype, page_size=PAGE_SIZE[name], max_cache_tokens=1024, max_live_requests=4))
    pm, rng, V = PlainModel(d), np.random.default_rng(1), tiny_config(name).vocab_size
    prompts = {f"r{i}": rng.integers(0, V, n).tolist() for i, n in enumerate(PROMPT_LENS[name][:3])}
    check_paths(run, lambda t: pm.logits(t)[-1].float(), prompts, V, 3, tol)


@pytest.mark.parametrize("dtype,tol", [("float32", 3e-5), ("bfloat16", 5e-2)])
@pytest.mark.parametrize("dim,streams", [(64, 3), (24, 0)])
def test_models_of_gated_attention(dtype, tol, dim, streams):
    """Windows, caps, sinks, gates, values mixed across layers, several residual streams; heads of 64 and of a size the tensor cores do not take."""
    rot = RotaryConfig(1e4, dim // 2)
    att = lambda window, mix, ff: TipezenLayer(type="attention", heads=4, kv_heads=2, dim=dim, vdim=dim, window=window, rot=rot, v_mix=mix, softcap=20.0,
                                               scale=dim ** -0.5, ff=ff)
    cfg = TipezenConfig("Tipezen", vocab_size=320, hidden_size=128, streams=streams, norm_eps=1e-5, layers=(att(24, True, 128), att(200, True, 0), att(9, True, 96)))
    sd = random_state_dict(cfg, 11, "bfloat16", norm_noise=0.2)
    run = ModelRunner(config=cfg, tensors=dict(sd), engine_config=EngineConfig(dtype=dtype, page_size=8, max_cache_tokens=1024, max_live_requests=4))
    rng, cj = np.random.default_rng(1), cfg.to_json_dict()
    prompts = {f"r{i}": rng.integers(0, 320, n).tolist() for i, n in enumerate((5, 70, 33))}
    check_paths(run, lambda t: plain_tipezen.forward(cj, sd, t)[-1].float(), prompts, 320, 3, tol, most=12)


def test_a_model_of_other_mixers_is_refused():
    cfg = TipezenConfig("Tipezen", vocab_size=64, hidden_size=64, streams=0, norm_eps=1e-5, layers=(
        TipezenLayer(type="retention", heads=2, dim=32, vdim=32, decay=(0.9, 0.99), ff=64),))
    run = ModelRunner(config=cfg, tensors=dict(random_state_dict(cfg, 1, "bfloat16")), engine_config=EngineConfig(dtype="float32", max_cache_tokens=256))
    run.add_request("a")
    with pytest.raises(RequestError, match="retention"):
        run.make_batch([StepEntry("a", [1, 2])], parents=[[-1, 0]])


def test_generation_over_trees_gives_the_tokens_of_single_steps(tmp_path):
    """A whole model checks drafted trees under penalties; some drafts are right, some wrong: the tokens are those of ordinary generation."""
    name, goal = "C", 30
    d, V = make_model_dir(tmp_path, name), tiny_config(name).vocab_size
    config = EngineConfig(dtype="float32", page_size=PAGE_SIZE[name], max_cache_tokens=1024, max_live_requests=4)
    rng = np.random.default_rng(8)
    prompts = [rng.integers(0, V, n).tolist() for n in (4, 19, 60)]
    from tffinfer_b200.sampling import SamplingParams
    settings = (1.3, 0.25, 0.125)
    single = Engine(d, config).generate(prompts, SamplingParams(max_new_tokens=goal, repetition_penalty=settings[0], frequency_penalty=settings[1],
                                                                presence_penalty=settings[2]))
    run = ModelRunner(d, config)
    for b in range(3):
        run.add_request(b)
    made, held, steps = [[] for _ in prompts], [list(p) for p in prompts], 0
    for b, p in enumerate(prompts):                    # all of a prompt but its last token, which is the first tree's root
        run.step([StepEntry(b, p[:-1])])
    while min(len(m) for m in made) < goal:
        steps += 1
        trees, tokens = [], []
        for b in range(3):
            ahead = single[b][len(made[b]):len(made[b]) + 3]
            right = [t if (steps + b) % 3 else (t + 1) % V for t in ahead]
            tree, words = [-1], [held[b][-1]]
            at = 0
            for t in right:                            # a wrong sibling ahead of each drafted token
                tree += [at, at]
                words += [(t + 7) % V, t]
                at = len(tree) - 1
            trees.append(tree)
            tokens.append(words)
        batch = run.make_batch([StepEntry(b, w, range(len(w))) for b, w in enumerate(tokens)], parents=trees)
        logits = run.run_batch(batch)
        past = [prompts[b] + made[b] for b in range(3)]
        prompt_len = [len(p) for p in prompts]
        # a tree's root is the last token of the history already: the kernel counts it on every row's path
        past = [h[:-1] for h in past]
        prompt_len = [min(n, len(h)) for n, h in zip(prompt_len, past)]
        start = np.cumsum([0] + [len(h) for h in past])
        c = LogitControls(batch.q_start, torch.tensor([settings] * 3, device=DEV), i32(np.concatenate(past)), i32(start[:-1]), i32([len(h) for h in past]),
                          i32(prompt_len), parents=batch.parents, tokens=batch.token_ids)
        out = torch.empty_like(logits)
        if steps == 1:                                 # (the first root is a prompt's token: it has not been generated)
            rows, first = batch.q_start[:-1].long(), LogitControls(
                i32(range(4)), torch.tensor([settings] * 3, device=DEV), i32(np.concatenate(prompts)), i32(np.cumsum([0] + [len(p) for p in prompts])[:-1]),
                i32([len(p) for p in prompts]), i32([len(p) for p in prompts]))
            out = logits[rows].contiguous()
            run.ops.control_logits(out, out, first)
            drawn = torch.empty(3, dtype=torch.int32, device=DEV)
            run.ops.argmax(out, drawn)
            for b, t in enumerate(drawn.tolist()):
                run.cache.commit(b, 1)
                made[b].append(t)
                held[b].append(t)
            continue
        run.ops.control_logits(logits, out, c)
        drawn = torch.empty(out.shape[0], dtype=torch.int32, device=DEV)
        run.ops.argmax(out, drawn)
        path, emitted, count = torch.empty(3, 8, dtype=torch.int32, device=DEV), torch.empty(3, 8, dtype=torch.int32, device=DEV), i32([0] * 3)
        run.ops.accept_tree(batch, batch.parents, drawn, path, emitted, count)
        for cache, table in zip(run.kv_caches, batch.block_tables):
            run.ops.keep_path(cache, batch, table, run.ecfg.page_size, path, count)
        for b, (e, n) in enumerate(zip(emitted.tolist(), count.tolist())):
            run.cache.commit(b, n)
            made[b] += e[:n]
            held[b] += e[:n]
    assert [m[:goal] for m in made] == single and steps < goal * 0.7
    run.ops.check_errors()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 48])
def test_arrays_of_a_larger_step_write_nothing_behind_this_one(ops, dtype, d):
    """A captured step whose arrays are exchanged for those of more nodes than it has rows: the rows that it has are right, those behind stay."""
    nq, nkv, T = 4, 2, 11
    gen = torch.Generator().manual_seed(d)
    rand = lambda *s: torch.randn(*s, generator=gen).to(dtype).to(DEV)
    cache, bt = rand(16, 1, 2, nkv, 16, d), i32(np.arange(16).reshape(4, 4))
    trees = [[-1, 0, 0], [-1, 0, 1, 1, 0], [-1, 0, 0, 1, 1, 2], [-1, 0]]        # 16 nodes: three of the third request's rows are there
    q, parents = rand(T, nq * d), i32(np.concatenate(trees)[:T])
    ctx, n = [5, 30, 20, 9], [len(t) for t in trees]
    for part in (dict(), dict(whole=0), dict(splits=2)):
        tc, general = ops._attention_tree_tc, ops._attention_tree_plain
        try:
            if "whole" in part:
                ops._attention_tree_tc = lambda *a: tc(*a, whole=0, least=1)
            if "splits" in part:
                ops._attention_tree_tc = lambda *a: False
                ops._attention_tree_plain = lambda *a: general(*a, splits=2)
            outs = []
            for counts in (n, [3, 5, 3]):
                batch = step_batch(ctx[:len(counts)], counts)
                store = torch.full((T + 8, nq * d), 7.0, dtype=dtype, device=DEV)
                ops.attention_tree(q, batch, parents, bt, cache, 0, 16, store[:T], nq, nkv, d, d, d ** -0.5)
                torch.cuda.synchronize()
                ops.check_errors()
                assert (store[T:] == 7).all()
                outs.append(store[:T].float())
            assert (outs[0] - outs[1]).abs().max() <= (2.0 ** -17 if dtype == torch.float32 else 2.0 ** -6) * outs[1].abs().max()
        finally:
            for name in ("_attention_tree_tc", "_attention_tree_plain"):
                ops.__dict__.pop(name, None)
