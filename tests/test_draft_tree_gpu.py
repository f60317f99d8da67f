"""Trees of drafted tokens on the GPU against plain implementations in 64 bits: attention over the cache, the walk that
accepts, the move of the accepted nodes' slots, and the controls of their logits."""
import math

import numpy as np
import pytest
import torch

import plain_tree as plain
from tffinfer_b200.kernels.library import CudaKernels, KernelError
from tffinfer_b200.sampling import LogitControls

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    return CudaKernels()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def tree_case(seed, dtype, nq, nkv, d, dv, page, ctx, nodes, padding=0, layers=2, layer=1, major=True):
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    trees = [plain.random_tree(rng, n, padding=padding if b % 2 == 0 else 0) for b, n in enumerate(nodes)]
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64).to(dtype).double()
    keys = [rand(c + n, nkv, d) for c, n in zip(ctx, nodes)]
    values = [rand(c + n, nkv, dv) for c, n in zip(ctx, nodes)]
    T = sum(nodes)
    q = rand(T, nq, d)
    held_k, held_v, held_q, t = [], [], q.clone(), 0
    for b, parents in enumerate(trees):            # what padding nodes bring is anything
        k, v = keys[b].clone(), values[b].clone()
        for i in range(len(parents)):
            if not plain.chain(parents, i):
                k[ctx[b] + i] = v[ctx[b] + i] = math.nan
                held_q[t] = math.nan
            t += 1
        held_k.append(k)
        held_v.append(v)
    cache, table = plain.paged(held_k, held_v, page, DEV, dtype, layers, layer, major, seed)
    batch = plain.step(ctx, trees, DEV)
    parents = i32(np.concatenate([np.asarray(t, dtype=np.int64) for t in trees] or [[]]))
    return dict(trees=trees, keys=keys, values=values, q=q, cache=cache, table=table, batch=batch, parents=parents, layer=layer, ctx=ctx,
                flat_q=held_q.reshape(T, nq * d).to(dtype).to(DEV), dtype=dtype, shape=(nq, nkv, d, dv), page=page)


def run_tree(ops, c, scale, rows_behind=3, **kw):
    nq, nkv, d, dv = c["shape"]
    T = c["flat_q"].shape[0]
    store = torch.full((T + rows_behind, nq * dv), 7.0, dtype=c["dtype"], device=DEV)
    ops.attention_tree(c["flat_q"], c["batch"], c["parents"], c["table"], c["cache"], c["layer"], c["page"], store[:T], nq, nkv, d, dv,
                       scale, **kw)
    torch.cuda.synchronize()
    ops.check_errors()
    assert (store[T:] == 7).all()
    return store[:T].view(T, nq, dv)


def check_tree(got, c, scale, **kw):
    nq, _, d, _ = c["shape"]
    kw["sink"] = kw.get("sink").cpu() if isinstance(kw.get("sink"), torch.Tensor) else torch.zeros(nq) if kw.get("sink") else None
    if kw.get("gates") is not None:
        kw["gates"] = kw["gates"].cpu()
    want, size, most = plain.attention(c["q"], c["keys"], c["values"], c["ctx"], c["trees"], nq, scale, **kw)
    got = got.cpu().double()
    longest = max(k.shape[0] for k in c["keys"])
    # float32: a score is off by (d + 4) roundings of the sum of its terms' sizes, a weight by twice that and the roundings of its
    # exponential and of the sums; sums of ``longest`` terms; the cap's tanh by a few roundings of the cap
    u = 2.0 ** -24
    score = (d + 4) * u * most + 8 * u * kw.get("softcap", 0.0)
    tol = size * (4 * score + (longest + 32) * 2 * u) + 1e-30
    if c["dtype"] == torch.bfloat16:
        # weights and results rounded to bfloat16 (2^-8 at most); the tensor core adds products of 24 bits (truncated: twice u)
        tol = 2 * tol + 2.0 ** -8 * (want.abs() + size) * 1.01 + 2.0 ** -17 * size
    assert torch.isfinite(got).all()
    worst = ((got - want).abs() / tol).max()
    assert worst <= 1, float(worst)
    t = 0
    for parents in c["trees"]:                     # padding gives zeros
        for i in range(len(parents)):
            if not plain.chain(parents, i):
                assert (got[t] == 0).all()
            t += 1


HEADS = [(4, 4, 64, 64), (8, 2, 128, 128), (10, 2, 128, 128), (16, 2, 64, 64), (3, 1, 128, 128), (16, 8, 128, 128)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("nq,nkv,d,dv", HEADS + [(4, 2, 80, 80), (6, 3, 40, 24), (2, 2, 9, 7), (4, 1, 192, 160), (2, 1, 512, 300)])
def test_head_layouts(ops, dtype, nq, nkv, d, dv):
    c = tree_case(nq * d, dtype, nq, nkv, d, dv, 16, [70, 0, 131], [9, 5, 1], padding=2)
    check_tree(run_tree(ops, c, d ** -0.5), c, d ** -0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ctx,nodes", [
    ([0], [1]), ([0], [64]), ([1], [2]), ([63], [1]), ([64], [1]), ([65], [66]), ([62], [7]), ([300], [256]), ([5, 1000, 0, 64], [0, 3, 12, 33]),
    ([2300], [16]), ([1023, 17, 513, 2], [31, 64, 1, 100]), ([127, 128, 129], [128, 127, 129])], ids=str)
def test_lengths(ops, dtype, ctx, nodes):
    c = tree_case(sum(ctx) + sum(nodes), dtype, 8, 2, 128, 128, 16, ctx, nodes, padding=3)
    check_tree(run_tree(ops, c, 0.09), c, 0.09)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page", [1, 8, 10, 16, 32, 64, 128])
def test_pages(ops, dtype, page):
    c = tree_case(page, dtype, 8, 2, 64, 64, page, [100, 37], [20, 41], padding=2, major=page % 16 != 0)
    check_tree(run_tree(ops, c, 0.125), c, 0.125)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("kw", [
    dict(window=1), dict(window=3), dict(window=64), dict(window=200), dict(window=40, keep=5), dict(window=2, keep=130), dict(softcap=5.0),
    dict(sink=True), dict(sink="learned"), dict(gates=True), dict(window=70, keep=4, softcap=8.0, sink="learned", gates=True)], ids=str)
def test_what_designs_add(ops, dtype, kw):
    nq = 8
    c = tree_case(len(str(kw)), dtype, nq, 2, 128, 128, 16, [150, 0, 128, 390], [40, 9, 17, 65], padding=3)
    kw = dict(kw)
    gen = torch.Generator().manual_seed(1)
    if kw.get("sink") == "learned":
        kw["sink"] = torch.randn(nq, generator=gen).to(DEV)
    if kw.get("gates"):
        kw["gates"] = torch.rand(c["flat_q"].shape[0], nq, generator=gen).to(DEV)
    check_tree(run_tree(ops, c, 0.1, **kw), c, 0.1, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_pages_that_a_window_has_given_back(ops, dtype):
    c = tree_case(5, dtype, 8, 2, 128, 128, 16, [500], [20])
    c["table"][0, :(500 - 100 + 1) // 16] = -1      # below the window's first page: given back (the first two are kept)
    free = sorted(set(range(c["cache"].shape[0])) - set(c["table"][0].tolist()))
    c["table"][0, :2] = torch.tensor(free[:2], dtype=torch.int32)
    for kind, held in ((0, c["keys"]), (1, c["values"])):
        for j in range(2):
            c["cache"][free[j], c["layer"], kind] = held[0][j * 16:(j + 1) * 16].transpose(0, 1).to(dtype).to(DEV)
    check_tree(run_tree(ops, c, 0.1, window=100, keep=20), c, 0.1, window=100, keep=20)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_parents_that_are_none(ops, dtype):
    """A parent behind its node, the node itself, numbers far outside: the node is not there, nor is what follows it."""
    c = tree_case(3, dtype, 4, 2, 128, 128, 16, [33, 90], [12, 10])
    bad = [[-1, 0, 5, 3, 2, 0, 1 << 20, 6, -1, 8, -7, 10], [3, -1, 1, 2, 99, -(1 << 31), 2, (1 << 31) - 1, -1, 9]]
    c["trees"], c["parents"] = bad, i32(np.concatenate(bad))
    check_tree(run_tree(ops, c, 0.1), c, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_chain_is_causal_attention(ops, dtype):
    c = tree_case(8, dtype, 8, 2, 128, 128, 16, [100, 300], [40, 9])
    c["trees"] = [list(range(-1, n - 1)) for n in (40, 9)]
    c["parents"] = i32(np.concatenate(c["trees"]))
    check_tree(run_tree(ops, c, 0.1), c, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_many_requests_and_a_long_one(ops, dtype):
    rng = np.random.default_rng(2)
    ctx = [int(x) for x in rng.integers(0, 90, 150)] + [4000]
    nodes = [int(x) for x in rng.integers(0, 6, 150)] + [30]
    c = tree_case(4, dtype, 8, 2, 64, 64, 16, ctx, nodes)
    check_tree(run_tree(ops, c, 0.1), c, 0.1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_scores(ops, dtype):
    """Weights between 1 and nothing: the maximum moves far from block to block."""
    c = tree_case(11, dtype, 8, 2, 128, 128, 16, [400], [20])
    ramp = torch.linspace(0.1, 12, 420, dtype=torch.float64)[:, None, None]
    for order in (ramp, ramp.flip(0)):
        c["keys"] = [(c["keys"][0] / c["keys"][0].abs().amax() * order).to(dtype).double()]
        c["cache"], c["table"] = plain.paged(c["keys"], c["values"], 16, DEV, dtype)
        check_tree(run_tree(ops, c, 1.0), c, 1.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_streams_graphs_and_repeated_calls(ops, dtype):
    """Captured and replayed behind new contexts and trees, twice over at once, and on another stream: the same bits."""
    a = tree_case(21, dtype, 8, 2, 128, 128, 16, [700, 60], [20, 33])
    b = tree_case(22, dtype, 8, 2, 128, 128, 16, [650, 90], [24, 29])
    want = [run_tree(ops, c, 0.1) for c in (a, b)]
    side = torch.cuda.Stream()
    outs = [torch.empty(53, 1024, dtype=dtype, device=DEV) for _ in range(2)]
    call = lambda c, out: ops.attention_tree(c["flat_q"], c["batch"], c["parents"], c["table"], c["cache"], 1, 16, out, 8, 2, 128, 128, 0.1)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            call(b, outs[1])
        call(a, outs[0])
    torch.cuda.synchronize()
    assert torch.equal(outs[0].view_as(want[0]), want[0]) and torch.equal(outs[1].view_as(want[1]), want[1])
    # one graph, its inputs exchanged between replays (max_kv_len of the captured batch bounds both)
    a["batch"].graph_bucket = 2
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call(a, outs[0])
    for src, expect in ((a, want[0]), (b, want[1]), (a, want[0])):
        held = {k: a[k].clone() for k in ("flat_q", "parents", "table")}
        arrays = {k: getattr(a["batch"], k).clone() for k in ("q_start", "pos_start")}
        cache = a["cache"].clone()
        if src is b:
            width = min(a["table"].shape[1], b["table"].shape[1])
            a["table"][:, :width].copy_(b["table"][:, :width])
            a["flat_q"].copy_(b["flat_q"]), a["parents"].copy_(b["parents"])
            for k in arrays:
                getattr(a["batch"], k).copy_(getattr(b["batch"], k))
            pages = b["cache"].shape[0]
            assert pages <= a["cache"].shape[0]
            a["cache"][:pages].copy_(b["cache"])
        g.replay()
        torch.cuda.synchronize()
        err = (outs[0].view_as(expect).double() - expect.double()).abs().max()
        assert err <= (2.0 ** -6 if dtype == torch.bfloat16 else 2.0 ** -18) * expect.double().abs().max()
        for k, t in held.items():
            a[k].copy_(t)
        for k, t in arrays.items():
            getattr(a["batch"], k).copy_(t)
        a["cache"].copy_(cache)
    ops.check_errors()


def test_tree_refusals(ops):
    c = tree_case(1, torch.bfloat16, 8, 2, 128, 128, 16, [30], [5])
    out = torch.empty(5, 1024, dtype=torch.bfloat16, device=DEV)
    def call(**kw):
        a = dict(q=c["flat_q"], parents=c["parents"], table=c["table"], cache=c["cache"], layer=1, page=16, out=out, nq=8, nkv=2, d=128, dv=128)
        a.update(kw)
        ops.attention_tree(a["q"], a.get("batch", c["batch"]), a["parents"], a["table"], a["cache"], a["layer"], a["page"], a["out"],
                           a["nq"], a["nkv"], a["d"], a["dv"], 0.1)
    call()
    big = plain.step([3], [[-1] * 257], DEV)
    for kw in (dict(parents=c["parents"][:4]), dict(parents=c["parents"].long()), dict(parents=c["parents"].cpu()), dict(layer=2), dict(layer=-1),
               dict(out=out.float()), dict(out=out[:4]), dict(q=c["flat_q"].float()), dict(page=8), dict(nkv=4), dict(d=64), dict(dv=64),
               dict(table=c["table"].long()), dict(cache=c["cache"].float()), dict(table=c["table"][:0]),
               dict(batch=big, parents=i32([-1] * 257), q=torch.zeros(257, 1024, dtype=torch.bfloat16, device=DEV),
                    out=torch.zeros(257, 1024, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(KernelError):
            call(**kw)


# ------------------------------------------------------------------ acceptance

@pytest.mark.parametrize("nodes,width,vocab", [([1], 4, 5), ([0, 3, 0], 8, 2), ([256, 255, 33, 32, 31], 40, 3), ([7] * 300, 5, 2),
                                               ([64] * 20, 64, 1), ([100, 1], 1, 2)], ids=str)
def test_acceptance(ops, nodes, width, vocab):
    rng = np.random.default_rng(len(nodes) + width)
    trees = [plain.random_tree(rng, n, padding=n // 5) for n in nodes]
    tokens, drawn = rng.integers(0, vocab, sum(nodes)), rng.integers(0, vocab, sum(nodes))
    batch = plain.step([3] * len(nodes), trees, DEV, tokens)
    B = len(nodes)
    path, emitted, count = (torch.full(s, 9, dtype=torch.int32, device=DEV) for s in ((B + 1, width), (B + 1, width), (B + 1,)))
    ops.accept_tree(batch, i32(np.concatenate(trees)), i32(drawn), path[:B], emitted[:B], count[:B])
    want = plain.accept(trees, tokens, drawn, width)
    assert [path[:B].tolist(), emitted[:B].tolist(), count[:B].tolist()] == [list(x) for x in want]
    assert (path[B] == 9).all() and (emitted[B] == 9).all() and count[B] == 9


def test_acceptance_of_trees_without_a_root(ops):
    trees, tokens, drawn = [[-2, 0, 0], [0, 0], [-1, 0, 7, 1, -5]], [1] * 10, [1] * 10
    batch = plain.step([0] * 3, trees, DEV, tokens)
    path, emitted = (torch.zeros(3, 6, dtype=torch.int32, device=DEV) for _ in range(2))
    count = torch.zeros(3, dtype=torch.int32, device=DEV)
    ops.accept_tree(batch, i32(np.concatenate(trees)), i32(drawn), path, emitted, count)
    assert count.tolist() == [0, 0, 3] and path[2].tolist() == [0, 1, 3, -1, -1, -1] and (path[:2] == -1).all()
    for bad in (dict(drawn=i32(drawn[:9])), dict(drawn=i32(drawn).long()), dict(path=path[:2]), dict(emitted=emitted[:, :5]), dict(count=count[:2])):
        a = dict(drawn=i32(drawn), path=path, emitted=emitted, count=count)
        a.update(bad)
        with pytest.raises(KernelError):
            ops.accept_tree(batch, i32(np.concatenate(trees)), a["drawn"], a["path"], a["emitted"], a["count"])


# ------------------------------------------------------------------ the accepted nodes' slots

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("page,heads,size,planes,layers,major", [(16, 2, 64, 2, 3, True), (8, 3, 40, 2, 2, False), (5, 1, 7, 1, 4, True),
                                                                 (64, 8, 128, 2, 5, True), (16, 4, 2, 2, 1, False)])
def test_slots_are_kept(ops, dtype, page, heads, size, planes, layers, major):
    rng, gen = np.random.default_rng(size), torch.Generator().manual_seed(size)
    ctx, nodes = [0, page - 1, 3 * page, 70, 11], [30, 40, 1, 21, 0]
    need = [-(-(c + n) // page) for c, n in zip(ctx, nodes)]
    pages = sum(need) + 2
    order, table, at = rng.permutation(pages), np.full((5, max(need)), -1), 0
    for b in range(5):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    cache = torch.randn((layers, pages, planes, heads, page, size) if major else (pages, layers, planes, heads, page, size), generator=gen).to(dtype).to(DEV)
    view = cache.permute(1, 0, 2, 3, 4, 5) if major else cache
    want = view.clone()
    path, count = np.full((5, 12), -1), [0] * 5
    for b, n in enumerate(nodes):
        if n:
            chosen = sorted({0, *rng.choice(n, min(n, 11), replace=False).tolist()})
            path[b, :len(chosen)], count[b] = chosen, len(chosen)
        for j in range(count[b]):
            src, dst = ctx[b] + path[b, j], ctx[b] + j
            want[table[b, dst // page], :, :, :, dst % page] = view[table[b, src // page], :, :, :, src % page]
    batch = plain.step(ctx, [[-1] * n for n in nodes], DEV)
    ops.keep_path(view, batch, i32(table), page, i32(path), i32(count))
    assert torch.equal(view, want)


def test_slots_of_paths_that_are_none(ops):
    """Slots behind the table, without a page, before the sequence; a count that is more than the path holds: nothing is moved there."""
    cache = torch.randn(4, 2, 2, 1, 8, 16, device=DEV)
    before, batch = cache.clone(), plain.step([6, 3, 0], [[-1] * 9] * 3, DEV)
    table = i32([[0, 1], [2, -1], [77, -5]])
    path, count = i32([[0, 500, -3, 1 << 30], [0, 6, 7, 8], [0, 5, 6, 9]]), i32([99, 4, 4])
    ops.keep_path(cache, batch, table, 8, path, count)
    assert torch.equal(cache, before)
    for bad in (dict(path=path[:2]), dict(count=count[:2]), dict(path=path.long()), dict(page=16), dict(table=table[:2]), dict(cache=cache[0]),
                dict(cache=cache.transpose(4, 5)), dict(cache=cache[..., :8]), dict(cache=cache.cpu())):
        a = dict(table=table, page=8, path=path, count=count, cache=cache)
        a.update(bad)
        with pytest.raises(KernelError):
            ops.keep_path(a["cache"], batch, a["table"], a["page"], a["path"], a["count"])


# ------------------------------------------------------------------ the controls of logits

def controls_case(seed, V, rows, tree=False, history=(0, 40), masked=True, biases=5, words_spare=0, repeat=False):
    """(logits, LogitControls' fields, what plain.control takes)."""
    rng, gen = np.random.default_rng(seed), torch.Generator().manual_seed(seed)
    R, B = sum(rows), len(rows)
    logits = torch.randn(R, V, generator=gen) * 4
    few = max(2, min(V, 12))
    requests, hist, start = [], [], []
    tokens = rng.integers(0, few, R)
    for b, n in enumerate(rows):
        h = rng.integers(-2 if b % 3 == 0 else 0, few, rng.integers(history[0], history[1] + 1)).tolist() + ([V - 1, V, V + 7] if b % 2 else [])
        setting = [(1.0, 0.0, 0.0), (1.3, 0.25, 0.5), (0.7, -0.3, 0.0), (1.0, 0.0, -0.4)][b % 4]
        some = sorted(rng.choice(min(V, 4 * few), min(V, biases), replace=repeat).tolist()) if b != 1 else []
        values = [-math.inf if rng.random() < 0.2 else float(np.float32(rng.normal())) for _ in some]
        requests.append((n, setting, h, int(rng.integers(0, len(h) + 1)), list(zip(some, values))))
        start.append(len(hist))
        hist += h
    c = dict(row_start=i32(np.concatenate([[0], np.cumsum(rows)])), settings=torch.tensor([r[1] for r in requests], device=DEV),
             history=i32(hist), history_start=i32(start), history_len=i32([len(r[2]) for r in requests]), prompt_len=i32([r[3] for r in requests]))
    if biases:
        flat = [x for r in requests for x in r[4]]
        c.update(bias_start=i32(np.concatenate([[0], np.cumsum([len(r[4]) for r in requests])])), bias_tokens=i32([t for t, _ in flat]),
                 bias_values=torch.tensor([v for _, v in flat], dtype=torch.float32, device=DEV))
    trees = masks = None
    if masked:
        words = -(-V // 32) + words_spare
        bits = rng.random((R // 2 + 1, words * 32)) < 0.5
        bits[0] = False                            # a state that allows nothing
        which = [int(rng.integers(-1, bits.shape[0])) for _ in range(R)]
        which[0] = 0
        masks = [bits[w, :V] if w >= 0 else None for w in which]
        c.update(mask=torch.from_numpy(np.packbits(bits, axis=1, bitorder="little").view(np.int32).copy()).to(DEV), mask_row=i32(which))
    if tree:
        trees = [plain.random_tree(rng, n, padding=n // 4) for n in rows]
        c.update(parents=i32(np.concatenate(trees)), tokens=i32(tokens))
    return logits, c, (requests, trees, tokens, masks)


def check_control(got, logits, given):
    want = plain.control(logits, *given)
    got = got.cpu().double()
    assert torch.equal(torch.isinf(got), torch.isinf(want)) and not torch.isnan(got).any()
    fine = torch.isfinite(want)
    # a rounding of each of up to five steps, none of whose values is larger than |x| * 1.5 + 40 * 0.3 + 0.5 + the biases
    tol = 5 * 2.0 ** -24 * (1.5 * logits.abs().double() + 60 * 0.3 + 0.5 + 30)
    assert ((got - want).abs() <= tol)[fine].all()
    same = fine & (want == logits.double())
    assert torch.equal(got[same], logits.double()[same])       # what no control touches keeps its bits


@pytest.mark.parametrize("V", [1, 2, 31, 33, 1000, 4097, 32768, 151936])
@pytest.mark.parametrize("rows,tree", [([1], False), ([1, 1, 1, 1, 1], False), ([3, 0, 17, 2], True), ([2, 1], False)], ids=str)
def test_controls(ops, V, rows, tree):
    logits, c, given = controls_case(V + len(rows), V, rows, tree)
    dev, out = logits.to(DEV), torch.full((sum(rows) + 1, V), 5.0, device=DEV)
    ops.control_logits(dev, out[:-1], LogitControls(**c))
    check_control(out[:-1], logits, given)
    assert (out[-1] == 5).all() and torch.equal(dev.cpu(), logits)
    if not tree:                                   # in place
        ops.control_logits(dev, dev, LogitControls(**c))
        assert torch.equal(dev, out[:-1])


@pytest.mark.parametrize("kw", [dict(masked=False), dict(biases=0), dict(masked=False, biases=0), dict(history=(0, 0)), dict(history=(3000, 5000)),
                                dict(biases=40, repeat=True), dict(words_spare=3), dict(tree=True, history=(0, 0), biases=30, repeat=True)], ids=str)
def test_what_controls_leave_out(ops, kw):
    logits, c, given = controls_case(77, 5003, [1, 2, 1, 4, 1], **{"tree": False, **kw})
    if kw.get("history") == (3000, 5000):          # up to 5,000 of one token: a larger bound than check_control's
        c["settings"][:, 1] *= 0.01
        given[0][:] = [(n, (s[0], float(np.float32(s[1]) * np.float32(0.01)), s[2]), h, p, b) for n, s, h, p, b in given[0]]
    out = torch.empty_like(logits, device=DEV)
    ops.control_logits(logits.to(DEV), out, LogitControls(**c))
    check_control(out, logits, given)


@pytest.mark.parametrize("V", [601, 40961])
def test_counts_of_long_histories(ops, V):
    # more tokens than 15 bits count, one of them most of the time; a request of few beside it
    rng = np.random.default_rng(V)
    logits = torch.randn(5, V, generator=torch.Generator().manual_seed(V)) * 4
    long = rng.permutation(np.concatenate([np.full(33000, V - 2), rng.integers(0, V, 7000)])).tolist()
    settings = [(1.2, float(np.float32(2e-4)), 0.5), (1.1, 0.25, 0.0)]
    trees, tokens = [[-1, 0, 0], [-1, 0]], np.array([V - 2, V - 2, 5, 3, 4])
    requests = [(3, settings[0], long, 300, [(V - 2, 1.0)]), (2, settings[1], [3, 4, 3], 1, [])]
    for tree in (False, True):
        c = LogitControls(i32([0, 3, 5]), torch.tensor(settings, device=DEV), i32(long + [3, 4, 3]), i32([0, len(long)]), i32([len(long), 3]), i32([300, 1]),
                          i32([0, 1, 1]), i32([V - 2]), torch.tensor([1.0], device=DEV), parents=i32(trees[0] + trees[1]) if tree else None,
                          tokens=i32(tokens) if tree else None)
        out = torch.empty_like(logits, device=DEV)
        ops.control_logits(logits.to(DEV), out, c)
        check_control(out, logits, (requests, trees if tree else None, tokens, None))


def test_controls_of_the_largest_tree_and_of_rows_behind_the_last(ops):
    logits, c, given = controls_case(3, 700, [256, 0, 1], True)
    wide = torch.cat([logits, torch.full((2, 700), math.nan)]).to(DEV)
    out = torch.full((259, 700), 3.0, device=DEV)
    c["mask_row"], c["parents"], c["tokens"] = (torch.cat([c[k], i32([0, 0])]) for k in ("mask_row", "parents", "tokens"))
    ops.control_logits(wide, out, LogitControls(**c))
    check_control(out[:257], logits, given)
    assert (out[257:] == 3).all()


def test_special_logits(ops):
    logits = torch.tensor([[math.inf, -math.inf, 0.0, -0.0, 1e38, -3e38, math.nan, 2.0]], device=DEV)
    c = LogitControls(i32([0, 1]), torch.tensor([[2.0, 0.5, 0.25]], device=DEV), i32([0, 1, 2, 3, 4, 5]), i32([0]), i32([6]), i32([0]),
                      i32([0, 1]), i32([7]), torch.tensor([-math.inf], device=DEV), i32([[0b10111111]]))
    out = torch.empty_like(logits)
    ops.control_logits(logits, out, c)
    assert out[0, :6].tolist() == [math.inf, -math.inf, -0.75, -0.75, float(np.float32(np.float32(1e38) / 2)), -math.inf]
    assert out[0, 6] == -math.inf and out[0, 7] == -math.inf     # a banned NaN, a banned token


def test_control_refusals(ops):
    logits, c, _ = controls_case(5, 100, [2, 3], True)
    dev, out = logits.to(DEV), torch.empty(5, 100, device=DEV)
    ops.control_logits(dev, out, LogitControls(**c))
    cut = lambda k: {k: c[k][:-1].contiguous()}
    for bad in (cut("row_start"), cut("settings"), cut("history_len"), cut("prompt_len"), cut("history_start"), cut("bias_start"), cut("bias_values"),
                cut("mask_row"), cut("parents"), cut("tokens"), dict(mask=c["mask"][:, :3].contiguous()), dict(mask=None), dict(tokens=None), dict(parents=None),
                dict(bias_start=None), dict(settings=c["settings"].double()), dict(history=c["history"].long()), dict(tokens=c["tokens"].cpu())):
        with pytest.raises(KernelError):
            ops.control_logits(dev, out, LogitControls(**{**c, **bad}))
    for a, b in ((dev, dev), (dev.bfloat16(), out), (dev, out.double()), (dev, out[:4]), (dev[:, ::2], out[:, ::2])):
        with pytest.raises(KernelError):
            ops.control_logits(a, b, LogitControls(**c))
    plain_c = LogitControls(**{k: v for k, v in c.items() if k not in ("parents", "tokens")})
    store = torch.zeros(6, 100, device=DEV)
    with pytest.raises(KernelError):                # the outputs overlap the logits one row on
        ops.control_logits(store[:5], store[1:], plain_c)


def test_empty_steps(ops):
    e = torch.empty
    batch = plain.step([], [], DEV)
    none = i32([])
    ops.attention_tree(e(0, 256, device=DEV), batch, none, i32(np.zeros((0, 4))), e(3, 1, 2, 2, 16, 64, device=DEV), 0, 16, e(0, 256, device=DEV), 4, 2, 64,
                       64, 0.1)
    ops.accept_tree(batch, none, none, i32(np.zeros((0, 4))), i32(np.zeros((0, 4))), none)
    ops.keep_path(e(3, 1, 2, 2, 16, 64, device=DEV), batch, i32(np.zeros((0, 4))), 16, i32(np.zeros((0, 4))), none)
    ops.control_logits(e(0, 50, device=DEV), e(0, 50, device=DEV), LogitControls(i32([0]), e(0, 3, device=DEV), none, none, none, none))
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_tables_without_a_page(ops, dtype):
    """A table that ends early or has no page in its middle: nothing is read there (keys and values of zeros); the other request is as ever."""
    c = tree_case(31, dtype, 8, 2, 128, 128, 16, [100, 70], [9, 12])
    check_tree(run_tree(ops, c, 0.1), c, 0.1)
    lost = lambda b, lo, hi: [x[b][lo:hi].zero_() for x in (c["keys"], c["values"])]
    c["table"][0, 2] = -1
    lost(0, 32, 48)
    check_tree(run_tree(ops, c, 0.1), c, 0.1)
    c["table"][1, 0] = c["cache"].shape[0] + 5
    lost(1, 0, 16)
    check_tree(run_tree(ops, c, 0.1), c, 0.1)
    c["table"] = c["table"][:, :5].contiguous()              # request 0 wants seven pages, request 1 six
    lost(0, 80, 109), lost(1, 80, 82)
    check_tree(run_tree(ops, c, 0.1), c, 0.1)


def test_banned_tokens_are_never_drawn(ops):
    # Every second token is banned, and the numbers that are drawn with lie at the ends of the allowed tokens' stretches, within a
    # few roundings: whichever way those fall, the draw is an allowed token.
    V, near = 2048, 8
    x = torch.randn(V, generator=torch.Generator().manual_seed(3)) * 2
    bits = np.zeros(V, dtype=bool)
    bits[::2] = True
    mask = torch.from_numpy(np.packbits(bits, bitorder="little").view(np.int32).copy()).view(1, -1)
    ends = torch.cumsum(torch.exp(x[::2].double()), 0)
    u = (ends / ends[-1]).float().repeat_interleave(near)
    u = (u + (torch.arange(u.numel()) % near - near // 2) * u * 2.0**-24).clamp(0.0, 1.0 - 2.0**-24)
    R = u.numel()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    controls = LogitControls(i32([0, R]), torch.tensor([[1.0, 0.0, 0.0]], device="cuda"), i32([]), i32([0]), i32([0]), i32([0]), mask=mask.cuda(),
                             mask_row=torch.zeros(R, dtype=torch.int32, device="cuda"))
    logits = x.cuda().repeat(R, 1)
    ops.control_logits(logits, logits, controls)
    out = torch.empty(R, dtype=torch.int32, device="cuda")
    one = torch.ones(R, device="cuda")
    for filters in ({}, dict(top_k=i32([700] * R), top_p=one * 0.999, min_p=one * 0)):
        ops.sample(logits, one, u.cuda(), out, **filters)
        assert not (out % 2).any()
    # a row whose mask leaves nothing gives some token of the vocabulary
    logits.fill_(-math.inf)
    for filters in ({}, dict(top_k=i32([700] * R), top_p=one * 0.999, min_p=one * 0)):
        ops.sample(logits, one, u.cuda(), out, **filters)
        assert ((out >= 0) & (out < V)).all()
    ops.check_errors()
