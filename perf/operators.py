"""The operators that check drafted tokens, as cases that can be timed and compared.

A step of a request may bring a tree of drafted tokens behind its cached ones: node 0 is the token drawn last, every other
node continues its parent.  One pass of the model then gives the logits behind every node, and the drafted tokens that the
draws confirm are kept.  The operators are those that such a step needs beside what every step needs:

    tree      attention of the nodes: each sees the request's cached tokens, its ancestors and itself
    control   penalties for repeated tokens, biases and grammar masks on the logits, of decoded tokens and of nodes
    accept    the walk down a tree along the tokens that were drawn
    keep      the accepted nodes' keys and values moved to where the next step expects them, in every layer

Sizes are those of ``bench.py``: query heads, 8 key/value heads of 128 and the vocabulary of the Qwen3 family, the "2k"
model (16 query heads, 4 key/value heads, 8 layers, a vocabulary of 32,768).  ``listed`` gives the cases by name, ``draw`` more of the same ranges.

Fields of a case
    op        "tree", "control", "accept" or "keep"
    requests  requests of the step
    nodes     most nodes of a request's tree (each has between half as many and as many); 0 (control): one row a request
    least, most   cached tokens of a request, or the length of its history (control)
    dtype, heads, kv_heads, head, window, page    (tree, keep) the attention's; ``window`` 0: every cached token is seen
    padded    (tree) some nodes are padding: they see nothing, are seen by none and give zeros
    vocab     (control, accept) size of the vocabulary
    masked    (control) every second request is held to a grammar, with a mask of its own for each of its rows
    biases    (control) biases of a request
    layers    (keep) layers of the cache
"""
import functools
import math

import numpy as np
import torch

own = False

DEV = "cuda"
LONGEST = 16                                   # nodes of a path down a tree
QWEN_VOCAB = 151936
HEADS = {"0.6B": 16, "4B": 32, "14B": 40, "32B": 64}


def _tree(dtype, heads, requests, nodes, least, most, name=None, kv_heads=8, head=128, window=0, page=16, padded=False):
    c = dict(op="tree", dtype=dtype, heads=heads, kv_heads=kv_heads, head=head, requests=requests, nodes=nodes, least=least,
             most=most, window=window, page=page, padded=padded)
    return c if name is None else dict(c, name=name)


def _control(requests, nodes, least, most, vocab, masked, biases, name=None):
    c = dict(op="control", requests=requests, nodes=nodes, least=least, most=most, vocab=vocab, masked=masked, biases=biases)
    return c if name is None else dict(c, name=name)


def _accept(requests, nodes, vocab, name=None):
    c = dict(op="accept", requests=requests, nodes=nodes, least=100, most=4000, vocab=vocab)
    return c if name is None else dict(c, name=name)


def _keep(dtype, requests, nodes, kv_heads, head, layers, least, most, name=None, page=16):
    c = dict(op="keep", dtype=dtype, requests=requests, nodes=nodes, kv_heads=kv_heads, head=head, layers=layers, least=least,
             most=most, page=page)
    return c if name is None else dict(c, name=name)


def listed():
    return [
        # one user, a small tree behind a short conversation: latency
        _tree("bf16", 16, 1, 7, 300, 600, "tree_1_short"),
        # a served batch of the 8B shape: 8 requests behind the benchmark's 2,048 tokens, 32 nodes each
        _tree("bf16", 32, 8, 32, 2048, 2304, "tree_8_of_32"),
        # many users, small trees, contexts of very different lengths
        _tree("bf16", 32, 64, 8, 200, 6000, "tree_64_ragged"),
        # one long document of the 32B shape, a large tree
        _tree("bf16", 64, 1, 64, 32000, 32768, "tree_1_long"),
        # the 32-bit mode: two users, padded trees
        _tree("f32", 16, 2, 13, 400, 700, "tree_f32", padded=True),
        # one decoded token: penalties and a few biases
        _control(1, 0, 700, 800, QWEN_VOCAB, False, 10, "control_1"),
        # 64 users who decode, half of them held to a grammar
        _control(64, 0, 200, 6000, QWEN_VOCAB, True, 20, "control_64"),
        # the rows of 8 trees of 32 nodes
        _control(8, 32, 2048, 2304, QWEN_VOCAB, True, 5, "control_8_of_32"),
        # one user's tree
        _accept(1, 8, QWEN_VOCAB, "accept_1"),
        # 64 users, large trees
        _accept(64, 64, QWEN_VOCAB, "accept_64"),
        # one user of the "2k" model
        _keep("bf16", 1, 8, 4, 128, 8, 300, 600, "keep_1"),
        # 64 users of the 8B shape (short contexts: only their last pages are touched)
        _keep("bf16", 64, 32, 8, 128, 36, 60, 130, "keep_64"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "tree", "tree", "control", "control", "control", "accept", "keep"])
    if op == "tree":
        if rng.random() < 0.2:                     # the 32-bit mode: few requests
            least = _log(rng, 16, 800)
            return _tree("f32", rng.choice([8, 16, 32]), rng.randint(1, 3), _log(rng, 1, 24), least, least + rng.randrange(200),
                         kv_heads=rng.choice([4, 8]), head=rng.choice([64, 96, 128]), padded=rng.random() < 0.5)
        requests, nodes = _log(rng, 1, 64), _log(rng, 1, 64)
        least = _log(rng, 16, min(32000, 200000 // requests, 2000000 // (requests * nodes)))
        return _tree("bf16", HEADS[rng.choice(sorted(HEADS))], requests, nodes, least,
                     int(least * rng.uniform(1, 1.3)) + 1, head=rng.choice([64, 128, 128]), window=rng.choice([0, 0, 0, 512, 1000]),
                     page=rng.choice([16, 16, 32, 64]), padded=rng.random() < 0.3)
    if op == "control":
        requests, nodes = rng.choice([(_log(rng, 1, 128), 0), (_log(rng, 1, 8), _log(rng, 2, 32))])
        least = _log(rng, 16, 8000)
        return _control(requests, nodes, least, int(least * rng.uniform(1, 2)) + 1, rng.choice([32768, 32001, QWEN_VOCAB, QWEN_VOCAB]),
                        rng.random() < 0.6, rng.choice([0, _log(rng, 1, 300)]))
    if op == "accept":
        return _accept(_log(rng, 1, 128), _log(rng, 1, 200), rng.choice([32768, QWEN_VOCAB]))
    least = _log(rng, 16, 200)
    return _keep(rng.choice(["bf16", "bf16", "f32"]), _log(rng, 1, 32), _log(rng, 2, 64), rng.choice([4, 8]), rng.choice([64, 128]),
                 rng.choice([8, 28, 36]), least, least + rng.randrange(100), page=rng.choice([16, 16, 64]))


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """Nodes and cached tokens (or history) of every request; they belong to the case, whatever the seed is."""
    B, N = case["requests"], case["nodes"]
    rng = np.random.default_rng([B, N, case["least"], case["most"]])
    n = rng.integers(max(1, (N + 1) // 2), N + 1, B) if N else np.ones(B, dtype=np.int64)
    if N:
        n[rng.integers(B)] = N
    return n, rng.integers(case["least"], case["most"] + 1, B)


def _parents(n, rng, padded=False):
    """A tree of n nodes: node 0 is its root, no path has more than LONGEST nodes; -2 marks padding."""
    parent, depth = np.full(n, -1), np.zeros(n, dtype=np.int64)
    for i in range(1, n):
        p = int(rng.integers(max(0, i - 8), i))
        while depth[p] >= LONGEST - 1:
            p = int(parent[p])
        parent[i], depth[i] = p, depth[p] + 1
    if padded and n > 2:
        parent[n - 1 - int(rng.integers(0, n // 3 + 1)):] = -2
    return parent


def _int(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(DEV)


def _step(n, ctx, parents, tokens):
    """The step's arrays, as the engine keeps them for a step of these trees (engine/batch.py: StepBatch)."""
    B, start = len(n), np.concatenate([[0], np.cumsum(n)])
    depth = np.zeros(start[-1], dtype=np.int64)
    for b in range(B):
        for i in range(1, n[b]):
            p = parents[b][i]
            depth[start[b] + i] = depth[start[b] + p] + 1 if p >= 0 else 0
    req, order = np.repeat(np.arange(B), n), np.lexsort((-(ctx + n), n))
    return dict(num_tokens=int(start[-1]), num_requests=B, num_logit_rows=int(start[-1]), max_q_len=int(n.max()),
                max_kv_len=int((ctx + n).max()), token_ids=_int(tokens), positions=_int(ctx[req] + depth), tok_req=_int(req),
                q_start=_int(start), pos_start=_int(ctx), kv_len=_int(ctx + n), slots=_int(np.arange(B)),
                logit_rows=_int(np.arange(start[-1])), req_order=_int(order), h_q_lens=n, h_pos_start=ctx,
                h_sorted_q_lens=n[order], h_sorted_kv_lens=(ctx + n)[order], real_requests=B, real_logit_rows=int(start[-1]))


def _pages(case, n, ctx, rng):
    """A block table of pages in no order, and how many pages the cache has."""
    need = -(-(ctx + n) // case["page"])
    total, width = int(need.sum()), int(need.max())
    order, table, at = rng.permutation(total), np.full((len(n), width), -1), 0
    for b in range(len(n)):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
    return _int(table), total


def prepare(case, seed):
    rng = np.random.default_rng(seed)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    randn = lambda *s, dtype=torch.float32: torch.randn(*s, generator=gen, device=DEV, dtype=dtype)
    n, ctx = _lengths(case)
    parents = [_parents(int(k), rng, case.get("padded", False)) for k in n]
    T, op = int(n.sum()), case["op"]
    s = dict(case=case, parents=_int(np.concatenate(parents)))
    if op in ("tree", "keep"):
        dt = torch.float32 if case["dtype"] == "f32" else torch.bfloat16
        s["table"], pages = _pages(case, n, ctx, rng)
        s["step"] = _step(n, ctx, parents, np.zeros(T))
        # the layers outermost, as the engine stores them
        shape = (case.get("layers", 1), pages, 2, case["kv_heads"], case["page"], case["head"])
        s["store"] = torch.empty(shape, dtype=dt, device=DEV).normal_(generator=gen)
        s["cache"] = s["store"].permute(1, 0, 2, 3, 4, 5)
    if op == "tree":
        width = case["heads"] * case["head"]
        s["q"] = (randn(T, width) * 1.5).to(dt)              # normed, rotated queries: scores of a few units
        s["out"] = torch.empty(T, width, dtype=dt, device=DEV)
        s["scale"] = case["head"] ** -0.5
    elif op == "keep":
        path, count = np.full((len(n), LONGEST), -1), np.zeros(len(n))
        for b, parent in enumerate(parents):                 # to a node somewhere in the tree
            i, chain = int(rng.integers(len(parent))), []
            while i >= 0:
                chain.append(i)
                i = parent[i]
            path[b, :len(chain)], count[b] = chain[::-1], len(chain)
        s["path"], s["count"] = _int(path), _int(count)
    elif op == "accept":
        tokens, drawn = rng.integers(0, case["vocab"], T), rng.integers(0, case["vocab"], T)
        at = 0
        for parent in parents:
            for i in range(1, len(parent)):
                if rng.random() < 0.5:                       # the token that was drawn behind the parent (also for two siblings)
                    tokens[at + i] = drawn[at + parent[i]]
            at += len(parent)
        s["step"], s["drawn"] = _step(n, ctx, parents, tokens), _int(drawn)
        s["answer"] = [torch.empty(len(n), LONGEST, dtype=torch.int32, device=DEV) for _ in range(2)] + \
            [torch.empty(len(n), dtype=torch.int32, device=DEV)]
    else:
        B, V, tree = len(n), case["vocab"], case["nodes"] > 0
        word = lambda *size: (V * rng.random(size) ** 3).astype(np.int64)          # few tokens are used often
        held, biases = int(ctx.max()), case["biases"]
        c = dict(row_start=_int(np.concatenate([[0], np.cumsum(n)])),
                 settings=torch.tensor(np.stack([rng.choice([1.0, 1.05, 1.2], B), rng.choice([0.0, 0.1, 0.5], B),
                                                 rng.choice([0.0, 0.3], B)], 1), dtype=torch.float32, device=DEV),
                 history=_int(word(B * held)), history_start=_int(np.arange(B) * held), history_len=_int(ctx),
                 prompt_len=_int((ctx * rng.random(B)).astype(np.int64)))
        if biases:
            some = np.sort(np.stack([rng.choice(V, biases, replace=False) for _ in range(B)]), 1)
            value = rng.normal(0, 3, some.shape)
            value[rng.random(some.shape) < 0.1] = -np.inf     # tokens that a request must not give
            c.update(bias_start=_int(np.arange(B + 1) * biases), bias_tokens=_int(some.reshape(-1)),
                     bias_values=torch.tensor(value.reshape(-1), dtype=torch.float32, device=DEV))
        if case["masked"]:
            row = np.full(T, -1)
            own_mask = np.repeat(np.arange(B) % 2 == 1, n) if B > 1 else np.ones(T, dtype=bool)
            row[own_mask] = np.arange(own_mask.sum())
            bits = torch.randint(-2 ** 31, 2 ** 31, (int(own_mask.sum()), (V + 31) // 32), generator=gen, device=DEV, dtype=torch.int64)
            few = torch.randint(-2 ** 31, 2 ** 31, (bits.shape[0], bits.shape[1], 3), generator=gen, device=DEV, dtype=torch.int64)
            few = few[..., 0] & few[..., 1] & few[..., 2]     # a state of the grammar that allows few tokens
            c.update(mask=torch.where((torch.arange(bits.shape[0], device=DEV) % 2 == 0)[:, None], few, bits).to(torch.int32),
                     mask_row=_int(row))
        if tree:
            c.update(parents=s["parents"], tokens=_int(word(T)))
        s["controls"] = c
        s["logits"], s["out"] = randn(T, V) * 4, torch.empty(T, V, device=DEV)
    return s


# ------------------------------------------------------------------ the framework's calls

@functools.lru_cache(maxsize=None)
def _kernels():
    from tffinfer_b200.kernels.library import CudaKernels
    return CudaKernels(verbose_build=False)


def _own(s):
    from tffinfer_b200.engine.batch import StepBatch
    from tffinfer_b200.sampling import LogitControls
    ops, case, op = _kernels(), s["case"], s["case"]["op"]
    if op == "control":
        ops.control_logits(s["logits"], s["out"], LogitControls(**s["controls"]))
        return s["out"]
    batch = StepBatch(**s["step"])
    if op == "tree":
        ops.attention_tree(s["q"], batch, s["parents"], s["table"], s["cache"], 0, case["page"], s["out"], case["heads"],
                           case["kv_heads"], case["head"], case["head"], s["scale"], window=case["window"])
        return s["out"]
    if op == "accept":
        ops.accept_tree(batch, s["parents"], s["drawn"], *s["answer"])
        return s["answer"]
    ops.keep_path(s["cache"], batch, s["table"], case["page"], s["path"], s["count"])
    return s["store"]


# ------------------------------------------------------------------ the plain forms

def _padded(start, B, N):
    """Flat row of node i of request b, and whether there is one."""
    n = start[1:] - start[:-1]
    i = torch.arange(N, device=DEV)
    there = i[None] < n[:, None]
    return torch.where(there, start[:-1, None] + i[None], 0), there


def _ancestors(parent, there):
    """[b, i, j]: node j is i or an ancestor of i, for the nodes whose ancestors are all there (parent -1 at their end)."""
    N = parent.shape[1]
    i = torch.arange(N, device=DEV)
    edge = (parent[:, :, None] == i) & (parent[:, :, None] >= 0) & (i < i[:, None]) & there[:, :, None]
    reach = torch.matrix_power(torch.eye(N, device=DEV, dtype=torch.float64) + edge, max(1, N)) > 0
    rooted = (reach & (there & (parent == -1))[:, None]).any(-1) & there
    return reach & rooted[:, :, None]


def _plain_tree(s):
    case, st = s["case"], s["step"]
    B, N, page, d, kv = st["num_requests"], st["max_q_len"], case["page"], case["head"], case["kv_heads"]
    G, L = case["heads"] // kv, st["max_kv_len"]
    at, there = _padded(st["q_start"].long(), B, N)
    ctx = st["pos_start"].long()
    sees = _ancestors(torch.where(there, s["parents"].long()[at], -2), there)
    pos = ctx[:, None] + sees.sum(-1) - 1
    n = torch.arange(L, device=DEV)
    j = n[None] - ctx[:, None]                               # node of a key, below 0: a cached token
    node = (j >= 0) & (j < there.sum(-1)[:, None])
    jj = j.clamp(0, N - 1)
    key_pos = torch.where(node, pos.gather(1, jj), n[None])
    seen = torch.where(node[:, None], sees.gather(2, jj[:, None].expand(B, N, L)), (j < 0)[:, None]) & sees.any(-1)[..., None]
    if case["window"]:
        seen &= pos[..., None] - key_pos[:, None] < case["window"]
    held = torch.arange(L, device=DEV)[None] < st["kv_len"][:, None]
    pages = torch.where(held, s["table"].long()[:, n // page], 0)
    off = (n % page).expand(B, L)
    k, v = (torch.where(held[..., None, None], s["store"][0][pages, x, :, off], 0).float() for x in (0, 1))       # [B, L, kv, d]
    q = s["q"].float().view(-1, kv, G, d)[at] * there[..., None, None, None]
    q = q.permute(0, 2, 3, 1, 4).reshape(B, kv, G * N, d)
    x = torch.matmul(q, k.permute(0, 2, 3, 1)).view(B, kv, G, N, L).mul_(s["scale"])
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul((x / total.clamp(min=1e-30)).view(B, kv, G * N, L), v.permute(0, 2, 1, 3)).view(B, kv, G, N, d)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(B, N, -1)[there])
    return s["out"]


def _plain_control(s):
    c, x = s["controls"], s["logits"]
    R, V = x.shape
    start = c["row_start"].long()
    B = start.numel() - 1
    req = torch.repeat_interleave(torch.arange(B, device=DEV), start[1:] - start[:-1])
    held = c["history"].numel() // B
    i = torch.arange(held, device=DEV)[None]
    where = c["history_start"].long()[:, None] + i
    token = c["history"].long()[where.clamp(max=c["history"].numel() - 1)]
    valid = i < c["history_len"][:, None]
    seen = torch.zeros(B, V, device=DEV).scatter_add_(1, token, valid.float())[req]
    count = torch.zeros(B, V, device=DEV).scatter_add_(1, token, (valid & (i >= c["prompt_len"][:, None])).float())[req]
    if "parents" in c:
        N = int(s["case"]["nodes"])
        at, there = _padded(start, B, N)
        on = _ancestors(torch.where(there, c["parents"].long()[at], -2), there)[there].float()        # [R, N]: the path of a row
        words = c["tokens"].long()[at][req]
        seen.scatter_add_(1, words, on)
        count.scatter_add_(1, words, on)
    r, f, p = (t[req][:, None] for t in c["settings"].unbind(1))
    y = torch.where(seen > 0, torch.where(x > 0, x / r, x * r), x) - (f * count + p * (count > 0))
    if "bias_tokens" in c:
        n = c["bias_start"].long()
        whose = torch.repeat_interleave(torch.arange(B, device=DEV), n[1:] - n[:-1])
        y += torch.zeros(B, V, device=DEV).index_put_((whose, c["bias_tokens"].long()), c["bias_values"], accumulate=True)[req]
    if "mask" in c:
        t = torch.arange(V, device=DEV)
        allowed = (c["mask"][c["mask_row"].clamp(min=0).long()][:, t // 32] >> (t % 32).int()) & 1
        y.masked_fill_((allowed == 0) & (c["mask_row"] >= 0)[:, None], -math.inf)
    s["out"].copy_(y)
    return s["out"]


def _plain_accept(s):
    st = s["step"]
    B, N = st["num_requests"], st["max_q_len"]
    at, there = _padded(st["q_start"].long(), B, N)
    parent = torch.where(there, s["parents"].long()[at], -2)
    token, drawn = st["token_ids"].long()[at], s["drawn"].long()[at]
    i = torch.arange(N, device=DEV)
    fits = there & (parent >= 0) & (parent < i) & (token == drawn.gather(1, parent.clamp(min=0)))
    same = (parent[:, :, None] == parent[:, None]) & fits[:, None] & (i < i[:, None])          # an earlier sibling that fits too
    step = torch.where(fits & ~same.any(-1), parent, -2)
    step[:, 0] = parent[:, 0]
    on = _ancestors(step, there)[:, :, 0] & (parent[:, :1] == -1)
    place = on.cumsum(1) - 1
    on &= place < LONGEST
    path, emitted, count = s["answer"]
    full = torch.full((B, LONGEST + 1), -1, device=DEV, dtype=torch.int64)
    slot = torch.where(on, place, LONGEST)
    path.copy_(full.scatter(1, slot, i.expand(B, N))[:, :LONGEST])
    emitted.copy_(full.scatter(1, slot, drawn)[:, :LONGEST])
    count.copy_(on.sum(1))
    return s["answer"]


def _plain_keep(s):
    page, path = s["case"]["page"], s["path"].long()
    j = torch.arange(path.shape[1], device=DEV)
    b, j = torch.nonzero(j[None] < s["count"][:, None], as_tuple=True)
    ctx, table, store = s["step"]["pos_start"].long()[b], s["table"].long(), s["store"]
    to, at = ctx + j, ctx + path[b, j]
    store[:, table[b, to // page], :, :, to % page] = store[:, table[b, at // page], :, :, at % page]
    return store


def run(s):
    if own:
        return _own(s)
    return {"tree": _plain_tree, "control": _plain_control, "accept": _plain_accept, "keep": _plain_keep}[s["case"]["op"]](s)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    n, ctx = _lengths(case)
    B, T, op = case["requests"], int(n.sum()), case["op"]
    size = 4 if case.get("dtype") == "f32" else 2
    deep = np.minimum(n, 4)                                   # nodes of a path, about
    if op == "tree":
        seen = np.minimum(ctx, case["window"]) if case["window"] else ctx
        kv, q = case["kv_heads"] * case["head"], case["heads"] * case["head"]
        return {"bytes": size * (2 * int((seen + n).sum()) * kv + 2 * T * q), "flops": 4 * q * int((n * (seen + deep)).sum())}
    if op == "keep":
        return {"bytes": 2 * int(deep.sum()) * case["layers"] * 2 * case["kv_heads"] * case["head"] * size, "flops": 0}
    if op == "accept":
        return {"bytes": 4 * (3 * T + B * (2 * LONGEST + 2)), "flops": 0}
    masks = int(n[1::2].sum()) if B > 1 else T
    return {"bytes": T * case["vocab"] * 8 + 4 * int(ctx.sum()) + 8 * B * case["biases"] + (masks * case["vocab"] // 8 if case["masked"] else 0),
            "flops": T * case["vocab"]}


# ------------------------------------------------------------------ the definitions in 64 bits

def _chain(parent, i):
    """Node i and its ancestors, or none where one of them is not there."""
    out = []
    while i >= 0:
        out.append(i)
        p = int(parent[i])
        if p >= i or p < -1:
            return []
        i = p
    return out


def _exact_tree(case, s):
    st, kv, d, page = s["step"], case["kv_heads"], case["head"], case["page"]
    G, parents, start, table = case["heads"] // kv, s["parents"].tolist(), st["q_start"].tolist(), s["table"].long()
    out = torch.zeros(st["num_tokens"], kv, G, d, dtype=torch.float64, device=DEV)
    for b, ctx in enumerate(st["pos_start"].tolist()):
        parent = parents[start[b]:start[b + 1]]
        n = len(parent)
        slot = torch.arange(ctx + n, device=DEV)
        key = s["store"][0][table[b, slot // page], 0, :, slot % page].double()
        val = s["store"][0][table[b, slot // page], 1, :, slot % page].double()
        depth = [len(_chain(parent, i)) - 1 for i in range(n)]
        where = torch.cat([slot[:ctx], torch.tensor([ctx + max(x, 0) for x in depth], device=DEV)])
        for i in range(n):
            chain = _chain(parent, i)
            if not chain:
                continue
            lo = max(0, ctx + depth[i] - case["window"] + 1) if case["window"] else 0
            pick = torch.cat([slot[min(lo, ctx):ctx], torch.tensor(sorted(ctx + j for j in chain), device=DEV)])
            pick = pick[where[pick] >= lo]
            q = s["q"][start[b] + i].double().view(kv, G, d)
            x = torch.einsum("hgd,nhd->hgn", q, key[pick]) * s["scale"]
            out[start[b] + i] = torch.einsum("hgn,nhd->hgd", torch.softmax(x, -1), val[pick])
    return out.view(st["num_tokens"], -1)


def _exact_control(case, s):
    c, x = s["controls"], s["logits"].double()
    V, held = case["vocab"], c["history"].cpu().numpy()
    start, first, last = (c[k].tolist() for k in ("row_start", "history_start", "history_len"))
    for b, (r, f, p) in enumerate(c["settings"].double().tolist()):
        past = held[first[b]:first[b] + last[b]]
        drawn = past[int(c["prompt_len"][b]):]
        seen, count = (torch.from_numpy(np.bincount(t, minlength=V)).to(DEV).double() for t in (past, drawn))
        bias = torch.zeros(V, dtype=torch.float64, device=DEV)
        if "bias_tokens" in c:
            lo, hi = c["bias_start"][b:b + 2].tolist()
            bias[c["bias_tokens"][lo:hi].long()] = c["bias_values"][lo:hi].double()
        parent = c["parents"][start[b]:start[b + 1]].tolist() if "parents" in c else None
        for row in range(start[b], start[b + 1]):
            sn, ct = seen, count
            if parent is not None:
                path = c["tokens"][torch.tensor(_chain(parent, row - start[b]), device=DEV) + start[b]].cpu().numpy()
                more = torch.from_numpy(np.bincount(path, minlength=V)).to(DEV)
                sn, ct = seen + more, count + more
            y = torch.where(sn > 0, torch.where(x[row] > 0, x[row] / r, x[row] * r), x[row]) - f * ct - p * (ct > 0) + bias
            if "mask" in c and int(c["mask_row"][row]) >= 0:
                words = c["mask"][int(c["mask_row"][row])].cpu().numpy().view(np.uint32).view(np.uint8)
                allowed = torch.from_numpy(np.unpackbits(words, bitorder="little")[:V].astype(bool)).to(DEV)
                y = torch.where(allowed, y, -math.inf)
            x[row] = y
    return x


def _exact_accept(case, s):
    st = s["step"]
    B, parents, tokens, drawn, start = (st["num_requests"], s["parents"].tolist(), st["token_ids"].tolist(), s["drawn"].tolist(),
                                        st["q_start"].tolist())
    path, emitted = torch.full((B, LONGEST), -1, dtype=torch.int32), torch.full((B, LONGEST), -1, dtype=torch.int32)
    count = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        at, i, k = start[b], 0, 0
        while i is not None and k < LONGEST:
            path[b, k], emitted[b, k], k = i, drawn[at + i], k + 1
            i = next((j for j in range(i + 1, start[b + 1] - at) if parents[at + j] == i and tokens[at + j] == drawn[at + i]), None)
        count[b] = k
    return [path.to(DEV), emitted.to(DEV), count.to(DEV)]


def _exact_keep(case, s):
    out, page, table = s["store"].double(), case["page"], s["table"].tolist()
    for b, (ctx, k) in enumerate(zip(s["step"]["pos_start"].tolist(), s["count"].tolist())):
        for j, i in enumerate(s["path"][b, :k].tolist()):
            src, dst = ctx + i, ctx + j
            out[:, table[b][dst // page], :, :, dst % page] = s["store"][:, table[b][src // page], :, :, src % page].double()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "control": _exact_control, "accept": _exact_accept, "keep": _exact_keep}[case["op"]](case, s)
