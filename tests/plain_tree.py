"""The operators that check trees of drafted tokens, written from their definitions in 64 bits on the CPU."""
import math
from types import SimpleNamespace

import numpy as np
import torch


def chain(parents, i):
    """Node i and its ancestors, node first; nothing for a node that is not there."""
    out = []
    while i >= 0:
        out.append(i)
        p = int(parents[i])
        if p >= i or p < -1:
            return []
        i = p
    return out


def random_tree(rng, n, spread=6, padding=0):
    parents = [-1] + [int(rng.integers(max(0, i - spread), i)) for i in range(1, n)] if n else []
    for i in range(max(1, n - padding), n):
        parents[i] = -2
    return parents


def step(ctx, trees, device, tokens=None, table=None):
    """What the kernels read of a step's batch."""
    n = np.array([len(t) for t in trees], dtype=np.int64)
    start = np.concatenate([[0], np.cumsum(n)])
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device=device)
    return SimpleNamespace(num_requests=len(trees), num_tokens=int(start[-1]), max_q_len=int(n.max(initial=0)),
                           max_kv_len=int((np.asarray(ctx) + n).max(initial=0)), q_start=i32(start), pos_start=i32(ctx),
                           tok_req=i32(np.repeat(np.arange(len(trees)), n)), token_ids=i32(tokens if tokens is not None else np.zeros(start[-1])),
                           h_q_lens=n, h_pos_start=np.asarray(ctx), req_order=None)


def paged(keys, values, page, device, dtype, layers=2, layer=1, major=True, seed=0, spare=3):
    """A cache whose layer ``layer`` holds keys[b] and values[b] ([slots, heads, size]) of every request in pages of no order;
    everything else in it is NaN.  (cache, block table with -1 where a request has no page)."""
    heads, size = keys[0].shape[1], max(keys[0].shape[2], values[0].shape[2])
    need = [-(-k.shape[0] // page) for k in keys]
    pages = sum(need) + spare
    order = np.random.default_rng(seed).permutation(pages)
    table = np.full((len(keys), max(max(need), 1) + 1), -1)
    store = torch.full((pages, layers, 2, heads, page, size), math.nan, dtype=torch.float64)
    at = 0
    for b, (k, v) in enumerate(zip(keys, values)):
        for j in range(need[b]):
            table[b, j] = order[at]
            part = slice(j * page, (j + 1) * page)
            store[order[at], layer, 0, :, :k[part].shape[0], :k.shape[2]] = k[part].transpose(0, 1)
            store[order[at], layer, 1, :, :v[part].shape[0], :v.shape[2]] = v[part].transpose(0, 1)
            at += 1
    cache = store.to(dtype).to(device)
    if major:                                    # stored with the layers outermost, as the engine does
        cache = cache.permute(1, 0, 2, 3, 4, 5).contiguous().permute(1, 0, 2, 3, 4, 5)
    return cache, torch.tensor(table, dtype=torch.int32, device=device)


def sees(parents, ctx, i, window=0, keep=0):
    """The cache slots that node i sees."""
    line = chain(parents, i)
    if not line:
        return []
    at = ctx + len(line) - 1
    slots = [(n, n) for n in range(ctx)] + [(at - k, ctx + a) for k, a in reversed(list(enumerate(line)))]
    return [slot for pos, slot in slots if not window or at - pos < window or pos < keep]


def attention(q, keys, values, ctx, trees, nq, scale, window=0, softcap=0.0, sink=None, gates=None, keep=0):
    """(out [T, nq, dv], sum of |weight * value|, largest sum of |q k| scale): q [T, nq, d], keys[b] and values[b] [slots, nkv, .]."""
    out, size, most, t = [], [], 0.0, 0
    for b, parents in enumerate(trees):
        nkv = keys[b].shape[1]
        for i in range(len(parents)):
            slots = sees(parents, ctx[b], i, window, keep)
            o = torch.zeros(nq, values[b].shape[2], dtype=torch.float64)
            a = o.clone()
            if slots:
                k, v = keys[b][slots].double(), values[b][slots].double()
                k, v = (x.repeat_interleave(nq // nkv, 1) for x in (k, v))
                s = torch.einsum("hd,nhd->hn", q[t].double(), k) * scale
                most = max(most, float(torch.einsum("hd,nhd->hn", q[t].double().abs(), k.abs()).max()) * scale)
                if softcap > 0:
                    s = softcap * torch.tanh(s / softcap)
                if sink is not None:
                    s = torch.cat([s, sink.double()[:, None]], 1)
                w = torch.softmax(s, 1)[:, :len(slots)]
                if gates is not None:
                    w = w * gates[t].double()[:, None]
                o, a = torch.einsum("hn,nhd->hd", w, v), torch.einsum("hn,nhd->hd", w.abs(), v.abs())
            out.append(o)
            size.append(a)
            t += 1
    return torch.stack(out), torch.stack(size), most


def accept(trees, tokens, drawn, width):
    path, emitted, count, at = [], [], [], 0
    for parents in trees:
        n, i, p, e = len(parents), 0, [], []
        if n == 0 or parents[0] != -1:
            i = None
        while i is not None and len(p) < width:
            p.append(i)
            e.append(int(drawn[at + i]))
            i = next((j for j in range(i + 1, n) if parents[j] == i and int(tokens[at + j]) == int(drawn[at + i])), None)
        path.append(p + [-1] * (width - len(p)))
        emitted.append(e + [-1] * (width - len(e)))
        count.append(len(p))
        at += n
    return path, emitted, count


def control(logits, requests, trees=None, tokens=None, masks=None):
    """requests: (rows, (repetition, frequency, presence), history, prompt length, [(token, bias)]); masks[row]: allowed or None."""
    x = logits.double().clone()
    V, row = x.shape[1], 0
    for b, (rows, (rep, freq, pres), history, prompt, biases) in enumerate(requests):
        for i in range(rows):
            path = [int(tokens[row - i + a]) for a in chain(trees[b], i)] if trees is not None else []
            made = list(history[prompt:]) + path
            for t in set(list(history) + path):
                if 0 <= t < V:
                    x[row, t] = x[row, t] / rep if x[row, t] > 0 else x[row, t] * rep
            for t in set(made):
                if 0 <= t < V:
                    x[row, t] -= freq * made.count(t) + pres
            for t, v in biases:
                if 0 <= t < V:
                    x[row, t] = -math.inf if v == -math.inf else x[row, t] + v
            if masks is not None and masks[row] is not None:
                x[row][~torch.tensor(masks[row])] = -math.inf
            row += 1
    return x
