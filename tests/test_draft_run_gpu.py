"""The operators of drafted trees used together, as a step that checks drafted tokens uses them: what it emits and what it leaves in the
cache are those of decoding one token at a time.  And generation under controls, against plain logits."""
import math

import numpy as np
import pytest
import torch

import plain_tree as plain
from helpers import make_model_dir, tiny_config, PAGE_SIZE
from plain_qwen3 import PlainModel
from tffinfer_b200.config import EngineConfig
from tffinfer_b200.engine import Engine
from tffinfer_b200.kernels.library import CudaKernels
from tffinfer_b200.sampling import LogitControls, SamplingParams

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
V, WIDTH, LAYERS, NQ, NKV, D, PAGE = 61, 96, 3, 4, 2, 64, 16


class Tiny:
    """A decoder of attention layers only: its products are plain, its attention, controls, draws and cache moves the framework's."""

    def __init__(self, ops, dtype, requests, slots, seed):
        gen = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=gen).to(DEV)
        self.ops, self.dtype = ops, dtype
        self.table_of, self.place = rand(V, WIDTH), rand(400, WIDTH) * 0.3
        self.wq, self.wk = (rand(LAYERS, WIDTH, h * D) / WIDTH ** 0.5 for h in (NQ, NKV))
        self.wv, self.wo = rand(LAYERS, WIDTH, NKV * D) / WIDTH ** 0.5, rand(LAYERS, NQ * D, WIDTH) / (NQ * D) ** 0.5
        self.head = rand(WIDTH, V)
        pages = -(-slots // PAGE)
        store = torch.full((LAYERS, requests * pages + 1, 2, NKV, PAGE, D), math.nan, dtype=dtype, device=DEV)
        self.cache = store.permute(1, 0, 2, 3, 4, 5)
        order = torch.randperm(requests * pages, generator=gen)
        self.table = order.view(requests, pages).int().to(DEV)

    def logits(self, batch, parents, tokens, positions):
        x = self.table_of[tokens] + self.place[positions]
        req, T = batch.tok_req.long(), tokens.numel()
        at = batch.pos_start.long()[req] + torch.arange(T, device=DEV) - batch.q_start.long()[req]        # the nodes' slots
        page, off = self.table.long()[req, at // PAGE], at % PAGE
        for layer in range(LAYERS):
            h = x / x.norm(dim=1, keepdim=True) * WIDTH ** 0.5
            q = (h @ self.wq[layer]).to(self.dtype)
            self.cache[page, layer, 0, :, off] = (h @ self.wk[layer]).to(self.dtype).view(T, NKV, D)
            self.cache[page, layer, 1, :, off] = (h @ self.wv[layer]).to(self.dtype).view(T, NKV, D)
            o = torch.empty(T, NQ * D, dtype=self.dtype, device=DEV)
            self.ops.attention_tree(q, batch, parents, self.table, self.cache, layer, PAGE, o, NQ, NKV, D, D, D ** -0.5)
            x = x + o.float() @ self.wo[layer]
        return (x @ self.head).contiguous()


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def controls(batch, histories, prompts, settings, bans, tree, parents, tokens):
    """Penalties, a bias each, and a grammar for every second request that bans a token after each token (token 7 k + 3 after k)."""
    start = batch.q_start
    words = -(-V // 32)
    mask = np.full((len(tokens), words), -1, dtype=np.int32)
    for r, (t, b) in enumerate(zip(tokens, batch.tok_req.tolist())):
        if b % 2:
            banned = (7 * t + 3) % V
            mask[r, banned // 32] &= ~np.int32(np.uint32(1 << banned % 32).view(np.int32))
    held = np.concatenate([[0], np.cumsum([len(h) for h in histories])])
    return LogitControls(start, torch.tensor(settings, dtype=torch.float32, device=DEV), i32(np.concatenate(histories).astype(np.int64)), i32(held[:-1]),
                         i32([len(h) for h in histories]), i32(prompts), i32(np.arange(len(bans) + 1)), i32([t for t, _ in bans]),
                         torch.tensor([v for _, v in bans], device=DEV), i32(mask), None, parents if tree else None, i32(tokens) if tree else None)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_checked_trees_emit_what_single_steps_emit(dtype):
    ops = CudaKernels()
    B, goal = 3, 40
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, V, n).tolist() for n in (5, 17, 33)]
    settings, bans = [[1.2, 0.3, 0.2], [1.0, 0.0, 0.0], [1.1, 0.0, 0.4]], [(4, -math.inf), (9, 2.0), (0, -1.0)]

    def run(drafts):
        m = Tiny(ops, dtype, B, 400, 5)
        ctx, made = [0] * B, [[] for _ in range(B)]
        pending = [list(p) for p in prompts]                 # tokens that are known and not in the cache; the last is node 0
        steps = 0
        while any(len(x) < goal for x in made):
            steps += 1
            trees, tokens = [], []
            for b in range(B):
                first = pending[b][:-1] if not made[b] else []                    # a prompt comes as a chain ahead of its last token
                t, parent = list(first) + [pending[b][-1]], list(range(-1, len(first)))
                if drafts and made[b]:
                    for extra, up in drafts(b, made[b]):     # (token, index among the drafted: -1 the root)
                        t.append(extra)
                        parent.append(0 if up < 0 else up + 1)
                trees.append(parent)
                tokens += t
            batch = plain.step(ctx, trees, DEV, tokens)
            parents = i32(np.concatenate(trees))
            depth = [len(plain.chain(p, i)) - 1 for p in trees for i in range(len(p))]
            positions = batch.pos_start.long()[batch.tok_req.long()] + torch.tensor(depth, device=DEV)
            logits = m.logits(batch, parents, batch.token_ids.long(), positions)
            prompt_step = not made[0]
            histories = [prompts[b] + made[b][:-1] if made[b] else [] for b in range(B)]
            out = torch.empty_like(logits)
            # (in the prompt's step its tokens are nodes, which count as generated: the histories there are the prompts, one row each)
            if prompt_step:
                last = batch.q_start[1:].long() - 1
                one = plain.step(ctx, [[-1]] * B, DEV)
                c = controls(one, prompts, [len(p) for p in prompts], settings, bans, False, None, [p[-1] for p in prompts])
                rows = logits[last].contiguous()
                ops.control_logits(rows, rows, c)
                drawn = torch.empty(B, dtype=torch.int32, device=DEV)
                ops.argmax(rows, drawn)
                for b, t in enumerate(drawn.tolist()):
                    ctx[b] += len(prompts[b])
                    made[b].append(t)
                    pending[b] = [t]
                continue
            c = controls(batch, histories, [len(p) for p in prompts], settings, bans, True, parents, tokens)
            ops.control_logits(logits, out, c)
            drawn = torch.empty(len(tokens), dtype=torch.int32, device=DEV)
            ops.argmax(out, drawn)
            path, emitted = (torch.empty(B, 8, dtype=torch.int32, device=DEV) for _ in range(2))
            count = torch.empty(B, dtype=torch.int32, device=DEV)
            ops.accept_tree(batch, parents, drawn, path, emitted, count)
            ops.keep_path(m.cache, batch, m.table, PAGE, path, count)
            for b, (e, n) in enumerate(zip(emitted.tolist(), count.tolist())):
                assert n >= 1
                made[b] += e[:n]
                ctx[b] += n
                pending[b] = [e[n - 1]]
        ops.check_errors()
        return [x[:goal] for x in made], steps, m, ctx

    single, steps_one, one, ctx_one = run(None)

    def drafts(b, made):
        """Two guesses a level for three levels; of every second tree one is what follows indeed, of the others all are wrong."""
        known = single[b][len(made):len(made) + 3]
        wrong = lambda k: (single[b][min(len(made), goal - 1)] + 11 + k) % V
        right = [known[k] if k < len(known) and (len(made) + b) % 3 else wrong(k) for k in range(3)]
        # level by level: (a wrong one, the right one), children of the right one before
        return [(wrong(7), -1), (right[0], -1), (wrong(8), 1), (right[1], 1), (right[1], 0), (right[2], 3), (wrong(9), 3)]

    tree, steps_tree, two, ctx_two = run(drafts)
    if dtype == torch.float32:
        assert tree == single and steps_tree < 0.6 * steps_one
        # the cache holds what single steps leave there, where both have got to
        for b in range(B):
            n = min(ctx_one[b], ctx_two[b])
            at = torch.arange(n, device=DEV)
            held = [m.cache[m.table[b].long()[at // PAGE], :, :, :, at % PAGE] for m in (one, two)]
            assert (held[0] - held[1]).abs().max() <= 1e-4 * held[0].abs().max()
    else:
        # (a draw between two nearly equal logits may differ in bfloat16: the tokens agree up to there)
        assert steps_tree < 0.8 * steps_one and sum(a == b for x, y in zip(tree, single) for a, b in zip(x, y)) >= B * goal // 2


def _plain_generate(pm, prompt, params):
    toks = list(prompt)
    for _ in range(params.max_new_tokens):
        row = pm.logits(toks)[-1:].float()
        made = toks[len(prompt):]
        mask = params.token_mask(made) if params.token_mask is not None else None
        allowed = None
        if mask is not None:
            allowed = np.unpackbits(np.ascontiguousarray(mask).view(np.uint8), bitorder="little")[:row.shape[1]].astype(bool)
        row = plain.control(row, [(1, (params.repetition_penalty, params.frequency_penalty, params.presence_penalty), toks, len(prompt), list(params.logit_bias))],
                            masks=[allowed])
        top = torch.topk(row[0], 2)
        assert float(top.values[0] - top.values[1]) > 1e-4             # the choice does not hang on rounding
        toks.append(int(top.indices[0]))
    return toks[len(prompt):]


@pytest.mark.parametrize("async_steps", [False, True])
def test_generation_under_controls(tmp_path, async_steps):
    name = "C"                                     # (an odd vocabulary)
    d = make_model_dir(tmp_path, name)
    vocab = tiny_config(name).vocab_size
    words = -(-vocab // 32)

    def even(made):                                # a grammar: tokens alternate between even and odd
        bits = np.zeros(words * 32, dtype=bool)
        bits[len(made) % 2::2] = True
        return np.packbits(bits, bitorder="little").view(np.int32)

    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, vocab, n).tolist() for n in (9, 4, 21, 6)]
    params = [SamplingParams(max_new_tokens=12, frequency_penalty=0.7, presence_penalty=0.4, repetition_penalty=1.3),
              SamplingParams(max_new_tokens=12, token_mask=even), SamplingParams(max_new_tokens=12, logit_bias=((3, 1.5), (11, -math.inf), (5, -0.5))),
              SamplingParams(max_new_tokens=12)]
    eng = Engine(d, EngineConfig(dtype="float32", page_size=PAGE_SIZE[name], max_cache_tokens=512, max_live_requests=4, async_steps=async_steps))
    got = eng.generate(prompts, params)
    eng.runner.ops.check_errors()
    pm = PlainModel(d)
    assert got == [_plain_generate(pm, p, sp) for p, sp in zip(prompts, params)]
    assert all((t % 2) == (i % 2) for i, t in enumerate(got[1]))
