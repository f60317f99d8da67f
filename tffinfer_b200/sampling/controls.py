"""What changes a request's logits ahead of a draw: penalties for tokens that it has had, biases, a grammar's mask.

The penalty helper of the reference (src/core/sampler/LLMSampler.cpp:21-34) works on one row on the host and is never
called.  Here the rows of a whole step, single tokens or the nodes of drafted trees, are one kernel call
(``CudaKernels.control_logits``)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Sequence

import numpy as np
import torch

from .params import SamplingParams


def mask_of(params: SamplingParams, made: Sequence[int], vocab: int) -> Optional[np.ndarray]:
    """What the grammar of ``params`` allows behind the generated tokens ``made``: 32-bit words, or None for no limit.  Raises what the
    grammar raises, and ValueError for anything else that it gives."""
    mask = params.token_mask(list(made)) if params.token_mask is not None else None
    if mask is None:
        return None
    mask, words = np.array(mask, order="C"), -(-vocab // 32)          # (a copy: a grammar may fill one array for several requests)
    if mask.dtype.itemsize != 4 or mask.dtype.kind not in "iu" or mask.shape != (words,):
        raise ValueError(f"a token mask is {words} 32-bit words for {vocab} tokens, got {mask.dtype} {mask.shape}")
    if not mask[:-1].any() and not int(mask.view(np.uint32)[-1]) << (32 * words - vocab) & 0xffffffff:
        raise ValueError(f"a token mask allows no token of {vocab}")
    return mask


@dataclass
class LogitControls:
    """The controls of a step's logit rows, tensors on the device (int32 unless said otherwise).  B requests, R rows.

    For the logit x of token t in a row of request b, in this order:
      ``settings[b]`` = (repetition, frequency, presence)
        a token of the history or of the row's path:  x / repetition if x > 0, else x * repetition
        one that was generated n > 0 times (behind the prompt, or on the path):  x - (frequency * n + presence)
      the biases of t:  x + bias; a bias of -infinity bans the token; finite or -infinity
      the row's mask:   -infinity where it has no bit for t

    row_start [B + 1]           the rows of request b are row_start[b] .. row_start[b + 1] - 1; rows behind row_start[B] are left alone
    settings float32 [B, 3]
    history [..], history_start [B], history_len [B], prompt_len [B]
                                request b's tokens are history[history_start[b]] and the history_len[b] - 1 behind it, the
                                first prompt_len[b] of them the prompt
    bias_start [B + 1], bias_tokens [..], bias_values float32 [..]
                                request b's biases, in ascending order of their tokens; those of one token add up
    mask [M, words], mask_row [R]
                                bit t % 32 of word t // 32: token t is allowed.  Row r has mask mask_row[r], none if that is
                                not in [0, M); without mask_row it has mask r
    parents [R], tokens [R]     the rows of a request are the nodes of a tree of drafted tokens: parents as in
                                ``CudaKernels.attention_tree``, and as many as there are (a tree of more than 256 takes longer a
                                node).  A row's path is its node and that node's ancestors; node 0, the token drawn last, is on every
                                path, and so not in the history
    """
    row_start: torch.Tensor
    settings: torch.Tensor
    history: torch.Tensor
    history_start: torch.Tensor
    history_len: torch.Tensor
    prompt_len: torch.Tensor
    bias_start: Optional[torch.Tensor] = None
    bias_tokens: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    mask: Optional[torch.Tensor] = None
    mask_row: Optional[torch.Tensor] = None
    parents: Optional[torch.Tensor] = None
    tokens: Optional[torch.Tensor] = None

    def problem(self, rows: int, vocab: int) -> Optional[str]:
        """What is wrong with the sizes of these controls for logits [rows, vocab], or None."""
        B = self.row_start.numel() - 1
        if B < 0 or self.settings.shape != (B, 3):
            return "row_start has one element more than settings has rows of three"
        if self.history_start.numel() != B or self.history_len.numel() != B or self.prompt_len.numel() != B:
            return "history_start, history_len and prompt_len have an element a request"
        if self.bias_start is not None or self.bias_tokens is not None or self.bias_values is not None:
            if self.bias_start is None or self.bias_tokens is None or self.bias_values is None:
                return "bias_start, bias_tokens and bias_values come together"
            if self.bias_start.numel() != B + 1 or self.bias_tokens.numel() != self.bias_values.numel():
                return "bias_start has an element more than there are requests, bias_tokens as many as bias_values"
        if self.mask is not None:
            if self.mask.dim() != 2 or self.mask.shape[1] * 32 < vocab:
                return f"a mask has a bit for each of {vocab} tokens"
        elif self.mask_row is not None:
            return "mask_row without a mask"
        if self.mask_row is not None and self.mask_row.numel() != rows:
            return "mask_row has an element a row"
        if self.parents is not None or self.tokens is not None:
            if self.parents is None or self.tokens is None:
                return "parents and tokens come together"
            if self.parents.numel() != rows or self.tokens.numel() != rows:
                return "parents and tokens have an element a row"
        return None

    @classmethod
    def of(cls, params: Sequence[SamplingParams], prompts: Sequence[int], histories: Sequence[Sequence[int]], vocab: int,
           device, masks: Optional[Sequence[Optional[np.ndarray]]] = None) -> "LogitControls":
        """The controls of one row a request: its settings, the length of its prompt and its tokens so far.  ``masks``: what the
        requests' grammars have given already (``mask_of``); None: they are asked here."""
        B = len(params)
        lens = np.fromiter((len(h) for h in histories), dtype=np.int64, count=B)
        start = np.concatenate([[0], np.cumsum(lens)])
        biases = [sorted(p.logit_bias) for p in params]
        count = np.concatenate([[0], np.cumsum([len(x) for x in biases])])
        if masks is None:
            masks = [mask_of(p, h[n:], vocab) for p, n, h in zip(params, prompts, histories)]
        words, held = -(-vocab // 32), [m for m in masks if m is not None]
        row = np.cumsum([m is not None for m in masks]) - 1
        row[[m is None for m in masks]] = -1
        # one buffer of 32-bit words, one copy
        parts = [np.arange(B + 1), np.concatenate(list(histories) + [[]]), start[:-1], lens, np.asarray(prompts), count,
                 [t for x in biases for t, _ in x], row]
        ints = [np.asarray(p, dtype=np.int64).astype(np.int32) for p in parts]
        floats = [np.array([[p.repetition_penalty, p.frequency_penalty, p.presence_penalty] for p in params], dtype=np.float32),
                  np.array([v for x in biases for _, v in x], dtype=np.float32)]
        flat = ints + [f.reshape(-1).view(np.int32) for f in floats] + [m.view(np.int32) for m in held]
        host = torch.from_numpy(np.concatenate(flat))
        dev = (host.pin_memory() if torch.device(device).type == "cuda" else host).to(device, non_blocking=True)
        at, out = 0, []
        for f in flat:
            out.append(dev[at:at + f.size])
            at += f.size
        rs, hist, hs, hl, pl, bs, bt, mr, settings, values = out[:10]
        some = count[-1] > 0
        return cls(rs, settings.view(torch.float32).view(B, 3), hist, hs, hl, pl, bs if some else None, bt if some else None,
                   values.view(torch.float32) if some else None,
                   dev[at - words * len(held):at].view(len(held), words) if held else None, mr if held else None)
