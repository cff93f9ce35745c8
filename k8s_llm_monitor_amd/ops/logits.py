"""Controls of logits ahead of the sampler: penalties for repeated tokens, biases and allowed-token masks.

A request's controls lie in a slot of :class:`LogitControls`, set once; a row of logits names its slot.  The tokens that a row has seen are read
from a token cache: ``[pages, 16]`` int32 ids beside the KV cache's pages, by the same block tables, written by :func:`cache_tokens` where
the KV write is - so that preemption, prefix reuse and captured decode steps need nothing more.

Of a row with controls, in this order: tokens of prompt or answer, ``x > 0 ? x / repetition : x * repetition``; tokens of the answer,
``x - frequency * count - presence``; biased tokens, ``x + bias``; tokens that are not allowed, -inf.  All in 32 bits, rounded once.
"""
from __future__ import annotations

from typing import Iterable, NamedTuple, Optional

import torch

from . import _gpu, native

PAGE = 16
MAX_BIAS = 2046  # biased tokens a slot
LARGEST = 1e30  # of a penalty or a finite bias


class LogitControls(NamedTuple):
    """Slots of controls, on the device of the logits."""

    params: torch.Tensor  # [slots, 3] fp32: repetition, presence, frequency
    info: torch.Tensor  # [slots, 2] int32: tokens of the prompt; whether the mask counts
    bias_ids: torch.Tensor  # [slots, m] int32, < 0: none; of several entries with one token the first counts
    bias_vals: torch.Tensor  # [slots, m] fp32
    masks: torch.Tensor  # [slots, ceil(V / 32)] int32: bit v % 32 of word v / 32 set where token v is allowed

    def set(self, slot: int, prompt_len: int, repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0,
            bias: Optional[dict] = None, allowed: Optional[Iterable[int]] = None) -> None:
        """Fills a slot: the penalties, ``bias`` {token: addend}, ``allowed`` token ids (None: all).  A few small copies to the device, in the
        order of the current stream; the host does not wait for what runs there."""
        if not 0 <= slot < self.params.shape[0]:
            raise ValueError(f"LogitControls.set: slot {slot} of {self.params.shape[0]}")
        check_controls(repetition, presence, frequency, bias)
        m, words = self.bias_ids.shape[1], self.masks.shape[1]
        bias = bias or {}
        if len(bias) > m:
            raise ValueError(f"LogitControls.set: {len(bias)} biased tokens, room for {m}")
        n = len(bias)
        mask = allowed_mask(allowed, words * 32) if allowed is not None else None
        # pinned memory, the allocator's own until the copies out of it are done: a copy from pageable memory would wait for the stream
        stage = torch.empty(5 + 2 * m + (words if mask is not None else 0), dtype=torch.int32, pin_memory=self.params.is_cuda)
        info, params, ids, vals = stage[:2], stage[2:5].view(torch.float32), stage[5:5 + m], stage[5 + m:5 + 2 * m].view(torch.float32)
        info.copy_(torch.tensor([prompt_len, int(mask is not None)], dtype=torch.int32))
        params.copy_(torch.tensor([repetition, presence, frequency], dtype=torch.float32))
        ids[:n] = torch.tensor([int(t) for t in bias], dtype=torch.int32)
        ids[n:] = -1
        vals[:n] = torch.tensor([float(x) for x in bias.values()], dtype=torch.float32)
        vals[n:] = 0
        if mask is not None:
            self.masks[slot].copy_(stage[5 + 2 * m:].copy_(mask), non_blocking=True)
        if m:
            self.bias_ids[slot].copy_(ids, non_blocking=True)
            self.bias_vals[slot].copy_(vals, non_blocking=True)
        self.params[slot].copy_(params, non_blocking=True)
        self.info[slot].copy_(info, non_blocking=True)


def check_controls(repetition: float = 1.0, presence: float = 0.0, frequency: float = 0.0, bias: Optional[dict] = None) -> None:
    """ValueError for controls without a meaning, or so large that sums of them would pass 32 bits (2^20 times a frequency penalty is the most)."""
    import math
    if not 1 / LARGEST <= repetition <= LARGEST:
        raise ValueError(f"repetition penalty {repetition}: a positive number, {1 / LARGEST} to {LARGEST}")
    if not (abs(presence) <= LARGEST and abs(frequency) <= LARGEST):
        raise ValueError(f"presence {presence} and frequency {frequency}: numbers up to {LARGEST}")
    for t, x in (bias or {}).items():
        if int(t) != t or t < 0 or not (abs(float(x)) <= LARGEST or math.isinf(x)):
            raise ValueError(f"bias {x!r} of token {t!r}: token ids and numbers up to {LARGEST}, or infinite")


def allowed_mask(allowed: Iterable[int], vocab: int) -> torch.Tensor:
    """int32 words with the bits of the ``allowed`` token ids set (ids outside the vocabulary are an error)."""
    ids = torch.as_tensor(list(allowed), dtype=torch.int64)
    if ids.numel() and (int(ids.min()) < 0 or int(ids.max()) >= vocab):
        raise ValueError(f"allowed tokens {int(ids.min())} .. {int(ids.max())}: the vocabulary has {vocab}")
    words = torch.zeros((vocab + 31) // 32, 32, dtype=torch.int64)
    words.view(-1)[ids] = 1
    w = (words << torch.arange(32)).sum(1)
    return torch.where(w >= 1 << 31, w - (1 << 32), w).to(torch.int32)


def logit_controls(slots: int, vocab: int, max_bias: int = 64, device=None) -> LogitControls:
    """Empty slots (no penalty, no bias, every token allowed)."""
    if not 0 <= max_bias <= MAX_BIAS:
        raise ValueError(f"logit_controls: at most {MAX_BIAS} biased tokens a slot")
    params = torch.zeros(slots, 3, dtype=torch.float32, device=device)
    params[:, 0] = 1.0
    return LogitControls(params, torch.zeros(slots, 2, dtype=torch.int32, device=device),
                         torch.full((slots, max_bias), -1, dtype=torch.int32, device=device),
                         torch.zeros(slots, max_bias, dtype=torch.float32, device=device),
                         torch.full((slots, (vocab + 31) // 32), -1, dtype=torch.int32, device=device))


def cache_tokens(token_cache: torch.Tensor, ids: torch.Tensor, slot_mapping: torch.Tensor, src: Optional[torch.Tensor] = None,
                 prev: Optional[torch.Tensor] = None) -> None:
    """Token ``ids`` [T] into the pages of ``slot_mapping`` (< 0: not written).  ``src``, ``prev``: as ``resolve_ids`` has them - where src[i] >= 0
    the id is prev[src[i]], the token that the step before sampled."""
    if _gpu(token_cache):
        native().cache_tokens(token_cache, ids, slot_mapping, src, prev)
        return
    if src is not None:
        r = src[: ids.numel()].long()
        ids = torch.where((r >= 0) & (r < prev.numel()), prev[r.clamp(0, max(0, prev.numel() - 1))], ids)
    sm = slot_mapping[: ids.numel()].long()
    ok = (sm >= 0) & (sm < token_cache.numel())
    token_cache.view(-1)[sm[ok]] = ids[ok]


def control_logits(logits: torch.Tensor, controls: LogitControls, rows: torch.Tensor, token_cache: torch.Tensor, block_tables: torch.Tensor,
                   seq_lens: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The controlled logits [B, V]: row b by slot ``rows[b]`` (outside the slots: as it is), its history the ``seq_lens[b]`` tokens of its pages
    (ids outside the vocabulary and pages outside the cache count for nothing), the first ``info[slot, 0]`` of them the prompt.  ``out``:
    ``logits`` itself (in place), or a tensor of its type or of float32.  A row whose mask allows nothing is all -inf."""
    if out is None:
        out = torch.empty_like(logits)
    if _gpu(logits):
        native().logit_controls(out, logits, *controls, rows, token_cache, block_tables, seq_lens)
        return out
    y = logits.to(torch.float32, copy=True)
    V = logits.shape[1]
    for b in range(logits.shape[0]):
        s = int(rows[b])
        if not 0 <= s < controls.params.shape[0]:
            continue
        n = max(0, min(int(seq_lens[b]), block_tables.shape[1] * PAGE))
        p = block_tables[b, : (n + PAGE - 1) // PAGE].long()
        there = (p >= 0) & (p < token_cache.shape[0])
        ids = torch.where(there[:, None], token_cache[p.clamp(0, token_cache.shape[0] - 1)], -1).reshape(-1)[:n].long()
        prompt, masked = controls.info[s].tolist()
        rep, pres, freq = controls.params[s]
        known = (ids >= 0) & (ids < V)
        seen = torch.zeros(V, dtype=torch.bool)
        seen[ids[known]] = True
        answer = ids[max(0, prompt):]
        count = torch.bincount(answer[(answer >= 0) & (answer < V)], minlength=V).float()
        x = y[b]
        x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
        x = torch.where(count > 0, x - freq * count - pres, x)
        add = {}
        for t, a in zip(controls.bias_ids[s].tolist(), controls.bias_vals[s].tolist()):
            if 0 <= t < V:
                add.setdefault(t, a)
        for t, a in add.items():
            x[t] += a
        if masked:
            bits = (controls.masks[s][:, None] >> torch.arange(32)) & 1
            x = torch.where(bits.reshape(-1)[:V] > 0, x, torch.full_like(x, float("-inf")))
        y[b] = x
    return out.copy_(y)
