"""Beam search on a paged cache, restated in 64 bits: selection over beams and vocabulary, and the reordering of
tables and partly filled pages.  Test infrastructure only."""

from __future__ import annotations

import math

import torch


def candidates(logits: torch.Tensor, scores: torch.Tensor, finished=None, end_token: int = 0) -> torch.Tensor:
    """float64 ``[B, W, V]``: ``score + logit - logsumexp``; a NaN logit counts as -inf; rows with nothing finite, or a
    score that is not finite, are -inf throughout; a finished beam has its end token at its own score."""
    B, W = scores.shape
    x = logits.double().view(B, W, -1)
    x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    lse = torch.logsumexp(x, -1, keepdim=True)
    s = scores.double().unsqueeze(-1)
    live = torch.isfinite(lse) & torch.isfinite(s)
    cand = torch.where(live, s + (x - torch.where(live, lse, torch.zeros_like(lse))), torch.full_like(x, -math.inf))
    if finished is not None:
        kept = torch.full_like(x, -math.inf)
        kept[:, :, end_token] = torch.where(torch.isfinite(scores), scores.double(), torch.full_like(scores.double(), -math.inf))
        cand = torch.where(finished.unsqueeze(-1), kept, cand)
    return cand


def select(cand: torch.Tensor, n_out: int):
    """Largest first, equal ones by the lowest flat index -> (tokens, parents, float64 scores)."""
    B, W, V = cand.shape
    value, at = torch.sort(cand.view(B, -1), dim=1, descending=True, stable=True)
    return at[:, :n_out] % V, at[:, :n_out] // V, value[:, :n_out]


def reorder(beam_table, own_table, parents, lengths, page_size, caches, scales=None, own_rows=None):
    """The tables, caches and scales after the reordering (new tensors)."""
    B, W = parents.shape
    table = beam_table.clone()
    caches = [c.clone() for c in caches]
    scales = [s.clone() for s in scales] if scales else []
    for b in range(B):
        full, rest = divmod(int(lengths[b]), page_size)
        before = [(c.clone() if rest else c) for c in caches]
        before_s = [s.clone() for s in scales]
        for w in range(W):
            q = int(parents[b, w])
            if not 0 <= q < W or q == w:
                continue
            table[b * W + w, :full] = beam_table[b * W + q, :full]
            if rest:
                row = [int(own_rows[b * W + i]) if own_rows is not None else b * W + i for i in (w, q)]
                dst, src = int(own_table[row[0], full]), int(own_table[row[1], full])
                for c, old in zip(caches, before):
                    c[dst, :, :rest] = old[src, :, :rest]
                for s, old in zip(scales, before_s):
                    s[dst] = old[src]
    return table, caches, scales
