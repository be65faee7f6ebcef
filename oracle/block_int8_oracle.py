"""int8 pools with one scale per block (one page of one KV head), restated in 64 bits.  Test infrastructure only.

A block's bytes go by the rows it holds, not by the calls that brought them, so the oracle quantises whole blocks:
``s`` is the power of two with ``64 s <= max |x| < 128 s`` (0 for zeros, at least 2^-126), the code ``floor(x / s)``, the
value ``(code + 1/2) s``.
"""

from __future__ import annotations

import math

import torch


def block_scale(amax: float) -> float:
    if amax == 0.0:
        return 0.0
    return max(2.0 ** (math.frexp(amax)[1] - 7), 2.0 ** -126)


def quantize_block(rows: torch.Tensor) -> tuple[torch.Tensor, float]:
    """``rows [n, D]`` of one block and head -> (int8 codes, scale).  Infinities saturate, NaN is code 0."""
    x = rows.double()
    finite = x[torch.isfinite(x)]
    s = block_scale(float(finite.abs().max()) if finite.numel() else 0.0)
    code = torch.floor(x / s) if s > 0 else torch.zeros_like(x)
    code = torch.where(torch.isnan(x), torch.zeros_like(x), code)
    code = torch.where(torch.isposinf(x), torch.full_like(x, 127.0), code)
    code = torch.where(torch.isneginf(x), torch.full_like(x, -128.0), code)
    return code.to(torch.int8), s


def quantize_blocks(rows: torch.Tensor, live: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The same for finite ``rows [B, P, D]`` of many blocks at once; ``live [B, P]``: the rows that exist (codes of the
    others are 0)."""
    x = torch.where(live.unsqueeze(-1), rows.double(), torch.zeros((), dtype=torch.float64, device=rows.device))
    amax = x.abs().amax((1, 2))
    _, e = torch.frexp(amax)
    s = torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), (e - 7).clamp(min=-126)), torch.zeros_like(amax))
    code = torch.where(s.view(-1, 1, 1) > 0, torch.floor(x / s.view(-1, 1, 1).clamp(min=2.0 ** -126)), torch.zeros_like(x))
    return code.to(torch.int8), s


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """``[n_pages, H, P, D]`` codes and ``[n_pages, H]`` scales -> float64 values."""
    return (codes.double() + 0.5) * scales.double()[:, :, None, None]


def attention(q, k_codes, k_scales, v_codes, v_scales, page_table, seqused_k, *, scale, causal=True, window=None,
              rows=None, visible_until=None):
    """float64 paged attention.  ``q [B, Sq, Hq, D]``; ``rows[b]``: valid query rows.  Returns ``(out, lse, weight,
    score, reach)``: the output and log-sum-exp, and what rounding errors are proportional to: per output element ``sum_j p_j
    |v_j|``, per row the largest ``scale * sum_d |q_d k_d|`` and the largest ``scale * max|q| * sum_d |k_d|``.  Rows without a key: zeros and -inf."""
    B, Sq, Hq, D = q.shape
    Hkv, P = k_codes.shape[1], k_codes.shape[2]
    g = Hq // Hkv
    dev = q.device
    out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device=dev)
    weight = torch.zeros_like(out)
    lse = torch.full((B, Hq, Sq), -math.inf, dtype=torch.float64, device=dev)
    score = torch.zeros(B, Sq, Hq, 1, dtype=torch.float64, device=dev)
    reach = torch.zeros_like(score)
    for b in range(B):
        n = int(seqused_k[b])
        sq = Sq if rows is None else int(rows[b])
        if n <= 0 or sq <= 0:
            continue
        pages = page_table[b, :-(-n // P)].long()
        K = dequantize(k_codes[pages], k_scales[pages]).transpose(1, 2).reshape(-1, Hkv, D)[:n].repeat_interleave(g, 1)
        V = dequantize(v_codes[pages], v_scales[pages]).transpose(1, 2).reshape(-1, Hkv, D)[:n].repeat_interleave(g, 1)
        x = q[b, :sq].double()
        z = torch.einsum("jhd,nhd->hjn", x, K) * scale
        za = torch.einsum("jhd,nhd->hjn", x.abs(), K.abs()) * scale
        j = torch.arange(sq, device=dev).view(-1, 1)
        at = torch.arange(n, device=dev).view(1, -1)
        ok = torch.ones(sq, n, dtype=torch.bool, device=dev)
        if causal or window is not None:
            last = j if visible_until is None else torch.maximum(j, visible_until[b, :sq].view(-1, 1).to(j).clamp(max=sq - 1))
            ok &= at <= n - sq + last
        if window is not None:
            ok &= at > n - sq + j - window
        z = z.masked_fill(~ok, -math.inf)
        p = torch.nan_to_num(torch.softmax(z, -1))
        out[b, :sq] = torch.einsum("hjn,nhd->jhd", p, V)
        weight[b, :sq] = torch.einsum("hjn,nhd->jhd", p, V.abs())
        lse[b, :, :sq] = torch.logsumexp(z, -1)
        ka = (K.abs().sum(-1).transpose(0, 1).unsqueeze(1) * scale).expand(Hq, sq, n).masked_fill(~ok, 0.0).amax(-1)
        reach[b, :sq] = (ka.transpose(0, 1) * x.abs().amax(-1)).unsqueeze(-1)
        score[b, :sq] = za.masked_fill(~ok, 0.0).amax(-1).transpose(0, 1).unsqueeze(-1)
    return out, lse, weight, score, reach
