"""int8 pools with a scale per block: the append against the exact 64-bit quantisation, attention against float64.

Append: power-of-two scales make codes and scales exactly determined, whatever the split over calls: bytes are compared.

Attention: the pool's values are exact in both computations, so an output element may be off by
  u_out |o|                                   its own rounding (u = half a step: bf16 2^-8, fp16 2^-11)
  u_p A                                       the rounding of the softmax weights, A = sum_j p_j |v_j|
  A (4 D 2^-24 S + 2^-20 + 2 n 2^-24)         fp32 products of D terms (S = scale * sum |q k| of the row, twice for an accumulator
                                              that truncates, numerator and denominator), the exponential, sums of n terms
  A 2 R 2^-15.9                               up to 16 packed rows the query is a 16-bit number relative to its row's largest, off by
                                              max|q| / 65024 at most: R = scale * max|q| * sum |k| of the row's worst key
  A 4 D 2^-24 scale 128 k_scale sum |q|       17 to 64 packed rows: K enters the products as code + 128, an offset taken out again
  n 2^-25 max|v|                              weights below f16's normal range
with u_p = 2^-8 where the products run on bf16 operands (prompt chunks of bf16 queries) and 2^-11 elsewhere.
"""

import math

import pytest
import torch

from kestrel_b200 import KVMemoryPool, PagedKVCache, PageTable, _native, kernels, paged_attention
from oracle import block_int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _views(*pools):
    return [p.permute(0, 2, 1, 3) for p in pools]


def _append(k, v, kc, vc, ks, vs, slots):
    kernels.reshape_and_cache_block_int8(k, v, *_views(kc, vc), ks, vs, slots)


def _clear_status():
    _native.device_status(0, clear=True)


# ---------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------

def _pools(n_pages, H, P, D):
    g = torch.Generator().manual_seed(1)
    kc, vc = (torch.randint(-128, 128, (n_pages, H, P, D), generator=g, dtype=torch.int8).to(DEV) for _ in range(2))
    ks, vs = (torch.rand(n_pages, H, generator=g).to(DEV) for _ in range(2))
    return kc, vc, ks, vs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("P,H,D", [(1, 2, 64), (4, 3, 128), (16, 8, 128), (24, 1, 48), (64, 2, 128), (128, 2, 64)])
def test_bytes_do_not_depend_on_the_split(dtype, P, H, D):
    """Sequences of odd lengths appended in pieces of 1, 3, P - 1, 40, 100.. tokens: every live byte and scale is
    that of the whole block at once; pages of nobody stay as they were."""
    g = torch.Generator().manual_seed(P * 131 + D)
    lengths = [1, P, P + 1, 2 * P + 3, 201]
    pages = [-(-n // P) for n in lengths]
    n_pages = sum(pages) + 3
    perm = torch.randperm(n_pages, generator=g)
    kc, vc, ks, vs = _pools(n_pages, H, P, D)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    # magnitudes climb along a sequence, so that scales grow in mid-block
    rows = [[(torch.randn(n, H, D, generator=g) * torch.exp2(torch.randint(-6, 7, (n, H, 1), generator=g).float())).to(dtype)
             for n in lengths] for _ in range(2)]
    at = [0] * len(lengths)
    base, tables = 0, []
    for c in pages:
        tables.append(perm[base:base + c])
        base += c
    pieces = [1, 3, max(1, P - 1), 40, 1, 100]
    step = 0
    while any(a < n for a, n in zip(at, lengths)):
        take = [min(pieces[(step + i) % len(pieces)], n - a) for i, (a, n) in enumerate(zip(at, lengths))]
        slots, parts = [], [[], []]
        for i, t in enumerate(take):
            pos = torch.arange(at[i], at[i] + t)
            slots.append(tables[i][pos // P] * P + pos % P)
            for kv in range(2):
                parts[kv].append(rows[kv][i][at[i]:at[i] + t])
            at[i] += t
        _append(*(torch.cat(p).to(DEV) for p in parts), kc, vc, ks, vs, torch.cat(slots).to(DEV))
        step += 1
    for kv, (cache, scale) in enumerate(((kc, ks), (vc, vs))):
        cache, scale = cache.cpu(), scale.cpu()
        used = set()
        for i, n in enumerate(lengths):
            for c, page in enumerate(tables[i].tolist()):
                live = rows[kv][i][c * P:(c + 1) * P]
                used.add(page)
                for h in range(H):
                    code, s = O.quantize_block(live[:, h])
                    assert float(scale[page, h]) == s, (i, c, h)
                    assert torch.equal(cache[page, h, :live.shape[0]], code), (i, c, h)
        for page in set(range(n_pages)) - used:
            assert torch.equal(cache[page], before[kv][page].cpu()) and torch.equal(scale[page], before[2 + kv][page].cpu())


@pytest.mark.parametrize("dtype,P,H,D", [(torch.bfloat16, 64, 8, 128), (torch.float16, 16, 8, 64), (torch.float32, 128, 8, 64),
                                         (torch.bfloat16, 256, 8, 128), (torch.bfloat16, 24, 16, 32), (torch.float32, 4, 8, 128)])
@pytest.mark.parametrize("aligned", [True, False])
def test_many_tokens(dtype, P, H, D, aligned):
    """Prompt chunks in numbers that give every warp a window of its own: two calls per sequence, the second one starting
    inside a page; a NaN, an infinity, a skipped token and equal slots among them."""
    _clear_status()
    g = torch.Generator(device=DEV).manual_seed(P + D)
    lengths = [1 + (i * 977) % 1500 for i in range(28)]
    pages = [-(-n // P) for n in lengths]
    n_pages = sum(pages) + 2
    perm = torch.randperm(n_pages, generator=g, device=DEV)
    table = torch.zeros(len(lengths), max(pages), dtype=torch.int64, device=DEV)
    at = 0
    for b, c in enumerate(pages):
        table[b, :c] = perm[at:at + c]
        at += c
    seq = torch.cat([torch.full((n,), b, device=DEV) for b, n in enumerate(lengths)])
    pos = torch.cat([torch.arange(n, device=DEV) for n in lengths])
    T = len(pos)
    extra = 0 if aligned else 1        # rows off the 16-byte boundary
    k, v = (torch.randn(T * H * D + 1, generator=g, device=DEV).to(dtype)[extra:extra + T * H * D].view(T, H, D) for _ in range(2))
    slots = table[seq, pos // P] * P + pos % P
    kc, vc, ks, vs = _pools(n_pages, H, P, D)
    first = pos < torch.tensor([n * 2 // 3 for n in lengths], device=DEV)[seq]
    for part in (first, ~first):
        i = torch.nonzero(part).view(-1)
        a, b = k[i], v[i]
        if not aligned:
            a, b = (torch.cat([x.reshape(-1)[:1], x.reshape(-1)])[1:].view(x.shape) for x in (a, b))
        _append(a, b, kc, vc, ks, vs, slots[i])
    block = table[seq, pos // P]
    live = torch.zeros(n_pages, P, dtype=torch.bool, device=DEV)
    live[block, pos % P] = True
    for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
        for h in range(H):
            rows = torch.zeros(n_pages, P, D, dtype=dtype, device=DEV)
            rows[block, pos % P] = x[:, h]
            code, s = O.quantize_blocks(rows, live)
            used = live.any(1)
            assert torch.equal(scale[used, h].double(), s[used]), h
            assert torch.equal(cache[:, h][live], code[live]), h
    assert _native.device_status(0)[0] == 0
    # the same once more in one call, with what does not belong there
    k2 = k.clone()
    long = lengths.index(max(lengths))
    at = int(torch.nonzero(seq == long)[0])
    k2[at + 3, 0, :3] = torch.tensor([math.nan, math.inf, -math.inf], dtype=dtype, device=DEV)
    slots2 = slots.clone()
    slots2[at + min(P, 3) - 1 + P * 2] = -1 if P > 4 else slots2[at + min(P, 3) - 1 + P * 2]
    if P > 8:
        slots2[at + P + 5] = slots2[at + P + 4]       # the later row counts
    _append(k2, v, kc, vc, ks, vs, slots2)
    assert _native.device_status(0)[0] == _native.STATUS_NOT_FINITE
    for c in range(2):
        page = int(table[long, c])
        toks = [t for t in range(at + c * P, at + min(lengths[long], (c + 1) * P)) if int(slots2[t]) >= 0]
        code, s = O.quantize_block(k2[toks, 0].cpu())
        assert float(ks[page, 0]) == s
        for j, t in enumerate(toks):
            if int(slots2[t]) not in slots2[t + 1:at + (c + 1) * P].tolist():
                assert torch.equal(kc[page, 0, int(slots2[t]) % P].cpu(), code[j]), (c, j)


def test_strides_alignment_negative_and_equal_slots():
    """Rows that are slices of a fused projection, rows off the 16-byte boundary, skipped tokens, equal slots in a run."""
    g = torch.Generator().manual_seed(3)
    H, D, P, T = 2, 64, 16, 90
    fused = torch.randn(T, 3 * H, D, generator=g).to(torch.bfloat16).to(DEV)
    flat = torch.randn(T * H * D + 1, generator=g).to(torch.bfloat16).to(DEV)
    for k, v in ((fused[:, H:2 * H], fused[:, 2 * H:]), (flat[1:].view(T, H, D), flat[1:].view(T, H, D))):
        kc, vc, ks, vs = _pools(12, H, P, D)
        before = kc.clone()
        slots = torch.arange(T) + 2 * P
        slots[5] = -1                     # splits its block's run in two neighbours' worth: moved to another page below
        slots[6:16] = torch.arange(10) + 10 * P
        slots[40] = slots[39]             # the later row counts
        slots[41] = slots[39]
        _append(k, v, kc, vc, ks, vs, slots.to(DEV))
        for x, cache, scale in ((k, kc, ks), (v, vc, vs)):
            x, cache, scale = x.cpu(), cache.cpu(), scale.cpu()
            where = {}
            amax = {}
            for t, s in enumerate(slots.tolist()):
                if s >= 0:
                    where[s] = t
                    amax.setdefault(s // P, []).append(t)
            for page, toks in amax.items():
                for h in range(H):
                    s = O.block_scale(float(x[toks, h].double().abs().max()))
                    assert float(scale[page, h]) == s
                    for slot, t in where.items():
                        if slot // P == page:
                            assert torch.equal(cache[page, h, slot % P], torch.floor(x[t, h].double() / s).to(torch.int8)), (page, slot)
        assert torch.equal(kc[0].cpu(), before[0].cpu())


def test_extremes():
    """Zeros, the smallest and the largest numbers, NaN and infinities, a growth by more than eight powers of two."""
    _clear_status()
    H, D, P = 1, 16, 4
    big = torch.finfo(torch.float32).max
    rows = torch.zeros(6, H, D)
    rows[1, 0, :3] = torch.tensor([1e-45, -1e-45, 1e-39])
    rows[2, 0, :4] = torch.tensor([big, -big, 1e-30, -1e-30])
    rows[3, 0, :4] = torch.tensor([math.nan, math.inf, -math.inf, 1.0])
    rows[4, 0, :2] = torch.tensor([1.0, -1.0])
    rows[5, 0, :2] = torch.tensor([-64.0, 2.0 ** -140])
    rows = rows.to(DEV)
    kc, vc, ks, vs = _pools(8, H, P, D)
    _append(rows, rows, kc, vc, ks, vs, (torch.arange(6) * P).to(DEV))
    for i in range(6):
        code, s = O.quantize_block(rows[i].cpu())
        assert float(ks[i, 0]) == s and torch.equal(kc[i, 0, :1].cpu(), code), i
        assert float(vs[i, 0]) == s and torch.equal(vc[i, 0, :1].cpu(), code), i
    assert _native.device_status(0)[0] == _native.STATUS_NOT_FINITE
    # a block of 2^-40, then 1.0: the codes become those of 2^-40 under the new scale, 0 and -1
    x = torch.full((2, H, D), 2.0 ** -40)
    x[0, 0, 1] = -2.0 ** -40
    x[1] = 1.0
    x = x.to(DEV)
    for t in range(2):
        _append(x[t:t + 1], x[t:t + 1], kc, vc, ks, vs, torch.tensor([7 * P + t], device=DEV))
    code, s = O.quantize_block(x[:, 0].cpu())
    assert float(ks[7, 0]) == s and torch.equal(kc[7, 0, :2].cpu(), code)
    assert _native.device_status(0)[0] == 0


def test_slots_past_the_pool_are_reported_and_skipped():
    _clear_status()
    kc, vc, ks, vs = _pools(2, 1, 4, 16)
    before = [t.clone() for t in (kc, vc, ks, vs)]
    x = torch.ones(3, 1, 16, device=DEV)
    _append(x, x, kc, vc, ks, vs, torch.tensor([8, 1 << 40, -5], device=DEV))
    assert _native.device_status(0)[0] == _native.STATUS_BAD_SLOT
    assert all(torch.equal(a, b) for a, b in zip(before, (kc, vc, ks, vs)))


def test_append_refusals():
    kc, vc, ks, vs = _pools(4, 2, 4, 32)
    x = torch.zeros(3, 2, 32, device=DEV)
    s = torch.arange(3, device=DEV)
    ok = dict(key=x, value=x, key_cache=kc.permute(0, 2, 1, 3), value_cache=vc.permute(0, 2, 1, 3), key_scales=ks,
              value_scales=vs, slot_mapping=s)
    kernels.reshape_and_cache_block_int8(**ok)
    for bad, err in ((dict(key=x[:2]), ValueError), (dict(slot_mapping=s.int()), ValueError), (dict(slot_mapping=s[:2]), RuntimeError),
                     (dict(key_cache=kc), ValueError), (dict(key_scales=ks.half()), ValueError), (dict(value_scales=vs[:2]), ValueError),
                     (dict(key=x.double(), value=x.double()), ValueError), (dict(key=x.cpu()), RuntimeError),
                     (dict(key_scales=ks.t().contiguous().t(), value_scales=vs.t().contiguous().t()), ValueError),
                     (dict(key_cache=kc.view(torch.uint8).permute(0, 2, 1, 3), value_cache=vc.view(torch.uint8).permute(0, 2, 1, 3)), ValueError)):
        with pytest.raises(err):
            kernels.reshape_and_cache_block_int8(**{**ok, **bad})
    odd = torch.zeros(4, 2, 4, 24, dtype=torch.int8, device=DEV).permute(0, 2, 1, 3)
    with pytest.raises(NotImplementedError, match="head_dim 24"):
        y = torch.zeros(3, 2, 24, device=DEV)
        kernels.reshape_and_cache_block_int8(y, y, odd, odd.clone(memory_format=torch.preserve_format), ks, vs, s)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

def _problem(seed, lengths, Hq, Hkv, D, P, Sq, dtype, spread=3, spare=2):
    g = torch.Generator().manual_seed(seed)
    pages = [-(-n // P) for n in lengths]
    n_pages = sum(pages) + spare
    perm = (torch.randperm(n_pages - 1, generator=g) + 1).to(torch.int32)
    table = torch.full((len(lengths), max(pages + [1]) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    codes = [(torch.randn(n_pages, Hkv, P, D, generator=g) * 27).floor().clamp(-128, 127).to(torch.int8) for _ in range(2)]
    scales = [torch.exp2(-torch.randint(5 - spread // 2, 6 + spread // 2, (n_pages, Hkv), generator=g).float()) for _ in range(2)]
    scales[1][torch.rand(n_pages, Hkv, generator=g) < 0.05] = 0.0           # blocks of zeros
    scales[0][torch.rand(n_pages, Hkv, generator=g) < 0.05] = 0.0
    q = torch.randn(len(lengths), Sq, Hq, D, generator=g).to(dtype)
    return dict(q=q.to(DEV), kc=codes[0].to(DEV), vc=codes[1].to(DEV), ks=scales[0].to(DEV), vs=scales[1].to(DEV),
                table=table.to(DEV), lens=torch.tensor(lengths, dtype=torch.int32, device=DEV), scale=D ** -0.5)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check(got, p, *, lse=None, bf16_products=False, **kw):
    out, want_lse, weight, score, reach = O.attention(p["q"], p["kc"], p["ks"], p["vc"], p["vs"], p["table"], p["lens"], scale=p["scale"], **kw)
    D = p["q"].shape[-1]
    n = int(p["lens"].max())
    vmax = float((128 * p["vs"].max()).double())
    u_p = _half_step(torch.bfloat16) if bf16_products and p["q"].dtype == torch.bfloat16 else _half_step(torch.float16)
    reach = reach / 65024 * 2
    offset = 4 * D * 2.0 ** -24 * p["scale"] * 128 * float(p["ks"].max()) * p["q"].double().abs().sum(-1, keepdim=True)
    reach = reach + offset
    rel = u_p + 4 * D * 2.0 ** -24 * score + reach + 2.0 ** -20 + 2 * n * 2.0 ** -24
    tol = weight * rel + n * 2.0 ** -25 * vmax
    tol = tol + _half_step(p["q"].dtype) * (out.abs() + tol) + 1e-30
    err = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    assert bool((err <= tol).all()), (float((err / tol).max()), float(err.max()))
    if lse is not None:
        same = torch.isinf(want_lse) == torch.isinf(lse)
        assert bool(same.all())
        d = (lse.double() - want_lse).abs()[torch.isfinite(want_lse)]
        # fp32 scores and sum: the same relative terms as the weights', and the value's own rounding
        most = 4 * D * 2.0 ** -24 * float(score.max()) + float(reach.max()) + 2.0 ** -19 + 2 * n * 2.0 ** -24 + 2.0 ** -22 * float(want_lse[torch.isfinite(want_lse)].abs().max())
        assert float(d.max()) <= most


def _run(p, **kw):
    return kernels.flash_attn_fwd(p["q"], *_views(p["kc"], p["vc"]), page_table=p["table"], seqused_k=p["lens"], softmax_scale=p["scale"],
                                  k_block_scale=p["ks"], v_block_scale=p["vs"], return_lse=True, **kw)


LENGTHS = [1, 700, 0, 33, 129, 16, 1537, 64]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Hq,Hkv,D", [(8, 2, 128), (4, 4, 64), (16, 2, 64), (8, 1, 128)])
@pytest.mark.parametrize("P", [1, 2, 4, 16, 32, 64, 256])
@pytest.mark.parametrize("Sq", [1, 3])
def test_decode_and_verify(dtype, Hq, Hkv, D, P, Sq):
    """The transposed kernel (up to 8 packed rows) and the 16-row kernel, gathered and copied by boxes; lengths of 0
    and 1, lengths shorter than the query rows."""
    p = _problem(P * 7 + Sq, LENGTHS, Hq, Hkv, D, P, Sq, dtype)
    out, lse = _run(p, causal=True)
    _check(out, p, lse=lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,P,Sq", [(128, 16, 5), (64, 1, 6), (128, 64, 8), (64, 4, 12), (128, 2, 16), (64, 128, 11)])
def test_rows32(dtype, D, P, Sq):
    """17 to 64 packed rows per KV head."""
    p = _problem(Sq, LENGTHS, 8, 2, D, P, Sq, dtype)
    out, lse = _run(p, causal=True)
    _check(out, p, lse=lse)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,P,Sq", [(128, 16, 17), (64, 16, 32), (128, 64, 40), (128, 1, 70), (64, 4, 100), (128, 256, 130), (64, 2, 129)])
def test_prefill(dtype, D, P, Sq):
    """More packed rows: the tensor-memory kernel with and without its key split."""
    p = _problem(Sq, [Sq, 0, 700, 129, 1537, 3], 8, 2, D, P, Sq, dtype)
    out, lse = _run(p, causal=True)
    _check(out, p, lse=lse, bf16_products=True)


def test_prefill_key_split_at_a_cta_per_sm():
    """33 to 64 packed rows go to the tensor-memory kernel once the batch gives every SM a CTA."""
    p = _problem(9, [37 + 11 * (i % 40) for i in range(80)], 8, 2, 128, 16, 10, torch.bfloat16)
    out, lse = _run(p, causal=True)
    _check(out, p, lse=lse, bf16_products=True)


@pytest.mark.parametrize("Sq", [1, 4, 9, 40])
@pytest.mark.parametrize("window", [1, 17, 200])
def test_sliding_window(Sq, window):
    p = _problem(Sq + window, LENGTHS, 8, 2, 128, 16, Sq, torch.bfloat16)
    out, lse = _run(p, window_size_left=window - 1, window_size_right=0)
    _check(out, p, lse=lse, window=window, bf16_products=True)


@pytest.mark.parametrize("Sq", [1, 4, 12, 80])
def test_no_mask_and_short_rows(Sq):
    """causal=False, and seqused_q: rows past a sequence's own are left as they were."""
    p = _problem(Sq, [5, 300, 80, 1], 8, 2, 64, 16, Sq, torch.float16)
    out, lse = _run(p, causal=False)
    _check(out, p, lse=lse, causal=False)
    rows = torch.tensor([1, Sq, max(1, Sq // 2), 0], dtype=torch.int32, device=DEV)
    out = torch.full_like(p["q"], 7.0)
    _run(p, causal=True, seqused_q=rows, out=out)
    keep = torch.arange(Sq, device=DEV).view(1, -1) >= rows.view(-1, 1)
    assert bool((out[keep] == 7.0).all())
    out[keep] = 0
    _check(out, p, rows=rows)


@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 0, 1, 7], [40, 1, 90, 2]])
def test_packed_rows(counts):
    p = _problem(sum(counts), [100, 17, 300, 64], 8, 2, 128, 16, max(counts), torch.bfloat16)
    cu = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist(), dtype=torch.int32, device=DEV)
    q = torch.cat([p["q"][b, :c] for b, c in enumerate(counts)])
    got, _ = kernels.flash_attn_fwd(q, *_views(p["kc"], p["vc"]), page_table=p["table"], seqused_k=p["lens"], cu_seqlens_q=cu,
                                    max_seqlen_q=max(counts), softmax_scale=p["scale"], causal=True, k_block_scale=p["ks"], v_block_scale=p["vs"])
    out = torch.zeros_like(p["q"])
    for b, c in enumerate(counts):
        out[b, :c] = got[int(cu[b]):int(cu[b + 1])]
    _check(out, p, rows=counts, bf16_products=True)


@pytest.mark.parametrize("Sq", [1, 3, 7, 40])
def test_blocks_of_very_different_scales(Sq):
    """Scales from 2^-16 to 2^4 side by side: weights are kept relative to the largest V scale, whose own block may
    hardly be attended to."""
    p = _problem(Sq, [900, 130], 8, 2, 128, 16, Sq, torch.bfloat16, spread=0)
    g = torch.Generator().manual_seed(4)
    p["vs"] = torch.exp2(torch.randint(-16, 5, p["vs"].shape, generator=g).float()).to(DEV)
    p["ks"] = torch.exp2(torch.randint(-12, -3, p["ks"].shape, generator=g).float()).to(DEV)
    out, lse = _run(p, causal=True)
    _check(out, p, lse=lse, bf16_products=True)


@pytest.mark.parametrize("Sq", [1, 4])
def test_shared_prefix(Sq):
    """The batch's common pages read once: same result up to the rounding of the two partial outputs to q's type."""
    p = _problem(11, [160 + 16 + 3 * b + Sq for b in range(24)], 8, 2, 64, 16, Sq, torch.bfloat16)
    p["table"][:, :10] = p["table"][0, :10].clone()
    out, _ = _run(p, causal=True, shared_prefix_pages=10)
    plain, _ = _run(p, causal=True)
    # three roundings to bf16 (two partials and the sum) and bf16 weights in the prefix pass, on values up to A
    _, _, weight, _, _ = O.attention(p["q"], p["kc"], p["ks"], p["vc"], p["vs"], p["table"], p["lens"], scale=p["scale"])
    assert bool(((out.double() - plain.double()).abs() <= 5 * 2.0 ** -8 * weight + 1e-6).all())


def test_image_block_mask():
    Sq = 50
    p = _problem(2, [Sq, Sq + 70], 8, 2, 64, 16, Sq, torch.float16)
    ids = torch.full((2, Sq), -1, dtype=torch.int32, device=DEV)
    ids[0, 5:30] = 0
    ids[1, 20:49] = 3
    out, lse = _run(p, mask_mod=kernels.block_bidirectional_mask, aux_tensors=[ids])
    _check(out, p, lse=lse, visible_until=kernels.block_visibility(ids))


def test_bad_pages_are_reported_and_read_as_nothing():
    _clear_status()
    p = _problem(1, [64, 64], 8, 2, 128, 16, 1, torch.bfloat16)
    p["table"][1, 2] = 10 ** 6
    out, _ = _run(p, causal=True)
    assert torch.isfinite(out).all()
    assert _native.device_status(0)[0] & _native.STATUS_BAD_PAGE


def test_attention_refusals():
    p = _problem(1, [10], 8, 2, 64, 16, 1, torch.bfloat16)
    for change, err in ((dict(k_block_scale=None), ValueError), (dict(v_block_scale=p["vs"][:, :1]), ValueError),
                        (dict(v_block_scale=p["vs"].half()), ValueError), (dict(k_block_scale=p["ks"].cpu()), RuntimeError)):
        kw = dict(k_block_scale=p["ks"], v_block_scale=p["vs"])
        kw.update(change)
        with pytest.raises(err):
            kernels.flash_attn_fwd(p["q"], *_views(p["kc"], p["vc"]), page_table=p["table"], seqused_k=p["lens"], causal=True, **kw)
    with pytest.raises(ValueError, match="int8"):
        kernels.flash_attn_fwd(p["q"], *_views(p["kc"].to(torch.bfloat16), p["vc"].to(torch.bfloat16)), page_table=p["table"],
                               seqused_k=p["lens"], causal=True, k_block_scale=p["ks"], v_block_scale=p["vs"])


def test_callers_built_before_the_int8_pools(monkeypatch):
    """The argument struct without its last three fields is still served; any other size is refused."""
    g = torch.Generator().manual_seed(2)
    kc, vc = (torch.randn(6, 2, 16, 64, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    q = torch.randn(2, 1, 8, 64, generator=g).to(torch.bfloat16).to(DEV)
    table = torch.tensor([[1, 2], [3, 4]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([20, 31], dtype=torch.int32, device=DEV)
    call = lambda: kernels.flash_attn_fwd(q, *_views(kc, vc), page_table=table, seqused_k=lens, causal=True)[0]  # noqa: E731
    want = call()
    sizeof = kernels.C.sizeof
    before = _native.AttnArgs.k_block_scale.offset
    for size, served in ((before, True), (before - 8, False), (before + 8, False)):
        kernels._ws_bytes_cache.clear()
        monkeypatch.setattr(kernels.C, "sizeof", lambda t, size=size: size if t is _native.AttnArgs else sizeof(t))
        if served:
            assert torch.equal(call(), want)
        else:
            with pytest.raises(ValueError, match="size mismatch"):
                call()
    monkeypatch.undo()
    kernels._ws_bytes_cache.clear()


def test_large_pool_offsets_pass_32_bits():
    """A pool of over 2^32 bytes: pages at both ends."""
    P, D, H = 256, 128, 8
    n_pages = (1 << 32) // (P * D * H) + 3
    kc = torch.zeros(n_pages, H, P, D, dtype=torch.int8, device=DEV)
    vc = torch.zeros_like(kc)
    ks, vs = torch.zeros(n_pages, H, device=DEV), torch.zeros(n_pages, H, device=DEV)
    g = torch.Generator().manual_seed(8)
    rows = [torch.randn(300, H, D, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2)]
    pages = torch.tensor([n_pages - 1, n_pages - 2])
    pos = torch.arange(300)
    _append(*rows, kc, vc, ks, vs, (pages[pos // P] * P + pos % P).to(DEV))
    code, s = O.quantize_block(rows[0][:P, H - 1].cpu())
    assert torch.equal(kc[n_pages - 1, H - 1].cpu(), code) and float(ks[n_pages - 1, H - 1]) == s
    for Sq in (1, 40):
        p = dict(q=torch.randn(1, Sq, 16, D, generator=g).to(torch.bfloat16).to(DEV), kc=kc, vc=vc, ks=ks, vs=vs,
                 table=pages.to(torch.int32).view(1, 2).to(DEV), lens=torch.tensor([300], dtype=torch.int32, device=DEV), scale=D ** -0.5)
        out, lse = _run(p, causal=True)
        _check(out, p, lse=lse, bf16_products=True)


# ---------------------------------------------------------------------------
# through the cache classes
# ---------------------------------------------------------------------------

def test_cache_layer_append_rotary_copy_and_attention():
    """PagedKVCache(dtype=int8): update, rope_update, copy-on-write with the scales, paged_attention; on a side stream."""
    g = torch.Generator().manual_seed(5)
    H, D, P = 2, 64, 16
    pool = KVMemoryPool(device=DEV)
    pt = PageTable(n_pages=32, page_size=P, max_batch_size=4, device=DEV)
    layer = PagedKVCache(pt, n_heads=H, head_dim=D, dtype=torch.int8, pool=pool)
    row = pt.allocate()
    pt.reserve(row, 60)
    pt.commit_block_table()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        pos = torch.arange(41, device=DEV).view(1, -1)
        k, v, q = (torch.randn(1, 41, n, D, generator=g).to(torch.bfloat16).to(DEV) for n in (H, H, 4 * H))
        idx = torch.tensor([row], device=DEV)
        layer.update(pos[:, :40], k[:, :40], v[:, :40], slot_mapping=pt.build_slot_mapping(idx, pos[:, :40]))
        ang = torch.outer(torch.arange(64).float(), torch.rand(D // 2, generator=g))
        cs = torch.cat([ang.cos(), ang.sin()], 1).to(DEV)
        qr, kr = q[:, 40:].clone(), k[:, 40:].clone()
        layer.rope_update(pos[:, 40:], qr, kr, v[:, 40:], cs, slot_mapping=pt.build_slot_mapping(idx, pos[:, 40:]))
        want_q, want_k = q[:, 40:].clone(), k[:, 40:].clone()
        kernels.rotary_embedding(pos[:, 40:], want_q, want_k, D, cs)
        assert torch.equal(qr, want_q) and torch.equal(kr, want_k)
        table = pt.page_table[row:row + 1]
        lens = torch.tensor([41], dtype=torch.int32, device=DEV)
        out = paged_attention(qr.transpose(1, 2), paged_kv_layer=layer, page_table=table, paged_kv_seqlens_k=lens, scaling=D ** -0.5)
        p = dict(q=qr, kc=layer.k_cache, vc=layer.v_cache, ks=layer.k_block_scale, vs=layer.v_block_scale, table=table, lens=lens, scale=D ** -0.5)
        _check(out, p)
        live = torch.cat([k[0, :40], kr[0]])
        pages = pt.get_pages(row, 0, 3)
        for c, page in enumerate(pages):
            for h in range(H):
                code, s = O.quantize_block(live[c * P:(c + 1) * P, h].cpu())
                assert float(layer.k_block_scale[page, h]) == s and torch.equal(layer.k_cache[page, h, :code.shape[0]].cpu(), code)
        from kestrel_b200 import copy_kv_pages
        src, dst = pt.cow_page(row, 2)
        copy_kv_pages([layer], *pt.take_pending_page_copies())
        assert torch.equal(layer.v_cache[dst], layer.v_cache[src]) and torch.equal(layer.v_block_scale[dst], layer.v_block_scale[src])
        assert torch.equal(layer.k_block_scale[dst], layer.k_block_scale[src])
        with pytest.raises(NotImplementedError):
            layer.rope_update(pos[:, 40:], qr, kr, v[:, 40:], cs, slot_mapping=pt.build_slot_mapping(idx, pos[:, 40:]), write_k=False)
        torch.cuda.current_stream().synchronize()
    with pytest.raises(ValueError, match="scale per block"):
        PagedKVCache(pt, n_heads=H, head_dim=D, dtype=torch.int8, pool=pool, k_scale=1.0, v_scale=1.0)
