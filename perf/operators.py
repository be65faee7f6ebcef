"""Cases of the block-scaled int8 cache (append, attention), of the step tables built from request lengths and of
beam search (selection, reordering of paged states): their inputs, their plain forms and what they cost.

``own`` false: ``run`` computes the plain form with elementary torch operations.  ``own`` true: ``run`` makes the calls
a user makes of ``kestrel_b200``.

An int8 pool ``[n_pages, H, P, D]`` holds codes; a block is one page of one head, with one fp32 scale in
``[n_pages, H]``.  An element is ``(code + 1/2) * scale``; the scale is the power of two ``s`` with
``64 s <= max |x| < 128 s`` over the block's rows (0 for a block of zeros) and the code is ``floor(x / s)``.  Codes and
scales are therefore determined exactly: they are returned as they lie in the pools, and are equal or wrong.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f16": 2, "f32": 4, "int8": 1}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 256 sequences: one token each, most of them into a page that already holds some
        dict(name="append decode 256", op="append", seqs=256, tokens_lo=1, tokens_hi=1, heads=8, head_dim=128, page=16, dtype="bf16"),
        # eight prompt chunks of ragged lengths, starting anywhere in a page
        dict(name="append chunks 8x2k", op="append", seqs=8, tokens_lo=1500, tokens_hi=2600, heads=8, head_dim=128, page=64, dtype="bf16"),
        # a single sequence's decode call: latency
        dict(name="attend one 900", op="attention", batch=1, len_lo=900, len_hi=900, q_heads=32, kv_heads=8, head_dim=128, page=16,
             q_len=1, window=0, dtype="bf16"),
        # a decode batch of mixed context lengths, larger than L2
        dict(name="attend 64 U[2k,16k]", op="attention", batch=64, len_lo=2048, len_hi=16384, q_heads=32, kv_heads=8, head_dim=128,
             page=16, q_len=1, window=0, dtype="bf16"),
        # a verify step of four tokens, heads of 64, one sequence without keys, odd lengths
        dict(name="attend verify4 h64", op="attention", batch=48, len_lo=0, len_hi=5003, q_heads=16, kv_heads=4, head_dim=64,
             page=32, q_len=4, window=0, dtype="f16"),
        # prompt chunks on cached tokens: bound by the products
        dict(name="attend chunk 512", op="attention", batch=4, len_lo=2048, len_hi=4608, q_heads=32, kv_heads=8, head_dim=128,
             page=64, q_len=512, window=0, dtype="bf16"),
        # a decode step's tables: every request one token
        dict(name="tables decode 256", op="tables", batch=256, len_lo=1, len_hi=8192, new_lo=1, new_hi=1, page=16),
        # chunked prefill and decode rows in one step
        dict(name="tables mixed 1000", op="tables", batch=1000, len_lo=0, len_hi=4096, new_lo=1, new_hi=255, page=16),
        # a few beams of one request: latency
        dict(name="beams 1x4", op="beam", batch=1, beams=4, out=8, vocab=51200, finished=0, dtype="bf16"),
        # a serving batch: 512 rows of a large vocabulary
        dict(name="beams 64x8", op="beam", batch=64, beams=8, out=16, vocab=151936, finished=1, dtype="bf16"),
        # moving the partly filled pages of 24 layers, a small 16-bit batch and a large int8 one
        dict(name="reorder 2x4", op="reorder", batch=2, beams=4, len_lo=700, len_hi=900, new=48, layers=24, heads=8, head_dim=128,
             page=16, kind="bf16"),
        dict(name="reorder 32x8 int8", op="reorder", batch=32, beams=8, len_lo=200, len_hi=1200, new=64, layers=24, heads=8, head_dim=128,
             page=16, kind="int8"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attention", "attention", "tables", "beam", "reorder"])
    if op == "append":
        lo = _log_int(rng, 1, 1500)
        hi = lo + rng.randrange(0, lo + 1)
        heads, head_dim = rng.choice([(8, 128), (4, 64), (32, 64), (2, 128), (1, 128)])
        most = max(1, 16000 * 1024 // (hi * heads * head_dim))
        return dict(op=op, seqs=_log_int(rng, 1, min(512, most)), tokens_lo=lo, tokens_hi=hi, heads=heads, head_dim=head_dim,
                    page=rng.choice([1, 4, 16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16", "f32"]))
    if op == "attention":
        q_heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (16, 4, 64), (32, 32, 64), (8, 1, 128), (16, 2, 128)])
        q_len = rng.choice([1, 1, 1, 2, 4, 7, 16, 33, 150, 400])
        hi = _log_int(rng, 40, 12000 if q_len <= 16 else 4000)
        lo = rng.randrange(0, hi + 1)
        most = min(64 * 16384 * 1024 // (hi * kv_heads * head_dim * 2), (1 << 28) // (hi * q_heads * q_len))
        return dict(op=op, batch=_log_int(rng, 1, max(1, min(96, most))), len_lo=lo, len_hi=hi, q_heads=q_heads, kv_heads=kv_heads,
                    head_dim=head_dim, page=rng.choice([1, 4, 16, 32, 64, 128]), q_len=q_len,
                    window=rng.choice([0, 0, 0, rng.randrange(1, 1500)]), dtype=rng.choice(["bf16", "f16"]))
    if op == "tables":
        hi = _log_int(rng, 1, 600)
        return dict(op=op, batch=_log_int(rng, 1, 1000), len_lo=0, len_hi=_log_int(rng, 1, 8192), new_lo=rng.randrange(0, hi + 1), new_hi=hi,
                    page=rng.choice([1, 4, 16, 64, 256]))
    if op == "beam":
        beams = rng.choice([1, 2, 3, 4, 5, 8, 10, 16])
        vocab = _log_int(rng, 1000, 200000)
        most = max(1, 64 * 8 * 151936 // (beams * vocab * 2))
        return dict(op=op, batch=_log_int(rng, 1, min(128, most)), beams=beams, out=rng.choice([beams, 2 * beams]), vocab=vocab,
                    finished=rng.randrange(2), dtype=rng.choice(["bf16", "f16", "f32"]))
    beams = rng.choice([2, 3, 4, 6, 8, 12])
    lo = _log_int(rng, 20, 1000)
    return dict(op=op, batch=_log_int(rng, 1, 192 // beams), beams=beams, len_lo=lo, len_hi=lo + rng.randrange(0, 200), new=rng.randrange(1, 65),
                layers=rng.choice([1, 7, 24]), heads=rng.choice([2, 8]), head_dim=rng.choice([64, 128]),
                page=rng.choice([1, 4, 16, 32]), kind=rng.choice(["bf16", "int8"]))


def _ints(case, what, n, lo, hi):
    """``n`` whole numbers of [lo, hi] that go by the case alone: lengths and parents, which decide the work."""
    r = random.Random("%s %s" % (what, sorted((k, v) for k, v in case.items() if k != "name")))
    return [r.randint(lo, hi) for _ in range(n)]


def _lengths(case):
    got = _ints(case, "len", case["batch"], case["len_lo"], case["len_hi"])
    if case["len_lo"] == 0:
        got[0] = 0
    got[-1] = case["len_hi"]
    return got


def _append_lengths(case):
    """(tokens held before, tokens appended) of every sequence."""
    new = _ints(case, "new", case["seqs"], case["tokens_lo"], case["tokens_hi"])
    return _ints(case, "held", case["seqs"], 0, 4 * case["page"]), new


def _parents(case):
    return _ints(case, "parents", case["batch"] * case["beams"], 0, case["beams"] - 1)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _pages(gen, counts, spare=8):
    """A random page table of ``counts[i]`` pages per row (page 0 stays out), -1 behind; and the number of pages."""
    total = sum(counts)
    n_pages = total + spare
    perm = torch.randperm(n_pages - 1, generator=gen, device="cuda")[:total].to(torch.int32) + 1
    table = torch.full((len(counts), max(counts + [1])), -1, dtype=torch.int32, device="cuda")
    cols = torch.arange(table.shape[1], device="cuda")
    table[cols < torch.tensor(counts, device="cuda").view(-1, 1)] = perm
    return table, n_pages


def _codes(gen, shape):
    """Codes as the quantiser leaves them for normal values, and scales that are powers of two."""
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    flat = codes.view(shape[0], -1)
    step = max(1, (1 << 27) // max(1, flat.shape[1]))
    for i in range(0, shape[0], step):
        x = torch.randn(flat[i:i + step].shape, generator=gen, device="cuda", dtype=torch.float16)
        flat[i:i + step] = (x * 27).floor_().clamp_(-128, 127).to(torch.int8)
    return codes, torch.exp2(-torch.randint(4, 7, shape[:2], generator=gen, device="cuda").float())


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    s = SimpleNamespace(case=dict(case), op=case["op"])
    if s.op == "append":
        held, new = _append_lengths(case)
        P, H, D, dt = case["page"], case["heads"], case["head_dim"], _DTYPES[case["dtype"]]
        table, n_pages = _pages(gen, [-(-(h + n) // P) for h, n in zip(held, new)])
        T = sum(new)
        held_t, new_t = torch.tensor(held, device=dev), torch.tensor(new, device=dev)
        row = torch.repeat_interleave(torch.arange(len(new), device=dev), new_t)
        pos = held_t[row] + torch.arange(T, device=dev) - (torch.cumsum(new_t, 0) - new_t)[row]
        s.slots = table[row, pos // P].long() * P + pos % P
        # rows as a fused projection leaves them: K and V are slices of one buffer, magnitudes differ between heads
        fused = torch.randn(T, 4 * H, D, generator=gen, device=dev)
        fused *= torch.exp2(torch.randint(-2, 3, (4 * H, 1), generator=gen, device=dev).float())
        fused = fused.to(dt)
        s.key, s.value = fused[:, 2 * H:3 * H], fused[:, 3 * H:]
        # what the blocks hold already: codes and scales of the tokens before
        s.k_cache, s.k_scale = _codes(gen, (n_pages, H, P, D))
        s.v_cache, s.v_scale = _codes(gen, (n_pages, H, P, D))
        return s
    if s.op == "attention":
        L, P = _lengths(case), case["page"]
        s.table, n_pages = _pages(gen, [-(-n // P) for n in L])
        s.lengths = torch.tensor(L, dtype=torch.int32, device=dev)
        dt = _DTYPES[case["dtype"]]
        s.q = torch.randn(case["batch"], case["q_len"], case["q_heads"], case["head_dim"], generator=gen, device=dev).to(dt)
        shape = (n_pages, case["kv_heads"], P, case["head_dim"])
        k, ks = _codes(gen, shape)
        v, vs = _codes(gen, shape)
        s.layer = SimpleNamespace(k_cache=k, v_cache=v, k_block_scale=ks, v_block_scale=vs)
        s.scaling = case["head_dim"] ** -0.5
        s.window = case["window"] or None
        return s
    if s.op == "tables":
        L, P, B = _lengths(case), case["page"], case["batch"]
        new = _ints(case, "new", B, case["new_lo"], case["new_hi"])
        held = [-(-n // P) for n in L]
        cols = -(-(case["len_hi"] + case["new_hi"]) // P) + 1
        table, n_pages = _pages(gen, held, spare=8 + sum(new))
        order = torch.randperm(B, generator=gen, device=dev) + 1          # the requests' rows; row 0 is the padding row
        s.table = torch.full((B + 1, cols), -1, dtype=torch.int32, device=dev)
        s.table[0] = 0
        s.table[order, :table.shape[1]] = table
        s.rows = order.to(torch.int32)
        used = torch.zeros(n_pages, dtype=torch.bool, device=dev)
        used[table[table >= 0].long()] = True
        used[0] = True
        free = torch.nonzero(~used).view(-1).to(torch.int32)
        free = free[torch.randperm(free.numel(), generator=gen, device=dev)]
        s.free, s.free_count = free, torch.tensor([free.numel()], dtype=torch.int32, device=dev)
        s.lengths = torch.tensor(L, dtype=torch.int32, device=dev)
        s.new = torch.tensor(new, dtype=torch.int32, device=dev)
        s.n_tokens = sum(new) + 37                                        # a bucket: its tail holds no tokens
        s.n_pages = n_pages
        s.out_table = torch.full((B, cols), -1, dtype=torch.int32, device=dev)
        return s
    if s.op == "beam":
        B, W, V = case["batch"], case["beams"], case["vocab"]
        s.logits = torch.empty(B * W, V, dtype=_DTYPES[case["dtype"]], device=dev)
        for i in range(0, B * W, 64):
            s.logits[i:i + 64] = torch.randn(s.logits[i:i + 64].shape, generator=gen, device=dev) * 3
        s.scores = -torch.rand(B, W, generator=gen, device=dev) * 6 - 20
        s.finished = (torch.rand(B, W, generator=gen, device=dev) < 0.2) if case["finished"] else None
        s.end = 2
        return s
    if s.op == "reorder":
        B, W, P, n = case["batch"], case["beams"], case["page"], case["new"]
        L = _lengths(case)
        R = B * W
        # every request's prompt lies in shared pages, what its beams add in pages of their own
        shared = [max(0, x - n) // P for x in L]
        cols = max(-(-(x + 1) // P) for x in L)
        table, n_shared = _pages(gen, shared, spare=1)
        own_pages = [-(-(x + 1) // P) - k for x, k in zip(L, shared)]
        counts = [k for k in own_pages for _ in range(W)]
        perm, n_own = _pages(gen, counts, spare=8)
        n_pages = n_shared + n_own
        s.own_table = torch.full((R, cols), -1, dtype=torch.int32, device=dev)
        row, col = torch.arange(R, device=dev).view(-1, 1), torch.arange(cols, device=dev).view(1, -1)
        first = torch.tensor(shared, device=dev).repeat_interleave(W).view(-1, 1)
        last = first + torch.tensor(counts, device=dev).view(-1, 1)
        from_prompt = table[:, torch.arange(cols, device=dev).clamp(max=table.shape[1] - 1)].repeat_interleave(W, 0)
        mine = perm.gather(1, (col - first).clamp(0, perm.shape[1] - 1)) + n_shared
        s.own_table = torch.where(col < first, from_prompt, torch.where(col < last, mine, s.own_table)).contiguous()
        # the table that is read: a full page of its own may by now be another beam's
        full = torch.tensor([x // P for x in L], device=dev).repeat_interleave(W).view(-1, 1)
        other = torch.randint(0, W, (R, cols), generator=gen, device=dev) + row // W * W
        s.table = torch.where((col >= first) & (col < full), s.own_table.gather(0, other), s.own_table).contiguous()
        s.parents = torch.tensor(_parents(case), device=dev).view(B, W)
        s.lengths = torch.tensor(L, dtype=torch.int32, device=dev)
        shape = (2 * case["layers"], n_pages, case["heads"], P, case["head_dim"])
        if case["kind"] == "int8":
            s.pools = torch.randint(-128, 128, shape, generator=gen, dtype=torch.int8, device=dev)
            s.scales = torch.exp2(-torch.randint(3, 9, shape[:3], generator=gen, device=dev).float())
        else:
            s.pools = torch.empty(shape, dtype=torch.bfloat16, device=dev).normal_(generator=gen)
            s.scales = None
        s.pool_list, s.scale_list = list(s.pools.unbind(0)), None if s.scales is None else list(s.scales.unbind(0))
        return s
    raise ValueError(s.op)


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------

def _pow2_scale(amax):
    """The power of two s with 64 s <= amax < 128 s; 0 for 0 (fp32 in, fp32 out)."""
    _, e = torch.frexp(amax)                     # amax = m 2^e, 1/2 <= m < 1
    return torch.where(amax > 0, torch.ldexp(torch.ones_like(amax), e - 7), torch.zeros_like(amax))


def _plain_append_one(rows, cache, scale, slots):
    P = cache.shape[2]
    page, off = slots // P, slots % P
    x = rows.float()
    start = torch.zeros(cache.shape[0], dtype=torch.bool, device=x.device)
    start[page[off == 0]] = True                 # a block whose first token is written starts anew
    touched = torch.zeros_like(start)
    touched[page] = True
    old = torch.where(start.view(-1, 1), torch.zeros_like(scale), scale)
    new = old.clone().scatter_reduce_(0, page.view(-1, 1).expand(-1, x.shape[1]), _pow2_scale(x.abs().amax(-1)), "amax")
    grown = torch.nonzero(touched & ~start & (new > old).any(1)).view(-1)
    k = torch.where(old[grown] > 0, torch.log2(new[grown] / old[grown]), torch.zeros_like(old[grown])).clamp(max=31)
    cache[grown] = torch.floor(cache[grown].float() * torch.exp2(-k)[:, :, None, None]).to(torch.int8)
    s = new[page].unsqueeze(-1)
    code = torch.where(s > 0, torch.floor(x / s.clamp(min=1e-38)), torch.zeros_like(x))
    cache[page, :, off] = code.to(torch.int8)
    scale.copy_(new)


def _plain_attention(s):
    c, layer = s.case, s.layer
    B, Sq, Hq, D = s.q.shape
    Hkv, P = c["kv_heads"], c["page"]
    table = s.table.clamp(min=0).long()
    n = table.shape[1] * P

    def values(cache, scale):
        v = (cache[table].float() + 0.5) * scale[table][:, :, :, None, None]          # [B, pages, H, P, D]
        return v.permute(0, 2, 1, 3, 4).reshape(B, Hkv, n, D)

    q = s.q.float().view(B, Sq, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    score = (q @ values(layer.k_cache, layer.k_block_scale).transpose(2, 3)) * s.scaling
    score = score.view(B, Hkv, Hq // Hkv, Sq, n)
    key = torch.arange(n, device=q.device).view(1, 1, n)
    limit = (s.lengths.view(B, 1) - Sq + torch.arange(Sq, device=q.device).view(1, Sq)).unsqueeze(-1)
    seen = (key <= limit) & (key < s.lengths.view(B, 1, 1))
    if s.window is not None:
        seen &= key > limit - s.window
    score = score.masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    w = torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = w.sum(-1, keepdim=True)
    w = (w / torch.where(total > 0, total, torch.ones_like(total))).view(B, Hkv, -1, n)
    out = w @ values(layer.v_cache, layer.v_block_scale)
    return out.view(B, Hkv, Hq // Hkv, Sq, D).permute(0, 3, 1, 2, 4).reshape(B, Sq, Hq, D).to(s.q.dtype)


def _plain_tables(s):
    P, B = s.case["page"], s.case["batch"]
    dev = s.table.device
    rows, L, new = s.rows.long(), s.lengths.long(), s.new.long()
    held, want = (L + P - 1) // P, (L + new + P - 1) // P
    need = want - held
    cum, cu = torch.cumsum(need, 0), torch.cumsum(new, 0)
    # page j that row i takes is free[count - cum[i] + j]
    entry = torch.repeat_interleave(torch.arange(B, device=dev), need)
    j = torch.arange(entry.numel(), device=dev) - (cum - need)[entry]
    s.table[rows[entry], held[entry] + j] = s.free[s.free_count.long() - cum[entry] + j]
    used = torch.arange(s.table.shape[1], device=dev).view(1, -1) < want.view(-1, 1)
    s.out_table[used] = s.table[rows][used]
    owner = torch.repeat_interleave(torch.arange(B, device=dev), new)
    pos = L[owner] + torch.arange(owner.numel(), device=dev) - (cu - new)[owner]
    slots = torch.full((s.n_tokens,), -1, dtype=torch.int64, device=dev)
    positions = torch.zeros(s.n_tokens, dtype=torch.int64, device=dev)
    slots[:pos.numel()] = s.table[rows[owner], pos // P].long() * P + pos % P
    positions[:pos.numel()] = pos
    return dict(page_table=s.table, out_page_table=s.out_table, seqused_k=(L + new).int(),
                cu_seqlens_q=torch.cat([cu.new_zeros(1), cu]).int(), slot_mapping=slots, positions=positions,
                free_count=s.free_count - need.sum().int(), pages_taken=need.sum().int().view(1))


def _plain_beam(s):
    B, W = s.scores.shape
    V, K = s.logits.shape[1], s.case["out"]
    x = s.logits.double().view(B, W, V)          # 64 bits: candidates of different beams lie close to one another
    top = x.amax(-1, keepdim=True)
    cand = s.scores.double().unsqueeze(-1) + (x - top - torch.log(torch.exp(x - top).sum(-1, keepdim=True)))
    if s.finished is not None:                   # a finished beam goes on as itself, by the end token alone
        at_end = torch.arange(V, device=x.device).view(1, 1, V) == s.end
        kept = torch.where(at_end, s.scores.double().unsqueeze(-1), torch.full_like(cand, -math.inf))
        cand = torch.where(s.finished.unsqueeze(-1), kept, cand)
    value, at = torch.sort(cand.view(B, W * V), dim=1, descending=True, stable=True)
    value, at = value[:, :K], at[:, :K]
    return dict(tokens=at % V, parents=at // V, scores=value.float())


def _plain_reorder(s):
    B, W = s.parents.shape
    P = s.case["page"]
    dev = s.table.device
    base = torch.arange(B, device=dev).view(B, 1) * W
    parent = (base + s.parents).view(-1)
    L = s.lengths.long().repeat_interleave(W)
    full, rest = L // P, L % P
    col = torch.arange(s.table.shape[1], device=dev).view(1, -1)
    s.table.copy_(torch.where(col < full.view(-1, 1), s.table[parent], s.table))
    row = torch.nonzero((parent != torch.arange(B * W, device=dev)) & (rest > 0)).view(-1)
    src, dst = s.own_table[parent[row], full[row]].long(), s.own_table[row, full[row]].long()
    live = (torch.arange(P, device=dev).view(1, P) < rest[row].view(-1, 1)).view(1, -1, 1, P, 1)
    s.pools[:, dst] = torch.where(live, s.pools[:, src], s.pools[:, dst])
    if s.scales is not None:
        s.scales[:, dst] = s.scales[:, src]
    return [s.table, s.pools] + ([] if s.scales is None else [s.scales])


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    c = s.case
    if s.op == "append":
        if own:
            from kestrel_b200 import kernels
            kernels.reshape_and_cache_block_int8(s.key, s.value, s.k_cache.permute(0, 2, 1, 3), s.v_cache.permute(0, 2, 1, 3),
                                                 s.k_scale, s.v_scale, s.slots)
        else:
            _plain_append_one(s.key, s.k_cache, s.k_scale, s.slots)
            _plain_append_one(s.value, s.v_cache, s.v_scale, s.slots)
        return dict(k_codes=s.k_cache, v_codes=s.v_cache, k_scale=s.k_scale, v_scale=s.v_scale)
    if s.op == "attention":
        if own:
            from kestrel_b200 import paged_attention
            return paged_attention(s.q.transpose(1, 2), paged_kv_layer=s.layer, page_table=s.table,
                                   paged_kv_seqlens_k=s.lengths, scaling=s.scaling, sliding_window=s.window)
        return _plain_attention(s)
    if s.op == "tables":
        if own:
            from kestrel_b200 import kernels
            r = kernels.build_ragged_step(s.table, s.rows, s.lengths, s.new, s.free, s.free_count, c["page"], n_pages=s.n_pages,
                                          n_tokens=s.n_tokens, out_page_table=s.out_table)
            return dict(page_table=s.table, out_page_table=s.out_table, seqused_k=r.seqused_k, cu_seqlens_q=r.cu_seqlens_q,
                        slot_mapping=r.slot_mapping, positions=r.positions, free_count=r.free_count, pages_taken=r.pages_taken)
        return _plain_tables(s)
    if s.op == "beam":
        if own:
            from kestrel_b200 import kernels
            r = kernels.beam_step_from_logits(s.logits, s.scores, c["out"], finished=s.finished, end_token=s.end)
            return dict(tokens=r.tokens, parents=r.parents, scores=r.scores)
        return _plain_beam(s)
    if own:
        from kestrel_b200 import kernels
        kernels.reorder_beam_pages(s.table, s.own_table, s.parents, s.lengths, c["page"], s.pool_list, scales=s.scale_list)
        return [s.table, s.pools] + ([] if s.scales is None else [s.scales])
    return _plain_reorder(s)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "append":
        held, new = _append_lengths(case)
        T, P = sum(new), case["page"]
        n = T * case["heads"] * case["head_dim"]
        blocks = sum(-(-(h + m) // P) - h // P for h, m in zip(held, new) if m)
        return {"bytes": 2 * n * (_BYTES[case["dtype"]] + 1) + 8 * T + 2 * 4 * blocks * case["heads"], "flops": 2 * 3 * n}
    if case["op"] == "attention":
        L, Sq, D, win = _lengths(case), case["q_len"], case["head_dim"], case["window"]
        pairs = keys = blocks = 0
        for n in L:
            first = 0 if not win else max(0, n - Sq - win + 1)
            keys += n - first
            blocks += -(-n // case["page"]) - first // case["page"]
            for j in range(Sq):
                seen = max(0, n - Sq + j + 1)
                pairs += min(seen, win) if win else seen
        rows = case["batch"] * Sq * case["q_heads"] * D * 2
        return {"bytes": 2 * keys * case["kv_heads"] * D + blocks * (8 * case["kv_heads"] + 4) + 2 * rows,
                "flops": 4 * case["q_heads"] * D * pairs}
    if case["op"] == "tables":
        L, P = _lengths(case), case["page"]
        new = _ints(case, "new", case["batch"], case["new_lo"], case["new_hi"])
        have = sum(-(-n // P) for n in L)
        want = sum(-(-(n + m) // P) for n, m in zip(L, new))
        return {"bytes": 4 * have + 4 * want + 8 * (want - have) + 16 * (sum(new) + 37) + 24 * case["batch"], "flops": 4 * sum(new)}
    if case["op"] == "beam":
        n = case["batch"] * case["beams"] * case["vocab"]
        return {"bytes": n * _BYTES[case["dtype"]] + 4 * case["batch"] * case["beams"] + 20 * case["batch"] * case["out"], "flops": 4 * n}
    L, W, P, parents = _lengths(case), case["beams"], case["page"], _parents(case)
    tokens = blocks = table = 0
    for b, n in enumerate(L):
        mine = parents[b * W:(b + 1) * W]
        moved = [p for w, p in enumerate(mine) if p != w]
        if n % P:
            tokens += (len(set(moved)) + len(moved)) * (n % P)
            blocks += len(set(moved)) + len(moved)
        table += (len(set(moved)) + len(moved)) * (n // P)
    pools = 2 * case["layers"] * case["heads"]
    more = 4 * pools * blocks if case["kind"] == "int8" else 0
    return {"bytes": tokens * pools * case["head_dim"] * _BYTES[case["kind"]] + more + 4 * table + 12 * len(parents), "flops": 0}


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    if s.op == "append":
        got = {}
        P = case["page"]
        for name, rows, scale in (("k_scale", s.key, s.k_scale), ("v_scale", s.value, s.v_scale)):
            want = scale.double().cpu()
            size = rows.double().abs().amax(-1).cpu()
            page, off = (s.slots // P).cpu(), (s.slots % P).cpu()
            begun = page[off == 0]
            want[begun] = 0.0
            s_row = torch.where(size > 0, 2.0 ** (torch.floor(torch.log2(size.clamp(min=1e-300))) - 6), torch.zeros_like(size))
            for h in range(want.shape[1]):
                want[:, h].index_reduce_(0, page, s_row[:, h], "amax")
            got[name] = want
        return dict(k_codes=None, v_codes=None, **got)
    if s.op == "attention":
        B, Sq, Hq, D = s.q.shape
        P, g = case["page"], Hq // case["kv_heads"]
        out = torch.zeros(B, Sq, Hq, D, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s.lengths.tolist()):
            if n == 0:
                continue
            pages = s.table[b, :-(-n // P)].long()

            def rows(cache, scale):
                return ((2.0 * cache[pages].double() + 1.0) * (0.5 * scale[pages].double())[..., None, None]).transpose(1, 2).flatten(0, 1)[:n]
            K, V = rows(s.layer.k_cache, s.layer.k_block_scale), rows(s.layer.v_cache, s.layer.v_block_scale)
            at = torch.arange(n, device="cuda").view(1, -1)
            for js in torch.arange(Sq, device="cuda").split(64):
                last = (n - Sq + js).view(-1, 1)                 # the last key that each query position sees
                ok = (at <= last) if not s.window else (at <= last) & (at > last - s.window)
                z = torch.einsum("jhgd,nhd->hgjn", s.q[b, js].double().view(len(js), -1, g, D), K) * s.scaling
                p = torch.nan_to_num(torch.softmax(z.masked_fill(~ok, -math.inf), -1))
                out[b, js] = torch.einsum("hgjn,nhd->jhgd", p, V).reshape(len(js), Hq, D)
        return out
    if s.op == "beam":
        B, W = s.scores.shape
        V, K = case["vocab"], case["out"]
        best = torch.empty(B, K, dtype=torch.float64)
        for b in range(B):
            lp = torch.log_softmax(s.logits[b * W:(b + 1) * W].double(), -1) + s.scores[b].double().view(W, 1)
            if s.finished is not None:
                for w in torch.nonzero(s.finished[b]).view(-1).tolist():
                    lp[w] = -math.inf
                    lp[w, s.end] = s.scores[b, w].double()
            best[b] = torch.topk(lp.flatten(), K).values.cpu()
        return dict(tokens=None, parents=None, scores=best)
    return None
