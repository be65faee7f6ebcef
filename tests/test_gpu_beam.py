"""Beam search: selection against float64 candidates, reordering against plain copies.

Tokens and parents are compared exactly; the random cases are chosen so that neighbouring candidates of different
value differ by more than the kernel's error, which is asserted on the oracle's values.  That error: a row's sum of exponentials
is off by at most 2^-21 relatively (fp32 exponentials of 2 ulp, an argument rounded once; 64 bits across threads), so a log-sum-exp
by 2^-21, and a score by that and its own rounding, 2^-24 of its value.
"""

import math

import pytest
import torch

from kestrel_b200 import KVMemoryPool, PagedKVCache, PageTable, _native, kernels, paged_attention, reorder_beams
from oracle import beam_oracle as S
from oracle import block_int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
NEAR = 2.0 ** -19


def _select(logits, scores, K, finished=None, end=0):
    cand = S.candidates(logits, scores, finished, end)
    tokens, parents, value = S.select(cand, min(K + 1, cand.shape[1] * cand.shape[2]))
    gap = (value[:, :-1] - value[:, 1:])
    near = (gap > 0) & (gap < NEAR)
    assert not bool(near.any()), "inputs of this test: candidates closer than the kernel can tell apart"
    r = kernels.beam_step_from_logits(logits.to(DEV), scores.to(DEV), K, finished=finished.to(DEV) if finished is not None else None, end_token=end)
    assert torch.equal(r.tokens.cpu(), tokens[:, :K]) and torch.equal(r.parents.cpu(), parents[:, :K])
    got, want = r.scores.cpu().double(), value[:, :K]
    assert torch.equal(torch.isinf(got), torch.isinf(want))
    ok = torch.isfinite(want)
    assert bool(((got - want).abs()[ok] <= 2.0 ** -21 + 2.0 ** -24 * want.abs()[ok] + 2.0 ** -40).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,W,V,K", [(1, 1, 5, 5), (1, 4, 51200, 8), (3, 2, 1003, 4), (2, 5, 32000, 10), (9, 8, 20011, 16), (1, 64, 700, 64),
                                     (40, 4, 30000, 8), (2, 3, 262144, 6)])
def test_selection(dtype, B, W, V, K):
    g = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(B * W, V, generator=g) * 3).to(dtype)
    _select(logits, -torch.rand(B, W, generator=g) * 8, K)


def test_selection_strided_rows():
    """Row strides and a start that rule out 16-byte loads, and ones that allow them."""
    g = torch.Generator().manual_seed(1)
    for off, stride in ((0, 1024), (3, 1001)):
        base = torch.randn(6 * stride + off, generator=g).to(torch.bfloat16)
        logits = base.as_strided((6, 1000), (stride, 1), off)
        scores = -torch.rand(2, 3, generator=g)
        want = S.select(S.candidates(logits, scores), 6)
        dev = base.to(DEV).as_strided((6, 1000), (stride, 1), off)
        r = kernels.beam_step_from_logits(dev, scores.to(DEV), 6)
        assert torch.equal(r.tokens.cpu(), want[0]) and torch.equal(r.parents.cpu(), want[1])


def test_ties_go_to_the_lowest_index():
    """All logits equal, -0 next to 0, equal rows: beam 0's first tokens, then the next beam's."""
    for V in (3, 40, 9000):
        for x in (torch.zeros(2, V), torch.zeros(2, V).index_fill_(1, torch.tensor([1]), -0.0)):
            _select(x, torch.zeros(1, 2), min(6, 2 * V))
    # 64 of 64 equal rows: over a thousand elements of a slice and candidates of the request reach the thresholds
    _select(torch.zeros(64, 20000), torch.zeros(1, 64), 64)


def test_first_step_and_dead_rows():
    """Beams that do not exist yet (-inf), rows of -inf, NaN, a row with +inf, a NaN score: only -inf candidates, lowest first."""
    g = torch.Generator().manual_seed(2)
    x = torch.randn(8, 3000, generator=g)
    scores = torch.tensor([[0.0, -math.inf, -math.inf, -math.inf], [-1.0, -2.0, math.nan, -0.5]])
    x[1, 5] = 50.0                      # (beam 1 of request 0 does not exist)
    x[4] = -math.inf
    x[5, :10] = math.nan
    x[7, 17] = math.inf
    _select(x, scores, 8)
    x[0, 4:] = -math.inf                # four tokens left: the rest of the candidates are -inf, lowest flat index first
    _select(x, scores, 8)


@pytest.mark.parametrize("K", [3, 6])
def test_finished_beams(K):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(9, 500, generator=g)
    scores = -torch.rand(3, 3, generator=g)
    finished = torch.tensor([[True, False, False], [True, True, True], [False, False, True]])
    for end in (0, 2, 499):
        _select(x, scores, K, finished, end)


def test_many_survivors():
    """Every good candidate in few threads' hands: the merge cannot rank them at once and goes round by round."""
    g = torch.Generator().manual_seed(4)
    W, V, K = 64, 65536, 64
    x = torch.randn(W, V, generator=g)
    x[3, 8192:8192 + 4000] += 30
    x[7, :4000] += 30
    for w in range(0, 64, 2):
        x[w, 8192 * 2:8192 * 2 + 2000] += 40
        x[w, 8192 * 5:8192 * 5 + 2000] += 40
    scores = torch.zeros(1, W)
    cand = S.candidates(x, scores)
    tokens, parents, value = S.select(cand, K)
    r = kernels.beam_step_from_logits(x.to(DEV), scores.to(DEV), K)
    # (thousands of candidates lie close together: each choice is one of the best up to the kernel's error)
    got = cand[0, r.parents.cpu()[0], r.tokens.cpu()[0]]
    assert bool(((got - value[0]).abs() <= NEAR).all())
    assert len(set(zip(r.parents.cpu()[0].tolist(), r.tokens.cpu()[0].tolist()))) == K
    assert bool(((r.scores.cpu()[0].double() - got).abs() <= 2.0 ** -21 + 2.0 ** -24 * got.abs()).all())


def test_out_graph_and_streams():
    """Written into the caller's tensors; captured and replayed on new logits; another stream at the same time."""
    g = torch.Generator().manual_seed(5)
    B, W, V, K = 2, 4, 5000, 8
    x, s = torch.randn(B * W, V, generator=g).to(DEV), torch.zeros(B, W, device=DEV)
    out = kernels.BeamStep(torch.empty(B, K, dtype=torch.int64, device=DEV), torch.empty(B, K, dtype=torch.int64, device=DEV),
                           torch.empty(B, K, device=DEV))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert kernels.beam_step_from_logits(x, s, K, out=out).tokens is out.tokens
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kernels.beam_step_from_logits(x, s, K, out=out)
    for i in range(3):
        x.copy_(torch.randn(B * W, V, generator=g))
        torch.cuda.synchronize()
        graph.replay()
        other = kernels.beam_step_from_logits(x, s, K)
        torch.cuda.synchronize()
        tokens, parents, _ = S.select(S.candidates(x.cpu(), s.cpu()), K)
        assert torch.equal(out.tokens.cpu(), tokens) and torch.equal(out.parents.cpu(), parents)
        assert torch.equal(other.tokens, out.tokens) and torch.equal(other.scores, out.scores)


def test_selection_refusals():
    x, s = torch.zeros(6, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    for a, err in (((x, s, 0), ValueError), ((x, s.double(), 2), ValueError), ((x[:5], s, 2), ValueError), ((x.t(), s, 2), ValueError),
                   ((x.long(), s, 2), ValueError), ((x, s, 65), NotImplementedError), ((x, s, 31), ValueError), ((x.cpu(), s, 2), RuntimeError)):
        with pytest.raises(err):
            kernels.beam_step_from_logits(*a)
    f = torch.zeros(2, 3, dtype=torch.bool, device=DEV)
    with pytest.raises(ValueError):
        kernels.beam_step_from_logits(x, s, 2, finished=f, end_token=10)
    with pytest.raises(ValueError):
        kernels.beam_step_from_logits(x, s, 2, finished=f.int())
    assert kernels.beam_step_from_logits(x[:0], s[:0], 2).tokens.shape == (0, 2)
    assert kernels.beam_step_from_logits(x, s, 30).tokens[0].tolist() == list(range(10)) * 3


# ---------------------------------------------------------------------------
# reordering
# ---------------------------------------------------------------------------

def _beams(seed, lengths, W, P, H, D, dtype, n_pools, scaled=False, row_map=False):
    g = torch.Generator().manual_seed(seed)
    B, R = len(lengths), len(lengths) * W
    cols = max(-(-(n + 1) // P) for n in lengths) + 1
    n_rows = R + 3 if row_map else R
    n_pages = n_rows * cols + 1
    own = (torch.randperm(n_pages - 1, generator=g)[:n_rows * cols] + 1).to(torch.int32).view(n_rows, cols)
    own_rows = torch.randperm(n_rows, generator=g)[:R] if row_map else None
    table = (own if own_rows is None else own[own_rows]).clone()
    for b, n in enumerate(lengths):
        for c in range(n // P):      # full pages may be another beam's
            pick = torch.randint(0, W, (W,), generator=g) + b * W
            table[b * W:(b + 1) * W, c] = (own if own_rows is None else own[own_rows])[pick, c]
    if dtype == torch.int8:
        caches = [torch.randint(-128, 128, (n_pages, H, P, D), generator=g, dtype=torch.int8) for _ in range(n_pools)]
    else:
        caches = [torch.randn(n_pages, H, P, D, generator=g).to(dtype) for _ in range(n_pools)]
    scales = [torch.rand(n_pages, H, generator=g) for _ in range(n_pools)] if scaled else None
    return g, table, own, own_rows, caches, scales


def _reorder(table, own, own_rows, parents, lengths, P, caches, scales):
    L = torch.tensor(lengths, dtype=torch.int32)
    want = S.reorder(table, own, parents, L, P, caches, scales, own_rows)
    t, c = table.to(DEV), [x.to(DEV) for x in caches]
    s = [x.to(DEV) for x in scales] if scales else None
    kernels.reorder_beam_pages(t, own.to(DEV), parents.to(DEV), L.to(DEV), P, c, scales=s,
                               own_rows=own_rows.to(DEV) if own_rows is not None else None)
    assert torch.equal(t.cpu(), want[0])
    for a, b in zip(c, want[1]):
        assert torch.equal(a.cpu(), b)
    for a, b in zip(s or [], want[2]):
        assert torch.equal(a.cpu(), b)


@pytest.mark.parametrize("W", [1, 2, 4, 7, 16, 32])
@pytest.mark.parametrize("P,H,D,dtype", [(16, 2, 64, torch.bfloat16), (1, 4, 64, torch.float16), (4, 3, 20, torch.bfloat16), (16, 2, 128, torch.int8),
                                         (8, 1, 8, torch.float32)])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_reorder(W, P, H, D, dtype, idx):
    """Random parents, the identity, all from one beam, a rotation, a swap: lengths of 0, inside the first page, at a page's end."""
    lengths = [0, 1, P, 3 * P + P // 2, 5 * P + 1]
    g, table, own, own_rows, caches, scales = _beams(W + P, lengths, W, P, H, D, dtype, 3, scaled=dtype == torch.int8, row_map=W % 2 == 0)
    n = torch.arange(W)
    for parents in (torch.randint(0, W, (5, W), generator=g), n.expand(5, W), torch.full((5, W), W - 1), n.roll(1).expand(5, W), n.flip(0).expand(5, W)):
        _reorder(table, own, own_rows, parents.to(idx).contiguous(), lengths, P, caches, scales)


def test_reorder_many_pools_and_requests():
    """More pools than one launch takes, more requests than SMs; scale arrays of 100 layers."""
    g, table, own, own_rows, caches, scales = _beams(1, [5, 21], 3, 8, 1, 16, torch.int8, 200, scaled=True)
    _reorder(table, own, own_rows, torch.tensor([[2, 0, 1], [1, 1, 0]]), [5, 21], 8, caches, scales)
    lengths = [1 + 3 * (i % 17) for i in range(200)]
    g, table, own, own_rows, caches, scales = _beams(2, lengths, 4, 4, 1, 16, torch.bfloat16, 2)
    _reorder(table, own, own_rows, torch.randint(0, 4, (200, 4), generator=g), lengths, 4, caches, scales)


def test_reorder_bad_parents_and_pages_are_reported():
    _native.device_status(0, clear=True)
    g, table, own, own_rows, caches, scales = _beams(3, [6, 6], 2, 4, 1, 16, torch.bfloat16, 2)
    _reorder(table, own, own_rows, torch.tensor([[-1, 5], [1, 0]]), [6, 6], 4, caches, scales)     # out of range: stays as it is
    assert _native.device_status(0)[0] == _native.STATUS_BAD_ROW
    t, c = table.to(DEV), [x.to(DEV) for x in caches]
    bad = own.clone()
    bad[0, 1] = 10 ** 6
    kernels.reorder_beam_pages(t, bad.to(DEV), torch.tensor([[1, 0], [0, 1]], device=DEV), torch.tensor([6, 6], dtype=torch.int32, device=DEV), 4, c)
    assert _native.device_status(0)[0] == _native.STATUS_BAD_PAGE
    assert all(torch.equal(a.cpu(), b) for a, b in zip(c, caches))
    kernels.reorder_beam_pages(t, own.to(DEV), torch.tensor([[1, 0], [0, 1]], device=DEV), torch.tensor([400, 6], dtype=torch.int32, device=DEV), 4, c)
    assert _native.device_status(0)[0] == _native.STATUS_BAD_ROW


def test_reorder_refusals():
    g, table, own, own_rows, caches, scales = _beams(4, [6], 2, 4, 1, 16, torch.bfloat16, 2)
    t, o, c = table.to(DEV), own.to(DEV), [x.to(DEV) for x in caches]
    p, L = torch.tensor([[1, 0]], device=DEV), torch.tensor([6], dtype=torch.int32, device=DEV)
    ok = dict(beam_table=t, own_table=o, parents=p, lengths=L, page_size=4, caches=c)
    kernels.reorder_beam_pages(**ok)
    for bad, err in ((dict(own_table=t), ValueError), (dict(beam_table=t[:1]), ValueError), (dict(parents=p[0]), ValueError), (dict(lengths=L.long()), ValueError),
                     (dict(page_size=8), ValueError), (dict(caches=[c[0], c[1].half()]), ValueError), (dict(caches=[c[0].cpu()]), RuntimeError),
                     (dict(caches=[c[0], c[1], c[0]]), ValueError),
                     (dict(scales=[torch.zeros(3, 1, device=DEV)]), ValueError), (dict(own_rows=p), ValueError)):
        with pytest.raises(err):
            kernels.reorder_beam_pages(**{**ok, **bad})
    with pytest.raises(NotImplementedError):
        kernels.reorder_beam_pages(torch.zeros(33, 3, dtype=torch.int32, device=DEV), torch.zeros(33, 3, dtype=torch.int32, device=DEV),
                                   torch.zeros(1, 33, dtype=torch.int64, device=DEV), L, 4, c)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
@pytest.mark.parametrize("P", [1, 8])
def test_beam_search_on_the_paged_cache(dtype, P):
    """Two requests of three beams for twenty steps over two layers: what each beam's attention reads is, bit for bit, the
    K / V rows of the tokens its own history chose."""
    B, W, H, g_, D, V, layers = 2, 3, 2, 2, 64, 50, 2
    gen = torch.Generator().manual_seed(P)
    prompt = [2 * P, 2 * P + P]          # whole pages, shared by the beams
    pt = PageTable(n_pages=200 * (1 if P > 1 else 4), page_size=P, max_batch_size=B * W + 1, device=DEV)
    pool = KVMemoryPool(device=DEV)
    cache = [PagedKVCache(pt, n_heads=H, head_dim=D, dtype=dtype, pool=pool) for _ in range(layers)]
    emb = torch.randn(layers, 2, V + 40, H, D, generator=gen).to(torch.bfloat16).to(DEV)      # token -> its K and V rows
    head = torch.randn(H * g_ * D, V, generator=gen).to(DEV)
    rows, history = [], [[] for _ in range(B * W)]
    for b in range(B):
        shared = pt.allocate_pages(prompt[b] // P)
        for w in range(W):
            row = pt.allocate()
            pt.map_pages(row, 0, shared)
            pt.reserve(row, prompt[b] + 24)
            rows.append(row)
            history[b * W + w] = [V + (t * 7 + b) % 40 for t in range(prompt[b])]
    pt.commit_block_table()
    own_rows = torch.tensor(rows, device=DEV)
    beam_table = pt.page_table[own_rows].contiguous()
    lengths = torch.tensor(prompt, dtype=torch.int32, device=DEV)

    def append(idx, toks, pos):
        slots = pt.build_slot_mapping(idx, pos)
        for i, layer in enumerate(cache):
            layer.update(pos, emb[i, 0][toks], emb[i, 1][toks], slot_mapping=slots)

    for b in range(B):
        append(own_rows[b * W:b * W + 1], torch.tensor([history[b * W]], device=DEV), torch.arange(prompt[b], device=DEV).view(1, -1))
    scores = torch.tensor([[0.0] + [-math.inf] * (W - 1)] * B, device=DEV)
    q = torch.randn(B * W, 1, H * g_, D, generator=gen).to(torch.bfloat16).to(DEV)
    for step in range(20):
        seq = lengths.repeat_interleave(W)
        outs = [paged_attention(q.transpose(1, 2), paged_kv_layer=layer, page_table=beam_table, paged_kv_seqlens_k=seq, scaling=D ** -0.5)
                for layer in cache]
        for r in range(B * W):       # what each beam reads against its own history
            n = len(history[r])
            pages = beam_table[r, :-(-n // P)].long()
            for i, layer in enumerate(cache):
                for kv, name in enumerate(("k", "v")):
                    rows_ = emb[i, kv][torch.tensor(history[r], device=DEV)]
                    codes = getattr(layer, name + "_cache")[pages].transpose(1, 2).reshape(-1, H, D)[:n]
                    if dtype == torch.int8:
                        scale = getattr(layer, name + "_block_scale")[pages]
                        for c in range(len(pages)):
                            for h in range(H):
                                code, s = O.quantize_block(rows_[c * P:(c + 1) * P, h].cpu())
                                assert float(scale[c, h]) == s
                                assert torch.equal(codes[c * P:c * P + code.shape[0], h].cpu(), code)
                    else:
                        assert torch.equal(codes, rows_)
        logits = sum(o.float().view(B * W, -1) for o in outs) @ head * 0.05
        want = S.select(S.candidates(logits.cpu(), scores.cpu()), W)
        r = kernels.beam_step_from_logits(logits, scores, W)
        assert torch.equal(r.tokens.cpu(), want[0]) and torch.equal(r.parents.cpu(), want[1])
        reorder_beams(cache, beam_table, pt.page_table, r.parents, lengths, own_rows=own_rows)
        parents, tokens = r.parents.cpu(), r.tokens.cpu()
        history = [history[b * W + int(parents[b, w])] + [int(tokens[b, w])] for b in range(B) for w in range(W)]
        append(own_rows, r.tokens.view(-1, 1), lengths.repeat_interleave(W).view(-1, 1).long())
        scores = r.scores
        lengths += 1
