"""The tables of a ragged step built on the GPU, against the host page table: whole numbers, compared exactly."""

import pytest
import torch

from kestrel_b200 import DevicePageTable, KVMemoryPool, PagedKVCache, PageTable, _native, kernels
from oracle import block_int8_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _clear_status():
    _native.device_status(0, clear=True)


def _int(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def _out_table(pt, B, fill=-7):
    return torch.full((B, pt.page_table.shape[1]), fill, dtype=torch.int32, device=DEV)


def _check_step(r, host, rows, lengths, new, P, n_tokens, cols):
    """Against the host table after the same reservations."""
    total = sum(new)
    assert r.seqused_k.tolist() == [n + m for n, m in zip(lengths, new)]
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    assert r.cu_seqlens_q.tolist() == cu
    slots, pos = [], []
    for row, n, m in zip(rows, lengths, new):
        pages = host[row]
        for t in range(n, n + m):
            slots.append(pages[t // P] * P + t % P)
            pos.append(t)
    assert r.slot_mapping.tolist() == slots + [-1] * (n_tokens - total)
    assert r.positions.tolist() == pos + [0] * (n_tokens - total)
    table = r.page_table.cpu()
    for i, (row, n, m) in enumerate(zip(rows, lengths, new)):
        want = -(-(n + m) // P)
        assert table[i, :want].tolist() == host[row][:want]
        assert bool((table[i, want:] == -7).all())


@pytest.mark.parametrize("P", [1, 3, 16, 128])
@pytest.mark.parametrize("B", [1, 2, 33, 300, 1500])
@pytest.mark.parametrize("idx", [torch.int32, torch.int64])
def test_steps_like_the_host_table(P, B, idx):
    """Several steps of decode rows, idle rows and prompt chunks, then rows leave and others come: pages are handed out in
    the host's order, the free lists end up the same."""
    g = torch.Generator().manual_seed(P * 1000 + B)
    n_pages = 3 + 4 * B * (1 + 60 // P)
    host = PageTable(n_pages=n_pages, page_size=P, max_batch_size=B + 1, device="cpu")
    pt = DevicePageTable(n_pages, P, B + 1, DEV, pages_per_row=2 + 260 // P)
    rows = [host.allocate() for _ in range(B)]
    order = torch.randperm(B, generator=g).tolist()
    rows = [rows[i] for i in order]
    lengths = [0] * B
    for step in range(4):
        new = torch.randint(0, 61 if step == 0 else 3, (B,), generator=g).tolist()
        for row, n, m in zip(rows, lengths, new):
            host.reserve(row, n + m)
        n_tokens = sum(new) + (5 if step % 2 else 0)
        out = _out_table(pt, B)
        r = pt.step(_int(rows, idx), _int(lengths), _int(new), n_tokens, out_page_table=out)
        _check_step(r, host.page_table_cpu, rows, lengths, new, P, n_tokens, pt.page_table.shape[1])
        assert int(r.pages_taken) == sum(-(-(n + m) // P) - -(-n // P) for n, m in zip(lengths, new))
        lengths = [n + m for n, m in zip(lengths, new)]
        assert int(pt.free_count) == len(host.free_pages) and pt.free_pages[:int(pt.free_count)].tolist() == host.free_pages
        for row, n in zip(rows, lengths):
            c = -(-n // P)
            assert pt.page_table[row, :c].tolist() == host.page_table_cpu[row][:c]
        if B > 2:   # a third of the rows leaves, some with a cached prefix that stays allocated
            gone = list(range(step, B, 3))
            keep = [min(i % 3, -(-lengths[i] // P)) for i in gone]
            pt.release(_int([rows[i] for i in gone], idx), _int([lengths[i] for i in gone]), _int(keep))
            for i, k in zip(gone, keep):
                host.erase(rows[i], k)
                lengths[i] = 0
            for i in reversed(gone):
                assert host.allocate() == rows[i]
            assert pt.free_pages[:int(pt.free_count)].tolist() == host.free_pages
            for i, k in zip(gone, keep):
                assert bool((pt.page_table[rows[i], k:] == -1).all())


def test_padding_rows_and_empty_batches():
    """Entries of row 0 get page 0 and take nothing; a batch without entries, a step without tokens."""
    pt = DevicePageTable(20, 4, 4, DEV)
    out = _out_table(pt, 4)
    r = pt.step(_int([2, 0, 0, 1]), _int([0, 0, 3, 0]), _int([5, 1, 1, 2]), 12, out_page_table=out)
    # (the free list ends in 3, 2, 1: two pages are its last two, in the list's order)
    assert r.slot_mapping.tolist() == [4 * 2, 4 * 2 + 1, 4 * 2 + 2, 4 * 2 + 3, 4 * 1] + [0, 3] + [4 * 3, 4 * 3 + 1] + [-1] * 3
    assert int(r.pages_taken) == 3 and int(pt.free_count) == 16
    assert out[1, :1].tolist() == [0] and out[2, :1].tolist() == [0]
    empty = pt.step(_int([]), _int([]), _int([]), 3, out_page_table=out)
    assert empty.cu_seqlens_q.tolist() == [0] and empty.slot_mapping.tolist() == [-1] * 3 and int(empty.pages_taken) == 0
    none = pt.step(_int([1]), _int([2]), _int([0]), 0, out_page_table=out)
    assert none.seqused_k.tolist() == [2] and none.slot_mapping.numel() == 0 and int(pt.free_count) == 16


@pytest.mark.parametrize("why", ["pages", "tokens"])
def test_a_step_that_does_not_fit_takes_nothing(why):
    _clear_status()
    pt = DevicePageTable(6, 4, 4, DEV)
    before = pt.page_table.clone()
    out = _out_table(pt, 2)
    r = pt.step(_int([1, 2]), _int([0, 0]), _int([12, 12] if why == "pages" else [4, 4]), 30 if why == "pages" else 7, out_page_table=out)
    assert int(r.pages_taken) == -1 and r.seqused_k.tolist() == [0, 0] and r.cu_seqlens_q.tolist() == [0, 0, 0]
    assert bool((r.slot_mapping == -1).all()) and torch.equal(pt.page_table, before) and int(pt.free_count) == 5
    assert _native.device_status(0)[0] == _native.STATUS_NO_PAGES
    r = pt.step(_int([1, 2]), _int([0, 0]), _int([12, 8]), 30, out_page_table=out)      # exactly what is there
    assert int(r.pages_taken) == 5 and int(pt.free_count) == 0


def test_entries_out_of_range_get_nothing():
    _clear_status()
    pt = DevicePageTable(40, 4, 4, DEV, pages_per_row=5)
    out = _out_table(pt, 6)
    r = pt.step(_int([1, 9, -1, 2, 3, 2 ** 31 - 1]), _int([0, 0, 0, 19, -4, 0]), _int([3, 3, 3, 2, 1, 1]), 20, out_page_table=out)
    assert r.seqused_k.tolist() == [3, 0, 0, 0, 0, 0] and r.cu_seqlens_q.tolist() == [0, 3, 3, 3, 3, 3, 3]
    assert int(r.pages_taken) == 1 and bool((out[1:] == -7).all())
    assert _native.device_status(0)[0] == _native.STATUS_BAD_ROW
    pt.release(_int([9, 1]), _int([4, 3]))
    assert int(pt.free_count) == 39 and _native.device_status(0)[0] == _native.STATUS_BAD_ROW
    # a table entry that is no page: the token has no slot
    pt.page_table[2, 0] = 40
    r = pt.step(_int([2]), _int([1]), _int([2]), 2, out_page_table=out)
    assert r.slot_mapping.tolist() == [-1, -1] and _native.device_status(0)[0] == _native.STATUS_BAD_PAGE
    # more pages than were ever handed out: nothing changes
    pt.release(_int([1, 2, 3]), _int([20, 20, 20]))
    assert int(pt.free_count) == 39 and _native.device_status(0)[0] == _native.STATUS_NO_PAGES


def test_a_captured_step_advances_its_own_state():
    """lengths and the free count written in place; two graphs over one table, replayed in turn."""
    P, B = 4, 3
    pt = DevicePageTable(60, P, B + 1, DEV)
    host = PageTable(n_pages=60, page_size=P, max_batch_size=B + 1, device="cpu")
    rows = [host.allocate() for _ in range(B)]
    idx, lengths, new = _int(rows), _int([0] * B), _int([1, 2, 0])
    out = [_out_table(pt, B) for _ in range(2)]
    outs = [dict(out_cu_seqlens_q=torch.empty(B + 1, dtype=torch.int32, device=DEV), out_slot_mapping=torch.empty(5, dtype=torch.int64, device=DEV),
                 out_positions=torch.empty(5, dtype=torch.int64, device=DEV), out_pages_taken=torch.empty(1, dtype=torch.int32, device=DEV))
            for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            pt.step(idx, lengths, new, 5, out_page_table=out[i], out_seqused_k=lengths, **outs[i])
        graphs.append(graph)
    held = [0] * B
    for step in range(9):
        adds = [[1, 2, 0], [2, 2, 1], [0, 0, 5]][step % 3]
        new.copy_(_int(adds))
        graphs[step % 2].replay()
        for row, n, m in zip(rows, held, adds):
            host.reserve(row, n + m)
        want = [host.page_table_cpu[row][t // P] * P + t % P for row, n, m in zip(rows, held, adds) for t in range(n, n + m)]
        held = [n + m for n, m in zip(held, adds)]
        assert lengths.tolist() == held
        assert outs[step % 2]["out_slot_mapping"].tolist() == want + [-1] * (5 - len(want))
        assert pt.free_pages[:int(pt.free_count)].tolist() == host.free_pages


def test_refusals():
    pt = DevicePageTable(10, 4, 4, DEV)
    out = _out_table(pt, 2)
    ok = dict(batch_idx=_int([1, 2]), lengths=_int([0, 0]), new_tokens=_int([1, 1]), n_tokens=4, out_page_table=out)
    pt.step(**ok)
    for bad in (dict(lengths=_int([0])), dict(new_tokens=_int([1, 1], torch.int64)), dict(batch_idx=_int([[1, 2]])),
                dict(n_tokens=-1), dict(out_page_table=out[:1]), dict(out_page_table=out.long()), dict(lengths=_int([0, 0, 0, 0])[::2]),
                dict(out_slot_mapping=torch.empty(3, dtype=torch.int64, device=DEV))):
        with pytest.raises(ValueError):
            pt.step(**{**ok, **bad})
    with pytest.raises(RuntimeError):
        pt.step(**{**ok, "lengths": torch.zeros(2, dtype=torch.int32)})
    many = torch.zeros(8193, dtype=torch.int32, device=DEV)
    with pytest.raises(NotImplementedError, match="8192"):
        pt.step(many, many, many, 0, out_page_table=_out_table(pt, 8193))


@pytest.mark.parametrize("dtype", [torch.int8, torch.bfloat16])
def test_ragged_serving_steps(dtype):
    """Tables, append and packed attention of mixed steps, int8 and 16-bit pools, captured once and replayed: each
    step's output against float64 attention over everything its requests have appended."""
    P, H, g_, D, B, n_tokens = 16, 2, 4, 64, 5, 48
    gen = torch.Generator().manual_seed(6)
    pt = DevicePageTable(120, P, B + 1, DEV)
    layer = PagedKVCache(pt, n_heads=H, head_dim=D, dtype=dtype, pool=KVMemoryPool(device=DEV))
    idx, lengths, new = _int([3, 1, 5, 2, 4]), _int([0] * B), _int([0] * B)
    table = torch.zeros(B, pt.page_table.shape[1], dtype=torch.int32, device=DEV)
    k, v = (torch.zeros(1, n_tokens, H, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    q = torch.zeros(n_tokens, H * g_, D, dtype=torch.bfloat16, device=DEV)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=DEV)
    slots, positions = (torch.empty(n_tokens, dtype=torch.int64, device=DEV) for _ in range(2))
    taken = torch.empty(1, dtype=torch.int32, device=DEV)
    out = torch.empty_like(q)
    scales = dict(k_block_scale=layer.k_block_scale, v_block_scale=layer.v_block_scale) if dtype == torch.int8 else {}

    def step():
        pt.step(idx, lengths, new, n_tokens, out_page_table=table, out_seqused_k=lengths, out_cu_seqlens_q=cu, out_slot_mapping=slots,
                out_positions=positions, out_pages_taken=taken)
        layer.update(positions.view(1, -1), k, v, slot_mapping=slots.view(1, -1))
        kernels.flash_attn_fwd(q, layer.k_cache.permute(0, 2, 1, 3), layer.v_cache.permute(0, 2, 1, 3), page_table=table, seqused_k=lengths,
                               cu_seqlens_q=cu, max_seqlen_q=n_tokens, causal=True, out=out, **scales)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()                      # (no tokens: sizes the scratch)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.synchronize()
    past = [[torch.zeros(0, H, D, dtype=torch.bfloat16) for _ in range(2)] for _ in range(B)]
    for adds in ([20, 1, 0, 17, 3], [1, 1, 1, 1, 1], [0, 40, 1, 1, 1], [1, 1, 1, 1, 0], [30, 1, 1, 1, 15]):
        n = sum(adds)
        fresh = [torch.randn(n, h, D, generator=gen).to(torch.bfloat16) for h in (H, H, H * g_)]
        k[0, :n], v[0, :n], q[:n] = (t.to(DEV) for t in fresh)
        new.copy_(_int(adds))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        at = 0
        for b, m in enumerate(adds):
            for i in range(2):
                past[b][i] = torch.cat([past[b][i], fresh[i][at:at + m]])
            L = past[b][0].shape[0]
            if m:
                pools = []
                for rows in past[b]:
                    if dtype == torch.int8:   # the pool's own values are exact: block by block
                        blocks = [[O.quantize_block(rows[c:c + P, h]) for h in range(H)] for c in range(0, L, P)]
                        rows = torch.cat([torch.stack([(c.double() + 0.5) * s for c, s in blk], 1) for blk in blocks])
                    pools.append(rows.double().repeat_interleave(g_, 1))
                x = fresh[2][at:at + m].double()
                z = torch.einsum("jhd,nhd->hjn", x, pools[0]) * D ** -0.5
                z = z.masked_fill(torch.arange(L).view(1, -1) > L - m + torch.arange(m).view(-1, 1), float("-inf"))
                p = torch.softmax(z, -1)
                want = torch.einsum("hjn,nhd->jhd", p, pools[1])
                weight = torch.einsum("hjn,nhd->jhd", p, pools[1].abs())
                got = out[at:at + m].cpu().double()
                # output and weights rounded to bf16 (2^-8 each), fp32 terms below 2^-12 at these sizes
                assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -11) * weight + 1e-6).all()), (adds, b)
            at += m
        assert bool((out[n:] == 9.0).all())       # rows behind the last sequence stay as they were
