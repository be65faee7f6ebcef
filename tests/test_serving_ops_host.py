"""The int8, ragged-step and beam-search entry points without a GPU: CPU tensors are refused, and the oracles do what they say."""

import math

import pytest
import torch

from kestrel_b200 import DevicePageTable, KVMemoryPool, PagedKVCache, PageTable, get_runtime, kernels, reorder_beams
from oracle import beam_oracle as S
from oracle import block_int8_oracle as O


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 1, 16)
    pool = torch.zeros(3, 1, 4, 16, dtype=torch.int8).permute(0, 2, 1, 3)
    scale = torch.zeros(3, 1)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 3, dtype=torch.int32)
    for call in (lambda: kernels.reshape_and_cache_block_int8(x, x, pool, pool, scale, scale, torch.zeros(2, dtype=torch.int64)),
                 lambda: kernels.build_ragged_step(table, i32, i32, i32, i32, i32, 4, n_pages=3, n_tokens=1, out_page_table=table),
                 lambda: kernels.release_rows(table, i32, i32, i32, i32, 4),
                 lambda: kernels.beam_step_from_logits(torch.zeros(2, 5), torch.zeros(1, 2), 2),
                 lambda: kernels.reorder_beam_pages(table, table.clone(), torch.zeros(1, 2, dtype=torch.int64), i32[:1], 4, [])):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="at least one layer"):
        reorder_beams([None], table, table, i32, i32)


def test_runtime_offers_the_operators():
    rt = get_runtime()
    assert rt.cache.reshape_and_cache_block_int8 is kernels.reshape_and_cache_block_int8
    assert rt.cache.build_ragged_step is kernels.build_ragged_step and rt.cache.release_rows is kernels.release_rows
    assert rt.cache.reorder_beam_pages is kernels.reorder_beam_pages
    assert rt.sampling.beam_step_from_logits is kernels.beam_step_from_logits


def test_int8_layers_and_device_tables_on_the_host():
    pt = PageTable(n_pages=4, page_size=4, max_batch_size=2, device="cpu")
    pool = KVMemoryPool(device="cpu")
    layer = PagedKVCache(pt, n_heads=2, head_dim=16, dtype=torch.int8, pool=pool)
    assert layer.k_cache.dtype == torch.int8 and layer.k_block_scale.shape == (4, 2) and layer.block_scaled and not layer.quantized
    with pytest.raises(ValueError, match="scale per block"):
        PagedKVCache(pt, n_heads=2, head_dim=16, dtype=torch.int8, pool=pool, k_scale=1.0)
    dt = DevicePageTable(5, 4, 3, "cpu", pages_per_row=2)
    assert dt.free_pages[:int(dt.free_count)].tolist() == PageTable(n_pages=5, page_size=4, max_batch_size=3, device="cpu").free_pages
    assert dt.page_table.tolist() == [[0, 0], [-1, -1], [-1, -1]]
    for bad in ((0, 4, 3), (5, 0, 3), (5, 4, 0)):
        with pytest.raises(ValueError):
            DevicePageTable(*bad, "cpu")
    with pytest.raises(ValueError):
        DevicePageTable(5, 4, 3, "cpu", pages_per_row=0)


@pytest.mark.parametrize("amax,scale", [(0.0, 0.0), (64.0, 1.0), (127.99, 1.0), (128.0, 2.0), (1.0, 2.0 ** -6), (1e-45, 2.0 ** -126)])
def test_block_scale(amax, scale):
    assert O.block_scale(amax) == scale


def test_quantised_values_are_within_half_a_step_and_coding_again_is_a_shift():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(32, 16, generator=g)
    code, s = O.quantize_block(x)
    assert float(((code.double() + 0.5) * s - x.double()).abs().max()) <= s / 2
    y = torch.cat([x, torch.full((1, 16), 50.0)])
    code2, s2 = O.quantize_block(y)
    assert torch.equal(code2[:32], code >> round(math.log2(s2 / s)))


def test_beam_candidates():
    cand = S.candidates(torch.tensor([[0.0, 0.0], [1.0, -math.inf]]), torch.tensor([[0.0, -1.0]]))
    tokens, parents, value = S.select(cand, 4)
    assert tokens.tolist() == [[0, 1, 0, 1]] and parents.tolist() == [[0, 0, 1, 1]]
    assert torch.allclose(value, torch.tensor([[math.log(0.5), math.log(0.5), -1.0, -math.inf]], dtype=torch.float64))
