"""Paged serving: numbers beyond 32 bits are refused, not cut to their low half."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_layers_and_sizes_beyond_32_bits(cuda_device):
    import smallaios_b200 as sa

    pool = sa.GpuKvPages(1, 1, 64, 4, device=cuda_device)
    x = torch.ones(1, 1, 64, device=cuda_device)
    table, lens = torch.zeros(1, 2, dtype=torch.int32, device=cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for layer in (2**32, -2**32, 2**31):
        with pytest.raises(sa.InvalidAttribute, match="layer_idx"):
            pool.append(layer, x, x, table, lens)
        with pytest.raises(sa.InvalidAttribute, match="layer_idx"):
            sa.gqa_paged_attend(x, pool, layer, table, lens, num_heads=1)
        with pytest.raises(sa.InvalidAttribute, match="layer_idx"):
            pool.view(layer)
    assert not pool.view(0).k_meta.any()
    for kw in (dict(num_pages=2**32 + 4), dict(num_layers=2**32 + 1), dict(head_dim=2**32 + 64), dict(bits=2**32 + 4),
               dict(num_heads=2**32 + 1), dict(kv_head_begin=2**32), dict(kv_head_count=2**32 + 1), dict(num_kv_heads=2**32 + 1)):
        with pytest.raises(sa.InvalidAttribute, match=next(iter(kw))):
            sa.GpuKvPages(**{**dict(num_layers=1, num_kv_heads=1, head_dim=64, num_pages=4), **kw}, device=cuda_device)


def test_shapes_beyond_32_bits(cuda_device):
    """Rows of 2^32 and more pages or groups, of memory that is never written (17 GB)."""
    import smallaios_b200 as sa

    pool = sa.GpuKvPages(1, 1, 64, 4, device=cuda_device)
    x = torch.ones(1, 1, 64, device=cuda_device)
    lens = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    wide = torch.empty(2**32 + 4, dtype=torch.int32, device=cuda_device)
    with pytest.raises(sa.ShapeMismatch, match="pages"):
        pool.append(0, x, x, wide[None], lens)
    with pytest.raises(sa.ShapeMismatch, match="pages"):
        sa.gqa_paged_attend(x, pool, 0, wide[None], lens, num_heads=1)
    with pytest.raises(sa.InvalidAttribute, match="beams"):
        pool.reorder_beams(wide[:, None], wide, wide[None])
    with pytest.raises(sa.InvalidAttribute, match="groups"):
        pool.reorder_beams(wide[:, None], wide, wide[:, None])
    scores = wide.view(torch.float32)
    with pytest.raises(sa.InvalidAttribute, match="beams"):
        sa.beam_select(scores[:, None], scores[None], keep=4)
    with pytest.raises(sa.InvalidAttribute, match="groups"):
        sa.beam_select(scores[:, None], scores[:, None])
    del wide, scores
    torch.cuda.empty_cache()
