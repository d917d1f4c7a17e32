"""The beams' page tables: tables and results that lie between each other's rows, other streams, captured steps, and
pages behind 32-bit offsets."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pool(device, layers=1, h=1, d=64, pages=64, bits=8):
    import smallaios_b200 as sa

    return sa.GpuKvPages(layers, h, d, pages, bits=bits, device=device)


def _case(device, width=3):
    """Two groups of four beams, 70 tokens each, one beam of each continued twice."""
    table = torch.arange(8 * width, dtype=torch.int32, device=device).view(8, width)
    lens = torch.full((8,), 70, dtype=torch.int32, device=device)
    parents = torch.tensor([[0, 0, 2, 3], [1, 1, 1, 3]], dtype=torch.int32, device=device)
    return table, lens, parents


def test_column_slices_of_one_tensor_do_not_overlap(cuda_device):
    import smallaios_b200 as sa

    table, lens, parents = _case(cuda_device)
    want = _pool(cuda_device).reorder_beams(table, lens, parents)
    for old, new, width in ((0, 3, 6), (3, 0, 6), (1, 5, 8), (4, 1, 7)):
        wide = torch.full((8, width), -9, dtype=torch.int32, device=cuda_device)
        wide[:, old:old + 3] = table
        pool = _pool(cuda_device)
        out = wide[:, new:new + 3]
        assert pool.reorder_beams(wide[:, old:old + 3], lens, parents, out=out) is out
        assert torch.equal(out, want) and torch.equal(wide[:, old:old + 3], table)
        rest = [i for i in range(width) if not (old <= i < old + 3 or new <= i < new + 3)]
        assert (wide[:, rest] == -9).all() and pool.device_status() == 0
    # halves of one tensor by rows, and tables that share a column or an element
    both = torch.zeros(16, 3, dtype=torch.int32, device=cuda_device)
    both[8:] = table
    assert torch.equal(_pool(cuda_device).reorder_beams(both[8:], lens, parents, out=both[:8]), want)
    wide = torch.zeros(9, 8, dtype=torch.int32, device=cuda_device)
    for old, new in ((wide[:8, :3], wide[:8, 2:5]), (wide[:8, 2:5], wide[:8, :3]), (wide[:8, 5:], wide[:8, 5:]),
                     (wide[:8, :3], wide[1:, :3]), (wide[1:, 2:5], wide[:8, :3]),
                     (wide.view(-1)[:24].view(8, 3), wide.view(-1)[23:47].view(8, 3))):
        with pytest.raises(sa.InvalidAttribute, match="overlaps"):
            _pool(cuda_device).reorder_beams(old, lens, parents, out=new)
