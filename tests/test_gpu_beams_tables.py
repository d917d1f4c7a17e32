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


def test_scores_and_marks_of_other_strides_are_refused(cuda_device):
    import smallaios_b200 as sa

    x, wide = torch.zeros(8, 50, device=cuda_device), torch.zeros(2, 8, device=cuda_device)
    for scores in (wide[:, :4], wide[:, ::2], torch.zeros(4, 2, device=cuda_device).t()):
        with pytest.raises(ValueError, match="scores"):
            sa.beam_select(x, scores)
    with pytest.raises(ValueError, match="finished"):
        sa.beam_select(x, torch.zeros(2, 4, device=cuda_device), finished=wide.bool()[:, :4])


@pytest.mark.parametrize("handles", [False, True])
def test_appending_and_reordering_on_another_stream(cuda_device, handles):
    """The stream's own order holds: inputs written there just before, and a result allocated for it, while the current
    stream takes and gives back memory."""
    import smallaios_b200 as sa

    table, lens, parents = _case(cuda_device)
    k, v = (torch.randn(8, 70, 64, device=cuda_device) for _ in range(2))
    zero = torch.zeros_like(lens)
    want_pool = _pool(cuda_device)
    want_pool.append(0, k, v, table, zero)
    want = want_pool.reorder_beams(table, lens, parents)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    stream = s.cuda_stream if handles else s
    for _ in range(4):
        pool = _pool(cuda_device)
        sk, sv, st, sp = (torch.zeros_like(x) for x in (k, v, table, parents))
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
            for dst, src in ((sk, k), (sv, v), (st, table), (sp, parents)):
                dst.copy_(src)
        pool.append(0, sk, sv, st, zero, stream=stream)
        got = pool.reorder_beams(st, lens, sp, stream=stream)
        for _ in range(8):
            torch.full(table.shape, -1, dtype=torch.int32, device=cuda_device)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and pool.device_status() == 0
        for name in ("k_codes", "v_codes", "k_meta", "v_meta"):
            assert torch.equal(getattr(pool.view(0), name), getattr(want_pool.view(0), name))


def test_a_captured_reordering_replays_with_new_parents(cuda_device):
    """Append, selection's place taken by given parents, and reordering, captured once; the table goes back and forth
    between two buffers."""
    import smallaios_b200 as sa

    r = np.random.default_rng(3)
    steps, b, k, layers, h, d = 24, 2, 4, 2, 2, 64
    keys = [torch.randn(b * k, 1, h * d, device=cuda_device) for _ in range(steps)]
    choices = [torch.from_numpy(r.integers(-1, k, (b, k)).astype(np.int32)).to(cuda_device) for _ in range(steps)]
    pools = [_pool(cuda_device, layers, h, d, b * k * 3, 4) for _ in range(2)]
    first = torch.from_numpy(r.permutation(b * k * 3).astype(np.int32).reshape(b * k, 3)).to(cuda_device)
    start = torch.full((b * k,), 55, dtype=torch.int32, device=cuda_device)
    prompt = torch.randn(b * k, 55, h * d, device=cuda_device)
    for pool in pools:
        for i in range(layers):
            pool.append(i, prompt, prompt, first, torch.zeros_like(start))

    def step(pool, x, table, new, lens, parents):
        for i in range(layers):
            pool.append(i, x, x * (i + 1), table, lens)
        lens.add_(1)
        pool.reorder_beams(table, lens, parents, out=new)

    # step by step
    table, lens = first.clone(), start.clone()
    for x, p in zip(keys, choices):
        new = torch.empty_like(table)
        step(pools[0], x, table, new, lens, p)
        table = new
    # two steps captured, replayed
    x, p, lens2 = [keys[0].clone() for _ in range(2)], [choices[0].clone() for _ in range(2)], start.clone()
    tables = [first.clone(), torch.empty_like(first)]
    held = [[t.clone() for t in (v.k_codes, v.v_codes, v.k_meta, v.v_meta)] for v in map(pools[1].view, range(layers))]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):  # what a first call sets up is not part of the graph
        step(pools[1], x[0], tables[0], tables[1], lens2, p[0])
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for i in range(2):
            step(pools[1], x[i], tables[i], tables[1 - i], lens2, p[i])
    tables[0].copy_(first)
    lens2.copy_(start)
    for i, arrays in enumerate(held):
        v = pools[1].view(i)
        for dst, src in zip((v.k_codes, v.v_codes, v.k_meta, v.v_meta), arrays):
            dst.copy_(src)
    for at in range(0, steps, 2):
        for i in range(2):
            x[i].copy_(keys[at + i])
            p[i].copy_(choices[at + i])
        graph.replay()
    assert torch.equal(tables[0], table) and torch.equal(lens2, lens)
    assert [pool.device_status() for pool in pools] == [0, 0]
    for i in range(layers):
        a, e = pools[1].view(i), pools[0].view(i)
        for name in ("k_codes", "v_codes", "k_meta", "v_meta"):
            assert torch.equal(getattr(a, name), getattr(e, name))


def test_copies_between_pages_behind_32_bit_offsets(cuda_device):
    """The second layer of a pool of more than 4 GB a layer, pages from both ends."""
    import smallaios_b200 as sa

    h, d, pages, k = 4, 128, 64000, 3  # 18432 bytes a head and page: 4.7 GB a layer
    lens = torch.full((k,), 100, dtype=torch.int32, device=cuda_device)
    parents = torch.tensor([[1, 1, 1]], dtype=torch.int32, device=cuda_device)
    x = torch.randn(k, 100, h * d, device=cuda_device)
    got = []
    for n, ids in ((pages, [63999, 7, 31000, 63998, 0, 63997]), (6, [5, 1, 2, 4, 0, 3])):
        pool = _pool(cuda_device, 2, h, d, n, 8)
        table = torch.tensor(ids, dtype=torch.int32, device=cuda_device).view(k, 2)
        for layer in range(2):
            pool.append(layer, x + layer, x - layer, table, torch.zeros_like(lens))
        new = pool.reorder_beams(table, lens, parents)
        assert pool.device_status() == 0
        assert new.flatten().tolist() == [ids[2], ids[1], ids[2], ids[3], ids[2], ids[5]]
        views = [pool.view(layer) for layer in range(2)]
        got.append([getattr(v, name)[new.long()] for v in views for name in ("k_codes", "v_codes", "k_meta", "v_meta")])
        pool.close()
    for a, e in zip(*got):
        assert torch.equal(a, e)
    for a in got[0]:  # 36 rows of the page in use: two blocks of V and 4 tokens of the third
        rows = a[:, 1, :, :36] if a.shape[3] == 64 else a[:, 1, :, :2]
        assert torch.equal(rows[0], rows[1]) and torch.equal(rows[0], rows[2])
