"""Buffers of the serving operators: outputs in place of the queries, and tensors that start at any element."""
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _lists, _query, _random, _trees

pytestmark = pytest.mark.gpu


def _shifted(t):
    """A contiguous copy of `t` that starts one element past an aligned address."""
    buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    view = buf[1:].view(t.shape)
    view.copy_(t)
    assert view.is_contiguous() and view.data_ptr() % 16 == t.element_size()
    return view


@pytest.mark.parametrize("bits,d,g,b,s", [(4, 128, 4, 2, 6), (8, 64, 8, 3, 1), (4, 128, 8, 2, 1), (4, 64, 1, 600, 2),
                                          (3, 64, 4, 2, 5), (4, 256, 2, 1, 3), (8, 32, 5, 2, 4)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_in_place_and_unaligned(cuda_device, bits, d, g, b, s, dtype):
    import smallaios_b200 as sa

    h, past, n = 2, 64 * 3 + 9, s
    r, kc, km, vc, vm = _random(6, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, dtype, cuda_device)
    parents, ids = _device(_trees(r, b, n), cuda_device), _device(_lists(r, b, n, h, 3, past), cuda_device)
    means = sa.kv_block_means(cache, 0, 0, past // 64)
    calls = {
        "tree": (lambda q, ints, **kw: sa.gqa_tree_attend(q, cache, 0, ints, num_heads=h * g, **kw), parents),
        "sparse": (lambda q, ints, **kw: sa.gqa_sparse_attend(q, cache, 0, ints, num_heads=h * g, **kw), ids),
    }
    for name, (call, ints) in calls.items():
        want = call(q, ints)
        x = q.clone()
        assert call(x, ints, out=x) is x and torch.equal(x, want), name
        out = _shifted(torch.zeros_like(q))
        assert torch.equal(call(_shifted(q), _shifted(ints), out=out), want), name
    sel = lambda q, **kw: sa.gqa_select_blocks(q, cache, 0, means, num_heads=h * g, max_blocks=3, **kw)  # noqa: E731
    want = sel(q)
    assert torch.equal(sel(_shifted(q), out=_shifted(torch.zeros_like(want))), want)
    with pytest.raises(sa.UnsupportedOp, match="aligned"):
        sa.gqa_select_blocks(q, cache, 0, _shifted(means), num_heads=h * g, max_blocks=3)
    with pytest.raises(sa.UnsupportedOp, match="aligned"):
        sa.kv_block_means(cache, 0, 0, past // 64, out=_shifted(means))
    cache.close()
