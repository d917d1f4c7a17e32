"""Rows of a draft tree are independent: a finite query of any size in one node, or in a slot that holds no node,
leaves the other rows as they are."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _query, _random

pytestmark = pytest.mark.gpu

PARENTS = np.array([[-1, 0, 1, -2, 2, -1, 0, 5, 6, 3]], np.int32)  # slots 3 and 9 hold no node


@pytest.mark.parametrize("bits,d,g", [(4, 128, 4), (8, 64, 8), (8, 128, 1), (4, 64, 7), (3, 64, 4)])
@pytest.mark.parametrize("dtype,big", [("f32", 1e30), ("f32", 1e6), ("f32", -3e37), ("bf16", 1e30), ("bf16", 3e38),
                                       ("f16", 65504.0), ("f32", 1e-30)])
@pytest.mark.parametrize("at", [3, 5])
def test_other_rows_keep_their_values(cuda_device, bits, d, g, dtype, big, at):
    """The other rows' bound is that of their own queries; what a slot without a node holds does not change a bit."""
    import smallaios_b200 as sa

    b, h, past, n = 1, 2, 300, 10
    r, kc, km, vc, vm = _random(10, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, dtype, cuda_device)
    others = [j for j in range(n) if j not in (3, 9, at)]
    outs = []
    for value in (0.0, big):
        q[0, at] = value
        q[0, at, 1::2] = -value / 2
        outs.append(sa.gqa_tree_attend(q, cache, 0, _device(PARENTS, cuda_device), num_heads=h * g))
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = np.repeat(ref.tree_sees(PARENTS, past)[:, :, None], h, axis=2)
    want = ref.attend(q64[:, others], k, v, sees[:, others])
    bound = ref.row_bound(dtype, q64[:, others], k, v, vc, vm, want)
    for out in outs:
        ref.assert_rows(out.double().cpu().numpy()[:, others], want, bound, d)
    if at == 3:
        assert torch.equal(*outs)
    assert (outs[1][0, [3, 9]] == 0).all()
    cache.close()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_heads_of_different_size(cuda_device, dtype):
    """Heads whose queries differ by a factor of 2^24 in size, each against its own bound."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 1, 1, 4, 128, 4, 400, 12
    r, kc, km, vc, vm = _random(12, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, dtype, cuda_device)
    q.view(b, n, g, d)[:] *= torch.tensor([1.0, 2.0 ** -20, 2.0 ** 4, 2.0 ** -4], device=cuda_device, dtype=q.dtype)[:, None]
    q64 = q.double().cpu().numpy().reshape(b, n, h, g, d)
    parents = np.arange(-1, n - 1, dtype=np.int32)[None]
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g).double().cpu().numpy()
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2)
    want = ref.attend(q64, k, v, sees)
    got, want = out.reshape(b, n, g, d), want.reshape(b, n, g, d)
    for e in range(g):
        bound = ref.row_bound(dtype, q64[:, :, :, e:e + 1], k, v, vc, vm, want[:, :, e])
        ref.assert_rows(got[:, :, e], want[:, :, e], bound, d)
    cache.close()
