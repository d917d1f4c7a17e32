"""Draft-tree attention over values whose scales are zero or tiny: constant vectors, zeroed rows, values near zero."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _query, _random, _trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,d,g", [(4, 128, 4), (8, 64, 8), (8, 128, 1), (3, 64, 2)])
@pytest.mark.parametrize("kind", ["constant", "tiny", "zero rows", "constant tokens", "small"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_small_value_scales(cuda_device, bits, d, g, kind, dtype):
    import smallaios_b200 as sa

    b, h, past, n = 2, 2, 600, 9
    total = past + n
    r, kc, km, vc, vm = _random(3, b, h, d, bits, total)
    if kind == "zero rows":
        for x in (kc, km, vc, vm):
            x[:, :, :400] = 0
    elif kind == "tiny":
        vm[:, :, :, 0] = 1e-35
    elif kind == "small":
        vm[:] *= np.float32(1e-12 if dtype != "f16" else 1e-2)
    else:
        vm[:, :, slice(5, None, 3) if kind == "constant tokens" else slice(None), 0] = 0.0
    cache = _cache(b, h, g, d, bits, total, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, dtype, cuda_device)
    parents = _trees(r, b, n)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, k, v, np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound(dtype, q64, k, v, vc, vm, want), d)
    cache.close()


@pytest.mark.parametrize("bits", [4, 8])
def test_constant_values_over_a_long_context(cuda_device, bits):
    """300,000 tokens whose value vectors are all the same constant: that vector, not an overflow of the sums."""
    import smallaios_b200 as sa

    d, g, past, n = 64, 2, 300_000, 3
    cache = _cache(1, 1, g, d, bits, past + n, cuda_device)
    view = cache.view(0)
    torch.manual_seed(0)
    view.k_codes.random_(0, 256)
    view.v_codes.random_(0, 256)
    view.k_meta[..., 0], view.k_meta[..., 1] = 2.0 ** -bits, -0.5
    view.v_meta[..., 0], view.v_meta[..., 1] = 0.0, 500.0
    cache.set_position(past)
    q = torch.randn(1, n, g * d, device=cuda_device)
    parents = torch.tensor([[-1, 0, 0]], dtype=torch.int32, device=cuda_device)
    out = sa.gqa_tree_attend(q, cache, 0, parents, num_heads=g).double().cpu().numpy().reshape(n, g, d)
    signs = view.signs.double().cpu().numpy()
    want = ref.walsh(np.full((1, d), 500.0)) * signs / np.sqrt(d)
    # one vector of norm 500 sqrt(d), so the weights' errors cancel but for their sum's: 2^-20 of it
    assert np.abs(out - want).max() < 2.0 ** -20 * 500 * d ** 0.5 * 8
    cache.close()
