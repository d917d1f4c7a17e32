"""Block-sparse attention over values whose scales are zero or tiny: constant vectors, zeroed rows, values near zero."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _query, _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,d,g", [(4, 128, 4), (4, 128, 8), (8, 128, 3), (8, 64, 8), (4, 64, 1), (8, 128, 5), (3, 64, 2)])
@pytest.mark.parametrize("kind", ["constant", "tiny", "zero rows", "constant first", "constant last", "constant tokens",
                                  "small"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_small_value_scales(cuda_device, bits, d, g, kind, dtype):
    import smallaios_b200 as sa

    b, h, past, s, k = 2, 2, 64 * 12 + 30, 2, 6
    total = past + s
    r, kc, km, vc, vm = _random(3, b, h, d, bits, total)
    at = {"constant first": slice(0, 64 * 6), "constant last": slice(64 * 6, None),
          "constant tokens": slice(5, None, 3)}.get(kind, slice(None))
    if kind == "zero rows":  # as a cache holds that was never written below its position
        at = slice(0, 64 * 4)
        for x in (kc, km, vc, vm):
            x[:, :, at] = 0
    elif kind == "tiny":
        vm[:, :, :, 0] = 1e-35
    elif kind == "small":
        vm[:] *= np.float32(1e-12)
    else:
        vm[:, :, at, 0] = 0.0
    cache = _cache(b, h, g, d, bits, total, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, s, h, g, d, dtype, cuda_device)
    ids = np.broadcast_to(np.array([0, 1, 3, 5, 8, 12], np.int32), (b, s, h, k))
    out = sa.gqa_sparse_attend(q, cache, 0, _device(ids, cuda_device), num_heads=h * g)
    kk, vv = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, kk, vv, ref.sparse_sees(ids, past, total))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound(dtype, q64, kk, vv, vc, vm, want), d)
    assert cache.device_status() == 0
    cache.close()


def test_all_values_zero(cuda_device):
    """Nothing but zeros behind the lists: zeros, not NaN."""
    import smallaios_b200 as sa

    for g in (2, 8):
        cache = _cache(1, 1, g, 128, 4, 64 * 9, cuda_device)
        cache.set_position(64 * 8)
        q = torch.randn(1, 1, g * 128, device=cuda_device)
        ids = torch.tensor([[[[0, 2, 8]]]], dtype=torch.int32, device=cuda_device)
        assert (sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=g) == 0).all()
        cache.close()
