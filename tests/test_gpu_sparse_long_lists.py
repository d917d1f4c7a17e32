"""Block lists longer than 32-bit token counts reach are refused; long ones that are almost empty are read."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _query, _random

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,d", [(4, 128), (3, 64)])
def test_lists_past_the_limit_are_refused(cuda_device, bits, d):
    import smallaios_b200 as sa

    cache = _cache(1, 1, 1, d, bits, 64, cuda_device)
    q = torch.zeros(1, 1, d, device=cuda_device)
    ids = torch.full((1, 1, 1, 1 << 25), -1, dtype=torch.int32, device=cuda_device)
    with pytest.raises(sa.UnsupportedOp, match="at most"):
        sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=1)
    cache.close()


@pytest.mark.parametrize("bits,d,g", [(4, 128, 2), (8, 64, 8), (3, 64, 1)])
def test_a_long_list_of_few_blocks(cuda_device, bits, d, g):
    import smallaios_b200 as sa

    past, k = 64 * 7 + 3, 20_000
    r, kc, km, vc, vm = _random(4, 1, 1, d, bits, past + 1)
    cache = _cache(1, 1, g, d, bits, past + 1, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, 1, 1, 1, g, d, "f32", cuda_device)
    ids = np.full((1, 1, 1, k), -1, np.int32)
    ids[..., 17], ids[..., 9_001], ids[..., k - 1] = 2, 7, 5
    out = sa.gqa_sparse_attend(q, cache, 0, _device(ids, cuda_device), num_heads=g)
    kk, vv = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, kk, vv, ref.sparse_sees(ids, past, past + 1))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound("f32", q64, kk, vv, vc, vm, want), d)
    cache.close()
