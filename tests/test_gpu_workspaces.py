"""Whose workspace a serving call uses: the caller's where the size is not 0, else the cache's own."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _lists, _query, _random, _trees

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64), (3, 128), (3, 64), (4, 16), (4, 32), (8, 256)])
def test_sizes(cuda_device, bits, d):
    from smallaios_b200 import _lib

    cache = _cache(2, 2, 4, d, bits, 300, cuda_device)
    own = bits == 3 or d not in (64, 128)
    for code in (_lib.SA_DTYPE_FLOAT, _lib.SA_DTYPE_FLOAT16, _lib.SA_DTYPE_BFLOAT16):
        assert (_lib.lib.sa_gqa_tree_workspace_bytes(cache.handle, 8, code) == 0) == own
    assert _lib.lib.sa_gqa_sparse_workspace_bytes(cache.handle, 1) == 0
    assert (_lib.lib.sa_gqa_sparse_workspace_bytes(cache.handle, 2) == 0) == own
    cache.close()


def test_calls_with_workspaces_of_their_own_may_overlap(cuda_device):
    """One cache, three streams: a tree, block lists of several tokens, and a dense chunk on the cache's workspace."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 4, 4, 4, 128, 4, 64 * 40, 8
    r, kc, km, vc, vm = _random(2, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, "bf16", cuda_device)
    parents, ids = _device(_trees(r, b, n), cuda_device), _device(_lists(r, b, n, h, 9, past), cuda_device)
    calls = [lambda s=None: sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g, stream=s),
             lambda s=None: sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g, stream=s),
             lambda s=None: sa.gqa_attend(q, cache, 0, num_heads=h * g, do_rotary=False, stream=s)]
    want = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                torch.cuda._sleep(500_000)
                got.append(c(s))
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    cache.close()
