"""Layer views are zero-copy: while a tensor of one lives, so does the cache's memory."""
import gc
import weakref

import pytest

pytestmark = pytest.mark.gpu


def test_views_keep_the_cache_alive(cuda_device):
    import smallaios_b200 as sa

    cache = sa.GpuKvCache(1, 2, 64, 64, batch=1, bits=4, device=cuda_device)
    seen = weakref.ref(cache)
    codes = cache.view(0).k_codes
    del cache
    gc.collect()
    assert seen() is not None and seen().handle  # not freed: `codes` still points into it
    assert int(codes.sum()) == 0
    del codes
    gc.collect()
    assert seen() is None
