"""A decoder layer over pages against the one over the contiguous cache."""
import numpy as np
import pytest
import torch

from tests.test_gpu_serving_layer import BITS, D, HKV, HQ, _near, _rows, _tables, _weights

pytestmark = pytest.mark.gpu


def test_paged_layer_is_the_contiguous_layer(cuda_device):
    """Rows of different lengths, each against a cache of one sequence.  The paged step rounds q once less (its rotation
    stays in 32 bits; 2^-9 of scores of a few units move them by about 1%), so 2e-2."""
    import smallaios_b200 as sa

    r = np.random.default_rng(1)
    w = _weights(r, cuda_device)
    lens = [0, 63, 64, 130]
    b = len(lens)
    cos, sin = _tables(max(lens) + 4, cuda_device)
    rope = dict(cos_cache=cos, sin_cache=sin)
    prompts = [_rows(r, max(n, 1), cuda_device) for n in lens]
    caches, pool = [], sa.GpuKvPages(1, HKV, D, 16, num_heads=HQ, bits=BITS, device=cuda_device)
    table = torch.full((b + 1, 3), -1, dtype=torch.int32, device=cuda_device)  # the last row takes no part
    table[:b] = torch.randperm(16, device=cuda_device)[:b * 3].view(b, 3)
    view = pool.view(0)
    for i, n in enumerate(lens):
        cache = sa.GpuKvCache(1, HKV, D, max(lens) + 4, batch=1, num_heads=HQ, bits=BITS, device=cuda_device)
        if n:
            sa.prefill_layer_step(prompts[i], None, w, cache, 0, batch=1, seq_len=n, **rope)
            cache.advance_position(n)
        caches.append(cache)
        held = cache.view(0)
        for j in range((n + 63) // 64):  # a block of 64 cached tokens is a page
            page = int(table[i, j])
            view.k_codes[page], view.k_meta[page] = held.k_codes[0, :, 64 * j:64 * j + 64], held.k_meta[0, :, 64 * j:64 * j + 64]
            view.v_codes[page], view.v_meta[page] = held.v_codes[0, :, 4 * j:4 * j + 4], held.v_meta[0, :, 64 * j:64 * j + 64]
    seq_lens = torch.tensor(lens + [-1], dtype=torch.int32, device=cuda_device)
    for _ in range(3):
        x, resid = _rows(r, b + 1, cuda_device), _rows(r, b + 1, cuda_device)
        d, pre = sa.paged_layer_step(x, resid, w, pool, 0, page_table=table, seq_lens=seq_lens, **rope)
        assert pool.device_status() == 0
        for i, cache in enumerate(caches):
            want, want_pre = sa.decoder_layer_step(x[i:i + 1], resid[i:i + 1], w, cache, 0, **rope)
            cache.advance_position(1)
            _near(d[i:i + 1], want, 2e-2)
            _near(pre[i:i + 1], want_pre, 2e-2)
        seq_lens[:b] += 1
