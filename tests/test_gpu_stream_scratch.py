"""Calls launched on a stream that is not the current one: their scratch is not handed out while they run."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _lists, _query, _random, _trees

pytestmark = pytest.mark.gpu


def _problem(seed, device, dtype="bf16", b=4, h=4, g=4, d=128, bits=4, past=64 * 30, n=8):
    import smallaios_b200 as sa

    r, kc, km, vc, vm = _random(seed, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, dtype, device)
    parents = _device(_trees(r, b, n), device)
    ids = _device(_lists(r, b, n, h, 5, past), device)
    means = sa.kv_block_means(cache, 0, 0, past // 64)
    calls = {
        "tree": lambda stream=None: sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g, stream=stream),
        "sparse": lambda stream=None: sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g, stream=stream),
        "select": lambda stream=None: sa.gqa_select_blocks(q, cache, 0, means, num_heads=h * g, max_blocks=6, stream=stream),
        "means": lambda stream=None: sa.kv_block_means(cache, 0, 0, past // 64, stream=stream),
    }
    sizes = (cache.tree_workspace_bytes(n, 16), sa._lib.lib.sa_gqa_sparse_workspace_bytes(cache.handle, n),
             q.numel() * q.element_size())
    return cache, calls, sizes


@pytest.mark.parametrize("handles", [False, True])
@pytest.mark.parametrize("op", ["tree", "sparse", "select", "means"])
def test_two_streams_beside_a_busy_current_one(cuda_device, op, handles):
    problems = [_problem(seed, cuda_device) for seed in (1, 2)]
    want = [calls[op]() for _, calls, _ in problems]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in problems]
    for _ in range(5):
        got = []
        for s, (_, calls, _) in zip(streams, problems):
            with torch.cuda.stream(s):
                torch.cuda._sleep(2_000_000)  # the call's kernels start about a millisecond after it returned
            got.append(calls[op](s.cuda_stream if handles else s))
        for size in problems[0][2]:
            for _ in range(4):
                torch.full((max(size, 1),), 255, dtype=torch.uint8, device=cuda_device)
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    for cache, _, _ in problems:
        cache.close()


def test_handle_zero_is_the_default_stream(cuda_device):
    cache, calls, _ = _problem(3, cuda_device)
    want = calls["tree"]()
    assert torch.equal(calls["tree"](0), want)
    cache.close()
