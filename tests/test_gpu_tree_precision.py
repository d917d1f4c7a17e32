"""Precision of the draft-tree attention: its error against 64 bits beside the rounding of the outputs' type."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests.test_gpu_serving import _cache, _device, _query, _random, _trees

pytestmark = pytest.mark.gpu


def _error(dtype, bits, d, g, past, n, device, b=2, h=2, full=False):
    """Error of the outputs over the error of the exact values rounded once to their type, both as norms."""
    import smallaios_b200 as sa

    r, kc, km, vc, vm = _random(past + n, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    if full:
        cache.set_tree_precision(True)
    q, q64 = _query(r, b, n, h, g, d, dtype, device)
    parents = _trees(r, b, n, ragged=False)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, k, v, np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2))
    rounded = torch.from_numpy(want).to(out.dtype).double().numpy()
    cache.close()
    return np.linalg.norm(out.double().cpu().numpy() - want) / np.linalg.norm(rounded - want)


@pytest.mark.parametrize("bits,d,g,past,n", [(4, 128, 4, 2000, 16), (8, 128, 8, 1500, 8), (4, 64, 2, 1000, 20), (8, 64, 4, 3000, 4)])
def test_f16_outputs_are_rounded_once(cuda_device, bits, d, g, past, n):
    """Two planes of q^ and u hold 22 bits, and f32 sums over 25 tiles lose less than 2^-17: next to the 2^-12.2 of
    the type's rounding (2^-11 / sqrt(12), over the mean significand) that adds in quadrature below 0.1%.  A tenth is
    allowed; one plane of u adds 0.2 and more."""
    assert _error("f16", bits, d, g, past, n, cuda_device) < 1.1


@pytest.mark.parametrize("bits,d,g,past,n", [(4, 128, 4, 2000, 16), (8, 64, 4, 3000, 4)])
def test_bf16_outputs_by_default(cuda_device, bits, d, g, past, n):
    """One plane each of q^ and u: 2^-12 / sqrt(3) or so apiece against 2^-9.2, in quadrature about 2%."""
    assert _error("bf16", bits, d, g, past, n, cuda_device) < 1.05


@pytest.mark.parametrize("bits,d,g,past,n", [(4, 128, 4, 2000, 16), (8, 64, 4, 3000, 4), (4, 128, 8, 700, 64), (4, 64, 1, 900, 3)])
def test_bf16_outputs_are_rounded_once_by_choice(cuda_device, bits, d, g, past, n):
    """22 bits of q^ and u, 2^-17 of f32 sums: below 0.1% beside 2^-9.2.  A hundredth is allowed."""
    assert _error("bf16", bits, d, g, past, n, cuda_device, full=True) < 1.01


def test_the_choice_is_the_caches(cuda_device):
    """Workspace and results follow the setting; f32 callers see no difference."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 2, 2, 4, 128, 4, 300, 12
    r, kc, km, vc, vm = _random(1, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    parents = _device(_trees(r, b, n), cuda_device)
    for dtype, differs in (("bf16", True), ("f32", False)):
        q, _ = _query(r, b, n, h, g, d, dtype, cuda_device)
        outs = []
        for full in (False, True, False):
            cache.set_tree_precision(full)
            outs.append(sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g))
        assert torch.equal(outs[0], outs[2])
        assert torch.equal(outs[0], outs[1]) != differs
    cache.close()
