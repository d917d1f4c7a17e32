"""Precision of attention over pages: its error against 64 bits beside the rounding of the outputs' type."""
import ctypes

import numpy as np
import pytest
import torch

from tests.test_gpu_pages import DT, _attend_case

pytestmark = pytest.mark.gpu


def _error(dtype, bits, d, g, lens, device, full):
    """Error of the outputs over the error of the exact values rounded once to their type, both as norms."""
    import smallaios_b200 as sa

    pool, q, table, ln, kw, want, _ = _attend_case(device, bits, d, 2, g, dtype, lens, 1, None, "half", seed=3)
    pool.set_precision(full)
    got = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw).double().cpu().numpy().reshape(want.shape)
    rounded = torch.from_numpy(want).to(DT[dtype]).double().numpy()
    pool.close()
    return np.linalg.norm(got - want) / np.linalg.norm(rounded - want)


SHAPES = [(4, 128, 4, [2000, 700]), (8, 128, 8, [1500, 64]), (4, 64, 2, [1000]), (8, 64, 11, [900, 5, 77]), (4, 128, 1, [3000])]


@pytest.mark.parametrize("bits,d,g,lens", SHAPES)
def test_outputs_are_rounded_once_by_choice(cuda_device, bits, d, g, lens):
    """24 bits of q' and of the weights, and sums in f32, are some 1e-6 of the output: beside the 2^-12.2 of f16's rounding
    (2^-11 / sqrt(12), over the mean significand) that adds 1e-5 in quadrature.  A thousandth is allowed; 16 bits add
    more than 1e-2 (below)."""
    assert _error("f16", bits, d, g, lens, cuda_device, True) < 1.001
    assert _error("bf16", bits, d, g, lens, cuda_device, True) < 1.001


@pytest.mark.parametrize("bits,d,g,lens", SHAPES)
def test_outputs_by_default(cuda_device, bits, d, g, lens):
    """16 bits: a query's digits move a weight by 0.29 max|q'| / 32639 |k| / sqrt(D), 4e-5 for components of one, a weight's
    own by 0.29 / 65535 of the largest, some 16 times itself: 8e-5.  Beside 2.1e-4 (f16) and 1.7e-3 (bf16) that adds 8%
    and a thousandth in quadrature."""
    assert _error("f16", bits, d, g, lens, cuda_device, False) < 1.15
    assert _error("bf16", bits, d, g, lens, cuda_device, False) < 1.005


def test_the_choice_is_the_pools(cuda_device):
    """Workspace and results follow the setting; f32 callers see no difference."""
    import smallaios_b200 as sa
    from smallaios_b200._lib import lib

    for dtype, code, differs in (("f16", 10, True), ("bf16", 16, True), ("f32", 1, False)):
        pool, q, table, ln, kw, _, _ = _attend_case(cuda_device, 4, 128, 2, 8, dtype, [300, 0, 64], 1, None, "half")
        outs, sizes = [], []
        for full in (False, True, False):
            pool.set_precision(full)
            sizes.append(pool.workspace_bytes(3, 1, code))
            assert sizes[-1] == lib.sa_gqa_paged_workspace_bytes(pool.handle, 3, 1, code)
            ws = torch.full((sizes[-1],), 255, dtype=torch.uint8, device=cuda_device)
            outs.append(sa.gqa_paged_attend(q, pool, 0, table, ln, workspace=ws, **kw))
            assert torch.equal(outs[-1], sa.gqa_paged_attend(q, pool, 0, table, ln, **kw))
        assert torch.equal(outs[0], outs[2]) and sizes[0] == sizes[2]
        assert torch.equal(outs[0], outs[1]) != differs
    assert lib.sa_kv_pages_set_precision(ctypes.c_void_p(), 1) == 9
    pool.close()
    with pytest.raises(RuntimeError, match="close"):
        pool.set_precision(True)
