"""Host-side checks of paged serving and beam search that answer without a GPU."""
import ctypes

import pytest
import torch


def _cfg(**kw):
    from smallaios_b200 import _lib

    c = _lib.KvPagesConfig()
    base = dict(num_layers=1, num_pages=4, num_heads=8, num_kv_heads=2, kv_head_begin=0, kv_head_count=2, head_dim=64, bits=4,
                seed=42)
    for k, v in {**base, **kw}.items():
        setattr(c, k, v)
    return c


@pytest.mark.parametrize("kw,status,msg", [
    (dict(head_dim=32), 3, b"head_dim 32"),
    (dict(head_dim=256), 3, b"head_dim 256"),
    (dict(bits=3), 3, b"bits must be 4 or 8"),
    (dict(num_pages=0), 9, b"zero dimension"),
    (dict(num_layers=-1), 9, b"zero dimension"),
    (dict(num_heads=7), 1, b"num_heads must be a positive multiple"),
    (dict(kv_head_begin=1), 1, b"kv head range"),
    (dict(kv_head_begin=2**31 - 1, kv_head_count=1), 1, b"kv head range"),
])
def test_pool_config_validation_without_gpu(kw, status, msg):
    from smallaios_b200._lib import lib

    h = ctypes.c_void_p()
    assert lib.sa_kv_pages_create(ctypes.byref(_cfg(**kw)), ctypes.byref(h)) == status
    assert msg in lib.sa_last_error_string()
    assert not h.value


@pytest.mark.parametrize("kw", [
    dict(num_pages=2**31 - 1, num_layers=2**31 - 1), dict(num_pages=2**30, num_layers=2**10),
    dict(num_heads=2**30, num_kv_heads=2**30, kv_head_count=2**30, num_pages=2**20, num_layers=2**20),
])
def test_a_pool_beyond_any_memory_is_refused_before_it_is_counted_in_bytes(kw):
    from smallaios_b200._lib import lib

    h = ctypes.c_void_p()
    assert lib.sa_kv_pages_create(ctypes.byref(_cfg(**kw)), ctypes.byref(h)) == 5
    assert b"256 GiB" in lib.sa_last_error_string()
    assert not h.value


def test_null_handles_are_rejected():
    from smallaios_b200._lib import lib

    none = [None] * 3
    assert lib.sa_kv_pages_destroy(None) == 0
    assert lib.sa_kv_pages_create(None, None) == 9
    assert lib.sa_kv_pages_get_config(None, None) == 9
    assert lib.sa_kv_pages_layer_view(None, 0, None) == 9
    assert lib.sa_kv_pages_device_status(None, None, 0) == 9
    assert lib.sa_kv_pages_append(None, 0, None, None, 0, 0, 1, 1, 1, None, 0, 0, *none, None, 0, 0, 0, None) == 9
    assert lib.sa_gqa_paged_attend(None, 0, None, 0, 0, None, 1, 1, 1, 8, 0, 0.0, None, 0, 0, *none, None, 0, 0, 0, None, 0,
                                   None) == 9
    assert lib.sa_kv_pages_reorder(None, None, 0, None, 0, 0, None, None, 1, 1, None) == 9
    assert lib.sa_gqa_paged_workspace_bytes(None, 1, 1, 1) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=7), 3), (dict(beams=0), 1), (dict(beams=33), 1), (dict(keep=0), 1), (dict(keep=65), 1), (dict(vocab=0), 2),
    (dict(vocab=100, stride=99), 2), (dict(batch=-1), 2), (dict(vocab=2**31), 3), (dict(vocab=2**29, beams=8), 3),
    (dict(batch=2**29, beams=8), 3), (dict(logits=None), 9), (dict(logits=1027), 9), (dict(workspace_bytes=1), 9),
    (dict(workspace=1024 + 16), 9), (dict(batch=0), 0),
])
def test_selection_arguments_without_gpu(kw, status):
    """No launch follows a refusal, so the pointers are never followed."""
    from smallaios_b200._lib import lib

    a = {**dict(logits=1024, dtype=1, batch=2, beams=4, vocab=1000, keep=4, workspace=1024, workspace_bytes=1 << 40), **kw}
    stride = a.get("stride", a["vocab"])
    assert lib.sa_beam_select(a["logits"], stride, a["dtype"], 1024, None, a["batch"], a["beams"], a["vocab"], 2, a["keep"], 1024,
                              1024, 1024, a["workspace"], a["workspace_bytes"], None) == status


def test_selection_workspace_is_zero_for_what_is_refused():
    from smallaios_b200._lib import lib

    assert lib.sa_beam_select_workspace_bytes(2, 4, 1000) > 0
    for args in ((0, 4, 1000), (2, 33, 1000), (2, 4, 0), (2, 4, 2**30)):
        assert lib.sa_beam_select_workspace_bytes(*args) == 0


def test_python_checks_want_gpu_tensors():
    import smallaios_b200 as sa

    class Pool:  # what the checks read of a pool
        query_width, kv_width, half_dim, device = 64, 64, 32, torch.device("cuda", 0)

    with pytest.raises(TypeError):
        sa.gqa_paged_attend(torch.zeros(1, 1, 64), Pool(), 0, torch.zeros(1, 1), torch.zeros(1), num_heads=1)
    with pytest.raises(TypeError):
        sa.GpuKvPages.append(Pool(), 0, torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), None, None)
    with pytest.raises(TypeError):
        sa.GpuKvPages.reorder_beams(Pool(), None, None, torch.zeros(1, 1, dtype=torch.int32))
    with pytest.raises(TypeError):
        sa.beam_select(torch.zeros(2, 5), torch.zeros(1, 2))
