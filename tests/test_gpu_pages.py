"""Paged serving on the GPU: appending to pages against the oracle's codes, attention over pages against its plain
64-bit form (tests/pages_reference.py)."""
import numpy as np
import pytest
import torch

import tests.pages_reference as pr
import tests.serving_reference as ref
from tests.helpers import oracle_append, rope_tables

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _pool(layers, h, g, d, bits, pages, device, **kw):
    import smallaios_b200 as sa

    return sa.GpuKvPages(layers, h, d, pages, num_heads=h * g, bits=bits, device=device, **kw)


def _to(x, device):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device)


def _arrays(view):
    return [x.cpu().numpy().copy() for x in (view.k_codes, view.v_codes_tokens(), view.k_meta, view.v_meta)]


def _expect(held, table, b, pos, token):
    """Token `token` of an oracle append into the held arrays, at position pos of row b."""
    page, t = table[b, pos // pr.PAGE], pos % pr.PAGE
    for a, x in zip(held, token):
        a[page, :, t] = x


# ---- append ---------------------------------------------------------------------------------------
APPENDS = [  # bits, d, h, dtype, S, lens, counts, rotation (None, half, interleaved)
    (4, 128, 8, "bf16", 1, [0, 1, 63, 64, 700], None, "half"),
    (8, 128, 3, "f32", 1, [5, -1, 130], None, "interleaved"),
    (8, 64, 1, "f16", 1, [127] * 9, None, "half"),
    (4, 64, 2, "f32", 1, [0], None, None),
    (4, 128, 2, "bf16", 200, [0, 61, 3], [200, 77, 0], "half"),
    (4, 128, 3, "f32", 7, [2, 59, 64, 120], None, "interleaved"),
    (8, 128, 2, "f16", 67, [0, 1, 2], [67, 66, 1], "half"),
    (8, 64, 4, "bf16", 33, [31, 0], [5, 33], "interleaved"),
    (4, 64, 5, "f16", 129, [6], None, "half"),
    (8, 64, 1, "f32", 2, [63, -3, 62], [2, 2, 9], None),
]


@pytest.mark.parametrize("bits,d,h,dtype,s,lens,counts,rotation", APPENDS)
def test_append_writes_the_oracles_codes(cuda_device, bits, d, h, dtype, s, lens, counts, rotation):
    r = np.random.default_rng(hash((bits, d, h, s)) % 2**32)
    b = len(lens)
    n = [0 if ln < 0 else s if counts is None else min(counts[i], s) for i, ln in enumerate(lens)]
    pages, table = pr.tables(r, [max(ln, 0) + m for ln, m in zip(lens, n)])
    pool = _pool(2, h, 1, d, bits, pages, cuda_device)
    view = pool.view(1)
    for x in (view.k_codes, view.v_codes):
        x.copy_(torch.randint(0, 256, x.shape, device=cuda_device, dtype=torch.uint8))
    for x in (view.k_meta, view.v_meta):
        x.copy_(torch.randn(x.shape, device=cuda_device))
    want, other = _arrays(view), _arrays(pool.view(0))
    cos, sin = rope_tables(max(max(lens), 0) + s, d)
    k = torch.from_numpy(r.standard_normal((b, s, h * d)).astype(np.float32)).to(DT[dtype])
    v = torch.from_numpy(r.standard_normal((b, s, h * d)).astype(np.float32)).to(DT[dtype])
    signs = view.signs.cpu().numpy()
    for i in range(b):
        if n[i] <= 0:
            continue
        x = [t[i:i + 1, :n[i]].float().numpy().reshape(1, n[i], h, d) for t in (k, v)]
        kc, km, vc, vm = oracle_append(*x, signs, bits, lens[i], cos, sin, do_rotary=rotation is not None,
                                       interleaved=rotation == "interleaved")
        for j in range(n[i]):
            _expect(want, table, i, lens[i] + j, (kc[0, :, j], vc[0, :, j], km[0, :, j], vm[0, :, j]))
    pool.append(1, k.to(cuda_device), v.to(cuda_device), _to(table, cuda_device),
                torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=cuda_device),
                do_rotary=rotation is not None, rotary_interleaved=rotation == "interleaved",
                cos_cache=_to(cos, cuda_device), sin_cache=_to(sin, cuda_device))
    assert pool.device_status() == 0
    for got, x in zip(_arrays(view), want):
        assert np.array_equal(got.view(np.uint32 if got.dtype == np.float32 else np.uint8),
                              x.view(np.uint32 if x.dtype == np.float32 else np.uint8))
    for got, x in zip(_arrays(pool.view(0)), other):
        assert np.array_equal(got, x)


@pytest.mark.parametrize("s", [1, 12])
@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64)])
def test_append_of_special_vectors_equals_the_contiguous_caches(cuda_device, bits, d, s):
    """Zeros of both signs, constants, the ends of the range, infinities, NaN, and values that lie on code borders."""
    import smallaios_b200 as sa

    r = np.random.default_rng(3)
    h, b = 4, 6
    x = r.standard_normal((2, b, s, h, d)).astype(np.float32)
    special = [np.zeros(d), -np.zeros(d), np.where(np.arange(d) % 2, 0.0, -0.0), np.full(d, 3.25), np.full(d, 1e30),
               np.full(d, 1e-40), np.eye(d)[5] * 1e-38, np.eye(d)[0] * 3e38, np.full(d, 3e38), np.eye(d)[1] * np.inf,
               np.full(d, np.nan), np.where(np.arange(d) == 7, np.nan, 1.0), np.where(np.arange(d) < 2, np.inf, 0.0),
               np.where(np.arange(d) == 3, -np.inf, 2.0), np.arange(d) % 16, np.where(np.arange(d) % 3 == 0, 1.0, -1.0),
               np.where(np.arange(d) < d // 2, 1.0, 2.0), np.eye(d)[9] * 2.0 ** 100]
    for i in range(2 * b * s * h):
        if i % 3 != 2:
            x.reshape(-1, d)[i] = special[(i - i // 3) % len(special)]
    k, v = (torch.from_numpy(a.reshape(b, s, h * d)).to(cuda_device) for a in x)
    cache = sa.GpuKvCache(1, h, d, 64, batch=b, bits=bits, device=cuda_device)
    pool = _pool(1, h, 1, d, bits, b, cuda_device)
    table = torch.randperm(b, device=cuda_device).to(torch.int32)[:, None].contiguous()
    cache.append(0, k, v)
    pool.append(0, k, v, table, torch.zeros(b, dtype=torch.int32, device=cuda_device))
    got, want, at = pool.view(0), cache.view(0), table[:, 0].long()
    assert torch.equal(got.k_codes[at][:, :, :s], want.k_codes[:, :, :s])
    assert torch.equal(got.v_codes_tokens()[at][:, :, :s], want.v_codes_tokens()[:, :, :s])
    for a, e in ((got.k_meta, want.k_meta), (got.v_meta, want.v_meta)):
        a, e = a[at][:, :, :s], e[:, :, :s]
        same = (a.contiguous().view(torch.int32) == e.contiguous().view(torch.int32)) | (a.isnan() & e.isnan())
        assert same.all()


# ---- attention ------------------------------------------------------------------------------------
ATTENDS = [  # bits, d, h, g, dtype, lens before the new tokens, S, counts, rotation
    (8, 64, 2, 4, "f32", [511], 1, None, "half"),
    (4, 128, 8, 4, "bf16", [0, 1, 62, 63, 64, 65, 1000], 1, None, "half"),
    (4, 128, 2, 8, "f16", [129, -1, 4095], 1, None, "interleaved"),
    (4, 128, 3, 8, "f32", [129, -1, 700], 1, None, "interleaved"),
    (8, 128, 1, 1, "f32", [33, 31, 32, 0], 1, None, None),
    (8, 128, 2, 3, "bf16", [333, 100, 95], 1, None, "half"),
    (4, 64, 2, 7, "f16", [64 * 9 - 1], 1, None, "half"),
    (8, 64, 1, 2, "bf16", [3, 900, 17], 1, None, None),
    (4, 128, 2, 16, "bf16", [200, 70], 1, None, "half"),   # two blocks of query heads
    (8, 64, 1, 11, "f32", [77], 1, None, "half"),          # three, the last one of three heads
    (4, 128, 2, 4, "f32", [60, 0, 300], 9, None, "half"),
    (4, 128, 2, 5, "bf16", [60, 5, 300], 9, [9, 0, 3], "interleaved"),
    (4, 64, 1, 1, "f32", [-1, -5], 1, None, "half"),
    (4, 128, 4, 4, "f32", [(i * 37) % 230 for i in range(150)], 1, None, "half"),   # more units than warps
    (4, 64, 1, 1, "bf16", [(i * 7) % 70 - 1 for i in range(2500)], 1, None, None),  # more rows than a launch takes
    (8, 128, 8, 4, "bf16", [1500, 0, 3], 1, None, "half"),
]


def _attend_case(device, bits, d, h, g, dtype, lens, s, counts, rotation, seed=0, scale=None, poison=False, layers=1):
    r = np.random.default_rng(seed)
    b = len(lens)
    pages, table = pr.tables(r, [max(ln + s, 0) for ln in lens])
    kc, km = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    vc, vm = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    pool = _pool(layers, h, g, d, bits, pages, device)
    signs = pr.fill(pool.view(layers - 1), kc, km, vc, vm)
    cos, sin = rope_tables(max(max(lens), 0) + s, d)
    q = torch.from_numpy((r.standard_normal((b, s, h * g * d)) * 1.3).astype(np.float32)).to(DT[dtype])
    qr = q.double().numpy().reshape(b, s, h, g, d).copy()
    sees = np.zeros((b, s), np.int64)
    for i in range(b):
        for j in range(s):
            if lens[i] >= 0 and (counts is None or j < counts[i]):
                sees[i, j] = lens[i] + j + 1
                if rotation:
                    qr[i, j] = pr.rotate(qr[i, j], lens[i] + j, cos, sin, rotation == "interleaved")
    want, size = pr.attend(qr, kc, km, vc, vm, signs, table, sees, bits, scale)
    limit = pr.bound(dtype, qr, size, want, scale)
    kw = dict(num_heads=h * g, do_rotary=rotation is not None, rotary_interleaved=rotation == "interleaved",
              cos_cache=_to(cos, device), sin_cache=_to(sin, device), scale=scale,
              counts=None if counts is None else torch.tensor(counts, dtype=torch.int32, device=device))
    if poison:  # what lies behind a row's tokens is never used
        view = pool.view(layers - 1)
        for i in range(b):
            n = max(lens[i] + s, 0)
            if n % pr.PAGE:
                page = int(table[i, n // pr.PAGE])
                view.k_meta[page, :, n % pr.PAGE:] = float("nan")
                view.v_meta[page, :, n % pr.PAGE:] = float("inf")
    return pool, q.to(device), _to(table, device), torch.tensor(lens, dtype=torch.int32, device=device), kw, want, limit


@pytest.mark.parametrize("bits,d,h,g,dtype,lens,s,counts,rotation", ATTENDS)
def test_attend_matches_the_plain_form(cuda_device, bits, d, h, g, dtype, lens, s, counts, rotation):
    import smallaios_b200 as sa

    pool, q, table, ln, kw, want, limit = _attend_case(cuda_device, bits, d, h, g, dtype, lens, s, counts, rotation,
                                                       poison=True)
    got = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
    assert pool.device_status() == 0
    pr.check(got.double().cpu().numpy().reshape(want.shape), want, limit)
    again = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
    assert torch.equal(got, again)
