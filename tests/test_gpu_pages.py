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


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.5])
def test_attend_with_a_scale_of_its_own(cuda_device, dtype, scale):
    import smallaios_b200 as sa

    pool, q, table, ln, kw, want, limit = _attend_case(cuda_device, 4, 128, 2, 4, dtype, [300, 0, 64], 1, None, "half",
                                                       seed=3, scale=scale)
    got = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
    pr.check(got.double().cpu().numpy().reshape(want.shape), want, limit)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("bits", [4, 8])
def test_attend_over_values_of_no_or_little_scale(cuda_device, bits, dtype):
    """Constant value vectors (a scale of 1, codes of 0), scales of 0 and of 1e-30, and a token that takes all weight."""
    import smallaios_b200 as sa

    r = np.random.default_rng(4)
    h, g, d, n = 2, 4, 128, 200
    pages, table = pr.tables(r, [n])
    kc, km = ref.random_vectors(r, (pages, h, 64, d), bits)
    vc, vm = ref.random_vectors(r, (pages, h, 64, d), bits)
    vm[:, :, ::3, 0] = 0.0
    vm[:, :, 1::3, 0] = 1e-30
    vm[:, 1, :, 0] = 0.0                    # a head whose values all have none
    km[int(table[0, 1]), :, 5] *= 40.0      # far the largest scores, of either sign
    pool = _pool(1, h, g, d, bits, pages, cuda_device)
    signs = pr.fill(pool.view(0), kc, km, vc, vm)
    q = torch.from_numpy(r.standard_normal((1, 1, h * g * d)).astype(np.float32)).to(DT[dtype])
    qr = q.double().numpy().reshape(1, 1, h, g, d)
    want, size = pr.attend(qr, kc, km, vc, vm, signs, table, np.array([[n]]), bits)
    got = sa.gqa_paged_attend(q.to(cuda_device), pool, 0, _to(table, cuda_device),
                              torch.tensor([n - 1], dtype=torch.int32, device=cuda_device), num_heads=h * g)
    pr.check(got.double().cpu().numpy().reshape(want.shape), want, pr.bound(dtype, qr, size, want))


def test_attend_equals_the_contiguous_caches_attention(cuda_device):
    """Pages and a GpuKvCache filled by the same appends give the same answer within both paths' precision."""
    import smallaios_b200 as sa

    r = np.random.default_rng(5)
    b, h, g, d, n = 3, 4, 4, 128, 130
    cos, sin = (_to(x, cuda_device) for x in rope_tables(n, d))
    x = [torch.from_numpy(r.standard_normal((b, n, w * d)).astype(np.float32)).to(cuda_device) for w in (h, h, h * g)]
    kw = dict(cos_cache=cos, sin_cache=sin, do_rotary=True)
    cache = sa.GpuKvCache(1, h, d, n, batch=b, num_heads=h * g, device=cuda_device)
    cache.append(0, x[0], x[1], **kw)
    cache.set_position(n - 1)
    pages, table = pr.tables(r, [n] * b)
    pool = _pool(1, h, g, d, 4, pages, cuda_device)
    table = _to(table, cuda_device)
    lens = torch.zeros(b, dtype=torch.int32, device=cuda_device)
    for lo, hi in ((0, 1), (1, 64), (64, 129), (129, 130)):  # in steps
        pool.append(0, x[0][:, lo:hi], x[1][:, lo:hi], table, lens + lo, **kw)
    q = x[2][:, n - 1:].contiguous()
    want = sa.gqa_attend(q, cache, 0, num_heads=h * g, **kw)
    got = sa.gqa_paged_attend(q, pool, 0, table, lens + n - 1, num_heads=h * g, **kw)
    # both are within 1e-5 of the exact sum at scores of a few units and values of one
    assert (got - want).abs().max() < 2e-5


def test_appends_and_queries_from_slices_at_any_element(cuda_device):
    """Keys, values and queries as columns of one projection, aligned and not; tables as columns of a wider one."""
    import smallaios_b200 as sa

    r = np.random.default_rng(6)
    h, g, d, b, s = 2, 3, 64, 3, 5
    w = (g + 2) * h * d
    lens = [3, 60, 126]
    pages, table = pr.tables(r, [n + s for n in lens])
    cos, sin = (_to(x, cuda_device) for x in rope_tables(200, d))
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda_device)
    for dtype in DT.values():
        wide = torch.randn(b, s, w + 3, device=cuda_device).to(dtype)
        for first in (0, 1, 3):
            x = wide[..., first:first + w]
            q, k, v = x[..., :g * h * d], x[..., g * h * d:(g + 1) * h * d], x[..., (g + 1) * h * d:]
            outs = []
            for parts in ((q, k, v), [t.contiguous() for t in (q, k, v)]):
                pool = _pool(1, h, g, d, 8, pages, cuda_device)
                tab = _to(table, cuda_device)
                if parts[0] is q:
                    tab = torch.full((b, tab.shape[1] + 4), -7, dtype=torch.int32, device=cuda_device)[:, 1:-3]
                    tab.copy_(_to(table, cuda_device))
                kw = dict(do_rotary=True, cos_cache=cos, sin_cache=sin)
                pool.append(0, parts[1], parts[2], tab, ln, **kw)
                out = torch.empty(b * s * g * h * d + 1, dtype=dtype, device=cuda_device)[1:].view(b, s, -1)
                got = sa.gqa_paged_attend(parts[0], pool, 0, tab, ln, num_heads=g * h, out=out if parts[0] is q else None, **kw)
                view = pool.view(0)
                outs.append([got, view.k_codes, view.v_codes, view.k_meta, view.v_meta])
                assert pool.device_status() == 0
            assert all(torch.equal(x, y) for x, y in zip(*outs))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("s", [1, 9])
def test_rotary_tables_that_start_at_any_element(cuda_device, s, interleaved):
    import smallaios_b200 as sa

    h, g, d, b = 2, 3, 128, 2
    tables = [_to(x, cuda_device) for x in rope_tables(100, d)]
    shifted = [torch.cat([x.new_zeros(1), x.flatten()])[1:].view(x.shape) for x in tables]
    assert all(x.data_ptr() % 16 for x in shifted)
    k, v, q = (torch.randn(b, s, w * d, device=cuda_device) for w in (h, h, h * g))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([3, 60], dtype=torch.int32, device=cuda_device)
    outs = []
    for cos, sin in (tables, shifted):
        pool = _pool(1, h, g, d, 4, 4, cuda_device)
        kw = dict(do_rotary=True, rotary_interleaved=interleaved, cos_cache=cos, sin_cache=sin)
        pool.append(0, k, v, table, lens, **kw)
        outs.append([sa.gqa_paged_attend(q, pool, 0, table, lens, num_heads=h * g, **kw), pool.view(0).k_codes, pool.view(0).k_meta])
    assert all(torch.equal(x, y) for x, y in zip(*outs))


def test_attend_in_place_and_into_a_given_workspace(cuda_device):
    import smallaios_b200 as sa

    pool, q, table, ln, kw, _, _ = _attend_case(cuda_device, 4, 128, 2, 4, "bf16", [100, 3], 2, None, "half")
    want = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
    need = pool.workspace_bytes(2, 2, 16)
    ws = torch.full((need,), 255, dtype=torch.uint8, device=cuda_device)
    assert torch.equal(sa.gqa_paged_attend(q, pool, 0, table, ln, workspace=ws, **kw), want)
    x = q.clone()
    assert sa.gqa_paged_attend(x, pool, 0, table, ln, out=x, **kw) is x and torch.equal(x, want)
    with pytest.raises(sa.InvalidAttribute, match="workspace"):
        sa.gqa_paged_attend(q, pool, 0, table, ln, workspace=ws[:need - 1], **kw)
    with pytest.raises(sa.InvalidAttribute, match="aligned"):
        sa.gqa_paged_attend(q, pool, 0, table, ln, workspace=torch.empty(need + 16, dtype=torch.uint8, device=cuda_device)[16:], **kw)


def test_pages_far_behind_the_first(cuda_device):
    """A pool of more than 4 GB: the last pages lie past 32-bit offsets."""
    import smallaios_b200 as sa

    h, g, d, bits, pages = 4, 2, 128, 8, 64000  # 18432 bytes a head and page: 4.7 GB
    pool = _pool(1, h, g, d, bits, pages, cuda_device)
    small = _pool(1, h, g, d, bits, 3, cuda_device)
    k, v = (torch.randn(1, 150, h * d, device=cuda_device) for _ in range(2))
    q = torch.randn(1, 1, h * g * d, device=cuda_device)
    zero, last = (torch.tensor([n], dtype=torch.int32, device=cuda_device) for n in (0, 149))
    outs = []
    for p, ids in ((pool, [63999, 31000, 63998]), (small, [2, 0, 1])):
        table = torch.tensor([ids], dtype=torch.int32, device=cuda_device)
        p.append(0, k, v, table, zero)
        outs.append(sa.gqa_paged_attend(q, p, 0, table, last, num_heads=h * g))
        assert p.device_status() == 0
    assert torch.equal(*outs)
    pool.close()
    small.close()


def test_what_the_device_meets_is_reported(cuda_device):
    """Pages outside the pool and behind the table, positions behind the rotary tables: left out, and a status bit."""
    import smallaios_b200 as sa

    r = np.random.default_rng(7)
    h, g, d = 2, 2, 128
    pool = _pool(1, h, g, d, 4, 4, cuda_device)
    kw = dict(num_heads=h * g)
    x = [torch.from_numpy(r.standard_normal((3, 1, w * d)).astype(np.float32)).to(cuda_device) for w in (h, h, h * g)]
    good = torch.tensor([[0, 1], [2, 3], [-1, -1]], dtype=torch.int32, device=cuda_device)
    lens = torch.tensor([70, 5, -1], dtype=torch.int32, device=cuda_device)
    pool.append(0, x[0], x[1], good, lens)
    want = sa.gqa_paged_attend(x[2], pool, 0, good, lens, **kw)
    assert pool.device_status() == 0 and not want[2].any()
    held = pool.view(0).k_codes.clone()

    for bad in (-1, 4, 2**31 - 1, -2**31):
        table = good.clone()
        table[1, 0] = bad
        pool.append(0, x[1], x[0], table, torch.tensor([-1, 5, -1], dtype=torch.int32, device=cuda_device))
        assert pool.device_status(clear=True) == 2
        got = sa.gqa_paged_attend(x[2], pool, 0, table, lens, **kw)
        assert pool.device_status(clear=True) == 2
        assert torch.equal(got[0], want[0]) and not got[1].any()  # a row whose pages are all bad sees nothing
        table[0, 1] = bad  # the second page of row 0: its first 64 tokens are attended to
        got = sa.gqa_paged_attend(x[2], pool, 0, table, lens, **kw)
        first = sa.gqa_paged_attend(x[2], pool, 0, good, torch.tensor([63, 5, -1], dtype=torch.int32, device=cuda_device), **kw)
        assert torch.equal(got[0], first[0])
        assert pool.device_status(clear=True) == 2
    far = torch.tensor([200, 5, 2**31 - 1], dtype=torch.int32, device=cuda_device)  # more tokens than two pages hold
    pool.append(0, x[1], x[0], good, torch.tensor([200, -1, 2**31 - 1], dtype=torch.int32, device=cuda_device))
    assert pool.device_status(clear=True) == 2
    got = sa.gqa_paged_attend(x[2], pool, 0, good, far, **kw)
    assert pool.device_status(clear=True) == 2 and torch.equal(got[1], want[1])
    assert torch.equal(pool.view(0).k_codes, held)

    cos, sin = (_to(t, cuda_device) for t in rope_tables(70, d))
    rope = dict(do_rotary=True, cos_cache=cos, sin_cache=sin)
    pool.append(0, x[1], x[0], good, torch.tensor([70, -1, -1], dtype=torch.int32, device=cuda_device), **rope)
    assert pool.device_status(clear=True) == 4 and torch.equal(pool.view(0).k_codes, held)
    got = sa.gqa_paged_attend(x[2], pool, 0, good, lens, **kw, **rope)
    assert pool.device_status(clear=True) == 4 and not got[0].any() and got[1].any()


def test_refused_arguments(cuda_device):
    import smallaios_b200 as sa

    h, g, d = 2, 2, 64
    pool = _pool(2, h, g, d, 4, 4, cuda_device)
    k = torch.zeros(2, 3, h * d, device=cuda_device)
    q = torch.zeros(2, 3, h * g * d, device=cuda_device)
    table = torch.zeros(2, 2, dtype=torch.int32, device=cuda_device)
    lens = torch.zeros(2, dtype=torch.int32, device=cuda_device)
    cos = torch.zeros(8, d // 2, device=cuda_device)

    def both(error, match=None, layer=0, table=table, lens=lens, x=None, **kw):
        with pytest.raises(error, match=match):
            pool.append(layer, *((k, k) if x is None else (x(k), x(k))), table, lens, **kw)
        with pytest.raises(error, match=match):
            sa.gqa_paged_attend(q if x is None else x(q), pool, layer, table, lens, num_heads=h * g, **kw)

    both(sa.InvalidAttribute, "layer_idx", layer=2)
    both(sa.InvalidAttribute, "layer_idx", layer=-1)
    both(sa.UnsupportedOp, "int32", table=table.long())
    both(sa.UnsupportedOp, "int32", lens=lens.long())
    both(sa.UnsupportedOp, "int32", counts=lens.long())
    both(sa.ShapeMismatch, "page_table", table=table[:1])
    both(sa.ShapeMismatch, "page_table", table=table[0])
    both(sa.ShapeMismatch, "entries", lens=lens[:1])
    both(sa.ShapeMismatch, "entries", counts=lens[:1])
    both(ValueError, "page_table", table=torch.zeros(2, 4, dtype=torch.int32, device=cuda_device)[:, ::2])
    both(TypeError, "page_table", table=table.cpu())
    both(TypeError, "seq_lens", lens=None)
    both(sa.ShapeMismatch, "hidden size", x=lambda t: t[..., :-1].contiguous())
    both(sa.ShapeMismatch, "rank-3", x=lambda t: t[0])
    both(ValueError, "contiguous rows", x=lambda t: torch.zeros(*t.shape[:2], 2 * t.shape[2], device=cuda_device)[..., ::2])
    both(ValueError, "contiguous rows", x=lambda t: t[:, :1].expand(t.shape))
    both(sa.UnsupportedOp, "dtype", x=lambda t: t.double())
    both(sa.ShapeMismatch, "cos_cache", do_rotary=True)
    both(sa.ShapeMismatch, "come together", cos_cache=cos)
    both(sa.ShapeMismatch, "cos and sin", cos_cache=cos, sin_cache=cos[:4].contiguous(), do_rotary=True)
    both(sa.ShapeMismatch, "cos and sin", cos_cache=cos[:, :-1].contiguous(), sin_cache=cos[:, :-1].contiguous(), do_rotary=True)
    both(sa.UnsupportedOp, "float32", cos_cache=cos.half(), sin_cache=cos.half(), do_rotary=True)
    both(sa.ShapeMismatch, "tables of 0", cos_cache=cos[:0], sin_cache=cos[:0], do_rotary=True)
    with pytest.raises(sa.ShapeMismatch, match="equal shapes"):
        pool.append(0, k, k[:, :2], table, lens)
    with pytest.raises(sa.UnsupportedOp, match="differ"):
        pool.append(0, k, k.half(), table, lens)
    with pytest.raises(ValueError, match="same strides"):
        pool.append(0, k, torch.zeros(2, 3, 2 * h * d, device=cuda_device)[..., :h * d], table, lens)
    with pytest.raises(sa.ShapeMismatch, match="num_heads"):
        sa.gqa_paged_attend(q, pool, 0, table, lens, num_heads=h)
    for out in (q[:1], q.half()):
        with pytest.raises(sa.ShapeMismatch, match="out"):
            sa.gqa_paged_attend(q, pool, 0, table, lens, num_heads=h * g, out=out)
    with pytest.raises(sa._lib.SaError):
        pool.view(2)
    # nothing to do is no error
    for b, s in ((0, 3), (2, 0)):
        pool.append(0, k[:b, :s], k[:b, :s], table[:b], lens[:b])
        assert sa.gqa_paged_attend(q[:b, :s], pool, 0, table[:b], lens[:b], num_heads=h * g).shape == (b, s, h * g * d)
    none = table[:, :0].contiguous()
    pool.append(0, k, k, none, lens)
    assert not sa.gqa_paged_attend(q, pool, 0, none, lens, num_heads=h * g).any()
    assert pool.device_status(clear=True) == 2
    pool.append(0, k, k, none, lens - 1)
    assert pool.device_status() == 0
    pool.close()
    with pytest.raises(RuntimeError, match="close"):
        pool.append(0, k, k, table, lens)


# ---- streams, graphs, threads ---------------------------------------------------------------------------
@pytest.mark.parametrize("handles", [False, True])
def test_calls_on_other_streams(cuda_device, handles):
    """Two pools on two streams beside a busy current one: scratch and outputs are the streams' own."""
    import smallaios_b200 as sa

    cases = [_attend_case(cuda_device, 4, 128, 4, 4, "bf16", [900, 64 * 20, 3], 1, None, "half", seed=s) for s in (1, 2)]
    want = [sa.gqa_paged_attend(c[1], c[0], 0, c[2], c[3], **c[4]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(4):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                torch.cuda._sleep(2_000_000)
            got.append(sa.gqa_paged_attend(c[1], c[0], 0, c[2], c[3], **c[4], stream=s.cuda_stream if handles else s))
        for n in (cases[0][0].workspace_bytes(3, 1, 16), cases[0][1].numel() * 2):
            for _ in range(4):
                torch.full((n,), 255, dtype=torch.uint8, device=cuda_device)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_two_calls_on_one_pool_at_once(cuda_device):
    """Attention calls on one pool may overlap: each has a workspace of its own."""
    import smallaios_b200 as sa

    pool, q, table, ln, kw, _, _ = _attend_case(cuda_device, 4, 128, 8, 4, "bf16", [3000 + i for i in range(16)], 1, None, "half")
    want = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
    other = sa.gqa_paged_attend(q.flip(0).contiguous(), pool, 0, table, ln, **kw)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        a = sa.gqa_paged_attend(q, pool, 0, table, ln, stream=streams[0], **kw)
        streams[1].wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[1]):
            b = sa.gqa_paged_attend(q.flip(0).contiguous(), pool, 0, table, ln, **kw)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, other)


def test_a_captured_step_replays_with_new_lengths(cuda_device):
    """Append and attention, captured once; tables, lengths and inputs change between replays."""
    import smallaios_b200 as sa

    r = np.random.default_rng(8)
    b, h, g, d, steps = 3, 2, 4, 128, 70
    lens0 = [0, 50, 130]
    pages, table = pr.tables(r, [n + steps for n in lens0])
    cos, sin = (_to(x, cuda_device) for x in rope_tables(300, d))
    rope = dict(do_rotary=True, cos_cache=cos, sin_cache=sin)
    inputs = [[torch.from_numpy(r.standard_normal((b, 1, w * d)).astype(np.float32)).to(cuda_device).bfloat16()
               for w in (h, h, h * g)] for _ in range(steps)]
    fill = [torch.randn(b, 130, h * d, device=cuda_device).bfloat16() for _ in range(2)]
    outs = []
    for captured in (False, True):
        pool = _pool(1, h, g, d, 4, pages, cuda_device)
        tab = _to(table, cuda_device)
        lens = torch.tensor(lens0, dtype=torch.int32, device=cuda_device)
        pool.append(0, *fill, tab, torch.zeros_like(lens), counts=lens, **rope)
        x = [t.clone() for t in inputs[0]]

        def step():
            pool.append(0, x[0], x[1], tab, lens, **rope)
            out = sa.gqa_paged_attend(x[2], pool, 0, tab, lens, num_heads=h * g, **rope)
            lens.add_(1)
            return out

        got = []
        if captured:
            keep = lens.clone()
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            lens.copy_(keep)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
            lens.copy_(keep)
        for i in range(steps):
            for dst, src in zip(x, inputs[i]):
                dst.copy_(src)
            if captured:
                graph.replay()
                got.append(out.clone())
            else:
                got.append(step())
        assert pool.device_status() == 0
        outs.append(torch.cat(got))
    assert torch.equal(*outs)


def test_pools_of_several_threads(cuda_device):
    import smallaios_b200 as sa
    from tests.test_gpu_serving_threads import _run

    def job(seed, bits, d):
        pool, q, table, ln, kw, want, limit = _attend_case(cuda_device, bits, d, 2, 4, "f32", [200 + seed, 7], 1, None, "half",
                                                           seed=seed)

        def run():
            for _ in range(50):
                got = sa.gqa_paged_attend(q, pool, 0, table, ln, **kw)
            pr.check(got.double().cpu().numpy().reshape(want.shape), want, limit)
        return run

    jobs = [job(i, bits, d) for i, (bits, d) in enumerate(((4, 128), (8, 128), (4, 64), (8, 64), (4, 128)))]
    torch.cuda.synchronize()
    _run(jobs)


def test_a_shard_of_the_heads_holds_what_the_whole_pool_does(cuda_device):
    import smallaios_b200 as sa

    h, g, d = 4, 2, 64
    k, v, q = (torch.randn(1, 90, w * d, device=cuda_device) for w in (h, h, h * g))
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=cuda_device)
    zero, last = (torch.tensor([n], dtype=torch.int32, device=cuda_device) for n in (0, 89))
    whole = _pool(2, h, g, d, 4, 2, cuda_device)
    whole.append(1, k, v, table, zero)
    want = sa.gqa_paged_attend(q[:, -1:].contiguous(), whole, 1, table, last, num_heads=h * g)
    part = sa.GpuKvPages(2, h, d, 2, num_heads=h * g, bits=4, kv_head_begin=1, kv_head_count=2, device=cuda_device)
    part.append(1, k[..., d:3 * d], v[..., d:3 * d], table, zero)
    assert torch.equal(part.view(1).k_codes, whole.view(1).k_codes[:, 1:3])
    assert torch.equal(part.view(1).v_codes, whole.view(1).v_codes[:, 1:3])
    got = sa.gqa_paged_attend(q[:, -1:, g * d:3 * g * d], part, 1, table, last, num_heads=h * g)
    assert torch.equal(got, want[..., g * d:3 * g * d])
