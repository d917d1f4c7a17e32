"""Serving operators on the GPU against their plain 64-bit forms (tests/serving_reference.py): attention of a
draft tree, keeping accepted drafts, block means, block selection and block-sparse attention."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _cache(b, h, g, d, bits, tokens, device, layers=1, **kw):
    import smallaios_b200 as sa

    return sa.GpuKvCache(layers, h, d, tokens, batch=b, num_heads=h * g, bits=bits, device=device, **kw)


def _random(seed, b, h, d, bits, tokens):
    r = np.random.default_rng(seed)
    kc, km = ref.random_vectors(r, (b, h, tokens, d), bits)
    vc, vm = ref.random_vectors(r, (b, h, tokens, d), bits)
    return r, kc, km, vc, vm


def _query(r, b, s, h, g, d, dtype, device, spread=1.3):
    q = torch.from_numpy((r.standard_normal((b, s, h * g * d)) * spread).astype(np.float32)).to(DT[dtype])
    return q.to(device), q.double().numpy().reshape(b, s, h, g, d)


def _trees(r, b, n, ragged=True):
    parents = np.full((b, n), -2, np.int32)
    for i in range(b):
        size = n if i == 0 or not ragged else int(r.integers(0, n + 1))
        for j in range(size):
            parents[i, j] = int(r.integers(-1, j)) if j else -1
    return parents


def _device(x, device):
    return torch.from_numpy(np.ascontiguousarray(x)).to(device)


# ---- draft trees ---------------------------------------------------------------------------------
TREES = [  # bits, d, g, dtype, b, h, past, n
    (8, 64, 4, "f32", 1, 2, 512, 8),
    (4, 128, 4, "bf16", 2, 2, 1000, 16),
    (4, 128, 8, "f16", 2, 1, 700, 64),
    (4, 128, 4, "f32", 2, 3, 333, 26),
    (8, 128, 3, "f32", 2, 2, 257, 33),
    (8, 128, 1, "bf16", 3, 1, 129, 64),
    (4, 64, 7, "f16", 1, 2, 191, 19),
    (4, 64, 2, "f32", 5, 2, 64, 7),
    (8, 64, 5, "f32", 1, 1, 127, 50),
    (4, 128, 4, "f32", 2, 2, 0, 13),     # nothing cached yet
    (4, 128, 4, "f32", 1, 1, 0, 1),      # one token in all
    (4, 128, 1, "f32", 1, 2, 1, 1),
    (4, 128, 4, "f16", 1, 2, 63, 2),     # the drafts straddle a block
    (4, 128, 4, "f32", 40, 4, 300, 4),   # more units than SMs
    (4, 128, 2, "f32", 1, 1, 9000, 3),   # few rows, long context
    (4, 64, 1, "bf16", 600, 8, 70, 2),   # more row blocks than one launch takes
    (4, 128, 8, "bf16", 11, 8, 199, 56), # many rows over a short context: several per warp of the merge
    (8, 64, 2, "f16", 30, 8, 300, 40),   # the same with units cut between ranges
    (3, 64, 4, "f32", 2, 2, 100, 9),     # formats of the general kernel
    (4, 32, 4, "f16", 2, 2, 77, 5),
    (8, 16, 2, "f32", 2, 2, 40, 6),
    (4, 256, 8, "bf16", 1, 2, 150, 12),
]


@pytest.mark.parametrize("bits,d,g,dtype,b,h,past,n", TREES)
def test_tree_attend(cuda_device, bits, d, g, dtype, b, h, past, n):
    import smallaios_b200 as sa

    r, kc, km, vc, vm = _random(past * 131 + n, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n + 5, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, dtype, cuda_device)
    parents = _trees(r, b, n)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2)
    want = ref.attend(q64, k, v, sees)
    got = out.double().cpu().numpy()
    ref.assert_rows(got, want, ref.row_bound(dtype, q64, k, v, vc, vm, want), d)
    assert (got.reshape(b, n, -1)[~sees.any(-1)[:, :, 0]] == 0).all()
    assert cache.device_status() == 0
    cache.close()


@pytest.mark.parametrize("scale", [0.01, 1.0, 3.0])
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_tree_attend_scale_and_peaked_scores(cuda_device, scale, dtype):
    """The scale attribute, up to scores of several hundred (one token takes all the weight)."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 2, 2, 4, 128, 4, 500, 10
    r, kc, km, vc, vm = _random(5, b, h, d, bits, past + n)
    km[:, :, 100:200] *= 3.0  # later tokens outgrow the first ones: the running maximum moves
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, dtype, cuda_device)
    parents = _trees(r, b, n)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g, scale=scale)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, k, v, np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2), scale)
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound(dtype, q64, k, v, vc, vm, want, scale), d)
    cache.close()


@pytest.mark.parametrize("vscale", [1e-6, 1e5])
def test_tree_attend_value_range(cuda_device, vscale):
    """Values far from 1, and of magnitudes that differ between tokens."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 1, 2, 4, 128, 4, 400, 10
    r, kc, km, vc, vm = _random(6, b, h, d, bits, past + n)
    vm = (vm * vscale * 2.0 ** r.integers(-6, 7, (b, h, past + n, 1))).astype(np.float32)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, "f32", cuda_device)
    parents = _trees(r, b, n)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, k, v, np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound("f32", q64, k, v, vc, vm, want), d)
    cache.close()


@pytest.mark.parametrize("bits,d,g,dtype", [(4, 128, 4, "f32"), (4, 128, 4, "bf16"), (8, 64, 8, "f32"), (3, 64, 2, "f32")])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3.0e38])
def test_tree_attend_masked_places_take_no_part(cuda_device, bits, d, g, dtype, bad):
    """NaN, infinities and the largest values in drafts that a node does not see, and past the drafts."""
    import smallaios_b200 as sa

    b, h, past, n = 2, 2, 100, 12
    tokens = past + n + 40
    r, kc, km, vc, vm = _random(9, b, h, d, bits, tokens)
    parents = np.tile(np.array([-1, 0, 0, 1, 2, 2, -1, 6, -2, 8, 5, 20], np.int32), (b, 1))
    spoiled = [3, 7, 8, 9, 11]  # leaves and slots without a node
    km[:, :, [past + j for j in spoiled]] = bad
    vm[:, :, [past + j for j in spoiled]] = bad
    km[:, :, past + n:] = bad
    vm[:, :, past + n:] = bad
    cache = _cache(b, h, g, d, bits, tokens, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, dtype, cuda_device)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    clean = [j for j in range(n) if j not in (3, 7)]
    with np.errstate(all="ignore"):
        k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
        sees = np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2)
        want = ref.attend(q64[:, clean], k, v, sees[:, clean])
    good = [t for t in range(past + n) if t - past not in spoiled]
    bound = ref.row_bound(dtype, q64, k[:, :, good], v[:, :, good], vc[:, :, good], vm[:, :, good], want)
    ref.assert_rows(out.double().cpu().numpy()[:, clean], want, bound, d)
    cache.close()


def test_tree_attend_rejects_nothing_finite_in_one_row(cuda_device):
    """A query row of NaN or infinity spoils its own rows only."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 1, 1, 4, 128, 4, 300, 9
    r, kc, km, vc, vm = _random(10, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, q64 = _query(r, b, n, h, g, d, "f32", cuda_device)
    q[0, 2] = float("nan")
    q[0, 5] = float("inf")
    parents = _trees(r, b, n)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    clean = [0, 1, 3, 4, 6, 7, 8]
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2)
    want = ref.attend(q64[:, clean], k, v, sees[:, clean])
    ref.assert_rows(out.double().cpu().numpy()[:, clean], want,
                    ref.row_bound("f32", q64[:, clean], k, v, vc, vm, want), d)
    assert torch.isnan(out[0, 2]).all()
    cache.close()


@pytest.mark.parametrize("lowrank", [None, 2])
def test_tree_chain_is_causal_attention(cuda_device, lowrank):
    """A chain of drafts, appended through the cache, is what gqa_attend computes for a chunk."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 2, 2, 4, 64, 4, 130, 11
    r = np.random.default_rng(3)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device, lowrank_k=lowrank)
    for count in (past, n):
        kv = [torch.from_numpy(r.standard_normal((b, count, h * d)).astype(np.float32)).to(cuda_device) for _ in "kv"]
        cache.append(0, *kv)
        if count == past:
            cache.advance_position(past)
    q, _ = _query(r, b, n, h, g, d, "f32", cuda_device)
    parents = np.tile(np.arange(-1, n - 1, dtype=np.int32), (b, 1))
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    want = sa.gqa_attend(q, cache, 0, num_heads=h * g, do_rotary=False)
    # both within their own error of the same value: 2^-20 (|q||k| scale about 20, twice) of values near 4
    assert (out - want).abs().max().item() < 4e-4
    cache.close()


# ---- keeping accepted drafts -----------------------------------------------------------------------
@pytest.mark.parametrize("bits,d,qjl,path", [
    (4, 128, False, [[0, 3, 7], [0, 1, 2]]),
    (8, 64, True, [[5, 0, 3], [2, 1, 0]]),           # any order: rows are read before any is written
    (3, 64, False, [[7, 7, 7], [0, 0, 1]]),          # a row may be kept more than once
    (4, 32, True, [[4], [0]]),
    (4, 256, False, [[0, 1, 2, 3, 4, 5, 6, 7], [7, 6, 5, 4, 3, 2, 1, 0]]),
    (4, 16, False, [[3, 5], [1, 6]]),
])
@pytest.mark.parametrize("past", [0, 13, 62])
def test_keep_drafts(cuda_device, bits, d, qjl, path, past):
    b, h, layers, drafted = 2, 3, 2, 8
    cache = _cache(b, h, 1, d, bits, past + drafted + 3, cuda_device, layers=layers, qjl_residual=qjl)
    r = np.random.default_rng(past)
    want = []
    for layer in range(layers):
        view = cache.view(layer)
        arrays = [view.k_codes, view.v_codes, view.k_meta, view.v_meta]
        arrays += [view.k_qjl_bits, view.v_qjl_bits, view.k_qjl_mag, view.v_qjl_mag] if qjl else []
        for a in arrays:
            x = r.integers(0, 256, a.shape).astype(np.uint8) if a.dtype == torch.uint8 else r.standard_normal(a.shape)
            a.copy_(_device(x, cuda_device))
        tokens = [view.k_codes, view.v_codes_tokens()] + arrays[2:]
        want.append([a.cpu().numpy().copy() for a in tokens])
    cache.set_position(past)
    p = np.array(path, np.int32)
    cache.keep_drafts(_device(p, cuda_device), drafted=drafted)
    for layer in range(layers):
        view = cache.view(layer)
        got = [view.k_codes, view.v_codes_tokens(), view.k_meta, view.v_meta]
        got += [view.k_qjl_bits, view.v_qjl_bits, view.k_qjl_mag, view.v_qjl_mag] if qjl else []
        for a, w in zip(got, want[layer]):
            src = w.copy()
            for i in range(b):
                w[i, :, past:past + p.shape[1]] = src[i, :, past + p[i]].transpose(1, 0, *range(2, w.ndim - 1))
            np.testing.assert_array_equal(a.cpu().numpy(), w)
    assert cache.device_status() == 0 and cache.current_position() == past
    cache.close()


def test_keep_drafts_flags_entries_outside_the_drafts(cuda_device):
    cache = _cache(1, 1, 1, 64, 4, 32, cuda_device)
    view = cache.view(0)
    view.k_codes.copy_(torch.arange(64, device=cuda_device, dtype=torch.uint8).view(1, 1, 64, 1).expand_as(view.k_codes))
    cache.set_position(4)
    cache.keep_drafts(torch.tensor([[2, 6, -1, 3]], dtype=torch.int32, device=cuda_device), drafted=6)
    assert view.k_codes[0, 0, 4:8, 0].tolist() == [6, 5, 6, 7]  # entries 1 and 2 left as they were
    assert cache.device_status(clear=True) == 2 and cache.device_status() == 0
    cache.close()


# ---- block means -----------------------------------------------------------------------------------
@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64), (3, 64), (3, 128), (4, 32), (4, 16), (8, 256), (4, 256)])
def test_block_means_are_exact(cuda_device, bits, d):
    import smallaios_b200 as sa

    b, h, blocks = 2, 3, 5
    r, kc, km, vc, vm = _random(bits * d, b, h, d, bits, blocks * 64)
    # blocks of every kind: one token outweighs the rest; zeros; values out of range; tiny; huge
    km[0, 0, 70] *= 1e6
    km[0, 1, 64:128] = 0.0
    km[0, 2, 64], km[0, 2, 65], km[0, 2, 66, 0], km[0, 2, 67, 1] = np.nan, np.inf, -np.inf, 2.0 ** 100
    km[1, 0, 64:128] *= 1e-38
    km[1, 1, 64:128] *= 1e29
    km[1, 2, 128:192, 1] = 0.0
    kc[1, 2, 128:192] = 2 ** bits - 1  # the largest sums
    km[1, 2, 128:192, 0] = np.nextafter(np.float32(1.0), np.float32(0.0))
    cache = _cache(b, h, 1, d, bits, blocks * 64, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    got = sa.kv_block_means(cache, 0, 0, blocks)
    want = ref.block_means(kc, km, 0, blocks)
    np.testing.assert_array_equal(got.double().cpu().numpy(), want)
    # a slice of a kept tensor
    kept = torch.full((b, h, blocks + 2, d), 7.0, dtype=torch.bfloat16, device=cuda_device)
    sa.kv_block_means(cache, 0, 1, 4, out=kept[:, :, 1:4])
    np.testing.assert_array_equal(kept[:, :, 1:4].double().cpu().numpy(), want[:, :, 1:4])
    assert (kept[:, :, 0] == 7).all() and (kept[:, :, 4:] == 7).all()
    assert sa.kv_block_means(cache, 0, 2, 2).shape == (b, h, 0, d)
    cache.close()


# ---- block selection ---------------------------------------------------------------------------------
SELECT = [  # d, g, dtype, b, h, past, s, k, sink, local
    (128, 4, "bf16", 2, 2, 64 * 40 + 5, 1, 8, 1, 1),
    (128, 8, "f16", 2, 1, 64 * 130, 1, 16, 1, 1),
    (64, 3, "f32", 1, 3, 64 * 70 + 60, 9, 5, 0, 2),  # the query tokens cross a block
    (128, 1, "f32", 1, 1, 64 * 300 + 1, 2, 64, 2, 3),
    (32, 2, "f32", 2, 2, 64 * 20, 3, 4, 1, 1),
    (16, 4, "f16", 2, 2, 64 * 20, 3, 4, 1, 1),
    (256, 8, "bf16", 1, 2, 64 * 33 + 2, 2, 7, 1, 1),
    (128, 4, "f32", 2, 2, 64 * 7 + 3, 1, 8, 1, 1),   # as many blocks as the list takes
    (128, 4, "f32", 2, 2, 64 * 3, 1, 8, 1, 1),       # fewer
    (128, 4, "f32", 2, 2, 0, 1, 2, 1, 1),            # the first token
    (64, 4, "f32", 1, 2, 64 * 9, 1, 1, 0, 1),        # its own block only
    (128, 4, "f32", 1, 2, 64 * 1100 + 9, 1, 33, 1, 1),
    (128, 4, "bf16", 40, 8, 64 * 127 + 63, 1, 32, 1, 1),  # more CTAs than fit at once, up to 128 blocks
    (128, 8, "bf16", 40, 8, 64 * 127 + 63, 1, 32, 1, 1),
    (64, 2, "f32", 20, 8, 64 * 60 + 62, 3, 5, 1, 2),
    (16, 1, "f16", 76, 4, 64 * 30, 1, 4, 1, 1),
    (32, 3, "f32", 76, 4, 64 * 128, 1, 4, 1, 1),          # 129 blocks
]


@pytest.mark.parametrize("d,g,dtype,b,h,past,s,k,sink,local", SELECT)
def test_select_blocks_is_exact(cuda_device, d, g, dtype, b, h, past, s, k, sink, local):
    import smallaios_b200 as sa

    r = np.random.default_rng(past + k)
    cache = _cache(b, h, g, d, 4, past + s, cuda_device)
    signs = cache.view(0).signs.cpu().numpy().astype(np.float64)
    cache.set_position(past)
    blocks = (past + s + 63) // 64
    means = (r.integers(-255, 256, (b, h, blocks, d)) * 2.0 ** r.integers(-12, -9, (b, h, blocks, 1))).astype(np.float32)
    if blocks > 12:
        means[:, :, 3:11] = means[:, :, 3:4]  # ties
    q, q64 = _query(r, b, s, h, g, d, dtype, cuda_device)
    got = sa.gqa_select_blocks(q, cache, 0, _device(means, cuda_device).bfloat16(), num_heads=h * g, max_blocks=k,
                               sink_blocks=sink, local_blocks=local)
    want = ref.select(q64, signs, means.astype(np.float64), past, k, sink, local)
    np.testing.assert_array_equal(got.cpu().numpy(), want)
    cache.close()


def test_select_blocks_edges(cuda_device):
    """All scores equal (zero queries), queries out of range, and means held in a larger tensor."""
    import smallaios_b200 as sa

    b, h, g, d, past, k = 1, 2, 4, 128, 64 * 50, 6
    r = np.random.default_rng(0)
    cache = _cache(b, h, g, d, 4, past + 1, cuda_device)
    signs = cache.view(0).signs.cpu().numpy().astype(np.float64)
    cache.set_position(past)
    means = torch.zeros(b, h, 64, d, dtype=torch.bfloat16, device=cuda_device)
    means[:, :, :51] = _device(r.integers(-255, 256, (b, h, 51, d)).astype(np.float32), cuda_device)
    sel = lambda q: sa.gqa_select_blocks(q, cache, 0, means[:, :, :51], num_heads=h * g, max_blocks=k)  # noqa: E731
    q, q64 = _query(r, b, 1, h, g, d, "f32", cuda_device)
    assert sel(torch.zeros_like(q)).tolist() == [[[[0, 1, 2, 3, 4, 50]] * h]]
    for bad in (float("nan"), float("inf"), -3e38, 1e-45):
        q[0, 0, 3 * d + 7] = bad
        q64[0, 0, 0, 3, 7] = bad
        want = ref.select(q64, signs, means.double().cpu().numpy(), past, k)
        np.testing.assert_array_equal(sel(q).cpu().numpy(), want)
    cache.close()


# ---- block-sparse attention ----------------------------------------------------------------------------
SPARSE = [  # bits, d, g, dtype, b, h, past, s, k
    (4, 128, 4, "bf16", 2, 2, 64 * 30 + 17, 1, 8),
    (4, 128, 4, "f32", 2, 2, 64 * 30 + 63, 1, 9),
    (4, 128, 8, "f16", 2, 1, 64 * 50, 1, 16),
    (4, 128, 8, "f32", 1, 2, 64 * 50 + 1, 1, 3),
    (8, 128, 4, "f32", 1, 2, 64 * 20 + 31, 1, 5),
    (8, 128, 6, "f32", 1, 2, 64 * 20 + 32, 1, 5),
    (8, 64, 3, "f32", 2, 2, 64 * 12 + 40, 30, 4),   # the query tokens cross a block
    (4, 64, 1, "f16", 2, 3, 64 * 5, 3, 2),
    (4, 64, 7, "f32", 1, 1, 64 * 9 + 5, 5, 20),     # longer lists than blocks
    (4, 128, 4, "f32", 1, 1, 0, 1, 1),              # one token
    (4, 128, 2, "f32", 20, 4, 64 * 6 + 1, 4, 3),    # more units than SMs
    (4, 64, 1, "f32", 3, 4, 10, 1400, 2),           # more query rows than one launch takes
    (3, 64, 4, "f32", 1, 2, 64 * 8 + 9, 2, 3),      # formats of the general kernel
    (4, 256, 2, "f16", 1, 2, 64 * 8 + 9, 2, 3),
    (8, 32, 8, "f32", 1, 2, 64 * 8 + 9, 2, 3),
]


def _lists(r, b, s, h, k, past):
    ids = np.full((b, s, h, k), -1, np.int32)
    for i in range(b):
        for j in range(s):
            own = (past + j) // 64
            for e in range(h):
                n = min(k, own + 1)
                rest = r.permutation(own)[:n - 1]
                ids[i, j, e, :n] = np.sort(np.append(rest, own))
    return ids


@pytest.mark.parametrize("bits,d,g,dtype,b,h,past,s,k", SPARSE)
def test_sparse_attend(cuda_device, bits, d, g, dtype, b, h, past, s, k):
    import smallaios_b200 as sa

    total = past + s
    r, kc, km, vc, vm = _random(past + s, b, h, d, bits, total)
    cache = _cache(b, h, g, d, bits, total + 70, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    view = cache.view(0)
    for meta in (view.k_meta, view.v_meta):
        meta[:, :, total:] = float("nan")  # rows past the query tokens take no part
    cache.set_position(past)
    q, q64 = _query(r, b, s, h, g, d, dtype, cuda_device)
    ids = _lists(r, b, s, h, k, past)
    out = sa.gqa_sparse_attend(q, cache, 0, _device(ids, cuda_device), num_heads=h * g)
    kk, vv = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, kk, vv, ref.sparse_sees(ids, past, total))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound(dtype, q64, kk, vv, vc, vm, want), d)
    assert cache.device_status() == 0
    cache.close()


@pytest.mark.parametrize("g,d,bits", [(4, 128, 4), (8, 128, 4), (4, 64, 8), (8, 64, 8), (8, 128, 8), (2, 64, 3)])
def test_sparse_attend_lists_of_any_shape(cuda_device, g, d, bits):
    """Empty lists, holes, ids outside the cache and blocks after the query's own position."""
    import smallaios_b200 as sa

    b, h, past, s, k = 1, 2, 64 * 10 + 20, 4, 7
    total = past + s
    r, kc, km, vc, vm = _random(11, b, h, d, bits, total)
    cache = _cache(b, h, g, d, bits, 64 * 13, cuda_device)
    signs = ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    ids = np.array([[-1] * 7, [-1, 3, -1, -1, 5, -1, 10], [2, 1 << 30, 9, -7, -1, 13, -1], [10, -1, -1, -1, -1, 12, 0]],
                   np.int32)
    ids = np.broadcast_to(ids[None, :, None, :], (b, s, h, k))
    q, q64 = _query(r, b, s, h, g, d, "f32", cuda_device)
    out = sa.gqa_sparse_attend(q, cache, 0, _device(ids, cuda_device), num_heads=h * g)
    kk, vv = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    kept = np.where((ids >= 0) & (ids <= 10), ids, -1)
    want = ref.attend(q64, kk, vv, ref.sparse_sees(kept, past, total))
    got = out.double().cpu().numpy()
    ref.assert_rows(got, want, ref.row_bound("f32", q64, kk, vv, vc, vm, want), d)
    assert (got[:, 0] == 0).all()
    cache.close()


def test_sparse_step_over_every_block_is_dense_decode(cuda_device):
    """Means kept while appending, selection and sparse attention: with room for every block, gqa_attend."""
    import smallaios_b200 as sa

    b, h, g, d, bits, past = 3, 2, 4, 128, 4, 64 * 6 + 10
    r = np.random.default_rng(1)
    cache = _cache(b, h, g, d, bits, past + 1, cuda_device)
    for count in (past, 1):
        cache.append(0, *[torch.from_numpy(r.standard_normal((b, count, h * d)).astype(np.float32)).to(cuda_device)
                          for _ in "kv"])
        if count == past:
            cache.advance_position(past)
    means = sa.kv_block_means(cache, 0, 0, past // 64)
    q, _ = _query(r, b, 1, h, g, d, "f32", cuda_device)
    ids = sa.gqa_select_blocks(q, cache, 0, means, num_heads=h * g, max_blocks=9)
    assert ids[0, 0, 0].tolist() == [0, 1, 2, 3, 4, 5, 6, -1, -1]
    out = sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g)
    want = sa.gqa_attend(q, cache, 0, num_heads=h * g, do_rotary=False)
    assert (out - want).abs().max().item() < 4e-4
    cache.close()


def test_offsets_past_32_bits(cuda_device):
    """A layer of 4.3 GB of key codes: blocks at the end of the last unit."""
    import smallaios_b200 as sa

    b, h, g, d, bits, tokens = 1, 9, 2, 128, 8, 1 << 22
    past = tokens - 100
    cache = _cache(b, h, g, d, bits, tokens, cuda_device)
    view = cache.view(0)
    lo = past - 64 * 5 - past % 64
    n = tokens - lo
    r, kc, km, vc, vm = _random(2, b, h, d, bits, n)
    view.k_codes[:, :, lo:] = _device(ref.pack(kc, bits), cuda_device)
    packed = ref.pack(vc, bits).reshape(b, h, n // 16, 4, 4, d // 4, 4).transpose(0, 1, 2, 5, 3, 6, 4)
    view.v_codes[:, :, lo // 16:] = _device(packed, cuda_device)
    view.k_meta[:, :, lo:] = _device(km.astype(np.float32), cuda_device)
    view.v_meta[:, :, lo:] = _device(vm.astype(np.float32), cuda_device)
    signs = view.signs.cpu().numpy().astype(np.float64)
    cache.set_position(past)
    first = lo // 64
    means = sa.kv_block_means(cache, 0, first, first + 5)
    np.testing.assert_array_equal(means.double().cpu().numpy(), ref.block_means(kc, km, 0, 5))
    q, q64 = _query(r, b, 2, h, g, d, "f32", cuda_device)
    ids = np.broadcast_to(np.array([first, first + 2, first + 5], np.int32), (b, 2, h, 3))
    out = sa.gqa_sparse_attend(q, cache, 0, _device(ids, cuda_device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    want = ref.attend(q64, k, v, ref.sparse_sees(ids - first, past - lo, n))
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound("f32", q64, k, v, vc, vm, want), d)
    # a tree at the end of the last head: the zeroed prefix has scores of zero and values of zero
    parents = np.array([[-1, 0]], np.int32)
    out = sa.gqa_tree_attend(q, cache, 0, _device(parents, cuda_device), num_heads=h * g)
    sees = np.repeat(ref.tree_sees(parents, past - lo)[:, :, None], h, axis=2)
    w = np.einsum("bshgd,bhtd->bshgt", q64, k[:, :, :past - lo + 2]) / np.sqrt(d)
    w = np.where(sees[:, :, :, None], np.exp(w), 0.0)
    want = np.einsum("bshgt,bhtd->bshgd", w, v[:, :, :past - lo + 2]) / (w.sum(-1, keepdims=True) + lo)
    want = want.reshape(b, 2, -1)
    ref.assert_rows(out.double().cpu().numpy(), want, ref.row_bound("f32", q64, k, v, vc, vm, want), d)
    cache.keep_drafts(torch.tensor([[1]], dtype=torch.int32, device=cuda_device), drafted=2)
    assert torch.equal(view.k_codes[:, :, past], view.k_codes[:, :, past + 1])
    cache.close()


# ---- streams, buffers, refusals --------------------------------------------------------------------------
def test_operators_on_another_stream(cuda_device):
    import smallaios_b200 as sa

    b, h, g, d, bits, past, n = 4, 4, 4, 128, 4, 64 * 20, 8
    r, kc, km, vc, vm = _random(4, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, "f32", cuda_device)
    parents = _device(_trees(r, b, n), cuda_device)

    def step(stream=None):
        means = sa.kv_block_means(cache, 0, 0, past // 64, stream=stream)
        ids = sa.gqa_select_blocks(q, cache, 0, means, num_heads=h * g, max_blocks=6, stream=stream)
        return (means, ids, sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g, stream=stream),
                sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g, stream=stream))

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(side)
    side.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)  # no order of anything changes a result
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    graph.replay()
    torch.cuda.synchronize()
    for x, y in zip(captured, want):
        assert torch.equal(x, y)
    cache.close()


def test_given_outputs_and_workspace(cuda_device):
    import smallaios_b200 as sa
    from smallaios_b200 import _lib

    b, h, g, d, bits, past, n = 2, 2, 4, 128, 4, 300, 6
    r, kc, km, vc, vm = _random(8, b, h, d, bits, past + n)
    cache = _cache(b, h, g, d, bits, past + n, cuda_device)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    q, _ = _query(r, b, n, h, g, d, "bf16", cuda_device)
    parents = _device(_trees(r, b, n), cuda_device)
    want = sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g)
    size = _lib.lib.sa_gqa_tree_workspace_bytes(cache.handle, n, _lib.SA_DTYPE_BFLOAT16)
    ws = torch.full((max(size, 256),), 255, dtype=torch.uint8, device=cuda_device)  # its contents do not matter
    out = torch.full_like(q, float("nan"))
    assert sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g, out=out, workspace=ws) is out
    assert torch.equal(out, want)
    if size:
        with pytest.raises(sa.InvalidAttribute, match="workspace of"):
            sa.gqa_tree_attend(q, cache, 0, parents, num_heads=h * g, workspace=ws[:size - 1])
    ids = _device(_lists(r, b, n, h, 3, past), cuda_device)
    want = sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g)
    size = _lib.lib.sa_gqa_sparse_workspace_bytes(cache.handle, n)
    ws = torch.full((max(size, 256),), 255, dtype=torch.uint8, device=cuda_device)
    out = torch.full_like(q, float("nan"))
    assert sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=h * g, out=out, workspace=ws) is out
    assert torch.equal(out, want)
    cache.close()


def test_no_query_tokens(cuda_device):
    import smallaios_b200 as sa

    cache = _cache(2, 2, 4, 64, 4, 64, cuda_device)
    q = torch.empty(2, 0, 512, device=cuda_device)
    assert sa.gqa_tree_attend(q, cache, 0, torch.empty(2, 0, dtype=torch.int32, device=cuda_device), num_heads=8).shape == q.shape
    means = sa.kv_block_means(cache, 0, 0, 1)
    ids = sa.gqa_select_blocks(q, cache, 0, means, num_heads=8, max_blocks=3)
    assert ids.shape == (2, 0, 2, 3)
    assert sa.gqa_sparse_attend(q, cache, 0, ids, num_heads=8).shape == q.shape
    cache.keep_drafts(torch.empty(2, 0, dtype=torch.int32, device=cuda_device), drafted=4)
    cache.close()


def test_refusals(cuda_device):
    import smallaios_b200 as sa

    dev = cuda_device
    cache = _cache(2, 2, 4, 64, 4, 200, dev)
    cache.set_position(130)
    q = torch.zeros(2, 5, 512, device=dev)
    parents = torch.zeros(2, 5, dtype=torch.int32, device=dev)
    means = torch.zeros(2, 2, 3, 64, dtype=torch.bfloat16, device=dev)
    ids = torch.zeros(2, 5, 2, 3, dtype=torch.int32, device=dev)
    tree = lambda q=q, p=parents, layer=0, heads=8, **kw: sa.gqa_tree_attend(q, cache, layer, p, num_heads=heads, **kw)  # noqa: E731
    sel = lambda q=q, m=means, k=3, **kw: sa.gqa_select_blocks(q, cache, 0, m, num_heads=8, max_blocks=k, **kw)  # noqa: E731
    att = lambda q=q, i=ids, **kw: sa.gqa_sparse_attend(q, cache, 0, i, num_heads=8, **kw)  # noqa: E731

    def refused(error, call, *a, **kw):
        with pytest.raises(error):
            call(*a, **kw)

    refused(TypeError, tree, q=q.cpu())
    refused(ValueError, tree, q=q.transpose(0, 1))
    refused(sa.ShapeMismatch, tree, q=q[0])
    refused(sa.ShapeMismatch, tree, q=q[:, :, :256].contiguous())
    refused(sa.UnsupportedOp, tree, q=q.double())
    refused(sa.UnsupportedOp, tree, p=parents.long())
    refused(sa.ShapeMismatch, tree, p=parents[:, :4].contiguous())
    refused(sa.ShapeMismatch, tree, heads=4)
    refused(sa.InvalidAttribute, tree, layer=1)
    refused(sa.ShapeMismatch, tree, out=q[:, :4].contiguous())
    refused(sa.UnsupportedOp, tree, q=torch.zeros(2, 65, 512, device=dev), p=torch.zeros(2, 65, dtype=torch.int32, device=dev))
    cache.set_position(150)
    refused(sa.CapacityError, tree, q=torch.zeros(2, 64, 512, device=dev), p=torch.zeros(2, 64, dtype=torch.int32, device=dev))
    cache.set_position(130)
    refused(sa.InvalidAttribute, sel, k=1)
    refused(sa.InvalidAttribute, sel, k=0)
    refused(sa.InvalidAttribute, sel, local_blocks=0)
    refused(sa.ShapeMismatch, sel, m=means[:, :, :1])
    refused(sa.UnsupportedOp, sel, m=means.float())
    refused(ValueError, sel, m=means.transpose(2, 3).contiguous().transpose(2, 3))
    refused(sa.ShapeMismatch, att, i=ids[:, :4].contiguous())
    refused(sa.UnsupportedOp, att, i=ids.long())
    refused(sa.InvalidAttribute, att, i=ids[..., :0].contiguous())
    refused(sa.ShapeMismatch, sa.kv_block_means, cache, 0, 0, 5)
    refused(sa.ShapeMismatch, sa.kv_block_means, cache, 0, 2, 1)
    refused(sa.InvalidAttribute, sa.kv_block_means, cache, 3, 0, 1)
    refused(sa.ShapeMismatch, sa.kv_block_means, cache, 0, 0, 2, out=means)
    path = torch.zeros(2, 3, dtype=torch.int32, device=dev)
    refused(sa.ShapeMismatch, cache.keep_drafts, path, drafted=2)
    refused(sa.UnsupportedOp, cache.keep_drafts, path, drafted=65)
    refused(sa.ShapeMismatch, cache.keep_drafts, path[:1].contiguous(), drafted=5)
    refused(sa.UnsupportedOp, cache.keep_drafts, path.long(), drafted=5)
    cache.set_position(198)
    refused(sa.CapacityError, cache.keep_drafts, path, drafted=5)
    cache.close()
    low = _cache(1, 1, 1, 64, 4, 64, dev, lowrank_k=1)
    refused(sa.UnsupportedOp, sa.kv_block_means, low, 0, 0, 1)
    refused(sa.UnsupportedOp, low.keep_drafts, torch.zeros(1, 1, dtype=torch.int32, device=dev), drafted=1)
    low.close()
