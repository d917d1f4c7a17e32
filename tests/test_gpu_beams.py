"""Beam search on the GPU: selection over beams and vocabulary, and the beams' pages, against plain forms."""
import numpy as np
import pytest
import torch

import tests.pages_reference as pr
import tests.serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- selection --------------------------------------------------------------------------------------
def _select(logits, scores, finished, end, keep):
    """(parents, tokens, scores) in 64 bits; logits (B, K, V)."""
    b, k, v = logits.shape
    parents, tokens = np.full((2, b, keep), -1, np.int64)
    out = np.full((b, keep), -np.inf)
    with np.errstate(all="ignore"):
        for i in range(b):
            x = logits[i].astype(np.float64)
            top = x.max(-1, keepdims=True)
            x = x - (top + np.log(np.exp(x - top).sum(-1, keepdims=True)))
            x = x + scores[i].astype(np.float64)[:, None]
            for j in range(k):
                if finished is not None and finished[i, j]:
                    x[j] = -np.inf
                    if 0 <= end < v:
                        x[j, end] = scores[i, j]
            x = np.where(np.isnan(x), -np.inf, x).ravel()
            order = np.lexsort((np.arange(k * v), -x))[:keep]
            order = order[x[order] > -np.inf]
            n = len(order)
            parents[i, :n], tokens[i, :n], out[i, :n] = order // v, order % v, x[order]
    return parents, tokens, out


def _run(logits, scores, finished, end, keep, device):
    """logits (B, K, V) tensor."""
    import smallaios_b200 as sa

    b, k, v = logits.shape
    got = sa.beam_select(logits.reshape(b * k, v).to(device), torch.from_numpy(scores).to(device),
                         finished=None if finished is None else torch.from_numpy(finished).to(device), end_token=end, keep=keep)
    return [x.cpu().numpy() for x in got]


def _same(got, want, logits, scores):
    """Places are equal; a score is off by the rounding of the result to f32, and by the logarithm's error: sums of
    exponentials that are off by a relative 2^-21 each at most (the instruction and its rounded argument)."""
    assert np.array_equal(got[0], want[0])
    assert np.array_equal(got[1], want[1])
    lost = want[2] == -np.inf
    assert np.array_equal(got[2] == -np.inf, lost)
    off = np.abs(got[2].astype(np.float64)[~lost] - want[2][~lost])
    assert (off <= 2.0 ** -24 * np.abs(want[2][~lost]) + 2.0 ** -21).all()


@pytest.mark.parametrize("b,k,v,keep,dtype,done", [
    (1, 4, 32000, 4, "f32", False),
    (3, 5, 50257, 10, "f16", True),
    (7, 8, 1000, 8, "bf16", True),
    (2, 1, 255, 1, "f32", False),
    (2, 1, 7, 3, "bf16", False),
    (40, 3, 1, 3, "f16", False),     # one token: as many continuations as beams
    (2, 2, 2, 9, "f32", True),       # fewer continuations than asked for
    (1, 32, 4099, 64, "bf16", True),
    (2, 16, 777, 64, "f32", False),
    (150, 2, 513, 4, "f16", False),
])
def test_selection_matches_the_plain_form(cuda_device, b, k, v, keep, dtype, done):
    r = np.random.default_rng(b * 1000 + v)
    logits = torch.from_numpy((r.standard_normal((b, k, v)) * 3).astype(np.float32)).to(DT[dtype])
    scores = (-np.cumsum(r.random((b, k)), 1) * 2).astype(np.float32)
    finished = r.random((b, k)) < 0.3 if done else None
    want = _select(logits.double().numpy(), scores, finished, 1, keep)
    _same(_run(logits, scores, finished, 1, keep, cuda_device), want, logits, scores)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_selection_of_equal_scores_takes_the_lowest(cuda_device, dtype):
    """Constant rows, equal beams, and plateaus that cross groups."""
    r = np.random.default_rng(5)
    for v, keep in ((3000, 20), (600, 64), (5, 12)):
        x = np.zeros((4, 3, v), np.float32)
        x[1] = r.integers(0, 3, v)                  # three equal beams with many equal tokens
        x[2, 1:] = -1.5
        x[3, :, v // 2:] = 2.0
        scores = np.zeros((4, 3), np.float32)
        scores[3] = [-1, 0, -1]
        logits = torch.from_numpy(x).to(DT[dtype])
        want = _select(logits.double().numpy(), scores, None, -1, keep)
        _same(_run(logits, scores, None, -1, keep, cuda_device), want, logits, scores)


def test_selection_with_masked_tokens_infinities_and_nan(cuda_device):
    r = np.random.default_rng(6)
    v = 1300
    x = (r.standard_normal((8, 4, v)) * 2).astype(np.float32)
    low = np.finfo(np.float32).min
    x[0, :, 5:] = -np.inf                            # five tokens are left
    x[1] = -np.inf                                   # none is
    x[2, 1] = -np.inf                                # one beam has none
    x[3, 2, 77] = np.nan
    x[4, 0, 1299] = np.inf
    x[5] = low                                       # the type's lowest value, everywhere
    x[6, :, 3:] = low
    x[7, :, ::2] = -np.inf
    scores = (-r.random((8, 4))).astype(np.float32)
    scores[7] = [-np.inf, 0.5, np.nan, -np.inf]      # beams without a score offer nothing
    logits = torch.from_numpy(x)
    for finished, end in ((None, -1), (r.random((8, 4)) < 0.4, 9), (np.ones((8, 4), bool), v), (np.ones((8, 4), bool), v - 1)):
        want = _select(x, scores, finished, end, 24)
        _same(_run(logits, scores, finished, end, 24, cuda_device), want, logits, scores)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_selection_over_slices_of_wider_rows(cuda_device, dtype):
    """Rows that begin and end at any element."""
    import smallaios_b200 as sa

    r = np.random.default_rng(7)
    for first, v, width in ((1, 513, 521), (3, 1000, 1003), (7, 250, 264), (0, 8, 9), (5, 2, 7)):
        wide = torch.from_numpy((r.standard_normal((6, width)) * 3).astype(np.float32)).to(DT[dtype])
        wide[:, :first] = 50.0
        wide[:, first + v:] = float("nan")
        scores = -r.random((2, 3)).astype(np.float32)
        x = wide[:, first:first + v]
        want = _select(x.double().numpy().reshape(2, 3, v), scores, None, -1, 5)
        got = sa.beam_select(wide.to(cuda_device)[:, first:first + v], torch.from_numpy(scores).to(cuda_device), keep=5)
        _same([t.cpu().numpy() for t in got], want, x, scores)


# ---- the beams' pages ---------------------------------------------------------------------------------
def _reorder(table, arrays, parents, n):
    """One group: table (K, W), arrays of (P, H, 64, X) per layer (tokens in order).  In place on copies."""
    k, w = table.shape
    full, fill = divmod(n, pr.PAGE)
    p = [x if x != -1 else i for i, x in enumerate(parents)]
    out = table.copy()
    out[:, :full] = table[p, :full]
    children = {x: [i for i in range(k) if p[i] == x] for x in range(k)}
    free = [x for x in range(k) if not children[x]]
    if fill:
        for i in range(k):
            heir = p[i] if p[i] in children[p[i]] else children[p[i]][0]
            if heir == i:
                out[i, full] = table[p[i], full]
            else:
                page = table[free.pop(0), full]
                out[i, full] = page
                for layer in arrays:
                    for a in layer:
                        a[page, :, :fill] = a[table[p[i], full], :, :fill]
    return out


def _tokens(view):
    return [x.cpu().numpy().copy() for x in (view.k_codes, view.v_codes_tokens(), view.k_meta, view.v_meta)]


@pytest.mark.parametrize("layers,b,k,h,d,bits,lens,width", [
    (2, 1, 4, 2, 64, 8, [200], 5),
    (1, 3, 8, 3, 128, 4, [64, 1, 129], 4),
    (3, 2, 32, 1, 64, 4, [63, 127], 2),
    (1, 5, 3, 2, 128, 8, [0, -1, 5, 300, 66], 6),
    (1, 1, 1, 1, 64, 4, [70], 2),
    (2, 17, 5, 1, 128, 4, list(range(60, 77)), 3),
])
def test_reorder_matches_the_plain_form(cuda_device, layers, b, k, h, d, bits, lens, width):
    import smallaios_b200 as sa

    r = np.random.default_rng(layers * 100 + b * 10 + k)
    pages = b * k * width + 2
    pool = sa.GpuKvPages(layers, h, d, pages, bits=bits, device=cuda_device)
    for i in range(layers):
        view = pool.view(i)
        for x in (view.k_codes, view.v_codes):
            x.copy_(torch.randint(0, 256, x.shape, device=cuda_device, dtype=torch.uint8))
        for x in (view.k_meta, view.v_meta):
            x.copy_(torch.randn(x.shape, device=cuda_device))
    table = r.permutation(pages)[:b * k * width].astype(np.int32).reshape(b * k, width)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda_device).repeat_interleave(k)
    current = torch.from_numpy(table).to(cuda_device)
    arrays = [_tokens(pool.view(i)) for i in range(layers)]
    for turn in range(4):  # several steps, one on the other's table
        parents = r.integers(-1, k, (b, k)).astype(np.int32)
        if turn == 2:
            parents[:] = r.integers(0, k)  # one beam goes on in all slots
        want = table.copy()
        for i in range(b):
            if lens[i] > 0:
                want[i * k:(i + 1) * k] = _reorder(table[i * k:(i + 1) * k], arrays, parents[i], lens[i])
        current = pool.reorder_beams(current, ln, torch.from_numpy(parents).to(cuda_device))
        assert pool.device_status() == 0
        assert np.array_equal(current.cpu().numpy(), want)
        table = want
        for i in range(layers):
            for got, x in zip(_tokens(pool.view(i)), arrays[i]):
                assert np.array_equal(got, x)
