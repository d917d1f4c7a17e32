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


@pytest.mark.parametrize("bad", [9, -2, 2**31 - 1])
def test_beams_that_do_not_match_stay_and_are_reported(cuda_device, bad):
    import smallaios_b200 as sa

    pool = sa.GpuKvPages(1, 1, 64, 40, bits=8, device=cuda_device)
    table = torch.arange(24, dtype=torch.int32, device=cuda_device).view(8, 3)
    before = pool.view(0).k_codes.copy_(torch.randint(0, 256, pool.view(0).k_codes.shape, device=cuda_device,
                                                      dtype=torch.uint8)).clone()
    lens = torch.full((8,), 70, dtype=torch.int32, device=cuda_device)
    parents = torch.tensor([[0, 0, 2, 3], [1, 1, 1, 1]], dtype=torch.int32, device=cuda_device)
    uneven = lens.clone()
    uneven[5] = 71
    got = pool.reorder_beams(table, uneven, parents)  # the second group's beams differ in length
    assert pool.device_status(clear=True) == 8 and torch.equal(got[4:], table[4:]) and got[1].tolist() == [0, 4, 5]
    pool.view(0).k_codes.copy_(before)
    stray = parents.clone()
    stray[0, 3] = bad                                  # a parent outside the group: that beam stays
    assert torch.equal(pool.reorder_beams(table, lens, stray), pool.reorder_beams(table, lens, parents))
    assert pool.device_status(clear=True) == 8
    broken = table.clone()
    broken[1, 1] = 40                                  # the page to copy to is outside the pool
    pool.view(0).k_codes.copy_(before)
    pool.reorder_beams(broken, lens, parents[:1].repeat(2, 1))
    assert pool.device_status(clear=True) == 2
    long = torch.full((8,), 193, dtype=torch.int32, device=cuda_device)  # more tokens than three pages hold
    assert torch.equal(pool.reorder_beams(table, long, parents), table) and pool.device_status(clear=True) == 2


def test_numbers_beyond_32_bits_are_not_cut(cuda_device):
    """An end token outside the vocabulary offers nothing, also one whose low 32 bits name a token."""
    import smallaios_b200 as sa

    x, scores = torch.zeros(4, 100, device=cuda_device), torch.zeros(1, 4, device=cuda_device)
    done = torch.ones(1, 4, dtype=torch.bool, device=cuda_device)
    for end in (-1, 100, 2**32 + 5, -2**32 + 5):
        parents, tokens, out = sa.beam_select(x, scores, finished=done, end_token=end)
        assert (parents == -1).all() and (tokens == -1).all() and (out == -float("inf")).all()
    with pytest.raises(sa.InvalidAttribute, match="keep"):
        sa.beam_select(x, scores, keep=2**32 + 4)


def test_refused_arguments(cuda_device):
    import smallaios_b200 as sa

    x = torch.zeros(8, 100, device=cuda_device)
    scores = torch.zeros(2, 4, device=cuda_device)
    done = torch.zeros(2, 4, dtype=torch.bool, device=cuda_device)
    for error, match, args, kw in (
            (sa.ShapeMismatch, "logits", (x[:7], scores), {}), (sa.ShapeMismatch, "logits", (x[0], scores), {}),
            (sa.ShapeMismatch, "logits", (x, scores[0]), {}), (sa.UnsupportedOp, "float32", (x, scores.half()), {}),
            (sa.UnsupportedOp, "dtype", (x.double(), scores), {}), (sa.UnsupportedOp, "finished", (x, scores), dict(finished=done.int())),
            (sa.ShapeMismatch, "finished", (x, scores), dict(finished=done[:1])), (ValueError, "rows", (x[:, ::2], scores), {}),
            (ValueError, "rows", (x[:1].expand(8, 100), scores), {}), (sa.InvalidAttribute, "keep", (x, scores), dict(keep=0)),
            (sa.InvalidAttribute, "keep", (x, scores), dict(keep=65)), (sa.ShapeMismatch, "rows of 0", (x[:, :0], scores), {}),
            (sa.InvalidAttribute, "33 beams", (torch.zeros(33, 9, device=cuda_device), torch.zeros(1, 33, device=cuda_device)), {}),
            (sa.InvalidAttribute, "workspace", (x, scores), dict(workspace=torch.empty(16, dtype=torch.uint8, device=cuda_device))),
            (TypeError, "logits", (x.cpu(), scores), {}), (TypeError, "scores", (x, scores.cpu()), {})):
        with pytest.raises(error, match=match):
            sa.beam_select(*args, **kw)
    assert [t.shape for t in sa.beam_select(x[:0], scores[:0])] == [(0, 4)] * 3

    pool = sa.GpuKvPages(1, 1, 64, 8, device=cuda_device)
    table = torch.zeros(8, 2, dtype=torch.int32, device=cuda_device)
    lens, parents = torch.zeros(8, dtype=torch.int32, device=cuda_device), torch.zeros(2, 4, dtype=torch.int32, device=cuda_device)
    for error, match, args, kw in (
            (sa.UnsupportedOp, "parents", (table, lens, parents.long()), {}), (sa.ShapeMismatch, "parents", (table, lens, parents[0]), {}),
            (sa.ShapeMismatch, "page_table", (table[:7], lens, parents), {}), (sa.ShapeMismatch, "entries", (table, lens[:7], parents), {}),
            (sa.ShapeMismatch, "out", (table, lens, parents), dict(out=table[:7])), (sa.UnsupportedOp, "out", (table, lens, parents), dict(out=table.long())),
            (sa.InvalidAttribute, "overlaps", (table, lens, parents), dict(out=table)),
            (sa.InvalidAttribute, "beams", (torch.zeros(33, 2, dtype=torch.int32, device=cuda_device),
                                            torch.zeros(33, dtype=torch.int32, device=cuda_device),
                                            torch.zeros(1, 33, dtype=torch.int32, device=cuda_device)), {}),
            (TypeError, "page_table", (table.cpu(), lens, parents), {})):
        with pytest.raises(error, match=match):
            pool.reorder_beams(*args, **kw)
    assert pool.reorder_beams(table[:0], lens[:0], parents[:0]).shape == (0, 2)
    wide = torch.full((8, 5), 7, dtype=torch.int32, device=cuda_device)
    pool.reorder_beams(table, lens, parents, out=wide[:, 1:3])
    assert wide.tolist() == [[7, 0, 0, 7, 7]] * 8


def test_selection_on_another_stream_and_in_a_graph(cuda_device):
    import smallaios_b200 as sa

    r = np.random.default_rng(9)
    x = torch.from_numpy((r.standard_normal((3, 32, 5000)) * 3).astype(np.float32)).to(cuda_device).bfloat16()
    scores = -torch.rand(8, 4, device=cuda_device)
    want = [sa.beam_select(t, scores, keep=6) for t in x]
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for handle in (s, s.cuda_stream):
        with torch.cuda.stream(s):
            torch.cuda._sleep(2_000_000)
        got = sa.beam_select(x[0], scores, keep=6, stream=handle)
        for _ in range(4):
            torch.full((1 << 20,), 255, dtype=torch.uint8, device=cuda_device)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
    static = x[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sa.beam_select(static, scores, keep=6)
    for t, w in zip(x, want):
        static.copy_(t)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, w))


# ---- all of it -----------------------------------------------------------------------------------------
@pytest.mark.parametrize("lift", [2.0, 9.0])  # of the end token's logits: few beams end, or most
def test_a_beam_search_over_pages(cuda_device, lift):
    """Appending, attention, selection and reordering as a serving loop runs them, against histories kept apart: every
    beam's keys and values encoded by the oracle, attention and selection in 64 bits."""
    import smallaios_b200 as sa
    from tests.helpers import oracle_append, rope_tables

    r = np.random.default_rng(10)
    b, k, h, g, d, bits, vocab, steps, end = 2, 4, 1, 2, 64, 8, 300, 75, 7
    prompt = [50, 61]
    tk, tv = (r.standard_normal((vocab, h * d)).astype(np.float32) for _ in range(2))
    tq = (r.standard_normal((vocab, h * g * d)) * 1.5).astype(np.float32)
    wout = (r.standard_normal((h * g * d, vocab)) * 1.2).astype(np.float32)
    rows = max(prompt) + steps + 1
    cos, sin = rope_tables(rows, d)
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(cuda_device)  # noqa: E731
    gk, gv, gq, gw, gcos, gsin = (dev(x) for x in (tk, tv, tq, wout, cos, sin))
    rope = dict(do_rotary=True, cos_cache=gcos, sin_cache=gsin)

    width = (rows + 63) // 64
    pool = sa.GpuKvPages(1, h, d, b * k * width, num_heads=h * g, bits=bits, device=cuda_device)
    signs = pool.view(0).signs.cpu().numpy()
    table = dev(r.permutation(b * k * width).astype(np.int32).reshape(b * k, width))
    words = [r.integers(0, vocab, n) for n in prompt]
    longest = max(prompt)
    ids = np.zeros((b * k, longest), np.int64)
    for i in range(b * k):
        ids[i, :prompt[i // k]] = words[i // k]
    counts = dev(np.repeat(prompt, k).astype(np.int32))
    lens = torch.zeros_like(counts)
    pool.append(0, gk[dev(ids)], gv[dev(ids)], table, lens, counts=counts, **rope)
    lens += counts

    # what a token at a position holds, as the oracle encodes it
    held = {}

    def vectors(token, pos):
        if (token, pos) not in held:
            kc, km, vc, vm = oracle_append(tk[token].reshape(1, 1, h, d), tv[token].reshape(1, 1, h, d), signs, bits, pos, cos, sin,
                                           do_rotary=True)
            held[token, pos] = [ref.decode(ref.unpack(c, bits, d), m, signs.astype(np.float64))[0, :, 0] for c, m in ((kc, km), (vc, vm))]
        return held[token, pos]

    hist = [[list(words[i]) for _ in range(k)] for i in range(b)]
    scores = np.full((b, k), -np.inf, np.float32)
    scores[:, 0] = 0.0
    tokens = np.array([[w[-1]] * k for w in words])  # the first new token repeats the prompt's last one
    finished = np.zeros((b, k), bool)
    ended = 0
    for step in range(steps):
        tok = dev(tokens.reshape(-1))
        pool.append(0, gk[tok][:, None], gv[tok][:, None], table, lens, **rope)
        attn = sa.gqa_paged_attend(gq[tok][:, None].contiguous(), pool, 0, table, lens, num_heads=h * g, **rope)
        logits = attn[:, 0] @ gw
        logits[:, end] += lift
        got = [x.cpu().numpy() for x in sa.beam_select(logits, dev(scores), finished=dev(finished), end_token=end)]
        lens += 1
        table = pool.reorder_beams(table, lens, dev(got[0]))

        want_logits = np.zeros((b, k, vocab))
        for i in range(b):
            for j in range(k):
                hist[i][j].append(int(tokens[i, j]))
                n = len(hist[i][j])
                kv = [vectors(t, p) for p, t in enumerate(hist[i][j])]
                q = pr.rotate(tq[tokens[i, j]].reshape(h, g, d), n - 1, cos, sin, False)
                w = np.einsum("hgd,thd->hgt", q, np.stack([x[0] for x in kv])) / np.sqrt(d)
                w = np.exp(w - w.max(-1, keepdims=True))
                o = np.einsum("hgt,thd->hgd", w / w.sum(-1, keepdims=True), np.stack([x[1] for x in kv]))
                want_logits[i, j] = o.reshape(-1) @ wout
                want_logits[i, j, end] += lift
        want = _select(want_logits, scores, finished, end, k)
        # attention is off by 1e-5 at most, a logit by that times the norm of a column of wout
        live = want[2] > -np.inf
        assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1]), step
        assert np.abs(got[2][live] - want[2][live]).max() < 1e-3
        parents = np.where(got[0] < 0, np.arange(k), got[0])
        hist = [[list(hist[i][p]) for p in parents[i]] for i in range(b)]
        scores, tokens, finished = got[2], np.maximum(got[1], 0), got[1] == end
        ended += int(finished.sum())
    assert pool.device_status() == 0 and (lift < 5 or ended > 0)
