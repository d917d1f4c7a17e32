"""Plain forms of paged serving on the host: sequences in pages, and the error bound of attention over pages."""
from __future__ import annotations

import numpy as np

import tests.serving_reference as ref

PAGE = 64
ROUND = ref.ROUND


def tables(r, needs, width=None, spare=3):
    """(pages in the pool, (B, width) int32 table): distinct random pages for each row's `needs[b]` tokens; -1 behind."""
    pages = [(n + PAGE - 1) // PAGE for n in needs]
    width = max(pages) if width is None else width
    total = sum(pages) + spare
    order = r.permutation(total).astype(np.int32)
    table = np.full((len(needs), width), -1, np.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = order[at:at + n]
        at += n
    return total, table


def fill(view, kc, km, vc, vm):
    """Codes (P, H, 64, D) and metadata (P, H, 64, 2) into a layer's pages; the signs (H, D)."""
    import torch

    p, h, t, d = kc.shape
    dev = view.k_codes.device
    to = lambda x: torch.from_numpy(np.ascontiguousarray(x)).to(dev)  # noqa: E731
    view.k_codes.copy_(to(ref.pack(kc, view.bits)))
    vp = ref.pack(vc, view.bits)
    cb = vp.shape[-1]
    view.v_codes.copy_(to(vp.reshape(p, h, 4, 4, 4, cb // 4, 4).transpose(0, 1, 2, 5, 3, 6, 4)))
    view.k_meta.copy_(to(km.astype(np.float32)))
    view.v_meta.copy_(to(vm.astype(np.float32)))
    return view.signs.cpu().numpy().astype(np.float64)


def tokens_of(a, row, n):
    """(P, H, 64, X) -> (H, n, X): the first n tokens of a table row."""
    pages = row[:(n + PAGE - 1) // PAGE]
    return a[pages].transpose(1, 0, 2, 3).reshape(a.shape[1], -1, a.shape[3])[:, :n]


def rotate(x, pos, cos, sin, interleaved):
    """Rotary embedding of (..., D) at one position, in 64 bits."""
    x, c, s = x.astype(np.float64), cos[pos].astype(np.float64), sin[pos].astype(np.float64)
    d = x.shape[-1]
    a, b = (np.s_[..., 0::2], np.s_[..., 1::2]) if interleaved else (np.s_[..., :d // 2], np.s_[..., d // 2:])
    y = np.empty_like(x)
    y[a], y[b] = c * x[a] - s * x[b], s * x[a] + c * x[b]
    return y


def attend(q, kc, km, vc, vm, signs, table, lens, bits, scale=None):
    """q (B, S, H, G, D) rotated; lens (B, S) tokens each query token sees.  -> outputs and bounds (B, S, H, G, ...)."""
    b, s, h, g, d = q.shape
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out = np.zeros((b, s, h, g, d))
    size = np.zeros((b, s, h, 4))  # |k|, |v|, the largest value scale, |c - middle|
    mid = 8 if bits == 4 else 128
    for i in range(b):
        n = int(lens[i].max())
        if n == 0:
            continue
        kt, vt, kmt, vmt = (tokens_of(a, table[i], n) for a in (kc, vc, km, vm))
        k = ref.decode(kt[None], kmt[None], signs)[0]
        v = ref.decode(vt[None], vmt[None], signs)[0]
        for j in range(s):
            m = int(lens[i, j])
            if m == 0:
                continue
            w = np.einsum("hgd,htd->hgt", q[i, j], k[:, :m]) * scale
            w = np.exp(w - w.max(-1, keepdims=True))
            out[i, j] = np.einsum("hgt,htd->hgd", w / w.sum(-1, keepdims=True), v[:, :m])
            norm = lambda x: np.sqrt((x * x).sum(-1)).max(-1)  # noqa: E731
            size[i, j] = np.stack([norm(k[:, :m]), norm(v[:, :m]), np.abs(vmt[:, :m, 0]).max(-1),
                                   norm(vt[:, :m] - float(mid))], -1)
    return out, size


def bound(dtype, q, size, want, scale=None):
    """Bound on the 2-norm of the error of each output vector.

    The query's digits are off by half a step of max|q'| / Q (Q = 32639 or 8355711) in each of D dimensions, so
    a score by e_q |q||k| scale with e_q = sqrt(D) / (2 Q), a weight by a relative 2 e_q |q||k| scale, and the output
    by that times max|v|.  A weight's digit is off by half a step of its chunk's largest weight times value scale
    (U = 65535 or 2^24 - 1); over the up to 64 tokens of a chunk, and the chunks' largest weights adding up to no more
    than the sum of all, that moves the output by (32 / U) max vs max|c - middle|.  f32 arithmetic of scores and
    sums adds 2^-20 |q||k| scale to a score, and 2^-19 |v|.
    """
    d = q.shape[-1]
    scale = 1.0 / np.sqrt(d) if scale is None else abs(scale)
    steps, top = (8355711, 2.0 ** 24 - 1) if dtype == "f32" else (32639, 65535.0)
    qn = np.sqrt((q * q).sum(-1))  # (B, S, H, G)
    kn, vn, vs, cn = (size[..., None, x] for x in range(4))
    e_q = np.sqrt(d) / (2 * steps) + 2.0 ** -20
    rows = np.sqrt((want * want).sum(-1))
    return 2 * e_q * qn * kn * scale * vn + 32 / top * vs * cn + 2.0 ** -19 * vn + ROUND[dtype] * rows


def check(got, want, limit):
    assert np.isfinite(got).all(), "not finite"
    off = np.sqrt(((got - want) ** 2).sum(-1))
    bad = off > limit
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} rows off by up to {off[bad].max():.3e} (bound {limit[bad].max():.3e})"
