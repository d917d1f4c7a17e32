"""Plain 64-bit forms of the serving operators (draft trees, block means, block selection, block-sparse
attention) on the host, from a cache's arrays, and the error bound of the attention kernels."""
from __future__ import annotations

import numpy as np

BLOCK = 64


def unpack(codes: np.ndarray, bits: int, d: int) -> np.ndarray:
    """(..., CB) packed bytes -> (..., D) codes: a little-endian stream of `bits`-bit numbers."""
    stream = np.unpackbits(codes, axis=-1, bitorder="little").reshape(*codes.shape[:-1], d, bits)
    return (stream.astype(np.int64) << np.arange(bits)).sum(-1)


def pack(c: np.ndarray, bits: int) -> np.ndarray:
    stream = ((c[..., None] >> np.arange(bits)) & 1).astype(np.uint8)
    return np.packbits(stream.reshape(*c.shape[:-1], -1), axis=-1, bitorder="little")


def walsh(x: np.ndarray) -> np.ndarray:
    d = x.shape[-1]
    h = np.array([[1.0]])
    while h.shape[0] < d:
        h = np.block([[h, h], [h, -h]])
    return x @ h


def random_vectors(r, shape, bits):
    """Codes (B, H, T, D) and {scale, zero point} (B, H, T, 2) of quantized Gaussian vectors."""
    x = r.standard_normal(shape)
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    scale = ((hi - lo) / (2 ** bits - 1)).astype(np.float32)
    lo = lo.astype(np.float32)
    c = np.clip(np.rint((x - lo) / scale), 0, 2 ** bits - 1).astype(np.int64)
    return c, np.concatenate([scale, lo], -1)


def fill_cache(cache, layer, kc, km, vc, vm):
    """Codes (B, H, T, D) and metadata (B, H, T, 2) of tokens [0, T) into a cache's arrays."""
    import torch

    view = cache.view(layer)
    b, h, t, _ = kc.shape
    cap, cb = view.k_codes.shape[2], view.k_codes.shape[3]
    dev = view.k_codes.device
    kp, vp = (np.zeros((b, h, cap, cb), np.uint8) for _ in range(2))
    kp[:, :, :t], vp[:, :, :t] = pack(kc, view.bits), pack(vc, view.bits)
    view.k_codes.copy_(torch.from_numpy(kp).to(dev))
    blocks = vp.reshape(b, h, cap // 16, 4, 4, cb // 4, 4).transpose(0, 1, 2, 5, 3, 6, 4)
    view.v_codes.copy_(torch.from_numpy(np.ascontiguousarray(blocks)).to(dev))
    view.k_meta[:, :, :t].copy_(torch.from_numpy(km.astype(np.float32)).to(dev))
    view.v_meta[:, :, :t].copy_(torch.from_numpy(vm.astype(np.float32)).to(dev))
    return view.signs.cpu().numpy().astype(np.float64)


def decode(c, meta, signs):
    """The vectors (B, H, T, D) that codes stand for; signs (H, D)."""
    meta = meta.astype(np.float32).astype(np.float64)
    x = c * meta[..., :1] + meta[..., 1:]
    return walsh(x) * signs[None, :, None, :] / np.sqrt(c.shape[-1])


def attend(q, k, v, sees, scale=None):
    """q (B, S, H, G, D), k / v (B, H, T, D), sees (B, S, H, T) -> (B, S, H*G*D); empty rows are zero.
    Tokens that a row does not see take no part, whatever their vectors hold."""
    b, s, h, g, d = q.shape
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out = np.zeros((b, s, h, g, d))
    for i in range(b):
        for j in range(s):
            for e in range(h):
                at = np.flatnonzero(sees[i, j, e])
                if not len(at):
                    continue
                w = q[i, j, e] @ k[i, e, at].T * scale
                w = np.exp(w - w.max(-1, keepdims=True))
                out[i, j, e] = (w / w.sum(-1, keepdims=True)) @ v[i, e, at]
    return out.reshape(b, s, h * g * d)


def tree_sees(parents, past):
    """(B, N, past + N): node i sees the prefix, its ancestors and itself; absent nodes see nothing."""
    b, n = parents.shape
    sees = np.zeros((b, n, past + n), bool)
    for i in range(b):
        present = np.zeros(n, bool)
        for j in range(n):
            p = parents[i, j]
            present[j] = p == -1 or (0 <= p < j and present[p])
            if present[j]:
                if p >= 0:
                    sees[i, j] = sees[i, p]
                else:
                    sees[i, j, :past] = True
                sees[i, j, past + j] = True
    return sees


def sparse_sees(ids, pos0, total):
    """ids (B, S, H, k) -> (B, S, H, total)."""
    b, s, h, _ = ids.shape
    sees = np.zeros((b, s, h, total), bool)
    for i in range(b):
        for j in range(s):
            for e in range(h):
                for x in ids[i, j, e]:
                    if x >= 0:
                        sees[i, j, e, x * BLOCK:(x + 1) * BLOCK] = True
                sees[i, j, e, pos0 + j + 1:] = False
    return sees


def _exponent(x):
    """Least e >= -100 with x < 2^e."""
    return max(-100, int(np.frexp(np.float64(x))[1])) if x > 0 else -100


def _grid(x):
    x = np.asarray(x, np.float64)
    with np.errstate(invalid="ignore"):
        return np.where(np.abs(x) < 2.0 ** 100, x, 0.0)


def block_means(c, meta, lo, hi):
    """c (B, H, T, D), meta (B, H, T, 2) -> (B, H, hi - lo, D) by the whole-number definition."""
    b, h, _, d = c.shape
    out = np.zeros((b, h, hi - lo, d))
    for i in range(b):
        for e in range(h):
            for n in range(lo, hi):
                at = slice(n * BLOCK, (n + 1) * BLOCK)
                m = _grid(meta[i, e, at].astype(np.float32))
                x = _exponent(np.abs(m).max())
                g = np.rint(m * 2.0 ** (15 - x)).astype(np.int64)
                total = (g[:, :1] * c[i, e, at]).sum(0) + g[:, 1].sum()
                drop = max(0, int(np.abs(total).max()).bit_length() - 8)
                out[i, e, n - lo] = ((total + ((1 << drop) >> 1)) >> drop) * 2.0 ** (drop + x - 21)
    return out


def select(q, signs, means, pos0, k, sink=1, local=1):
    """q (B, S, H, G, D), means (B, H, blocks, D) -> ids (B, S, H, k)."""
    b, s, h, _, _ = q.shape
    ids = np.full((b, s, h, k), -1, np.int64)
    for i in range(b):
        for j in range(s):
            own = (pos0 + j) // BLOCK
            for e in range(h):
                x = _grid(q[i, j, e])
                n = np.rint(x * 2.0 ** (12 - _exponent(np.abs(x).max())))
                r = walsh(n * signs[e])
                drop = max(0, int(np.abs(r).max()).bit_length() - 7)
                r8 = np.clip(np.rint(r / 2.0 ** drop), -127, 127)
                score = {}
                for a in range(own + 1):
                    forced = a < sink or a > own - local
                    score[a] = np.inf if forced else (r8 @ means[i, e, a]).max()
                best = sorted(score, key=lambda a: (-score[a], a))[:k]
                ids[i, j, e, :len(best)] = sorted(best)
    return ids


# unit roundoff of the outputs' types, and what the operands of the products may lose
ROUND = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
OPERAND = {"f32": 2.0 ** -21, "f16": 2.0 ** -21, "bf16": 2.0 ** -11}


def row_bound(dtype, q, k, v, vc, vm, want, scale=None):
    """Bound on the 2-norm of the error of each output vector (D values).

    With operands that lose a relative eps (16 bits of significand: bf16 callers get one fp16 plane, others
    two) a score moves by at most eps |q||k| scale, a weight by a relative 2 eps |q||k| scale, the output by
    that times max|v|; the weights' own rounding adds eps times the sum's terms vs|c|, twice (numerator and
    denominator).  f32 arithmetic adds 2^-20 to eps; the output's rounding is relative to it.
    """
    d = q.shape[-1]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    norm = lambda x: np.nanmax(np.where(np.isfinite(x), x, np.nan))  # noqa: E731
    with np.errstate(invalid="ignore", over="ignore"):
        qn, kn, vn = (norm(np.sqrt((x * x).sum(-1))) for x in (q, k, v))
        cn = norm(vm[..., 0].astype(np.float64) * np.sqrt((vc * vc).sum(-1)))
    eps = OPERAND[dtype] + 2.0 ** -20
    rows = np.sqrt((want.reshape(*want.shape[:-1], -1, d) ** 2).sum(-1))
    return eps * (2 * qn * kn * abs(scale) * vn + 2 * (cn + vn)) + ROUND[dtype] * rows


def assert_rows(got, want, bound, d):
    off = np.sqrt(((got - want).reshape(*want.shape[:-1], -1, d) ** 2).sum(-1))
    assert np.isfinite(got).all(), "not finite"
    bad = off > bound
    assert not bad.any(), f"{int(bad.sum())} of {bad.size} rows off by up to {off[bad].max():.3e} (bound {bound[bad].max():.3e})"
