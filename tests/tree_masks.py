"""Draft trees whose drafts carry the weight: queries and drafted keys share a direction, so every draft that a node sees
has a fair part of its output, and a mask that is wrong by one draft moves the row by more than any rounding."""
import numpy as np

import tests.serving_reference as ref

# bits, d, g, dtype, b, h, past, n, shape of the tree
CASES = [
    (4, 128, 4, "bf16", 2, 2, 1000, 16, "random"),
    (4, 128, 4, "bf16", 2, 1, 120, 30, "random"),   # the drafts straddle two tiles, the rows two blocks
    (4, 64, 1, "bf16", 12, 2, 70, 2, "random"),
    (8, 128, 8, "bf16", 1, 2, 383, 64, "wide"),     # 512 rows
    (8, 64, 3, "bf16", 2, 2, 0, 21, "chain"),       # no prefix
    (4, 128, 1, "bf16", 3, 1, 255, 18, "chain"),
    (4, 64, 7, "bf16", 1, 2, 191, 19, "forest"),
    (8, 128, 2, "bf16", 2, 1, 640, 24, "holes"),
    (4, 128, 4, "f16", 2, 2, 100, 26, "random"),
    (8, 64, 8, "f16", 1, 1, 300, 40, "holes"),
    (4, 128, 4, "f32", 2, 1, 127, 33, "random"),
    (8, 128, 5, "f32", 1, 1, 500, 17, "forest"),
    (3, 64, 4, "bf16", 1, 2, 100, 12, "random"),
    (4, 256, 2, "f16", 1, 1, 90, 9, "holes"),
]
# Largest error of a row, as a part of the largest row: eight roundings of the output's type for f32 sums and the
# type itself, and for the operands' 2^-11 (bf16) or 2^-21 ten times over, the size of the scores.
TOLERANCE = {"bf16": 8 * 2.0 ** -9 + 10 * 2.0 ** -11, "f16": 8 * 2.0 ** -12 + 10 * 2.0 ** -21, "f32": 2.0 ** -16}


def parents_of(r, b, n, kind):
    """(B, N) parents: chains, forests of several roots, wide trees, trees with slots that hold no node."""
    p = np.full((b, n), -1, np.int32)
    for i in range(b):
        for j in range(1, n):
            if kind == "chain":
                p[i, j] = j - 1
            elif kind == "wide":
                p[i, j] = (j - 1) // 4
            elif kind == "forest":
                p[i, j] = -1 if j % 5 == 0 else r.integers(j - j % 5, j)
            else:
                p[i, j] = r.integers(max(-1, j - 7), j)
            if kind == "holes" and j % 6 == 4:
                p[i, j] = [-2, j, n + 3][j % 3]
    return p


def encode(x, signs, bits):
    """Codes and {scale, zero point} of vectors (B, H, T, D) in the rotated frame of the heads' signs."""
    y = ref.walsh(x * signs[None, :, None, :]) / np.sqrt(x.shape[-1])
    lo, hi = y.min(-1, keepdims=True), y.max(-1, keepdims=True)
    scale = ((hi - lo) / (2 ** bits - 1)).astype(np.float32)
    lo = lo.astype(np.float32)
    return np.clip(np.rint((y - lo) / scale), 0, 2 ** bits - 1).astype(np.int64), np.concatenate([scale, lo], -1)


def problem(case, signs):
    """Queries (B, N, H, G, D), codes and metadata of K and V, parents."""
    bits, d, g, _, b, h, past, n, kind = case
    r = np.random.default_rng(past * 64 + n)
    u = r.choice([-1.0, 1.0], (b, 1, h, 1, d))
    want = np.log(past + 1.0) + 2.0  # a draft's score above the prefix's
    q = u * (want / np.sqrt(d)) + 0.2 * r.standard_normal((b, n, h, g, d))
    k = 0.5 * r.standard_normal((b, h, past + n, d))
    k[:, :, past:] = u[:, 0].repeat(n, axis=2) + 0.1 * r.standard_normal((b, h, n, d))
    v = 0.5 * r.standard_normal((b, h, past + n, d))
    v[:, :, past:] = 4.0 * r.choice([-1.0, 1.0], (b, h, n, d))
    return (q, *encode(k, signs, bits), *encode(v, signs, bits), parents_of(r, b, n, kind))


def off(got, want, d):
    """Error of each output vector as a part of the largest one."""
    rows = lambda x: np.sqrt((x.reshape(*x.shape[:-1], -1, d) ** 2).sum(-1))  # noqa: E731
    return rows(got - want) / rows(want).max()
