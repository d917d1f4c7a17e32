"""The tolerance of the tree-mask tests rejects every mask that is wrong by a single draft (plain form, no GPU)."""
import numpy as np
import pytest

import tests.serving_reference as ref
from tests import tree_masks as tm


def _wrong(sees, past, how):
    """A mask that errs, and the rows (B, N) that it errs in."""
    x = sees.copy()
    drafts = x[:, :, past:]
    b, n = x.shape[:2]
    present = sees.any(-1)
    for i in range(b):
        for j in range(n):
            if not present[i, j]:
                continue
            seen = np.flatnonzero(sees[i, j, past:])
            unseen = np.setdiff1d(np.arange(n), seen)
            if how == "drop an ancestor" and len(seen) > 1:
                drafts[i, j, seen[(i + j) % (len(seen) - 1)]] = False
            elif how == "drop itself" and len(seen) > 1:
                drafts[i, j, j] = False
            elif how == "add one" and len(unseen):
                drafts[i, j, unseen[(i + j) % len(unseen)]] = True
            elif how == "every draft":
                drafts[i, j] = True
            elif how == "causal":
                drafts[i, j, :j + 1] = True
    return x, (x != sees).any(-1)


@pytest.mark.parametrize("how", ["drop an ancestor", "drop itself", "add one", "every draft", "causal"])
@pytest.mark.parametrize("case", tm.CASES, ids=str)
def test_a_wrong_mask_is_out_of_tolerance(case, how):
    bits, d, g, dtype, b, h, past, n, kind = case
    signs = np.random.default_rng(7).choice([-1.0, 1.0], (h, d))
    q, kc, km, vc, vm, parents = tm.problem(case, signs)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = ref.tree_sees(parents, past)
    wrong, rows = _wrong(sees, past, how)
    if not rows.any():
        assert kind == "chain" and how == "causal"
        return
    plain = [ref.attend(q, k, v, np.repeat(m[:, :, None], h, axis=2)) for m in (sees, wrong)]
    assert tm.off(plain[1], plain[0], d)[rows].min() > 2 * tm.TOLERANCE[dtype]
