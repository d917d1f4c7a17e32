"""Which drafts each node of a tree sees, on trees whose drafts carry the weight (tests/tree_masks.py)."""
import numpy as np
import pytest
import torch

import tests.serving_reference as ref
from tests import tree_masks as tm
from tests.test_gpu_serving import DT, _cache, _device

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("case,full", [(c, f) for c in tm.CASES for f in ((False, True) if c[3] == "bf16" else (False,))],
                         ids=str)
def test_each_node_sees_its_path(cuda_device, case, full):
    import smallaios_b200 as sa

    bits, d, g, dtype, b, h, past, n, _ = case
    cache = _cache(b, h, g, d, bits, past + n + 3, cuda_device)
    signs = cache.view(0).signs.double().cpu().numpy()
    q, kc, km, vc, vm, parents = tm.problem(case, signs)
    ref.fill_cache(cache, 0, kc, km, vc, vm)
    cache.set_position(past)
    cache.set_tree_precision(full)
    qd = torch.from_numpy(q.reshape(b, n, h * g * d)).to(DT[dtype])
    out = sa.gqa_tree_attend(qd.to(cuda_device), cache, 0, _device(parents, cuda_device), num_heads=h * g)
    k, v = ref.decode(kc, km, signs), ref.decode(vc, vm, signs)
    sees = np.repeat(ref.tree_sees(parents, past)[:, :, None], h, axis=2)
    want = ref.attend(qd.double().numpy().reshape(q.shape), k, v, sees)
    got = out.double().cpu().numpy()
    assert tm.off(got, want, d).max() < tm.TOLERANCE[dtype]
    assert (got[~sees.any(-1)[:, :, 0]] == 0).all()
    cache.close()
