"""Attention of rows that share pages: beams after a reordering, and prompts in common, at sizes where ranges cross rows."""
import numpy as np
import pytest
import torch

import tests.pages_reference as pr
import tests.serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits,d,h,g", [(4, 128, 2, 4), (8, 128, 1, 8), (8, 64, 2, 2)])
@pytest.mark.parametrize("common", [0, 3, 40])  # pages
def test_rows_that_share_pages(cuda_device, bits, d, h, g, dtype, common):
    """Two groups of five beams: a common prompt, then pages of their own of several lengths.  The last beam of a group is
    its first one's twin, all pages and the query included: within the bound, since ranges cut the two apart elsewhere."""
    import smallaios_b200 as sa

    r = np.random.default_rng(common + d)
    k, own = 5, [70, 1, 64, 130, 70]
    b, width = 2 * k, common + 3
    total = 2 * common + 6 * k + 1
    ids = r.permutation(total).astype(np.int32)
    table = np.full((b, width), -1, np.int32)
    lens = np.zeros(b, np.int64)
    for i in range(b):
        table[i, :common] = ids[(i // k) * common:(i // k + 1) * common]
        table[i, common:] = ids[2 * common + 3 * i:2 * common + 3 * i + 3]
        lens[i] = 64 * common + own[i % k]
    table[4], table[9] = table[0], table[5]  # the last beam is the first one's twin
    kc, km = ref.random_vectors(r, (total, h, pr.PAGE, d), bits)
    vc, vm = ref.random_vectors(r, (total, h, pr.PAGE, d), bits)
    pool = sa.GpuKvPages(1, h, d, total, num_heads=h * g, bits=bits, device=cuda_device)
    signs = pr.fill(pool.view(0), kc, km, vc, vm)
    q = (r.standard_normal((b, 1, h * g * d)) * 1.3).astype(np.float32)
    q[4], q[9] = q[0], q[5]
    q = torch.from_numpy(q).to(DT[dtype])
    qr = q.double().numpy().reshape(b, 1, h, g, d)
    want, size = pr.attend(qr, kc, km, vc, vm, signs, table, lens[:, None], bits)
    got = sa.gqa_paged_attend(q.to(cuda_device), pool, 0, torch.from_numpy(table).to(cuda_device),
                              torch.from_numpy((lens - 1).astype(np.int32)).to(cuda_device), num_heads=h * g)
    assert pool.device_status() == 0
    pr.check(got.double().cpu().numpy().reshape(want.shape), want, pr.bound(dtype, qr, size, want))
