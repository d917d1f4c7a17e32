"""Attention over pages: the position that a query is rotated to, for rows with more tokens than their tables have pages."""
import numpy as np
import pytest
import torch

import tests.pages_reference as pr
import tests.serving_reference as ref
from tests.helpers import rope_tables

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_queries_behind_their_tables_are_rotated_to_their_own_positions(cuda_device, interleaved, dtype):
    """Tokens without a page are not attended to; the query stays where it is.  Rows that end at, before and far behind
    their table's last token, several new tokens each."""
    import smallaios_b200 as sa

    r = np.random.default_rng(11)
    bits, d, h, g, s = 4, 128, 2, 3, 4
    lens, width = [126, 200, 100, 124, -1], 2
    b, most = len(lens), 64 * width
    pages, table = pr.tables(r, [most] * b)
    kc, km = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    vc, vm = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    pool = sa.GpuKvPages(1, h, d, pages, num_heads=h * g, bits=bits, device=cuda_device)
    signs = pr.fill(pool.view(0), kc, km, vc, vm)
    cos, sin = rope_tables(300, d)
    q = torch.from_numpy((r.standard_normal((b, s, h * g * d)) * 1.3).astype(np.float32)).to(DT[dtype])
    qr = q.double().numpy().reshape(b, s, h, g, d).copy()
    sees = np.zeros((b, s), np.int64)
    for i in range(b):
        for j in range(s):
            if lens[i] >= 0:
                sees[i, j] = min(lens[i] + j + 1, most)
                qr[i, j] = pr.rotate(qr[i, j], lens[i] + j, cos, sin, interleaved)
    want, size = pr.attend(qr, kc, km, vc, vm, signs, table, sees, bits)
    dev = lambda x: torch.from_numpy(x).to(cuda_device)  # noqa: E731
    got = sa.gqa_paged_attend(q.to(cuda_device), pool, 0, dev(table), torch.tensor(lens, dtype=torch.int32, device=cuda_device),
                              num_heads=h * g, do_rotary=True, rotary_interleaved=interleaved, cos_cache=dev(cos), sin_cache=dev(sin))
    assert pool.device_status(clear=True) == 2
    pr.check(got.double().cpu().numpy().reshape(want.shape), want, pr.bound(dtype, qr, size, want))
