"""The serving operators on a cache that holds a part of the KV heads: the heads' part of the whole cache's results."""
import pytest
import torch

from tests.test_gpu_serving import DT, _cache, _device, _lists, _trees
import numpy as np

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits,d,g", [(4, 128, 4), (8, 64, 8), (3, 64, 2), (4, 32, 3)])
@pytest.mark.parametrize("begin,count", [(0, 1), (2, 2), (3, 1)])
def test_heads_of_a_shard(cuda_device, bits, d, g, begin, count):
    import smallaios_b200 as sa

    b, h, past, n, drafted = 2, 4, 64 * 9 + 20, 6, 6
    r = np.random.default_rng(bits + d)
    kv = [torch.from_numpy(r.standard_normal((b, c, h, d)).astype(np.float32)).to(cuda_device)
          for c in (past, past, n, n)]
    q = torch.from_numpy(r.standard_normal((b, n, h, g * d)).astype(np.float32)).to(DT["f16"]).to(cuda_device)
    parents, ids = _device(_trees(r, b, n), cuda_device), _device(_lists(r, b, n, h, 4, past), cuda_device)
    path = torch.tensor([[0, 2, 5], [1, 3, 4]], dtype=torch.int32, device=cuda_device)
    outs = []
    for lo, c in ((0, h), (begin, count)):
        part = slice(lo, lo + c)
        cache = _cache(b, h, g, d, bits, past + n, cuda_device, layers=2, kv_head_begin=lo, kv_head_count=c)
        cut = lambda t: t[:, :, part].reshape(b, t.shape[1], -1).contiguous()  # noqa: E731
        cache.append(1, cut(kv[0]), cut(kv[1]))
        cache.advance_position(past)
        cache.append(1, cut(kv[2]), cut(kv[3]))
        means = sa.kv_block_means(cache, 1, 0, past // 64)
        qc = cut(q)
        got = [means, sa.gqa_select_blocks(qc, cache, 1, means, num_heads=h * g, max_blocks=5),
               sa.gqa_tree_attend(qc, cache, 1, parents, num_heads=h * g).view(b, n, c, g * d),
               sa.gqa_sparse_attend(qc, cache, 1, ids[:, :, part].contiguous(), num_heads=h * g).view(b, n, c, g * d)]
        cache.keep_drafts(path, drafted=drafted)
        view = cache.view(1)
        got += [x[:, :, past:past + 3] for x in (view.k_codes, view.v_codes_tokens(), view.k_meta, view.v_meta)]
        outs.append([t.clone() for t in got])
        assert cache.device_status() == 0
        cache.close()
    part = slice(begin, begin + count)
    whole, own = outs
    for i in (0, 4, 5, 6, 7):  # (B, H, ...)
        assert torch.equal(whole[i][:, part], own[i]), i
    assert torch.equal(whole[1][:, :, part], own[1])
    for i in (2, 3):  # the ranges that the work is cut into differ, and with them the order of f32 sums
        x, y = whole[i][:, :, part].float(), own[i].float()
        # f16 rounding of either, and 2^-17 of f32 sums
        assert ((x - y).norm() / y.norm()).item() < 2.0 ** -11, i
