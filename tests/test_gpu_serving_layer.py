"""The serving operators together, as a serving loop runs them: a tree of drafts verified by a layer, its accepted
path kept, decoding from there; a decode loop over selected blocks with its block means kept up to date."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, HQ, HKV, D, F, BITS = 512, 8, 2, 64, 1024, 4
DT = torch.bfloat16


def _weights(r, device):
    import smallaios_b200 as sa

    def w(n, k):
        codes = torch.from_numpy(r.integers(0, 256, (n, k // 32, 16), dtype=np.uint8)).to(device)
        scales = torch.from_numpy(r.uniform(0.002, 0.006, (n, k // 32)).astype(np.float32)).to(DT).to(device)
        return codes, scales

    norm = [torch.from_numpy(r.uniform(0.5, 1.5, HIDDEN).astype(np.float32)).to(DT).to(device) for _ in range(2)]
    wqkv, wo, wgu, wdn = w((HQ + 2 * HKV) * D, HIDDEN), w(HIDDEN, HQ * D), w(2 * F, HIDDEN), w(HIDDEN, F)
    return sa.LayerWeights(*wqkv, *wo, *wgu, *wdn, *norm)


def _tables(rows, device):
    t = np.arange(rows)[:, None] * 10000.0 ** (-np.arange(D // 2) / (D // 2))[None]
    return [torch.from_numpy(f(t).astype(np.float32)).to(device) for f in (np.cos, np.sin)]


def _rows(r, n, device):
    return torch.from_numpy(r.standard_normal((n, HIDDEN)).astype(np.float32)).to(DT).to(device)


def _near(got, want, bar):
    err = (got.float() - want.float()).norm() / want.float().norm()
    assert err < bar, f"relative error {err:.2e}"


def test_chain_tree_is_a_prefill_chunk(cuda_device):
    """A chain of drafts through tree_layer_step is the chunk prefill_layer_step computes.  The tree path rounds the
    rotated q and k to bf16 once more (2^-9 each: scores of a few units move by about 1%), so 2e-2."""
    import smallaios_b200 as sa

    b, past, n = 2, 150, 20
    r = np.random.default_rng(1)
    w = _weights(r, cuda_device)
    cos, sin = _tables(past + n, cuda_device)
    x0, x1 = _rows(r, b * past, cuda_device), _rows(r, b * n, cuda_device)
    outs = []
    for tree in (False, True):
        cache = sa.GpuKvCache(1, HKV, D, past + n, batch=b, num_heads=HQ, bits=BITS, device=cuda_device)
        sa.prefill_layer_step(x0, None, w, cache, 0, batch=b, seq_len=past, cos_cache=cos, sin_cache=sin)
        cache.advance_position(past)
        if tree:
            parents = torch.arange(-1, n - 1, dtype=torch.int32, device=cuda_device).repeat(b, 1)
            ids = (past + torch.arange(n, dtype=torch.int32, device=cuda_device)).repeat(b, 1)
            outs.append(sa.tree_layer_step(x1, None, w, cache, 0, parents=parents, position_ids=ids, cos_cache=cos,
                                           sin_cache=sin))
        else:
            outs.append(sa.prefill_layer_step(x1, None, w, cache, 0, batch=b, seq_len=n, cos_cache=cos, sin_cache=sin))
        assert cache.current_position() == past
        cache.close()
    for got, want in zip(outs[1], outs[0]):
        _near(got, want, 2e-2)


def test_verify_keep_and_decode(cuda_device):
    """After keep_drafts the cache is the one that only ever saw the accepted tokens: same bytes, same next outputs."""
    import smallaios_b200 as sa

    b, past, n, layers = 2, 90, 9, 2
    path = [[0, 2, 5, 8], [1, 3, 4, 7]]
    depth = len(path[0])
    parents = torch.tensor([[-1, 0, 0, 1, 2, 2, 3, 4, 5], [-1, -1, 0, 1, 3, 2, 5, 4, 7]], dtype=torch.int32)
    r = np.random.default_rng(2)
    kv = [[torch.from_numpy(r.standard_normal((b, c, HKV * D)).astype(np.float32)).to(DT).to(cuda_device)
           for _ in range(2 * layers)] for c in (past, n, 1)]
    q = torch.from_numpy(r.standard_normal((b, n, HQ * D)).astype(np.float32)).to(DT).to(cuda_device)
    got, want = (sa.GpuKvCache(layers, HKV, D, past + n + 1, batch=b, num_heads=HQ, bits=BITS, qjl_residual=True,
                               device=cuda_device) for _ in range(2))
    for cache in (got, want):
        for layer in range(layers):
            cache.append(layer, *kv[0][2 * layer:2 * layer + 2])
        cache.advance_position(past)
    p = torch.tensor(path, device=cuda_device)
    for layer in range(layers):
        k, v = kv[1][2 * layer:2 * layer + 2]
        got.append(layer, k, v)
        sa.gqa_tree_attend(q, got, layer, parents.to(cuda_device), num_heads=HQ)
        pick = p[..., None].expand(-1, -1, HKV * D)
        want.append(layer, k.gather(1, pick), v.gather(1, pick))
    got.keep_drafts(p.to(torch.int32), drafted=n)
    for cache in (got, want):
        cache.advance_position(depth)
    for layer in range(layers):
        outs = [sa.group_query_attention(q[:, :1].contiguous(), *kv[2][2 * layer:2 * layer + 2], cache, layer,
                                         num_heads=HQ, kv_num_heads=HKV, do_rotary=False) for cache in (got, want)]
        assert torch.equal(*outs)
        a, c = got.view(layer), want.view(layer)
        end = past + depth + 1
        for name in ("k_codes", "k_meta", "v_meta", "k_qjl_bits", "v_qjl_bits", "k_qjl_mag", "v_qjl_mag"):
            assert torch.equal(getattr(a, name)[:, :, :end], getattr(c, name)[:, :, :end]), name
        assert torch.equal(a.v_codes_tokens()[:, :, :end], c.v_codes_tokens()[:, :, :end])
    got.close()
    want.close()


@pytest.mark.parametrize("max_blocks,bar", [(8, 1e-2), (3, None)])
def test_decode_over_selected_blocks(cuda_device, max_blocks, bar):
    """Decode steps that cross two block ends.  With room for every block the layer is the dense one (rounding flips
    of bf16 propagate: 1e-2); the means that the steps leave are those of the whole cache."""
    import smallaios_b200 as sa

    b, past, steps = 2, 190, 70
    r = np.random.default_rng(3)
    w = _weights(r, cuda_device)
    cos, sin = _tables(past + steps, cuda_device)
    x0 = _rows(r, b * past, cuda_device)
    caches = [sa.GpuKvCache(1, HKV, D, past + steps, batch=b, num_heads=HQ, bits=BITS, device=cuda_device) for _ in "ab"]
    for cache in caches:
        sa.prefill_layer_step(x0, None, w, cache, 0, batch=b, seq_len=past, cos_cache=cos, sin_cache=sin)
        cache.advance_position(past)
    means = torch.zeros(b, HKV, (past + steps + 63) // 64, D, dtype=DT, device=cuda_device)
    sa.kv_block_means(caches[1], 0, 0, past // 64, out=means[:, :, :past // 64])
    for _ in range(steps):
        x = _rows(r, b, cuda_device)
        want = sa.decoder_layer_step(x, None, w, caches[0], 0, cos_cache=cos, sin_cache=sin)
        got = sa.decoder_layer_step(x, None, w, caches[1], 0, cos_cache=cos, sin_cache=sin, block_means=means,
                                    max_blocks=max_blocks)
        if bar:
            _near(got[0], want[0], bar)
        assert torch.isfinite(got[0]).all()
        for cache in caches:
            cache.advance_position(1)
    full = (past + steps) // 64
    assert torch.equal(means[:, :, :full], sa.kv_block_means(caches[1], 0, 0, full))
    for cache in caches:
        assert cache.device_status() == 0
        cache.close()
