"""What one token's metadata costs the other tokens of its page, in attention over pages: constant vectors (which the
append gives a scale of 1 and codes of 0) and large scales without weight, against 64 bits."""
import numpy as np
import pytest
import torch

import tests.pages_reference as pr
import tests.serving_reference as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEPS = {"f32": (8355711, 2.0 ** 24 - 1), "f16": (32639, 65535.0), "bf16": (32639, 65535.0)}  # of queries, of weights


def _held(view, bits, d):
    """A layer's codes (P, H, 64, D) and metadata (P, H, 64, 2), and the signs (H, D)."""
    codes = (ref.unpack(x.cpu().numpy(), bits, d) for x in (view.k_codes, view.v_codes_tokens()))
    kc, vc = codes
    return kc, view.k_meta.cpu().numpy().copy(), vc, view.v_meta.cpu().numpy().copy(), view.signs.cpu().numpy().astype(np.float64)


def _expect(dtype, q, kc, km, vc, vm, signs, row, n, bits, scale):
    """q (H, G, D), one row of n tokens -> outputs (H, G, D) and bounds on the 2-norms of their errors.

    A query's digits are off by half a step of max|q'| in each dimension, f32 arithmetic by 2^-20 of the scores' size:
    a weight by a relative e_t = (2 e_q + 2^-20) |q||k_t| scale, the output by sum w_t e_t |v_t - out|.  (2 e_q: first
    order, and the largest component of q' may be any part of |q|.)
    A weight times its value scale is off by half a step of the largest such product of its page, and that moves the
    output by as much times |c_t - middle|; not for a token whose codes are all 0, whose value is its zero point.
    f32 sums: 2^-19 of the terms, which are w_t (vs_t |c_t - middle| + sqrt(D) |vz_t + middle vs_t|); zero points alone
    for such a token.
    """
    d = q.shape[-1]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    mid, (steps, top) = (8 if bits == 4 else 128), STEPS[dtype]
    kc, vc, km, vm = (pr.tokens_of(a, row, n) for a in (kc, vc, km, vm))
    k, v = (ref.decode(c[None], m[None], signs)[0] for c, m in ((kc, km), (vc, vm)))
    km, vm = km.astype(np.float64), vm.astype(np.float64)
    w = np.einsum("hgd,htd->hgt", q, k) * scale
    w = np.exp(w - w.max(-1, keepdims=True))
    w /= w.sum(-1, keepdims=True)
    out = np.einsum("hgt,htd->hgd", w, v)
    norm = lambda x: np.sqrt((x * x).sum(-1))  # noqa: E731
    e = (2 * np.sqrt(d) / (2 * steps) + 2.0 ** -20) * norm(q)[..., None] * norm(k)[:, None] * abs(scale)
    limit = (w * e * norm(v[:, None] - out[:, :, None])).sum(-1)
    some = vc.any(-1)  # (H, T)
    vs = np.where(some, vm[..., 0], 0.0)
    size = norm(vc - float(mid)) * some  # |c_t - middle|
    for t in range(0, n, pr.PAGE):
        part = np.s_[..., t:t + pr.PAGE]
        step = (w[part] * np.maximum(vs, 2.0 ** -64)[:, None][part]).max(-1) / (2 * top)
        limit += step * size[part].sum(-1)[:, None]
    terms = vs * size + np.sqrt(d) * np.abs(vm[..., 1] + mid * vs)
    limit += 2.0 ** -19 * (w * terms[:, None]).sum(-1) + ref.ROUND[dtype] * norm(out)
    return out, limit


def _attend(pool, q, table, n, device, **kw):
    import smallaios_b200 as sa

    got = sa.gqa_paged_attend(q.to(device), pool, 0, torch.from_numpy(table).to(device),
                              torch.tensor([n - 1], dtype=torch.int32, device=device), **kw)
    assert pool.device_status() == 0
    return got.double().cpu().numpy()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scale", [0.0, None])
@pytest.mark.parametrize("std", [0.1, 0.001])
@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64)])
def test_constant_values_cost_their_neighbours_nothing(cuda_device, bits, d, std, scale, dtype):
    """Padded tokens' values, all zero, and vectors that rotate into a constant, appended beside small ordinary ones."""
    import smallaios_b200 as sa

    r = np.random.default_rng(bits + d)
    h, g, n = 2, 4, 200
    pages, table = pr.tables(r, [n])
    pool = sa.GpuKvPages(1, h, d, pages, num_heads=h * g, bits=bits, device=cuda_device)
    k, v = r.standard_normal((n, h, d)), r.standard_normal((n, h, d)) * std
    v[3::7] = 0.0
    v[5::50] = np.eye(d)[0] * std
    v[130:, 1] = 0.0  # a head whose last pages hold nothing else
    k, v = (torch.from_numpy(x.astype(np.float32).reshape(1, n, h * d)).to(cuda_device) for x in (k, v))
    pool.append(0, k, v, torch.from_numpy(table).to(cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device))
    held = _held(pool.view(0), bits, d)
    used = pr.tokens_of(held[2], table[0], n), pr.tokens_of(held[3], table[0], n)
    assert not used[0][:, 3::7].any() and (used[1][:, 3::7, 0] == 1.0).all()  # as the format has them
    q = torch.from_numpy(r.standard_normal((1, 1, h * g * d)).astype(np.float32)).to(DT[dtype])
    want, limit = _expect(dtype, q.double().numpy().reshape(h, g, d), *held, table[0], n, bits, scale)
    got = _attend(pool, q, table, n, cuda_device, num_heads=h * g, scale=scale)
    pr.check(got.reshape(h, g, d), want, limit)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64)])
def test_a_large_scale_without_weight_costs_its_neighbours_nothing(cuda_device, bits, d, dtype):
    """A value of scale 1 whose score is 40 below the others', whose scales are a thousandth.

    The query is a row of the transform: q' has one component, which its digits hold exactly, so that the weights'
    own digits are what is seen."""
    import smallaios_b200 as sa

    r = np.random.default_rng(bits * d)
    h, g, n = 2, 2, 170
    pages, table = pr.tables(r, [n])
    kc, km = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    vc, vm = ref.random_vectors(r, (pages, h, pr.PAGE, d), bits)
    vm *= 0.001 / vm[..., :1].mean()
    vm[:, :, 9::32] = np.array([1.0, -3.0], np.float32)
    km[:, :, 9::32, 1] -= 40.0
    pool = sa.GpuKvPages(1, h, d, pages, num_heads=h * g, bits=bits, device=cuda_device)
    signs = pr.fill(pool.view(0), kc, km, vc, vm)
    one = signs[:, None] * ref.walsh(np.eye(d)[[3, d - 6]])[None]  # (H, G, D) of +-1
    q = torch.from_numpy(one.astype(np.float32).reshape(1, 1, -1)).to(DT[dtype])
    want, limit = _expect(dtype, one, kc, km, vc, vm, signs, table[0], n, bits, None)
    got = _attend(pool, q, table, n, cuda_device, num_heads=h * g)
    pr.check(got.reshape(h, g, d), want, limit)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("bits,d", [(4, 128), (8, 128), (4, 64), (8, 64)])
def test_constant_keys_score_what_they_are(cuda_device, bits, d, dtype):
    """Zero keys between small ones: a score of 0 has no digits of the query to be off by."""
    import smallaios_b200 as sa

    r = np.random.default_rng(bits * d + 1)
    h, g, n = 2, 4, 200
    pages, table = pr.tables(r, [n])
    pool = sa.GpuKvPages(1, h, d, pages, num_heads=h * g, bits=bits, device=cuda_device)
    k, v = r.standard_normal((n, h, d)) * 0.02, r.standard_normal((n, h, d)) * 0.1 + 1.0
    k[::2] = 0.0
    v[::2] *= -1.0  # the two halves' weights are what the output is made of
    k, v = (torch.from_numpy(x.astype(np.float32).reshape(1, n, h * d)).to(cuda_device) for x in (k, v))
    pool.append(0, k, v, torch.from_numpy(table).to(cuda_device), torch.zeros(1, dtype=torch.int32, device=cuda_device))
    held = _held(pool.view(0), bits, d)
    q = torch.from_numpy((r.standard_normal((1, 1, h * g * d)) * 3).astype(np.float32)).to(DT[dtype])
    want, limit = _expect(dtype, q.double().numpy().reshape(h, g, d), *held, table[0], n, bits, None)
    got = _attend(pool, q, table, n, cuda_device, num_heads=h * g)
    pr.check(got.reshape(h, g, d), want, limit)
