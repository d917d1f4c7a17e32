"""Serving operators over the compressed KV cache: what is measured, and their plain forms.

Four operators, each over the cache's own format (per vector: D codes c of 4 or 8 bits, a scale s and a
zero point z, standing for S.H.(s c + z)/sqrt(D), H the Walsh-Hadamard matrix, S the head's signs):

  tree       attention of N drafted tokens per sequence that form a tree: node i sees the cached prefix,
             its ancestors and itself
  keep       the accepted path of drafted tokens moves to the front of the drafts, in every layer
  means      the mean rotated key of every block of 64 tokens, on a grid of 8 bits under one exponent
  sparse     every query token picks blocks by an exact integer score of those means, then attends to
             the tokens of the picked blocks only

The plain forms compute in 32 bits with elementary torch operations on the raw arrays of a cache; the
framework's operators read the same bytes from a GpuKvCache.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls the framework's operators

SEED = 0xDEADBEEFCAFE1234  # the cache's default seed of the head signs
BLOCK = 64                 # tokens of a block
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MASK64 = (1 << 64) - 1


# ---- the cases -------------------------------------------------------------------------------------
def listed():
    return [
        # the smallest decode layer, one sequence and a short int8 cache, eight drafts: latency
        dict(name="tree_small", op="tree", B=1, H=2, G=4, D=64, bits=8, dtype="f32", past=512, N=8),
        # a few users of the 32-head, 8-KV-head layer; odd context and odd tree, ragged between sequences
        dict(name="tree_odd", op="tree", B=8, H=8, G=4, D=128, bits=4, dtype="bf16", past=4093, N=26),
        # the headline decode configuration (batch 64, context 8192, int4) verifying 16 drafts each
        dict(name="tree_batch64", op="tree", B=64, H=8, G=4, D=128, bits=4, dtype="bf16", past=8176, N=16),
        # the 64-head layer with the widest tree: 512 query rows per KV head
        dict(name="tree_wide", op="tree", B=16, H=8, G=8, D=128, bits=4, dtype="f16", past=16300, N=64),
        # one sequence accepts two of eight drafts in every layer of a small model: latency
        dict(name="keep_small", op="keep", L=16, B=1, H=2, D=64, bits=8, past=200, N=8, n=2),
        # 64 sequences accept 11 of 48 drafts
        dict(name="keep_batch64", op="keep", L=16, B=64, H=8, D=128, bits=4, past=301, N=48, n=11),
        # a decode step that filled one block in each of 64 sequences
        dict(name="means_step", op="means", B=64, H=8, D=128, bits=4, first=127, blocks=1),
        # the whole of eight prompts of 32768 tokens
        dict(name="means_prompt", op="means", B=8, H=8, D=128, bits=8, first=0, blocks=512),
        # one user, 4096 tokens, 16 blocks: latency
        dict(name="sparse_one", op="sparse", B=1, H=8, G=4, D=128, bits=4, dtype="bf16", past=4095, S=1, k=16),
        # the headline decode configuration with a quarter of its blocks
        dict(name="sparse_batch64", op="sparse", B=64, H=8, G=4, D=128, bits=4, dtype="bf16", past=8191, S=1, k=32),
        # long contexts of the 64-head layer: an eighth of 32768 tokens
        dict(name="sparse_long", op="sparse", B=32, H=8, G=8, D=128, bits=4, dtype="f16", past=32767, S=1, k=64),
        # several query tokens per sequence, int8 cache, three heads per KV head, odd context
        dict(name="sparse_multi", op="sparse", B=3, H=4, G=3, D=64, bits=8, dtype="f32", past=9001, S=21, k=23),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "keep", "means", "sparse", "sparse"])
    bits, d = rng.choice([4, 4, 8]), rng.choice([64, 128, 128])
    case = dict(op=op, B=_log_int(rng, 1, 64), H=rng.choice([1, 2, 3, 4, 8]), D=d, bits=bits)
    if op == "keep":
        n_drafts = rng.randint(2, 64)
        case.update(L=rng.randint(1, 16), past=_log_int(rng, 1, 320), N=n_drafts, n=rng.randint(1, (n_drafts + 1) // 2))
        return case
    if op == "means":
        blocks = _log_int(rng, 1, 512)
        case.update(first=rng.randint(0, 8), blocks=min(blocks, max(1, 32768 // (case["B"] * case["H"]))))
        return case
    case.update(G=rng.choice([1, 2, 3, 4, 7, 8]), dtype=rng.choice(["bf16", "bf16", "f16", "f32"]))
    # the same cache bytes and query rows at most as the listed cases have
    tokens = _log_int(rng, 64, 32768)
    tokens = min(tokens, max(64, (64 * 8 * 8192 * 128) // (case["B"] * case["H"] * d * (2 if bits == 8 else 1))))
    if op == "tree":
        most = (16 * 8 * 512 * 16384) // (case["B"] * case["H"] * case["G"] * tokens * 2)
        case.update(past=tokens, N=max(1, min(_log_int(rng, 1, 64), most)))
    else:
        k = _log_int(rng, 2, 64)
        most = (32 * 8 * 64) // (case["B"] * case["H"] * k)
        case.update(past=tokens, S=max(1, min(_log_int(rng, 1, 32), most)), k=k)
    return case


def _capacity(case):
    op = case["op"]
    tokens = {"tree": lambda: case["past"] + case["N"], "keep": lambda: case["past"] + case["N"],
              "means": lambda: (case["first"] + case["blocks"]) * BLOCK,
              "sparse": lambda: case["past"] + case["S"]}[op]()
    return (tokens + BLOCK - 1) // BLOCK * BLOCK


def work(case):
    op, d = case["op"], case["D"]
    cb = d * case["bits"] // 8
    units = case["B"] * case["H"]
    if op == "keep":  # codes, scale and zero point of K and V, read once and written once
        return {"bytes": 2.0 * case["L"] * units * case["n"] * (2 * cb + 16) + 4.0 * case["B"] * case["n"], "flops": 0.0}
    if op == "means":
        tokens = units * case["blocks"] * BLOCK
        return {"bytes": tokens * (cb + 8.0) + units * case["blocks"] * d * 2.0, "flops": 2.0 * tokens * d}
    width = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if op == "tree":
        rows, tokens = case["N"] * case["G"], case["past"] + case["N"]
        return {"bytes": units * (tokens * (2 * cb + 16.0) + 2 * rows * d * width) + 4.0 * case["B"] * case["N"],
                "flops": 4.0 * units * rows * d * (case["past"] + 1)}
    # sparse: the means of every earlier block once per sequence and head, the picked blocks of each query token
    # (a cache block that several tokens of a sequence pick is read once at best; no more than the context)
    blocks = (case["past"] + case["S"] + BLOCK - 1) // BLOCK
    picked = min(case["k"], blocks)
    read = min(picked * case["S"], blocks)
    rows = case["S"] * case["G"]
    return {"bytes": units * (blocks * d * 2.0 + read * BLOCK * (2 * cb + 16.0) + 2 * rows * d * width + 4.0 * case["S"] * case["k"]),
            "flops": units * rows * d * (2.0 * blocks + 4.0 * picked * BLOCK)}


# ---- inputs ----------------------------------------------------------------------------------------
def _signs(layer, heads, d):
    """The +-1 signs of a layer's heads, from the cache's seed (Xorshift64)."""
    out = np.empty((heads, d), np.float32)
    for h in range(heads):
        x = (SEED * 0x9E3779B97F4A7C15 + layer * heads + h) & MASK64 or 0x5EEDDEADBEEFCAFE
        for i in range(d):
            x ^= (x << 13) & MASK64
            x ^= x >> 7
            x ^= (x << 17) & MASK64
            out[h, i] = 1.0 if (x & 1) == 0 else -1.0
    return torch.from_numpy(out).cuda()


def _pack(c, bits):
    """Codes (..., D) -> bytes (..., D*bits/8), the low nibble first."""
    return c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)


def _vectors(gen, shape, bits, spread):
    """Codes, {scale, zero point} of rotated vectors: Gaussian about a direction that neighbours share."""
    b, h, t, d = shape
    codes = torch.empty(b, h, t, d * bits // 8, dtype=torch.uint8, device="cuda")
    meta = torch.empty(b, h, t, 2, device="cuda")
    for i in range(b):  # one sequence at a time: the floats of a whole cache would not fit
        x = torch.randn(h, t, d, generator=gen, device="cuda")
        topic = torch.randn(h, (t + 31) // 32, d, generator=gen, device="cuda") * spread
        x += topic.repeat_interleave(32, dim=1)[:, :t]
        lo, hi = x.aminmax(dim=-1, keepdim=True)
        scale = (hi - lo) / (2 ** bits - 1)
        codes[i] = _pack(((x - lo) / scale).round_().clamp_(0, 2 ** bits - 1).to(torch.uint8), bits)
        meta[i] = torch.cat([scale, lo], dim=-1)
    return codes, meta


def _to_cache_v(v):
    """Token-major V codes (B, H, T, CB) -> the cache's 16-token blocks (B, H, T/16, CB/4, 4, 4, 4)."""
    b, h, t, cb = v.shape
    return v.view(b, h, t // 16, 4, 4, cb // 4, 4).permute(0, 1, 2, 5, 3, 6, 4)


def _trees(gen_np, b, n):
    """Parents (B, N): -1 is a root (it follows the prefix), -2 a slot without a node; trees differ in size."""
    parents = np.full((b, n), -2, np.int32)
    for i in range(b):
        size = n if i == 0 else int(gen_np.integers((n + 1) // 2, n + 1))
        for j in range(size):
            parents[i, j] = int(gen_np.integers(max(0, j - 6), j)) if j and gen_np.random() < 0.9 else -1
    return parents


def _paths(gen_np, b, n_drafts, n):
    """Accepted nodes (B, n), ascending: the root, then nodes at n or later, so that no move overwrites a source."""
    rest = np.stack([np.sort(gen_np.permutation(np.arange(n, n_drafts))[:n - 1]) for _ in range(b)])
    return np.concatenate([np.zeros((b, 1)), rest], axis=1).astype(np.int32)


def prepare(case, seed):
    op, b, h, d, bits = case["op"], case["B"], case["H"], case["D"], case["bits"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gen_np = np.random.default_rng(seed)
    t = _capacity(case)
    layers, g = case.get("L", 1), case.get("G", 1)
    st = dict(case=case)
    cache = None
    if own:
        import smallaios_b200 as sa

        cache = sa.GpuKvCache(layers, h, d, t, batch=b, num_heads=h * g, bits=bits, device="cuda")
        st["sa"], st["cache"] = sa, cache

    if op == "keep":
        cb = d * bits // 8
        st["path"] = torch.from_numpy(_paths(gen_np, b, case["N"], case["n"])).cuda()
        arrays = []
        for i in range(layers):
            k = torch.randint(0, 256, (b, h, t, cb), generator=gen, device="cuda", dtype=torch.uint8)
            v = torch.randint(0, 256, (b, h, t // 16, cb // 4, 4, 4, 4), generator=gen, device="cuda", dtype=torch.uint8)
            km = torch.randn(b, h, t, 2, generator=gen, device="cuda")
            vm = torch.randn(b, h, t, 2, generator=gen, device="cuda")
            if own:
                view = cache.view(i)
                for dst, src in ((view.k_codes, k), (view.v_codes, v), (view.k_meta, km), (view.v_meta, vm)):
                    dst.copy_(src)
                arrays.append([view.k_codes, view.v_codes, view.k_meta, view.v_meta])
            else:
                arrays.append([k, v, km, vm])
        if own:
            cache.set_position(case["past"])
            st["arrays"] = arrays
        else:  # one array for all layers of each kind
            st["stacked"] = [torch.stack(a) for a in zip(*arrays)]
        return st

    k, km = _vectors(gen, (b, h, t, d), bits, 0.5)
    if op == "means":
        if own:
            view = cache.view(0)
            view.k_codes.copy_(k)
            view.k_meta.copy_(km)
        else:
            st.update(k=k, km=km)
        return st

    v, vm = _vectors(gen, (b, h, t, d), bits, 0.2)
    s = case["N"] if op == "tree" else case["S"]
    # queries as the projection gives them, rotated to their positions; scores of standard deviation near 1.5
    st["q"] = (torch.randn(b, s, h * g * d, generator=gen, device="cuda") * 1.3).to(DTYPES[case["dtype"]])
    if op == "tree":
        st["parents"] = torch.from_numpy(_trees(gen_np, b, s)).cuda()
    else:
        # block means are state that the cache's user keeps up to date while appending
        st["means"] = _means(_unpack(k, bits), km)
    if own:
        view = cache.view(0)
        view.k_codes.copy_(k)
        view.k_meta.copy_(km)
        view.v_codes.copy_(_to_cache_v(v))
        view.v_meta.copy_(vm)
        cache.set_position(case["past"])
    else:
        st.update(k=k, km=km, v=v, vm=vm, signs=_signs(0, h, d))
    return st


# ---- plain forms -----------------------------------------------------------------------------------
def _unpack(codes, bits):
    if bits == 8:
        return codes
    return torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)


def _hadamard(d):
    """Walsh-Hadamard matrix: entry (i, j) is -1 to the number of common set bits of i and j."""
    i = torch.arange(d, device="cuda")
    common = (i[:, None] & i[None, :])[..., None] >> torch.arange(8, device="cuda")
    return 1.0 - 2.0 * ((common & 1).sum(-1) % 2).float()


def _vectors_of(codes, meta, bits):
    """The rotated vectors s c + z."""
    return _unpack(codes, bits).float() * meta[..., :1] + meta[..., 1:]


def _rotated_queries(st, hadamard):
    """(B, H, S, G, D): the queries in the cache's rotated frame, and the signs that rotate back."""
    case = st["case"]
    b, h, g, d = case["B"], case["H"], case["G"], case["D"]
    q = st["q"].float().view(b, -1, h, g, d).transpose(1, 2)
    signs = st["signs"].view(1, h, 1, 1, d)
    return (q * signs) @ hadamard, signs


def _softmax_rows(scores, allowed):
    """Rows of softmax over the allowed places; rows without any are zero."""
    top = torch.where(allowed, scores, -math.inf).amax(-1, keepdim=True)
    e = torch.where(allowed, (scores - torch.where(top > -math.inf, top, 0.0)).exp(), 0.0)
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _tree_plain(st):
    case = st["case"]
    b, h, g, d, n, past, bits = (case[x] for x in ("B", "H", "G", "D", "N", "past", "bits"))
    hadamard = _hadamard(d)
    q, signs = _rotated_queries(st, hadamard)
    total = past + n
    k = _vectors_of(st["k"][:, :, :total], st["km"][:, :, :total], bits)
    scores = q.reshape(b, h, n * g, d) @ k.transpose(-1, -2) * (1.0 / d)  # 1/sqrt(D) of the rotation, 1/sqrt(D) of attention
    del k
    # ancestors: the powers of (I + parent) are nonzero where one node is above another
    parents = st["parents"].long()
    node = torch.arange(n, device="cuda")
    up = (parents[:, :, None] == node).float() + torch.eye(n, device="cuda")
    sees = (torch.linalg.matrix_power(up, n) > 0) & (parents[:, :, None] >= -1)
    allowed = torch.cat([(parents >= -1)[:, :, None].expand(b, n, past), sees], dim=-1)
    p = _softmax_rows(scores.view(b, h, n, g, total), allowed[:, None, :, None, :])
    del scores
    v = _vectors_of(st["v"][:, :, :total], st["vm"][:, :, :total], bits)
    o = (p.view(b, h, n * g, total) @ v).view(b, h, n, g, d)
    o = (o @ hadamard) * (signs / math.sqrt(d))
    return o.transpose(1, 2).reshape(b, n, h * g * d).to(st["q"].dtype)


def _keep_plain(st):
    case = st["case"]
    past, n = case["past"], case["n"]
    k, v, km, vm = st["stacked"]
    src = (past + st["path"].long())  # (B, n)
    dst = past + torch.arange(n, device="cuda").expand_as(src)
    row = torch.arange(case["B"], device="cuda")[:, None]
    k[:, row, :, dst] = k[:, row, :, src]  # the right side is read whole before anything is written
    km[:, row, :, dst] = km[:, row, :, src]
    vm[:, row, :, dst] = vm[:, row, :, src]
    v[:, row, :, dst // 16, :, dst % 16 // 4, :, dst % 4] = v[:, row, :, src // 16, :, src % 16 // 4, :, src % 4]
    return [[k[i], v[i], km[i], vm[i]] for i in range(case["L"])]


def _small(x):
    """Values of magnitude under 2^100; the others (infinities and NaN among them) count as zero."""
    return torch.where(x.abs() < 2.0 ** 100, x, 0.0)


def _exponent(x):
    """The least e with x < 2^e, and -100 where that is less."""
    return torch.where(x > 0, torch.frexp(x)[1].clamp_min(-100), -100)


def _power(e):
    """2^e in 32 bits, exactly, for whole numbers -126 <= e <= 127."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _means(codes, meta):
    """Means of blocks of 64 rotated keys, (B, H, T, D) and (B, H, T, 2) -> bf16 (B, H, T/64, D).

    All in whole numbers: scale and zero point of the block's tokens as 15-bit multiples of one power of two,
    the sums over the tokens, and these rounded to 8 bits under the largest one's exponent."""
    b, h, t, d = codes.shape
    meta = _small(meta).view(b, h, t // BLOCK, BLOCK, 2)
    e = _exponent(meta.abs().amax((-1, -2), keepdim=True))
    grid = (meta * _power(15 - e)).round().to(torch.int32)
    total = (codes.view(b, h, t // BLOCK, BLOCK, d).to(torch.int32) * grid[..., :1] + grid[..., 1:]).sum(3, dtype=torch.int32)
    bits = torch.frexp(total.abs().amax(-1, keepdim=True).double())[1]
    shift = (bits - 8).clamp_min(0)
    rounded = (total + ((1 << shift) >> 1)) >> shift
    return (rounded.float() * _power(shift + e[..., 0] - 21)).to(torch.bfloat16)


def _means_plain(st):
    case = st["case"]
    lo, hi = case["first"] * BLOCK, (case["first"] + case["blocks"]) * BLOCK
    return _means(_unpack(st["k"][:, :, lo:hi], case["bits"]), st["km"][:, :, lo:hi])


def _picked_blocks(st, hadamard):
    """Block ids (B, S, H, k), ascending, -1 after the last: the first block, the query's own block, and those
    with the largest scores (of the best query head of the KV head; ties to the lower block)."""
    case = st["case"]
    b, h, g, d, s, past, k = (case[x] for x in ("B", "H", "G", "D", "S", "past", "k"))
    # queries on a 12-bit grid, rotated exactly, rounded to 8 bits
    q = _small(st["q"].float()).view(b, s, h, g, d).transpose(1, 2)
    grid = (q * _power(12 - _exponent(q.abs().amax((-1, -2), keepdim=True)))).round()
    r = (grid * st["signs"].view(1, h, 1, 1, d)) @ hadamard
    shift = (torch.frexp(r.abs().amax((-1, -2), keepdim=True))[1] - 7).clamp_min(0)
    r8 = (r * _power(-shift)).round().clamp(-127, 127)
    blocks = (past + s + BLOCK - 1) // BLOCK
    m = st["means"][:, :, None, :blocks].float()
    score = (r8 @ m.transpose(-1, -2)).amax(-2)  # (B, H, S, blocks), exact: whole numbers under 2^24 times a power of two
    block = torch.arange(blocks, device="cuda")
    last = (past + torch.arange(s, device="cuda")[:, None]) // BLOCK
    score = torch.where((block == 0) | (block == last), math.inf, score)
    score = torch.where(block > last, -math.inf, score)
    top, ids = torch.sort(score, dim=-1, descending=True, stable=True)
    ids = torch.where(top > -math.inf, ids, 1 << 30)[..., :k].sort(-1)[0]
    ids = torch.where(ids < 1 << 30, ids, -1).to(torch.int32).transpose(1, 2)
    return torch.nn.functional.pad(ids, (0, k - ids.shape[-1]), value=-1).contiguous()


def _sparse_plain(st):
    case = st["case"]
    b, h, g, d, s, past, k, bits = (case[x] for x in ("B", "H", "G", "D", "S", "past", "k", "bits"))
    hadamard = _hadamard(d)
    ids = _picked_blocks(st, hadamard)
    q, signs = _rotated_queries(st, hadamard)  # (B, H, S, G, D)
    at = ids.transpose(1, 2).long()            # (B, H, S, k)
    seq, head = torch.arange(b, device="cuda")[:, None, None, None], torch.arange(h, device="cuda")[:, None, None]
    blocks = lambda a: a.view(b, h, -1, BLOCK, a.shape[-1])[seq, head, at.clamp_min(0)]  # noqa: E731
    kk = _vectors_of(blocks(st["k"]), blocks(st["km"]), bits).view(b, h, s, k * BLOCK, d)
    scores = q @ kk.transpose(-1, -2) * (1.0 / d)
    del kk
    token = at[..., None] * BLOCK + torch.arange(BLOCK, device="cuda")
    allowed = (at[..., None] >= 0) & (token <= past + torch.arange(s, device="cuda")[:, None, None])
    p = _softmax_rows(scores, allowed.view(b, h, s, 1, k * BLOCK))
    vv = _vectors_of(blocks(st["v"]), blocks(st["vm"]), bits).view(b, h, s, k * BLOCK, d)
    o = ((p @ vv) @ hadamard) * (signs / math.sqrt(d))
    return [ids, o.transpose(1, 2).reshape(b, s, h * g * d).to(st["q"].dtype)]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"tree": _tree_plain, "keep": _keep_plain, "means": _means_plain, "sparse": _sparse_plain}[op](state)
    sa, cache = state["sa"], state["cache"]
    if op == "tree":
        return sa.gqa_tree_attend(state["q"], cache, 0, state["parents"], num_heads=case["H"] * case["G"])
    if op == "keep":
        cache.keep_drafts(state["path"], drafted=case["N"])
        return state["arrays"]
    if op == "means":
        return sa.kv_block_means(cache, 0, case["first"], case["first"] + case["blocks"])
    ids = sa.gqa_select_blocks(state["q"], cache, 0, state["means"], num_heads=case["H"] * case["G"], max_blocks=case["k"])
    return [ids, sa.gqa_sparse_attend(state["q"], cache, 0, ids, num_heads=case["H"] * case["G"])]


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _walsh64(x):
    """Walsh-Hadamard transform of the last axis, by butterflies."""
    d = x.shape[-1]
    step = 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(x.shape)
        step *= 2
    return x


def _decode64(codes, meta, bits, signs):
    """Vectors of one head (T, D) as the cache's codes define them."""
    if bits == 4:
        c = torch.empty(*codes.shape[:-1], 2 * codes.shape[-1], dtype=torch.float64, device=codes.device)
        c[..., 0::2] = (codes & 15).double()
        c[..., 1::2] = (codes >> 4).double()
    else:
        c = codes.double()
    x = c * meta[:, :1].double() + meta[:, 1:].double()
    return signs.double() * _walsh64(x) / math.sqrt(x.shape[-1])


def _power64(e):
    """2^e in 64 bits, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _means64(st):
    """The block means by their definition, with 64-bit whole numbers and floats."""
    case = st["case"]
    b, h, d, n = case["B"], case["H"], case["D"], case["blocks"]
    out = torch.zeros(b, h, n, d, dtype=torch.float64, device="cuda")
    for i in range(n):
        at = (case["first"] + i) * BLOCK
        byte = st["k"][:, :, at:at + BLOCK].long()
        code = byte if case["bits"] == 8 else torch.stack([byte % 16, byte // 16], dim=-1).reshape(b, h, BLOCK, d)
        pair = st["km"][:, :, at:at + BLOCK].double()
        pair = torch.where(pair.abs() < 2.0 ** 100, pair, 0.0)
        top = pair.abs().reshape(b, h, -1).max(-1)[0]
        e = torch.where(top > 0, torch.frexp(top)[1].clamp_min(-100), -100)[..., None]
        s, z = (torch.round(pair[..., x] * _power64(15 - e)).long() for x in (0, 1))
        m = torch.einsum("bht,bhtd->bhd", s.double(), code.double()) + z.sum(-1, keepdim=True).double()
        shift = (torch.frexp(m.abs().max(-1, keepdim=True)[0])[1] - 8).clamp_min(0)
        out[:, :, i] = torch.floor(m * _power64(-shift) + 0.5 * (shift > 0)) * _power64(shift + e - 21)
    return out


def exact(case, seed):
    global own
    op = case["op"]
    if op == "keep":
        return None  # bytes that move
    was, own = own, False
    try:
        st = prepare(case, seed)
        ids = _picked_blocks(st, _hadamard(case["D"])) if op == "sparse" else None
    finally:
        own = was
    if op == "means":
        return _means64(st)
    b, h, g, d, past, bits = (case[x] for x in ("B", "H", "G", "D", "past", "bits"))
    s = case["N"] if op == "tree" else case["S"]
    q = st["q"].double().view(b, s, h, g, d)
    out = torch.zeros(b, s, h, g, d, dtype=torch.float64, device="cuda")
    parents = st["parents"].tolist() if op == "tree" else None
    for i in range(b):
        seen = []  # the tokens that each query token sees
        if op == "tree":
            for j in range(s):
                mask = torch.zeros(past + s, dtype=torch.bool)
                at = j if parents[i][j] >= -1 else -1
                mask[:past] = at >= 0
                while at >= 0:
                    mask[past + at] = True
                    at = parents[i][at]
                seen.append(mask)
            seen = torch.stack(seen).cuda()
        for e in range(h):
            total = past + s
            k = _decode64(st["k"][i, e, :total], st["km"][i, e, :total], bits, st["signs"][e])
            v = _decode64(st["v"][i, e, :total], st["vm"][i, e, :total], bits, st["signs"][e])
            if op == "sparse":
                block = torch.zeros(s, (total + BLOCK - 1) // BLOCK + 1, dtype=torch.bool, device="cuda")
                block.scatter_(1, ids[i, :, e].long() % block.shape[1], True)  # -1 lands in the spare last column
                token = torch.arange(total, device="cuda")
                mask = block[:, :-1].repeat_interleave(BLOCK, dim=1)[:, :total] & (token <= past + torch.arange(s, device="cuda")[:, None])
            else:
                mask = seen
            w = torch.einsum("sgd,td->sgt", q[i, :, e], k) / math.sqrt(d)
            w = w.masked_fill(~mask[:, None], -math.inf)
            w = torch.nan_to_num(torch.softmax(w, dim=-1))  # a row that sees nothing is zero
            out[i, :, e] = torch.einsum("sgt,td->sgd", w, v)
    out = out.view(b, s, h * g * d)
    return [None, out] if op == "sparse" else out
