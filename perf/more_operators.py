"""Operators of paged serving over the compressed KV format: what is measured, and their plain forms.

Four operators, each over pages of 64 tokens that hold, per (page, KV head) and token, D codes c of 4 or 8 bits, a
scale s and a zero point z, standing for S.H.(s c + z)/sqrt(D) (H the Walsh-Hadamard matrix, S the head's signs):

  append    keys and values of new tokens are rotated to their positions (keys), quantized and written into the
            pages of their sequences; sequences differ in length, and in how many tokens they add
  attend    one new token of each sequence attends to all tokens of its pages; its query is rotated on the way
  select    beam search: the best continuations over all beams and the whole vocabulary
  reorder   the beams take over the pages of the beams they continue; a page that several beams would go on
            filling is copied

The plain forms compute in 32 bits (codes: with every step rounded to 32 bits, as the format defines them; the
selection: in 64 bits, since scores of different beams lie close) with elementary torch operations on raw arrays;
the framework's operators work on a GpuKvPages with the same bytes.
"""
import math

import numpy as np
import torch

own = False  # True: run() calls the framework's operators

SEED = 0xDEADBEEFCAFE1234  # the pool's default seed of the head signs
PAGE = 64                  # tokens of a page
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MASK64 = (1 << 64) - 1


# ---- the cases -------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a batch of 64 in the 32-head, 8-KV-head layer: latency
        dict(name="append_step", op="append", B=64, S=1, H=8, D=128, bits=4, dtype="bf16", past=8191, ragged=True,
             interleaved=False),
        # a few chunks of f32 prompts of odd lengths, interleaved rotation, int8, small heads
        dict(name="append_odd", op="append", B=3, S=333, H=4, D=64, bits=8, dtype="f32", past=77, ragged=True,
             interleaved=True),
        # eight whole prompts of up to 2048 tokens (the prefill configuration)
        dict(name="append_prompts", op="append", B=8, S=2048, H=8, D=128, bits=4, dtype="bf16", past=0, ragged=True,
             interleaved=False),
        # the smallest decode layer: one sequence, a short int8 context: latency
        dict(name="attend_one", op="attend", B=1, H=2, G=4, D=64, bits=8, dtype="f32", past=511, ragged=False,
             interleaved=False),
        # a server's mixed batch: 48 sequences between their first token and 16000
        dict(name="attend_ragged", op="attend", B=48, H=8, G=4, D=128, bits=4, dtype="bf16", past=16000, ragged=True,
             interleaved=False),
        # the headline decode configuration (batch 64, context 8192, int4)
        dict(name="attend_batch64", op="attend", B=64, H=8, G=4, D=128, bits=4, dtype="bf16", past=8191, ragged=False,
             interleaved=False),
        # long contexts of the 64-head layer, eight query heads per KV head
        dict(name="attend_long", op="attend", B=32, H=8, G=8, D=128, bits=4, dtype="f16", past=32767, ragged=False,
             interleaved=False),
        # one user with four beams: latency
        dict(name="select_one", op="select", B=1, K=4, V=32000, keep=4, dtype="f32"),
        # a vocabulary of odd size, twice as many candidates as beams
        dict(name="select_odd", op="select", B=32, K=5, V=50257, keep=10, dtype="f16"),
        # 64 users with eight beams each over a large vocabulary
        dict(name="select_batch64", op="select", B=64, K=8, V=128256, keep=8, dtype="bf16"),
        # one user with four beams in a small model: latency
        dict(name="reorder_one", op="reorder", L=12, B=1, K=4, H=2, D=64, bits=8, past=200),
        # 16 users with eight beams
        dict(name="reorder_batch16", op="reorder", L=8, B=16, K=8, H=8, D=128, bits=4, past=1005),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "select", "select", "reorder"])
    if op == "select":
        k = rng.randint(1, 16)
        case = dict(op=op, K=k, V=_log_int(rng, 1000, 128256), keep=min(32, k * rng.choice([1, 1, 2])),
                    dtype=rng.choice(["bf16", "f16", "f32"]))
        width = 4 if case["dtype"] == "f32" else 2
        return dict(case, B=_log_int(rng, 1, max(1, min(64, 64 * 8 * 128256 * 2 // (k * case["V"] * width)))))
    case = dict(op=op, H=rng.choice([1, 2, 3, 4, 8]), D=rng.choice([64, 128, 128]), bits=rng.choice([4, 4, 8]))
    if op == "reorder":
        k, layers = rng.randint(2, 16), rng.randint(1, 15)
        most = 16 * 8 * 8 * 8 * 128 * 4 // (k * layers * case["H"] * case["D"] * case["bits"])
        return dict(case, L=layers, K=k, B=_log_int(rng, 1, max(1, min(16, most))), past=_log_int(rng, 1, 1005))
    case.update(dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), ragged=rng.random() < 0.7,
                interleaved=rng.random() < 0.3)
    if op == "append":
        s = _log_int(rng, 1, 2048)
        most = 8 * 2048 * 8 * 128 * 2 // (s * case["H"] * case["D"] * (4 if case["dtype"] == "f32" else 2))
        case.update(S=s, B=_log_int(rng, 1, max(1, min(64, most))))
        held = 64 * 4096 * 8 * 128 * 4 // (case["B"] * case["H"] * case["D"] * case["bits"])  # tokens of a sequence
        return dict(case, past=_log_int(rng, 1, max(2, min(8192, held))))
    tokens = _log_int(rng, 1, 32768)
    # the same pages and multiplications at most as the listed cases have
    case["G"] = rng.choice([1, 2, 3, 4, 7, 8])
    most = 32 * 8 * 128 * 4 * 32768 // (tokens * case["H"] * case["D"] * case["bits"])
    return dict(case, B=_log_int(rng, 1, max(1, min(64, most))), past=tokens - 1)


def _lengths(case):
    """Tokens cached before the call, of each sequence: `past` each, or spread between 0 and `past` where ragged."""
    past, b = case["past"], case["B"]
    if not case.get("ragged"):
        return [past] * b
    return [past if i == 0 else int(past * ((i * 0.6180339887) % 1.0) ** 1.5) for i in range(b)]


def _counts(case):
    """Tokens that each sequence appends: S, or fewer where ragged prompts are padded."""
    s = case["S"]
    return [s if i == 0 or not case["ragged"] or s == 1 else 1 + int((s - 1) * ((i * 0.7548776662) % 1.0))
            for i in range(case["B"])]


def work(case):
    op = case["op"]
    if op == "select":
        width = 4 if case["dtype"] == "f32" else 2
        n = case["B"] * case["K"] * case["V"]
        return {"bytes": n * width + 5.0 * case["B"] * case["K"] + 12.0 * case["B"] * case["keep"], "flops": 4.0 * n}
    d = case["D"]
    row = d * case["bits"] // 8 + 8  # codes, scale and zero point of a vector
    if op == "reorder":
        # the rows of the page in use that more than one beam continues, read once and written for each further beam;
        # the table's used part is read and written
        copies = case["B"] * _further_beams(case["K"])
        rows = case["L"] * case["H"] * (case["past"] % PAGE)
        entries = case["B"] * case["K"] * ((case["past"] + PAGE) // PAGE)
        return {"bytes": 2.0 * copies * rows * 2 * row + 8.0 * entries, "flops": 0.0}
    width = 4 if case["dtype"] == "f32" else 2
    if op == "append":
        vectors = 2.0 * sum(_counts(case)) * case["H"]
        return {"bytes": vectors * (d * width + row), "flops": vectors * d * (math.log2(d) + 6)}
    tokens = sum(n + 1 for n in _lengths(case))
    rows = case["B"] * case["H"] * case["G"] * d
    return {"bytes": 2.0 * tokens * case["H"] * row + 2.0 * rows * width,
            "flops": 4.0 * tokens * case["H"] * case["G"] * d}


def _further_beams(k):
    """Beams of k that end; as many others go on in a second slot."""
    return (k + 1) // 3


# ---- inputs ----------------------------------------------------------------------------------------
def _signs(layer, heads, d):
    """The +-1 signs of a layer's heads, from the pool's seed (Xorshift64)."""
    out = np.empty((heads, d), np.float32)
    for h in range(heads):
        x = (SEED * 0x9E3779B97F4A7C15 + layer * heads + h) & MASK64 or 0x5EEDDEADBEEFCAFE
        for i in range(d):
            x ^= (x << 13) & MASK64
            x ^= x >> 7
            x ^= (x << 17) & MASK64
            out[h, i] = 1.0 if (x & 1) == 0 else -1.0
    return torch.from_numpy(out).cuda()


def _tables(positions, d):
    """Cosines and sines of the rotary angles, (positions, D/2), from angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
    angle = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _vectors(gen, pages, heads, d, bits, spread):
    """Codes (P, H, 64, CB) and {scale, zero point} of rotated vectors: Gaussian about a direction of the page."""
    codes = torch.empty(pages, heads, PAGE, d * bits // 8, dtype=torch.uint8, device="cuda")
    meta = torch.empty(pages, heads, PAGE, 2, device="cuda")
    step = max(1, (1 << 26) // (heads * PAGE * d))
    for i in range(0, pages, step):  # a part of the pool at a time: the floats of all would not fit
        n = min(step, pages - i)
        x = torch.randn(n, heads, PAGE, d, generator=gen, device="cuda")
        x += torch.randn(n, heads, 1, d, generator=gen, device="cuda") * spread
        lo, hi = x.aminmax(dim=-1, keepdim=True)
        scale = (hi - lo) / (2 ** bits - 1)
        c = ((x - lo) / scale).round_().clamp_(0, 2 ** bits - 1).to(torch.uint8)
        codes[i:i + n] = c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)
        meta[i:i + n] = torch.cat([scale, lo], dim=-1)
    return codes, meta


def _to_pool_v(v):
    """Token-major V codes (P, H, 64, CB) -> the pool's 16-token blocks (P, H, 4, CB/4, 4, 4, 4)."""
    p, h, t, cb = v.shape
    return v.view(p, h, t // 16, 4, 4, cb // 4, 4).permute(0, 1, 2, 5, 3, 6, 4)


def _parents(gen_np, b, k):
    """(B, K) the beam that each slot continues: about a third of the beams end, and as many others take their place."""
    out, n = np.empty((b, k), np.int32), _further_beams(k)
    for i in range(b):
        ended = gen_np.permutation(k)[:n]
        alive = np.setdiff1d(np.arange(k), ended)
        out[i] = gen_np.permutation(np.concatenate([alive, gen_np.choice(alive, n)]))
    return out


def _pool(case, pages):
    import smallaios_b200 as sa

    return sa, sa.GpuKvPages(case.get("L", 1), case["H"], case["D"], pages, num_heads=case["H"] * case.get("G", 1),
                             bits=case["bits"], device="cuda")


def prepare(case, seed):
    op = case["op"]
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gen_np = np.random.default_rng(seed)
    st = dict(case=case)
    if op == "select":
        b, k, v = case["B"], case["K"], case["V"]
        # logits of standard deviation near 2.5 with a few tokens far above; some tokens are forbidden
        x = torch.randn(b * k, v, generator=gen, device="cuda") * 2.5
        hot = torch.randint(0, v, (b * k, 24), generator=gen, device="cuda")
        x.scatter_add_(1, hot, torch.rand(b * k, 24, generator=gen, device="cuda") * 6)
        x.scatter_(1, torch.randint(0, v, (b * k, 7), generator=gen, device="cuda"), -math.inf)
        st["logits"] = x.to(DTYPES[case["dtype"]])
        st["scores"] = -torch.rand(b, k, generator=gen, device="cuda").mul_(0.7).cumsum(1) - 20
        st["finished"] = torch.rand(b, k, generator=gen, device="cuda") < 0.15
        if own:
            import smallaios_b200 as sa

            st["sa"] = sa
        return st

    h, d, bits, b = case["H"], case["D"], case["bits"], case["B"]
    cb = d * bits // 8
    if op == "reorder":
        k, past = case["K"], case["past"]
        used = past // PAGE  # full pages, shared by the beams; each beam has one page of its own behind them
        pages = b * (used + k)
        order = torch.from_numpy(gen_np.permutation(pages).astype(np.int32)).cuda()
        shared, mine = order[:b * used].view(b, 1, used), order[b * used:].view(b, k, 1)
        st["table"] = torch.cat([shared.expand(b, k, used), mine], dim=-1).reshape(b * k, used + 1).contiguous()
        st["out"] = torch.empty_like(st["table"])
        st["lens"] = torch.full((b * k,), past, dtype=torch.int32, device="cuda")
        st["parents"] = torch.from_numpy(_parents(gen_np, b, k)).cuda()
        arrays = []
        if own:
            st["sa"], st["pages"] = _pool(case, pages)
        for i in range(case["L"]):
            layer = [torch.randint(0, 256, (pages, h, PAGE, cb), generator=gen, device="cuda", dtype=torch.uint8),
                     torch.randint(0, 256, (pages, h, 4, cb // 4, 4, 4, 4), generator=gen, device="cuda", dtype=torch.uint8),
                     torch.randn(pages, h, PAGE, 2, generator=gen, device="cuda"),
                     torch.randn(pages, h, PAGE, 2, generator=gen, device="cuda")]
            if own:
                view = st["pages"].view(i)
                held = [view.k_codes, view.v_codes, view.k_meta, view.v_meta]
                for dst, src in zip(held, layer):
                    dst.copy_(src)
                layer = held
            arrays.append(layer)
        st["arrays"] = arrays
        return st

    lens = _lengths(case)
    counts = _counts(case) if op == "append" else [1] * b
    need = [(n + c + PAGE - 1) // PAGE for n, c in zip(lens, counts)]
    pages, width = sum(need) + 1, max(need)  # one page that no sequence uses
    order = gen_np.permutation(pages).astype(np.int32)
    table = np.full((b, width), -1, np.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    st["table"] = torch.from_numpy(table).cuda()
    st["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    st["cos"], st["sin"] = _tables(width * PAGE, d)
    if own:
        st["sa"], st["pages"] = _pool(case, pages)
    else:
        st["signs"], st["lens_host"] = _signs(0, h, d), lens
    dtype = DTYPES[case["dtype"]]
    if op == "append":
        s = case["S"]
        if case["ragged"] and s > 1:
            st["counts"] = torch.tensor(counts, dtype=torch.int32, device="cuda")
        st["k"] = torch.randn(b, s, h * d, generator=gen, device="cuda").to(dtype)
        st["v"] = (torch.randn(b, s, h * d, generator=gen, device="cuda") * 0.5).to(dtype)
        arrays = [torch.randint(0, 256, (pages, h, PAGE, cb), generator=gen, device="cuda", dtype=torch.uint8),
                  torch.randint(0, 256, (pages, h, 4, cb // 4, 4, 4, 4), generator=gen, device="cuda", dtype=torch.uint8),
                  torch.randn(pages, h, PAGE, 2, generator=gen, device="cuda"),
                  torch.randn(pages, h, PAGE, 2, generator=gen, device="cuda")]
    else:
        # queries as the projection gives them; scores of standard deviation near 1.5
        st["q"] = (torch.randn(b, 1, h * case["G"] * d, generator=gen, device="cuda") * 1.3).to(dtype)
        k, km = _vectors(gen, pages, h, d, bits, 0.5)
        v, vm = _vectors(gen, pages, h, d, bits, 0.2)
        arrays = [k, _to_pool_v(v) if own else v, km, vm]
    if own:
        view = st["pages"].view(0)
        held = [view.k_codes, view.v_codes, view.k_meta, view.v_meta]
        for dst, src in zip(held, arrays):
            dst.copy_(src)
        arrays = held
    st["arrays"] = arrays
    return st


# ---- plain forms -----------------------------------------------------------------------------------
def _hadamard(d):
    """Walsh-Hadamard matrix: entry (i, j) is -1 to the number of common set bits of i and j."""
    i = torch.arange(d, device="cuda")
    common = (i[:, None] & i[None, :])[..., None] >> torch.arange(8, device="cuda")
    return 1.0 - 2.0 * ((common & 1).sum(-1) % 2).float()


def _rotate(x, positions, cos, sin, interleaved):
    """Rotary embedding of (..., n, heads, D) floats at positions (..., n); each product is rounded before the sum."""
    c, s = cos[positions][..., None, :], sin[positions][..., None, :]
    if interleaved:
        x0, x1 = x[..., 0::2], x[..., 1::2]
        return torch.stack([c * x0 - s * x1, s * x0 + c * x1], dim=-1).flatten(-2)
    x0, x1 = x.chunk(2, dim=-1)
    return torch.cat([c * x0 - s * x1, s * x0 + c * x1], dim=-1)


def _inv_sqrt(d):
    """The format's 1/sqrt(D): ten Newton steps from D, each operation rounded to 32 bits."""
    x = s = np.float32(d)
    for _ in range(10):
        s = np.float32(0.5) * np.float32(s + np.float32(x / s))
    return float(np.float32(1.0) / s)


def _encode(x, signs, bits):
    """Codes and {scale, zero point} of vectors (..., heads, D), every step rounded to 32 bits."""
    x = x * signs
    d, step = x.shape[-1], 1
    while step < d:
        y = x.unflatten(-1, (d // (2 * step), 2, step))
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).flatten(-3)
        step *= 2
    x = x * torch.tensor(_inv_sqrt(d), device="cuda")
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = hi - lo
    levels = torch.tensor(float(2 ** bits - 1), device="cuda")
    scale = torch.where(span > 0, span / levels, 1.0)
    t = (x - lo) / scale
    whole = t.trunc()
    c = (whole + (t - whole >= 0.5).float()).clamp(max=float(levels)).to(torch.uint8)  # half away from zero
    c = c if bits == 8 else c[..., 0::2] | (c[..., 1::2] << 4)
    return c, torch.cat([scale, lo], dim=-1)


def _append_plain(st):
    case = st["case"]
    b, s, h, d, bits = (case[x] for x in ("B", "S", "H", "D", "bits"))
    token = torch.arange(s, device="cuda")
    at = st["lens"].long()[:, None] + token  # (B, S) positions
    live = token < (st["counts"][:, None] if "counts" in st else s)
    k = _rotate(st["k"].float().view(b, s, h, d), torch.where(live, at, 0), st["cos"], st["sin"], case["interleaved"])
    k_codes, v_codes, k_meta, v_meta = st["arrays"]
    row, col = torch.where(live.expand(b, s))
    p = at[row, col]
    page, t = st["table"][row, p // PAGE].long(), p % PAGE
    c, m = _encode(k[row, col], st["signs"], bits)
    k_codes[page, :, t], k_meta[page, :, t] = c, m
    c, m = _encode(st["v"].float().view(b, s, h, d)[row, col], st["signs"], bits)
    v_codes[page, :, t // 16, :, t % 16 // 4, :, t % 4] = c.unflatten(-1, (-1, 4))
    v_meta[page, :, t] = m
    return [k_codes, v_codes, k_meta, v_meta]


def _attend_plain(st):
    case = st["case"]
    b, h, g, d, bits = (case[x] for x in ("B", "H", "G", "D", "bits"))
    k_codes, v_codes, k_meta, v_meta = st["arrays"]
    hadamard, signs = _hadamard(d), st["signs"].view(h, 1, d)
    q = _rotate(st["q"].float().view(b, 1, h * g, d), st["lens"].long()[:, None], st["cos"], st["sin"],
                case["interleaved"]).view(b, h, g, d)
    q = (q * signs) @ hadamard  # the pages' rotated frame

    def vectors(codes, meta, pages, n):  # (H, n, D)
        c = codes[pages].transpose(0, 1).flatten(1, 2)[:, :n]
        c = c if bits == 8 else torch.stack([c & 15, c >> 4], dim=-1).flatten(-2)
        m = meta[pages].transpose(0, 1).flatten(1, 2)[:, :n]
        return c.float() * m[..., :1] + m[..., 1:]

    out = torch.empty(b, h, g, d, device="cuda")
    for i, past in enumerate(st["lens_host"]):
        n = past + 1
        pages = st["table"][i, :(n + PAGE - 1) // PAGE].long()
        w = q[i] @ vectors(k_codes, k_meta, pages, n).transpose(-1, -2) * (1.0 / d)  # 1/sqrt(D) of rotation and scores
        e = (w - w.amax(-1, keepdim=True)).exp()
        out[i] = (e / e.sum(-1, keepdim=True)) @ vectors(v_codes, v_meta, pages, n)
    out = (out @ hadamard) * (signs / math.sqrt(d))
    return out.view(b, 1, h * g * d).to(st["q"].dtype)


def _select_plain(st):
    case = st["case"]
    b, k, v, keep = (case[x] for x in ("B", "K", "V", "keep"))
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - (top + (x - top).exp().sum(-1, keepdim=True).log())
    score = st["scores"].double().view(b * k, 1)
    done = st["finished"].view(b * k, 1)
    end = torch.arange(v, device="cuda") == END
    x = torch.where(done, torch.where(end, score, -math.inf), x + score)
    x = torch.where(x.isnan(), -math.inf, x).view(b, k * v)
    places = torch.arange(k * v, device="cuda")
    parents, tokens, scores = [], [], []
    for _ in range(keep):  # the best, the lowest place among equals; then the best of the others
        best = x.amax(-1, keepdim=True)
        place = torch.where(x == best, places, k * v).amin(-1, keepdim=True)
        x.scatter_(1, place, -math.inf)
        some = best > -math.inf
        parents.append(torch.where(some, place // v, -1))
        tokens.append(torch.where(some, place % v, -1))
        scores.append(best)
    return [torch.cat(parents, 1).int(), torch.cat(tokens, 1).int(), torch.cat(scores, 1).float()]


END = 2  # the token that ends a sequence


def _reorder_plain(st):
    case = st["case"]
    b, k, past = case["B"], case["K"], case["past"]
    used, fill = past // PAGE, past % PAGE
    parents = st["parents"].long()
    table = st["table"].view(b, k, -1)
    out = table.clone()
    out[:, :, :used] = table[:, :, :used].gather(1, parents[..., None].expand(b, k, used))
    # the page in use: a beam that goes on in its own slot keeps it, else the first slot that continues it; the
    # others take the pages of the beams that ended, in order, with a copy of the parent's rows
    slot = torch.arange(k, device="cuda")
    child = parents[:, :, None] == slot  # (B, slot, parent)
    first = torch.where(child, slot[:, None], k).amin(1)  # (B, parent)
    heir = torch.where(child.diagonal(dim1=1, dim2=2), slot, first)
    heirs = heir.gather(1, parents) == slot  # (B, slot)
    ended = ~child.any(1)
    rank = (~heirs).long().cumsum(1) - 1     # the number of a slot among those that take a page
    free = torch.where(ended, slot, k).sort(1)[0]
    source = torch.where(heirs, parents, free.gather(1, rank.clamp_min(0)).clamp_max(k - 1))
    if fill:
        out[:, :, used] = table[:, :, used].gather(1, source)
        copied = ~heirs
        dst = out[:, :, used][copied].long()
        src = table[:, :, used].gather(1, parents)[copied].long()
        t = torch.arange(fill, device="cuda")
        for k_codes, v_codes, k_meta, v_meta in st["arrays"]:
            for a in (k_codes, k_meta, v_meta):
                a[dst, :, :fill] = a[src, :, :fill]
            v_codes[dst[:, None], :, t // 16, :, t % 16 // 4, :, t % 4] = \
                v_codes[src[:, None], :, t // 16, :, t % 16 // 4, :, t % 4]
    return [out.view(b * k, -1), st["arrays"]]


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"append": _append_plain, "attend": _attend_plain, "select": _select_plain,
                "reorder": _reorder_plain}[op](state)
    sa, pages = state["sa"], state.get("pages")
    if op == "append":
        pages.append(0, state["k"], state["v"], state["table"], state["lens"], counts=state.get("counts"), do_rotary=True,
                     rotary_interleaved=case["interleaved"], cos_cache=state["cos"], sin_cache=state["sin"])
        return state["arrays"]
    if op == "attend":
        return sa.gqa_paged_attend(state["q"], pages, 0, state["table"], state["lens"], num_heads=case["H"] * case["G"],
                                   do_rotary=True, rotary_interleaved=case["interleaved"], cos_cache=state["cos"],
                                   sin_cache=state["sin"])
    if op == "select":
        return list(sa.beam_select(state["logits"], state["scores"], finished=state["finished"], end_token=END,
                                   keep=case["keep"]))
    return [pages.reorder_beams(state["table"], state["lens"], state["parents"], out=state["out"]), state["arrays"]]


# ---- the definitions in 64 bits ----------------------------------------------------------------------
def _walsh64(x):
    """Walsh-Hadamard transform of the last axis, by butterflies."""
    d, step = x.shape[-1], 1
    while step < d:
        y = x.reshape(*x.shape[:-1], d // (2 * step), 2, step)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], dim=-2).reshape(x.shape)
        step *= 2
    return x


def _round32(x):
    """64-bit values rounded to 32 bits: a sum, product or quotient of 32-bit values comes out as 32 bits give it."""
    return x.float().double()


def _append_exact(st):
    """The format's definition: each operation is exact, then rounded to 32 bits."""
    case = st["case"]
    b, h, d, bits = case["B"], case["H"], case["D"], case["bits"]
    out = [a.clone() for a in st["arrays"]]
    signs, root = st["signs"].double(), _inv_sqrt(d)
    counts = _counts(case)
    for i in range(b):
        p = st["lens_host"][i] + torch.arange(counts[i], device="cuda")
        page, t = st["table"][i].long()[p // PAGE], p % PAGE
        cos, sin = st["cos"][p].double()[:, None], st["sin"][p].double()[:, None]
        for which, name in enumerate(("k", "v")):
            x = st[name][i, :counts[i]].double().view(-1, h, d)
            if which == 0:
                pair = (slice(0, None, 2), slice(1, None, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
                x0, x1 = x[..., pair[0]].clone(), x[..., pair[1]].clone()
                x[..., pair[0]] = _round32(_round32(cos * x0) - _round32(sin * x1))
                x[..., pair[1]] = _round32(_round32(sin * x0) + _round32(cos * x1))
            x = x * signs
            for step in [1 << j for j in range(d.bit_length() - 1)]:
                index = torch.arange(d, device="cuda")
                other = x[..., index ^ step]
                x = _round32(torch.where((index & step) == 0, x + other, other - x))
            x = _round32(x * root)
            lo = x.min(-1, keepdim=True)[0]
            span = _round32(x.max(-1, keepdim=True)[0] - lo)
            scale = torch.where(span > 0, _round32(span / (2 ** bits - 1)), 1.0)
            code = torch.floor(_round32(_round32(x - lo) / scale) + 0.5).clamp(max=2 ** bits - 1).to(torch.uint8)
            if bits == 4:
                code = code[..., 0::2] + 16 * code[..., 1::2]
            if which == 0:
                out[0][page, :, t] = code
            else:
                for j in range(4):  # byte j of each group of four, in the pool's order of V
                    out[1][page, :, t // 16, :, t % 16 // 4, j, t % 4] = code[..., j::4]
            out[2 + which][page, :, t] = torch.cat([scale, lo], dim=-1).float()
    return out


def _attend_exact(st):
    case = st["case"]
    b, h, g, d, bits = (case[x] for x in ("B", "H", "G", "D", "bits"))
    k_codes, v_codes, k_meta, v_meta = st["arrays"]
    out = torch.zeros(b, h, g, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = st["lens_host"][i] + 1
        pages = st["table"][i, :(n + PAGE - 1) // PAGE].long()
        q = st["q"][i, 0].double().view(h, g, d)
        c, s = st["cos"][n - 1].double(), st["sin"][n - 1].double()
        r = torch.empty_like(q)
        pair = (slice(0, None, 2), slice(1, None, 2)) if case["interleaved"] else (slice(0, d // 2), slice(d // 2, d))
        r[..., pair[0]] = c * q[..., pair[0]] - s * q[..., pair[1]]
        r[..., pair[1]] = s * q[..., pair[0]] + c * q[..., pair[1]]
        for e in range(h):
            def head(codes, meta):  # the vectors themselves, (n, D)
                byte = codes[pages, e].reshape(-1, codes.shape[-1])[:n]
                if bits == 4:
                    x = torch.empty(n, d, dtype=torch.float64, device="cuda")
                    x[:, 0::2], x[:, 1::2] = (byte % 16).double(), (byte // 16).double()
                else:
                    x = byte.double()
                m = meta[pages, e].reshape(-1, 2)[:n].double()
                return st["signs"][e].double() * _walsh64(x * m[:, :1] + m[:, 1:]) / math.sqrt(d)

            w = torch.softmax(torch.einsum("gd,td->gt", r[e], head(k_codes, k_meta)) / math.sqrt(d), dim=-1)
            out[i, e] = torch.einsum("gt,td->gd", w, head(v_codes, v_meta))
    return out.view(b, 1, h * g * d)


def _select_exact(st):
    case = st["case"]
    b, k, v, keep = (case[x] for x in ("B", "K", "V", "keep"))
    parents = torch.full((b, keep), -1, dtype=torch.int32, device="cuda")
    tokens, scores = parents.clone(), torch.full((b, keep), -math.inf, dtype=torch.float64, device="cuda")
    for i in range(b):
        total = torch.log_softmax(st["logits"][i * k:(i + 1) * k].double(), dim=-1) + st["scores"][i].double()[:, None]
        for j in range(k):
            if st["finished"][i, j]:
                total[j] = -math.inf
                total[j, END] = st["scores"][i, j].double()
        flat = torch.nan_to_num(total.flatten(), nan=-math.inf, neginf=-math.inf)
        value, place = torch.sort(flat, descending=True, stable=True)
        n = min(keep, int((value > -math.inf).sum()))
        parents[i, :n], tokens[i, :n], scores[i, :n] = (place[:n] // v).int(), (place[:n] % v).int(), value[:n]
    return [parents, tokens, scores]


def exact(case, seed):
    global own
    if case["op"] == "reorder":
        return None  # bytes that move
    was, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = was
    return {"append": _append_exact, "attend": _attend_exact, "select": _select_exact}[case["op"]](st)
