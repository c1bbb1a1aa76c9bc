"""Timed cases of the paged packed-cache operators: appending rotated keys and values to a paged
1-bit-per-plane cache, decode attention over its pages (capped, biased and windowed scores), and
decode attention of a batch that shares a prefix.

A cache tensor (K or V) is a pool of pages: code and res are int32 words [pages, kv_heads,
page_size, D/32] (element i at bit i & 31 of word i >> 5), norms and rnorms float32 [pages,
kv_heads, page_size].  A row stands for  d * H(norm c[code] / sqrt(D) + rnorm g / D sign)  with H
the Walsh-Hadamard matrix, g = 1 for keys and sqrt(2/pi) for values.
"""
import math
import sys

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_C = math.sqrt(2.0 / math.pi)  # the two levels of N(0, 1)


def listed():
    return [
        # one new token of one sequence: the smallest append, all latency
        _append("append: one token", 1, 8, 128, "bf16", 128, False, 64),
        # one decode step of a batch of 64
        _append("append: batch step", 64, 8, 128, "bf16", 128, False, 64),
        # the prompts of four sequences of 8192 tokens
        _append("append: prompts", 32768, 8, 128, "bf16", 128, False, 64),
        # one prompt of an odd length, wide heads, a quarter of each head rotated in adjacent pairs
        _append("append: odd prompt, D 256", 5003, 4, 256, "fp16", 64, True, 48),
        # one short conversation, grouped queries
        _decode("decode: one sequence", 1, 8, 4, 128, "bf16", 1537, 64),
        # a serving batch of uneven conversations, grouped queries
        _decode("decode: ragged batch", 32, 8, 4, 128, "bf16", 8192, 64),
        # long contexts, a query head for each cached head, capped scores
        _decode("decode: long, capped", 8, 16, 1, 128, "fp32", 40000, 64, softcap=30.0),
        # wide heads, a sliding window and a bias by distance, pages of an odd size
        _decode("decode: window, slopes, D 256", 24, 4, 8, 256, "fp16", 16384, 48, window=4096, slopes=True),
        # four samples of one short prompt
        _prefix("prefix: four samples", 4, 8, 4, 128, "bf16", 1024, 128, 64),
        # requests behind one system prompt
        _prefix("prefix: system prompt", 64, 8, 4, 128, "bf16", 8192, 512, 64),
        # many questions about one long document
        _prefix("prefix: long document", 128, 8, 4, 128, "bf16", 32768, 1024, 64),
        # an odd batch, odd grouping, wide heads, capped scores
        _prefix("prefix: odd, D 256, capped", 13, 4, 7, 256, "fp16", 5001, 700, 48, softcap=50.0),
    ]


def _append(name, tokens, heads, dim, dtype, rot, inter, page):
    return {"name": name, "op": "append", "tokens": tokens, "kv_heads": heads, "dim": dim, "dtype": dtype,
            "rot": rot, "interleaved": inter, "page": page}


def _decode(name, batch, heads, nq, dim, dtype, length, page, window=0, softcap=0.0, slopes=False):
    return {"name": name, "op": "decode", "batch": batch, "kv_heads": heads, "n_q": nq, "dim": dim,
            "dtype": dtype, "prefix": 0, "length": length, "page": page, "window": window,
            "softcap": softcap, "slopes": slopes}


def _prefix(name, batch, heads, nq, dim, dtype, prefix, suffix, page, softcap=0.0):
    return {"name": name, "op": "prefix", "batch": batch, "kv_heads": heads, "n_q": nq, "dim": dim,
            "dtype": dtype, "prefix": prefix, "length": suffix, "page": page, "window": 0,
            "softcap": softcap, "slopes": False}


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "prefix", "prefix"])
    dim = rng.choice([128, 128, 256])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    heads = rng.choice([1, 2, 4, 5, 8])
    page = rng.choice([16, 32, 48, 64, 100, 128, 256])
    if op == "append":
        tokens = _between(rng, 1, 16000)
        rot = rng.choice([dim, dim, dim // 2, 64, 32])
        c = _append("", tokens, heads, dim, dtype, rot, rng.random() < 0.3, page)
    elif op == "decode":
        batch, nq = _between(rng, 1, 48), rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        length = _between(rng, 2, min(32768, 3000000 // (batch * heads * (dim // 128))))
        c = _decode("", batch, heads, nq, dim, dtype, length, page, window=rng.choice([0, 0, max(1, length // 3)]),
                    softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3)
    else:
        batch, nq = _between(rng, 2, 96), rng.choice([1, 2, 3, 4, 5, 6, 7, 8])
        prefix = _between(rng, 64, 16000)
        suffix = _between(rng, 1, 700)
        c = _prefix("", batch, heads, nq, dim, dtype, prefix, suffix, page, softcap=rng.choice([0.0, 0.0, 50.0]))
    del c["name"]
    return c


def work(case):
    D, H = case["dim"], case["kv_heads"]
    elt = 4 if case["dtype"] == "fp32" else 2
    row = 2 * (D // 4 + 8)  # K and V: two planes and two norms each
    if case["op"] == "append":
        T, R = case["tokens"], case["rot"]
        rows = 2 * T * H
        return {"bytes": rows * D * elt + T * H * row + T * (4 * R + 16), "flops": rows * D * (math.log2(D) + 6) + 3 * T * H * R}
    B, nq = case["batch"], case["n_q"]
    lens = _lengths(case)
    keep = [min(n, case["window"]) if case["window"] else n for n in lens]
    rows = case["prefix"] + sum(n - case["prefix"] for n in keep)
    pairs = sum(keep) * H * nq
    return {"bytes": rows * H * row + 2 * B * H * nq * D * elt, "flops": 4.0 * D * pairs}


def _lengths(case):
    """Cached tokens of each sequence: the longest has them all, the others spread below it."""
    B, n, P = case["batch"], case["length"], case["prefix"]
    return [P + max(1, n - (n * 7 * b // 8) // max(1, B - 1)) for b in range(B)]


def _hadamard(D, dtype, device):
    h = torch.ones(1, 1, dtype=dtype, device=device)
    while h.shape[0] < D:
        h = torch.cat([torch.cat([h, h], 1), torch.cat([h, -h], 1)], 0)
    return h


def _levels(D):
    c = torch.tensor(_C / math.sqrt(D), dtype=torch.float32)
    return torch.stack([-c, c])


def _signs(D, g):
    return (torch.randint(0, 2, (D,), generator=g) * 2 - 1).to(torch.float32)


def _words(bits):
    """Truth values [..., D] as int32 words [..., D/32]."""
    b = bits.reshape(*bits.shape[:-1], -1, 32).to(torch.int64)
    w = (b << torch.arange(32, device=b.device)).sum(-1)
    return (w - ((w >> 31) << 32)).to(torch.int32)


def _bits(words):
    """int32 words [..., W] as truth values [..., 32 W]."""
    b = (words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return b.reshape(*words.shape[:-1], -1) != 0


def _encode(x, d, c):
    """Rows of x (64 bits): their code and residual bits and both norms."""
    D = x.shape[-1]
    norm = x.square().sum(-1, keepdim=True).sqrt()
    norm = torch.where(norm == 0, torch.full_like(norm, 1e-8), norm)
    y = (x * d) @ _hadamard(D, x.dtype, x.device) / math.sqrt(D) / norm
    bit = y > (c[0] + c[1]) / 2
    v = y - torch.where(bit, c[1], c[0])
    rnorm = norm * v.square().sum(-1, keepdim=True).sqrt()
    rnorm = torch.where(rnorm == 0, torch.full_like(rnorm, 1e-8), rnorm)
    return bit, v >= 0, norm[..., 0], rnorm[..., 0]


# ------------------------------------------------------------------ inputs


def prepare(case, seed):
    return _prepare_append(case, seed) if case["op"] == "append" else _prepare_attend(case, seed)


def _generators(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed)), torch.Generator().manual_seed(int(seed) + 7)


def _empty_pool(pages, H, page, D):
    return {"code": torch.zeros(pages, H, page, D // 32, dtype=torch.int32, device="cuda"),
            "res": torch.zeros(pages, H, page, D // 32, dtype=torch.int32, device="cuda"),
            "norms": torch.zeros(pages, H, page, dtype=torch.float32, device="cuda"),
            "rnorms": torch.zeros(pages, H, page, dtype=torch.float32, device="cuda")}


def _kv(shape, g, scale):
    """Normal values with a few large channels, as keys and values have them."""
    x = torch.randn(*shape, device="cuda", generator=g)
    x[..., 5::47] *= scale
    return x


def _prepare_append(case, seed):
    g, gc = _generators(seed)
    T, H, D, R, page = case["tokens"], case["kv_heads"], case["dim"], case["rot"], case["page"]
    dt = _TYPES[case["dtype"]]
    pages = -(-T // page) + 3
    # a sequence's tokens lie in its pages in order, the pages anywhere in the pool
    order = torch.randperm(pages, device="cuda", generator=g)
    at = torch.arange(T, device="cuda") + 1
    s = {"op": "append", "slots": order[at // page] * page + at % page,
         "positions": torch.arange(T, device="cuda") + 4000, "interleaved": case["interleaved"]}
    s["k"] = _kv((T, H, D), g, 6.0).to(dt)
    s["v"] = _kv((T, H, D), g, 3.0).to(dt)
    angle = torch.arange(4000 + T, dtype=torch.float64, device="cuda")[:, None] * \
        10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64, device="cuda") / R)
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    s["dk"], s["dv"], s["c"] = _signs(D, gc), _signs(D, gc), _levels(D)
    s["kc"], s["vc"] = _empty_pool(pages, H, page, D), _empty_pool(pages, H, page, D)
    return s


def _fill(pool, d, c, g, scale):
    """Every row of the pool, the unused ones too, from rows of normal values."""
    n = pool["norms"].numel()
    D = d.numel()
    hd = d[:, None] * _hadamard(D, torch.float32, "cuda") / math.sqrt(D)
    for a in range(0, n, 1 << 20):
        x = _kv((min(1 << 20, n - a), D), g, scale)
        norm = x.square().sum(-1).sqrt()
        y = x @ hd / norm[:, None]
        bit = y > 0
        v = y - torch.where(bit, c[1], c[0])
        b = a + x.shape[0]
        pool["code"].view(n, -1)[a:b] = _words(bit)
        pool["res"].view(n, -1)[a:b] = _words(v >= 0)
        pool["norms"].view(n)[a:b] = norm
        pool["rnorms"].view(n)[a:b] = norm * v.square().sum(-1).sqrt()


def _prepare_attend(case, seed):
    g, gc = _generators(seed)
    B, H, nq, D, page, P = (case[k] for k in ("batch", "kv_heads", "n_q", "dim", "page", "prefix"))
    dt = _TYPES[case["dtype"]]
    lens = _lengths(case)
    shared = P // page  # whole pages of the prefix; a page that it ends in is each sequence's own
    width = -(-max(lens) // page)
    owned = [-(-n // page) - shared for n in lens]
    pages = shared + sum(owned) + 2
    order = torch.randperm(pages, generator=gc).to(torch.int32)
    table = torch.zeros(B, width, dtype=torch.int32)
    at = shared
    for b in range(B):
        table[b, :shared] = order[:shared]
        table[b, shared:shared + owned[b]] = order[at:at + owned[b]]
        at += owned[b]
    s = {"op": case["op"], "prefix": P, "max_len": max(lens), "window": case["window"],
         "softcap": case["softcap"], "table": table.cuda(),
         "lengths": torch.tensor(lens, dtype=torch.int32, device="cuda")}
    s["dk"], s["dv"], s["c"] = _signs(D, gc), _signs(D, gc), _levels(D)
    s["kc"], s["vc"] = _empty_pool(pages, H, page, D), _empty_pool(pages, H, page, D)
    cc = s["c"].cuda()
    _fill(s["kc"], s["dk"].cuda(), cc, g, 4.0)
    _fill(s["vc"], s["dv"].cuda(), cc, g, 2.0)
    if P % page:  # the tail of the prefix is in every sequence's copy of that page
        first = table[0, shared].item()
        for pool in (s["kc"], s["vc"]):
            for t in pool.values():
                t[s["table"][:, shared].long(), :, :P % page] = t[first, :, :P % page].clone()
    s["q"] = torch.randn(B, H * nq, D, device="cuda", generator=g).to(dt)
    s["slopes"] = None
    if case["slopes"]:
        s["slopes"] = 2.0 ** (-8.0 * (torch.arange(H * nq, device="cuda", dtype=torch.float32) + 1) / (H * nq))
    return s


# ------------------------------------------------------------------ passes


def run(s):
    if own:
        if "kudahitam-quant_b200" not in sys.path:
            sys.path.insert(0, "kudahitam-quant_b200")
        from kudahitam import ops
        kc, vc = _packed(ops, s["kc"]), _packed(ops, s["vc"])
        if s["op"] == "append":
            ops.paged_append(s["k"], s["v"], kc, vc, s["slots"], s["dk"], s["dv"], s["c"],
                             positions=s["positions"], cos=s["cos"], sin=s["sin"],
                             interleaved=s["interleaved"])
            return [s["kc"], s["vc"]]
        if s["op"] == "prefix":
            return ops.paged_prefix_attention(s["q"], kc, vc, s["table"], s["lengths"], s["prefix"],
                                              s["dk"], s["dv"], s["c"], max_len=s["max_len"],
                                              softcap=s["softcap"])
        return ops.paged_decode_attention(s["q"], kc, vc, s["table"], s["lengths"], s["dk"], s["dv"],
                                          s["c"], max_len=s["max_len"], window=s["window"],
                                          softcap=s["softcap"], slopes=s["slopes"])
    return _plain_append(s) if s["op"] == "append" else _plain_attend(s)


def _packed(ops, pool):
    P, H, page, W = pool["code"].shape
    return ops.PackedKV((P, H, page, 32 * W), 1, pool["code"].view(-1, W), pool["norms"].view(-1),
                        pool["res"].view(-1, W), pool["rnorms"].view(-1))


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] elements of each row turned by their angles."""
    R = 2 * cos.shape[-1]
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    p, q = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([p, q], -1).flatten(-2) if interleaved else torch.cat([p, q], -1)
    return torch.cat([turned, x[..., R:]], -1)


def _plain_append(s):
    # bits next to a border need 64 bits
    c = s["c"].double().cuda()
    cos, sin = s["cos"].double()[s["positions"]][:, None], s["sin"].double()[s["positions"]][:, None]
    k = _rotate(s["k"].double(), cos, sin, s["interleaved"])
    page = s["kc"]["norms"].shape[2]
    at, off = s["slots"] // page, s["slots"] % page
    _put(s["kc"], at, off, _encode(k, s["dk"].double().cuda(), c))
    _put(s["vc"], at, off, _encode(s["v"].double(), s["dv"].double().cuda(), c))
    return [s["kc"], s["vc"]]


def _put(pool, at, off, coded):
    bit, res, norm, rnorm = coded
    pool["code"][at, :, off] = _words(bit)
    pool["res"][at, :, off] = _words(res)
    pool["norms"][at, :, off] = norm.float()
    pool["rnorms"][at, :, off] = rnorm.float()


def _values(pool, c, at, off, gain):
    """Rows at (page, offset) in the transformed domain: [..., H, D] in 32 bits."""
    D = 32 * pool["code"].shape[-1]
    a = torch.where(_bits(pool["code"][at, :, off]), c[1], c[0]) * (pool["norms"][at, :, off] * gain[0])[..., None]
    r = (pool["rnorms"][at, :, off] * (gain[1] / D))[..., None]
    return torch.where(_bits(pool["res"][at, :, off]), a + r, a - r)


def _plain_attend(s):
    page, H = s["kc"]["norms"].shape[2], s["kc"]["norms"].shape[1]
    B, Hq, D = s["q"].shape
    P, c = s["prefix"], s["c"].cuda()
    kgain, vgain = (1.0, math.sqrt(D)), (1.0 / math.sqrt(D), math.sqrt(2.0 / math.pi))
    q = (s["q"].float() * s["dk"].cuda()) @ _hadamard(D, torch.float32, "cuda") / math.sqrt(D)
    q = q.view(B, H, Hq // H, D)
    pos = torch.arange(s["max_len"], device="cuda")
    own_pos = pos[P:]
    at, off = s["table"].long()[:, own_pos // page], (own_pos % page).expand(B, -1)
    k = _values(s["kc"], c, at, off, kgain)  # [B, S, H, D]
    t = torch.einsum("bhnd,bshd->bhns", q, k)
    del k
    if P:
        first = s["table"].long()[0, pos[:P] // page]
        k = _values(s["kc"], c, first, pos[:P] % page, kgain)  # [P, H, D]
        t = torch.cat([torch.einsum("bhnd,shd->bhns", q, k), t], -1)
        del k
    t = t / math.sqrt(D)
    if s["softcap"]:
        t = s["softcap"] * torch.tanh(t / s["softcap"])
    last = (s["lengths"].long() - 1)[:, None, None, None]
    if s["slopes"] is not None:
        t = t - s["slopes"].view(1, H, -1, 1) * (last - pos)
    hidden = pos > last
    if s["window"]:
        hidden = hidden | (pos <= last - s["window"])
    t = t.masked_fill(hidden, -math.inf)
    p = (t - t.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    p = p.double() if s["q"].dtype == torch.float32 else p  # a long sum of values of either sign
    v = _values(s["vc"], c, at, off, vgain).to(p.dtype)
    o = torch.einsum("bhns,bshd->bhnd", p[..., P:], v)
    del v
    if P:
        o = o + torch.einsum("bhns,shd->bhnd", p[..., :P], _values(s["vc"], c, first, pos[:P] % page, vgain).to(p.dtype))
    o = o.float() @ _hadamard(D, torch.float32, "cuda") * s["dv"].cuda()
    return o.reshape(B, Hq, D).to(s["q"].dtype)


# ------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if s["op"] == "append" else _exact_attend(s)


def _walsh(x):
    """The Walsh-Hadamard sums of the rows of x, one butterfly after another."""
    D, h = x.shape[-1], 1
    while h < D:
        y = x.reshape(*x.shape[:-1], D // (2 * h), 2, h)
        x = torch.stack([y[..., 0, :] + y[..., 1, :], y[..., 0, :] - y[..., 1, :]], -2).reshape(x.shape)
        h *= 2
    return x


def _exact_append(s):
    R, D = 2 * s["cos"].shape[1], s["k"].shape[-1]
    k = s["k"].to(torch.float64).clone()
    half = torch.arange(R // 2, device="cuda")
    i, j = (2 * half, 2 * half + 1) if s["interleaved"] else (half, half + R // 2)
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"]].unsqueeze(1)
    z = torch.complex(k[..., i], k[..., j]) * turn
    k[..., i], k[..., j] = z.real, z.imag
    c0, c1 = s["c"].double().tolist()
    for x, d, pool in ((k, s["dk"], s["kc"]), (s["v"].double(), s["dv"], s["vc"])):
        norm = x.square().sum(-1).sqrt().clamp_min(1e-8)
        y = _walsh(x * d.double().cuda()) / (norm * math.sqrt(D))[..., None]
        near = ((y - c1).abs() < (y - c0).abs())
        left = y - (c0 + (c1 - c0) * near.double())
        rnorm = (norm * left.square().sum(-1).sqrt()).clamp_min(1e-8)
        page = pool["norms"].shape[2]
        for name, value in (("norms", norm), ("rnorms", rnorm)):
            pool[name] = pool[name].double().transpose(1, 2).reshape(-1, x.shape[1]).index_copy(0, s["slots"], value)
            pool[name] = pool[name].view(-1, page, x.shape[1]).transpose(1, 2).contiguous()
        pool["code"] = pool["res"] = None
    return [s["kc"], s["vc"]]


def _exact_attend(s):
    B, Hq, D = s["q"].shape
    H, page = s["kc"]["norms"].shape[1:3]
    c0, c1 = s["c"].double().tolist()
    qt = _walsh(s["q"].double() * s["dk"].double().cuda()) / math.sqrt(D)
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    lens = s["lengths"].tolist()

    def rows(pool, ids, h, wide, gain):
        take = lambda t: t[:, h].reshape(-1, *t.shape[3:])[ids]  # noqa: E731
        word = torch.arange(D, device="cuda")
        code = (take(pool["code"])[:, word // 32] >> (word % 32).int()) % 2
        res = (take(pool["res"])[:, word // 32] >> (word % 32).int()) % 2
        return take(pool["norms"]).double()[:, None] * wide * (c0 + (c1 - c0) * code) + \
            take(pool["rnorms"]).double()[:, None] * gain * (2 * res - 1)

    for b in range(B):
        n = lens[b]
        lo = max(0, n - s["window"]) if s["window"] else 0
        pos = torch.arange(lo, n, device="cuda")
        ids = s["table"].long()[b, pos // page] * page + pos % page
        for h in range(H):
            heads = slice(h * (Hq // H), (h + 1) * (Hq // H))
            t = qt[b, heads] @ rows(s["kc"], ids, h, 1.0, 1.0 / math.sqrt(D)).T / math.sqrt(D)
            if s["softcap"]:
                t = torch.tanh(t / s["softcap"]) * s["softcap"]
            if s["slopes"] is not None:
                t = t + s["slopes"][heads].double()[:, None] * (pos - (n - 1))
            v = rows(s["vc"], ids, h, 1.0 / math.sqrt(D), math.sqrt(2.0 / math.pi) / D)
            out[b, heads] = torch.softmax(t, -1) @ v
    return _walsh(out) * s["dv"].double().cuda()
