"""Plain 64-bit forms of the paged cache operators, and paged inputs, for the tests."""
from __future__ import annotations

import math

import torch

import khtest as K
from kudahitam import lloyd_max, ops, rademacher

G = math.sqrt(2.0 / math.pi)


def hadamard(D: int) -> torch.Tensor:
    return torch.from_numpy(K.hadamard(D))


def unpack(words: torch.Tensor) -> torch.Tensor:
    w = words.long().unsqueeze(-1) >> torch.arange(32)
    return (w & 1).reshape(*words.shape[:-1], -1)


def rotate(x, cos, sin, interleaved):
    """x [T, H, D] in 64 bits, cos / sin [T, R/2]."""
    R = 2 * cos.shape[-1]
    cos, sin = cos.double()[:, None], sin.double()[:, None]
    y = x.clone()
    a = slice(0, R, 2) if interleaved else slice(0, R // 2)
    b = slice(1, R, 2) if interleaved else slice(R // 2, R)
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., b] * cos + x[..., a] * sin
    return y


def compress(x, d, c):
    """(code, res, norm, rnorm) of the rows of x in 64 bits; bits as 0 / 1."""
    D = x.shape[-1]
    norm = x.square().sum(-1).sqrt()
    norm = torch.where(norm == 0, 1e-8, norm)
    y = (x * d.double()) @ hadamard(D) / (norm * math.sqrt(D)).unsqueeze(-1)
    c = c.double()
    code = (y > (c[0] + c[1]) / 2).long()
    v = y - c[code]
    rn = norm * v.square().sum(-1).sqrt()
    return code, (v >= 0).long(), norm, torch.where(rn == 0, 1e-8, rn)


def rows(p: ops.PackedKV, c, key: bool) -> torch.Tensor:
    """Rotated-domain values of every row of a pool (keys: the score's vector)."""
    D = p.head_dim
    code, res = unpack(p.code.cpu()), unpack(p.res.cpu())
    n, rn = p.norms.cpu().double(), p.rnorms.cpu().double()
    a, b = (1.0, 1.0 / math.sqrt(D)) if key else (1.0 / math.sqrt(D), G / D)
    return n[:, None] * a * c.double()[code] + rn[:, None] * b * (2 * res - 1)


def attention(q, kc, vc, table, lengths, dk, dv, c, sm_scale=None, starts=None, window=0,
              softcap=0.0, slopes=None):
    """(out, lse, spread, reach, peak, largest): 64-bit attention of every query
    row; spread is sum p |V_hat|, reach the largest |q| |K| sm_scale among its
    rows, peak the same with sqrt(D) max |q~| for |q|, largest the rows' largest
    p |V_hat| times the square root of their number."""
    B, Hq, D = q.shape
    P, H, page, _ = kc.shape
    nq = Hq // H
    scale = 1 / math.sqrt(D) if sm_scale is None else sm_scale
    kv, vv = rows(kc, c, True).view(P, H, page, D), rows(vc, c, False).view(P, H, page, D)
    qt = (q.cpu().double() * dk.double()) @ hadamard(D) / math.sqrt(D)
    out = torch.zeros(B, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    spread, reach, peak, largest = (torch.zeros(B, Hq, dtype=torch.float64) for _ in range(4))
    table = table.cpu().long()
    for b in range(B):
        n = int(lengths[b])
        lo = max(0, int(starts[b]) if starts is not None else 0, n - window if window else 0)
        if lo >= n:
            continue
        j = torch.arange(lo, n)
        pg, off = table[b, j // page], j % page
        for hq in range(Hq):
            h = hq // nq
            k, v = kv[pg, h, off], vv[pg, h, off]
            t = k @ qt[b, hq] * scale
            if softcap:
                t = softcap * torch.tanh(t / softcap)
            if slopes is not None:
                t = t - float(slopes[hq]) * (n - 1 - j)
            lse[b, hq] = torch.logsumexp(t, 0)
            p = torch.exp(t - lse[b, hq])
            out[b, hq] = p @ v
            spread[b, hq] = p @ v.norm(dim=-1) * math.sqrt(D)
            reach[b, hq] = k.norm(dim=-1).max() * qt[b, hq].norm() * abs(scale)
            peak[b, hq] = k.norm(dim=-1).max() * qt[b, hq].abs().max() * math.sqrt(D) * abs(scale)
            largest[b, hq] = (p * v.norm(dim=-1)).max() * math.sqrt(D * len(p))
    return (out @ hadamard(D)) * dv.double(), lse, spread, reach, peak, largest


def check(got, lse, want, dtype):
    """Holds an output (and lse, or None) to the accuracy that the operators document.

    A score is off by at most `ds` (the cap and the bias do not enlarge that):
      fp32 queries: 2^-20 |q| |K| sm_scale (32-bit transforms, q~ in 32-bit fixed
      point, sums of whole numbers);
      16-bit ones: q~ in fixed point, off by 2^-13 of its largest element for a
      quarter of the elements, half of that for the next and so on, in the
      2-norm sqrt(D / 4 (1 + 1/4 + 1/16 + 1/64)) 2^-13 max |q~|, which is under
      2^-13.7 sqrt(D) max |q~|;  bf16 may take the tensor-core prefix instead:
      two operands rounded to fp16, 2^-11 |q| |K| sm_scale.
    p is off by twice that, relatively, as numerator and denominator move
    apart.  The weighted sum adds `dw` sum p |V_hat| (2^-20; 2^-11 for bf16, two
    fp16 operands) and roundings of the weights to 2^-14 (2^-24 for fp32 queries)
    of the largest weight of a unit: independent, so the root of their number
    counts, 1 / sqrt(12) of a step each; a whole 2^-14 is over 3 deviations.
    The output's own rounding is half a step."""
    out, ref_lse, spread, reach, peak, largest = want
    ds, dw = 2.0 ** -20 * reach, 2.0 ** -20
    if dtype != torch.float32:
        ds = ds + 2.0 ** -13.7 * peak
    if dtype == torch.bfloat16:
        ds, dw = torch.maximum(ds, 2.0 ** -11 * reach), 2.0 ** -11
    extra = 2.0 ** (-24 if dtype == torch.float32 else -14) * largest
    got = got.detach().cpu().double()
    # a value past the type's largest rounds to an infinity of its sign
    over = torch.isinf(got) & (out.abs() >= torch.finfo(dtype).max) & (got.sign() == out.sign())
    got = torch.where(over, out, got)
    off = (got - out).norm(dim=-1)
    most = (2 * ds + dw) * spread + extra + torch.finfo(dtype).eps / 2 * out.norm(dim=-1)
    bad = off > most
    assert torch.isfinite(got).all()
    assert not bad.any(), (off[bad].max(), most[bad].min(), bad.nonzero()[:4].tolist())
    if lse is not None:
        lse = lse.detach().cpu().double()
        none = torch.isinf(ref_lse)
        assert torch.equal(torch.isinf(lse), none) and (lse[none] < 0).all()
        # the logarithm and its parts are 32-bit: 2^-22 of its size
        dl = (lse - ref_lse).abs()[~none]
        ml = (ds + 2.0 ** -20 + 2.0 ** -22 * ref_lse.abs())[~none]
        assert (dl <= ml).all(), (dl.max(), ml.min())


def pools(pages, H, page, D, seed, scale=3.0):
    """Two pools whose every row is a compressed row, built by the 64-bit form."""
    g = torch.Generator().manual_seed(seed)
    dk, dv, c = rademacher(D, 2 * seed), rademacher(D, 2 * seed + 1), lloyd_max(1, D)
    out = []
    for d in (dk, dv):
        x = torch.randn(pages * H * page, D, generator=g, dtype=torch.float64)
        x[:, 3::41] *= scale
        code, res, norm, rnorm = compress(x, d, c)
        out.append(ops.PackedKV((pages, H, page, D), 1, words(code), norm.float(), words(res),
                                rnorm.float()))
    return out[0], out[1], dk, dv, c


def words(bits):
    b = bits.reshape(*bits.shape[:-1], -1, 32) << torch.arange(32)
    w = b.sum(-1)
    return (w - ((w >> 31) << 32)).int()


def cuda(p: ops.PackedKV) -> ops.PackedKV:
    return ops.PackedKV(p.shape, p.bits, p.code.cuda(), p.norms.cuda(), p.res.cuda(),
                        p.rnorms.cuda())


def tables(lengths, page, pages, seed, prefix=0):
    """A block table of distinct pages per sequence (whole pages of the prefix
    shared); entries past a sequence's length are far out of range."""
    g = torch.Generator().manual_seed(seed)
    order = torch.randperm(pages, generator=g).int()
    shared = prefix // page
    width = max(1, max(-(-n // page) for n in lengths))
    t = torch.full((len(lengths), width), 1 << 30, dtype=torch.int32)
    at = shared
    for b, n in enumerate(lengths):
        need = -(-n // page)
        t[b, :min(shared, need)] = order[:min(shared, need)]
        own = max(0, need - shared)
        t[b, shared:shared + own] = order[at:at + own]
        at += own
    assert at <= pages
    return t


def poison(kc, vc, table, lengths, starts=None):
    """Norms of every row that no sequence attends become NaN, its bits all set."""
    P, H, page, D = kc.shape
    used = torch.zeros(P, page, dtype=torch.bool)
    for b, n in enumerate(lengths):
        j = torch.arange(min(n, max(0, int(starts[b]))) if starts is not None else 0, n)
        if len(j):
            used[table[b, j // page].long(), j % page] = True
    idle = (~used)[:, None].expand(P, H, page).reshape(-1)
    for p in (kc, vc):
        p.norms[idle] = float("nan")
        p.rnorms[idle] = float("inf")
        p.code[idle] = -1
        p.res[idle] = -1
