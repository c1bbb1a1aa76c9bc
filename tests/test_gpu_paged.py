"""The paged packed cache on the GPU against its plain 64-bit forms: appending
rotated keys and values, decode attention over pages with caps, biases,
windows and empty rows, and attention of a batch that shares a prefix."""
import math

import pytest
import torch

import paged_ref as R
from kudahitam import _lib, lloyd_max, ops, rademacher

pytestmark = pytest.mark.gpu

BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(autouse=True)
def _no_device_error():
    _lib.call("kh_clear_device_error")
    yield
    assert _lib.device_error() == 0


def _tables(n, rot):
    a = torch.arange(n, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    return a.cos().float(), a.sin().float()


def _want_append(k, v, dk, dv, c, pos=None, cos=None, sin=None, inter=False):
    x = k.double()
    if pos is not None:
        x = R.rotate(x, cos[pos], sin[pos], inter)
    return R.compress(x, dk, c), R.compress(v.double(), dv, c)


def _check_rows(pool, slots, want):
    """The pool's rows at `slots` are the 64-bit form's bits and norms."""
    P, H, page, D = pool.shape
    code, res, norm, rnorm = want
    at = (slots // page, slice(None), slots % page)
    get = lambda t, *w: t.cpu().view(P, H, page, *w)[at]  # noqa: E731
    assert torch.equal(get(pool.code, D // 32), R.words(code))
    assert torch.equal(get(pool.res, D // 32), R.words(res))
    # sums of D squares in 32 bits, a root and a product: D / 32 + 5 + 4 roundings
    tol = (D / 32 + 9) * 2.0 ** -24
    assert ((get(pool.norms).double() / norm - 1).abs() <= tol).all()
    assert ((get(pool.rnorms).double() / rnorm - 1).abs() <= 4 * tol).all()


@pytest.mark.parametrize("D,dtype,T,H,page,rot,inter", [
    (128, BF, 1, 8, 64, 128, False),
    (128, BF, 65, 3, 48, 128, True),
    (128, FL, 33, 2, 1, 64, False),
    (128, HF, 700, 5, 100, 2, False),
    (256, HF, 129, 2, 16, 256, False),
    (256, BF, 40, 4, 7, 64, True),
    (256, FL, 17, 1, 32, 34, False),
    (128, BF, 2500, 8, 64, 128, False),
    (128, HF, 2501, 7, 64, 96, True),
    (256, BF, 1203, 8, 64, 128, False),
    (128, FL, 1501, 3, 64, 128, False),
    (256, FL, 1100, 4, 64, 64, True),
    (256, HF, 1302, 4, 48, 256, False),
    (128, BF, 4100, 1, 64, 34, False),
    (128, FL, 2301, 3, 64, 128, False),
    (256, FL, 1700, 4, 64, 64, True),
    (256, HF, 1702, 4, 48, 256, False),
    (256, BF, 3400, 2, 64, 256, True),
    (128, BF, 6700, 1, 64, 34, False),
])
def test_append_is_the_64_bit_encoding(D, dtype, T, H, page, rot, inter):
    g = torch.Generator().manual_seed(T + D)
    dk, dv, c = rademacher(D, 1), rademacher(D, 2), lloyd_max(1, D)
    k = (torch.randn(T, H, D, generator=g) * 4).to(dtype)
    v = torch.randn(T, H, D, generator=g).to(dtype)
    k[T // 2, 0] = 0  # a row of zeros: norm 1e-8, index 0
    v[0, H - 1, 1:] = 0  # one element: every |y| equal
    pages = -(-T // page) + 2
    slots = torch.randperm(pages * page, generator=g)[:T]
    pos = torch.randint(0, 5000, (T,), generator=g)
    cos, sin = _tables(5000, rot)
    kc, vc = (ops.empty_paged(pages, H, page, D, "cuda") for _ in range(2))
    for p in (kc, vc):
        p.norms.fill_(-3)
        p.code.fill_(7)
    ops.paged_append(k.cuda(), v.cuda(), kc, vc, slots.cuda(), dk, dv, c, pos.cuda(), cos.cuda(),
                     sin.cuda(), inter)
    wk, wv = _want_append(k, v, dk, dv, c, pos, cos, sin, inter)
    _check_rows(kc, slots, wk)
    _check_rows(vc, slots, wv)
    # rows of other slots stay as they were
    idle = torch.ones(pages * page, dtype=torch.bool)
    idle[slots] = False
    at = idle.nonzero()[:, 0]
    for p in (kc, vc):
        n = p.norms.cpu().view(pages, H, page)[at // page, :, at % page]
        assert (n == -3).all()
        w = p.code.cpu().view(pages, H, page, -1)[at // page, :, at % page]
        assert (w == 7).all()


def test_append_without_rotation_strided_inputs_and_padding():
    D, H, T, page = 128, 4, 50, 16
    g = torch.Generator().manual_seed(0)
    dk, dv, c = rademacher(D, 3), rademacher(D, 4), lloyd_max(1, D)
    both = torch.randn(H, T, 2 * D + 8, generator=g).to(BF).cuda()
    k, v = both[:, :, :D].transpose(0, 1), both[:, :, D + 3:2 * D + 3].transpose(0, 1)
    slots = torch.randperm(4 * page, generator=g)[:T]
    slots[::7] = -1
    kc, vc = (ops.empty_paged(4, H, page, D, "cuda") for _ in range(2))
    ops.paged_append(k, v, kc, vc, slots.cuda(), dk, dv, c)
    on = slots >= 0
    wk, wv = _want_append(k.cpu()[on], v.cpu()[on], dk, dv, c)
    _check_rows(kc, slots[on], wk)
    _check_rows(vc, slots[on], wv)
    assert int((kc.norms > 0).sum()) == int(on.sum()) * H
    # one value for every token, without a copy of it; and elements apart
    one = torch.randn(H, D, generator=g).to(BF)
    wide = torch.randn(T, H, 2 * D, generator=g).to(BF)
    ops.paged_append(one.cuda().expand(T, H, D), wide.cuda()[:, :, ::2], kc, vc, slots.cuda(), dk,
                     dv, c)
    wk, wv = _want_append(one.expand(T, H, D)[on], wide[:, :, ::2][on], dk, dv, c)
    _check_rows(kc, slots[on], wk)
    _check_rows(vc, slots[on], wv)


@pytest.mark.parametrize("times", [1, 110])
def test_append_extreme_values_and_ties(times):
    """Squares that leave 32 bits, and sums that are exactly zero."""
    D, H = 128, 1
    dk, dv, c = rademacher(D, 5), rademacher(D, 6), lloyd_max(1, D)
    g = torch.Generator().manual_seed(1)
    k = torch.randn(64, H, D, generator=g)
    k[:16] *= 1e-25
    k[16:32] *= 1e18
    k[32:48] = torch.randint(-2, 3, (16, H, D), generator=g).float()  # many sums are zero
    k[48:] = torch.where(torch.rand(16, H, D, generator=g) < 0.5, 1.0, -1.0)
    k = k.repeat(times, 1, 1)
    kc, vc = (ops.empty_paged(times, H, 64, D, "cuda") for _ in range(2))
    slots = torch.arange(64 * times)
    ops.paged_append(k.cuda(), k.cuda(), kc, vc, slots.cuda(), dk, dv, c)
    wk, wv = _want_append(k, k, dk, dv, c)
    _check_rows(kc, slots, wk)
    _check_rows(vc, slots, wv)


@pytest.mark.parametrize("T", [20, 2100, 3400])
def test_append_with_uneven_levels(T):
    """Two levels that are not -c, c, and tokens without a slot among many."""
    D, H = 128, 2
    dk, dv = rademacher(D, 5), rademacher(D, 6)
    c = torch.tensor([-0.05, 0.09])
    g = torch.Generator().manual_seed(T)
    k = torch.randn(T, H, D, generator=g).to(BF)
    kc, vc = (ops.empty_paged(T // 16 + 1, H, 16, D, "cuda") for _ in range(2))
    slots = torch.arange(T)
    slots[3::5] = -1
    for cb in (c, lloyd_max(1, D)):
        ops.paged_append(k.cuda(), k.cuda(), kc, vc, slots.cuda(), dk, dv, cb)
        on = slots >= 0
        wk, wv = _want_append(k[on], k[on], dk, dv, cb)
        _check_rows(kc, slots[on], wk)
        _check_rows(vc, slots[on], wv)
        assert int((kc.norms > 0).sum()) == int(on.sum()) * H


def test_append_matches_compress_away_from_borders():
    """The engine's own compressor writes the same planes, but for elements so
    near a border that its 32-bit sums may fall on the other side: D additions
    in at most 16 roundings of 2^-23 of sum |x| <= sqrt(D) norm are 2^-19 of
    y = u / (norm sqrt(D)), the norm's own error is far below; twice that."""
    D, H, T = 128, 4, 512
    dk, dv, c = rademacher(D, 7), rademacher(D, 8), lloyd_max(1, D)
    x = torch.randn(T, H, D, device="cuda").to(BF)
    kc, vc = (ops.empty_paged(1, H, T, D, "cuda") for _ in range(2))
    ops.paged_append(x, x, kc, vc, torch.arange(T, device="cuda"), dk, dv, c)
    rows = x.transpose(0, 1).contiguous()
    p = ops.compress(rows, dk, c)
    z = rows.cpu().double().view(H * T, D)
    y = (z * dk.double()) @ R.hadamard(D) / (z.norm(dim=-1, keepdim=True) * math.sqrt(D))
    off = torch.stack([y.abs()] + [(y - float(b)).abs() for b in c]).amin(0)
    for a, b in ((p.code, kc.code), (p.res, kc.res)):
        other = R.unpack(a.cpu().view(H * T, -1)) != R.unpack(b.cpu().view(H * T, -1))
        assert (off[other] <= 2.0 ** -18).all()
        assert int(other.sum()) < 0.001 * other.numel()


def test_append_flags_bad_slots_and_positions():
    D, H = 128, 2
    dk, dv, c = rademacher(D, 1), rademacher(D, 2), lloyd_max(1, D)
    x = torch.randn(6, H, D, device="cuda")
    kc, vc = (ops.empty_paged(1, H, 8, D, "cuda") for _ in range(2))
    cos, sin = (t.cuda() for t in _tables(10, 128))
    slots = torch.tensor([0, 8, -2, 1 << 60, 3, 4], device="cuda")
    pos = torch.tensor([0, 1, 2, 3, 10, -1], device="cuda")
    ops.paged_append(x, x, kc, vc, slots, dk, dv, c, pos, cos, sin)
    assert _lib.device_error() == 8
    _lib.call("kh_clear_device_error")
    live = kc.norms.view(H, 8)[0] > 0
    assert live.nonzero()[:, 0].tolist() == [0]


# ------------------------------------------------------------------ attention


def _attend(lengths, H, nq, D, dtype, page, prefix=0, seed=0, starts=None, max_len=None, pad=0,
            **kw):
    need = prefix // page + sum(max(0, -(-n // page) - prefix // page) for n in lengths)
    kc, vc, dk, dv, c = R.pools(need + 2, H, page, D, seed)
    table = R.tables(lengths, page, need + 2, seed, prefix)
    if prefix % page:  # each sequence's copy of the page that the prefix ends in
        s = prefix // page
        for p in (kc, vc):
            for t in (p.code, p.res, p.norms, p.rnorms):
                w = t.view(need + 2, H, page, -1)
                src = w[int(table[0, s]), :, :prefix % page].clone()
                for b, n in enumerate(lengths):
                    if n > s * page:
                        w[int(table[b, s]), :, :prefix % page] = src
    R.poison(kc, vc, table, lengths, starts)
    g = torch.Generator().manual_seed(seed + 99)
    q = torch.randn(len(lengths), H * nq, D, generator=g).to(dtype)
    if pad:  # a slice of a wider table
        table = torch.cat([table, torch.full((len(lengths), pad), -5, dtype=torch.int32)], 1)
    t = table.cuda()[:, :table.shape[1] - pad]
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda()
    sl = kw.get("slopes")
    opts = dict(kw, starts=st, slopes=None if sl is None else sl.cuda(), max_len=max_len,
                return_lse=True)
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), t, ln)
    if prefix:
        out, lse = ops.paged_prefix_attention(*a, prefix, dk, dv, c, **opts)
    else:
        out, lse = ops.paged_decode_attention(*a, dk, dv, c, **opts)
    assert out.dtype == dtype and out.shape == q.shape and lse.dtype == FL
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c, starts=starts, **kw)
    R.check(out, lse, want, dtype)
    none = torch.isinf(want[1])
    assert (out.cpu()[none] == 0).all()


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("lengths,H,nq,page", [
    ([1], 1, 1, 1),
    ([0], 2, 2, 16),
    ([0, 1, 2, 15, 16, 17, 31, 32, 33], 2, 4, 16),
    ([127, 128, 129, 63, 64, 65, 300, 0], 3, 1, 48),
    ([1000, 7], 1, 8, 100),
    ([2, 333], 2, 3, 32),
    ([77, 500, 1], 1, 5, 64),
    ([40, 91], 2, 9, 7),
    ([65, 130], 1, 16, 256),
    ([31, 260], 1, 33, 16),
])
def test_decode_matches_the_64_bit_form(dtype, D, lengths, H, nq, page):
    _attend(lengths, H, nq, D, dtype, page, seed=len(lengths) + nq)


@pytest.mark.parametrize("dtype,D,nq", [(BF, 128, 4), (FL, 128, 1), (HF, 256, 8), (FL, 128, 6),
                                        (BF, 256, 16)])
def test_decode_long_sequences_over_several_chunks(dtype, D, nq):
    _attend([5001, 1025, 2048, 4095], 1, nq, D, dtype, 64, seed=3, max_len=5100 // 64 * 64)


@pytest.mark.parametrize("kw", [
    dict(softcap=2.0), dict(softcap=50.0), dict(window=1), dict(window=33), dict(window=10 ** 6),
    dict(slopes=True), dict(starts=[0, 5, 700, 64, 1]),
    dict(starts=[-3, 129, 200, 1, 128], window=100, softcap=20.0, slopes=True, sm_scale=0.3),
])
@pytest.mark.parametrize("dtype,D,nq", [(BF, 128, 4), (FL, 256, 2), (HF, 128, 7), (BF, 128, 12)])
def test_decode_caps_biases_windows_and_starts(dtype, D, nq, kw):
    lengths = [600, 130, 700, 65, 1]
    kw = dict(kw)
    if kw.pop("slopes", False):
        kw["slopes"] = 2.0 ** -torch.arange(1, 2 * nq + 1, dtype=FL) * 4
    _attend(lengths, 2, nq, D, dtype, 48, seed=nq, pad=3, **kw)


@pytest.mark.parametrize("dtype,D", [(BF, 128), (HF, 256), (FL, 128)])
def test_decode_units_of_many_thousand_rows(dtype, D):
    """So many rows that a unit is longer than what 32-bit sums hold: sequences
    of a million rows, five pages over and over, which is attention over the
    five once."""
    page, pages, times, B, nq = 500, 5, 420, 8, 256
    n = page * pages
    kc, vc, dk, dv, c = R.pools(pages, 1, page, D, 21)
    table = torch.arange(pages, dtype=torch.int32).repeat(B, times)
    lengths = [n * times, 3] + [n * times - 1] * (B - 2)
    q = torch.randn(B, nq, D, generator=torch.Generator().manual_seed(21)) / 8
    q = q.to(dtype)
    out, lse = ops.paged_decode_attention(q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
                                          torch.tensor(lengths, dtype=torch.int32).cuda(), dk, dv,
                                          c, return_lse=True)
    few = q[:2, :3]
    want = list(R.attention(few, kc, vc, table[:2], [n, 3], dk, dv, c))
    want[1][0] += math.log(times)
    R.check(out[:2, :3], lse[:2, :3], want, dtype)


def test_decode_negative_scale_and_large_values():
    """A negative scale, and rows whose norms span many orders."""
    _attend([400, 90], 1, 4, 128, FL, 16, seed=5, sm_scale=-0.2)
    lengths, page, H, D = [257, 64], 16, 1, 128
    kc, vc, dk, dv, c = R.pools(23, H, page, D, 6)
    g = torch.Generator().manual_seed(6)
    f = 10.0 ** (torch.rand(vc.norms.numel(), generator=g) * 12 - 6)
    vc.norms *= f
    vc.rnorms *= f
    table = R.tables(lengths, page, 23, 6)
    for dtype, nq in ((FL, 2), (BF, 4), (HF, 6)):
        q = (torch.randn(2, nq, D, generator=g) * 20).to(dtype)
        out, lse = ops.paged_decode_attention(q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
                                              torch.tensor(lengths, dtype=torch.int32).cuda(), dk,
                                              dv, c, return_lse=True)
        R.check(out, lse, R.attention(q, kc, vc, table, lengths, dk, dv, c), dtype)


@pytest.mark.parametrize("dtype,D,B,nq", [(BF, 128, 3, 4), (FL, 256, 2, 2), (BF, 128, 12, 4),
                                          (BF, 256, 20, 2)])
def test_attention_with_uneven_levels(dtype, D, B, nq):
    """A caller's codebook need not be symmetric, nor around zero."""
    prefix, page = 200, 16
    lengths = [prefix + 30 + b for b in range(B)]
    kc, vc, dk, dv, _ = R.pools(prefix // page + 1 + 6 * B, 1, page, D, 8)
    c = torch.tensor([-0.3, 1.7])
    table = R.tables(lengths, page, kc.shape[0], 8, prefix // page * page)
    g = torch.Generator().manual_seed(8)
    q = torch.randn(B, nq, D, generator=g).to(dtype)
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
         torch.tensor(lengths, dtype=torch.int32).cuda())
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
    R.check(*ops.paged_decode_attention(*a, dk, dv, c, return_lse=True), want, dtype)
    R.check(*ops.paged_prefix_attention(*a, prefix // page * page, dk, dv, c, return_lse=True),
            want, dtype)


@pytest.mark.parametrize("dtype,D,nq", [(BF, 128, 4), (FL, 128, 3), (HF, 256, 2), (FL, 256, 1)])
def test_decode_with_values_that_are_not_finite(dtype, D, nq):
    """A NaN or an infinity among a sequence's norms, or in one of its queries,
    makes that result NaN and no other."""
    lengths, page, H = [200, 150, 90], 16, 2
    kc, vc, dk, dv, c = R.pools(32, H, page, D, 31)
    table = R.tables(lengths, page, 32, 31)
    g = torch.Generator().manual_seed(31)
    q = torch.randn(3, H * nq, D, generator=g).to(dtype)
    ln = torch.tensor(lengths, dtype=torch.int32).cuda()
    run = lambda x: ops.paged_decode_attention(  # noqa: E731
        x.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln, dk, dv, c).cpu().float()
    R.check(run(q), None, R.attention(q, kc, vc, table, lengths, dk, dv, c), dtype)
    for pool in (kc, vc):
        for norms in (pool.norms, pool.rnorms):
            for bad in (math.nan, math.inf):
                for j in (0, 37, 149):
                    row = (int(table[1, j // page]) * H + 1) * page + j % page
                    old = norms[row].clone()
                    norms[row] = bad
                    out = run(q)
                    norms[row] = old
                    if not (pool is kc and bad == math.inf):  # may be a weight of zero
                        assert torch.isnan(out[1, nq:]).all()
                    assert torch.isfinite(out[[0, 2]]).all() and torch.isfinite(out[1, :nq]).all()
    for bad in (math.nan, math.inf, -math.inf):
        for e in (0, 5):
            x = q.clone()
            x[2, nq - 1, e] = bad
            out = run(x)
            assert torch.isnan(out[2, nq - 1]).all()
            out[2, nq - 1] = 0
            assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype,D,H,nq,page,prefix,suffix", [
    (BF, 128, 2, 4, 64, 640, [3, 1, 100, 64]),
    (BF, 128, 1, 8, 48, 1001, [0, 7, 300]),
    (HF, 128, 2, 3, 16, 129, [1] * 9),
    (HF, 256, 1, 7, 48, 501, [70, 1, 0, 33, 200]),
    (FL, 128, 1, 4, 32, 700, [5, 40]),
    (FL, 256, 2, 1, 100, 64, [1, 2, 3]),
    (BF, 128, 1, 1, 64, 2100, [10] * 40),
    (BF, 256, 1, 16, 64, 260, [9, 90, 30]),
    (BF, 128, 1, 5, 64, 1, [1, 0]),
    (BF, 128, 2, 4, 64, 1500, [20] * 37),
    (HF, 128, 1, 12, 64, 300, [17] * 12),
])
def test_prefix_matches_the_64_bit_form(dtype, D, H, nq, page, prefix, suffix):
    _attend([prefix + s for s in suffix], H, nq, D, dtype, page, prefix=prefix, seed=prefix)


@pytest.mark.parametrize("dtype,D,nq", [(BF, 128, 4), (HF, 128, 4), (FL, 128, 2), (BF, 256, 8)])
def test_prefix_with_caps_biases_windows_and_short_sequences(dtype, D, nq):
    """Sequences that end or start inside the prefix, windows that reach into
    it, and one that attends nothing."""
    prefix, lengths = 400, [500, 401, 400, 300, 1, 0, 450]
    starts = [0, 390, 100, 299, 0, 0, 450]
    slopes = 2.0 ** -torch.arange(1, 2 * nq + 1, dtype=FL)
    _attend(lengths, 2, nq, D, dtype, 64, prefix=prefix, seed=1, softcap=15.0, window=150,
            slopes=slopes, starts=starts)
    _attend(lengths, 2, nq, D, dtype, 64, prefix=prefix, seed=2)


@pytest.mark.parametrize("D,B,nq", [(128, 12, 4), (128, 70, 4), (256, 9, 6)])
@pytest.mark.parametrize("extra", [False, True])
def test_prefix_of_many_queries_with_masks(D, B, nq, extra):
    """Enough queries for the tensor-core prefix, each with limits of its own."""
    prefix = 777
    lengths = [prefix + (37 * b) % 90 for b in range(B)]
    lengths[3:6] = [500, 0, 777]
    starts = [(53 * b) % 1000 for b in range(B)]
    kw = dict(softcap=12.0, slopes=2.0 ** -torch.arange(1, 2 * nq + 1, dtype=FL)) if extra else {}
    _attend(lengths, 2, nq, D, BF, 48, prefix=prefix, seed=B, starts=starts, window=400, **kw)
    _attend(lengths, 2, nq, D, BF, 64, prefix=prefix, seed=B + 1, **kw)


def test_prefix_of_many_queries_with_large_and_bad_values():
    """Norms over twelve orders in the prefix; then a NaN in one attended row,
    which must reach every query that attends it and no other."""
    prefix, page, H, D, B, nq = 512, 64, 1, 128, 10, 4
    lengths = [prefix + 5] * B
    lengths[2] = 100
    kc, vc, dk, dv, c = R.pools(prefix // page + B, H, page, D, 12)
    g = torch.Generator().manual_seed(12)
    f = 10.0 ** (torch.rand(vc.norms.numel(), generator=g) * 12 - 6)
    vc.norms *= f
    vc.rnorms *= f
    table = R.tables(lengths, page, prefix // page + B, 12, prefix)
    q = (torch.randn(B, nq, D, generator=g) * 8).to(BF)
    run = lambda: ops.paged_prefix_attention(  # noqa: E731
        q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(), prefix, dk, dv, c, return_lse=True)
    R.check(*run(), R.attention(q, kc, vc, table, lengths, dk, dv, c), BF)
    for pool in (kc, vc):
        row = int(table[0, 300 // page]) * page + 300 % page
        old = pool.norms[row].clone()
        pool.norms[row] = float("nan")
        out = run()[0].cpu().float()
        assert torch.isfinite(out[2]).all()
        assert torch.isnan(out[[b for b in range(B) if b != 2]]).all()
        pool.norms[row] = old


def test_prefix_equals_decode():
    """The shared read is the same attention as each sequence's own."""
    lengths, prefix, page = [1100, 1030, 1024], 1024, 64
    kc, vc, dk, dv, c = R.pools(20, 2, page, 128, 11)
    table = R.tables(lengths, page, 20, 11, prefix)
    q = torch.randn(3, 8, 128)
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
         torch.tensor(lengths, dtype=torch.int32).cuda())
    x = ops.paged_prefix_attention(*a, prefix, dk, dv, c)
    y = ops.paged_decode_attention(*a, dk, dv, c)
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
    R.check(x, None, want, FL)
    R.check(y, None, want, FL)


def test_attention_flags_bad_pages_and_lengths():
    kc, vc, dk, dv, c = R.pools(4, 1, 16, 128, 2)
    q = torch.randn(2, 2, 128)
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    bad = table.clone()
    bad[1, 0] = 4  # past the pool: those 16 rows are not attended
    ln = torch.tensor([20, 30], dtype=torch.int32)
    args = (dk, dv, c)
    got = ops.paged_decode_attention(q.cuda(), R.cuda(kc), R.cuda(vc), bad.cuda(), ln.cuda(), *args)
    assert _lib.device_error() == 8
    _lib.call("kh_clear_device_error")
    want = R.attention(q, kc, vc, table, [20, 30], *args, starts=[0, 16])
    R.check(got, None, want, FL)
    ln = torch.tensor([33, -1], dtype=torch.int32)  # clamped to 32 and 0
    got, lse = ops.paged_decode_attention(q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
                                          ln.cuda(), *args, return_lse=True)
    assert _lib.device_error() == 8
    _lib.call("kh_clear_device_error")
    R.check(got, lse, R.attention(q, kc, vc, table, [32, 0], *args), FL)


def test_append_then_attend_in_a_graph_and_on_another_stream():
    """A decode loop as a server runs it: each step appends one token per
    sequence and attends; captured once, replayed with new contents, and the
    results equal the same calls made one by one."""
    D, H, nq, B, page, steps = 128, 2, 4, 3, 16, 5
    dk, dv, c = rademacher(D, 1), rademacher(D, 2), lloyd_max(1, D)
    cos, sin = (t.cuda() for t in _tables(200, D))
    g = torch.Generator().manual_seed(3)
    ks, vs = (torch.randn(steps, B, H, D, generator=g).to(BF).cuda() for _ in range(2))
    qs = torch.randn(steps, B, H * nq, D, generator=g).to(BF).cuda()
    table = torch.randperm(6, generator=g).int().view(B, 2).cuda()
    start = torch.tensor([14, 0, 7])

    def pools():
        return [ops.empty_paged(6, H, page, D, "cuda") for _ in range(2)]

    def at(i):
        n = (start + i).cuda()
        slot = table.long()[torch.arange(B, device="cuda"), n // page] * page + n % page
        return slot, n, (n + 1).int()

    def step(kc, vc, k, v, q, slot, pos, ln):
        ops.paged_append(k, v, kc, vc, slot, dk, dv, c, pos, cos, sin)
        return ops.paged_decode_attention(q, kc, vc, table, ln, dk, dv, c)

    first = [torch.randn(14, H, D, generator=g).to(BF).cuda() for _ in range(2)]

    def fill(kc, vc):
        for b in range(B):
            n = int(start[b])
            if n:
                p = torch.arange(n, device="cuda")
                slot = table.long()[b, p // page] * page + p % page
                ops.paged_append(first[0][:n], first[1][:n], kc, vc, slot, dk, dv, c, p, cos, sin)

    kc, vc = pools()
    fill(kc, vc)
    want = [step(kc, vc, ks[i], vs[i], qs[i], *at(i)).clone() for i in range(steps)]

    side = torch.cuda.Stream()
    kc2, vc2 = pools()
    io = [ks[0].clone(), vs[0].clone(), qs[0].clone(), *at(0)]
    fill(kc2, vc2)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got0 = step(kc2, vc2, *io)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got0, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(kc2, vc2, *io)
    for i in range(steps):
        for dst, src in zip(io, (ks[i], vs[i], qs[i], *at(i))):
            dst.copy_(src)
        graph.replay()
        assert torch.equal(out, want[i]), i
    for a, b in ((kc, kc2), (vc, vc2)):
        assert torch.equal(a.code, b.code) and torch.equal(a.norms, b.norms)


def test_two_graphs_and_an_eager_call_do_not_share_scratch():
    kc, vc, dk, dv, c = R.pools(80, 1, 64, 128, 4)
    kc, vc = R.cuda(kc), R.cuda(vc)
    table = torch.arange(80, dtype=torch.int32).view(2, 40).cuda()
    ln = torch.tensor([2500, 1200], dtype=torch.int32).cuda()
    q = [torch.randn(2, 4, 128, device="cuda") for _ in range(3)]
    run = lambda x: ops.paged_decode_attention(x, kc, vc, table, ln, dk, dv, c)  # noqa: E731
    want = [run(x) for x in q]
    graphs, outs = [], []
    for x in q[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(run(x))
        graphs.append(gr)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        graphs[0].replay()
        with torch.cuda.stream(side):
            graphs[1].replay()
        eager = run(q[2])
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert torch.equal(eager, want[2])


def test_results_repeat_bit_for_bit():
    kc, vc, dk, dv, c = R.pools(60, 2, 48, 128, 8)
    kc, vc = R.cuda(kc), R.cuda(vc)
    table = torch.arange(60, dtype=torch.int32).view(2, 30).cuda()
    ln = torch.tensor([1440, 1000], dtype=torch.int32).cuda()
    for dtype in (BF, HF, FL):
        q = torch.randn(2, 8, 128, device="cuda").to(dtype)
        a = ops.paged_decode_attention(q, kc, vc, table, ln, dk, dv, c)
        for _ in range(3):
            assert torch.equal(a, ops.paged_decode_attention(q, kc, vc, table, ln, dk, dv, c))
        a = ops.paged_prefix_attention(q, kc, vc, table[:1].expand(2, -1).contiguous(), ln, 900,
                                       dk, dv, c)
        b = ops.paged_prefix_attention(q, kc, vc, table[:1].expand(2, -1).contiguous(), ln, 900,
                                       dk, dv, c)
        assert torch.equal(a, b)


def test_empty_calls():
    D, H, page = 128, 2, 16
    dk, dv, c = rademacher(D, 1), rademacher(D, 2), lloyd_max(1, D)
    kc, vc = (ops.empty_paged(1, H, page, D, "cuda") for _ in range(2))
    e = torch.empty(0, H, D, device="cuda")
    ops.paged_append(e, e, kc, vc, torch.empty(0, dtype=torch.int64, device="cuda"), dk, dv, c)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")  # noqa: E731
    q = torch.randn(2, 4, D, device="cuda")
    out = ops.paged_decode_attention(q[:0], kc, vc, i32(0, 1), i32(0), dk, dv, c)
    assert out.shape == (0, 4, D)
    out, lse = ops.paged_decode_attention(q, kc, vc, i32(2, 0), i32(2), dk, dv, c, return_lse=True)
    assert (out == 0).all() and torch.isinf(lse).all()
    out = ops.paged_decode_attention(q, kc, vc, i32(2, 1), i32(2), dk, dv, c, max_len=0)
    assert (out == 0).all()


def test_refusals_on_the_gpu_tensors():
    """Shapes, types and devices that do not fit are refused before a launch."""
    D, H = 128, 2
    dk, dv, c = rademacher(D, 0), rademacher(D, 1), lloyd_max(1, D)
    kc, vc = (ops.empty_paged(2, H, 16, D, "cuda") for _ in range(2))
    x = torch.zeros(3, H, D, device="cuda")
    s = torch.zeros(3, dtype=torch.int64, device="cuda")
    pos, cs = s.clone(), torch.zeros(4, 64, device="cuda")
    ap = lambda k=x, v=x, sl=s, **kw: ops.paged_append(k, v, kc, vc, sl, dk, dv, c, **kw)  # noqa: E731
    for bad in (dict(k=x.double(), v=x.double()), dict(v=x.half()), dict(k=x[:2]), dict(k=x[:, :1]),
                dict(k=x[..., :64], v=x[..., :64]), dict(sl=s.int()), dict(sl=s[:2]),
                dict(sl=s.cpu()), dict(positions=pos), dict(cos=cs, sin=cs),
                dict(positions=pos.int(), cos=cs, sin=cs), dict(positions=pos, cos=cs, sin=cs[:2]),
                dict(positions=pos, cos=cs.half(), sin=cs.half()),
                dict(positions=pos, cos=cs[:0], sin=cs[:0]),
                dict(positions=pos, cos=cs[:, ::2], sin=cs[:, ::2])):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ap(**bad)
    q = torch.zeros(2, 4, D, device="cuda")
    t = torch.zeros(2, 2, dtype=torch.int32, device="cuda")
    n = torch.zeros(2, dtype=torch.int32, device="cuda")
    at = lambda q=q, t=t, n=n, **kw: ops.paged_decode_attention(q, kc, vc, t, n, dk, dv, c, **kw)  # noqa: E731
    assert (at() == 0).all()
    for bad in (dict(q=q.double()), dict(q=q[:, :3]), dict(q=q[..., :64]), dict(q=q[:1]),
                dict(t=t.long()), dict(t=t[:1]), dict(n=n.long()), dict(n=n[:1]),
                dict(max_len=33), dict(max_len=-1), dict(window=-1), dict(softcap=-1.0),
                dict(softcap=float("nan")), dict(sm_scale=float("inf")),
                dict(slopes=torch.zeros(3, device="cuda")),
                dict(slopes=torch.zeros(4, device="cuda", dtype=torch.float64)),
                dict(starts=n.long()), dict(n=n.cpu()), dict(slopes=torch.zeros(4))):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            at(**bad)
    for prefix in (-1, 33):
        with pytest.raises(ValueError):
            ops.paged_prefix_attention(q, kc, vc, t, n, prefix, dk, dv, c)
    with pytest.raises(RuntimeError, match="levels|supported"):
        ops.paged_append(x, x, kc, vc, s, dk, dv, lloyd_max(2, D))
