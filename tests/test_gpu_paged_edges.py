"""The paged attention operators where their number formats end: one weight far
above thousands of others, values and norms at the ends of their types, and
batches whose places are not all in use."""
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


def _planted(D, page, targets, common, seed, sigma_v=1.0):
    """One KV head whose row j has score targets[j] (natural units) for a query
    `base`, and value rows that share `common` of their squared length.
    (base, K pool, V pool, dk, dv, c)"""
    n = len(targets)
    pages = -(-n // page)
    g = torch.Generator().manual_seed(seed)
    dk, dv, c = rademacher(D, 2 * seed), rademacher(D, 2 * seed + 1), lloyd_max(1, D)
    base = torch.randn(D, generator=g, dtype=torch.float64)
    qt = (base * dk.double()) @ R.hadamard(D) / math.sqrt(D)
    bits = (qt > 0).long()
    # every key has the query's signs: s_j = norm_j sum |q~| (c1 + 0.5 / sqrt(D))
    per = (qt.abs().sum() * (c[1].double() + 0.5 / math.sqrt(D))) / math.sqrt(D)
    norm = torch.ones(pages * page, dtype=torch.float64)
    norm[:n] = targets / per
    k = ops.PackedKV((pages, 1, page, D), 1, R.words(bits.expand(pages * page, D)), norm.float(),
                     R.words(bits.expand(pages * page, D)), (0.5 * norm).float())
    x = math.sqrt(1 - common) * torch.randn(pages * page, D, generator=g, dtype=torch.float64)
    x += math.sqrt(common) * torch.randn(D, generator=g, dtype=torch.float64)
    code, res, vn, vr = R.compress(x * sigma_v, dv, c)
    v = ops.PackedKV((pages, 1, page, D), 1, R.words(code), vn.float(), R.words(res), vr.float())
    return base, k, v, dk, dv, c


def _off(got, want):
    return ((got.detach().cpu().double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()


def _sink(n, share, sigma, D, common, seed, page=64):
    """A first row of weight `share` beside n - 1 others of spread sigma."""
    g = torch.Generator().manual_seed(seed + 1)
    t = 2.0 + sigma * torch.randn(n, generator=g, dtype=torch.float64).clamp(-3, 3)
    t[0] = torch.logsumexp(t[1:], 0) + math.log(share / (1 - share))
    return _planted(D, page, t.clamp_min(1e-3), common, seed)


def _queries(base, B, nq, dtype):
    """Query rows along base, up to 2% longer or shorter."""
    f = 1 + 0.02 * torch.linspace(-1, 1, B * nq, dtype=torch.float64)
    return (f.view(B, nq, 1) * base).to(dtype)


# Relative 2-norm of an output row's error.  The output's rounding: half a step
# eps / 2 at most, 0.43 of that in the mean square over a binade, within 15% over
# 128 elements: 1.9e-3 (bf16), 2.4e-4 (fp16).  The values' weights: 256 rows share the
# step of the heaviest, 2^-15 of it, later ones have steps of a half, a quarter and
# so on of that; 0.41 of a step a row (the difference of two remainders), at random:
# sqrt(256 4/3) 0.41 2^-15 = 2.3e-4.  Scores of up to 20 (in log2), 16-bit queries' fixed
# point 2^-13.7 sqrt(D) max |q~| / |q| of them at most, that over sqrt(D) in the mean
# square (5e-5), times 2 share (1 - share) <= 1/2: under 1e-4.  Root sums 1.92e-3 and 3.5e-4.
# fp32: exponents of 20 in three 32-bit roundings, 20 3 2^-24, a half of that as above:
# 1.8e-6; weights of 2^-30 of the heaviest, all of one sign: 256 (1 + 1/2 + ...) 2^-31: 2.4e-7.
WITHIN = {BF: 2e-3, HF: 4e-4, FL: 2.1e-6}


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("D,B,nq,n,share,sigma,common", [
    (128, 32, 4, 8192, 0.80, 0.0, 0.5), (128, 32, 4, 8192, 0.87, 0.5, 0.5),
    (128, 512, 4, 32768, 0.50, 0.0, 0.5), (128, 512, 4, 32768, 0.62, 0.5, 0.5),
    (128, 512, 4, 32768, 0.71, 1.0, 0.5), (128, 512, 4, 32768, 0.71, 1.0, 0.0),
    (128, 256, 7, 32768, 0.66, 0.5, 0.5), (256, 256, 3, 16384, 0.67, 0.0, 0.5),
    (256, 256, 8, 16384, 0.87, 1.0, 0.0), (128, 2, 2, 300, 0.90, 0.5, 0.5),
])
def test_small_weights_beside_a_large_one(dtype, D, B, nq, n, share, sigma, common):
    """A first row that takes most of the weight, as contexts have it, and a
    long tail whose rows each count little but together much."""
    base, k, v, dk, dv, c = _sink(n, share, sigma, D, common, n + nq)
    q = _queries(base, B, nq, dtype)
    pages = k.shape[0]
    table = torch.arange(pages, dtype=torch.int32).expand(B, -1).contiguous()
    out = ops.paged_decode_attention(q.cuda(), R.cuda(k), R.cuda(v), table.cuda(),
                                     torch.full((B,), n, dtype=torch.int32).cuda(), dk, dv, c)
    few = [0, B // 2, B - 1]
    want = R.attention(q[few], k, v, table[few], [n] * 3, dk, dv, c)[0]
    assert _off(out[few], want) <= WITHIN[dtype]
    # and the engine's attention over the same rows in one piece
    one = ops.decode_attention(q[:1].float().cuda(), R.cuda(k), R.cuda(v), dk, dv, c, length=n)
    assert _off(one, want[:1]) <= 1e-4
    assert _off(out[:1], one.cpu().double()) <= WITHIN[dtype] + 1e-4


@pytest.mark.parametrize("dtype,D,B,nq", [(BF, 128, 7, 4), (HF, 128, 16, 4), (HF, 256, 13, 7),
                                          (FL, 128, 8, 4)])
@pytest.mark.parametrize("n,share,sigma", [(8192, 0.8, 0.0), (32768, 0.62, 0.5)])
def test_small_weights_beside_a_large_one_in_a_prefix(dtype, D, B, nq, n, share, sigma):
    base, k, v, dk, dv, c = _sink(n, share, sigma, D, 0.5, n + B)
    q = _queries(base, B, nq, dtype)
    table = torch.arange(k.shape[0], dtype=torch.int32).expand(B, -1).contiguous()
    out = ops.paged_prefix_attention(q.cuda(), R.cuda(k), R.cuda(v), table.cuda(),
                                     torch.full((B,), n, dtype=torch.int32).cuda(), n, dk, dv, c)
    few = [0, B - 1]
    want = R.attention(q[few], k, v, table[few], [n] * 2, dk, dv, c)[0]
    assert _off(out[few], want) <= WITHIN[dtype]


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("D,nq", [(128, 4), (128, 8), (256, 4)])
def test_weights_that_rise_and_fall(dtype, D, nq):
    """Heavy rows anywhere, each of another size, with every row in between far
    below them and far above what came before."""
    n, B = 16384, 256
    g = torch.Generator().manual_seed(D + nq)
    t = 4.0 + 0.5 * torch.randn(n, generator=g, dtype=torch.float64)
    at = torch.tensor([0, 1, 31, 32, 255, 256, 257, 1000, 1031, 4000, 8191, 16383])
    t[at] += torch.tensor([5.0, 1, 6, 2, 5, 7, 4, 3, 8, 1, 7, 8], dtype=torch.float64)
    t[2000:3000] -= 3.0
    base, k, v, dk, dv, c = _planted(D, 64, t, 0.5, n + nq)
    q = _queries(base, B, nq, dtype)
    table = torch.arange(k.shape[0], dtype=torch.int32).expand(B, -1).contiguous()
    ln = torch.full((B,), n, dtype=torch.int32)
    out, lse = ops.paged_decode_attention(q.cuda(), R.cuda(k), R.cuda(v), table.cuda(), ln.cuda(),
                                          dk, dv, c, return_lse=True)
    few = [0, B - 1]
    want = R.attention(q[few], k, v, table[few], [n] * 2, dk, dv, c)
    assert _off(out[few], want[0]) <= WITHIN[dtype]
    assert (lse[few].cpu().double() - want[1]).abs().max() <= 2e-3


def _batch(lengths, page, H, D, nq, dtype, seed, pages=None):
    need = pages or sum(-(-n // page) for n in lengths) + 1
    kc, vc, dk, dv, c = R.pools(need, H, page, D, seed)
    table = R.tables(lengths, page, need, seed)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(len(lengths), H * nq, D, generator=g).to(dtype)
    return q, kc, vc, table, torch.tensor(lengths, dtype=torch.int32).cuda(), dk, dv, c


@pytest.mark.parametrize("dtype,D,nq", [(FL, 128, 2), (FL, 256, 1), (BF, 128, 4), (HF, 256, 5)])
def test_capped_scores_keep_nan(dtype, D, nq):
    """With a cap, too, a NaN in an attended row's norms or in a query (or an
    infinity, whose products are NaN) makes that result NaN and no other."""
    lengths, page, H = [200, 150, 90], 16, 2
    q, kc, vc, table, ln, dk, dv, c = _batch(lengths, page, H, D, nq, dtype, 41)
    run = lambda x: ops.paged_decode_attention(  # noqa: E731
        x.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln, dk, dv, c, softcap=8.0).cpu().float()
    R.check(run(q), None, R.attention(q, kc, vc, table, lengths, dk, dv, c, softcap=8.0), dtype)
    for pool in (kc, vc):
        for norms in (pool.norms, pool.rnorms):
            for j in (0, 37, 149):
                row = (int(table[1, j // page]) * H + 1) * page + j % page
                old = norms[row].clone()
                norms[row] = math.nan
                out = run(q)
                norms[row] = old
                assert torch.isnan(out[1, nq:]).all()
                assert torch.isfinite(out[[0, 2]]).all() and torch.isfinite(out[1, :nq]).all()
    for bad in (math.nan, math.inf, -math.inf):
        x = q.clone()
        x[2, nq - 1, 5] = bad
        out = run(x)
        assert torch.isnan(out[2, nq - 1]).all()
        out[2, nq - 1] = 0
        assert torch.isfinite(out).all()


@pytest.mark.parametrize("dtype,D,nq,B,prefix", [
    (FL, 128, 2, 3, 0), (BF, 128, 8, 3, 0), (HF, 256, 3, 3, 0), (BF, 128, 4, 3, 64), (BF, 128, 4, 12, 64),
    (BF, 256, 4, 9, 64)])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_infinite_norms_of_attended_rows(dtype, D, nq, B, prefix, softcap):
    """An infinity among the attended rows' norms has no average: NaN, whatever
    the score's sign and however small the row's weight."""
    page, H = 16, 1
    lengths = [150 + b for b in range(B)]
    q, kc, vc, table, ln, dk, dv, c = _batch(lengths, page, H, D, nq, dtype, 43)
    table[:, :prefix // page] = table[0, :prefix // page]
    # the row at 100 (or 7) counts nothing beside the last ones: 2^-500
    slopes = torch.full((nq,), 10.0)

    def run(sl):
        a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln)
        kw = dict(softcap=softcap, slopes=sl)
        if prefix:
            return ops.paged_prefix_attention(*a, prefix, dk, dv, c, **kw).cpu().float()
        return ops.paged_decode_attention(*a, dk, dv, c, **kw).cpu().float()

    assert torch.isfinite(run(None)).all() and torch.isfinite(run(slopes.cuda())).all()
    for j in (7, 100):
        hit = list(range(B)) if j < prefix else [1]
        miss = [b for b in range(B) if b not in hit]
        row = int(table[1, j // page]) * page + j % page
        for norms in (kc.norms, kc.rnorms, vc.norms, vc.rnorms):
            old = norms[row].clone()
            norms[row] = math.inf
            for sl in (None, slopes.cuda()):
                out = run(sl)
                assert torch.isnan(out[hit]).all(), (j, sl is None)
                assert torch.isfinite(out[miss]).all()
            norms[row] = old


@pytest.mark.parametrize("dtype,f", [(FL, 1e-32), (FL, 1e-38), (BF, 1e-36), (BF, 1e-38), (HF, 1e-7)])
@pytest.mark.parametrize("D,B,nq", [(128, 3, 4), (256, 2, 3), (128, 10, 4)])
def test_tiny_queries(dtype, f, D, B, nq):
    """Queries so small that every score is 0 in 32 bits: the rows' average."""
    lengths, page = [70 + 9 * b for b in range(B)], 16
    q, kc, vc, table, ln, dk, dv, c = _batch(lengths, page, 1, D, nq, FL, 47)
    q = (q * f).to(dtype)
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln)
    R.check(*ops.paged_decode_attention(*a, dk, dv, c, return_lse=True), want, dtype)
    # one shared page, that of sequence 0
    table[:, 0] = table[0, 0]
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln)
    R.check(*ops.paged_prefix_attention(*a, page, dk, dv, c, return_lse=True), want, dtype)


@pytest.mark.parametrize("dtype,D,nq", [(BF, 128, 4), (BF, 256, 4), (HF, 128, 2), (FL, 128, 3)])
@pytest.mark.parametrize("lengths", [
    [0] + [330 + 7 * b for b in range(11)],           # an unused place first
    [100, 0, 300, 319, 330] + [340] * 7,              # short ones first
    [0, 17, 160, 5, 200] + [130] * 7,                 # none reaches the prefix's end
    [0] * 12,
])
def test_prefix_of_a_batch_whose_first_places_are_short(dtype, D, nq, lengths):
    """The prefix is read through a sequence that has it: entries of the block
    table behind a sequence's last page are out of range, for every sequence."""
    prefix, page, H = 320, 32, 2
    kc, vc, dk, dv, c = R.pools(prefix // page + 24, H, page, D, 53)
    table = R.tables(lengths, page, kc.shape[0], 53, prefix)
    R.poison(kc, vc, table, lengths)
    q = torch.randn(len(lengths), H * nq, D, generator=torch.Generator().manual_seed(53)).to(dtype)
    # a captured graph's max_len, not the lengths, fixes the launch
    table = torch.cat([table, torch.full((len(lengths), 20 - table.shape[1]), 1 << 30,
                                         dtype=torch.int32)], 1)
    out, lse = ops.paged_prefix_attention(
        q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
        torch.tensor(lengths, dtype=torch.int32).cuda(), prefix, dk, dv, c, return_lse=True)
    want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
    R.check(out, lse, want, dtype)
    assert (out.cpu()[torch.isinf(want[1])] == 0).all()


def test_prefix_source_far_behind_in_a_large_batch():
    """Hundreds of unused places before the one that has the prefix."""
    prefix, page, D, nq = 64, 16, 128, 2
    for dtype in (BF, FL):
        for at in (127, 128, 129, 700):
            lengths = [3] * at + [70] + [0] * (705 - at - 1)
            kc, vc, dk, dv, c = R.pools(3000, 1, page, D, 59)
            table = R.tables(lengths, page, 3000, 59, prefix)
            q = torch.randn(705, nq, D, generator=torch.Generator().manual_seed(59)).to(dtype)
            out = ops.paged_prefix_attention(
                q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
                torch.tensor(lengths, dtype=torch.int32).cuda(), prefix, dk, dv, c).cpu()
            few = [0, at]
            want = R.attention(q[few], kc, vc, table[few], [3, 70], dk, dv, c)
            R.check(out[few], None, want, dtype)
            assert (out[at + 1:] == 0).all()


@pytest.mark.parametrize("D,page", [(128, 64), (256, 32)])
@pytest.mark.parametrize("gap", [12.97, 13.48, 14.18, 14.72])
def test_prefix_weights_of_a_tile_before_a_large_one(D, page, gap):
    """Tensor-core prefix: a heavy row late in a tile that is already full of
    weights far below it (2^-22.7 to 2^-25.2 times the first rows'); what those
    add keeps its size."""
    B, nq, n, last = 16, 4, 128, 127
    t = torch.full((n,), 2.0, dtype=torch.float64)
    mid = slice(32, 96) if D == 128 else slice(64, 96)  # a tile is 128 rows, or 64
    t[mid] += math.log(1000.0)
    t[last] += math.log(1000.0) + gap - math.log(64.0)
    base, k, v, dk, dv, c = _planted(D, page, t, 0.0, 61)
    # the rows before have one value, so that what they add shows along it
    w = k.shape[0] * page
    before = torch.arange(w) != last
    for x in (v.code, v.res, v.norms, v.rnorms):
        x[before] = x[0].clone()
    q = base.expand(B, nq, D).to(BF)
    table = torch.arange(k.shape[0], dtype=torch.int32).expand(B, -1).contiguous()
    out = ops.paged_prefix_attention(q.cuda(), R.cuda(k), R.cuda(v), table.cuda(),
                                     torch.full((B,), n, dtype=torch.int32).cuda(), n, dk, dv, c)
    want = R.attention(q[:1], k, v, table[:1], [n], dk, dv, c)[0]
    side = (R.rows(v, c, False)[0] @ R.hadamard(D)) * dv.double()
    side = side / side.norm()
    off = ((out[:1].cpu().double() - want) @ side).abs().max() / want.norm()
    # Along one direction the output's roundings (half steps, 2^-8 of elements that have
    # 1 / sqrt(D) of the norm each) are 2^-8 0.43 / sqrt(D) in the mean square, the heavy
    # row's (fp16) an eighth of that; two deviations are 3e-4 at D = 128.  The rest is the
    # mass of the rows before, under 0.01 for these gaps, to 2^-8 of itself.
    assert off <= 3e-4 + 0.01 * 2.0 ** -8


@pytest.mark.parametrize("n,share,sigma", [(131072, 0.87, 0.0), (131072, 0.62, 0.5), (32768, 0.71, 1.0)])
@pytest.mark.parametrize("D", [128, 256])
def test_prefix_in_one_chunk_with_a_heavy_row(n, share, sigma, D):
    """Tensor-core prefix, so many query rows that a CTA has all of it: small
    weights beside a large one.  WITHIN's bf16 output rounding 1.9e-3; a score of 17 (in
    natural units) whose keys' elements are one number with one rounding to fp16,
    2^-11 0.43 in the mean square, times share (1 - share) |V_0 - V| / |out| <= 0.19:
    6.8e-4; values and weights in fp16, 2^-11 0.43 each.  Root sum 2.1e-3."""
    per = 256 if D == 128 else 128
    nq = 64
    B = 148 * per // nq
    base, k, v, dk, dv, c = _sink(n, share, sigma, D, 0.5, n + D, page=256)
    q = _queries(base, B, nq, BF)
    table = torch.arange(k.shape[0], dtype=torch.int32).expand(B, -1).contiguous()
    out = ops.paged_prefix_attention(q.cuda(), R.cuda(k), R.cuda(v), table.cuda(),
                                     torch.full((B,), n, dtype=torch.int32).cuda(), n, dk, dv, c)
    few = [0, B - 1]
    want = R.attention(q[few][:, :4], k, v, table[few], [n] * 2, dk, dv, c)[0]
    assert _off(out[few][:, :4], want) <= 2.1e-3


@pytest.mark.parametrize("dtype,D,B,nq", [(FL, 128, 3, 2), (FL, 256, 2, 1), (BF, 128, 3, 4),
                                          (BF, 128, 10, 4), (BF, 256, 6, 4)])
@pytest.mark.parametrize("scale", [1e-14, 1e-20, 1e-25, 1e25, 1e30])
def test_values_of_any_size(dtype, D, B, nq, scale):
    """All values scaled: the result is, too.  Some rows have none at all."""
    lengths, page = [300 + 9 * b for b in range(B)], 16
    q, kc, vc, table, ln, dk, dv, c = _batch(lengths, page, 1, D, nq, dtype, 67)
    table[:, :16] = table[0, :16]
    vc.norms *= scale
    vc.rnorms *= scale
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln)
    for zeros in (False, True):
        if zeros:
            vc.norms[::3] = 0
            vc.rnorms[::3] = 0
            a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln)
        want = R.attention(q, kc, vc, table, lengths, dk, dv, c)
        R.check(*ops.paged_decode_attention(*a, dk, dv, c, return_lse=True), want, dtype)
        R.check(*ops.paged_prefix_attention(*a, 256, dk, dv, c, return_lse=True), want, dtype)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D,nq", [(128, 4), (128, 8), (256, 4)])
def test_scores_of_16_bit_queries(dtype, D, nq):
    """One row a sequence: lse is its score, computed from q~ in 16-bit fixed
    point.  A step is 2^-15 of the largest element, twice that for every other
    one: errors of 1 / sqrt(12) steps each are 0.456 2^-15 in the mean square, and
    over D elements, in units of |K| sqrt(D) max |q~|, 0.456 2^-15 / sqrt(D).  Of
    this many scores the root mean square is within 15% of that."""
    B, H, page = 128, 2, 16
    q, kc, vc, table, ln, dk, dv, c = _batch([1] * B, page, H, D, nq, dtype, 71)
    _, lse = ops.paged_decode_attention(q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(), ln, dk, dv,
                                        c, return_lse=True)
    _, want, _, _, peak, _ = R.attention(q, kc, vc, table, [1] * B, dk, dv, c)
    off = ((lse.cpu().double() - want) / peak).square().mean().sqrt()
    assert off <= 1.15 * 0.456 * 2.0 ** -15 / math.sqrt(D)


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("B,nq,n", [(7, 8, 13017), (64, 9, 2472), (64, 9, 11945), (64, 9, 2652),
                                    (16, 3, 300), (40, 4, 64)])
def test_prefix_chunks_of_a_few_tiles(D, B, nq, n):
    """Tensor-core prefix that is all there is: its sums leave after the last
    product, in every run."""
    page = 64
    kc, vc, dk, dv, c = R.pools(-(-n // page), 1, page, D, 73)
    q = torch.randn(B, nq, D, generator=torch.Generator().manual_seed(73)).to(BF)
    table = torch.randperm(kc.shape[0], generator=torch.Generator().manual_seed(n)).int()
    table = table.expand(B, -1).contiguous()
    a = (q.cuda(), R.cuda(kc), R.cuda(vc), table.cuda(),
         torch.full((B,), n, dtype=torch.int32).cuda(), n, dk, dv, c)
    out, lse = ops.paged_prefix_attention(*a, return_lse=True)
    few = [0, B - 1]
    want = R.attention(q[few], kc, vc, table[few], [n] * 2, dk, dv, c)
    R.check(out[few], lse[few], want, BF)
    for _ in range(20):
        assert torch.equal(ops.paged_prefix_attention(*a), out)


@pytest.mark.parametrize("dtype,D,B,nq", [(BF, 128, 12, 4), (BF, 256, 9, 4), (FL, 128, 3, 2)])
def test_prefix_in_a_graph_while_places_come_and_go(dtype, D, B, nq):
    """A captured call replayed with other lengths, the first place empty in
    some, beside eager calls on another stream."""
    prefix, page = 320, 32
    full = [prefix + 40 + b for b in range(B)]
    kc, vc, dk, dv, c = R.pools(prefix // page + 3 * B, 1, page, D, 79)
    table = R.tables(full, page, kc.shape[0], 79, prefix)
    q = torch.randn(B, nq, D, generator=torch.Generator().manual_seed(79)).to(dtype)
    kg, vg, tg, qg = R.cuda(kc), R.cuda(vc), table.cuda(), q.cuda()
    ln = torch.tensor(full, dtype=torch.int32).cuda()
    run = lambda n: ops.paged_prefix_attention(qg, kg, vg, tg, n, prefix, dk, dv, c)  # noqa: E731
    run(ln)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(ln)
    side = torch.cuda.Stream()
    other = torch.tensor([0] + [n - 7 for n in full[1:]], dtype=torch.int32).cuda()
    alone = run(other)
    for lengths in (full, [0] + full[1:], [5, 0] + [n - 30 for n in full[2:]], [0] * B, full):
        ln.copy_(torch.tensor(lengths, dtype=torch.int32))
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = [run(other) for _ in range(4)]
        for _ in range(4):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, alone) for x in beside)
        R.check(out, None, R.attention(q, kc, vc, table, lengths, dk, dv, c), dtype)
