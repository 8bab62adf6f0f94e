"""Attention over a paged K/V cache where numbers are at their limits."""
import math

import pytest
import torch

from kv_oracle import GROUP, U, quantise
from test_gpu_cache import KINDS, Call

pytestmark = pytest.mark.gpu


def _store(c, which, seq, rows, pos=0):
    """Other rows [n, kv, hd] at positions pos .. of a sequence of a call that was built already."""
    held = (c.keys if which == "k" else c.vals)[seq]
    held[pos:pos + rows.shape[0]] = c.pools.put(which, seq, pos, rows)
    (c.pools.dk if which == "k" else c.pools.dv).copy_(c.pools.k if which == "k" else c.pools.v)


def _query(c, q):
    """Other rows [used, H * hd]."""
    c.q[:c.rows.used, :c.H * c.hd] = q.to(c.q.dtype)
    c.dq.copy_(c.q)


# ---------------------------------------------------------------------------------------------------------------------
# groups that span more than 65504
# ---------------------------------------------------------------------------------------------------------------------
def _wide(gen, n, K, hd, most):
    """Rows whose groups of 32 go from -most to most."""
    x = (torch.rand(n, K, hd // GROUP, GROUP, generator=gen) * 2 - 1) * most
    x[..., 0], x[..., 1] = -most, most
    return x[..., torch.randperm(GROUP, generator=gen)].flatten(2)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,new,lens", [(1, [1], [200]), (12, [1, 1], [200, 70]), (2, [5], [200]), (2, [30], [90]), (2, [70], [100]), (1, [1], [3000])])
def test_wide_groups(pkg, kind, hd, H, new, lens):
    """Keys whose groups go from -40000 to 40000: codes times scale pass the halves' range (15 * 5332 = 79980), the values they stand for do not.  Every form of the
    attention takes them: the same tolerance as for other keys."""
    c = Call(pkg, kind, "q4", H, 1, hd, new, lens, seed=40, spread=0.02, scale=1e-3)
    gen = torch.Generator().manual_seed(41)
    for s, n in enumerate(lens):
        _store(c, "k", s, _wide(gen, n, 1, hd, 40000.0))
        assert c.keys[s].abs().max() < 65504 < 15 * float(quantise(_wide(gen, 1, 1, hd, 40000.0))[1][..., 1].min())
    c.check()


# ---------------------------------------------------------------------------------------------------------------------
# scores of -infinity
# ---------------------------------------------------------------------------------------------------------------------
SIGHTS = [([3], [3], 0), ([1], [200], 0), ([5, 1], [90, 300], 60), ([70], [100], 0), ([150], [400], 70), ([1], [9000], 0)]


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,lens,window", SIGHTS)
def test_nothing_but_minus_infinity(pkg, kind, cache, hd, new, lens, window):
    """An infinite element of q that meets one sign in every key: each score is -infinity, the softmax is undefined and the row NaN, as 0 / 0 is; not zero as for a row that
    sees nothing.  Its neighbours are as without it."""
    c = Call(pkg, kind, cache, 2, 1, hd, new, lens, window, 2, seed=50)
    for s, n in enumerate(lens):
        k = c.keys[s].float().clone()
        k[..., 7] = -1.5  # (over 4 bits not a group's minimum, whose code is zero: zero times infinity is no number anyway)
        k[..., 8] = -4.0
        _store(c, "k", s, k)
    clean = c.run().clone()
    c.dq[0, 7] = math.inf
    c.dq[c.rows.used - 1, hd + 7] = math.inf
    got = c.run()
    for i in range(c.rows.used):
        for h in range(2):
            a, b = got[i, hd * h:hd * h + hd], clean[i, hd * h:hd * h + hd]
            hit = (i, h) in ((0, 0), (c.rows.used - 1, 1))
            assert torch.isnan(a).all() if hit else torch.equal(a, b), (i, h)


@pytest.mark.parametrize("new,lens", [([3], [3]), ([1], [300]), ([40], [90]), ([1], [9000])])
def test_scores_that_overflow(pkg, new, lens):
    """fp32 products beyond the largest number: a row whose every score is one is NaN, keys with such a score beside others weigh nothing."""
    c = Call(pkg, "f32", "f32", 2, 1, 64, new, lens, seed=51)
    n = lens[0]
    k = torch.zeros(n, 1, 64)
    k[:, 0, 5] = -1e30
    k[::3, 0, 6] = 1e30
    _store(c, "k", 0, k)
    q = torch.zeros(new[0], 2, 64)
    q[:, 0, 5] = 1e30  # each score -infinity
    q[:, 1, 6] = -1e30  # of every third key
    _query(c, q.flatten(1))
    got = c.run().double()
    assert torch.isnan(got[:new[0], :64]).all()
    for i in range(new[0]):
        p = n - new[0] + i
        some = [j for j in range(p + 1) if j % 3]
        if not some:
            assert torch.isnan(got[i, 64:]).all()
            continue
        v = c.vals[0][some, 0]
        # equal weights: fp32 sums in any order, 64 terms of the size of the values at most between roundings
        assert ((got[i, 64:] - v.mean(0)).abs() <= (len(some) + 8) * 2.0 ** -24 * v.abs().mean(0)).all()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,lens", [([4, 2], [66, 70]), ([90, 2], [66, 9000]), ([4, 2], [66, 9000])])
def test_nothing_seen_is_zero(pkg, kind, cache, new, lens):
    """Rows at negative positions are zero whatever stands in them; with keys split over workgroups too."""
    c = Call(pkg, kind, cache, 2, 1, 64, new, lens, seed=52)
    c.rows.dlen.copy_(torch.tensor([new[0] - 3, lens[1]], dtype=torch.int32))
    c.dq[0], c.dq[1] = math.nan, math.inf
    got = c.run()
    assert (got[:3] == 0).all() and not (got[3:] == 0).any(1).all()


# ---------------------------------------------------------------------------------------------------------------------
# weights
# ---------------------------------------------------------------------------------------------------------------------
HALVES = [("f16", "f16"), ("f16", "q4"), ("bf16", "q4")]


@pytest.mark.parametrize("kind,cache", HALVES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new", [1, 6, 80])
def test_small_weights_of_a_long_sequence(pkg, kind, cache, hd, new):
    """One key whose score is 17 above those of 60000 others that make up the whole result, 60000 e^-17 = 0.0025: each weight is below half a step of the smallest halves.
    Weights are held to 2^-32 of the largest at least; maxLen keeps the keys in one workgroup, as they are in a call of many sequences."""
    n = 60000
    c = Call(pkg, kind, cache, 1, 1, hd, [new], [n], seed=53)
    k, v = torch.zeros(n, 1, hd), torch.ones(n, 1, hd)
    k[0], v[0] = 1.0, 0.0
    _store(c, "k", 0, k)
    _store(c, "v", 0, v)
    _query(c, torch.full((new, hd), 17.0 / math.sqrt(hd)))
    c.args.maxLen = 1
    c.work_for(c.args)
    assert c.args.workBytes == 0
    got = c.run().double()
    q = c.q.double()[0, 0]
    for i in range(new):
        others = (n - new + i) * math.exp(-float(q) * hd * c.scale)
        want = others / (1 + others)
        # scores of equal products: hd + 4 roundings; weights: 2^-32 of the largest each, or 2^-11 of their own size, the coarser one
        bound = U[kind] * want + want * (2 * 17 * (hd + 4) * 2.0 ** -24 + U["f16"] + 2.0 ** -18) + (n - new + i) * 2.0 ** -32 + (2.0 ** -25 if kind == "f16" else 0)
        assert ((got[i] - want).abs() <= bound).all(), (i, got[i, 0].item(), want, bound)


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,lens", [([1], [700]), ([6, 1], [300, 5000]), ([90], [400])])
def test_weights_sum_to_one(pkg, kind, cache, hd, new, lens):
    """Values that are all one: the result is one, whatever the weights are rounded to, as what is summed is what is multiplied.  (fp32 sums of both in their orders: off by a few
    2^-24 for each key, which a 16-bit result does not show; fp32 rows by twice that.)  One key in 16 weighs 1, the others 1/2 (1 + 0.45 steps): rounded, all err to one side."""
    weight = 0.5 * (1 + 0.45 * 2 * U[kind if cache == kind else "f16"])
    c = Call(pkg, kind, cache, 1, 1, hd, new, lens, seed=54, scale=-math.log(weight) / hd)
    for s, n in enumerate(lens):
        k = torch.full((n, 1, hd), -1.0)
        k[3::16] = 0.0
        _store(c, "k", s, k)
        _store(c, "v", s, torch.ones(n, 1, hd))
    _query(c, torch.ones(c.rows.used, hd))
    got = c.run().double()[:c.rows.used]
    if kind == "f32":
        assert ((got - 1).abs() <= 2 * max(lens) * 2.0 ** -24).all()
    else:
        assert (got == 1).all(), (got - 1).abs().max().item()


# ---------------------------------------------------------------------------------------------------------------------
# few fp16 rows over 4-bit pages: K as it is, weights to 22 bits
# ---------------------------------------------------------------------------------------------------------------------
FORMS = [(1, 1, 64), (1, 1, 128), (1, 20, 64), (1, 20, 128), (20, 1, 64), (20, 1, 128)]  # query heads, rows of a sequence, head size: a column for each group (the first two); 16 rows a workgroup


def _few(c, seq, keys, weights):
    """Results [n, H, hd] of a sequence in 64 bits, and their bound: K as the codes have it, weights to 2^-22 of their size or 2^-32 of the largest, values that are halves.
    Scores: fp32 sums of minimum * (sum of the row's elements) and of code * scale * element in two parts, a rounding of that size for each element that is not zero and 16 more;
    the row's sum as two halves, and elements of the row below 2^-24 of its largest.  keys: what the scores are of; weights: what is done to them (a mistake to be found)."""
    r0, n = int(c.rows.start[seq]), c.rows.new[seq]
    q = c.q[r0:r0 + n, :c.H * c.hd].double().unflatten(1, (c.H, c.hd))
    k, v = keys[:, 0], c.vals[seq][:, 0]
    low = k.unflatten(-1, (-1, GROUP)).amin(-1, keepdim=True).expand(-1, -1, GROUP).flatten(1)
    want, bound = torch.zeros(n, c.H, c.hd, dtype=torch.float64), torch.zeros(n, c.H, c.hd, dtype=torch.float64)
    for i in range(n):
        at = c.rows.lens[seq] - n + i + 1
        for h in range(c.H):
            s = k[:at] @ q[i, h] * c.scale
            size = (low[:at].abs() + (k - low)[:at].abs()) @ q[i, h].abs() * c.scale
            ds = size * (2 * int((q[i, h] != 0).sum()) + 16) * 2.0 ** -24 + 2.0 ** -22 * (low[:at].abs() @ q[i, h].abs()) * c.scale
            ds = ds + 2.0 ** -24 * q[i, h].abs().max() * (low.abs() + (k - low))[:at].sum(1) * c.scale + s.abs().max() * 2.0 ** -22
            p = weights(torch.exp(s - s.max()))
            l = p.sum()
            p = p / l
            want[i, h] = p @ v[:at]
            e = 2.0 ** -22 + 2 * (ds + (p * ds).sum()) + (at ** 0.5 + 16) * 2.0 ** -22
            bound[i, h] = (p * e) @ v[:at].abs() + 2.0 ** -32 / l * v[:at].abs().sum(0) + U["f16"] * want[i, h].abs() + 2.0 ** -25
    return want, bound


def _found(c, got, keys=lambda k: k, weights=lambda p: p):
    """The largest difference from that, in bounds."""
    worst = 0.0
    for s, n in enumerate(c.rows.new):
        want, bound = _few(c, s, keys(c.keys[s]), weights)
        g = got[int(c.rows.start[s]):int(c.rows.start[s]) + n, :c.H * c.hd].double().unflatten(1, (c.H, c.hd))
        worst = max(worst, ((g - want).abs() / bound).nan_to_num(1e9).max().item())
    return worst


def _two_of_a_row(gen, c):
    """Rows of two elements that are not zero: the roundings of longer sums would hide what is looked for."""
    q = torch.randn(c.rows.used, c.H, c.hd, generator=gen)
    some = torch.rand(c.rows.used, c.H, c.hd, generator=gen).argsort(-1) < 2
    return torch.where(some, q, torch.zeros_like(q)).flatten(1)


@pytest.mark.parametrize("H,rows,hd", FORMS)
def test_weights_of_few_rows(pkg, H, rows, hd):
    """Keys in pairs with almost the same score and opposite values, so that the result is a small difference of large sums: weights of 11 bits would miss the bound."""
    lens = [rows + i % 10 for i in range(1, 41)] if rows == 1 else [rows + 2 * i for i in range(1, 13)]
    c = Call(pkg, "f16", "q4", H, 1, hd, [rows] * len(lens), lens, seed=55, scale=0.1)
    gen = torch.Generator().manual_seed(56)
    for s, n in enumerate(lens):
        k = torch.randn((n + 1) // 2, 1, hd, generator=gen).repeat_interleave(2, 0)
        k[1::2] *= 1.01
        v = torch.where(torch.rand((n + 1) // 2, 1, hd // GROUP, generator=gen) < 0.5, 1.0, -1.0).repeat_interleave(2, 0)
        v[1::2] *= -1
        _store(c, "k", s, k[:n])
        _store(c, "v", s, v.repeat_interleave(GROUP, -1)[:n])  # (one value a group: exact)
        assert (c.vals[s].abs() == 1).all()
    _query(c, _two_of_a_row(gen, c))
    got = c.run()
    assert _found(c, got) <= 1
    assert _found(c, got, weights=lambda p: p.half().double()) > 2


@pytest.mark.parametrize("H,rows,hd", FORMS)
@pytest.mark.parametrize("low,span,scale,spread", [(1000.0, 2.0, 0.1, 1.0), (-40000.0, 80000.0, 1e-3, 0.02), (0.0, 1e-5, 2.0 ** 16, 1.0), (0.25, 3e-4, 2.0 ** 9, 1.0)])
def test_keys_of_few_rows(pkg, H, rows, hd, low, span, scale, spread):
    """Keys whose differences halves would lose (from 1000 to 1002), whose groups span more than they hold, and with scales below the normal halves: taken as they are."""
    lens = [rows + i % 10 for i in range(1, 41)] if rows == 1 else [rows + 3 * i for i in range(1, 13)]
    c = Call(pkg, "f16", "q4", H, 1, hd, [rows] * len(lens), lens, seed=57, scale=scale / 8)
    gen = torch.Generator().manual_seed(58)
    for s, n in enumerate(lens):
        x = torch.rand(n, 1, hd // GROUP, GROUP, generator=gen)
        x[..., 3], x[..., 9] = 0.0, 1.0
        _store(c, "k", s, (low + span * x).flatten(2))
        _store(c, "v", s, torch.where(torch.rand(n, 1, hd // GROUP, generator=gen) < 0.5, 1.0, -1.0).repeat_interleave(GROUP, -1))
    _query(c, _two_of_a_row(gen, c) * spread)
    got = c.run()
    assert _found(c, got) <= 1
    if low > 0:
        assert _found(c, got, keys=lambda k: k.half().double()) > 2
