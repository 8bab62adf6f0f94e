"""Operators on a paged K/V cache through the C ABI (rows in, rows back, attention with window and first positions), against the
64-bit restatement in kv_oracle.  Places where nothing is stored hold NaN throughout."""
import ctypes
import math

import pytest
import torch

from kv_oracle import PAGE, TORCH, U, Pools, Rows, attend, codes_of, tile_bytes

pytestmark = pytest.mark.gpu

KINDS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "q4"), ("bf16", "q4"), ("f16", "q4")]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen)


class Call:
    """One attention call over a filled cache."""

    def __init__(self, pkg, kind, cache, H, K, hd, new, lens, window=0, sinks=0, scale=0.0, seed=0, pad=0, spread=1.0, max_len=True, q_stride=0, out_stride=0):
        gen = torch.Generator().manual_seed(1000 + seed)
        self.pkg, self.kind, self.four, self.hd, self.H, self.window, self.sinks = pkg, kind, cache == "q4", hd, H, window, sinks
        self.pools = Pools(pkg, cache, K, hd, lens, seed)
        self.rows = Rows(pkg, kind, H, new, lens, pad)
        self.keys, self.vals = [], []
        for s, n in enumerate(lens):
            n = max(n, 0)
            k, v = (_normal(gen, n, K, hd).to(TORCH[kind]).float() for _ in range(2))
            self.keys.append(self.pools.put("k", s, 0, k) if n else torch.zeros(0, K, hd, dtype=torch.float64))
            self.vals.append(self.pools.put("v", s, 0, v) if n else torch.zeros(0, K, hd, dtype=torch.float64))
        qs, os = q_stride or H * hd, out_stride or H * hd
        self.q = torch.full((max(self.rows.rows, 1), qs), math.nan, dtype=TORCH[kind])
        self.q[:self.rows.used, :H * hd] = (_normal(gen, self.rows.used, H * hd) * spread).to(TORCH[kind])
        self.scale = scale or 1.0 / math.sqrt(hd)
        self.pools.to_gpu()
        self.dq = self.q.cuda()
        self.out = torch.full((max(self.rows.rows, 1), os), 77.0, dtype=TORCH[kind], device="cuda")
        self.cache, self.batch = self.pools.struct(), self.rows.struct()
        self.args = pkg.Attention(q=self.dq.data_ptr(), qStride=qs, out=self.out.data_ptr(), outStride=os, window=window, sinks=sinks, scale=scale,
                                  maxLen=max(max(lens), 1) if max_len else 0, maxNew=max(max(new), 1) if max_len else 0)
        self.work_for(self.args)

    def work_for(self, args):
        n = self.pkg.attention_work_bytes(self.cache, self.batch, args)
        self.work = torch.full((max(n, 16),), 255, dtype=torch.uint8, device="cuda")
        args.work, args.workBytes = self.work.data_ptr(), n

    def run(self, stream=None):
        self.pkg.attention(self.cache, self.batch, self.args, _stream() if stream is None else stream)
        torch.cuda.synchronize()
        return self.out.cpu()

    def want(self, s):
        r0, n = int(self.rows.start[s]), self.rows.new[s]
        q = self.q[r0:r0 + n, :self.H * self.hd].double().unflatten(1, (self.H, self.hd))
        return attend(q, self.keys[s], self.vals[s], self.rows.lens[s] - n, self.window, self.sinks, self.scale, self.kind, self.four)

    def check(self, got=None):
        got = self.run() if got is None else got
        for s, n in enumerate(self.rows.new):
            if n == 0:
                continue
            r0 = int(self.rows.start[s])
            g = got[r0:r0 + n, :self.H * self.hd].double().unflatten(1, (self.H, self.hd))
            want, bound = self.want(s)
            bad = ~((g - want).abs() <= bound)
            assert not bad.any(), (f"sequence {s}: {int(bad.sum())} of {bad.numel()} elements off, first at {bad.nonzero()[0].tolist()}: got {g[bad][0]} want {want[bad][0]} "
                                   f"bound {bound[bad][0]:.3e}; worst {((g - want).abs() / bound).nan_to_num(1e9).max():.3f} bounds")
        if got.shape[0] > self.rows.used:
            assert (got[self.rows.used:] == 77.0).all(), "rows behind the last sequence were written"
        if got.shape[1] > self.H * self.hd:
            assert (got[:, self.H * self.hd:] == 77.0).all(), "columns between rows were written"


SHAPES = [  # new rows and lengths of the sequences
    ([1], [1]), ([1], [64]), ([1], [65]), ([1], [577]), ([1] * 5, [1, 63, 200, 0, 129]),
    ([1, 0, 1, 3], [70, 50, 5, 130]), ([17], [17]), ([100, 1, 64], [100, 300, 70]), ([130, 5], [130, 260]), ([300], [1100]),
]
MASKS = [(0, 0), (1, 0), (5, 1), (64, 3), (100, 70), (1000, 4)]


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd,H,K", [(64, 4, 4), (128, 2, 2), (128, 8, 2), (64, 6, 2)])
def test_attention_small(pkg, kind, cache, hd, H, K):
    for i, (new, lens) in enumerate(SHAPES):
        if hd * H > 512 and sum(new) > 150:
            continue
        window, sinks = MASKS[(i + H + hd // 64) % len(MASKS)]
        Call(pkg, kind, cache, H, K, hd, new, lens, window, sinks, seed=i, pad=i % 3).check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("window,sinks", MASKS + [(2, 2), (63, 64), (65, 65), (128, 1)])
def test_masks(pkg, kind, cache, window, sinks):
    Call(pkg, kind, cache, 2, 1, 64, [70, 1, 1, 2], [270, 300, 64, 129], window, sinks, seed=window).check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("H,K", [(1, 1), (3, 1), (5, 1), (16, 1), (17, 1), (24, 3), (32, 1)])
def test_head_groups(pkg, kind, cache, H, K):
    Call(pkg, kind, cache, H, K, 64, [1, 2, 9], [150, 66, 9], 40, 2, seed=H).check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_long(pkg, kind, cache, hd):
    """Split over a long axis, alone and beside short ones; sharp weights; without the hints too."""
    Call(pkg, kind, cache, 4, 2, hd, [1], [9000], seed=1).check()
    Call(pkg, kind, cache, 2, 1, hd, [1, 1, 1], [5000, 3, 700], seed=2, spread=6.0).check()
    Call(pkg, kind, cache, 2, 2, hd, [1, 2], [4100, 900], 2000, 5, seed=3, max_len=False).check()
    Call(pkg, kind, cache, 2, 2, hd, [40], [3000], 0, 0, seed=4).check()


@pytest.mark.parametrize("kind,cache", KINDS)
def test_scale_and_strides(pkg, kind, cache):
    Call(pkg, kind, cache, 2, 2, 64, [5, 1], [80, 90], seed=5, scale=0.37, q_stride=3 * 128 + 16, out_stride=128 + 8, pad=2).check()
    Call(pkg, kind, cache, 2, 2, 64, [150], [150], 30, 1, seed=6, scale=0.01, q_stride=400, out_stride=136).check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,lens", [([70], [200]), ([1, 1], [200, 190]), ([300], [300])])
def test_nonfinite_in_masked_places(pkg, kind, cache, new, lens):
    """NaN and infinities at positions that some rows see and others do not: the others are as without them."""
    c = Call(pkg, kind, cache, 2, 1, 64, new, lens, 40, 2, seed=9)
    clean = c.run().clone()
    spots = [100, 150, lens[0] - 3]
    for at, x in zip(spots, (math.nan, math.inf, -math.inf)):
        c.pools.put("k", 0, at, torch.full((1, 1, 64), x))
        c.pools.put("v", 0, at, torch.full((1, 1, 64), x))
    c.pools.dk.copy_(c.pools.k)
    c.pools.dv.copy_(c.pools.v)
    got = c.run()
    for i in range(new[0]):
        p = lens[0] - new[0] + i
        hit = any(at <= p and (p - at < 40 or at < 2) for at in spots)
        assert torch.isnan(got[i]).any() if hit else torch.equal(got[i], clean[i]), f"position {p}"
    for i in range(new[0], sum(new)):
        assert torch.equal(got[i], clean[i])


def test_infinite_value_only(pkg):
    """An infinite value that is seen gives an infinity; a row that does not see it is untouched."""
    for kind in ("f32", "bf16", "f16"):
        c = Call(pkg, kind, kind, 1, 1, 64, [90], [90], 0, 0, seed=3)
        clean = c.run().clone()
        c.pools.v[c.pools.table[0, 0].long(), 50, 0, 7] = math.inf
        c.pools.dv.copy_(c.pools.v)
        got = c.run()
        assert torch.equal(got[:50], clean[:50])
        assert torch.isinf(got[50:, 7]).all()
        other = [d for d in range(64) if d != 7]
        assert torch.allclose(got[50:, other].float(), clean[50:, other].float(), rtol=4 * U[kind], atol=4 * U[kind])


@pytest.mark.parametrize("kind,cache", KINDS)
def test_pages(pkg, kind, cache):
    """Entries of pages that no row sees may be anything; a row that sees a page outside the pool is NaN."""
    c = Call(pkg, kind, cache, 2, 2, 64, [1, 3], [400, 260], 64, 3, seed=4)
    clean = c.run().clone()
    hidden = c.pools.dtable.clone()
    hidden[0, 1:5] = torch.tensor([-5, 10 ** 9, c.pools.pages, -2 ** 31], dtype=torch.int32)  # the window of position 399 begins at 336
    c.pools.dtable.copy_(hidden)
    assert torch.equal(c.run(), clean)
    c.pools.dtable[0, 0] = -1  # its first tokens
    got = c.run()
    assert torch.isnan(got[0]).all() and torch.equal(got[1:], clean[1:])
    c.pools.dtable.copy_(hidden)
    c.pools.dtable[1, 4] = c.pools.pages  # positions 256 ..: the newest of sequence 1
    got = c.run()
    assert torch.equal(got[0], clean[0]) and torch.isnan(got[2:4]).any(1).all()


def test_lengths_that_do_not_fit(pkg):
    """Rows at negative positions see nothing; a length beyond the page table is NaN, not a read behind it."""
    for kind, cache in KINDS:
        c = Call(pkg, kind, cache, 2, 2, 64, [4, 2], [66, 70], seed=4)
        clean = c.run().clone()
        c.rows.dlen.copy_(torch.tensor([2, 70], dtype=torch.int32))
        got = c.run()
        assert (got[:2] == 0).all() and not (got[2:4] == 0).all() and torch.equal(got[4:], clean[4:])
        c.rows.dlen.copy_(torch.tensor([-7, 70], dtype=torch.int32))
        got = c.run()
        assert (got[:4] == 0).all() and torch.equal(got[4:], clean[4:])
        c.rows.dlen.copy_(torch.tensor([66, 200], dtype=torch.int32))
        got = c.run()
        assert torch.equal(got[:4], clean[:4]) and torch.isnan(got[4:]).all()


@pytest.mark.parametrize("kind,cache", KINDS)
def test_offsets_beyond_32_bits(pkg, kind, cache):
    """Pages whose bytes and elements start behind 2^32."""
    if kind != "bf16" and kind != "f32":
        pytest.skip("the same offsets as bf16")
    K, hd = 16, 128
    c = Call(pkg, kind, cache, K, K, hd, [1, 20], [130, 70], seed=8)
    clean = c.run().clone()
    per = pkg.kv_page_bytes(codes_of(pkg)[cache], K, hd)
    pages = int(2 ** 32 * (1 if cache == "q4" else c.pools.k.element_size()) // per) + 40
    for name in ("dk", "dv"):
        small = getattr(c.pools, name)
        big = torch.empty((pages,) + tuple(small.shape[1:]), dtype=small.dtype, device="cuda")
        big[pages - small.shape[0]:] = small
        setattr(c.pools, name, big)
    c.pools.dtable += pages - c.pools.pages
    c.pools.pages = pages
    c.cache = c.pools.struct()
    assert torch.equal(c.run(), clean)


def test_graph_replays(pkg):
    """A captured call follows tables, lengths and rows as they are at each replay."""
    for kind, cache in (("bf16", "bf16"), ("f32", "q4"), ("f16", "q4")):
        c = Call(pkg, kind, cache, 4, 2, 64, [1, 1, 1], [2000, 300, 65], 0, 0, seed=11)
        eager = {}
        lens = {"a": [2000, 300, 65], "b": [1999, 7, 64], "c": [64, 1, 1]}
        for name, l in lens.items():
            c.rows.dlen.copy_(torch.tensor(l, dtype=torch.int32))
            eager[name] = c.run().clone()
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                pkg.attention(c.cache, c.batch, c.args, torch.cuda.current_stream().cuda_stream)
        for name in ("b", "a", "c", "a", "b"):
            c.rows.dlen.copy_(torch.tensor(lens[name], dtype=torch.int32))
            c.out.fill_(5.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert _same_bits(c.out.cpu(), eager[name]), name  # ("c" sees a position that holds NaN)
            torch.randn(1000, device="cuda").sum().item()


def test_graph_of_prompts(pkg):
    """The kernel of many rows in a graph: replays with other lengths, rows and hints than at the capture."""
    for kind, cache in (("bf16", "bf16"), ("f16", "q4"), ("f32", "f32")):
        c = Call(pkg, kind, cache, 4, 2, 128, [130, 90], [200, 90], 64, 2, seed=12)
        lens, starts = {"a": [200, 90], "b": [150, 64], "c": [129, 91]}, {"a": [0, 130, 220], "b": [0, 100, 101], "c": [0, 1, 200]}
        eager = {}
        for name in lens:
            c.rows.dlen.copy_(torch.tensor(lens[name], dtype=torch.int32))
            c.rows.dstart.copy_(torch.tensor(starts[name], dtype=torch.int32))
            c.out.fill_(5.0)
            eager[name] = c.run().clone()
            assert (eager[name][starts[name][-1]:] == 5.0).all()
        side = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            with torch.cuda.graph(g, stream=side):
                pkg.attention(c.cache, c.batch, c.args, torch.cuda.current_stream().cuda_stream)
        for name in ("b", "a", "c", "b"):
            c.rows.dlen.copy_(torch.tensor(lens[name], dtype=torch.int32))
            c.rows.dstart.copy_(torch.tensor(starts[name], dtype=torch.int32))
            c.out.fill_(5.0)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert _same_bits(c.out.cpu(), eager[name]), name  # ("c" sees a position that holds NaN)
            torch.randn(1000, device="cuda").sum().item()


@pytest.mark.parametrize("kind,cache", KINDS)
def test_hints_decide_nothing_else(pkg, kind, cache):
    """maxLen and maxNew that are too small, too large or missing: other kernels and splits, results within the bounds."""
    for max_len, max_new in ((1, 1), (0, 0), (100000, 5), (7, 1000)):
        for new, lens, window in (([1, 1], [1500, 3], 0), ([90, 40], [400, 40], 70)):
            c = Call(pkg, kind, cache, 4, 2, 64, new, lens, window, 3, seed=31)
            c.args.maxLen, c.args.maxNew = max_len, max_new
            c.work_for(c.args)
            c.check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd,lens", [(64, [17000, 40]), (128, [33100])])
def test_more_shares_than_lanes(pkg, kind, cache, hd, lens):
    """One K/V head and a long sequence: its keys are split over more workgroups than a wave has lanes."""
    c = Call(pkg, kind, cache, 3, 1, hd, [1] * len(lens), lens, seed=8)
    assert c.args.workBytes > 64 * 3 * len(lens) * (hd + 2) * 4
    c.check()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind,spread,scale", [("bf16", 1e30, 1e-30), ("bf16", 1e-25, 1e24), ("bf16", 3e4, 1e-5), ("f16", 1.2e4, 1e-5), ("f16", 1e-5, 1e4)])
def test_sizes_of_rows(pkg, kind, spread, scale, hd):
    """4-bit pages: rows far from one, large and small, with a scale that brings the scores back (they leave for powers of two and return)."""
    for new, lens in (([1, 1], [300, 65]), ([5], [200]), ([70], [100])):
        Call(pkg, kind, "q4", 2, 1, hd, new, lens, seed=23, spread=spread, scale=scale).check()


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("new,lens", [([3, 1], [90, 200]), ([150], [200])])
def test_nonfinite_rows(pkg, kind, cache, new, lens):
    """A row of q with NaN or infinities is none of its neighbours' business."""
    c = Call(pkg, kind, cache, 2, 1, 64, new, lens, 60, 2, seed=14)
    clean = c.run().clone()
    bad = [0, new[0] - 1]
    c.dq[bad[0], 5] = math.nan
    c.dq[bad[1], 70] = math.inf
    got = c.run()
    for i in range(sum(new)):
        for h in range(2):
            hit = (i == bad[0] and h == 0) or (i == bad[1] and h == 1)
            a, b = got[i, 64 * h:64 * h + 64], clean[i, 64 * h:64 * h + 64]
            assert torch.isnan(a).any() if hit else torch.equal(a, b), (i, h)


def test_many_sequences(pkg):
    """More sequences than a search step has places; some without rows."""
    new = [(7 * i) % 3 for i in range(150)]
    lens = [n + (11 * i) % 70 for i, n in enumerate(new)]
    for kind, cache in (("bf16", "bf16"), ("f32", "f32"), ("f16", "q4")):
        Call(pkg, kind, cache, 2, 1, 64, new, lens, 20, 1, seed=3, pad=4).check()
    a = Append(pkg, "bf16", "q4", 2, 1, 64, new, lens, seed=3, pad=4)
    a.run()
    a.expect()
    assert _same_bits(a.pools.dk.cpu(), a.pools.k) and _same_bits(a.pools.dv.cpu(), a.pools.v)


@pytest.mark.parametrize("n", [2, 8, 9, 33, 64, 65])
@pytest.mark.parametrize("kind,cache", [("bf16", "bf16"), ("f32", "q4"), ("f16", "q4")])
def test_order_of_sequences(pkg, kind, cache, n):
    """Sequences are taken longest first, up to 64 of them: single tokens, rows of every number, equal lengths, some without rows, the last rows of all untouched."""
    one = [1] * n
    some = [(5 * i + 2) % 4 for i in range(n)]
    most = [70 if i % 7 == 3 else (3 * i) % 5 for i in range(n)]
    for new in (one, some, most):
        lens = [m + (53 * i) % 130 if i % 3 else 80 for i, m in enumerate(new)]
        Call(pkg, kind, cache, 2, 1, 64, new, lens, 90, 2, seed=n, pad=3).check()


def test_small_work_is_refused(pkg):
    c = Call(pkg, "bf16", "bf16", 2, 1, 64, [1], [9000], seed=1)
    assert c.args.workBytes > 0
    for change in (dict(workBytes=c.args.workBytes - 1), dict(work=None), dict(work=c.args.work + 8)):
        c.work_for(c.args)
        for k, v in change.items():
            setattr(c.args, k, v)
        with pytest.raises(pkg.MlhError, match="work"):
            c.run()


def test_two_streams(pkg):
    """Calls on two streams at once, each with work memory of its own."""
    calls = [Call(pkg, "bf16", "bf16", 8, 2, 128, [1, 1], [6000, 5000], seed=i) for i in range(2)]
    alone = [c.run().clone() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(5):
        for c in calls:
            c.out.fill_(3.0)
        torch.cuda.synchronize()
        for c, st in zip(calls, streams):
            pkg.attention(c.cache, c.batch, c.args, st.cuda_stream)
        torch.cuda.synchronize()
        for c, want in zip(calls, alone):
            assert torch.equal(c.out.cpu(), want)


def test_same_answer_every_time(pkg):
    for kind, cache in KINDS:
        c = Call(pkg, kind, cache, 8, 2, 64, [1, 1, 30], [3000, 200, 500], seed=21)
        first = c.run().clone()
        for _ in range(4):
            c.work.random_(0, 255)
            assert torch.equal(c.run(), first)


# ---------------------------------------------------------------------------------------------------------------------
# rows in and back
# ---------------------------------------------------------------------------------------------------------------------
def _table(rows, hd):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd)
    return torch.stack([a.cos(), a.sin()], -1).flatten(1).float()


def _norm(x, gain):
    """Per-head norm in 64 bits, rounded to fp32: x [n, heads, hd] fp32."""
    d = x.double()
    return (gain.double().reshape(x.shape[1], x.shape[2]) * (d / (d.square().mean(-1, keepdim=True) + 1e-8).sqrt())).float()


def _turn(x, cs):
    a, b = x.double().unflatten(-1, (-1, 2)).unbind(-1)
    c, s = cs.double().unflatten(-1, (-1, 2))[:, None].unbind(-1)
    return torch.stack([c * a - s * b, s * a + c * b], -1).flatten(-2).float()


class Append:
    def __init__(self, pkg, kind, cache, H, K, hd, new, lens, rope=True, gains=False, with_q=True, pad=0, extra=0, in_place=False, seed=0, special=None):
        gen = torch.Generator().manual_seed(seed + 77)
        self.pkg, self.kind, self.H, self.K, self.hd = pkg, kind, H, K, hd
        self.pools = Pools(pkg, cache, K, hd, lens, seed)
        self.rows = Rows(pkg, kind, H, new, lens, pad)
        n, t = max(self.rows.rows, 1), TORCH[kind]
        self.q, self.k, self.v = (_normal(gen, n, w * hd + extra).to(t) for w in (H, K, K))
        if special is not None:
            special(self)
        self.rope = _table(max(lens), hd) if rope else None
        self.gains = [1 + 0.3 * torch.rand(w * hd, generator=gen) for w in (H, K)] if gains else None
        d = self.d = {"q": self.q.cuda(), "k": self.k.cuda(), "v": self.v.cuda()}
        if rope:
            d["rope"] = self.rope.cuda()
        if gains:
            d["gq"], d["gk"] = (g.cuda() for g in self.gains)
        d["qout"] = d["q"] if in_place else torch.full_like(d["q"], 77.0)
        self.with_q = with_q
        self.pools.to_gpu()
        self.cache, self.batch = self.pools.struct(), self.rows.struct()
        self.args = pkg.KvAppend(k=d["k"].data_ptr(), kStride=K * hd + extra, v=d["v"].data_ptr(), vStride=K * hd + extra,
                                 rope=d["rope"].data_ptr() if rope else None, ropeRows=max(lens) if rope else 0, kGain=d["gk"].data_ptr() if gains else None)
        if with_q:
            self.args.q, self.args.qOut, self.args.qStride, self.args.qOutStride = d["q"].data_ptr(), d["qout"].data_ptr(), H * hd + extra, H * hd + extra
            self.args.qGain = d["gq"].data_ptr() if gains else None

    def run(self):
        self.pkg.kv_append(self.cache, self.batch, self.args, _stream())
        torch.cuda.synchronize()

    def rotated(self, name, heads, gain):
        x = getattr(self, name)[:self.rows.used, :heads * self.hd].float().unflatten(1, (heads, self.hd))
        if gain is not None:
            x = _norm(x, gain)
        pos = torch.cat([torch.arange(n - m, n) for m, n in zip(self.rows.new, self.rows.lens)])
        return _turn(x, self.rope[pos]) if self.rope is not None and name != "v" else x

    def expect(self):
        q = self.rotated("q", self.H, self.gains[0] if self.gains else None).to(TORCH[self.kind])
        k, v = self.rotated("k", self.K, self.gains[1] if self.gains else None), self.rotated("v", self.K, None)
        for s, (m, n) in enumerate(zip(self.rows.new, self.rows.lens)):
            if m:
                r0 = int(self.rows.start[s])
                self.pools.put("k", s, n - m, k[r0:r0 + m])
                self.pools.put("v", s, n - m, v[r0:r0 + m])
        return q


def _same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("kind,cache", KINDS)
@pytest.mark.parametrize("hd,H,K", [(64, 4, 4), (128, 6, 2), (64, 33, 11), (128, 16, 16)])
@pytest.mark.parametrize("rope", [True, False])
def test_append(pkg, kind, cache, hd, H, K, rope):
    for i, (new, lens) in enumerate([([1], [1]), ([1, 1, 1], [65, 1, 200]), ([70, 0, 5], [70, 30, 133]), ([129], [300])]):
        a = Append(pkg, kind, cache, H, K, hd, new, lens, rope=rope, pad=i, extra=16 * (i % 2), seed=i)
        a.run()
        want = a.expect()
        got = a.d["qout"].cpu()
        assert _same_bits(got[:a.rows.used, :H * hd], want.flatten(1))
        assert (got[a.rows.used:] == 77).all() and (got[:, H * hd:] == 77).all()
        # the pools whole: what was stored, and everything else untouched
        assert _same_bits(a.pools.dk.cpu(), a.pools.k), f"keys, {new} {lens}"
        assert _same_bits(a.pools.dv.cpu(), a.pools.v), f"values, {new} {lens}"
        # and back, in every type
        for to, t in TORCH.items():
            back = [torch.full((a.rows.rows, K * hd + 8), 77.0, dtype=t, device="cuda") for _ in range(2)]
            batch = Rows(pkg, to, 1, new, lens, i)
            pkg.kv_read(a.cache, batch.struct(), pkg.KvRead(k=back[0].data_ptr(), v=back[1].data_ptr(), stride=K * hd + 8), _stream())
            torch.cuda.synchronize()
            for name, b in zip("kv", back):
                x = a.rotated(name, K, None)
                if cache == "q4":
                    x = Pools(pkg, "q4", K, hd, [a.rows.used], 0).put("k", 0, 0, x).float()
                else:
                    x = x.to(TORCH[cache]).float()
                assert _same_bits(b.cpu()[:a.rows.used, :K * hd], x.to(t).flatten(1))
                assert (b.cpu()[a.rows.used:] == 77).all() and (b.cpu()[:, K * hd:] == 77).all()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128])
def test_append_with_gains(pkg, kind, hd):
    """Norm in 64 bits: fp32 results differ from the restatement's by a rounding of fp32 at most (sums in another order), stored ones by that and
    their own rounding."""
    a = Append(pkg, kind, kind, 6, 3, hd, [3, 40], [80, 40], gains=True, in_place=True, seed=5)
    a.run()
    want = a.expect().double()
    got = a.d["q"].cpu()[:a.rows.used].double().unflatten(1, (6, hd))
    # a pair's sum of two products: relative to the products' size
    size = (want.unflatten(-1, (-1, 2)).square().sum(-1, keepdim=True).sqrt().expand(-1, -1, -1, 2)).flatten(-2)
    assert ((got - want).abs() <= 4 * 2.0 ** -24 * size + 2 * U[kind] * want.abs() + (2.0 ** -24 if kind == "f16" else 0)).all()
    for d, h in ((a.pools.dk, a.pools.k), (a.pools.dv, a.pools.v)):
        d, h = d.cpu().double(), h.double()
        there = ~h.isnan()
        assert torch.equal(there, ~d.isnan())
        big = (h.unflatten(-1, (-1, 2)).square().sum(-1, keepdim=True).sqrt().expand(*h.shape[:3], -1, 2)).flatten(-2)
        assert ((d - h).abs() <= 4 * 2.0 ** -24 * big + 2 * U[kind] * h.abs() + (2.0 ** -24 if kind == "f16" else 0))[there].all()


def test_append_four_bits_edges(pkg):
    """Groups of one value, ties between codes, subnormal scales, non-finite elements."""
    def special(a):
        x = a.v.view(-1, 4, 64)
        x[0, 0] = 3.25
        x[1, 0, :32] = torch.arange(32).float() / 2  # scale ~ 1: halves lie between codes
        x[1, 0, 31] = 15
        x[1, 0, 0] = 0
        x[2, 1, :32] *= 1e-7
        x[3, 1, 5] = math.nan
        x[3, 2, 40] = math.inf
        x[3, 3, 0] = -math.inf
        x[4, 0, :32] = 0
        x[5, 0, :2] = torch.tensor([-65504.0, 65504.0])
        x[6, 0, 0] = -1e30
    for kind in ("f32", "bf16"):
        a = Append(pkg, kind, "q4", 4, 4, 64, [9], [70], seed=3, special=special)
        a.run()
        a.expect()
        for d, h in ((a.pools.dk, a.pools.k), (a.pools.dv, a.pools.v)):
            p, w = d.cpu()[..., 64 * 32:].contiguous().view(torch.float16), h[..., 64 * 32:].contiguous().view(torch.float16)
            assert torch.equal(p.isnan(), w.isnan()) and _same_bits(p.nan_to_num(), w.nan_to_num())
            assert _same_bits(d.cpu()[..., :64 * 32], h[..., :64 * 32])


def test_append_refused_places(pkg):
    """Rows at negative positions, beyond the page table or the rope table, or in a page outside the pool store nothing, and their q is NaN."""
    for kind, cache in KINDS:
        a = Append(pkg, kind, cache, 4, 2, 64, [3, 2, 1], [40, 66, 130], seed=6)
        a.rows.dlen.copy_(torch.tensor([1, 66, 64 * a.pools.per + 1], dtype=torch.int32))  # positions -2 -1 0 | 64 65 | one behind the table
        a.pools.dtable[1, 1] = a.pools.pages
        before = a.pools.dk.cpu().clone()
        a.run()
        got = a.d["qout"].cpu()
        assert torch.isnan(got[:2]).all() and torch.isfinite(got[2]).all() and torch.isnan(got[3:]).all()
        changed = (before.view(torch.uint8) != a.pools.dk.cpu().view(torch.uint8)).flatten(1).any(1)
        assert changed.nonzero().flatten().tolist() == [int(a.pools.table[0, 0])]
        back = torch.zeros(2, a.rows.rows, 2 * 64, device="cuda")
        batch = Rows(pkg, "f32", 1, a.rows.new, a.rows.lens)
        st = batch.struct()
        batch.dlen.copy_(a.rows.dlen)
        pkg.kv_read(a.cache, st, pkg.KvRead(k=back[0].data_ptr(), v=back[1].data_ptr(), stride=128), _stream())
        assert torch.isnan(back[:, :2]).all() and torch.isfinite(back[:, 2]).all() and torch.isnan(back[:, 3:]).all()
        a.rows.dlen.copy_(torch.tensor([40, 64, 130], dtype=torch.int32))
        a.args.ropeRows = 39  # the last row of sequence 0 is at 39
        a.run()
        got = a.d["qout"].cpu()
        assert torch.isfinite(got[:2]).all() and torch.isnan(got[2:]).all()


def test_append_without_q(pkg):
    a = Append(pkg, "bf16", "bf16", 4, 2, 64, [5], [70], with_q=False, seed=2)
    a.run()
    a.expect()
    assert _same_bits(a.pools.dk.cpu(), a.pools.k) and _same_bits(a.pools.dv.cpu(), a.pools.v) and (a.d["qout"].cpu() == 77).all()


@pytest.mark.parametrize("kind,cache", KINDS)
def test_together(pkg, kind, cache):
    """A prompt, then single tokens, as a model's layer uses them: append, attention of the rotated queries, everything captured into one graph that is replayed
    for every token; against the restatement over the rows as stored."""
    H, K, hd, prompt, steps = 4, 2, 64, 90, 6
    lens = [prompt + steps, prompt + steps - 13]
    a = Append(pkg, kind, cache, H, K, hd, [prompt, prompt - 13], [prompt, prompt - 13], seed=4)
    gen = torch.Generator().manual_seed(5)
    a.pools = Pools(pkg, cache, K, hd, lens, 4).to_gpu()
    a.rope = _table(max(lens), hd)
    a.d["rope"] = a.rope.cuda()
    a.args.rope, a.args.ropeRows, a.cache = a.d["rope"].data_ptr(), max(lens), a.pools.struct()
    out = torch.zeros_like(a.d["q"])
    att = pkg.Attention(q=a.d["qout"].data_ptr(), qStride=H * hd, out=out.data_ptr(), outStride=H * hd, window=50, sinks=4)
    n = pkg.attention_work_bytes(a.cache, a.batch, att)
    work = torch.zeros(max(n, 16), dtype=torch.uint8, device="cuda")
    att.work, att.workBytes = work.data_ptr(), n
    keys, vals = ([torch.zeros(0, K, hd, dtype=torch.float64)] * 2 for _ in range(2))

    def check(new):
        nonlocal keys, vals
        q = a.rotated("q", H, None).to(TORCH[kind]).double()
        k, v = a.rotated("k", K, None), a.rotated("v", K, None)
        r = 0
        for s, m in enumerate(new):
            p0 = a.rows.lens[s] - m
            keys[s] = torch.cat([keys[s], a.pools.put("k", s, p0, k[r:r + m])])
            vals[s] = torch.cat([vals[s], a.pools.put("v", s, p0, v[r:r + m])])
            want, bound = attend(q[r:r + m], keys[s], vals[s], p0, 50, 4, hd ** -0.5, kind, cache == "q4")
            got = out.cpu()[r:r + m].double().unflatten(1, (H, hd))
            assert ((got - want).abs() <= bound).all(), f"sequence {s}, position {p0}: {((got - want).abs() / bound).max()}"
            r += m

    a.run()
    pkg.attention(a.cache, a.batch, att, _stream())
    torch.cuda.synchronize()
    check([prompt, prompt - 13])
    rows = Rows(pkg, kind, H, [1, 1], [prompt, prompt - 13])
    batch = rows.struct()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(g, stream=side):
            pkg.kv_append(a.cache, batch, a.args, torch.cuda.current_stream().cuda_stream)
            pkg.attention(a.cache, batch, att, torch.cuda.current_stream().cuda_stream)
    a.rows = rows
    for i in range(steps):
        rows.lens = [n + 1 for n in rows.lens]
        for x, w in ((a.q, H), (a.k, K), (a.v, K)):
            x[:2] = _normal(gen, 2, w * hd).to(x.dtype)
        for name in ("q", "k", "v"):
            a.d[name].copy_(getattr(a, name))
        rows.dlen.copy_(torch.tensor(rows.lens, dtype=torch.int32))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check([1, 1])
    assert _same_bits(a.pools.dk.cpu(), a.pools.k) and _same_bits(a.pools.dv.cpu(), a.pools.v)


def test_no_rows(pkg):
    a = Append(pkg, "bf16", "bf16", 4, 2, 64, [0], [5], seed=2)
    a.batch.rows = 0
    a.run()
    c = Call(pkg, "bf16", "bf16", 2, 2, 64, [0, 0], [5, 0], pad=3)
    c.check()
