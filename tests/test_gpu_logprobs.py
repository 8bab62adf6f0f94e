"""mlh_logprobs_device against its formula in 64 bits."""
import ctypes
import math

import pytest
import torch

import step_oracle as so

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


class Call:
    def __init__(self, pkg, x, tokens=None, top=0, t=0.0, pad=0, shift=0, entropy=True):
        """x [rows, vocab] in its type; pad: elements between rows (NaN); shift: elements that the first row starts behind an aligned address."""
        self.x, self.top, self.t = x, top, ctypes.c_float(t).value  # (the temperature of a call is a float)
        rows, vocab = x.shape
        self.tokens = torch.zeros(rows, 0, dtype=torch.int32) if tokens is None else tokens.to(torch.int32)
        given = self.tokens.shape[1]
        flat = torch.full((rows * (vocab + pad) + shift + 8,), NAN, dtype=x.dtype)
        flat[shift:shift + rows * (vocab + pad)].unflatten(0, (rows, vocab + pad))[:, :vocab] = x
        self.buf = flat.cuda()
        self.dtok = self.tokens.cuda()
        self.lp, self.ent = torch.full((rows + 1, given), 55.0, device="cuda"), torch.full((rows + 1,), 55.0, device="cuda")
        self.ids, self.tlp = torch.full((rows + 1, top), -55, dtype=torch.int32, device="cuda"), torch.full((rows + 1, top), 55.0, device="cuda")
        kind = {v: k for k, v in so.TORCH.items()}[x.dtype]
        self.args = pkg.LogProbs(logits=self.buf.data_ptr() + shift * x.element_size(), stride=vocab + pad, tokens=self.dtok.data_ptr() if given else None,
                                 logProb=self.lp.data_ptr() if given else None, entropy=self.ent.data_ptr() if entropy else None, topIds=self.ids.data_ptr() if top else None,
                                 topLogProb=self.tlp.data_ptr() if top else None, rows=rows, vocab=vocab, type=so.code_of(pkg, kind), given=given, top=top, temperature=t)
        size = pkg.logprobs_work_bytes(self.args)
        self.work = torch.full((max(size, 16) + 64,), 255, dtype=torch.uint8, device="cuda")
        self.args.work, self.args.workBytes = self.work.data_ptr(), size
        self.size, self.entropy = size, entropy

    def check(self, what=""):
        torch.cuda.synchronize()
        (lp, ent, ids, tlp), (blp, bent, btlp) = so.logprobs(self.x, self.tokens, self.top, self.t or 1.0)
        rows = self.x.shape[0]
        assert torch.equal(self.ids[:rows].cpu(), ids), f"{what}: ids {(self.ids[:rows].cpu() != ids).nonzero()[:4].tolist()}"
        so.close(self.lp[:rows].cpu(), lp, blp, what + " given")
        so.close(self.tlp[:rows].cpu(), tlp, btlp, what + " top")
        if self.entropy:
            so.close(self.ent[:rows].cpu(), ent, bent, what + " entropy")
            assert float(self.ent[rows]) == 55.0
        else:
            assert bool((self.ent == 55.0).all())
        assert bool((self.lp[rows] == 55.0).all()) and bool((self.tlp[rows] == 55.0).all()) and bool((self.ids[rows] == -55).all())
        assert bool((self.work[max(self.size, 0):] == 255).all())


def logits(kind, rows, vocab, seed, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, vocab, generator=gen) * spread).to(so.TORCH[kind]), gen


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,given,top,pad,shift", [(1, 1, 1, 1, 0, 0), (1, 8192, 1, 5, 0, 0), (3, 7, 2, 7, 0, 1), (5, 100, 1, 64, 4, 0), (2, 2049, 3, 20, 0, 3), (17, 4099, 1, 1, 1, 5),
                                                            (4, 20160, 0, 10, 0, 0), (64, 777, 1, 0, 0, 0), (7, 50257, 4, 64, 0, 7), (2, 131075, 1, 20, 0, 0), (1, 262144, 1, 50, 0, 0), (600, 513, 1, 3, 0, 0),
                                                            (1, 300001, 1, 64, 0, 1), (130, 9001, 2, 33, 7, 2)])
def test_against_the_formula(pkg, kind, rows, vocab, given, top, pad, shift):
    x, gen = logits(kind, rows, vocab, rows * 7 + vocab)
    c = Call(pkg, x, torch.randint(0, vocab, (rows, given), generator=gen), top, pad=pad, shift=shift)
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("t", [1e-4, 0.25, 1.0, 7.0, 1e4])
def test_temperatures(pkg, kind, t):
    x, gen = logits(kind, 6, 3001, 11)
    c = Call(pkg, x, torch.randint(0, 3001, (6, 2), generator=gen), 9, t)
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [97, 5003, 140001])
def test_masks(pkg, kind, vocab):
    """Rows with few tokens left, with one, with none; masks of -infinity and of the type's lowest value; +infinity and NaN."""
    x, gen = logits(kind, 14, vocab, vocab)
    low = torch.finfo(x.dtype).min
    keep = torch.rand(14, vocab, generator=gen) < 3.0 / vocab
    for r, fill in ((0, -INF), (1, low), (2, -INF), (3, low)):
        x[r][~keep[r]] = fill
    x[4] = -INF
    x[5] = low
    x[6] = -INF
    x[6, vocab // 2] = -3.0
    x[7] = low
    x[7, vocab - 1] = low / 2
    x[8, vocab // 3] = INF
    x[9, vocab // 5] = NAN
    x[10] = NAN
    x[11] = -INF
    x[11, 1::2] = NAN
    x[12] = torch.finfo(x.dtype).max
    x[13, :vocab // 2] = low
    x[13, vocab // 2:] = torch.finfo(x.dtype).max
    c = Call(pkg, x, torch.randint(0, vocab, (14, 3), generator=gen), 40)
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("order", ["up", "down", "equal", "steps", "stripes", "zeros", "last"])
@pytest.mark.parametrize("vocab", [2000, 33333, 131072])
def test_orders_and_ties(pkg, kind, order, vocab):
    """Rows in which the largest come last, in which many are equal, or in which they stand where one thread finds them all."""
    i = torch.arange(vocab, dtype=torch.float64)
    x = {"up": i / vocab * 8, "down": -i / vocab * 8, "equal": i * 0 + 1.5, "steps": (i // 700) % 11, "stripes": ((i // 8) % 256 == 17) * 3.0 + (i % 97) / 97, "zeros": torch.where(i % 2 == 0, -0.0, 0.0),
         "last": torch.where(i >= vocab - 70, 4.0, 0.0)}[order]
    x = x[None].repeat(3, 1).to(so.TORCH[kind])
    x[1] = x[1].flip(0)
    c = Call(pkg, x, torch.tensor([[0, vocab - 1], [5, 6], [vocab // 2, 1]]), 64)
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_a_nearly_certain_token_keeps_its_digits(pkg, kind):
    x, gen = logits(kind, 8, 30000, 5, 1.0)
    for r in range(8):
        x[r, 1000 + r] = 14.0 + 4 * r
    tok = torch.arange(1000, 1008)[:, None]
    c = Call(pkg, x, tok, 2)
    pkg.logprobs(c.args)
    c.check()
    assert float(c.lp[7, 0]) < 0  # (exp(-42 + ...) beside 1)


def test_tokens_that_are_none(pkg):
    x, _ = logits("bf16", 5, 1000, 1)
    x[4] = -INF
    c = Call(pkg, x, torch.tensor([[-1, 0], [999, 1000], [-2 ** 31, 2 ** 31 - 1], [3, -7], [-1, 5]]), 1, entropy=False)
    pkg.logprobs(c.args)
    c.check()


def test_entropy_alone_and_no_rows(pkg):
    x, _ = logits("f16", 33, 6007, 2)
    c = Call(pkg, x)
    c.args.rows = 0
    pkg.logprobs(c.args)
    torch.cuda.synchronize()
    assert bool((c.ent == 55.0).all())
    c.args.rows = 33
    pkg.logprobs(c.args)
    c.check()


def test_the_same_call_gives_the_same_bits(pkg):
    x, gen = logits("bf16", 70, 60001, 3)
    tok = torch.randint(0, 60001, (70, 2), generator=gen)
    c = Call(pkg, x, tok, 20)
    seen = []
    for _ in range(4):
        pkg.logprobs(c.args)
        torch.cuda.synchronize()
        seen.append([v.clone() for v in (c.lp, c.ent, c.ids, c.tlp)])
    for other in seen[1:]:
        assert all(torch.equal(a, b) for a, b in zip(seen[0], other))


@pytest.mark.parametrize("rows,vocab", [(2, 90001), (40, 5000)])
def test_on_a_stream_and_in_a_graph(pkg, rows, vocab):
    x, gen = logits("f32", rows, vocab, 4)
    c = Call(pkg, x, torch.randint(0, vocab, (rows, 1), generator=gen), 12)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    pkg.logprobs(c.args, st.cuda_stream)
    st.synchronize()
    c.check("stream")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        pkg.logprobs(c.args, st.cuda_stream)
    for i in range(4):
        c.x, gen = logits("f32", rows, vocab, 50 + i)
        c.buf[:rows * vocab] = c.x.flatten().cuda()
        c.tokens = torch.randint(0, vocab, (rows, 1), generator=gen, dtype=torch.int32)
        c.dtok.copy_(c.tokens)
        torch.cuda.synchronize()
        g.replay()
        c.check(f"replay {i}")
        y, _ = logits("bf16", 3, 4001, 90 + i)
        other = Call(pkg, y, top=3)
        pkg.logprobs(other.args)
        other.check("between")


@pytest.mark.parametrize("kind,rows,vocab,given,top,pad,shift", [("bf16", 1, 1 << 22, 2, 64, 0, 0), ("f32", 2, (1 << 22) - 1, 1, 3, 1, 3), ("f16", 70, 131080, 1, 2, 1, 1), ("bf16", 64, 65536, 1, 64, 1, 7),
                                                                 ("f32", 65, 65537, 0, 5, 0, 2), ("bf16", 128, 40960, 1, 20, 0, 1), ("f16", 129, 40960, 1, 20, 0, 1), ("f32", 128, 40959, 1, 20, 2, 1),
                                                                 ("bf16", 140, 140000, 1, 0, 0, 3), ("f32", 9, 1048573, 1, 64, 1, 3), ("bf16", 63, 65535, 64, 0, 0, 0), ("f32", 70000, 3, 1, 2, 0, 1), ("f16", 4, 70001, 64, 64, 0, 5)])
def test_largest_rows_and_many(pkg, kind, rows, vocab, given, top, pad, shift):
    x, gen = logits(kind, rows, vocab, vocab)
    c = Call(pkg, x, torch.randint(0, vocab, (rows, given), generator=gen), top, pad=pad, shift=shift)
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_parts_of_which_some_hold_nothing(pkg, kind):
    """Rows cut into parts (few of a long vocabulary): masked but for one part, or one token, or with a NaN or an infinity in one part only."""
    x, gen = logits(kind, 7, 200003, 3)
    x[0, :150000] = -INF
    x[1, 5:] = -INF
    x[2] = -INF
    x[2, 123456] = 2.0
    x[3] = -INF
    x[4, 7] = NAN
    x[5, 200002] = INF
    x[6, 8192:] = torch.finfo(x.dtype).min
    c = Call(pkg, x, torch.randint(0, 200003, (7, 5), generator=gen), 64, 0.5)
    assert c.size > 0
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("rows,vocab", [(3, 100001), (300, 7001)])
def test_two_calls_at_once(pkg, rows, vocab):
    """On two streams, of the same logits, each with work of its own."""
    x, gen = logits("bf16", rows, vocab, 8)
    tok = torch.randint(0, vocab, (rows, 2), generator=gen)
    calls = [Call(pkg, x, tok, 20), Call(pkg, x, tok, 20, 0.7)]
    calls[1].args.logits = calls[0].args.logits
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(3):
        for c, s in zip(calls, streams):
            pkg.logprobs(c.args, s.cuda_stream)
    for c in calls:
        c.check()


def test_more_rows_than_workgroups(pkg):
    rows = (1 << 22) + 77
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(rows, 2, device="cuda", generator=gen) * 3
    tok = torch.randint(0, 2, (rows, 1), device="cuda", dtype=torch.int32, generator=gen)
    lp, ent, ids, tlp = torch.zeros(rows, 1, device="cuda"), torch.zeros(rows, device="cuda"), torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), torch.zeros(rows, 1, device="cuda")
    pkg.logprobs(pkg.LogProbs(logits=x.data_ptr(), stride=2, tokens=tok.data_ptr(), logProb=lp.data_ptr(), entropy=ent.data_ptr(), topIds=ids.data_ptr(), topLogProb=tlp.data_ptr(), rows=rows,
                              vocab=2, type=pkg.DTYPE_F32, given=1, top=1))
    torch.cuda.synchronize()
    d = (x[:, 1] - x[:, 0]).double()
    p = torch.stack([-torch.nn.functional.softplus(d, threshold=100), -torch.nn.functional.softplus(-d, threshold=100)], 1)
    close = lambda got, want: float(((got.double() - want).abs() / (1e-3 + want.abs())).max()) < 1e-6  # (the exponent and the exponential: a few 2^-24 of them)
    assert close(lp[:, 0], p.gather(1, tok.long())[:, 0]) and close(ent, -(p.exp() * p).sum(1))
    assert torch.equal(ids[:, 0], (x[:, 1] > x[:, 0]).int()) and close(tlp[:, 0], p.max(1).values)


@pytest.mark.parametrize("vocab,top", [(1000, 5), (140003, 20)])
def test_far_offsets(pkg, vocab, top):
    """Rows 2^25 + 1 elements apart: the last one behind 2^31 elements."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB")
    rows, stride = 70, (1 << 25) + 1
    x, gen = logits("bf16", rows, vocab, 77)
    c = Call(pkg, x, torch.randint(0, vocab, (rows, 2), generator=gen), top)
    buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda")
    buf.view(rows, stride)[:, :vocab] = x.cuda()
    c.args.logits, c.args.stride = buf.data_ptr(), stride
    pkg.logprobs(c.args)
    c.check()


@pytest.mark.parametrize("kind,rows,top", [("bf16", 129, 0), ("f32", 129, 0), ("f16", 129, 0), ("bf16", 1030, 1)])
def test_entropy_of_equal_logits_does_not_drift(pkg, kind, rows, top):
    """Rows of 2^22 tokens that one workgroup has alone: eight tokens at 0, of which each wave meets one at its start, every other one at a distance below them
    that differs from row to row (8 to 16; such sums are all rounded the same way).

    Bound, with p the share of the others and d their logarithm: an exponential is off by (3 |d| + 4) 2^-24 of itself (as in the oracle), a product with its exponent by 3 more, the sums of
    sixteen by 9, of eight of those (the entropy's) by 8, and what is joined behind them in pairs (the threads of a wave) by 6; the entropy's own rounding."""
    vocab = 1 << 22
    if torch.cuda.mem_get_info()[0] < 2 * rows * vocab * 4:
        pytest.skip("needs twice the logits' memory")
    d = -(128 + torch.arange(rows, dtype=torch.float64) % 129) / 16  # (exact in every type)
    x = d.to(so.TORCH[kind]).cuda()[:, None].repeat(1, vocab)
    x[:, :2048:256] = 0
    ent, ids, tlp = torch.full((rows,), 55.0, device="cuda"), torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), torch.zeros(rows, 1, device="cuda")
    a = pkg.LogProbs(logits=x.data_ptr(), stride=vocab, entropy=ent.data_ptr(), rows=rows, vocab=vocab, type=so.code_of(pkg, kind), top=top, topIds=ids.data_ptr(), topLogProb=tlp.data_ptr())
    size = pkg.logprobs_work_bytes(a)
    work = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
    a.work, a.workBytes = work.data_ptr(), size
    pkg.logprobs(a)
    torch.cuda.synchronize()
    others = (vocab - 8) * torch.exp(d)
    logz, p = torch.log(8 + others), others / (8 + others)
    want = logz - p * d
    dz = p * (3 * d.abs() + 4 + 9 + 6) * 2.0 ** -24
    bound = 2.0 ** -24 * want + dz * (1 + want) + p * d.abs() * (3 * d.abs() + 4 + 3 + 9 + 8 + 6) * 2.0 ** -24
    so.close(ent.cpu(), want, bound, "entropy")
    if top:
        assert not bool(ids.any())
        so.close(tlp[:, 0].cpu(), -logz, 2.0 ** -24 * logz + dz, "top")
