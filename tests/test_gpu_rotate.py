"""mlh_rotate_device against its formula in 64 bits."""
import math
from decimal import Decimal, localcontext

import numpy as np
import pytest
import torch

import step_oracle as so

pytestmark = pytest.mark.gpu
NAN = math.nan


class Call:
    """Rows with a margin between and behind them (NaN where nothing may be written or read)."""

    def __init__(self, pkg, kind, rows, heads, kv, hd, rotated, halves, pos, freq, seed=0, amplitude=0.0, pad=0, inplace=False, spare=1):
        gen = torch.Generator().manual_seed(seed)
        self.pkg, self.kind, self.rows, self.heads, self.kv, self.hd, self.rotated, self.halves, self.amplitude = pkg, kind, rows, heads, kv, hd, rotated, halves, amplitude
        t = so.TORCH[kind]
        self.x, self.buf, self.out = {}, {}, {}
        for name, h in (("q", heads), ("k", kv)):
            if not h:
                continue
            self.x[name] = (torch.randn(rows, h, hd, generator=gen) * 1.5).to(t)
            b = torch.full((rows + spare, h * hd + pad), NAN, dtype=t)
            b[:rows, :h * hd] = self.x[name].flatten(1)
            self.buf[name] = b.cuda()
            self.out[name] = self.buf[name] if inplace else torch.full_like(self.buf[name], 77.0)
        self.pos, self.freq = torch.as_tensor(pos, dtype=torch.int32), torch.as_tensor(np.asarray(freq))
        self.dpos, self.dfreq = self.pos.cuda(), self.freq.cuda()
        args = dict(pos=self.dpos.data_ptr(), freq=self.dfreq.data_ptr(), rows=rows, type=so.code_of(pkg, kind), heads=heads, kvHeads=kv, headDim=hd, rotated=rotated,
                    layout=pkg.ROTATE_HALVES if halves else pkg.ROTATE_PAIRS, amplitude=amplitude)
        for name, o in (("q", "qOut"), ("k", "kOut")):
            if name in self.buf:
                args.update({name: self.buf[name].data_ptr(), name + "Stride": self.buf[name].shape[1], o: self.out[name].data_ptr(), name + "OutStride": self.out[name].shape[1]})
        self.args, self.inplace = pkg.Rotate(**args), inplace

    def check(self, what=""):
        torch.cuda.synchronize()
        for name, h in (("q", self.heads), ("k", self.kv)):
            if not h:
                continue
            want, bound = so.turned(self.x[name].double(), self.pos, self.freq, self.rotated, self.halves, self.amplitude or 1.0, self.kind)
            got = self.out[name].cpu()
            so.close(got[:self.rows, :h * self.hd].unflatten(1, (h, self.hd)), want, bound, f"{what} {name}")
            margin = torch.cat([got[self.rows:].flatten(), got[:self.rows, h * self.hd:].flatten()])
            assert bool((torch.isnan(margin) if self.inplace else margin == 77.0).all()), f"{what} {name}: written beyond the rows"


@pytest.mark.parametrize("halves", [False, True])
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,heads,kv,hd,rotated,pad", [(1, 12, 12, 64, 64, 0), (1, 1, 0, 8, 2, 0), (3, 5, 1, 80, 20, 8), (67, 4, 2, 96, 24, 0), (257, 8, 8, 128, 128, 64),
                                                          (33, 3, 3, 256, 128, 8), (130, 2, 1, 128, 32, 0), (19, 1, 1, 512, 512, 16), (9, 32, 4, 64, 62, 8), (5, 7, 7, 40, 16, 0)])
def test_against_the_formula(pkg, kind, rows, heads, kv, hd, rotated, pad, halves):
    gen = np.random.default_rng(rows * 131 + hd)
    pos = gen.integers(0, 5000, rows)
    c = Call(pkg, kind, rows, heads, kv, hd, rotated, halves, pos, pkg.rope_frequencies(rotated), seed=hd + rows, pad=pad)
    pkg.rotate(c.args)
    c.check()


@pytest.mark.parametrize("kind", ["f32", "f16"])
@pytest.mark.parametrize("halves", [False, True])
def test_far_and_negative_positions(pkg, kind, halves):
    pos = [0, 1, -1, 999999, -999999, 2 ** 31 - 1, -2 ** 31, 2 ** 24 + 1, 65535, -4097]
    c = Call(pkg, kind, len(pos), 3, 2, 128, 128, halves, pos, pkg.rope_frequencies(128, 500000.0), amplitude=1.25)
    pkg.rotate(c.args)
    c.check()


@pytest.mark.parametrize("rotated,hd", [(64, 64), (48, 128), (20, 80)])
def test_in_place_and_back(pkg, rotated, hd):
    """Rows turned where they stand, and back by the negative positions: what they were, but for the roundings of two calls."""
    pos = np.arange(40) * 37 - 300
    c = Call(pkg, "f32", 40, 6, 2, hd, rotated, True, pos, pkg.rope_frequencies(rotated), inplace=True, pad=4)
    pkg.rotate(c.args)
    c.check("there")
    c.dpos.neg_()
    pkg.rotate(c.args)
    torch.cuda.synchronize()
    for name, h in (("q", 6), ("k", 2)):
        got = c.out[name].cpu()[:40, :h * hd].unflatten(1, (h, hd)).double()
        x = c.x[name].double()
        size = x.abs().amax(-1, keepdim=True) * 2
        assert bool(((got - x).abs() <= 4 * 2.0 ** -24 * size).all())
        assert torch.equal(got[..., rotated:], x[..., rotated:])


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_what_is_no_number_stays_in_its_pair(pkg, kind):
    c = Call(pkg, kind, 6, 2, 1, 64, 32, True, [5] * 6, pkg.rope_frequencies(32))
    x = c.x["q"]
    x[0, 0, 3], x[1, 1, 17], x[2, 0, 40], x[3, 1, 63] = math.inf, NAN, math.inf, NAN
    c.buf["q"][:6, :128] = x.flatten(1).cuda()
    pkg.rotate(c.args)
    torch.cuda.synchronize()
    got = c.out["q"].cpu()[:6, :128].unflatten(1, (2, 64)).float()
    odd = ~torch.isfinite(got)
    want = torch.zeros_like(odd)
    for r, h, i in ((0, 0, 3), (0, 0, 19), (1, 1, 1), (1, 1, 17), (2, 0, 40), (3, 1, 63)):
        want[r, h, i] = True
    assert torch.equal(odd, want)
    assert float(got[2, 0, 40]) == math.inf


def test_no_rows_and_q_alone(pkg):
    c = Call(pkg, "bf16", 4, 2, 0, 64, 64, False, [1, 2, 3, 4], pkg.rope_frequencies(64))
    c.args.rows = 0
    pkg.rotate(c.args)
    torch.cuda.synchronize()
    assert bool((c.out["q"] == 77.0).all())
    c.args.rows = 4
    pkg.rotate(c.args)
    c.check()


def test_on_a_stream_and_in_a_graph(pkg):
    """Recorded once, replayed with other rows and positions, eager calls in between."""
    c = Call(pkg, "f16", 21, 4, 2, 128, 128, True, np.arange(21), pkg.rope_frequencies(128))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        pkg.rotate(c.args, st.cuda_stream)
    st.synchronize()
    c.check("stream")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        pkg.rotate(c.args, st.cuda_stream)
    for i in range(4):
        gen = torch.Generator().manual_seed(100 + i)
        c.pos = torch.randint(0, 100000, (21,), generator=gen, dtype=torch.int32)
        c.dpos.copy_(c.pos)
        for name, h in (("q", 4), ("k", 2)):
            c.x[name] = torch.randn(21, h, 128, generator=gen).half()
            c.buf[name][:21] = c.x[name].flatten(1).cuda()
            c.out[name].fill_(77.0)
        torch.cuda.synchronize()
        g.replay()
        c.check(f"replay {i}")
        other = Call(pkg, "f16", 3, 1, 1, 64, 64, False, [1, 2, 3], pkg.rope_frequencies(64), seed=i)
        pkg.rotate(other.args)
        other.check("between")


def test_more_rows_than_workgroups_and_far_offsets(pkg):
    """2^20 + 3 rows of which each fills a workgroup, 2^32 elements from the first to the last; two elements of 512 are turned."""
    rows, hd, stride = (1 << 20) + 3, 512, 4096
    free = torch.cuda.mem_get_info()[0]
    if free < 24 << 30:
        pytest.skip("needs 24 GiB")
    buf = torch.empty(rows * stride, dtype=torch.bfloat16, device="cuda").view(rows, stride)
    gen = torch.Generator(device="cuda").manual_seed(3)
    buf[:, :hd + 1] = torch.randn(rows, hd + 1, generator=gen, device="cuda").to(torch.bfloat16)
    out = torch.zeros(rows, hd, dtype=torch.bfloat16, device="cuda")
    pos = torch.randint(0, 1000, (rows,), generator=gen, device="cuda", dtype=torch.int32)
    freq = torch.tensor([0.37], dtype=torch.float64, device="cuda")
    pkg.rotate(pkg.Rotate(q=buf.data_ptr(), qStride=stride, qOut=out.data_ptr(), qOutStride=hd, pos=pos.data_ptr(), freq=freq.data_ptr(), rows=rows, type=pkg.DTYPE_BF16, heads=1,
                          headDim=hd, rotated=2, layout=pkg.ROTATE_PAIRS))
    torch.cuda.synchronize()
    assert torch.equal(out[:, 2:], buf[:, 2:hd])
    some = torch.cat([torch.arange(0, 3000), torch.arange(rows - 3000, rows), torch.arange(0, rows, 4001)])
    want, bound = so.turned(buf[some.cuda(), :hd].cpu().double()[:, None], pos[some.cuda()].cpu(), freq.cpu(), 2, False, 1.0, "bf16")
    so.close(out[some.cuda()].cpu()[:, None], want, bound, "rows far apart")
    angle = pos.double() * 0.37
    a, b = buf[:, 0].double(), buf[:, 1].double()
    assert float((out[:, 0].double() - (angle.cos() * a - angle.sin() * b)).abs().max()) < 2.0 ** -8 * float((a * a + b * b).sqrt().max()) + 1e-5


@pytest.mark.parametrize("fast", [1.0, 1e6])
def test_how_far_off_a_far_angle_is(pkg, fast):
    """Pairs (1, 0) become (cos, sin) of position times frequency as they stand, reduced with 60 digits; positions of 32 bits, frequencies up to `fast` times the usual ones.

    Bound: 2^-52 of the angle, the rounding to fp32, and 2^-51 for cosine and sine in 64 bits and the oracle's own."""
    pos = np.concatenate([[2 ** 31 - 1, -2 ** 31, 16777217, 1000003, -65537, 3], np.random.default_rng(5).integers(-2 ** 31, 2 ** 31, 1500)])
    freq = pkg.rope_frequencies(64) * fast
    c = Call(pkg, "f32", len(pos), 1, 0, 64, 64, True, pos, freq)
    row = torch.zeros(len(pos), 64)
    row[:, :32] = 1
    c.buf["q"][:len(pos), :64] = row.cuda()
    pkg.rotate(c.args)
    torch.cuda.synchronize()
    with localcontext() as digits:
        digits.prec = 60
        turn = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494459")
        angle = np.array([[float((Decimal(int(p)) * Decimal(float(f))).remainder_near(turn)) for f in freq] for p in pos])
    want = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1))
    size = torch.from_numpy(np.tile(np.abs(pos[:, None] * freq), 2))
    so.close(c.out["q"].cpu()[:len(pos), :64], want, 2.0 ** -52 * size + 2.0 ** -24 * want.abs() + 2.0 ** -51, "cosine and sine")
