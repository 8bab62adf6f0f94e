"""Matrices in 4 bits and mlh_gemm4_device against their definitions in 64 bits."""
import math

import pytest
import torch

import step_oracle as so

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def matrix(pkg, n, k, group):
    """(mlh_weights4 structure, its memory with a margin behind it)."""
    size = pkg.weights4_bytes(n, k, group)
    data = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
    return pkg.Weights4(data=data.data_ptr(), N=n, K=k, group=group), data


def codes_and_params(n, k, group, seed):
    gen = torch.Generator().manual_seed(seed)
    groups = (k + group - 1) // group
    codes = torch.randint(0, 16, (n, k), generator=gen, dtype=torch.int32)
    scale = 0.02 * (0.2 + torch.rand(n, groups, generator=gen))
    low = -scale * (7.5 + torch.randn(n, groups, generator=gen))
    return codes, torch.stack([low, scale], -1).half()


def set_from(pkg, n, k, group, seed):
    w, data = matrix(pkg, n, k, group)
    codes, params = codes_and_params(n, k, group, seed)
    dc, dp = so.packed4(codes).cuda(), params.cuda()
    pkg.weights4_set(w, dc.data_ptr(), dp.data_ptr())
    torch.cuda.synchronize()
    assert bool((data[-64:] == 255).all())
    return w, data, codes, params


SIZES = [(1, 32, 32), (16, 128, 128), (5, 96, 64), (17, 160, 128), (33, 2048, 64), (100, 352, 32), (257, 736, 128)]


@pytest.mark.parametrize("n,k,group", SIZES)
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_codes_come_back_as_their_values(pkg, n, k, group, kind):
    w, data, codes, params = set_from(pkg, n, k, group, n + k)
    out = torch.full((n + 1, k + 8), 9.0, dtype=so.TORCH[kind], device="cuda")
    pkg.weights4_read(w, so.code_of(pkg, kind), out.data_ptr(), k + 8)
    torch.cuda.synchronize()
    want = so.values4(codes, params, group).float().to(so.TORCH[kind])
    assert torch.equal(out[:n, :k].cpu(), want)
    assert bool((out[n] == 9.0).all()) and bool((out[:, k:] == 9.0).all())


@pytest.mark.parametrize("n,k,group", SIZES)
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_quantising(pkg, n, k, group, kind):
    gen = torch.Generator().manual_seed(n * k)
    x = (torch.randn(n, k, generator=gen) * 0.05).to(so.TORCH[kind])
    x[0, :32] = 0.25  # a group (or part of one) without spread
    if n > 4:
        x[1, 3], x[2, k - 1], x[3, 0] = INF, NAN, -INF
        x[4] *= 2e5 if kind != "f16" else 1e3
    src = torch.full((n, k + 16), NAN, dtype=x.dtype)
    src[:, :k] = x
    src = src.cuda()
    w, data = matrix(pkg, n, k, group)
    pkg.weights4_pack(w, so.code_of(pkg, kind), src.data_ptr(), k + 16)
    out = torch.zeros(n, k, device="cuda")
    pkg.weights4_read(w, pkg.DTYPE_F32, out.data_ptr(), k)
    torch.cuda.synchronize()
    assert bool((data[-64:] == 255).all())
    codes, params = so.quantise4(x.float(), group)
    want = so.values4(codes, params, group).float()
    assert torch.equal(torch.nan_to_num(out.cpu(), 1e9), torch.nan_to_num(want, 1e9))


class Product:
    def __init__(self, pkg, kind, m, n, k, group, epi="plain", seed=0, pad=0, weights=None, scale=1.0):
        self.pkg, self.kind, self.m, self.n, self.k, self.group, self.epi = pkg, kind, m, n, k, group, epi
        self.w, self.data, self.codes, self.params = weights or set_from(pkg, n, k, group, seed + n * 3 + k)
        gen = torch.Generator().manual_seed(seed + m)
        t = so.TORCH[kind]
        self.cols = n // 2 if epi == "swiglu" else n
        self.a = (torch.randn(m, k, generator=gen) * scale).to(t)
        self.da = torch.full((m, k + pad), NAN, dtype=t)
        self.da[:, :k] = self.a
        self.da = self.da.cuda()
        self.r = torch.randn(1 if epi == "bias" else m, self.cols, generator=gen).to(t) if epi in ("residual", "bias", "inplace") else None
        self.c = torch.full((m + 1, self.cols + pad), 33.0, dtype=t, device="cuda")
        self.args = pkg.Gemm4(a=self.da.data_ptr(), aStride=k + pad, c=self.c.data_ptr(), cStride=self.cols + pad, M=m, type=so.code_of(pkg, kind), swiglu=int(epi == "swiglu"))
        if epi == "inplace":
            self.c[:m, :self.cols] = self.r.cuda()
            self.args.r, self.args.rStride = self.args.c, self.args.cStride
        elif self.r is not None:
            self.dr = self.r.cuda()
            self.args.r, self.args.rStride = self.dr.data_ptr(), 0 if epi == "bias" else self.cols
        self.size = pkg.gemm4_work_bytes(self.w, self.args)
        self.work = torch.full((max(self.size, 16) + 64,), 255, dtype=torch.uint8, device="cuda")
        self.args.work, self.args.workBytes = self.work.data_ptr(), self.size

    def run(self, stream=None):
        self.pkg.gemm4(self.w, self.args, stream)
        return self

    def check(self, what=""):
        torch.cuda.synchronize()
        want, bound = so.product4(self.a.double(), self.codes, self.params, self.group, self.kind, None if self.r is None else self.r.double(), self.epi == "swiglu")
        got = self.c.cpu()
        so.close(got[:self.m, :self.cols], want, bound, what)
        assert bool((got[self.m] == 33.0).all()) and bool((got[:, self.cols:] == 33.0).all()), f"{what}: written beyond the result"
        assert bool((self.work[max(self.size, 0):] == 255).all())
        return got[:self.m, :self.cols]


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (1, 768, 768), (1, 48, 4096), (2, 17, 96), (4, 64, 1024), (5, 100, 2080), (8, 40, 512), (9, 33, 256), (16, 130, 1184), (17, 64, 640),
                                   (31, 18, 1056), (33, 257, 384), (48, 16, 2048), (49, 50, 160), (64, 300, 1536)])
def test_products(pkg, kind, group, m, n, k):
    Product(pkg, kind, m, n, k, group, pad=8 if (m + n) % 2 else 0).run().check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("epi", ["residual", "bias", "inplace", "swiglu"])
@pytest.mark.parametrize("m,n,k,group", [(1, 2, 32, 32), (1, 1408, 256, 64), (3, 50, 2048, 128), (16, 34, 736, 32), (20, 514, 384, 64), (64, 96, 1024, 128), (40, 22, 416, 32)])
def test_epilogues(pkg, kind, epi, m, n, k, group):
    Product(pkg, kind, m, n, k, group, epi, pad=16).run().check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m,n,k,group", [(1, 40000, 64, 32), (1, 32, 131072, 128), (7, 4112, 14336, 64), (64, 9000, 512, 32), (3, 16, 65536, 32)])
def test_wide_and_long(pkg, kind, m, n, k, group):
    Product(pkg, kind, m, n, k, group).run().check()


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_a_single_one_gives_the_weights(pkg, kind):
    """Rows of A with one 1 in them: the values, rounded; every place of a tile is met."""
    w = set_from(pkg, 48, 256, 32, 9)
    values = so.values4(w[2], w[3], 32)
    for k0 in range(0, 256, 64):
        p = Product(pkg, kind, 64, 48, 256, 32, weights=w)
        p.a = torch.zeros(64, 256, dtype=so.TORCH[kind])
        p.a[torch.arange(64), k0 + torch.arange(64)] = 1
        p.da.copy_(p.a)
        got = p.run().check(f"columns {k0}").double()
        want = values[:, k0:k0 + 64].T
        assert bool(((got - want).abs() <= (so.U[kind] + 4 * 2.0 ** -24) * want.abs() + 2.0 ** -23).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
def test_large_and_small_activations(pkg, kind):
    for scale in ({"f32": (1e30, 1e-30), "bf16": (1e30, 1e-30), "f16": (8000.0, 1e-6)}[kind]):
        Product(pkg, kind, 6, 70, 640, 64, scale=scale).run().check(f"scale {scale}")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("m", [1, 3, 20, 64])
def test_a_row_is_the_same_in_every_call(pkg, kind, m):
    """Bit for bit: alone, among others, twice, and beside rows that are no numbers."""
    w = set_from(pkg, 200, 1056, 64, 5)
    p = Product(pkg, kind, m, 200, 1056, 64, weights=w).run()
    torch.cuda.synchronize()
    first = p.c[:m, :200].clone()
    p.run()
    torch.cuda.synchronize()
    assert torch.equal(p.c[:m, :200], first)
    if m > 1:
        p.da[0, 5], p.da[m - 1, 7] = INF, NAN
        p.run()
        torch.cuda.synchronize()
        assert torch.equal(p.c[1:m - 1, :200], first[1:-1])
        assert not bool(torch.isfinite(p.c[0, :200]).any()) and not bool(torch.isfinite(p.c[m - 1, :200]).any())


def test_groups_that_are_no_numbers_stay_in_their_row(pkg):
    codes, params = codes_and_params(64, 256, 64, 3)
    params[5, 2, 0] = NAN
    params[40, 0] = torch.tensor([NAN, 0.0])
    w, data = matrix(pkg, 64, 256, 64)
    dc, dp = so.packed4(codes).cuda(), params.cuda()
    pkg.weights4_set(w, dc.data_ptr(), dp.data_ptr())
    for kind in ("f32", "bf16", "f16"):
        p = Product(pkg, kind, 3, 64, 256, 64, weights=(w, data, codes, params)).run()
        got = p.check()
        assert torch.equal(torch.isnan(got).any(0).nonzero().flatten(), torch.tensor([5, 40]))


def test_no_rows(pkg):
    p = Product(pkg, "f16", 4, 32, 64, 32)
    p.args.M = 0
    p.run()
    torch.cuda.synchronize()
    assert bool((p.c == 33.0).all())


@pytest.mark.parametrize("m,kind", [(1, "bf16"), (24, "f16"), (3, "f32"), (50, "f32")])
def test_on_a_stream_and_in_a_graph(pkg, m, kind):
    p = Product(pkg, kind, m, 700, 1312, 32, "residual")
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    p.run(st.cuda_stream)
    st.synchronize()
    p.check("stream")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        p.run(st.cuda_stream)
    for i in range(4):
        p.a = torch.randn(m, 1312, generator=torch.Generator().manual_seed(70 + i)).to(so.TORCH[kind])
        p.da.copy_(p.a)
        p.c.fill_(33.0)
        torch.cuda.synchronize()
        g.replay()
        p.check(f"replay {i}")
        Product(pkg, "bf16", 2, 50, 96, 32, seed=i).run().check("between")


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,k,group", [(3001, 736, 128), (1030, 544, 32), (4500, 416, 64), (6201, 1056, 32), (8190, 160, 128), (8193, 736, 64), (16383, 1184, 128), (16400, 288, 32), (20481, 416, 64)])
def test_every_way_that_waves_are_dealt(pkg, kind, n, k, group):
    """Rows of A and bands of W on both sides of every bound that chooses a kernel or its shape."""
    weights = set_from(pkg, n, k, group, n)
    for m in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64):
        Product(pkg, kind, m, n, k, group, weights=weights, pad=8).run().check(f"M {m}")
    if n % 2 == 0:
        Product(pkg, kind, 64, n, k, group, "swiglu", weights=weights).run().check("swiglu")


def test_two_products_at_once(pkg):
    """On two streams, of the same matrix and of the same A."""
    weights = set_from(pkg, 5000, 2048, 64, 3)
    p = [Product(pkg, "bf16", m, 5000, 2048, 64, weights=weights, seed=7) for m in (33, 33, 2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in p]
    for _ in range(3):
        for x, s in zip(p, streams):
            x.run(s.cuda_stream)
    for x in p:
        x.check()
    assert torch.equal(p[0].c, p[1].c)


@pytest.mark.parametrize("n,k,group", [(4097, 1184, 32), (1 << 16, 96, 64), (50, 1 << 17, 128)])
def test_laid_out_and_read_at_large_sizes(pkg, n, k, group):
    w, data, codes, params = set_from(pkg, n, k, group, 5)
    out = torch.full((n + 1, k), 9.0, device="cuda")
    pkg.weights4_read(w, pkg.DTYPE_F32, out.data_ptr(), k)
    want = so.values4(codes, params, group).float()
    assert torch.equal(out[:n].cpu(), want) and bool((out[n] == 9.0).all())
    again, other = matrix(pkg, n, k, group)
    pkg.weights4_pack(again, pkg.DTYPE_F32, out.data_ptr(), k)
    c2, p2 = so.quantise4(want, group)
    pkg.weights4_read(again, pkg.DTYPE_F32, out.data_ptr(), k)
    torch.cuda.synchronize()
    assert torch.equal(out[:n].cpu(), so.values4(c2, p2, group).float()) and bool((other[-64:] == 255).all())


def test_a_matrix_beyond_32_bit_offsets(pkg):
    """3.6 GB of codes: laid out, multiplied, read back; rows from all over it against the definition."""
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GiB")
    n, k, group, m = 110000, 1 << 16, 128, 3
    gen = torch.Generator(device="cuda").manual_seed(5)
    codes = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device="cuda", generator=gen)
    params = (torch.rand(n, k // group, 2, device="cuda", generator=gen) * 0.02 - 0.01).half()
    params[..., 1] = params[..., 1].abs()
    w, data = matrix(pkg, n, k, group)
    assert pkg.weights4_bytes(n, k, group) > 1 << 31
    pkg.weights4_set(w, codes.data_ptr(), params.data_ptr())
    some = torch.cat([torch.arange(0, 40), torch.arange(60000, 60020), torch.arange(n - 40, n)])
    packed = codes[some.cuda()].cpu().to(torch.int32)
    c = torch.stack([packed & 15, packed >> 4], -1).flatten(1)
    p = params[some.cuda()].cpu()
    for kind, rows in (("bf16", m), ("f16", 20), ("f32", 5)):
        t = so.TORCH[kind]
        a = torch.randn(rows, k, device="cuda", generator=gen).to(t)
        out = torch.zeros(rows, n, dtype=t, device="cuda")
        pkg.gemm4(w, pkg.Gemm4(a=a.data_ptr(), aStride=k, c=out.data_ptr(), cStride=n, M=rows, type=so.code_of(pkg, kind)))
        torch.cuda.synchronize()
        want, bound = so.product4(a.cpu().double(), c, p, group, kind)
        so.close(out[:, some.cuda()].cpu(), want, bound, kind)
    assert bool((data[-64:] == 255).all())


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("low", [0.0, 0.001, -7.5])
def test_how_far_off_a_single_product_is(pkg, kind, group, low):
    """Rows of A with one element in them, groups of scale 8 whose minimum is tiny beside it (or, -7.5 scales, an ordinary one): every kernel.

    Bound, in |a| 2^-24.  fp16: roundings of scale * code, of the minimum's product and of their sum, 3 (|min| + 15 scale).  bf16 and fp32 rows: the minimum - 16 scale is rounded to fp32, and so
    may be its product with a, each half a step of up to |min| + 16 scale; fp32 rows: the sum of a's planes by 16 + code and its product with the scale are rounded too, each by up to 31 scale.
    Then the result's own, in fp32 and in the type."""
    n, k, scale = 70, 384, 8.0
    codes, params = codes_and_params(n, k, group, 11)
    params[..., 0] = low * (scale if low < 0 else 1)
    params[..., 1] = scale
    w, data = matrix(pkg, n, k, group)
    dc, dp = so.packed4(codes).cuda(), params.cuda()
    pkg.weights4_set(w, dc.data_ptr(), dp.data_ptr())
    values = so.values4(codes, params, group)
    size = float(params[0, 0, 0].abs())
    roundings = {"f16": 3 * (size + 15 * scale), "bf16": 2 * (size + 16 * scale), "f32": 2 * (size + 16 * scale) + 2 * 31 * scale}[kind]
    for m in (1, 4, 8, 16, 32, 64):
        p = Product(pkg, kind, m, n, k, group, weights=(w, data, codes, params), seed=m)
        at, x = torch.arange(m) * 55 % k, p.a[:, 0].clone()
        p.a = torch.zeros(m, k, dtype=so.TORCH[kind])
        p.a[torch.arange(m), at] = x
        p.da.copy_(p.a)
        p.run()
        torch.cuda.synchronize()
        x = x.double()[:, None]
        want = x * values[:, at].T
        bound = x.abs() * roundings * 2.0 ** -24 + (2.0 ** -24 + so.U[kind]) * want.abs()
        so.close(p.c[:m, :n].cpu(), want, bound * (1 + so.U[kind]) + so.TINY[kind], f"M {m}")


@pytest.mark.parametrize("exponent", [-96, -109, -116, -126, -140])
def test_how_small_fp32_elements_may_be(pkg, exponent):
    """Elements of all 24 bits: three planes hold them down to 2^-110, below that what is left of them is off by half of a step of the smallest bf16, 2^-134, times 16 + code."""
    n, k, group = 70, 256, 64
    codes, params = codes_and_params(n, k, group, 12)
    params[..., 0], params[..., 1] = -7.5 * 1024, 1024
    w, data = matrix(pkg, n, k, group)
    dc, dp = so.packed4(codes).cuda(), params.cuda()
    pkg.weights4_set(w, dc.data_ptr(), dp.data_ptr())
    values = so.values4(codes, params, group)
    for m in (1, 8, 16, 64):
        p = Product(pkg, "f32", m, n, k, group, weights=(w, data, codes, params), seed=m)
        p.a = torch.ldexp(1 + p.a.abs().remainder(1), torch.tensor(exponent))
        p.da.copy_(p.a)
        p.run()
        torch.cuda.synchronize()
        want, bound = so.product4(p.a.double(), codes, params, group, "f32")
        so.close(p.c[:m, :n].cpu(), want, bound + (2.0 ** -134 * 31 * 1024 * k if exponent < -110 else 0), f"M {m}")
