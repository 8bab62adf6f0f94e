"""Plain 64-bit restatement (torch on the CPU) of the operators on a paged K/V cache, and a builder of their arguments."""
import math

import torch

PAGE, GROUP = 64, 32
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative


def codes_of(pkg):
    return {"f32": pkg.DTYPE_F32, "bf16": pkg.DTYPE_BF16, "f16": pkg.DTYPE_F16, "q4": pkg.CACHE_Q4}


def tile_bytes(hd):
    return PAGE * hd // 2 + PAGE * (hd // GROUP) * 4


def quantise(x):
    """x [.., hd] fp32 -> codes [.., hd] (0..15), parameters [.., groups, 2] as halves."""
    g = x.unflatten(-1, (-1, GROUP))
    bad = ~torch.isfinite(g).all(-1, keepdim=True)
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    base, scale = low.clamp(-65504, 65504).half(), ((high - low) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).half()
    bad |= torch.isinf(scale)
    step = scale.double()
    c = ((g.double() - base.double()) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
    c = torch.where((step > 0) & ~bad, c, torch.zeros_like(c))
    base = torch.where(bad, torch.full_like(base, math.nan), base)
    scale = torch.where(bad, torch.zeros_like(scale), scale)
    return c.flatten(-2).to(torch.int32), torch.cat([base, scale], -1)


def values(codes, params):
    """What codes [.., hd] and parameters [.., groups, 2] stand for, in 64 bits (rounded once to fp32, as defined)."""
    c = codes.double().unflatten(-1, (-1, GROUP))
    return (c * params[..., 1:].double() + params[..., :1].double()).float().double().flatten(-2)


class Pools:
    """Host copy of a cache's two pools and page table; device tensors on demand."""

    def __init__(self, pkg, cache, kv, hd, lens, seed, spare=2, fill=None):
        self.pkg, self.type, self.kv, self.hd, self.nseq = pkg, cache, kv, hd, len(lens)
        gen = torch.Generator().manual_seed(seed)
        used = [max(0, (n + PAGE - 1) // PAGE) for n in lens]
        self.pages, self.per = sum(used) + spare, max(max(used), 1)
        order = torch.randperm(self.pages, generator=gen).to(torch.int32)
        self.table = torch.full((self.nseq, self.per), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(used):
            self.table[i, :n] = order[at:at + n]
            at += n
        if cache == "q4":  # all ones: minima and scales are NaN where nothing is stored
            shape = (self.pages, kv, tile_bytes(hd))
            self.k, self.v = (torch.full(shape, 255, dtype=torch.uint8) for _ in range(2))
        else:
            shape = (self.pages, PAGE, kv, hd)
            self.k, self.v = (torch.full(shape, math.nan, dtype=TORCH[cache]) for _ in range(2))

    def put(self, which, seq, pos, rows):
        """Stores rows [n, kv, hd] (fp32) of sequence seq at positions pos .. pos + n - 1; returns what they stand for."""
        pool = self.k if which == "k" else self.v
        p = torch.arange(pos, pos + rows.shape[0])
        page, at = self.table[seq].long()[p // PAGE], p % PAGE
        if self.type != "q4":
            pool[page, at] = rows.to(pool.dtype)
            return rows.to(pool.dtype).double()
        c, m = quantise(rows)
        n = PAGE * self.hd // 2
        pool[..., :n].unflatten(2, (PAGE, self.hd // 2))[page, :, at] = (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8)
        pool[..., n:].view(torch.float16).unflatten(2, (PAGE, self.hd // GROUP, 2))[page, :, at] = m
        return values(c, m)

    def to_gpu(self):
        self.dk, self.dv, self.dtable = self.k.cuda(), self.v.cuda(), self.table.cuda()
        return self

    def struct(self):
        return self.pkg.KvCache(k=self.dk.data_ptr(), v=self.dv.data_ptr(), table=self.dtable.data_ptr(), type=codes_of(self.pkg)[self.type], heads=self.kv,
                                headDim=self.hd, numPages=self.pages, pagesPerSeq=self.per, nseq=self.nseq)


class Rows:
    """start and len of a call."""

    def __init__(self, pkg, kind, heads, new, lens, pad=0):
        self.pkg, self.kind, self.heads, self.new, self.lens = pkg, kind, heads, new, lens
        self.used = sum(new)
        self.rows = self.used + pad
        self.start = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
        self.len = torch.tensor(lens, dtype=torch.int32)

    def struct(self):
        self.dstart, self.dlen = self.start.cuda(), self.len.cuda()
        return self.pkg.KvBatch(start=self.dstart.data_ptr(), len=self.dlen.data_ptr(), rows=self.rows, type=codes_of(self.pkg)[self.kind], heads=self.heads)


def attend(q, k, v, first, window, sinks, scale, kind, four):
    """q [n, H, hd] at positions first .. first + n - 1 over k, v [len, K, hd] (64 bits).  Returns (out, bound of the error).

    Bound, per element: the output's rounding, u |o|, and sum_j p_j |v_j| e_j with e_j the relative error of weight and value j:
    the rounding of the weight to 16 bits and of 4-bit values to halves (u_p, u_v), and twice the absolute error of the score (the weight's
    own and its share of the sum): fp32 sums of hd products in any order, keys rounded to halves (4-bit pages), exp's argument reduction in
    fp32 and its result; and weights below the smallest half counting as 0."""
    n, H, hd = q.shape
    K = k.shape[1]
    out, bound = torch.zeros(n, H, hd, dtype=torch.float64), torch.zeros(n, H, hd, dtype=torch.float64)
    key = torch.arange(k.shape[0])
    pos = torch.arange(first, first + n)
    seen = key[None] <= pos[:, None]
    if window:
        seen &= (pos[:, None] - key[None] < window) | (key[None] < sinks)
    half = kind != "f32"
    u_p = 0.0 if not half else (U["f16"] if four else U[kind])
    u_v = U["f16"] if half and four else 0.0
    for h in range(H):
        kh, vh = k[:, h // (H // K)], v[:, h // (H // K)]
        for i in range(n):
            at = seen[i].nonzero().flatten()
            if at.numel() == 0:
                continue
            kk, vv = kh[at], vh[at]
            s = kk @ q[i, h] * scale
            size = kk.abs() @ q[i, h].abs() * scale
            ds = size * (hd + 4) * 2.0 ** -24 + s.abs().max() * 2.0 ** -22
            if half and four:
                ds = ds + size * U["f16"] + 2.0 ** -25 * q[i, h].abs().max() * kk.abs().sum(1) * scale
            p = torch.exp(s - s.max())
            l = p.sum()
            p = p / l
            out[i, h] = p @ vv
            e = u_p + u_v + 2 * (ds + (p * ds).sum()) + (at.numel() ** 0.5 + 16) * 2.0 ** -22
            bound[i, h] = (p * e) @ vv.abs() + U[kind] * out[i, h].abs() + (2.0 ** -24 if half else 0.0) / l * vv.abs().sum(0) + 1e-30
            if kind == "f16":
                bound[i, h] += 2.0 ** -25
    return out, bound
