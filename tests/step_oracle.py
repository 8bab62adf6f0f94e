"""Plain 64-bit restatement (torch on the CPU) of the operators around the paged cache: rotary positions, matrices in 4 bits, log probabilities."""
import math

import torch

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
TINY = {"f32": 2.0 ** -149, "bf16": 2.0 ** -133, "f16": 2.0 ** -24}  # a step of the smallest numbers


def code_of(pkg, kind):
    return {"f32": pkg.DTYPE_F32, "bf16": pkg.DTYPE_BF16, "f16": pkg.DTYPE_F16}[kind]


def turned(x, pos, freq, rotated, halves, amplitude, kind):
    """x [rows, heads, hd] (64 bits) -> (turned rows, bound of the error).

    Bound: the output's rounding, the angle's (2^-50 of itself and of a turn: two products, the reduction, cosine and sine in 64 bits), and with rows of 16 bits the
    roundings to fp32 of cosine or sine (with the amplitude), of two products and of their sum, 4 * 2^-24 of |c a| + |s b|."""
    half = rotated // 2
    angle = pos.double()[:, None] * freq.double()
    c, s = (angle.cos() * amplitude)[:, None], (angle.sin() * amplitude)[:, None]
    i = torch.arange(half) if halves else 2 * torch.arange(half)
    j = i + half if halves else i + 1
    y, bound = x.clone(), torch.zeros_like(x)
    a, b = x[..., i], x[..., j]
    turn = (2.0 ** -50 * (angle.abs() + 8))[:, None] * amplitude * (a.abs() + b.abs())
    for at, u, v in ((i, c * a, -s * b), (j, s * a, c * b)):
        y[..., at] = u + v
        bound[..., at] = U[kind] * (u + v).abs() + turn + TINY[kind]
        if kind != "f32":
            bound[..., at] += 4 * 2.0 ** -24 * (u.abs() + v.abs())
    return y, bound


# ---- matrices in 4 bits ----------------------------------------------------------------------------------------------
def quantise4(x, group):
    """x [n, k] fp32 -> codes [n, k] (0..15), parameters [n, groups, 2] as halves."""
    n, k = x.shape
    groups = (k + group - 1) // group
    codes, params = torch.zeros(n, k, dtype=torch.int32), torch.zeros(n, groups, 2, dtype=torch.float16)
    for g in range(groups):
        at = slice(g * group, min(k, (g + 1) * group))
        y = x[:, at]
        low, high = y.amin(1, keepdim=True), y.amax(1, keepdim=True)
        base, scale = low.clamp(-65504, 65504).half(), ((high - low) * torch.tensor(1.0 / 15.0, dtype=torch.float32)).half()
        bad = ~torch.isfinite(y).all(1, keepdim=True) | torch.isinf(scale)
        step = scale.double()
        c = ((y.double() - base.double()) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
        codes[:, at] = torch.where((step > 0) & ~bad, c, torch.zeros_like(c)).to(torch.int32)
        params[:, g] = torch.cat([torch.where(bad, torch.full_like(base, math.nan), base), torch.where(bad, torch.zeros_like(scale), scale)], 1)
    return codes, params


def values4(codes, params, group):
    """[n, k] in 64 bits, unrounded."""
    p = params.double().repeat_interleave(group, 1)[:, :codes.shape[1]]
    return codes.double() * p[..., 1] + p[..., 0]


def packed4(codes):
    """Codes [n, k] -> bytes [n, k / 2], the even element in the low half."""
    return (codes[:, 0::2] | (codes[:, 1::2] << 4)).to(torch.uint8)


def product4(a, codes, params, group, kind, r=None, swiglu=False):
    """a [m, k] (64 bits) -> (C, bound of the error).

    Bound: codes are multiplied exactly as code + 16 (bf16, fp32) or code (fp16) and corrected with the group's sum of a, so that the fp32 sums run over terms of
    |a| (scale (code + 16) + |min - 16 scale|); k of them in any order cost, as independent roundings, (sqrt(k) + 16) * 2^-24 of their total.  Then the epilogue, a few
    fp32 roundings, and the output's."""
    w = values4(codes, params, group)
    shift = 0.0 if kind == "f16" else 16.0
    p = params.double().repeat_interleave(group, 1)[:, :codes.shape[1]]
    size = p[..., 1].abs() * (codes.double() + shift) + (p[..., 0] - shift * p[..., 1]).abs()
    y, e = a @ w.T, (a.abs() @ size.T) * (math.sqrt(a.shape[1]) + 16) * 2.0 ** -24
    if swiglu:
        g, u, eg, eu = y[:, 0::2], y[:, 1::2], e[:, 0::2], e[:, 1::2]
        sig = torch.sigmoid(g)
        y = sig * g * u
        e = 1.1 * eg * (u.abs() + eu) + (sig * g).abs() * eu + 8 * 2.0 ** -24 * y.abs() * (1 + g.abs() / 4)
    elif r is not None:
        y = y + r
        e = e + 2.0 ** -24 * y.abs()
    return y, e + U[kind] * (y.abs() + e) + TINY[kind]


# ---- log probabilities -----------------------------------------------------------------------------------------------
def top_of(x, k):
    """Ids of the k largest of a row, of equal ones the lower first; NaN as -infinity."""
    y = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
    return torch.sort(y, descending=True, stable=True).indices[:k]


def logprobs(x, tokens, top, t):
    """x [rows, vocab] -> ((log p of tokens, entropy, ids, log p of those), (bounds of the three)).

    Bound: an exponential in fp32 is off by its argument's roundings (three of 2^-24 of |d|) and its own (2^-23), so that the sum Z, whose largest term is an exact 1, is off by
    dz = sum of p (3 |d| + 4) 2^-24 over the others, of itself; results are rounded to fp32.  Z is a sum in 64 bits with that 1 in it: each of up to vocab / 256 + 256
    additions behind the 1 is off by 2^-53.  The entropy's sum of p |d| is fp32 in parts of the row, of up to vocab / 256 terms each."""
    x = x.double()
    rows, vocab = x.shape
    lp = torch.full((rows, tokens.shape[1]), math.nan, dtype=torch.float64)
    ent = torch.full((rows,), math.nan, dtype=torch.float64)
    ids = torch.zeros(rows, top, dtype=torch.int32)
    tlp = torch.full((rows, top), math.nan, dtype=torch.float64)
    blp, bent, btlp = torch.zeros_like(lp), torch.zeros_like(ent), torch.zeros_like(tlp)
    for r in range(rows):
        ids[r] = top_of(x[r], top).to(torch.int32)
        m = x[r].max()
        sound = bool(torch.isfinite(m))
        if sound:
            d = (x[r] - m) / t
            e = torch.exp(d)
            first = int(x[r].argmax())
            rest = e.clone()
            rest[first] = 0
            z1 = float(rest.sum())
            logz = math.log1p(z1)
            p = e / (1 + z1)
            pd = torch.where(p > 0, p * d, torch.zeros_like(p))
            dz = float((torch.where(p > 0, rest / (1 + z1) * (3 * d.abs() + 4), torch.zeros_like(p))).sum()) * 2.0 ** -24 + (vocab / 256 + 256) * 2.0 ** -53
            ent[r] = logz - float(pd.sum())
            bent[r] = 2.0 ** -24 * ent[r] + dz * (1 + ent[r]) + float(pd.abs().sum()) * (math.sqrt(vocab / 256) + 24) * 2.0 ** -24 + float((pd * d).abs().nansum()) * 2.0 ** -22 + 1e-37
            tlp[r] = d[ids[r].long()] - logz
            btlp[r] = 2.0 ** -24 * tlp[r].abs() + dz + 1e-37
        for j, tok in enumerate(tokens[r].tolist()):
            if tok < 0:
                lp[r, j] = 0
            elif tok < vocab and sound:
                lp[r, j] = d[tok] - logz
                blp[r, j] = 2.0 ** -24 * lp[r, j].abs() + dz + 1e-37
    lp, tlp = (torch.where(v < -torch.finfo(torch.float32).max, torch.full_like(v, -math.inf), v) for v in (lp, tlp))  # (results are fp32)
    return (lp, ent, ids, tlp), (blp, bent, btlp)


def close(got, want, bound, what):
    got, want = got.double(), want.double()
    both = torch.isnan(got) & torch.isnan(want) | (got == want)
    off = (got - want).abs()
    bad = ~(both | (off <= bound))
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()}, the first at {bad.nonzero()[0].tolist()}: got {got[bad][0]!r}, want {want[bad][0]!r}, bound {bound.expand_as(got)[bad][0]!r}"
