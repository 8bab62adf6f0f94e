"""What is measured of the operators that stand around the paged cache in a caller's own model loop: rotary positions
(mlh_rotate_device), products with 4-bit weights (mlh_gemm4_device), and log probabilities of given tokens with entropy and
top alternatives (mlh_logprobs_device).

A state is what such a loop has in hand before the call: the rows on the device, weights that were laid out once, and the
filled argument structures.

  rotate    q and k rows of a call turned to their positions, out of place: adjacent pairs or halves, the whole head or its
            first elements, frequencies as they are or blended for long contexts.
  gemm4     C = A . W^T for 1 to 64 rows of A, W of 4-bit codes with a minimum and a scale (halves) for every group of a
            row's elements; plain, with a residual, or with the gate / up epilogue (rows 2j and 2j + 1 of W are gate and up).
  logprobs  rows of logits: log probabilities of given tokens, entropy, the k most likely tokens with theirs.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of the benchmark's decoder: nothing but latency
        {"name": "rotate-token", "op": "rotate", "type": "f32", "rows": 1, "heads": 12, "kv": 12, "hd": 64, "rotated": 64, "half": False,
         "far": 576, "factor": 1.0},
        # a call of prompts, grouped heads, halves, frequencies blended for eight times the length
        {"name": "rotate-prompts", "op": "rotate", "type": "bf16", "rows": 16384, "heads": 32, "kv": 8, "hd": 128, "rotated": 128, "half": True,
         "far": 65536, "factor": 8.0},
        # a chunk far into a long text, a quarter of each head turned
        {"name": "rotate-part", "op": "rotate", "type": "f16", "rows": 2500, "heads": 16, "kv": 16, "hd": 128, "rotated": 32, "half": True,
         "far": 1000000, "factor": 1.0},
        # one token through a projection of the benchmark's decoder, fp32 activations
        {"name": "gemm4-token", "op": "gemm4", "type": "f32", "m": 1, "n": 768, "k": 768, "group": 32, "epi": "plain"},
        # one token through gate and up of the large configuration
        {"name": "gemm4-gate-up", "op": "gemm4", "type": "bf16", "m": 1, "n": 11264, "k": 2048, "group": 64, "epi": "swiglu"},
        # a step of 5 sequences through a large down projection onto the residual rows
        {"name": "gemm4-down", "op": "gemm4", "type": "f16", "m": 5, "n": 8192, "k": 28672, "group": 32, "epi": "residual"},
        # a step of 19 sequences, a vocabulary's rows: the LM head in 4 bits
        {"name": "gemm4-head", "op": "gemm4", "type": "bf16", "m": 19, "n": 32000, "k": 2048, "group": 128, "epi": "plain"},
        # a step of 64 sequences through gate and up of a large model
        {"name": "gemm4-step", "op": "gemm4", "type": "f16", "m": 64, "n": 28672, "k": 8192, "group": 64, "epi": "swiglu"},
        # one token of the benchmark's decoder
        {"name": "logprobs-token", "op": "logprobs", "type": "f32", "rows": 1, "vocab": 8192, "given": 1, "top": 5, "t": 1.0, "masked": 0.0},
        # a step of 64 sequences over a large odd vocabulary, at a temperature, most tokens masked in a quarter of the rows
        {"name": "logprobs-step", "op": "logprobs", "type": "bf16", "rows": 64, "vocab": 131075, "given": 1, "top": 20, "t": 0.7, "masked": 0.25},
        # a text of the reference's own shape, scored
        {"name": "logprobs-text", "op": "logprobs", "type": "f32", "rows": 517, "vocab": 20160, "given": 1, "top": 10, "t": 1.0, "masked": 0.0},
        # many prompts, four candidates at every place: the largest call
        {"name": "logprobs-prompts", "op": "logprobs", "type": "bf16", "rows": 8192, "vocab": 50257, "given": 4, "top": 1, "t": 1.0, "masked": 0.0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op, kind = rng.choice(["rotate", "gemm4", "gemm4", "logprobs", "logprobs"]), rng.choice(["f32", "bf16", "f16"])
    case = {"op": op, "type": kind}
    if op == "rotate":  # up to 16384 rows
        hd = rng.choice([64, 80, 96, 128, 256])
        kv = rng.choice([1, 2, 4, 8, 12])
        case.update(rows=_log(rng, 1, 16384 if kind != "f32" else 8192), heads=kv * rng.choice([1, 2, 3, 4]), kv=kv, hd=hd,
                    rotated=rng.choice([hd, hd, hd // 2, hd // 4]), half=rng.random() < 0.5, far=_log(rng, 64, 1000000),
                    factor=rng.choice([1.0, 1.0, 4.0, 8.0, 32.0]))
        case["heads"] = min(case["heads"], 32) if hd < 256 else kv
    elif op == "gemm4":  # up to 64 rows, up to 200 million weights
        k = 32 * _log(rng, 2, 512)
        n = _log(rng, 16, min(40000, 200000000 // k))
        epi = rng.choice(["plain", "plain", "residual", "swiglu"])
        case.update(m=rng.choice([1, 1, 2, _log(rng, 1, 64), _log(rng, 1, 64)]), n=n + n % 2 if epi == "swiglu" else n, k=k,
                    group=rng.choice([32, 64, 128]), epi=epi)
    else:  # up to 8192 rows, up to 200 000 tokens
        vocab = _log(rng, 500, 200000)
        rows = _log(rng, 1, min(8192, 150000000 // vocab))
        case.update(rows=rows, vocab=vocab, given=rng.choice([1, 1, 1, 3]), top=rng.choice([0, 1, 5, 20, 50]), t=rng.choice([1.0, 1.0, 0.6, 1.5]),
                    masked=rng.choice([0.0, 0.0, 0.3]))
    return case


# --------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------
def _frequencies(case):
    """Radians a position of every pair.  With a factor: wavelengths beyond a full turn in 8192 positions are stretched by it, those
    with more than four turns kept, the ones between blended by their number of turns."""
    r = case["rotated"]
    f = 10000.0 ** (-torch.arange(0, r, 2, dtype=torch.float64) / r)
    if case["factor"] != 1.0:
        keep = ((8192.0 * f / (2 * math.pi) - 1.0) / 3.0).clamp(0.0, 1.0)
        f = f * keep + f / case["factor"] * (1.0 - keep)
    return f


def _inputs(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 1013 + 17)
    t = TYPES[case["type"]]
    s = {"case": case}

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    if case["op"] == "rotate":
        rows = case["rows"]
        s["q"], s["k"] = ((normal(rows, h, case["hd"]) * 1.5).to(t) for h in (case["heads"], case["kv"]))
        s["qout"], s["kout"] = torch.zeros_like(s["q"]), torch.zeros_like(s["k"])
        last = torch.randint(case["far"] // 2, case["far"], (1,), device=dev, generator=gen)
        s["pos"] = (last - torch.arange(rows, device=dev)).remainder(case["far"]).to(torch.int32)  # a text that ends there
        s["freq"] = _frequencies(case).to(dev)
    elif case["op"] == "gemm4":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        groups = (k + g - 1) // g
        s["a"] = normal(m, k).to(t)
        s["codes"] = torch.randint(0, 256, (n, k // 2), device=dev, generator=gen, dtype=torch.uint8)  # (two codes; the low half is the even element)
        scale = (0.4 + 0.2 * torch.rand(n, groups, device=dev, generator=gen)) / math.sqrt(k) / 4.0
        low = -scale * (7.5 + 0.5 * normal(n, groups))
        s["params"] = torch.stack([low, scale], -1).half()
        cols = n // 2 if case["epi"] == "swiglu" else n
        if case["epi"] == "residual":
            s["r"] = normal(m, cols).to(t)
        s["c"] = torch.zeros(m, cols, dtype=t, device=dev)
    else:
        rows, v = case["rows"], case["vocab"]
        x = torch.empty(rows, v, dtype=t, device=dev)
        sharp = 0.7 + 2.3 * torch.rand(rows, 1, device=dev, generator=gen)
        for r0 in range(0, rows, 1024):
            x[r0:r0 + 1024] = (normal(min(1024, rows - r0), v) * sharp[r0:r0 + 1024]).to(t)
        s["tokens"] = torch.randint(0, v, (rows, case["given"]), device=dev, generator=gen, dtype=torch.int32)
        lead = 12.0 * torch.rand(rows, device=dev, generator=gen)  # the first given token is likely as a rule
        at = s["tokens"][:, 0].long()
        x[torch.arange(rows, device=dev), at] += lead.to(t)
        if case["masked"]:  # only some tokens may follow (the given ones among them): the others are -infinity or the type's lowest value
            some = torch.arange(0, rows, max(1, int(round(1.0 / case["masked"]))), device=dev)
            seen = torch.randperm(v, device=dev, generator=gen)[:max(64, v // 1000)]
            seen = torch.cat([(seen + some[:, None] * 7919) % v, s["tokens"][some].long()], 1)
            kept = x[some].gather(1, seen)
            low = torch.where(some % 2 == 0, -math.inf, torch.finfo(t).min).to(t)
            x[some] = low[:, None].expand(-1, v).scatter(1, seen, kept)
        s["logits"] = x
        s["lp"] = torch.zeros(rows, case["given"], device=dev)
        s["entropy"] = torch.zeros(rows, device=dev)
        s["ids"] = torch.zeros(rows, case["top"], dtype=torch.int32, device=dev)
        s["toplp"] = torch.zeros(rows, case["top"], device=dev)
    return s


def _package():
    name = "mini_llm_cuda_amd"
    if name not in sys.modules:
        pkg = os.path.join(os.getcwd(), "mini-llm-cuda_amd")
        spec = importlib.util.spec_from_file_location(name, os.path.join(pkg, "__init__.py"), submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[name] = mod
        try:
            spec.loader.exec_module(mod)
        except Exception:
            del sys.modules[name]
            raise
    return sys.modules[name]


def prepare(case, seed):
    s = _inputs(case, seed)
    if not own:
        return s
    m = _package()
    kind = {"f32": m.DTYPE_F32, "bf16": m.DTYPE_BF16, "f16": m.DTYPE_F16}[case["type"]]
    if case["op"] == "rotate":
        q, k = case["heads"] * case["hd"], case["kv"] * case["hd"]
        s["args"] = m.Rotate(q=s["q"].data_ptr(), qStride=q, qOut=s["qout"].data_ptr(), qOutStride=q, k=s["k"].data_ptr(), kStride=k,
                             kOut=s["kout"].data_ptr(), kOutStride=k, pos=s["pos"].data_ptr(), freq=s["freq"].data_ptr(), rows=case["rows"], type=kind,
                             heads=case["heads"], kvHeads=case["kv"], headDim=case["hd"], rotated=case["rotated"],
                             layout=m.ROTATE_HALVES if case["half"] else m.ROTATE_PAIRS)
    elif case["op"] == "gemm4":
        n, k, g = case["n"], case["k"], case["group"]
        s["packed"] = torch.empty(m.weights4_bytes(n, k, g), dtype=torch.uint8, device="cuda:0")
        s["w"] = m.Weights4(data=s["packed"].data_ptr(), N=n, K=k, group=g)
        m.weights4_set(s["w"], s["codes"].data_ptr(), s["params"].data_ptr(), torch.cuda.current_stream().cuda_stream)
        cols = s["c"].shape[1]
        s["args"] = m.Gemm4(a=s["a"].data_ptr(), aStride=k, c=s["c"].data_ptr(), cStride=cols, M=case["m"], type=kind, swiglu=int(case["epi"] == "swiglu"))
        if case["epi"] == "residual":
            s["args"].r, s["args"].rStride = s["r"].data_ptr(), cols
        size = m.gemm4_work_bytes(s["w"], s["args"])
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda:0")
        s["args"].work, s["args"].workBytes = s["work"].data_ptr(), size
    else:
        s["args"] = m.LogProbs(logits=s["logits"].data_ptr(), stride=case["vocab"], tokens=s["tokens"].data_ptr(), logProb=s["lp"].data_ptr(),
                               entropy=s["entropy"].data_ptr(), topIds=s["ids"].data_ptr() if case["top"] else None,
                               topLogProb=s["toplp"].data_ptr() if case["top"] else None, rows=case["rows"], vocab=case["vocab"], type=kind,
                               given=case["given"], top=case["top"], temperature=case["t"])
        size = m.logprobs_work_bytes(s["args"])
        s["work"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda:0")
        s["args"].work, s["args"].workBytes = s["work"].data_ptr(), size
    return s


# --------------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------------
def _outputs(s):
    op = s["case"]["op"]
    if op == "rotate":
        return {"q": s["qout"], "k": s["kout"]}
    if op == "gemm4":
        return s["c"]
    return {"logprob": s["lp"], "entropy": s["entropy"], "ids": s["ids"], "top": s["toplp"]}


def _run_own(s):
    m, stream = _package(), torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "rotate":
        m.rotate(s["args"], stream)
    elif op == "gemm4":
        m.gemm4(s["w"], s["args"], stream)
    else:
        m.logprobs(s["args"], stream)
    return _outputs(s)


def _plain_rotate(s):
    case = s["case"]
    r = case["rotated"]
    angle = s["pos"].double()[:, None] * s["freq"]  # (a far position's angle has no digits behind the point in 32 bits)
    c, sn = angle.cos()[:, None], angle.sin()[:, None]
    for name in ("q", "k"):
        x = s[name]
        turned = x[..., :r].double()
        a, b = (turned[..., :r // 2], turned[..., r // 2:]) if case["half"] else (turned[..., 0::2], turned[..., 1::2])
        u, v = c * a - sn * b, sn * a + c * b
        y = torch.cat([u, v], -1) if case["half"] else torch.stack([u, v], -1).flatten(-2)
        s[name + "out"].copy_(torch.cat([y.to(x.dtype), x[..., r:]], -1))


def _weights(s):
    """[n, k] in fp32."""
    k, g = s["case"]["k"], s["case"]["group"]
    codes = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).flatten(-2).float()
    low, scale = (p.float().repeat_interleave(g, 1)[:, :k] for p in s["params"].unbind(-1))
    return low + codes * scale


def _plain_gemm4(s):
    case = s["case"]
    y = torch.matmul(s["a"].float(), _weights(s).t())
    if case["epi"] == "swiglu":
        gate, up = y[:, 0::2], y[:, 1::2]
        y = gate / (1.0 + torch.exp(-gate)) * up
    elif case["epi"] == "residual":
        y = y + s["r"].float()
    s["c"].copy_(y.to(s["c"].dtype))


def _plain_logprobs(s):
    case = s["case"]
    step = max(1, (1 << 28) // case["vocab"])
    for r0 in range(0, case["rows"], step):
        r1 = min(case["rows"], r0 + step)
        x = s["logits"][r0:r1].float()
        best = x.amax(1, keepdim=True)
        d = (x - best) / case["t"]
        e = torch.exp(d)
        z = e.sum(1, keepdim=True)
        logz = z.log()
        s["entropy"][r0:r1] = (logz - (e * d.clamp_min(-1e30)).sum(1, keepdim=True) / z)[:, 0]  # (a masked token adds nothing)
        s["lp"][r0:r1] = d.gather(1, s["tokens"][r0:r1].long()) - logz
        if case["top"]:
            at = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]  # (of equal ones the lowest index)
            s["ids"][r0:r1] = at.to(torch.int32)
            s["toplp"][r0:r1] = d.gather(1, at) - logz


def run(s):
    if own:
        return _run_own(s)
    {"rotate": _plain_rotate, "gemm4": _plain_gemm4, "logprobs": _plain_logprobs}[s["case"]["op"]](s)
    return _outputs(s)


# --------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["type"] == "f32" else 2
    if case["op"] == "rotate":
        heads = case["rows"] * (case["heads"] + case["kv"])
        return {"bytes": float(2 * heads * case["hd"] * e + case["rows"] * 4 + case["rotated"] * 4), "flops": 3.0 * heads * case["rotated"]}
    if case["op"] == "gemm4":
        m, n, k = case["m"], case["n"], case["k"]
        cols = n // 2 if case["epi"] == "swiglu" else n
        nbytes = n * k // 2 + n * ((k + case["group"] - 1) // case["group"]) * 4 + m * k * e + m * cols * e * (2 if case["epi"] == "residual" else 1)
        return {"bytes": float(nbytes), "flops": 2.0 * m * n * k}
    rows = case["rows"]
    return {"bytes": float(rows * (case["vocab"] * e + case["given"] * 8 + 4 + case["top"] * 8)), "flops": 6.0 * rows * case["vocab"]}


# --------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# --------------------------------------------------------------------------------------------------------------------
def _exact_rotate(s):
    case, out = s["case"], {}
    r, hd = case["rotated"], case["hd"]
    order = list(range(0, r, 2)) + list(range(1, r, 2)) if not case["half"] else list(range(r))  # first elements of the pairs, then their second ones
    order = torch.tensor(order + list(range(r, hd)), device="cuda:0")
    back = torch.argsort(order)
    turn = torch.polar(torch.ones(case["rows"], r // 2, dtype=torch.float64, device="cuda:0"), s["pos"].double().unsqueeze(1) * s["freq"].unsqueeze(0))
    for name in ("q", "k"):
        x = s[name].double().index_select(2, order)
        z = torch.complex(x[:, :, :r // 2].contiguous(), x[:, :, r // 2:r].contiguous()) * turn.unsqueeze(1)
        out[name] = torch.cat([z.real, z.imag, x[:, :, r:]], 2).index_select(2, back)
    return out


def _exact_gemm4(s):
    case = s["case"]
    n, k, g = case["n"], case["k"], case["group"]
    a = s["a"].double()
    out = torch.zeros(case["m"], n, dtype=torch.float64, device="cuda:0")
    for n0 in range(0, n, 4096):
        byte = s["codes"][n0:n0 + 4096].to(torch.int32)
        level = torch.empty(byte.shape[0], k, dtype=torch.float64, device="cuda:0")
        level[:, 0::2], level[:, 1::2] = byte % 16, byte // 16
        for k0 in range(0, k, g):  # group by group
            p = s["params"][n0:n0 + 4096, k0 // g].double()
            level[:, k0:k0 + g] = level[:, k0:k0 + g] * p[:, 1:] + p[:, :1]
        out[:, n0:n0 + 4096] = a @ level.T
    if case["epi"] == "swiglu":
        pair = out.reshape(case["m"], n // 2, 2)
        return torch.sigmoid(pair[:, :, 0]) * pair[:, :, 0] * pair[:, :, 1]
    return out + s["r"].double() if case["epi"] == "residual" else out


def _exact_logprobs(s):
    case = s["case"]
    rows, k = case["rows"], case["top"]
    lp, ent = torch.zeros(rows, case["given"], dtype=torch.float64, device="cuda:0"), torch.zeros(rows, dtype=torch.float64, device="cuda:0")
    ids, top = torch.zeros(rows, k, dtype=torch.int32, device="cuda:0"), torch.zeros(rows, k, dtype=torch.float64, device="cuda:0")
    step = max(1, (1 << 27) // case["vocab"])
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        x = s["logits"][r0:r1].double()
        logp = torch.log_softmax(x / case["t"], 1)
        p = logp.exp()
        ent[r0:r1] = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
        lp[r0:r1] = logp.gather(1, s["tokens"][r0:r1].long())
        free = torch.ones_like(x, dtype=torch.bool)
        place = torch.arange(case["vocab"], device="cuda:0").expand_as(x)
        for j in range(k):  # the largest that is left; of equal ones the lowest index
            best = x.masked_fill(~free, -math.inf).amax(1, keepdim=True)
            at = place.masked_fill(~free | (x != best), case["vocab"]).amin(1, keepdim=True)
            ids[r0:r1, j], top[r0:r1, j] = at[:, 0].to(torch.int32), logp.gather(1, at)[:, 0]
            free.scatter_(1, at, False)
    return {"logprob": lp, "entropy": ent, "ids": ids, "top": top}


def exact(case, seed):
    s = _inputs(case, seed)
    return {"rotate": _exact_rotate, "gemm4": _exact_gemm4, "logprobs": _exact_logprobs}[case["op"]](s)
