"""What is measured of the operators on a paged K/V cache: appending rows with their rotation (mlh_kv_append_device),
attention with a sliding window and first tokens that stay visible (mlh_attention_device), over pages of 32 or 16 bits
and over pages of 4.

A state is what a serving loop has in hand before a layer's call: the rows of the step's tokens, the pools, the page
table and lengths on the device, and the filled argument structures.  Tokens of sequence s are rows start[s] ..
start[s + 1] - 1, the last of them is position len[s] - 1.  Pages hold 64 positions; which page holds which positions
is dealt at random, as it is after a while of serving.  Sequences bring least_new to new rows each and hold least_held to
held positions before them.

  append   rows of q, k, v: q and k are rotated to their positions, k and v stored.  With 4-bit pages the pass also
           reads the stored rows back as the values they stand for (mlh_kv_read_device), as a caller does who moves a
           sequence to another cache.
  attend   the rows' queries over everything the sequences hold: single tokens, prompts, chunks behind a long context.
"""
import importlib.util
import math
import os
import sys

import torch

own = False

PAGE = 64
GROUP = 32  # elements that share a minimum and a scale in 4-bit pages
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# --------------------------------------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one sequence, heads of the benchmark's decoder, fp32 pages: nothing but latency
        {"name": "append-token", "op": "append", "type": "f32", "cache": "f32", "heads": 12, "kv": 12, "hd": 64,
         "nseq": 1, "new": 1, "least_new": 1, "held": 575, "least_held": 575},
        # a call of ragged prompts, grouped heads, 16-bit pages
        {"name": "append-prompts", "op": "append", "type": "bf16", "cache": "bf16", "heads": 32, "kv": 8, "hd": 128,
         "nseq": 23, "new": 1500, "least_new": 17, "held": 0, "least_held": 0},
        # the tokens of a step of many sequences into 4-bit pages
        {"name": "append4-step", "op": "append", "type": "bf16", "cache": "q4", "heads": 16, "kv": 16, "hd": 128,
         "nseq": 64, "new": 1, "least_new": 1, "held": 2047, "least_held": 40},
        # prompts into 4-bit pages
        {"name": "append4-prompts", "op": "append", "type": "f16", "cache": "q4", "heads": 32, "kv": 8, "hd": 128,
         "nseq": 5, "new": 4096, "least_new": 333, "held": 100, "least_held": 0},
        # one token of the benchmark's decoder over what its cache holds at most
        {"name": "token-f32", "op": "attend", "type": "f32", "cache": "f32", "heads": 12, "kv": 12, "hd": 64,
         "nseq": 1, "new": 1, "least_new": 1, "held": 575, "least_held": 575, "window": 256, "sinks": 4},
        # a step of 64 sequences of very different lengths, grouped heads, everything visible
        {"name": "step-bf16", "op": "attend", "type": "bf16", "cache": "bf16", "heads": 32, "kv": 8, "hd": 128,
         "nseq": 64, "new": 1, "least_new": 1, "held": 12000, "least_held": 100, "window": 0, "sinks": 0},
        # eight prompts of the large configuration's length, a window of half of it
        {"name": "prompts-bf16", "op": "attend", "type": "bf16", "cache": "bf16", "heads": 16, "kv": 16, "hd": 128,
         "nseq": 8, "new": 2048, "least_new": 2048, "held": 0, "least_held": 0, "window": 1024, "sinks": 4},
        # one long prompt: the largest call
        {"name": "long-prompt-f16", "op": "attend", "type": "f16", "cache": "f16", "heads": 32, "kv": 8, "hd": 128,
         "nseq": 1, "new": 16384, "least_new": 16384, "held": 0, "least_held": 0, "window": 4096, "sinks": 64},
        # a text of the reference's own shape, fp32
        {"name": "prompts-f32", "op": "attend", "type": "f32", "cache": "f32", "heads": 6, "kv": 6, "hd": 128,
         "nseq": 3, "new": 517, "least_new": 100, "held": 33, "least_held": 0, "window": 200, "sinks": 1},
        # one token behind a long context in 4 bits
        {"name": "token-long4", "op": "attend", "type": "bf16", "cache": "q4", "heads": 32, "kv": 8, "hd": 128,
         "nseq": 1, "new": 1, "least_new": 1, "held": 65000, "least_held": 65000, "window": 0, "sinks": 0},
        # a step of 48 sequences in 4 bits, a key head for each query head, a window
        {"name": "step4", "op": "attend", "type": "f16", "cache": "q4", "heads": 16, "kv": 16, "hd": 128,
         "nseq": 48, "new": 1, "least_new": 1, "held": 9000, "least_held": 50, "window": 4096, "sinks": 4},
        # a chunk of a prompt behind what is stored already in 4 bits
        {"name": "chunk4", "op": "attend", "type": "bf16", "cache": "q4", "heads": 32, "kv": 8, "hd": 64,
         "nseq": 2, "new": 777, "least_new": 512, "held": 7000, "least_held": 3000, "window": 0, "sinks": 0},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    cache = rng.choice(["f32", "bf16", "f16", "q4", "q4"])
    kind = cache if cache != "q4" else rng.choice(["f32", "bf16", "f16"])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 4, 6, 8, 12, 16])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 8] if kv <= 4 else [1, 1, 2, 3, 4] if kv <= 8 else [1, 2])
    case = {"op": "append" if rng.random() < 0.3 else "attend", "type": kind, "cache": cache, "heads": heads, "kv": kv, "hd": hd}
    shape = rng.choice(["step", "step", "prompts", "chunk"])
    if shape == "step":  # 1 to 64 single tokens, up to 200 000 positions in all
        nseq = _log(rng, 1, 64)
        longest = _log(rng, 2, min(50000, 400000 // nseq))
        case.update(nseq=nseq, new=1, least_new=1, held=longest, least_held=_log(rng, 1, longest) - 1)
    elif shape == "prompts":  # up to 8192 rows
        nseq = _log(rng, 1, 32)
        longest = _log(rng, 2, 4096 if nseq < 3 else 8192 // nseq)
        case.update(nseq=nseq, new=longest, least_new=_log(rng, 1, longest), held=0, least_held=0)
    else:  # up to 1024 rows behind up to 8000 positions each
        nseq = _log(rng, 1, 8)
        longest, held = _log(rng, 2, 1024 // nseq), _log(rng, 16, 8000)
        case.update(nseq=nseq, new=longest, least_new=_log(rng, 1, longest), held=held, least_held=_log(rng, 1, held))
    if case["op"] == "attend":
        case.update(window=rng.choice([0, _log(rng, 1, 4096), _log(rng, 64, 4096)]), sinks=rng.choice([0, 1, 4, 5, 64, 100]))
    return case


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, dealt in a scattered order."""
    if n == 1:
        return [hi]
    step = 7 if n % 7 else 5 if n % 5 else 3 if n % 3 else 1
    return [lo + (hi - lo) * ((i * step + 3) % n) // (n - 1) for i in range(n)]


def _shape(case):
    n = case["nseq"]
    new = _spread(case["least_new"], case["new"], n)
    held = _spread(case["least_held"], case["held"], n)[::-1]
    return new, [a + b for a, b in zip(new, held)]


# --------------------------------------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------------------------------------
def _page_bytes(case):
    """Bytes of one (page, head) tile of 4-bit pages: codes of 64 rows, then (minimum, scale) of every group of the rows."""
    return PAGE * case["hd"] // 2 + PAGE * (case["hd"] // GROUP) * 4


def _views4(pool, case):
    """Codes [pages, heads, 64, hd / 2] (low nibble: the even element) and parameters [pages, heads, 64, groups, 2] of a 4-bit pool."""
    hd, n = case["hd"], PAGE * case["hd"] // 2
    codes = pool[..., :n].unflatten(2, (PAGE, hd // 2))
    return codes, pool[..., n:].view(torch.float16).unflatten(2, (PAGE, hd // GROUP, 2))


def _quantise(x):
    """x [.., hd] in fp32 -> (codes [.., hd / 2] as bytes, parameters [.., groups, 2] as halves)."""
    g = x.unflatten(-1, (-1, GROUP))
    low, high = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    base, scale = low.half(), ((high - low) / 15.0).half()
    step = scale.double()
    codes = ((g.double() - base.double()) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
    codes = torch.where(step > 0, codes, torch.zeros_like(codes)).to(torch.uint8).flatten(-2)
    return codes[..., 0::2] | (codes[..., 1::2] << 4), torch.cat([base, scale], -1)


def _inputs(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 1009 + 11)
    new, length = _shape(case)
    H, K, hd, t = case["heads"], case["kv"], case["hd"], TYPES[case["type"]]
    rows, per = sum(new), max((n + PAGE - 1) // PAGE for n in length)
    used = [(n + PAGE - 1) // PAGE for n in length]
    pages = sum(used) + 3  # (a pool is never quite full)

    def normal(*shape):
        return torch.randn(*shape, device=dev, generator=gen)

    s = {"case": case, "start": torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device=dev),
         "len": torch.tensor(length, dtype=torch.int32, device=dev), "lengths": length, "new": new}
    order = torch.randperm(pages, device=dev, generator=gen).to(torch.int32)
    table = torch.zeros(len(new), per, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(used):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"], s["pages"] = table, pages
    s["q"] = (normal(rows, H, hd) * 1.5).to(t)
    if case["op"] == "append":
        s["k"], s["v"] = normal(rows, K, hd).to(t), normal(rows, K, hd).to(t)
        most = max(length)
        angle = torch.arange(most, device=dev, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, hd, 2, device=dev, dtype=torch.float64) / hd)
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).flatten(1).float().contiguous()
        s["qout"] = torch.zeros_like(s["q"])
    else:
        s["out"] = torch.zeros_like(s["q"])
    for name in ("pk", "pv"):
        if case["cache"] == "q4":
            pool = torch.zeros(pages, K, _page_bytes(case), dtype=torch.uint8, device=dev)
            if case["op"] == "attend":
                codes, params = _views4(pool, case)
                for p0 in range(0, pages, 256):
                    c, m = _quantise(normal(min(256, pages - p0), K, PAGE, hd))
                    codes[p0:p0 + 256], params[p0:p0 + 256] = c, m
        else:
            pool = torch.zeros(pages, PAGE, K, hd, dtype=TYPES[case["cache"]], device=dev)
            if case["op"] == "attend":
                for p0 in range(0, pages, 512):
                    pool[p0:p0 + 512] = normal(min(512, pages - p0), PAGE, K, hd).to(pool.dtype)
        s[name] = pool
    if case["op"] == "append" and case["cache"] == "q4":
        s["kback"], s["vback"] = (torch.zeros(rows, K, hd, dtype=torch.float32, device=dev) for _ in range(2))
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
    kinds = {"f32": m.DTYPE_F32, "bf16": m.DTYPE_BF16, "f16": m.DTYPE_F16, "q4": m.CACHE_Q4}
    H, K, hd = case["heads"], case["kv"], case["hd"]
    s["cache"] = m.KvCache(k=s["pk"].data_ptr(), v=s["pv"].data_ptr(), table=s["table"].data_ptr(), type=kinds[case["cache"]], heads=K, headDim=hd,
                           numPages=s["pages"], pagesPerSeq=s["table"].shape[1], nseq=case["nseq"])
    s["batch"] = m.KvBatch(start=s["start"].data_ptr(), len=s["len"].data_ptr(), rows=s["q"].shape[0], type=kinds[case["type"]], heads=H)
    if case["op"] == "append":
        s["args"] = m.KvAppend(q=s["q"].data_ptr(), qStride=H * hd, qOut=s["qout"].data_ptr(), qOutStride=H * hd, k=s["k"].data_ptr(), kStride=K * hd,
                               v=s["v"].data_ptr(), vStride=K * hd, rope=s["rope"].data_ptr(), ropeRows=s["rope"].shape[0])
        if case["cache"] == "q4":
            s["back"] = m.KvBatch(start=s["start"].data_ptr(), len=s["len"].data_ptr(), rows=s["q"].shape[0], type=m.DTYPE_F32, heads=K)
            s["read"] = m.KvRead(k=s["kback"].data_ptr(), v=s["vback"].data_ptr(), stride=K * hd)
    else:
        s["args"] = m.Attention(q=s["q"].data_ptr(), qStride=H * hd, out=s["out"].data_ptr(), outStride=H * hd, window=case["window"], sinks=case["sinks"],
                                maxLen=max(s["lengths"]), maxNew=max(s["new"]))
        n = m.attention_work_bytes(s["cache"], s["batch"], s["args"])
        s["work"] = torch.empty(max(n, 16), dtype=torch.uint8, device="cuda:0")
        s["args"].work, s["args"].workBytes = s["work"].data_ptr(), n
    return s


# --------------------------------------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------------------------------------
def _run_own(s):
    m, case, stream = _package(), s["case"], torch.cuda.current_stream().cuda_stream
    if case["op"] == "attend":
        m.attention(s["cache"], s["batch"], s["args"], stream)
        return s["out"]
    m.kv_append(s["cache"], s["batch"], s["args"], stream)
    if case["cache"] == "q4":
        m.kv_read(s["cache"], s["back"], s["read"], stream)
        return {"q": s["qout"], "k": s["kback"], "v": s["vback"]}
    return {"q": s["qout"], "k": s["pk"], "v": s["pv"]}


def _rotate(x, cs):
    """Adjacent pairs of x [rows, heads, hd] by the angles of cs [rows, hd] ((cos, sin) pairs); in 64 bits, rounded to fp32."""
    a, b = x.double().unflatten(-1, (-1, 2)).unbind(-1)
    c, s = cs.double().unflatten(-1, (-1, 2))[:, None].unbind(-1)
    return torch.stack([c * a - s * b, s * a + c * b], -1).flatten(-2).float()


def _plain_append(s):
    case, start, rows = s["case"], s["start"].long(), s["q"].shape[0]
    row = torch.arange(rows, device="cuda:0")
    seq = torch.bucketize(row, start[1:], right=True)
    pos = s["len"].long()[seq] - start[seq + 1] + row
    page, at = s["table"].long()[seq, pos // PAGE], pos % PAGE
    cs = s["rope"][pos]
    s["qout"].copy_(_rotate(s["q"], cs))
    out = {"q": s["qout"]}
    for name, x in (("k", _rotate(s["k"], cs)), ("v", s["v"].float())):
        if case["cache"] == "q4":
            codes, params = _views4(s["p" + name], case)
            c, m = _quantise(x)
            codes[page, :, at] = c
            params[page, :, at] = m
            out[name] = _dequantise(codes[page, :, at], params[page, :, at])
        else:
            s["p" + name][page, at] = x.to(s["p" + name].dtype)
            out[name] = s["p" + name]
    return out


def _dequantise(codes, params):
    """Codes [.., hd / 2], parameters [.., groups, 2] -> values [.., hd] in fp32 (minimum + code * scale, one rounding)."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, GROUP))
    return (c.double() * params[..., 1:].double() + params[..., :1].double()).float().flatten(-2)


def _held(s, name, i):
    """K or V of sequence i, [heads, len, hd] in fp32."""
    case, n = s["case"], s["lengths"][i]
    tiles = s["p" + name][s["table"][i, :(n + PAGE - 1) // PAGE].long()]
    if case["cache"] == "q4":
        x = _dequantise(*_views4(tiles, case)).transpose(1, 2)  # [pages, 64, heads, hd]
    else:
        x = tiles.float()
    return x.flatten(0, 1)[:n].transpose(0, 1).contiguous()


def _plain_attend(s):
    case, out = s["case"], s["out"]
    H, K, hd = case["heads"], case["kv"], case["hd"]
    at = 0
    for i, (new, n) in enumerate(zip(s["new"], s["lengths"])):
        k, v = _held(s, "k", i).transpose(1, 2).contiguous(), _held(s, "v", i)
        key = torch.arange(n, device="cuda:0")
        step = max(1, (1 << 28) // (H * n))
        for r0 in range(0, new, step):
            r1 = min(new, r0 + step)
            q = s["q"][at + r0:at + r1].float().unflatten(1, (K, H // K)).permute(1, 2, 0, 3).reshape(K, -1, hd)
            score = torch.matmul(q, k) * (1.0 / math.sqrt(hd))
            pos = torch.arange(n - new + r0, n - new + r1, device="cuda:0")[:, None]
            seen = key <= pos
            if case["window"]:
                seen &= (pos - key < case["window"]) | (key < case["sinks"])
            score = score.unflatten(1, (H // K, r1 - r0)).masked_fill(~seen, -math.inf).flatten(1, 2)
            p = torch.exp(score - score.amax(-1, keepdim=True))
            o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
            out[at + r0:at + r1] = o.unflatten(1, (H // K, r1 - r0)).permute(2, 0, 1, 3).reshape(r1 - r0, H, hd).to(out.dtype)
        at += new
    return out


def run(s):
    if own:
        return _run_own(s)
    return _plain_append(s) if s["case"]["op"] == "append" else _plain_attend(s)


# --------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------------------------------------
def _visible(pos, window, sinks):
    """Keys that position pos sees."""
    if not window or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    new, length = _shape(case)
    H, K, hd = case["heads"], case["kv"], case["hd"]
    e = 4 if case["type"] == "f32" else 2
    kept = hd * 5 / 8 if case["cache"] == "q4" else hd * (4 if case["cache"] == "f32" else 2)  # bytes of a head's row in the pool
    rows = sum(new)
    if case["op"] == "append":
        nbytes = rows * (2 * H + 2 * K) * hd * e + 2 * rows * K * kept + max(length) * hd * 4
        flops = rows * (H + K) * hd * 3.0
        if case["cache"] == "q4":
            nbytes += 2 * rows * K * (kept + 4 * hd)
            flops += 2 * rows * K * hd * 6.0
        return {"bytes": float(nbytes), "flops": float(flops)}
    nbytes, flops = 2.0 * rows * H * hd * e, 0.0
    for n, m in zip(new, length):
        first, w = m - n, case["window"]
        if not w or first < w:
            keys = m
        else:  # the window of the first new row and everything after it, and the first tokens
            keys = min(m, m - (first + 1 - w) + min(case["sinks"], first + 1 - w))
        nbytes += 2 * K * keys * kept
        flops += 4.0 * H * hd * sum(_visible(p, w, case["sinks"]) for p in range(first, m))
    return {"bytes": float(nbytes), "flops": float(flops)}


# --------------------------------------------------------------------------------------------------------------------
# the definition, in 64 bits
# --------------------------------------------------------------------------------------------------------------------
def _stored_values(x):
    """What 4-bit pages keep of x [rows, heads, hd] (fp64 holding fp32 values): per group of 32, minimum and scale as halves, 16 levels."""
    rows = x.reshape(-1, GROUP)
    low, high = rows.min(1).values, rows.max(1).values
    scale = ((high.float() - low.float()) / 15.0).half().double()
    low = low.half().double()
    best = torch.zeros_like(rows)
    for level in range(1, 16):  # the level's half-way border is passed (a value on it goes to the even level)
        border = low + (level - 0.5) * scale
        best += ((rows > border[:, None]) | ((rows == border[:, None]) & (level % 2 == 0))).double()
    return (low[:, None] + best * scale[:, None]).reshape(x.shape)


def _exact_append(s):
    case = s["case"]
    H, K, hd = case["heads"], case["kv"], case["hd"]
    places, owners = [], []
    for i, (new, n) in enumerate(zip(s["new"], s["lengths"])):
        places += range(n - new, n)
        owners += [i] * new
    pos = torch.tensor(places, device="cuda:0")
    turn = torch.view_as_complex(s["rope"].double()[pos].reshape(len(places), 1, hd // 2, 2).contiguous())

    def turned(x):
        return torch.view_as_real(torch.view_as_complex(x.double().reshape(len(places), -1, hd // 2, 2).contiguous()) * turn).reshape(x.shape)

    k, v = turned(s["k"]), s["v"].double()
    if case["cache"] == "q4":
        return {"q": turned(s["q"]), "k": _stored_values(k.float().double()), "v": _stored_values(v)}
    out = {"q": turned(s["q"])}
    slot = s["table"].long()[torch.tensor(owners, device="cuda:0"), pos // PAGE] * PAGE + pos % PAGE
    for name, x in (("k", k), ("v", v)):
        pool = torch.zeros(s["pages"] * PAGE, K, hd, dtype=torch.float64, device="cuda:0")
        pool.index_copy_(0, slot, x)
        out[name] = pool.reshape(s["pages"], PAGE, K, hd)
    return out


def _exact_values(s, name, i, head):
    """K or V of one head of sequence i, [len, hd] in 64 bits."""
    case, n, hd = s["case"], s["lengths"][i], s["case"]["hd"]
    pages = [int(p) for p in s["table"][i, :(n + PAGE - 1) // PAGE].tolist()]
    pool = s["p" + name][:, head] if case["cache"] == "q4" else s["p" + name][:, :, head]
    tiles = pool.index_select(0, torch.tensor(pages, device="cuda:0"))
    if case["cache"] != "q4":
        return tiles.reshape(-1, hd)[:n].double()
    byte = tiles[:, :PAGE * hd // 2].reshape(-1, hd // 2).to(torch.int32)
    level = torch.empty(byte.shape[0], hd, dtype=torch.float64, device="cuda:0")
    level[:, 0::2], level[:, 1::2] = byte % 16, byte // 16
    params = tiles[:, PAGE * hd // 2:].contiguous().view(torch.float16).double().reshape(-1, hd // GROUP, 2)
    return (params[:, :, 0].repeat_interleave(GROUP, 1) + level * params[:, :, 1].repeat_interleave(GROUP, 1))[:n]


def _exact_attend(s):
    case = s["case"]
    H, K, hd, w = case["heads"], case["kv"], case["hd"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda:0")
    at = 0
    for i, (new, n) in enumerate(zip(s["new"], s["lengths"])):
        for head in range(K):
            k, v = _exact_values(s, "k", i, head), _exact_values(s, "v", i, head)
            for r0 in range(0, new, 2048):
                r1 = min(new, r0 + 2048)
                lo, hi = n - new + r0, n - new + r1  # positions of these rows
                if w and lo >= w:  # only keys that one of them sees
                    first = max(lo + 1 - w, 0)
                    keep = torch.cat([torch.arange(min(case["sinks"], first)), torch.arange(first, hi)]).to("cuda:0")
                else:
                    keep = torch.arange(hi, device="cuda:0")
                back = torch.arange(lo, hi, device="cuda:0").unsqueeze(1) - keep
                hidden = back < 0
                if w:
                    hidden |= (back >= w) & (keep >= case["sinks"])
                for h in range(head * (H // K), (head + 1) * (H // K)):
                    a = s["q"][at + r0:at + r1, h].double() @ k[keep].T / hd ** 0.5
                    out[at + r0:at + r1, h] = torch.softmax(a.masked_fill(hidden, -math.inf), 1) @ v[keep]
        at += new
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attend(s)
