"""A caller's own model step out of the operators: products with 4-bit weights, rotary positions, the paged cache, log probabilities; and mlh_score, a context's use of the last."""
import math

import numpy as np
import pytest
import torch

import kv_oracle as kv
import step_oracle as so
from test_gpu_weights4 import set_from

pytestmark = pytest.mark.gpu

DIM, HEADS, KV, HD, ROT, FFN, VOCAB, GROUP = 256, 4, 2, 64, 48, 416, 1000, 32
EPS = 1e-6


class Weights:
    """Matrices of one block and a head, and what they stand for."""

    def __init__(self, pkg, seed):
        self.keep, self.w, self.values = [], {}, {}
        for i, (name, n, k) in enumerate((("qkv", (HEADS + 2 * KV) * HD, DIM), ("out", DIM, HEADS * HD), ("up", 2 * FFN, DIM), ("down", DIM, FFN), ("head", VOCAB, DIM))):
            w, data, codes, params = set_from(pkg, n, k, GROUP, seed * 10 + i)
            self.keep.append(data)
            self.w[name], self.values[name] = w, so.values4(codes, params, GROUP)


def norm(x):
    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)


def reference(W, xs, starts, freq, shake=None):
    """Logits of every row of sequences that bring xs[step][s] rows at a time, in 64 bits; shake: relative noise on every intermediate result."""
    def r(v):
        return v if shake is None else v * (1 + 2.0 ** -20 * (2 * torch.rand(v.shape, generator=shake, dtype=torch.float64) - 1))

    held = [None] * len(starts)
    out = []
    for rows in xs:
        logits = []
        for s, x in enumerate(rows):
            x = x.double()
            n = x.shape[0]
            at = 0 if held[s] is None else held[s][0].shape[0]
            pos = torch.arange(at, at + n)
            p = r(r(norm(x)) @ W.values["qkv"].T)
            q, k, v = p[:, :HEADS * HD].reshape(n, HEADS, HD), p[:, HEADS * HD:(HEADS + KV) * HD].reshape(n, KV, HD), p[:, (HEADS + KV) * HD:].reshape(n, KV, HD)
            q, k = (r(so.turned(t, pos, freq, ROT, True, 1.0, "f32")[0]) for t in (q, k))
            held[s] = (k, v) if held[s] is None else (torch.cat([held[s][0], k]), torch.cat([held[s][1], v]))
            K, V = held[s]
            mix = torch.zeros(n, HEADS, HD, dtype=torch.float64)
            for h in range(HEADS):
                score = q[:, h] @ K[:, h // (HEADS // KV)].T / math.sqrt(HD)
                score = score.masked_fill(torch.arange(K.shape[0])[None] > pos[:, None], -math.inf)
                mix[:, h] = torch.softmax(r(score), 1) @ V[:, h // (HEADS // KV)]
            h1 = r(r(mix).flatten(1) @ W.values["out"].T + x)
            g = r(r(norm(h1)) @ W.values["up"].T)
            u = r(torch.sigmoid(g[:, 0::2]) * g[:, 0::2] * g[:, 1::2])
            h2 = r(u @ W.values["down"].T + h1)
            logits.append(r(r(norm(h2)) @ W.values["head"].T))
        out.append(torch.cat(logits))
    return out


@pytest.mark.parametrize("graph", [False, True])
def test_steps_of_two_sequences(pkg, graph):
    """A prompt each (3 and 7 rows), then single tokens: log probabilities and best tokens of every row, fp32 rows and pages.

    Bound: the reference again with every intermediate result off by up to 2^-20 of itself (16 roundings to fp32, more than any operator's sums here make of their largest terms),
    eight times; four times the largest change that this makes to a logit."""
    W = Weights(pkg, 1)
    gen = torch.Generator().manual_seed(3)
    steps = [(3, 7), (1, 1), (1, 1), (1, 1)]
    xs = [[torch.randn(n, DIM, generator=gen) for n in rows] for rows in steps]
    freq = torch.from_numpy(pkg.rope_frequencies(ROT, 10000.0, pkg.ROPE_BLEND, 4.0, original=64))
    want = reference(W, xs, (0, 0), freq)
    bound = max(max(float((a - b).abs().max()) for a, b in zip(want, reference(W, xs, (0, 0), freq, torch.Generator().manual_seed(50 + i)))) for i in range(8)) * 4

    most, f32 = 10, pkg.DTYPE_F32
    pools = kv.Pools(pkg, "f32", KV, HD, [64, 64], 5).to_gpu()
    cache = pools.struct()

    def buf(*shape):
        return torch.zeros(*shape, device="cuda")

    x, xn, qkv, mix, h1, u, h2, logits = buf(most, DIM), buf(most, DIM), buf(most, (HEADS + 2 * KV) * HD), buf(most, HEADS * HD), buf(most, DIM), buf(most, FFN), buf(most, DIM), buf(most, VOCAB)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    start, length, pos, tokens = ints(0, 0, 0), ints(0, 0), torch.zeros(most, dtype=torch.int32, device="cuda"), torch.zeros(most, 1, dtype=torch.int32, device="cuda")
    lp, ent, tid, tlp = buf(most, 1), buf(most), torch.zeros(most, 5, dtype=torch.int32, device="cuda"), buf(most, 5)
    dfreq = freq.cuda()
    width = (HEADS + 2 * KV) * HD

    def product(name, m, a, c, r=None, swiglu=0):
        args = pkg.Gemm4(a=a.data_ptr(), aStride=a.shape[1], c=c.data_ptr(), cStride=c.shape[1], M=m, type=f32, swiglu=swiglu)
        if r is not None:
            args.r, args.rStride = r.data_ptr(), r.shape[1]
        assert pkg.gemm4_work_bytes(W.w[name], args) == 0
        pkg.gemm4(W.w[name], args, torch.cuda.current_stream().cuda_stream)

    def run(m):
        st = torch.cuda.current_stream().cuda_stream
        batch = pkg.KvBatch(start=start.data_ptr(), len=length.data_ptr(), rows=m, type=f32, heads=HEADS)
        kb, vb = qkv.data_ptr() + HEADS * HD * 4, qkv.data_ptr() + (HEADS + KV) * HD * 4
        xn.copy_(norm(x))
        product("qkv", m, xn, qkv)
        pkg.rotate(pkg.Rotate(q=qkv.data_ptr(), qStride=width, qOut=qkv.data_ptr(), qOutStride=width, k=kb, kStride=width, kOut=kb, kOutStride=width, pos=pos.data_ptr(), freq=dfreq.data_ptr(),
                              rows=m, type=f32, heads=HEADS, kvHeads=KV, headDim=HD, rotated=ROT, layout=pkg.ROTATE_HALVES), st)
        pkg.kv_append(cache, batch, pkg.KvAppend(q=qkv.data_ptr(), qStride=width, qOut=qkv.data_ptr(), qOutStride=width, k=kb, kStride=width, v=vb, vStride=width), st)
        pkg.attention(cache, batch, pkg.Attention(q=qkv.data_ptr(), qStride=width, out=mix.data_ptr(), outStride=HEADS * HD, maxLen=64, maxNew=most, work=work.data_ptr(), workBytes=work.numel()), st)
        product("out", m, mix, h1, x)
        xn.copy_(norm(h1))
        product("up", m, xn, u, swiglu=1)
        product("down", m, u, h2, h1)
        xn.copy_(norm(h2))
        product("head", m, xn, logits)
        pkg.logprobs(pkg.LogProbs(logits=logits.data_ptr(), stride=VOCAB, tokens=tokens.data_ptr(), logProb=lp.data_ptr(), entropy=ent.data_ptr(), topIds=tid.data_ptr(), topLogProb=tlp.data_ptr(),
                                  rows=m, vocab=VOCAB, type=f32, given=1, top=5), st)

    probe = pkg.Attention(q=qkv.data_ptr(), qStride=width, out=mix.data_ptr(), outStride=HEADS * HD, maxLen=64, maxNew=most)
    work = torch.zeros(max(16, pkg.attention_work_bytes(cache, pkg.KvBatch(start=start.data_ptr(), len=length.data_ptr(), rows=most, type=f32, heads=HEADS), probe)), dtype=torch.uint8, device="cuda")
    captured = None
    done = [0, 0]
    for i, rows in enumerate(xs):
        m = sum(len(r) for r in rows)
        done = [d + len(r) for d, r in zip(done, rows)]
        x[:m] = torch.cat(rows).cuda()
        start.copy_(ints(0, len(rows[0]), m))
        length.copy_(ints(*done))
        pos[:m] = torch.cat([torch.arange(d - len(r), d) for d, r in zip(done, rows)]).to(torch.int32).cuda()
        tokens[:m, 0] = (torch.arange(m) * 37 % VOCAB).to(torch.int32).cuda()
        torch.cuda.synchronize()
        if graph and i > 0:
            if captured is None:
                captured = torch.cuda.CUDAGraph()
                with torch.cuda.graph(captured):
                    run(m)
            captured.replay()
        else:
            run(m)
        torch.cuda.synchronize()
        got = logits[:m].cpu().double()
        assert float((got - want[i]).abs().max()) <= bound, (i, float((got - want[i]).abs().max()), bound)
        (elp, eent, eids, etlp), (blp, bent, btlp) = so.logprobs(logits[:m].cpu(), tokens[:m].cpu(), 5, 1.0)
        so.close(lp[:m].cpu(), elp, blp, f"step {i} given")
        so.close(ent[:m].cpu(), eent, bent, f"step {i} entropy")
        assert torch.equal(tid[:m].cpu(), eids)
        (wlp, _, wids, _), _ = so.logprobs(want[i].float(), tokens[:m].cpu(), 1, 1.0)
        assert float((lp[:m].cpu().double() - wlp).abs().max()) <= 2 * bound + 2.0 ** -22 * 20  # (a logit's and log Z's share; fp32 results of up to 20)
        for row in range(m):
            best = float(want[i][row].max())
            assert float(want[i][row, int(tid[row, 0])]) >= best - 2 * bound


def test_held_rows_move_to_other_positions(pkg):
    """Keys read back, turned by the distance and stored elsewhere are the keys of the other positions, but for the roundings of two more operators."""
    gen = torch.Generator().manual_seed(9)
    n, shift = 20, -70
    k, v = (torch.randn(n, KV, HD, generator=gen) for _ in range(2))
    freq = torch.from_numpy(pkg.rope_frequencies(HD))
    dfreq = freq.cuda()
    pools = kv.Pools(pkg, "f32", KV, HD, [128, 128], 2).to_gpu()
    cache = pools.struct()
    ints = lambda *t: torch.tensor(t, dtype=torch.int32, device="cuda")
    here, there = torch.arange(100, 100 + n), torch.arange(30, 30 + n)

    def turn(src, dst, pos):
        p = pos.to(torch.int32).cuda()
        pkg.rotate(pkg.Rotate(q=src.data_ptr(), qStride=KV * HD, qOut=dst.data_ptr(), qOutStride=KV * HD, pos=p.data_ptr(), freq=dfreq.data_ptr(), rows=n, type=pkg.DTYPE_F32, heads=KV, headDim=HD,
                              rotated=HD, layout=pkg.ROTATE_PAIRS))
        return p

    def batch(seq, last):
        start, length = (ints(0, n, n), ints(last + 1, 0)) if seq == 0 else (ints(0, 0, n), ints(0, last + 1))
        return (start, length), pkg.KvBatch(start=start.data_ptr(), len=length.data_ptr(), rows=n, type=pkg.DTYPE_F32, heads=KV)

    dk, dv, rk, rv = k.flatten(1).cuda(), v.flatten(1).cuda(), torch.zeros(n, KV * HD, device="cuda"), torch.zeros(n, KV * HD, device="cuda")
    keep = [turn(dk, dk, here)]
    t0, b0 = batch(0, 100 + n - 1)
    pkg.kv_append(cache, b0, pkg.KvAppend(k=dk.data_ptr(), kStride=KV * HD, v=dv.data_ptr(), vStride=KV * HD))
    pkg.kv_read(cache, b0, pkg.KvRead(k=rk.data_ptr(), v=rv.data_ptr(), stride=KV * HD))
    keep.append(turn(rk, rk, torch.full((n,), shift)))
    t1, b1 = batch(1, 30 + n - 1)
    pkg.kv_append(cache, b1, pkg.KvAppend(k=rk.data_ptr(), kStride=KV * HD, v=rv.data_ptr(), vStride=KV * HD))
    rk.zero_()
    pkg.kv_read(cache, b1, pkg.KvRead(k=rk.data_ptr(), v=rv.data_ptr(), stride=KV * HD))
    torch.cuda.synchronize()
    want, bound = so.turned(k.double(), there, freq, HD, False, 1.0, "f32")
    # the first rounding moves a pair by up to 2^-24 of its two elements, which the second turn mixes
    pair = want.unflatten(-1, (-1, 2)).abs().sum(-1, keepdim=True).expand(-1, -1, -1, 2).flatten(-2)
    so.close(rk.cpu().unflatten(1, (KV, HD)), want, bound + 2.0 ** -23 * pair, "keys")
    assert torch.equal(rv.cpu(), v.flatten(1))


# ---- mlh_score -------------------------------------------------------------------------------------------------------
def device(pkg, hp, seed):
    model = pkg.Model.generate(hp, seed)
    model.randomize_gains(seed)
    d = pkg.Device(hp, 0)
    d.upload(model)
    return d


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("kind,n,top,t", [("f32", 1, 3, 0.0), ("f32", 2, 0, 0.0), ("f32", 70, 64, 0.0), ("f32", 131, 5, 0.8), ("bf16", 40, 10, 1.5), ("bf16", 9, 1, 0.0)])
def test_score_is_what_the_logits_say(pkg, kind, n, top, t, mode):
    hp = pkg.config(1, weightDtype=pkg.DTYPE_BF16 if kind == "bf16" else pkg.DTYPE_F32, maxSeqs=2)
    d = device(pkg, hp, 4)
    d.set_prefill_mode(mode)
    ids = pkg.random_tokens(2, 0, hp.vocabSize, n)
    logits, _, nll = d.forward_full(0, ids, want_probs=False)
    lp, ent, tid, tlp = d.score(1, ids, top, t)
    nxt = torch.from_numpy(np.append(ids[1:], -1).astype(np.int32))[:, None]
    (wlp, went, wids, wtlp), (blp, bent, btlp) = so.logprobs(torch.from_numpy(logits), nxt, top, np.float32(t).item() or 1.0)
    so.close(torch.from_numpy(lp)[:, None], wlp, blp, "given")
    so.close(torch.from_numpy(ent), went, bent, "entropy")
    assert np.array_equal(tid, wids.numpy())
    so.close(torch.from_numpy(tlp), wtlp, btlp, "top")
    assert d.seq_len(0) == d.seq_len(1) == n
    if n > 1 and t == 0.0 and lp[:-1].min() > math.log(1e-4):
        assert abs(-float(lp[:-1].astype(np.float64).mean()) - nll) <= 1e-5 * max(1.0, abs(nll))
    again = d.score(1, ids[:1], top, t) if n + 1 <= hp.maxL else None  # the sequence goes on
    assert again is None or (d.seq_len(1) == n + 1 and float(again[0][0]) == 0.0)
    d.close()


def test_score_continues_where_a_prompt_stopped(pkg):
    """A text scored in two calls gives the rows of the second half that it gives in one, as far as the kernels of either length agree (fp32: 1e-4)."""
    hp = pkg.config(1, maxSeqs=2)
    d = device(pkg, hp, 5)
    ids = pkg.random_tokens(3, 1, hp.vocabSize, 90)
    whole = d.score(0, ids, 4)
    d.prefill(1, ids[:37])
    rest = d.score(1, ids[37:], 4)
    assert np.abs(rest[0] - whole[0][37:]).max() <= 1e-4 and np.abs(rest[1] - whole[1][37:]).max() <= 1e-4
    d.close()


def test_score_refuses(pkg):
    hp = pkg.config(1)
    d = device(pkg, hp, 6)
    ids = pkg.random_tokens(1, 0, hp.vocabSize, 4)
    for args, what in (((0, ids, 65), "top"), ((0, ids, -1), "top"), ((0, ids, 0, -1.0), "temperature"), ((0, ids, 0, math.nan), "temperature"), ((0, ids, 0, 2e4), "temperature"), ((1, ids, 0), "sequence"),
                       ((0, ids[:0], 0), "empty"), ((0, np.full(4, hp.vocabSize), 0), "token id"), ((0, np.zeros(hp.maxL + 1), 0), "maxL")):
        with pytest.raises(pkg.MlhError, match=what):
            d.score(*args)
    assert pkg.dev.mlh_score(d._h, 0, ids.ctypes.data, 4, 2, 0.0, None, None, None, None) == -1
    assert pkg.dev.mlh_score(None, 0, ids.ctypes.data, 4, 0, 0.0, None, None, None, None) == -1
    assert pkg.dev.mlh_score(d._h, 0, ids.ctypes.data, 4, 0, 0.0, None, None, None, None) == 0 and d.seq_len(0) == 4
    d.close()


def test_score_refuses_a_vocabulary_that_is_too_large_before_anything_else(pkg):
    """Before the sequence is looked at, let alone appended to: also from a context that has no weights yet."""
    hp = pkg.config(1, vocabSize=(1 << 22) + 1, dim=64, attnHeads=1, ffnDim=64, transformers=1, maxL=32)
    d = pkg.Device(hp, 0)
    with pytest.raises(pkg.MlhError, match="2\\^22"):
        d.score(0, np.array([1, 2, 3], dtype=np.int32), 2)
    assert d.seq_len(0) == 0
    d.close()
