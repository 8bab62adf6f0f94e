"""What rotary positions, matrices in 4 bits and log probabilities refuse: with a message, before anything reaches the device.  (The pointers here are none.)
And the frequencies of mll_rope_frequencies."""
import math

import numpy as np
import pytest

P = 1 << 20


def _rotate(pkg, **kw):
    d = dict(q=P, qStride=512, qOut=1 << 21, qOutStride=512, k=1 << 22, kStride=256, kOut=1 << 23, kOutStride=256, pos=P, freq=P, rows=5, type=pkg.DTYPE_BF16, heads=8, kvHeads=4, headDim=64,
             rotated=64)
    d.update(kw)
    return pkg.Rotate(**d)


@pytest.mark.parametrize("kw,what", [(dict(q=None), "q"), (dict(qOut=None), "qOut"), (dict(k=None), "both"), (dict(kOut=None), "both"), (dict(q=P + 8), "q: rows"), (dict(qStride=504), "q: "),
                                     (dict(qOutStride=516), "qOut"), (dict(kStride=248), "k: "), (dict(kOutStride=-256), "kOut"), (dict(kOutStride=1 << 33), "kOut"), (dict(pos=None), "null"),
                                     (dict(freq=None), "null"), (dict(pos=P + 2), "pos must"), (dict(freq=P + 4), "freq 8"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"),
                                     (dict(type=3), "type"), (dict(type=-1), "type"), (dict(heads=0), "heads"), (dict(kvHeads=0), "heads"), (dict(heads=5000), "heads"), (dict(headDim=4), "headDim"),
                                     (dict(headDim=60), "headDim"), (dict(headDim=520), "headDim"), (dict(rotated=63), "rotated"), (dict(rotated=0), "rotated"), (dict(rotated=66), "rotated"),
                                     (dict(layout=2), "layout"), (dict(layout=-1), "layout"), (dict(amplitude=-1.0), "amplitude"), (dict(amplitude=math.nan), "amplitude"),
                                     (dict(amplitude=math.inf), "amplitude"), (dict(qOut=P, qOutStride=520), "in place"), (dict(kOut=1 << 22, kOutStride=264), "in place")])
def test_rotate(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.rotate(_rotate(pkg, **kw))


def _weights(pkg, **kw):
    d = dict(data=P, N=48, K=256, group=64)
    d.update(kw)
    return pkg.Weights4(**d)


BAD_WEIGHTS = [dict(data=None), dict(data=P + 8), dict(N=0), dict(N=(1 << 20) + 1), dict(K=0), dict(K=48), dict(K=(1 << 17) + 32), dict(group=16), dict(group=0), dict(group=256), dict(K=-32)]


def _gemm4(pkg, **kw):
    d = dict(a=1 << 21, aStride=256, c=1 << 22, cStride=48, M=3, type=pkg.DTYPE_F16, work=1 << 24, workBytes=1 << 30)
    d.update(kw)
    return pkg.Gemm4(**d)


@pytest.mark.parametrize("kw", BAD_WEIGHTS)
def test_weights(pkg, kw):
    w = _weights(pkg, **kw)
    for call in (lambda: pkg.weights4_pack(w, pkg.DTYPE_F32, P, 256), lambda: pkg.weights4_set(w, P, P), lambda: pkg.weights4_read(w, pkg.DTYPE_F32, P, 256), lambda: pkg.gemm4(w, _gemm4(pkg))):
        with pytest.raises(pkg.MlhError, match="-1: ."):
            call()
    assert pkg.gemm4_work_bytes(w, _gemm4(pkg)) == 0
    if "data" not in kw:
        assert pkg.weights4_bytes(w.N, w.K, w.group) == 0


def test_weights_laid_out_and_read(pkg):
    w = _weights(pkg)
    for call in (lambda *a: pkg.weights4_pack(w, *a), lambda *a: pkg.weights4_read(w, *a)):
        for args, what in (((3, P, 256), "type"), ((pkg.DTYPE_F16, None, 256), "null"), ((pkg.DTYPE_F16, P + 8, 256), "aligned"), ((pkg.DTYPE_F32, P, 258), "aligned"), ((pkg.DTYPE_BF16, P, 248), "stride"),
                           ((pkg.DTYPE_BF16, P, 1 << 33), "stride")):
            with pytest.raises(pkg.MlhError, match=what):
                call(*args)
    for args, what in (((None, P), "null"), ((P, None), "null"), ((P + 8, P), "aligned"), ((P, P + 4), "aligned")):
        with pytest.raises(pkg.MlhError, match=what):
            pkg.weights4_set(w, *args)


def test_weights_bytes(pkg):
    assert pkg.weights4_bytes(16, 128, 32) == 16 * 128 * 5 // 8
    assert pkg.weights4_bytes(17, 160, 64) == 4 * 16 * 128 * 9 // 16  # (whole tiles of 16 x 128)
    assert pkg.weights4_bytes(1 << 20, 1 << 17, 128) == (1 << 37) * 17 // 32


@pytest.mark.parametrize("kw,what", [(dict(a=None), "a"), (dict(a=(1 << 21) + 2), "a: rows"), (dict(aStride=260), "a: "), (dict(aStride=248), "a: "), (dict(c=None), "c must"), (dict(c=(1 << 22) + 1), "aligned"),
                                     (dict(r=P + 1, rStride=48), "aligned"), (dict(cStride=47), "c: stride"), (dict(cStride=1 << 33), "c: stride"), (dict(r=P, rStride=40), "r: stride"),
                                     (dict(r=P, rStride=-48), "r: stride"), (dict(M=-1), "M must"), (dict(M=65), "M must"), (dict(type=5), "type"), (dict(swiglu=2), "swiglu"),
                                     (dict(swiglu=1, r=P, rStride=48), "swiglu"), (dict(r=1 << 22, rStride=56), "in place"), (dict(c=1 << 21, cStride=256), "not be a")])
def test_gemm4(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.gemm4(_weights(pkg), _gemm4(pkg, **kw))
    assert pkg.gemm4_work_bytes(_weights(pkg), _gemm4(pkg, **kw)) == 0


def test_gemm4_of_an_odd_number_of_gates_and_ups(pkg):
    with pytest.raises(pkg.MlhError, match="even"):
        pkg.gemm4(_weights(pkg, N=47), _gemm4(pkg, swiglu=1))


def _logprobs(pkg, **kw):
    d = dict(logits=P, stride=1000, tokens=1 << 21, logProb=1 << 22, entropy=1 << 23, topIds=1 << 24, topLogProb=1 << 25, rows=4, vocab=1000, type=pkg.DTYPE_BF16, given=2, top=5, work=1 << 26, workBytes=1 << 30)
    d.update(kw)
    return pkg.LogProbs(**d)


@pytest.mark.parametrize("kw,what", [(dict(logits=None), "null"), (dict(logits=P + 1), "aligned"), (dict(tokens=None), "null"), (dict(logProb=None), "null"), (dict(topIds=None), "null"),
                                     (dict(topLogProb=None), "null"), (dict(stride=999), "stride"), (dict(stride=1 << 33), "stride"), (dict(rows=-1), "rows"), (dict(rows=(1 << 24) + 1), "rows"),
                                     (dict(vocab=0), "vocab"), (dict(vocab=(1 << 22) + 1, stride=1 << 23), "vocab"), (dict(type=5), "type"), (dict(given=-1), "given"), (dict(given=65), "given"),
                                     (dict(top=-1), "top"), (dict(top=65), "top"), (dict(top=6, vocab=5), "top"), (dict(temperature=-1.0), "temperature"), (dict(temperature=1e-5), "temperature"),
                                     (dict(temperature=2e4), "temperature"), (dict(temperature=math.nan), "temperature"), (dict(tokens=P + 2), "4-byte"), (dict(logProb=P + 1), "4-byte"),
                                     (dict(entropy=P + 2), "4-byte"), (dict(topIds=P + 3), "4-byte"), (dict(topLogProb=P + 2), "4-byte")])
def test_logprobs(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.logprobs(_logprobs(pkg, **kw))
    assert pkg.logprobs_work_bytes(_logprobs(pkg, **kw)) == 0


@pytest.mark.parametrize("kw", [dict(work=None), dict(work=(1 << 26) + 8), dict(workBytes=0), dict(workBytes=-1)])
def test_logprobs_of_rows_in_parts_want_their_work(pkg, kw):
    long = dict(rows=2, vocab=200000, stride=200000)
    need = pkg.logprobs_work_bytes(_logprobs(pkg, **long))
    assert need > 0 and pkg.logprobs_work_bytes(_logprobs(pkg)) == 0
    if kw.get("workBytes") == -1:
        kw = dict(workBytes=need - 1)
    with pytest.raises(pkg.MlhError, match="work"):
        pkg.logprobs(_logprobs(pkg, **long, **kw))


@pytest.mark.parametrize("kw", [dict(), dict(rows=1, vocab=1 << 22, stride=1 << 22), dict(rows=500, vocab=150001, stride=150016), dict(top=0, given=0), dict(rows=300, vocab=5000, stride=5000)])
def test_the_work_of_logprobs_can_be_asked_before_there_are_pointers(pkg, kw):
    kw = {**dict(rows=2, vocab=200000, stride=200000), **kw}
    none = dict.fromkeys(("logits", "tokens", "logProb", "entropy", "topIds", "topLogProb", "work"))
    assert pkg.logprobs_work_bytes(_logprobs(pkg, **kw, **none)) == pkg.logprobs_work_bytes(_logprobs(pkg, **kw))
    assert (pkg.logprobs_work_bytes(_logprobs(pkg, **kw)) > 0) == (kw["vocab"] > 5000)


def test_null_structures(pkg):
    assert pkg.dev.mlh_rotate_device(None, None) == -1 and b"null" in pkg.dev.mlh_last_error(None)
    assert pkg.dev.mlh_logprobs_device(None, None) == -1 and b"null" in pkg.dev.mlh_last_error(None)
    assert pkg.dev.mlh_gemm4_device(None, _gemm4(pkg), None) == -1 and b"null" in pkg.dev.mlh_last_error(None)
    assert pkg.dev.mlh_gemm4_device(_weights(pkg), None, None) == -1 and b"null" in pkg.dev.mlh_last_error(None)
    assert pkg.dev.mlh_weights4_set_device(None, None, None, None) == -1
    assert pkg.dev.mlh_logprobs_work_bytes(None) == pkg.dev.mlh_gemm4_work_bytes(None, None) == 0


# ---- frequencies -------------------------------------------------------------------------------------------------------
def test_plain_frequencies_are_those_of_the_table(pkg):
    f = pkg.rope_frequencies(64)
    assert np.allclose(f, 10000.0 ** (-np.arange(0, 64, 2) / 64), rtol=1e-14, atol=0)
    tab = pkg.rope_table(40, 64)  # (float powf and cosf of up to 39 radians)
    angle = np.arange(40)[:, None] * f
    assert np.abs(tab[:, 0::2] - np.cos(angle)).max() < 1e-5 and np.abs(tab[:, 1::2] - np.sin(angle)).max() < 1e-5


def test_scaled_frequencies(pkg):
    f = pkg.rope_frequencies(128, 500000.0)
    assert np.allclose(pkg.rope_frequencies(128, 500000.0, pkg.ROPE_LINEAR, 4.0), f / 4, rtol=1e-15)
    g = pkg.rope_frequencies(128, 500000.0, pkg.ROPE_BASE, 8.0)
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 8, rel_tol=1e-12) and np.all(np.diff(g / f) < 0)
    b = pkg.rope_frequencies(128, 500000.0, pkg.ROPE_BLEND, 8.0, original=8192, low=1.0, high=4.0)
    turns = 8192 * f / (2 * np.pi)
    assert np.array_equal(b[turns >= 4], f[turns >= 4]) and np.allclose(b[turns <= 1], f[turns <= 1] / 8, rtol=1e-15)
    mid = (turns > 1) & (turns < 4)
    w = (turns[mid] - 1) / 3
    assert mid.any() and np.allclose(b[mid], f[mid] * w + f[mid] / 8 * (1 - w), rtol=1e-13)
    assert np.array_equal(pkg.rope_frequencies(128, 500000.0, pkg.ROPE_LINEAR, 1.0), f)


@pytest.mark.parametrize("kw", [dict(rotated=63), dict(rotated=0), dict(rotated=514), dict(base=1.0), dict(base=math.nan), dict(base=math.inf), dict(kind=4), dict(kind=-1), dict(kind=1, factor=0.5),
                                dict(kind=1, factor=math.nan), dict(kind=2, rotated=2, factor=2.0), dict(kind=3, factor=2.0, original=0), dict(kind=3, factor=2.0, original=8192, low=4.0, high=4.0),
                                dict(kind=3, factor=2.0, original=8192, low=-1.0), dict(kind=3, factor=2.0, original=math.inf), dict(kind=2, factor=1e300, base=1e300)])
def test_frequencies_that_are_none(pkg, kw):
    with pytest.raises(pkg.MlhError):
        pkg.rope_frequencies(**{"rotated": 64, **kw})
