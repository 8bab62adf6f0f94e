"""What the operators on a paged K/V cache refuse: with a message, before anything reaches the device.  (The pointers here are none.)"""
import pytest


def _cache(pkg, **kw):
    d = dict(k=1 << 20, v=1 << 21, table=1 << 22, type=pkg.DTYPE_BF16, heads=4, headDim=64, numPages=8, pagesPerSeq=2, nseq=3)
    d.update(kw)
    return pkg.KvCache(**d)


def _batch(pkg, **kw):
    d = dict(start=1 << 20, len=1 << 20, rows=5, type=pkg.DTYPE_BF16, heads=8)
    d.update(kw)
    return pkg.KvBatch(**d)


def _append(pkg, **kw):
    d = dict(q=1 << 20, qStride=512, qOut=1 << 23, qOutStride=512, k=1 << 24, kStride=256, v=1 << 25, vStride=256, rope=1 << 26, ropeRows=128)
    d.update(kw)
    return pkg.KvAppend(**d)


def _attention(pkg, **kw):
    d = dict(q=1 << 20, qStride=512, out=1 << 23, outStride=512)
    d.update(kw)
    return pkg.Attention(**d)


def _read(pkg, **kw):
    d = dict(k=1 << 24, v=1 << 25, stride=256)
    d.update(kw)
    return pkg.KvRead(**d)


COMMON_CACHE = [dict(k=None), dict(v=None), dict(table=None), dict(type=3), dict(type=9), dict(headDim=32), dict(headDim=96), dict(heads=0), dict(heads=5000), dict(numPages=0),
                dict(pagesPerSeq=0), dict(pagesPerSeq=(1 << 24) + 1), dict(nseq=0), dict(nseq=(1 << 20) + 1), dict(k=(1 << 20) + 8), dict(v=(1 << 20) + 2), dict(table=(1 << 20) + 2)]
COMMON_BATCH = [dict(start=None), dict(len=None), dict(rows=-1), dict(rows=(1 << 24) + 1), dict(type=5), dict(type=-1), dict(start=(1 << 20) + 1), dict(len=(1 << 20) + 2)]
HEADS = [dict(heads=6), dict(heads=2), dict(heads=0), dict(heads=4 * 33), dict(heads=-4)]


@pytest.mark.parametrize("kw", COMMON_CACHE)
def test_caches(pkg, kw):
    for call, args in ((pkg.kv_append, _append(pkg)), (pkg.attention, _attention(pkg)), (pkg.kv_read, _read(pkg))):
        with pytest.raises(pkg.MlhError, match="-1: ."):
            call(_cache(pkg, **kw), _batch(pkg), args)
    assert pkg.attention_work_bytes(_cache(pkg, **kw), _batch(pkg), _attention(pkg)) == 0


@pytest.mark.parametrize("kw", COMMON_BATCH)
def test_batches(pkg, kw):
    for call, args in ((pkg.kv_append, _append(pkg)), (pkg.attention, _attention(pkg)), (pkg.kv_read, _read(pkg))):
        with pytest.raises(pkg.MlhError, match="-1: ."):
            call(_cache(pkg), _batch(pkg, **kw), args)


@pytest.mark.parametrize("kw", HEADS)
def test_heads(pkg, kw):
    for call, args in ((pkg.kv_append, _append(pkg)), (pkg.attention, _attention(pkg))):
        with pytest.raises(pkg.MlhError, match="multiple"):
            call(_cache(pkg), _batch(pkg, **kw), args)


def test_types_must_match(pkg):
    for cache, rows in ((pkg.DTYPE_F32, pkg.DTYPE_BF16), (pkg.DTYPE_F16, pkg.DTYPE_BF16), (pkg.DTYPE_BF16, pkg.DTYPE_F32)):
        for call, args in ((pkg.kv_append, _append(pkg)), (pkg.attention, _attention(pkg))):
            with pytest.raises(pkg.MlhError, match="type of the cache"):
                call(_cache(pkg, type=cache), _batch(pkg, type=rows), args)


@pytest.mark.parametrize("kw,what", [(dict(q=None), "both"), (dict(qOut=None), "both"), (dict(k=None), "k"), (dict(v=None), "v"), (dict(k=(1 << 24) + 8), "k: rows"),
                                     (dict(qStride=504 + 4), "q: "), (dict(qStride=504), "q: "), (dict(qOutStride=500), "qOut"), (dict(kStride=248), "k: "), (dict(vStride=-256), "v: "),
                                     (dict(vStride=1 << 33), "v: "), (dict(rope=(1 << 20) + 4), "rope"), (dict(ropeRows=0), "ropeRows"), (dict(qGain=(1 << 20) + 2), "gains"),
                                     (dict(qOut=1 << 20, qOutStride=520), "in place"), (dict(q=None, qOut=None, qGain=1 << 20), "gain")])
def test_append(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.kv_append(_cache(pkg), _batch(pkg), _append(pkg, **kw))


@pytest.mark.parametrize("kw,what", [(dict(q=None), "q"), (dict(out=None), "out"), (dict(out=1 << 20), "not be q"), (dict(qStride=500), "q: "), (dict(outStride=8), "out: "),
                                     (dict(window=-1), "window"), (dict(sinks=-1), "window"), (dict(maxLen=-1), "window"), (dict(maxNew=-4), "window"), (dict(scale=-1.0), "scale"),
                                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q=(1 << 20) + 2), "q: ")])
def test_attention(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.attention(_cache(pkg), _batch(pkg), _attention(pkg, **kw))
    assert pkg.attention_work_bytes(_cache(pkg), _batch(pkg), _attention(pkg, **kw)) == 0


@pytest.mark.parametrize("kw,what", [(dict(k=None), "k"), (dict(v=None), "v"), (dict(stride=8), "stride"), (dict(stride=260), "aligned"), (dict(v=(1 << 20) + 4), "v: ")])
def test_read(pkg, kw, what):
    with pytest.raises(pkg.MlhError, match=what):
        pkg.kv_read(_cache(pkg), _batch(pkg), _read(pkg, **kw))


def test_null_structures(pkg):
    for args in ((None, _batch(pkg)), (_cache(pkg), None)):
        for fn, last in ((pkg.dev.mlh_kv_append_device, _append(pkg)), (pkg.dev.mlh_attention_device, _attention(pkg)), (pkg.dev.mlh_kv_read_device, _read(pkg))):
            assert fn(*args, last, None) == -1 and b"null" in pkg.dev.mlh_last_error(None)
    for fn in (pkg.dev.mlh_kv_append_device, pkg.dev.mlh_attention_device, pkg.dev.mlh_kv_read_device):
        assert fn(_cache(pkg), _batch(pkg), None, None) == -1 and b"null arguments" in pkg.dev.mlh_last_error(None)


def test_page_bytes(pkg):
    assert pkg.kv_page_bytes(pkg.DTYPE_F32, 12, 64) == 64 * 12 * 64 * 4
    assert pkg.kv_page_bytes(pkg.DTYPE_BF16, 8, 128) == pkg.kv_page_bytes(pkg.DTYPE_F16, 8, 128) == 64 * 8 * 128 * 2
    assert pkg.kv_page_bytes(pkg.CACHE_Q4, 8, 128) == 8 * 64 * 128 * 5 // 8
    for bad in ((3, 8, 128), (pkg.DTYPE_F32, 0, 128), (pkg.DTYPE_F32, 8, 96), (pkg.DTYPE_F32, 5000, 64)):
        assert pkg.kv_page_bytes(*bad) == 0
