"""Calls around the operators on a paged K/V cache: an earlier error of the program, what a context keeps, contexts of many sequences."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_cache import Append, Call, _same_bits, _stream
from test_gpu_cache_context import _hp, _model, rel
from kv_oracle import TORCH

pytestmark = pytest.mark.gpu


def _runtime():
    """The HIP runtime that is there already."""
    paths = {line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64.so" in line}
    assert len(paths) == 1, paths
    return ctypes.CDLL(paths.pop())


def test_errors_of_earlier_calls(pkg):
    """A call whose launches go well succeeds, whatever an earlier call of the program left behind."""
    a = Append(pkg, "bf16", "bf16", 4, 2, 64, [3], [70])
    c = Call(pkg, "bf16", "bf16", 2, 1, 64, [1], [9000], seed=1)  # (two launches)
    back = torch.zeros(2, 3, 128, dtype=TORCH["bf16"], device="cuda")
    want = c.run().clone()
    c.out.fill_(3.0)
    torch.cuda.synchronize()
    hip = _runtime()
    for call in (lambda: pkg.kv_append(a.cache, a.batch, a.args, _stream()),
                 lambda: pkg.kv_read(a.cache, a.batch, pkg.KvRead(k=back[0].data_ptr(), v=back[1].data_ptr(), stride=128), _stream()),
                 lambda: pkg.attention(c.cache, c.batch, c.args, _stream())):
        assert hip.hipSetDevice(1 << 20) != 0  # a device that does not exist
        try:
            call()
        finally:
            left = hip.hipGetLastError()
        assert left != 0  # still there for who caused it
    torch.cuda.synchronize()
    a.expect()
    assert _same_bits(a.pools.dk.cpu(), a.pools.k) and torch.equal(c.out.cpu(), want)


def test_reading_rows_keeps_no_workspace(pkg):
    """A context that reads its rows back, or sets the window that it has, keeps a few words of tables for it and not the memory that split keys need."""
    hp = _hp(pkg, 1, 128, 4, maxL=200)
    work = 2 * 768 * 16 * (128 + 2) * 4  # what shares of split keys need
    tokens = np.arange(30, dtype=np.int32)
    kept = []
    for _ in range(2):  # (the first context loads code)
        dev = pkg.Device(hp, 0)
        dev.upload(_model(pkg, hp))
        dev.prefill(0, tokens)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        dev.set_attention_window(0, 0)
        dev.read_kv(0, 0, 0, 30)
        kept.append(before - torch.cuda.mem_get_info()[0])
        dev.set_attention_window(20, 2)
        dev.prefill(0, tokens)
        assert np.isfinite(dev.logits(0)).all()
        dev.close()
    assert kept[1] < work // 2, kept


@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("seqs,flags,ple", [(20, 3, 32), (70, 1, 0), (70, 2, 32)])
def test_contexts_of_many_sequences(pkg, four, seqs, flags, ple):
    """Contexts of 16 sequences and more hand attention over in other ways than smaller ones: prefills of all, more than 64 segments, then decode steps; a window of everything, by the
    row step and by GEMVs, gives the default's logits over fp32 pages.  Over 4-bit pages the two agree, and each sequence with the same alone: a code next to a border may fall to its
    other side, which moves an element by 2/15 of half its group's range, 0.28 of the rows' spread, and a row of 256 by 0.28 / 16 = 1.8e-2 of its norm."""
    hp = _hp(pkg, 2, 64, 4, flags, ple, seqs=seqs, maxL=130)
    model = _model(pkg, hp, std=0.05)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    rng = np.random.default_rng(seqs)
    dev.set_page_table(rng.permutation(seqs * ((hp.maxL + 63) // 64)).astype(np.int32))
    prompts = [rng.integers(0, hp.vocabSize, 1 + (37 * i) % 100).astype(np.int32) for i in range(seqs)]
    feed = rng.integers(0, hp.vocabSize, (3, seqs)).astype(np.int32)

    def run(mode):
        dev.set_prefill_mode(mode)
        dev.reset()
        dev.prefill_batch(range(seqs), prompts)
        out = [np.stack([dev.logits(s) for s in range(seqs)])]
        for f in feed:
            dev.decode_step(f)
        return out + [np.stack([dev.logits(s) for s in range(seqs)])]

    before = [run(mode) for mode in (0, 1)]
    if four:
        dev.reset()
        dev.set_kv_type(pkg.CACHE_Q4)
    dev.set_attention_window(hp.maxL, 3)
    after = [run(mode) for mode in (0, 1)]
    if not four:
        for a, b in zip(after, before):
            assert all(rel(x, y) < 1e-5 for x, y in zip(a, b))
    else:
        assert all(rel(x, y) < 2e-2 for x, y in zip(*after))
        one = pkg.Device(_hp(pkg, 2, 64, 4, flags, ple, seqs=1, maxL=130), 0)
        one.upload(model)
        one.set_kv_type(pkg.CACHE_Q4)
        for s in (0, seqs // 2, seqs - 1):
            one.reset()
            one.prefill(0, prompts[s])
            assert rel(after[0][0][s], one.logits(0)) < 2e-2
            for f in feed:
                one.decode_step([f[s]])
            assert rel(after[0][1][s], one.logits(0)) < 2e-2
        one.close()
    dev.close()
