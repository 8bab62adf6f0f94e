"""Calls around the operators on a paged K/V cache."""
import ctypes

import numpy as np
import pytest
import torch

from test_gpu_cache import Append, Call, _same_bits, _stream
from test_gpu_cache_context import _hp, _model
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
