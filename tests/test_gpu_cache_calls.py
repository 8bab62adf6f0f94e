"""Calls around the operators on a paged K/V cache."""
import ctypes

import pytest
import torch

from test_gpu_cache import Append, Call, _same_bits, _stream
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
