"""Attention over a paged K/V cache where numbers are at their limits."""
import pytest
import torch

from kv_oracle import GROUP, quantise
from test_gpu_cache import Call

pytestmark = pytest.mark.gpu


def _store(c, which, seq, rows, pos=0):
    """Other rows [n, kv, hd] at positions pos .. of a sequence of a call that was built already."""
    held = (c.keys if which == "k" else c.vals)[seq]
    held[pos:pos + rows.shape[0]] = c.pools.put(which, seq, pos, rows)
    (c.pools.dk if which == "k" else c.pools.dv).copy_(c.pools.k if which == "k" else c.pools.v)


def _query(c, q):
    """Other rows [used, H * hd]."""
    c.q[:c.rows.used, :c.H * c.hd] = q.to(c.q.dtype)
    c.dq.copy_(c.q)


# ---------------------------------------------------------------------------------------------------------------------
# groups that span more than 65504
# ---------------------------------------------------------------------------------------------------------------------
def _wide(gen, n, K, hd, most):
    """Rows whose groups of 32 go from -most to most."""
    x = (torch.rand(n, K, hd // GROUP, GROUP, generator=gen) * 2 - 1) * most
    x[..., 0], x[..., 1] = -most, most
    return x[..., torch.randperm(GROUP, generator=gen)].flatten(2)


@pytest.mark.parametrize("kind", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("H,new,lens", [(1, [1], [200]), (12, [1, 1], [200, 70]), (2, [5], [200]), (2, [30], [90]), (2, [70], [100]), (1, [1], [3000])])
def test_wide_groups(pkg, kind, hd, H, new, lens):
    """Keys whose groups go from -40000 to 40000: codes times scale pass the halves' range (15 * 5332 = 79980), the values they stand for do not.  Every form of the
    attention takes them: the same tolerance as for other keys."""
    c = Call(pkg, kind, "q4", H, 1, hd, new, lens, seed=40, spread=0.02, scale=1e-3)
    gen = torch.Generator().manual_seed(41)
    for s, n in enumerate(lens):
        _store(c, "k", s, _wide(gen, n, 1, hd, 40000.0))
        assert c.keys[s].abs().max() < 65504 < 15 * float(quantise(_wide(gen, 1, 1, hd, 40000.0))[1][..., 1].min())
    c.check()
