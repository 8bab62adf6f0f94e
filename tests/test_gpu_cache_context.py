"""A context whose attention layers forget (mlh_set_attention_window) or keep 4-bit pages (mlh_set_kv_type), through prefill, decode, graphs and
teacher-forced scoring, against a 64-bit restatement of the decoder with that mask.  fp32 models: the logits of a few layers of fp32 sums, 1e-5 of their norm;
models with bf16 weights: the product's bar of 2e-2 relative (their prefills of more than 32 tokens hold activations as halves)."""
import numpy as np
import pytest

from conftest import assert_logits_close
from kv_oracle import values, quantise

import torch

pytestmark = pytest.mark.gpu


def rel(a, b):
    return np.linalg.norm(np.asarray(a, dtype=np.float64) - b) / np.linalg.norm(b)


def _bf16(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.bfloat16).double().numpy()


def _hp(pkg, n, hd=64, heads=2, flags=0, ple=0, gdn=0, seqs=1, maxL=200, bf16=0):
    hp = pkg.config(2, dim=hd * heads, attnHeads=heads, headDim=hd, ffnDim=192, transformers=n, vocabSize=301, maxL=maxL, maxSeqs=seqs, weightDtype=bf16,
                    qkRmsNorm=flags & 1, queryGating=flags >> 1, pleDim=ple, gdnHeads=heads if gdn else 0, gdnDk=hd if gdn else 0, gdnDv=hd if gdn else 0)
    pkg.set_layer_pattern(hp, gdn)
    return hp


def forward(pkg, model, tokens, window, sinks, stored=None):
    """Logits [n, V] and K, V [layer] -> [n, dim] of an attention-only model in 64 bits; stored: K and V rows to attend to instead of one's own."""
    hp = model.hparams
    d, H, hd, n = hp.dim, hp.attnHeads, hp.headDim, len(tokens)
    w = (lambda l, t: _bf16(model.tensor(l, t))) if hp.weightDtype else (lambda l, t: model.tensor(l, t).astype(np.float64))
    vec = lambda l, t: model.tensor(l, t).astype(np.float64).reshape(-1)
    rope = pkg.rope_table(hp.maxL, hd, hp.ropeDenomBase).astype(np.float64)[:n]
    c, s = rope[:, 0::2][:, None], rope[:, 1::2][:, None]
    norm = lambda x, g: g * x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-8)

    def turn(x):
        x = x.reshape(n, H, hd)
        a, b = x[..., 0::2], x[..., 1::2]
        return np.stack([c * a - s * b, s * a + c * b], -1).reshape(n, H, hd)

    pos = np.arange(n)
    seen = pos[None] <= pos[:, None]
    if window:
        seen &= (pos[:, None] - pos[None] < window) | (pos[None] < sinks)
    E = w(0, pkg.T_TOKEN_EMBEDDINGS)
    x = E[tokens]
    kv = {}
    for l in range(hp.transformers - 1, -1, -1):
        xn = norm(x, vec(l, pkg.T_RMS_GAMMA))
        q, k, v = (xn @ w(l, t).T for t in (pkg.T_QUERY, pkg.T_KEY, pkg.T_VALUE))
        if hp.qkRmsNorm:
            q = norm(q.reshape(n, H, hd), vec(l, pkg.T_QUERY_RMS_GAMMA).reshape(H, hd)).reshape(n, d)
            k = norm(k.reshape(n, H, hd), vec(l, pkg.T_KEY_RMS_GAMMA).reshape(H, hd)).reshape(n, d)
        q, k = turn(q), turn(k)
        kv[l] = (k.reshape(n, d), v)
        kk, vv = (k, v.reshape(n, H, hd)) if stored is None else (a.astype(np.float64).reshape(n, H, hd) for a in stored[l])
        a = np.empty((n, H, hd))
        for h in range(H):
            sc = np.where(seen, q[:, h] @ kk[:, h].T / np.sqrt(hd), -np.inf)
            p = np.exp(sc - sc.max(1, keepdims=True))
            a[:, h] = (p / p.sum(1, keepdims=True)) @ vv[:, h]
        a = a.reshape(n, d)
        if hp.queryGating:
            a = a / (1 + np.exp(-(xn @ w(l, pkg.T_GATED_QUERY).T)))
        h1 = x + a @ w(l, pkg.T_OUTPUT_PROJ).T
        if hp.pleDim:
            g = xn @ w(l, pkg.T_PLE_GATE).T
            h1 = h1 + (g / (1 + np.exp(-g)) * w(l, pkg.T_PLE_TABLE)[tokens]) @ w(l, pkg.T_PLE_UP).T
        hn = norm(h1, vec(l, pkg.T_RMS_GAMMA2))
        g = hn @ w(l, pkg.T_FFN_1A).T
        x = h1 + (g / (1 + np.exp(-g)) * (hn @ w(l, pkg.T_FFN_1B).T)) @ w(l, pkg.T_FFN_2).T
    return norm(x, vec(0, pkg.T_FINAL_RMS_GAMMA)) @ E.T, kv


def _model(pkg, hp, seed=3, std=0.08):
    model = pkg.Model.generate(hp, seed, std)
    model.randomize_gains(seed)
    return model


def _stored(dev, hp, seq, n):
    return {l: dev.read_kv(l, seq, 0, n) for l in range(hp.transformers) if hp.layerKinds[l] == 0}


@pytest.mark.parametrize("hd,heads,flags,ple", [(64, 2, 0, 0), (64, 3, 3, 32), (128, 1, 1, 0), (128, 2, 2, 32)])
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("n,window,sinks", [(40, 7, 2), (150, 33, 4), (150, 0, 0), (150, 64, 0)])
def test_logits(pkg, hd, heads, flags, ple, four, n, window, sinks):
    if not four and window == 0:
        pytest.skip("the default")
    hp = _hp(pkg, 2, hd, heads, flags, ple, maxL=n + 20)
    model = _model(pkg, hp)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    if four:
        dev.set_kv_type(pkg.CACHE_Q4)
    dev.set_attention_window(window, sinks)
    tokens = np.random.default_rng(n + window).integers(0, hp.vocabSize, n + 12).astype(np.int32)
    for mode in (0, 1):  # products over all tokens (row kernels up to 64, tiles beyond), token by token through GEMVs
        dev.set_prefill_mode(mode)
        assert dev.decode_route(1) == (pkg.DECODE_ROWS if mode == 0 else pkg.DECODE_GEMV)
        dev.reset()
        got, _, _ = dev.forward_full(0, tokens[:n])
        dev.reset()
        dev.prefill(0, tokens[:n - 9])
        dev.prefill(0, tokens[n - 9:n])  # a chunk behind a context
        chunked = dev.logits(0)
        more = []
        for t in tokens[n:]:
            dev.decode_step([t])
            more.append(dev.logits(0))
        stored = _stored(dev, hp, 0, n + 12)
        want, kv = forward(pkg, model, tokens, window, sinks, stored if four else None)
        assert rel(got, want[:n]) < 1e-5 if not four else rel(got, want[:n]) < 1e-4  # (the codes of the first pass may differ from the second's next to a border)
        assert rel(chunked, want[n - 1]) < 1e-5
        assert rel(np.stack(more), want[n:]) < 1e-5
        for l, (k, v) in stored.items():
            for a, b in zip((k, v), kv[l]):
                if not four:
                    assert rel(a, b) < 1e-5
                else:  # half a step of its group, or a whole one where fp32 and fp64 fall to different sides
                    _, par = quantise(torch.from_numpy(b).float().reshape(n + 12, heads, hd))
                    step = np.repeat(par[..., 1].double().numpy().reshape(n + 12, -1), 32, 1)
                    assert (np.abs(a - b) <= 0.51 * step + 2.0 ** -10 * np.abs(b)).mean() > 0.999 and (np.abs(a - b) <= 1.1 * step + 2.0 ** -10 * np.abs(b)).all()
    dev.close()


@pytest.mark.parametrize("four", [False, True])
def test_bf16_model(pkg, four):
    hp = _hp(pkg, 2, 128, 2, 3, 64, maxL=220, bf16=1)
    model = _model(pkg, hp)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    if four:
        dev.set_kv_type(pkg.CACHE_Q4)
    dev.set_attention_window(50, 3)
    tokens = np.random.default_rng(5).integers(0, hp.vocabSize, 200).astype(np.int32)
    for n in (20, 190):
        dev.reset()
        dev.prefill(0, tokens[:n])
        first = dev.logits(0)
        dev.decode_step([tokens[n]])
        second = dev.logits(0)
        want, _ = forward(pkg, model, tokens[:n + 1], 50, 3, _stored(dev, hp, 0, n + 1))
        if n > 32:
            # Halves: the normalised rows, the mixing output and the FFN units of two layers and the last normalised row, 9 vectors with 4 more of q, k, v and the weights of the
            # attention where they are halves, each off by at most 2^-11 of its norm.  An element of the logits is no measure: the last row alone may move one by
            # 2^-11 sum |x_i E_i| ~ 2^-11 * 256 * 0.8 * 0.064 = 6e-3, whatever its size (the largest is 4.2).
            assert rel(first, want[n - 1]) < 13 * 2.0 ** -11
        else:
            assert_logits_close(first, want[n - 1], 2e-2, "prefill")
        assert_logits_close(second, want[n], 2e-2, "decode")
    dev.close()


@pytest.mark.parametrize("gdn", [0, 1, 3])
def test_wide_window_is_the_default(pkg, gdn):
    """A window of all positions, several sequences, permuted pages: what the default gives, by other kernels; and back to the default."""
    hp = _hp(pkg, 4, 64, 4, 0, 32, gdn, seqs=5, maxL=300)
    model = _model(pkg, hp, std=0.05)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    rng = np.random.default_rng(7)
    per = (hp.maxL + 63) // 64
    dev.set_page_table(rng.permutation(5 * per).astype(np.int32))
    prompts = [rng.integers(0, hp.vocabSize, n).astype(np.int32) for n in (3, 150, 64, 65, 30)]
    feed = rng.integers(0, hp.vocabSize, (4, 5)).astype(np.int32)

    def run():
        dev.reset()
        dev.prefill_batch(range(5), prompts)
        out = [np.stack([dev.logits(s) for s in range(5)])]
        for f in feed:
            dev.decode_step(f)
        out.append(np.stack([dev.logits(s) for s in range(5)]))
        ids = dev.decode_loop(feed[-1], 6)
        return out, ids

    before, ids = run()
    route = dev.decode_route(5)
    dev.set_attention_window(hp.maxL, 9)
    assert dev.decode_route(5) == pkg.DECODE_ROWS and dev.decode_route(1) == pkg.DECODE_ROWS
    out, same = run()
    for a, b in zip(out, before):
        assert rel(a, b) < 1e-5
    assert np.array_equal(same, ids)
    for k in (1, 3):
        dev.set_graph(k)
        again, same = run()
        for a, b in zip(again, out):
            assert np.array_equal(a, b)
        assert np.array_equal(same, ids)
    dev.set_graph(0)
    dev.set_attention_window(0)
    assert dev.decode_route(5) == route
    again, same = run()
    for a, b in zip(again, before):
        assert np.array_equal(a, b)
    dev.close()


@pytest.mark.parametrize("four", [False, True])
def test_graphs_and_changes_of_the_window(pkg, four):
    """Replays of captured steps follow a new window; prefill and single steps agree on a hybrid model."""
    hp = _hp(pkg, 4, 64, 2, 1, 0, 1, seqs=2, maxL=260)
    model = _model(pkg, hp, std=0.05)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    if four:
        dev.set_kv_type(pkg.CACHE_Q4)
    rng = np.random.default_rng(8)
    tokens = rng.integers(0, hp.vocabSize, (2, 150)).astype(np.int32)
    for window, sinks in ((20, 1), (64, 0), (100, 70)):
        dev.set_attention_window(window, sinks)
        dev.set_graph(0)
        dev.reset()
        dev.prefill_batch([0, 1], [tokens[0, :140], tokens[1, :131]])
        eager = dev.decode_loop([5, 6], 9)
        logits = [dev.logits(s) for s in range(2)]
        dev.set_graph(4)
        dev.reset()
        dev.prefill_batch([0, 1], [tokens[0, :140], tokens[1, :131]])
        assert np.array_equal(dev.decode_loop([5, 6], 9), eager)
        assert all(np.array_equal(dev.logits(s), logits[s]) for s in range(2))
        dev.set_graph(0)
        if not four:  # (4-bit codes may fall to the other side of a border)
            whole = np.concatenate([tokens[0, :140], [5], eager[:-1, 0]]).astype(np.int32)
            dev.reset()
            dev.prefill(0, whole)
            assert rel(dev.logits(0), logits[0]) < 1e-5
    dev.close()


def test_kv_type_rules(pkg):
    hp = _hp(pkg, 2, 64, 2, maxL=100)
    model = _model(pkg, hp)
    dev = pkg.Device(hp, 0)
    dev.upload(model)
    tokens = np.arange(30, dtype=np.int32)
    dev.prefill(0, tokens)
    before = dev.logits(0)
    for bad in (pkg.DTYPE_BF16, pkg.DTYPE_F16, 3, -1):
        with pytest.raises(pkg.MlhError, match="MLH_DTYPE_F32 or MLH_CACHE_Q4"):
            dev.set_kv_type(bad)
    with pytest.raises(pkg.MlhError, match="empty"):
        dev.set_kv_type(pkg.CACHE_Q4)
    for w, s in ((-1, 0), (0, -1)):
        with pytest.raises(pkg.MlhError, match="negative"):
            dev.set_attention_window(w, s)
    for args in ((-1, 0, 0, 1), (2, 0, 0, 1), (0, 1, 0, 1), (0, 0, -1, 2), (0, 0, 0, 31), (0, 0, 30, 1), (0, 0, 0, 0)):
        with pytest.raises(pkg.MlhError):
            dev.read_kv(*args)
    k, v = dev.read_kv(1, 0, 3, 20)
    _, kv = forward(pkg, model, tokens, 0, 0)
    assert rel(k, kv[1][0][3:23]) < 1e-5 and rel(v, kv[1][1][3:23]) < 1e-5
    dev.reset()
    dev.set_kv_type(pkg.CACHE_Q4)
    dev.upload(model)  # weights anew: the pages stay as they are
    dev.prefill(0, tokens)
    k4, _ = dev.read_kv(1, 0, 3, 20)
    assert 1e-3 < rel(k4, k) < 0.15
    dev.time_decode([3], 4)
    dev.reset()
    dev.set_kv_type(pkg.DTYPE_F32)
    dev.prefill(0, tokens)
    assert np.array_equal(dev.logits(0), before)
    dev.close()


def test_measurement_and_sampling(pkg):
    """Timing of the attention part, a profile of steps and sampled tokens with a window and 4-bit pages."""
    hp = _hp(pkg, 3, 64, 2, 0, 0, 0, seqs=3, maxL=120)
    dev = pkg.Device(hp, 0)
    dev.upload(_model(pkg, hp))
    dev.set_kv_type(pkg.CACHE_Q4)
    dev.set_attention_window(30, 2)
    prompts = [np.arange(20 + s, dtype=np.int32) for s in range(3)]
    dev.prefill_batch(range(3), prompts)
    us, nbytes = dev.time_kernel(pkg.K_ATTN, 0, 3, 5)
    assert us > 0 and nbytes == sum(2 * 0.625 * hp.dim * n + 2 * 0.625 * hp.dim for n in (21, 22, 23))
    dev.reset()
    runs = []
    for k in (0, 2, 0):
        dev.set_graph(k)
        dev.reset()
        dev.prefill_batch(range(3), prompts)
        dev.set_sampling(0.8, 7)
        runs.append(dev.decode_loop([1, 2, 3], 20))
        dev.set_sampling(0.0)
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])
    dev.close()


def test_single_launch_shapes(pkg):
    """A model that the single-launch kernels cover leaves them for a window or other pages, and comes back with neither."""
    hp = _hp(pkg, 2, 64, 8, seqs=2, maxL=120)
    dev = pkg.Device(hp, 0)
    dev.upload(_model(pkg, hp))
    n, route = dev.single_launch_sequences(), dev.decode_route(1)
    assert n > 0 and route in (pkg.DECODE_XCD, pkg.DECODE_RANKS)
    dev.set_kv_type(pkg.CACHE_Q4)
    assert dev.single_launch_sequences() == 0 and dev.decode_route(1) == pkg.DECODE_ROWS
    dev.set_attention_window(40)
    dev.set_kv_type(pkg.DTYPE_F32)
    assert dev.single_launch_sequences() == 0 and dev.decode_route(1) == pkg.DECODE_ROWS
    dev.set_attention_window(0)
    assert dev.single_launch_sequences() == n and dev.decode_route(1) == route
    other = pkg.Device(hp, 0)  # the pages are new ones: every route finds them
    other.upload(_model(pkg, hp))
    tokens = np.arange(50, dtype=np.int32)
    for mode in (3, 0):
        got = []
        for d in (dev, other):
            d.set_persistent(mode)
            d.reset()
            d.prefill_batch([0, 1], [tokens, tokens[:9]])
            got.append((d.decode_loop([3, 4], 12), d.decode_loop([3], 12), d.logits(0)))
        assert all(np.array_equal(a, b) for a, b in zip(*got)), mode
    other.close()
    dev.close()


def test_model_without_attention(pkg):
    """Gated-delta-net layers have no window: nothing changes."""
    hp = _hp(pkg, 2, 64, 2, 0, 0, 1, seqs=1, maxL=60)
    for l in range(2):
        hp.layerKinds[l] = pkg.KIND_GDN
    dev = pkg.Device(hp, 0)
    dev.upload(_model(pkg, hp, std=0.05))
    tokens = np.arange(40, dtype=np.int32)
    dev.prefill(0, tokens)
    before, route = dev.logits(0), dev.decode_route(1)
    dev.set_attention_window(5, 1)
    dev.reset()
    dev.set_kv_type(pkg.CACHE_Q4)
    dev.prefill(0, tokens)
    assert np.array_equal(dev.logits(0), before) and dev.decode_route(1) == route
    with pytest.raises(pkg.MlhError, match="not an attention layer"):
        dev.read_kv(0, 0, 0, 1)
    dev.close()
