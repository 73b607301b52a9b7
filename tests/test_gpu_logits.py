"""lc_logits_process on the GPU: bit for bit against the f32 restatement (every
operation is rounded once in a fixed order), and against 64 bits within those
roundings."""
import numpy as np
import pytest

import logits_ref
from laguna_raw_halo_strix_b200 import lc

pytestmark = pytest.mark.gpu


def make(rng, m, n, hist, bias, masks, offset=0, vocab=None):
    """Host arrays of a batch whose lists are about hist / bias long, with ids outside the shard among them."""
    vocab = vocab or offset + n
    d = {}
    if hist:
        sizes = rng.integers(0, 2 * hist, m)
        sizes[rng.integers(m)] = 0
        d["hist_start"] = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        d["hist"] = (rng.random(sizes.sum()) ** 3 * (vocab + 20)).astype(np.int32) - 10
        d["gen_start"] = (d["hist_start"][:-1] + rng.integers(0, sizes + 1)).astype(np.int32)
        d["repetition"] = rng.uniform(0.7, 1.5, m).astype(np.float32)
        d["frequency"] = rng.uniform(-0.5, 1, m).astype(np.float32)
        d["presence"] = rng.uniform(-0.5, 1, m).astype(np.float32)
    if bias:
        sizes = rng.integers(0, 2 * bias, m)
        d["bias_start"] = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
        d["bias_tok"] = rng.integers(-5, vocab + 5, sizes.sum()).astype(np.int32)
        d["bias_tok"][::3] = d["bias_tok"][:1] if len(d["bias_tok"]) else 0  # the same id many times
        d["bias"] = rng.standard_normal(sizes.sum()).astype(np.float32)
    if masks:
        d["mask"] = rng.integers(0, 2 ** 32, (masks, (offset + n + 31) // 32 + 1), dtype=np.uint32)
        d["mask_row"] = rng.integers(-1, masks + 1, m).astype(np.int32)
    return d


def to_gpu(d, dev):
    import torch

    def one(a):
        return torch.from_numpy(a.view(np.int32) if a.dtype == np.uint32 else a).to(dev)

    return lc.LogitsRules(**{k: one(v) for k, v in d.items()})


def check(ctx, dev, x, d, offset=0, ld=None, shift=0, keys=True, out=True, in_place=False):
    import torch

    m, n = x.shape
    ld = ld or n
    buf = torch.full((m * ld + 8,), 7.0, device=dev)
    rows = torch.as_strided(buf, (m, n), (ld, 1), shift)
    rows.copy_(torch.from_numpy(x))
    obuf = buf if in_place else torch.full((m * ld + 8,), -7.0, device=dev)
    orows = torch.as_strided(obuf, (m, n), (ld, 1), shift)
    key = torch.zeros(m, dtype=torch.int64, device=dev) if keys else None
    rules = to_gpu(d, dev)
    ctx.logits_process(rows, rules, orows if out else None, key, m, n, offset, ld=ld, ld_out=ld if out else 0)
    torch.cuda.synchronize()
    ref, _, best = logits_ref.process(x, offset, **d)
    ref64, tol, _ = logits_ref.process(x, offset, **d, dtype=np.float64)
    if out:
        got = orows.cpu().numpy()
        assert np.array_equal(got.view(np.uint32), ref.view(np.uint32))
        inf = np.isinf(ref64)
        assert np.array_equal(np.isinf(got), inf)
        err = np.abs(np.where(inf, 0, got) - np.where(inf, 0, ref64))
        assert (err <= tol * (1 + 2.0 ** -20)).all()
        rest = torch.ones(m * ld + 8, dtype=torch.bool, device=dev)
        torch.as_strided(rest, (m, n), (ld, 1), shift)[:] = False
        assert (obuf[rest] == (7.0 if in_place else -7.0)).all()
    if keys:
        for r in range(m):
            k = int(key[r])
            assert lc.key_index(k) == offset + best[r], r
            assert np.float32(lc.key_value(k)).view(np.uint32) == ref[r, best[r]].view(np.uint32)


@pytest.mark.parametrize("m,n,hist,bias,masks", [(1, 1, 0, 0, 0), (1, 1, 3, 2, 1), (3, 7, 20, 5, 2), (5, 127, 50, 0, 0),
                                                 (2, 4095, 300, 10, 1), (4, 8192, 0, 100, 0), (3, 8193, 900, 0, 3),
                                                 (2, 50021, 3000, 200, 2), (1, 128256, 4000, 50, 1),
                                                 (7, 32000, 1000, 30, 7), (2, 262144, 0, 0, 2)])
def test_sizes(ctx, dev, m, n, hist, bias, masks):
    rng = np.random.default_rng(m * 1000 + n)
    x = (4 * rng.standard_normal((m, n))).astype(np.float32)
    check(ctx, dev, x, make(rng, m, n, hist, bias, masks))


@pytest.mark.parametrize("n,ld,shift", [(1000, 1003, 0), (1001, 1004, 4), (5000, 5001, 1), (9000, 9000, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_strides_and_in_place(ctx, dev, n, ld, shift, in_place):
    rng = np.random.default_rng(n)
    x = (4 * rng.standard_normal((6, n))).astype(np.float32)
    check(ctx, dev, x, make(rng, 6, n, 200, 20, 3), ld=ld, shift=shift, in_place=in_place)


@pytest.mark.parametrize("keys,out", [(True, False), (False, True)])
def test_only_one_output(ctx, dev, keys, out):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((4, 3001)).astype(np.float32)
    check(ctx, dev, x, make(rng, 4, 3001, 100, 20, 2), keys=keys, out=out)


@pytest.mark.parametrize("rule", ["repetition", "frequency", "presence", "gen_start", "mask_row"])
def test_missing_rules(ctx, dev, rule):
    rng = np.random.default_rng(4)
    x = rng.standard_normal((5, 2000)).astype(np.float32)
    d = make(rng, 5, 2000, 100, 20, 5)
    del d[rule]
    check(ctx, dev, x, d)


@pytest.mark.parametrize("offset", [1, 32, 16032, 2 ** 20 + 5])
def test_vocab_shards(ctx, dev, offset):
    rng = np.random.default_rng(offset)
    x = rng.standard_normal((3, 16032)).astype(np.float32)
    check(ctx, dev, x, make(rng, 3, 16032, 2000, 200, 2, offset=offset, vocab=offset + 2 * 16032), offset=offset)


def test_special_values(ctx, dev):
    """Infinities, NaN (kept where allowed, gone where masked), signed zeros, ties and rows with nothing allowed."""
    import torch

    n = 300
    x = np.zeros((6, n), np.float32)
    x[0, 5], x[0, 250] = np.inf, -np.inf
    x[1] = -np.inf
    x[2, 7] = np.nan                      # masked below
    x[3, 100], x[3, 200] = 2.0, 2.0       # a tie: the larger token
    x[4] = -0.0
    x[4, 3] = 0.0                         # +0 orders above -0
    x[5, 9] = 50.0
    mask = np.full((3, 10), 0xFFFFFFFF, np.uint32)
    mask[0, 0] &= ~np.uint32(1 << 7)
    mask[1] = 0
    d = dict(mask=mask, mask_row=np.array([2, 2, 0, 2, 2, 1], np.int32), hist=np.array([5, 250, 7], np.int32),
             hist_start=np.array([0, 2, 2, 3, 3, 3, 3], np.int32), repetition=np.full(6, 1.5, np.float32))
    rules = to_gpu(d, dev)
    xd = torch.from_numpy(x).to(dev)
    out, keys = torch.empty_like(xd), torch.empty(6, dtype=torch.int64, device=dev)
    ctx.logits_process(xd, rules, out, keys, 6, n)
    torch.cuda.synchronize()
    got = out.cpu().numpy()
    assert got[0, 5] == np.inf and got[0, 250] == -np.inf and got[2, 7] == -np.inf and not np.isnan(got).any()
    assert np.isinf(got[5]).all()
    best = [(lc.key_value(int(k)), lc.key_index(int(k))) for k in keys]
    assert best == [(np.inf, 5), (-np.inf, n - 1), (0.0, n - 1), (2.0, 200), (0.0, 3), (-np.inf, n - 1)]


def test_starts_outside_the_lists_are_held_inside(ctx, dev):
    """Start arrays that point before, behind and backwards read nothing outside their arrays."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((5, 1500)).astype(np.float32)
    d = make(rng, 5, 1500, 50, 10, 0)
    d["hist_start"] = np.array([-100, 20, 10, 2 ** 31 - 1, -(2 ** 31), 30], np.int32)
    d["bias_start"] = np.array([2 ** 30, -1, 5, 3, 2 ** 31 - 1, 7], np.int32)
    check(ctx, dev, x, d)


def test_matches_argmax_rows_without_rules(ctx, dev):
    import torch

    x = torch.randn(9, 7777, device=dev)
    x[:, 100] = x[:, 7000] = 9.0
    a, b = torch.empty(9, dtype=torch.int64, device=dev), torch.empty(9, dtype=torch.int64, device=dev)
    ctx.argmax_rows(x, 9, 7777, 64, a)
    ctx.logits_process(x, lc.LogitsRules(), None, b, 9, 7777, 64)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_two_streams_and_graph_replay(ctx, dev):
    """Calls on two streams at once, and a captured call that sees a list that grew."""
    import torch

    rng = np.random.default_rng(6)
    n = 20000
    x = (4 * rng.standard_normal((4, n))).astype(np.float32)
    d = make(rng, 4, n, 300, 30, 2)
    xd = torch.from_numpy(x).to(dev)
    rules = to_gpu(d, dev)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    ctxs = [lc.Context(0), lc.Context(0)]
    outs = [torch.empty_like(xd) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s, o in zip(ctxs, streams, outs):
            c.set_stream(s)
            c.logits_process(xd, rules, o, None, 4, n)
    torch.cuda.synchronize()
    ref, _, _ = logits_ref.process(x, **d)
    for o in outs:
        assert np.array_equal(o.cpu().numpy().view(np.uint32), ref.view(np.uint32))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        ctxs[0].logits_process(xd, rules, outs[0], None, 4, n)
    d["hist_start"][4] -= 7
    rules.held[1].copy_(torch.from_numpy(d["hist_start"]))
    graph.replay()
    torch.cuda.synchronize()
    ref, _, _ = logits_ref.process(x, **d)
    assert np.array_equal(outs[0].cpu().numpy().view(np.uint32), ref.view(np.uint32))
    del graph
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("m,n,hist,bias,masks", [(450, 7, 5, 2, 3), (700, 1500, 60, 10, 2), (460, 4097, 0, 20, 460),
                                                 (450, 9001, 30, 150, 1), (300, 20000, 100, 0, 0), (130, 50021, 300, 40, 2),
                                                 (20, 128256, 2000, 200, 3), (450, 8192, 3000, 5, 0),
                                                 (600, 1849, 2000, 3, 2)])
def test_many_rows(ctx, dev, m, n, hist, bias, masks):
    """More rows than the device takes at a time: lists of each row ahead of its logits, and in some
    sizes more tokens in one place than are kept, or a history longer than the vocabulary."""
    rng = np.random.default_rng(m + n)
    x = (4 * rng.standard_normal((m, n))).astype(np.float32)
    check(ctx, dev, x, make(rng, m, n, hist, bias, masks))


@pytest.mark.parametrize("n,ld,shift,offset", [(4099, 4100, 0, 0), (4101, 4103, 3, 16032), (6000, 6000, 0, 33)])
@pytest.mark.parametrize("in_place,keys,out", [(True, True, True), (False, False, True), (False, True, False)])
def test_many_rows_strides_and_shards(ctx, dev, n, ld, shift, offset, in_place, keys, out):
    rng = np.random.default_rng(n + offset)
    x = (4 * rng.standard_normal((500, n))).astype(np.float32)
    d = make(rng, 500, n, 40, 10, 7, offset=offset, vocab=offset + 2 * n)
    check(ctx, dev, x, d, offset=offset, ld=ld, shift=shift, in_place=in_place, keys=keys, out=out)


def test_many_rows_of_a_long_vocabulary(ctx, dev):
    """A CTA with more slices than groups of tokens kept for them."""
    import torch

    m, n = 444, 140000
    rng = np.random.default_rng(8)
    x = torch.randn(m, n, device=dev)
    d = make(rng, m, n, 300, 30, 2)
    out, keys = torch.empty_like(x), torch.empty(m, dtype=torch.int64, device=dev)
    ctx.logits_process(x, to_gpu(d, dev), out, keys, m, n)
    torch.cuda.synchronize()
    for r in (0, 1, 200, 443):
        one = {k: v[r:r + 1] for k, v in d.items() if k in ("gen_start", "repetition", "frequency", "presence", "mask_row")}
        one |= {k: d[k] for k in ("hist", "bias_tok", "bias", "mask")}
        one |= {k: d[k][r:r + 2] for k in ("hist_start", "bias_start")}
        ref, _, best = logits_ref.process(x[r:r + 1].cpu().numpy(), **one)
        assert np.array_equal(out[r].cpu().numpy().view(np.uint32), ref[0].view(np.uint32))
        assert lc.key_index(int(keys[r])) == best[0]


def test_many_rows_special_values(ctx, dev):
    """Rows of the order's lowest value, of -inf and of NaN among ordinary ones."""
    import torch

    m, n = 450, 5000
    x = torch.zeros(m, n, device=dev)
    x[1] = -float("inf")
    x[2].view(torch.int32)[:] = -1
    x[3, 17] = float("nan")
    x[449, 3] = 1.0
    out, keys = torch.empty_like(x), torch.empty(m, dtype=torch.int64, device=dev)
    ctx.logits_process(x, lc.LogitsRules(), out, keys, m, n)
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int32), x.view(torch.int32))
    at = [lc.key_index(int(k)) for k in keys.cpu()]
    assert at[1] == n - 1 and at[2] == n - 1 and at[3] == 17 and at[449] == 3 and at[4] == n - 1


def test_captured_calls_of_many_rows_on_two_streams(ctx, dev):
    """Replays side by side, and a list that grew between them."""
    import torch

    rng = np.random.default_rng(9)
    m, n = 460, 9000
    x = (4 * rng.standard_normal((m, n))).astype(np.float32)
    d = make(rng, m, n, 60, 10, 2)
    d["hist_start"][m] -= 7
    xd, rules = torch.from_numpy(x).to(dev), to_gpu(d, dev)
    streams, ctxs = [torch.cuda.Stream(), torch.cuda.Stream()], [lc.Context(0), lc.Context(0)]
    outs = [torch.empty_like(xd) for _ in range(2)]
    torch.cuda.synchronize()
    graphs = []
    for c, s, o in zip(ctxs, streams, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            c.set_stream(s)
            c.logits_process(xd, rules, o, None, m, n)
        graphs.append(g)
    for grow in (0, 7):
        d["hist_start"][m] += grow
        rules.held[1].copy_(torch.from_numpy(d["hist_start"]))
        torch.cuda.synchronize()
        for _ in range(10):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        ref, _, _ = logits_ref.process(x, **d)
        for o in outs:
            assert np.array_equal(o.cpu().numpy().view(np.uint32), ref.view(np.uint32))
