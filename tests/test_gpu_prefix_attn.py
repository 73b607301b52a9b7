"""lc_prefix_attn on the GPU against the definition in 64 bits.

Error of an output o = sum w_j v_j / sum w_j, with u the step of the input type
(half a step: 2^-9 of bf16's value is eps / 2 = 2^-8 relative, f16 2^-11):
  - scores: exact 16-bit products summed in f32 over head_dim terms, then scaled:
    (head_dim + 2) 2^-24 sum_d |q_d k_d| * scale * log2(e) in the exponent, which
    turns into that times ln 2 relative in w (S below);
  - exp2 about 2^-22 relative;
  - w rounded to the input type, eps / 2 relative (squared for f32 outputs, where
    a second plane holds what the first lost);
  - sums over n keys in f32: n 2^-24 of sum w_j |v_j| at most; taken as
    (sqrt(n) + 64) 2^-24, the tensor cores adding 16 products at a time
    and rounding errors being of both signs;
  - f16 weights below 2^-14 are subnormal: off by at most 2^-25 each, with
    sum w_j at least what it is relative to the largest score;
each applies to A = sum w_j |v_j| / sum w_j, and the normaliser doubles all but
the rounding of w.  The output's own rounding adds eps / 2 of |o|."""
import math

import pytest

from laguna_raw_halo_strix_b200 import lc

pytestmark = pytest.mark.gpu

IDS = {"f32": lc.F32, "f16": lc.F16, "bf16": lc.BF16}


def tt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


class Batch:
    """A batch on the GPU: counts[i] query rows and lens[i] own keys of sequence i."""

    def __init__(self, dev, src, dst, n_q, n_kv, hd, prefix, cap, counts, lens, seed=0, extra=0, spread=1.0, gap=0,
                 garbage=True):
        import torch

        g = torch.Generator(dev).manual_seed(seed)
        wk, wq, n = n_kv * hd, n_q * hd, len(counts)
        self.src, self.dst, self.n_q, self.n_kv, self.hd = src, dst, n_q, n_kv, hd
        self.prefix, self.cap, self.counts, self.lens = prefix, cap, counts, lens
        self.rows = sum(counts) + extra

        def rows(shape, width, fill=None):
            """[*shape, width] whose last rows are width + gap apart."""
            x = torch.randn(*shape, width + gap, generator=g, device=dev) * (spread if fill is None else 1)
            return x.to(tt(src))[..., :width]

        self.q = rows((self.rows,), wq)
        self.kp, self.vp = rows((max(prefix, 1),), wk), rows((max(prefix, 1),), wk, 1)
        self.ko, self.vo = rows((n, max(cap, 1)), wk), rows((n, max(cap, 1)), wk, 1)
        if garbage:  # what lies behind a sequence's rows must not matter
            for i, length in enumerate(lens):
                self.ko[i, max(length, 0):] = float("nan")
                self.vo[i, max(length, 0):] = float("inf")
        self.ld = wk + gap
        self.out = torch.full((self.rows, wq + gap), 77.0, device=dev).to(tt(dst))
        self.own_len = torch.tensor(lens, dtype=torch.int32, device=dev)
        start = [0]
        for c in counts:
            start.append(start[-1] + c)
        self.seq_start = torch.tensor(start, dtype=torch.int32, device=dev)
        self.scale = 1 / math.sqrt(hd)

    def kv(self):
        return lc.PrefixKV(self.kp, self.vp, self.prefix, self.ko, self.vo, self.cap, self.own_len, self.seq_start,
                           len(self.counts), ld_prefix=self.ld, ld_own=self.ld, own_stride=self.ko.stride(0))

    def run(self, ctx, causal=1):
        ctx.prefix_attn(IDS[self.src], IDS[self.dst], self.q, self.kv(), self.out, self.rows, self.n_q, self.n_kv,
                        self.hd, self.scale, causal, ldq=self.q.stride(0), ldo=self.out.stride(0))

    def check(self, causal=1):
        import torch

        torch.cuda.synchronize()
        hd, group, wq = self.hd, self.n_q // self.n_kv, self.n_q * self.hd
        eps_in = torch.finfo(tt(self.src)).eps / 2
        at = 0
        for i, (c, length) in enumerate(zip(self.counts, self.lens)):
            length = min(max(length, 0), self.cap)
            n = self.prefix + length
            k = torch.cat([self.kp[:self.prefix], self.ko[i, :length]]).double().view(n, self.n_kv, hd)
            v = torch.cat([self.vp[:self.prefix], self.vo[i, :length]]).double().view(n, self.n_kv, hd)
            q = self.q[at:at + c].double().view(c, self.n_kv, group, hd)
            s = torch.einsum("rhgd,khd->hgrk", q, k) * self.scale
            mag = torch.einsum("rhgd,khd->hgrk", q.abs(), k.abs()) * self.scale
            key = torch.arange(n, device=s.device)
            reach = torch.arange(c, device=s.device) + (length - c) if causal else \
                torch.full((c,), length, device=s.device)
            seen = (key < self.prefix) | (key - self.prefix <= reach[:, None])
            s = s.masked_fill(~seen, -math.inf)
            top = s.amax(-1, keepdim=True) if n else torch.zeros(*s.shape[:-1], 1, device=s.device).double()
            w = torch.where(seen, (s - top.clamp(min=-1e300)).exp(), 0.0)
            total = w.sum(-1, keepdim=True)
            flat = torch.einsum("hgrk,khd->rhgd", torch.where(total > 0, seen / total, 0.0), v.abs()).reshape(c, wq)
            w = torch.where(total > 0, w / total, 0.0)
            o = torch.einsum("hgrk,khd->rhgd", w, v).reshape(c, wq)
            a = torch.einsum("hgrk,khd->rhgd", w, v.abs()).reshape(c, wq)
            err_s = ((hd + 2) * 2.0 ** -24 * mag * seen).amax(-1) if n else torch.zeros(s.shape[:-1], device=s.device)
            err_s = err_s.permute(2, 0, 1).reshape(c, self.n_q, 1).expand(-1, -1, hd).reshape(c, wq)
            w_round = eps_in ** 2 if self.dst == "f32" else eps_in
            tol = a * (2 * (err_s * 1.01 + 2.0 ** -22 + (math.sqrt(n) + 64) * 2.0 ** -24) + w_round)
            if self.src == "f16":
                tol = tol + flat * 2.0 ** -25
            fo = torch.finfo(tt(self.dst))
            tol = tol * 1.001 + o.abs() * fo.eps / 2 + fo.smallest_normal * fo.eps
            got = self.out[at:at + c, :wq].double()
            bad = ~((got - o).abs() <= tol)
            assert not bad.any(), (i, int(bad.sum()), float(((got - o).abs() - tol).max()), bad.nonzero()[:4].tolist())
            at += c
        assert (self.out[at:] == 77.0).all(), "rows of no sequence"
        assert (self.out[:, wq:] == 77.0).all(), "columns behind a row"


TYPES = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "f32")]


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("prefix,cap,counts,lens", [
    (1, 1, [1], [1]), (0, 1, [1], [1]), (128, 0, [1], [0]), (127, 3, [1, 1], [1, 3]), (129, 130, [1, 1, 1], [130, 1, 64]),
    (300, 40, [1] * 9, [40, 1, 7, 16, 17, 31, 32, 33, 5]), (1000, 257, [3, 1, 16, 2], [257, 128, 16, 129])])
def test_small(ctx, dev, src, dst, hd, prefix, cap, counts, lens):
    b = Batch(dev, src, dst, 4, 2, hd, prefix, cap, counts, lens, seed=prefix)
    b.run(ctx)
    b.check()
    ctx.device_status()


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n_q,n_kv", [(1, 1), (5, 1), (8, 8), (32, 8), (24, 2), (48, 8), (3, 1), (9, 1), (17, 1), (40, 1),
                                       (64, 1), (100, 1), (128, 1)])
def test_head_layouts(ctx, dev, src, dst, n_q, n_kv):
    b = Batch(dev, src, dst, n_q, n_kv, 128, 500, 100, [1, 7, 2, 1], [33, 100, 60, 1], seed=n_q)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("src,dst", [("bf16", "f32"), ("f16", "f16")])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("counts,lens", [([300], [300]), ([130, 70, 257], [500, 70, 260]), ([64] * 6, [64, 99, 512, 65, 300, 130])])
def test_prompts(ctx, dev, src, dst, hd, causal, counts, lens):
    """Many query rows a sequence: several row tiles, causal limits inside tiles."""
    b = Batch(dev, src, dst, 8, 2, hd, 700, 512, counts, lens, seed=len(counts))
    b.run(ctx, causal)
    b.check(causal)


@pytest.mark.parametrize("src,dst", [("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("prefix", [0, 200])
def test_rows_that_see_little_or_nothing(ctx, dev, src, dst, prefix):
    """More query rows than own keys (the first see only the prefix, or nothing), empty sequences, rows of none."""
    b = Batch(dev, src, dst, 4, 2, 64, prefix, 30, [5, 0, 3, 1, 0, 4], [2, 9, 0, 1, 0, 30], extra=3, seed=5)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("prefix,cap", [(0, 0), (70, 0)])
def test_no_own_part(ctx, dev, prefix, cap):
    b = Batch(dev, "bf16", "f32", 4, 4, 64, prefix, cap, [1, 2, 1], [0, 0, 0], extra=1)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("src,dst", TYPES)
def test_strides(ctx, dev, src, dst):
    b = Batch(dev, src, dst, 8, 2, 64, 333, 77, [2, 1, 5], [77, 20, 5], extra=2, gap=24, seed=9)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("src,dst", TYPES)
def test_peaked_scores(ctx, dev, src, dst):
    """Scores of +-200: maxima that grow by far more than the rescaling threshold, tile after tile."""
    import torch

    b = Batch(dev, src, dst, 8, 2, 128, 1500, 300, [1, 2, 1, 4], [300, 150, 1, 40], seed=11, spread=4.0)
    order = (b.q[0, :128].float() @ b.kp[:, :128].float().T).argsort()
    b.kp[:] = b.kp[order].clone()
    assert torch.isfinite(b.kp).all()
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("lens", [[-5, 1000, 40], [2 ** 31 - 1, -(2 ** 31), 0]])
def test_lengths_outside_the_cache_are_held_inside(ctx, dev, lens):
    b = Batch(dev, "bf16", "f32", 4, 2, 64, 150, 60, [1, 1, 2], lens)
    b.run(ctx)
    b.check()


def test_starts_outside_the_rows_stay_in_bounds(ctx, dev):
    """Starts that run backwards or past the rows: which rows are computed is not said, the guard rows stay."""
    import torch

    b = Batch(dev, "bf16", "f32", 4, 2, 64, 150, 60, [2, 2, 2], [5, 6, 7])
    guard = torch.full((3 * b.rows, b.out.shape[1]), 77.0, device=dev)
    b.out = guard[b.rows:2 * b.rows]
    b.seq_start.copy_(torch.tensor([-7, 5, 2, 2 ** 31 - 1], dtype=torch.int32))
    b.run(ctx)
    torch.cuda.synchronize()
    assert (guard[:b.rows] == 77.0).all() and (guard[2 * b.rows:] == 77.0).all()
    ctx.device_status()


def test_one_sequence_agrees_with_mha_attn(ctx, dev):
    """One sequence whose cache is cut into prefix and own part against lc_mha_attn on the joined f32 rows."""
    import torch

    b = Batch(dev, "f16", "f32", 8, 2, 128, 200, 56, [16], [56], garbage=False)
    b.run(ctx)
    k = torch.cat([b.kp, b.ko[0]]).float().contiguous()
    v = torch.cat([b.vp, b.vo[0]]).float().contiguous()
    out = torch.empty(16, 8 * 128, device=dev)
    ctx.mha_attn(b.q.float().contiguous(), k, v, out, 16, 8, 2, 128, 256, b.scale, 240, 1)
    torch.cuda.synchronize()
    b.check()
    # both are within the derived bound of the exact value (lc_mha_attn keeps 22 bits of each factor)
    assert (out - b.out).abs().max() <= 2e-5 * out.abs().max()


def test_long_prefix(ctx, dev):
    """Many key splits (more than a warp's lanes in the merge) and many row tiles at once."""
    b = Batch(dev, "bf16", "bf16", 8, 1, 64, 40001, 200, [1] * 40, [(7 * i) % 200 + 1 for i in range(40)], seed=3)
    b.run(ctx)
    b.check()
    b = Batch(dev, "bf16", "f32", 2, 1, 128, 40001, 4000, [1], [3999], seed=4)
    b.run(ctx)
    b.check()


def test_offsets_past_32_bits(ctx, dev):
    """A cache whose last sequence starts past 2^32 elements."""
    import torch

    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 18 GB")
    b = Batch(dev, "bf16", "f32", 4, 2, 64, 90, 20, [1, 2, 1], [20, 11, 3])
    far = (1 << 31) + 64
    for name in ("ko", "vo"):
        big = torch.empty(2 * far + 20 * 128, device=dev, dtype=torch.bfloat16)
        view = torch.as_strided(big, (3, 20, 128), (far, 128, 1))
        view.copy_(getattr(b, name))
        setattr(b, name, view)
    b.run(ctx)
    b.check()


def test_graphs_grow_and_share_the_scratch(ctx, dev):
    """Two captured calls on one context, replayed in turn as lengths grow, with a larger eager call between
    (the scratch they hold must outlive its growth); capture before any call of the size is refused."""
    import torch

    c = lc.Context(0)
    s = torch.cuda.Stream()
    c.set_stream(s)
    a = Batch(dev, "bf16", "f32", 8, 2, 64, 400, 64, [1] * 5, [3, 9, 27, 40, 1], seed=1, garbage=False)
    b = Batch(dev, "f16", "f16", 8, 2, 128, 900, 64, [2] * 3, [5, 9, 60], seed=2, garbage=False)
    big = Batch(dev, "bf16", "bf16", 32, 8, 128, 3000, 300, [1] * 70, [100] * 70, seed=3)
    torch.cuda.synchronize()
    fresh = lc.Context(0)
    fresh.set_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        with pytest.raises(lc.LagunaError) as e:
            a.run(fresh)
    assert e.value.status == lc.LC_ERR_UNSUPPORTED and "capture" in str(e.value)
    del graph
    fresh.close()
    graphs = []
    for x in (a, b):
        x.run(c)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            x.run(c)
        graphs.append(g)
    for step in range(3):
        for x, g in zip((a, b), graphs):
            x.own_len += 1
            x.lens = [v + 1 for v in x.lens]
            x.out.fill_(77.0)
            torch.cuda.synchronize()
            with torch.cuda.stream(s):
                g.replay()
            torch.cuda.synchronize()
            x.check()
        if step == 0:
            big.run(c)
            torch.cuda.synchronize()
            big.check()
    del graphs, g
    c.close()


def test_repeats_bit_for_bit(ctx, dev):
    import torch

    b = Batch(dev, "bf16", "f32", 8, 2, 128, 3000, 200, [1] * 20, [(13 * i) % 200 + 1 for i in range(20)])
    b.run(ctx)
    torch.cuda.synchronize()
    first = b.out.clone()
    for _ in range(5):
        b.run(ctx)
    torch.cuda.synchronize()
    assert torch.equal(first, b.out)


@pytest.mark.parametrize("src", ["bf16", "f16"])
@pytest.mark.parametrize("n_q,n_kv,hd,counts,lens,prefix,cap", [
    (8, 2, 64, [343, 262, 393], [396, 262, 393], 5884, 431),     # states of many tiles
    (32, 8, 128, [343, 262, 393, 500], [396, 262, 393, 500], 1500, 512),  # rows written out by whole items
])
def test_long_sums_keep_their_digits(ctx, dev, src, n_q, n_kv, hd, counts, lens, prefix, cap):
    """f32 outputs: the tensor cores drop what lies below a sum's last bit, 2^-24 of it on the average, and at
    most 48 products (4 tiles of 64 keys, 16 at a time, in 3 planes) are summed there; scores, exponentials and
    planes of the weights add up to 4 times 2^-22.  All of the result's norm."""
    import torch

    b = Batch(dev, src, "f32", n_q, n_kv, hd, prefix, cap, counts, lens, seed=4)
    b.run(ctx)
    torch.cuda.synchronize()
    at, err, norm = 0, 0.0, 0.0
    for i, (c, length) in enumerate(zip(counts, lens)):
        k = torch.cat([b.kp[:prefix], b.ko[i, :length]]).double().view(-1, n_kv, hd)
        v = torch.cat([b.vp[:prefix], b.vo[i, :length]]).double().view(-1, n_kv, hd)
        hidden = torch.ones(c, length, dtype=torch.bool, device=dev).triu(length - c + 1)
        hidden = torch.cat([torch.zeros(c, prefix, dtype=torch.bool, device=dev), hidden], 1)
        for h in range(n_kv):
            group = n_q // n_kv
            q = b.q[at:at + c].double().view(c, n_kv, group, hd)[:, h]
            s = torch.einsum("rgd,kd->grk", q, k[:, h]) * b.scale
            o = torch.einsum("grk,kd->rgd", s.masked_fill(hidden, -math.inf).softmax(-1), v[:, h])
            got = b.out[at:at + c].double().view(c, n_kv, group, hd)[:, h]
            err, norm = err + float((got - o).square().sum()), norm + float(o.square().sum())
        at += c
    assert math.sqrt(err / norm) <= 48 * 2.0 ** -24 + 4 * 2.0 ** -22


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("n_q,n_kv,hd,prefix,cap,counts,lens", [
    (4, 1, 64, 10581, 206, [1], [200]), (2, 2, 128, 13851, 7, [1, 0, 1], [7, 3, 1]), (1, 1, 64, 0, 9000, [3], [8999]),
    (6, 2, 128, 700, 0, [1, 2], [0, 0])])
def test_few_rows_on_many_keys(ctx, dev, src, dst, n_q, n_kv, hd, prefix, cap, counts, lens):
    """Many states of a few rows, merged by several warps together; rows of no sequence among them."""
    b = Batch(dev, src, dst, n_q, n_kv, hd, prefix, cap, counts, lens, seed=6, extra=3)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("dst", ["f16", "f32"])
@pytest.mark.parametrize("hd,prefix,cap,counts,peak,second", [
    (64, 16384, 20, [1], 17.0, 0.0),          # few rows, many states
    (128, 4096, 100, [1, 1, 1], 12.0, 5.5),   # a later key of 2^7.9 times the first one's weight
    (64, 32768, 5, [1] * 40, 12.0, 0.0),
    (64, 0, 9000, [3], 15.0, 5.5),
    (128, 5000, 300, [300], 14.0, 0.0),       # whole row tiles
])
def test_a_dominant_first_key_keeps_the_others(ctx, dev, dst, hd, prefix, cap, counts, peak, second):
    """f16 keys, the first of them `peak` nats above the rest and with values of 0: the result is what the many small
    weights add up to.  Weights lie at 2^7 or more where the row's largest is, so that a subnormal one (spacing 2^-24) is
    off by at most 2^-25 of that scale, 2^-32 of the largest weight; else as above.  `second`: nats by which the last
    prefix (or own) key exceeds the first."""
    import torch

    n_q, n_kv = 4, 2
    lens = [cap] * len(counts)
    b = Batch(dev, "f16", dst, n_q, n_kv, hd, prefix, cap, counts, lens, seed=prefix + cap, garbage=False)
    b.q.view(-1, n_q, hd)[:, :, 0] = 8.0
    for x in (b.kp, b.ko):
        x.view(-1, n_kv, hd)[:, :, 0] = 0.0
    for x in (b.vp, b.vo):
        x.copy_((1 + 0.5 * x.float()).half())
    k, v = (b.kp, b.vp) if prefix else (b.ko[0], b.vo[0])
    step = math.sqrt(hd) / 8
    k.view(-1, n_kv, hd)[0, :, 0] = peak * step
    v[0] = 0.0
    if second:
        k.view(-1, n_kv, hd)[len(k) - sum(counts) - 1, :, 0] = (peak + second) * step
        v[len(k) - sum(counts) - 1] = 0.0
    b.run(ctx)
    torch.cuda.synchronize()
    at = 0
    for i, c in enumerate(counts):
        n = prefix + cap
        key, reach = torch.arange(n, device=dev), torch.arange(c, device=dev) + cap - c
        seen = (key < prefix) | (key - prefix <= reach[:, None])
        for h in range(n_kv):
            kk = torch.cat([b.kp[:prefix], b.ko[i]]).double().view(n, n_kv, hd)[:, h]
            vv = torch.cat([b.vp[:prefix], b.vo[i]]).double().view(n, n_kv, hd)[:, h]
            q = b.q[at:at + c].double().view(c, n_q, hd)[:, 2 * h:2 * h + 2]
            s = torch.einsum("rgd,kd->grk", q, kk) * b.scale
            mag = torch.einsum("rgd,kd->grk", q.abs(), kk.abs()) * b.scale
            s = s.masked_fill(~seen, -math.inf)
            w = (s - s.amax(-1, keepdim=True)).exp()
            total = w.sum(-1, keepdim=True)
            o, a = (w @ vv) / total, (w @ vv.abs()) / total
            flat = (seen.double() @ vv.abs()) / total
            err_s = ((hd + 2) * 2.0 ** -24 * mag * seen).amax(-1, keepdim=True)
            tol = a * (2 * (err_s * 1.01 + 2.0 ** -22 + (math.sqrt(n) + 64) * 2.0 ** -24) +
                       (2.0 ** -22 if dst == "f32" else 2.0 ** -11)) + flat * 2.0 ** -32
            fo = torch.finfo(tt(dst))
            tol = tol * 1.001 + o.abs() * fo.eps / 2 + fo.smallest_normal * fo.eps
            got = b.out[at:at + c].double().view(c, n_q, hd)[:, 2 * h:2 * h + 2].transpose(0, 1)
            err = (got - o).abs()
            assert (err <= tol).all(), (i, h, float((err / o.abs()).max()), float((tol / o.abs()).max()))
        at += c


def busy_batches(dev):
    """Two batches that keep the GPU some tens of microseconds, with many states each, and their results."""
    import torch

    a = Batch(dev, "bf16", "f32", 8, 2, 128, 6000, 300, [1] * 24, [(29 * i) % 300 + 1 for i in range(24)], seed=21)
    b = Batch(dev, "f16", "f16", 16, 4, 64, 9000, 200, [2] * 17, [(31 * i) % 199 + 2 for i in range(17)], seed=22)
    c = lc.Context(0)
    for x in (a, b):
        c.set_stream(torch.cuda.current_stream())
        x.run(c)
        x.check()
    c.close()
    return a, b, a.out.clone(), b.out.clone()


def test_streams_of_one_context_at_the_same_time(ctx, dev):
    """Calls of one context in turn on two streams that nothing orders: neither meets the other's states."""
    import torch

    a, b, want_a, want_b = busy_batches(dev)
    c, streams = lc.Context(0), [torch.cuda.Stream() for _ in range(2)]
    for x in (a, b):
        x.out.fill_(77.0)
    torch.cuda.synchronize()
    outs = []
    for _ in range(20):
        for x, s in zip((a, b), streams):
            c.set_stream(s)
            x.run(c)
            with torch.cuda.stream(s):
                outs.append((x, x.out.clone()))
    torch.cuda.synchronize()
    assert all(torch.equal(got, want_a if x is a else want_b) for x, got in outs)
    c.device_status()
    c.close()


def test_graphs_of_one_context_at_the_same_time(ctx, dev):
    """Two graphs captured on one stream of one context, replayed on two streams beside eager calls on a third."""
    import torch

    a, b, want_a, want_b = busy_batches(dev)
    e = Batch(dev, "bf16", "bf16", 8, 8, 64, 5000, 100, [1] * 30, [50] * 30, seed=23)
    c, streams = lc.Context(0), [torch.cuda.Stream() for _ in range(4)]
    c.set_stream(streams[3])
    e.run(c)
    e.check()
    want_e, graphs = e.out.clone(), []
    for x in (a, b):
        x.out.fill_(77.0)
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=streams[3]):
            for _ in range(3):
                x.run(c)
        graphs.append(g)
    for _ in range(10):
        for x, g, s in zip((a, b), graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        c.set_stream(streams[2])
        e.run(c)
    torch.cuda.synchronize()
    assert torch.equal(a.out, want_a) and torch.equal(b.out, want_b) and torch.equal(e.out, want_e)
    c.device_status()
    del graphs, g
    c.close()


def test_capture_after_a_call_that_needed_no_scratch(ctx, dev):
    """A large prompt is written out by whole items, a single row needs states: captured all the same."""
    import torch

    big = Batch(dev, "bf16", "bf16", 32, 8, 128, 1024, 2048, [2048], [2048], seed=31, garbage=False)
    one = Batch(dev, "bf16", "bf16", 32, 8, 128, 8192, 64, [1], [9], seed=32)
    c, s = lc.Context(0), torch.cuda.Stream()
    c.set_stream(s)
    torch.cuda.synchronize()
    big.run(c)
    torch.cuda.synchronize()
    assert c.scratch_bytes() == 0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        one.run(c)
    g.replay()
    one.check()
    del g
    c.close()


def test_captured_scratch_is_used_again(ctx, dev):
    """The scratch of a destroyed graph goes to the next one."""
    import gc
    import time

    import torch

    b = Batch(dev, "f16", "f32", 8, 2, 64, 3000, 64, [1] * 5, [3, 9, 27, 40, 1], seed=33)
    c, s = lc.Context(0), torch.cuda.Stream()
    c.set_stream(s)
    torch.cuda.synchronize()
    b.run(c)
    torch.cuda.synchronize()
    held = []
    for _ in range(6):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.run(c)
            b.run(c)
        b.out.fill_(77.0)
        torch.cuda.synchronize()
        g.replay()
        b.check()
        held.append(c.scratch_bytes())
        del g
        gc.collect()
        time.sleep(0.05)  # the release comes from a thread of the driver
    assert held[0] == held[-1], held
    c.close()


@pytest.mark.parametrize("src,dst", TYPES)
def test_one_long_prompt_beside_single_tokens(ctx, dev, src, dst):
    """Rows by the mean fill tiles, so that every sequence runs over the whole axis; the long one goes round."""
    b = Batch(dev, src, dst, 8, 2, 64, 300, 1000, [1, 900, 1, 1, 0, 1], [5, 950, 1000, 1, 7, 64], seed=41, extra=2)
    b.run(ctx)
    b.check()
    ctx.device_status()


def test_context_closed_before_its_graph(ctx, dev):
    """The graph is not replayed any more; that it goes later must not touch what the context freed."""
    import gc
    import time

    import torch

    b = Batch(dev, "bf16", "f32", 8, 2, 64, 3000, 64, [1] * 5, [3, 9, 27, 40, 1], seed=42)
    c, s = lc.Context(0), torch.cuda.Stream()
    c.set_stream(s)
    torch.cuda.synchronize()
    b.run(c)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        b.run(c)
    c.close()
    del g
    gc.collect()
    time.sleep(0.05)
    b.run(ctx)
    b.check()


@pytest.mark.parametrize("src,dst", TYPES)
@pytest.mark.parametrize("prefix,cap,counts,lens", [(500, 60, [3, 1, 20], [60, 9, 33]), (0, 300, [200], [300]),
                                                    (4000, 20, [1] * 12, [20] * 12)])
def test_without_the_causal_limit_at_any_stride(ctx, dev, src, dst, prefix, cap, counts, lens):
    b = Batch(dev, src, dst, 8, 4, 64, prefix, cap, counts, lens, seed=43, extra=1, gap=40)
    b.run(ctx, causal=0)
    b.check(causal=0)
