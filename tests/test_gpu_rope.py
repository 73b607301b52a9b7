"""lc_rope on the GPU against the rotation in 64 bits.

Error of one output value: the reduced angle is rounded to f32 (|a| <= pi: at
most 2^-23), sincosf is off by at most 2 ulp (2^-23), the scaled table value, the
two products and the sum are each rounded (4 * 2^-24): 8 * 2^-24 of
scale (|x1| + |x2|).  A 16-bit output adds half a step of the value."""
import numpy as np
import pytest

from laguna_raw_halo_strix_b200 import lc

pytestmark = pytest.mark.gpu

TYPES = {"f32": lc.F32, "f16": lc.F16, "bf16": lc.BF16}


def torch_type(t):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[t]


def reference(x, pos, freq, heads, hd, rd, pairs, scale):
    """x [m, heads * hd] in 64 bits -> (rotated, |x1| + |x2| of each output's pair)."""
    m = x.shape[0]
    x = x.reshape(m, heads, hd)
    y, mag = x.copy(), np.abs(x)
    a = pos.astype(np.float64)[:, None] * freq.astype(np.float64)
    c, s = scale * np.cos(a)[:, None], scale * np.sin(a)[:, None]
    i1 = np.arange(0, rd, 2) if pairs else np.arange(rd // 2)
    i2 = i1 + 1 if pairs else i1 + rd // 2
    y[..., i1] = x[..., i1] * c - x[..., i2] * s
    y[..., i2] = x[..., i2] * c + x[..., i1] * s
    mag[..., i1] = mag[..., i2] = scale * (np.abs(x[..., i1]) + np.abs(x[..., i2]))
    return y.reshape(m, -1), mag.reshape(m, -1)


def within(got, ref, mag, dst):
    import torch

    fi = torch.finfo(torch_type(dst))
    half_step = np.abs(ref) * fi.eps / 2 + fi.smallest_normal * fi.eps / 2 if dst != "f32" else 0.0
    err = np.abs(got.double().cpu().numpy() - ref)
    tol = mag * 8 * 2.0 ** -24 + half_step * (1 + 2.0 ** -10)
    assert (err <= tol).all(), float((err - tol).max())


@pytest.mark.parametrize("m,n_q,n_kv,hd,rd", [(1, 1, 0, 2, 2), (1, 32, 8, 128, 128), (16, 32, 8, 128, 128),
                                              (7, 3, 1, 80, 40), (5, 2, 2, 10, 6), (3, 4, 4, 64, 0),
                                              (33, 0, 2, 96, 48), (400, 6, 2, 64, 32), (2, 71, 1, 256, 256)])
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"),
                                     ("f16", "f16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("pairs", [False, True])
def test_against_64_bits(ctx, dev, m, n_q, n_kv, hd, rd, src, dst, pairs):
    import torch

    g = torch.Generator(dev).manual_seed(m * 100 + hd)
    freq = torch.from_numpy(lc.rope_freq(max(rd, 2), 500000.0)).to(dev)
    pos = torch.randint(-(2 ** 31), 2 ** 31 - 1, (m,), generator=g, device=dev).to(torch.int32)
    x = [torch.randn(m, h * hd, generator=g, device=dev).to(torch_type(src)) for h in (n_q, n_kv)]
    y = [torch.full((m, h * hd), float("nan"), device=dev, dtype=torch_type(dst)) for h in (n_q, n_kv)]
    ctx.rope(TYPES[src], TYPES[dst], int(pairs), x[0], y[0], n_q, x[1], y[1], n_kv, pos, freq, m, hd, rd, 1.25)
    torch.cuda.synchronize()
    for xi, yi, h in zip(x, y, (n_q, n_kv)):
        if h:
            ref, mag = reference(xi.double().cpu().numpy(), pos.cpu().numpy(), freq.cpu().numpy(), h, hd, rd, pairs,
                                 1.25)
            within(yi, ref, mag, dst)


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides_and_alignment_fused_in_place(ctx, dev, pairs, offset, t):
    """q, k, v columns of one buffer at odd offsets, rotated in place: v, the padding and the copied dims stay."""
    import torch

    m, n_q, n_kv, hd, rd, ld = 9, 4, 2, 48, 32, 48 * 8 + 13
    buf = torch.randn(m * ld + 8, device=dev).to(torch_type(t))
    before = buf.clone()
    rows = torch.as_strided(buf, (m, ld), (ld, 1), offset)
    q, k = rows[:, :n_q * hd], rows[:, n_q * hd:(n_q + n_kv) * hd]
    freq = torch.from_numpy(lc.rope_freq(rd, 10000.0)).to(dev)
    pos = torch.arange(1000, 1000 + m, device=dev, dtype=torch.int32)
    ctx.rope(TYPES[t], TYPES[t], int(pairs), q, q, n_q, k, k, n_kv, pos, freq, m, hd, rd, ldq=ld, ldq_out=ld, ldk=ld,
             ldk_out=ld)
    torch.cuda.synchronize()
    old = torch.as_strided(before, (m, ld), (ld, 1), offset)
    for a, b, h in ((q, old[:, :n_q * hd], n_q), (k, old[:, n_q * hd:(n_q + n_kv) * hd], n_kv)):
        ref, mag = reference(b.double().cpu().numpy(), pos.cpu().numpy(), freq.cpu().numpy(), h, hd, rd, pairs, 1.0)
        within(a, ref, mag, t)
        kept = torch.tensor([d % hd >= rd for d in range(h * hd)], device=dev)
        assert torch.equal(a[:, kept], b[:, kept])
    rest = torch.ones(m * ld + 8, dtype=torch.bool, device=dev)
    torch.as_strided(rest, (m, ld), (ld, 1), offset)[:, :(n_q + n_kv) * hd] = False
    assert torch.equal(buf[rest], before[rest])


def test_minus_pos_undoes_pos(ctx, dev):
    import torch

    m, h, hd = 64, 4, 128
    x = torch.randn(m, h * hd, device=dev)
    freq, scale = lc.rope_freq_scaled(hd, 500000.0, lc.ROPE_SCALE_YARN, 8.0, 4096)
    freq = torch.from_numpy(freq).to(dev)
    pos = torch.randint(0, 1 << 20, (m,), device=dev, dtype=torch.int32)
    y, z = torch.empty_like(x), torch.empty_like(x)
    ctx.rope(lc.F32, lc.F32, lc.ROPE_HALF, x, y, h, None, None, 0, pos, freq, m, hd, hd, scale)
    ctx.rope(lc.F32, lc.F32, lc.ROPE_HALF, y, z, h, None, None, 0, -pos, freq, m, hd, hd, 1 / scale)
    torch.cuda.synchronize()
    # two rotations, each within 8 * 2^-24 (|x1| + |x2|), the second on values up to sqrt(2) scale larger
    mag = x.abs().view(m, h, 2, hd // 2).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(m, -1)
    assert ((z - x).abs() <= (8 + 16 * 1.5 + 2) * 2.0 ** -24 * mag).all()


def test_agrees_with_qk_norm_rope_at_small_positions(ctx, dev):
    """With a weight that undoes nothing (rows of unit mean square) both rotate alike."""
    import torch

    m, h, hd = 16, 8, 128
    x = torch.randn(m, h * hd, device=dev)
    x = (x.view(m, h, hd) / x.view(m, h, hd).square().mean(-1, keepdim=True).sqrt()).reshape(m, -1).contiguous()
    freq = torch.from_numpy(lc.rope_freq(hd)).to(dev)
    a, b = torch.empty_like(x), torch.empty_like(x)
    ctx.qk_norm_rope(x, torch.ones(hd, device=dev), freq, a, m, h, hd, hd, 0.0, 3)
    ctx.rope(lc.F32, lc.F32, lc.ROPE_HALF, x, b, h, None, None, 0,
             torch.arange(3, 3 + m, device=dev, dtype=torch.int32), freq, m, hd, hd)
    torch.cuda.synchronize()
    # angles below 19: 19 * 2^-24 from the f32 product there, the norm (3 * 2^-24) and both rotations
    mag = x.abs().view(m, h, 2, hd // 2).sum(2, keepdim=True).expand(-1, -1, 2, -1).reshape(m, -1)
    assert ((a - b).abs() <= (19 + 8 + 8 + 16) * 2.0 ** -24 * mag).all()


def test_other_stream_and_graph(ctx, dev):
    import torch

    m, h, hd = 40, 4, 64
    x = torch.randn(m, h * hd, device=dev)
    freq = torch.from_numpy(lc.rope_freq(hd)).to(dev)
    pos = torch.arange(m, device=dev, dtype=torch.int32)
    ref, y = torch.empty_like(x), torch.zeros_like(x)
    ctx.rope(lc.F32, lc.F32, lc.ROPE_PAIRS, x, ref, h, None, None, 0, pos, freq, m, hd, hd)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    c = lc.Context(0)
    c.set_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        c.rope(lc.F32, lc.F32, lc.ROPE_PAIRS, x, y, h, None, None, 0, pos, freq, m, hd, hd)
    pos += 5  # a replay reads what the buffers hold then
    graph.replay()
    torch.cuda.synchronize()
    ctx.rope(lc.F32, lc.F32, lc.ROPE_PAIRS, x, ref, h, None, None, 0, pos, freq, m, hd, hd)
    torch.cuda.synchronize()
    assert torch.equal(y, ref)
    del graph
    c.close()


def test_offsets_past_32_bits(ctx, dev):
    """Rows so far apart that the last one starts past 2^32 elements."""
    import torch

    m, hd, ld = 3, 64, (1 << 31) + 8
    if torch.cuda.mem_get_info()[0] < 20 << 30:
        pytest.skip("needs 9 GB")
    buf = torch.zeros(2 * ld + hd, device=dev, dtype=torch.bfloat16)
    rows = torch.as_strided(buf, (m, hd), (ld, 1))
    rows.copy_(torch.randn(m, hd, device=dev))
    x = rows.double().cpu().numpy()
    freq = torch.from_numpy(lc.rope_freq(hd)).to(dev)
    pos = torch.tensor([5, 70000, 2 ** 31 - 1], device=dev, dtype=torch.int32)
    ctx.rope(lc.BF16, lc.BF16, lc.ROPE_HALF, rows, rows, 1, None, None, 0, pos, freq, m, hd, hd, ldq=ld, ldq_out=ld)
    torch.cuda.synchronize()
    ref, mag = reference(x, pos.cpu().numpy(), freq.cpu().numpy(), 1, hd, hd, False, 1.0)
    within(rows, ref, mag, "bf16")


@pytest.mark.parametrize("m,n_q,n_kv,hd,rd", [(5, 1, 1, 1022, 1022), (700, 3, 1, 600, 598), (2, 2, 1, 8192, 8192),
                                              (1500, 1, 0, 4, 2), (650, 5, 0, 254, 10), (3, 300, 7, 6, 4)])
@pytest.mark.parametrize("src,dst", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f32")])
@pytest.mark.parametrize("pairs", [False, True])
def test_items_and_threads_that_do_not_divide(ctx, dev, m, n_q, n_kv, hd, rd, src, dst, pairs):
    """Heads of more pieces than a CTA has threads, and few pieces with threads left over."""
    test_against_64_bits(ctx, dev, m, n_q, n_kv, hd, rd, src, dst, pairs)


def test_first_call_of_a_process_captured():
    """Neither lc_rope nor lc_logits_process needs a call before its capture."""
    import os
    import subprocess
    import sys

    code = """
import torch
from laguna_raw_halo_strix_b200 import lc
d = torch.device("cuda", 0)
x = torch.randn(2, 128, device=d); y = torch.zeros_like(x); l = torch.randn(3, 5000, device=d)
big = torch.randn(500, 5000, device=d)
pos = torch.arange(2, dtype=torch.int32, device=d); freq = torch.from_numpy(lc.rope_freq(64)).to(d)
keys, all_keys = torch.zeros(3, dtype=torch.int64, device=d), torch.zeros(500, dtype=torch.int64, device=d)
s = torch.cuda.Stream(); ctx = lc.Context(0); ctx.set_stream(s); g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g, stream=s):
    ctx.rope(lc.F32, lc.F32, lc.ROPE_HALF, x, y, 2, None, None, 0, pos, freq, 2, 64, 64)
    ctx.logits_process(l, lc.LogitsRules(), None, keys, 3, 5000)
    ctx.logits_process(big, lc.LogitsRules(), None, all_keys, 500, 5000)
g.replay(); torch.cuda.synchronize()
assert torch.equal(y[0], x[0]) and not torch.equal(y[1], x[1])
assert [lc.key_index(int(k)) for k in keys] == l.argmax(1).tolist()
assert [lc.key_index(int(k)) for k in all_keys] == big.argmax(1).tolist()
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


PI = 3141592653589793238462643383279502884197169399375105820974944592307816406286208999


def turned_past(pos, freq):
    """(how far the exact angle pos * freq is past the nearest multiple of pi, whether that is an odd one)."""
    from fractions import Fraction

    pi = Fraction(PI, 10 ** 81)
    a = Fraction(int(pos)) * Fraction(float(freq))
    k = round(a / pi)
    return float(a - k * pi), k % 2


@pytest.mark.parametrize("far", [131072, 2 ** 31 - 1])
@pytest.mark.parametrize("pairs", [False, True])
def test_angles_next_to_multiples_of_pi(ctx, dev, far, pairs):
    """Where the sine is small its value shows the angle's absolute error.  x = (1, 0) gives (cos a, sin a): the sine
    within 2 ulp of the function (2^-22), its correction and the angle's rounding (2^-23 each) of the value, and
    2^-50 for the reduction in 64 bits."""
    import torch

    rng = np.random.default_rng(far)
    f = rng.uniform(0.25, 1.0, 400000).astype(np.float32)
    p = rng.integers(far // 2, far, f.size)
    p *= rng.choice([-1, 1], f.size)
    turns = p.astype(np.longdouble) * f.astype(np.longdouble) / (np.longdouble(PI // 10 ** 63) / np.longdouble(10) ** 18)
    near = np.argsort(np.abs(turns - np.rint(turns)))[:64]
    f, p = f[near], p[near]
    half = near.size
    x = torch.zeros(half, 2 * half, device=dev)
    (x[:, 0::2] if pairs else x[:, :half]).fill_(1.0)
    y = torch.empty_like(x)
    ctx.rope(lc.F32, lc.F32, int(pairs), x, y, 1, None, None, 0, torch.from_numpy(p.astype(np.int32)).to(dev),
             torch.from_numpy(f).to(dev), half, 2 * half, 2 * half)
    torch.cuda.synchronize()
    got = y.cpu().numpy().astype(np.float64)
    cos, sin = (got[:, 0::2], got[:, 1::2]) if pairs else (got[:, :half], got[:, half:])
    odd_ones = 0
    for i in range(half):  # row i's pair i
        past, odd = turned_past(p[i], f[i])
        assert abs(past) < 1e-3
        want = -np.sin(past) if odd else np.sin(past)
        assert abs(sin[i, i] - want) <= abs(want) * 2.0 ** -21 + 2.0 ** -50, (i, sin[i, i], want, odd)
        assert abs(cos[i, i] - (-np.cos(past) if odd else np.cos(past))) <= 2.0 ** -22
        odd_ones += odd
    assert 0 < odd_ones < half
