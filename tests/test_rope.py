"""lc_rope and lc_rope_freq_scaled without a GPU: the frequency tables against
their formulas in 64 bits, and every refusal.  lc_rope decides them from its
arguments alone, before it looks into the context, so a blank one will do."""
import ctypes as C
import math

import numpy as np
import pytest

from laguna_raw_halo_strix_b200 import lc


def table64(dim, base, kind, factor, orig, fast, slow):
    """Frequencies and scale from the definition, one pair at a time."""
    out = []
    for i in range(dim // 2):
        b = base * factor ** (dim / (dim - 2)) if kind == lc.ROPE_SCALE_NTK else base
        w = b ** (-2 * i / dim)
        if kind == lc.ROPE_SCALE_LINEAR:
            w /= factor
        if kind == lc.ROPE_SCALE_YARN:
            # dimension whose wavelength 2 pi base^(2j/dim) fits n times into orig
            j = [dim * math.log(orig / (n * 2 * math.pi)) / (2 * math.log(base)) for n in (fast, slow)]
            lo, hi = max(math.floor(j[0]), 0), min(math.ceil(j[1]), dim - 1)
            t = min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0)
            w = w / factor * t + w * (1 - t)
        out.append(w)
    return np.array(out), 0.1 * math.log(factor) + 1 if kind == lc.ROPE_SCALE_YARN else 1.0


@pytest.mark.parametrize("dim,base", [(2, 10000.0), (64, 10000.0), (96, 500000.0), (128, 500000.0)])
@pytest.mark.parametrize("kind", [lc.ROPE_SCALE_NONE, lc.ROPE_SCALE_LINEAR, lc.ROPE_SCALE_NTK, lc.ROPE_SCALE_YARN])
@pytest.mark.parametrize("factor", [1.0, 4.0, 32.0])
def test_freq_tables(dim, base, kind, factor):
    if kind == lc.ROPE_SCALE_NTK and dim == 2:  # d / (d - 2)
        with pytest.raises(lc.LagunaError):
            lc.rope_freq_scaled(dim, base, kind, factor)
        return
    f, scale = lc.rope_freq_scaled(dim, base, kind, factor, 4096, 32.0, 1.0)
    ref, ref_scale = table64(dim, base, kind, factor, 4096, 32.0, 1.0)
    # one rounding to f32 (2^-24) and a few of 2^-53 before it
    assert np.abs(f / ref - 1).max() <= 2.0 ** -24 * 1.001
    assert abs(scale / ref_scale - 1) <= 2.0 ** -24 * 1.001


def test_none_agrees_with_the_plain_table():
    f, scale = lc.rope_freq_scaled(128, 500000.0)
    # lc_rope_freq forms powf, a reciprocal and 2i/d in f32: ln(base) * 2^-24 from
    # the exponent's rounding (13.2), 2 ulp of powf and one of the division
    assert np.abs(f / lc.rope_freq(128, 500000.0) - 1).max() <= (13.2 + 4) * 2.0 ** -24
    assert scale == 1.0


@pytest.mark.parametrize("args", [
    (127, 1e4, 0, 1.0, 0, 32.0, 1.0), (128, 1.0, 0, 1.0, 0, 32.0, 1.0), (128, float("nan"), 0, 1.0, 0, 32.0, 1.0),
    (128, 1e4, 4, 1.0, 0, 32.0, 1.0), (128, 1e4, -1, 1.0, 0, 32.0, 1.0), (128, 1e4, 1, 0.5, 0, 32.0, 1.0),
    (128, 1e4, 1, float("nan"), 0, 32.0, 1.0), (2, 1e4, 2, 2.0, 0, 32.0, 1.0), (128, 1e4, 3, 2.0, 0, 32.0, 1.0),
    (128, 1e4, 3, 2.0, 4096, 1.0, 32.0), (128, 1e4, 3, 2.0, 4096, 32.0, 0.0)])
def test_freq_refusals(args):
    with pytest.raises(lc.LagunaError) as e:
        lc.rope_freq_scaled(*args)
    assert e.value.status == lc.LC_ERR_INVALID


BLANK = C.create_string_buffer(4096)  # stands for an lc_ctx


def call(**over):
    a = dict(dtype=lc.F32, out_dtype=lc.F32, layout=lc.ROPE_HALF, q=0x10000, ldq=0, q_out=0x20000, ldq_out=0, n_q=2,
             k=0x30000, ldk=0, k_out=0x40000, ldk_out=0, n_kv=1, pos=0x50000, freq=0x60000, m=4, head_dim=64,
             rope_dim=64, scale=1.0)
    a.update(over)
    return lc.lib().lc_rope(C.cast(BLANK, C.c_void_p), *a.values())


INVALID = [
    dict(layout=2), dict(layout=-1), dict(head_dim=63, rope_dim=62), dict(head_dim=0, rope_dim=0), dict(rope_dim=33),
    dict(rope_dim=66), dict(q=None), dict(q_out=None), dict(k=None), dict(k_out=None), dict(pos=None), dict(freq=None),
    dict(ldq=127), dict(ldq_out=127), dict(ldk=63), dict(ldk_out=63), dict(ldq=2 ** 62), dict(q=0x10002),
    dict(k_out=0x40001), dict(pos=0x50002), dict(freq=0x60001),
    dict(q_out=0x10000 + 4 * 64),                        # shifted into its own input
    dict(k_out=0x10000),                                 # k over q
    dict(k_out=0x20000 + 4 * 100),                       # k over q's output
    dict(q_out=0x10000, ldq_out=256),                    # in place with another stride
    dict(q_out=0x10000, dtype=lc.F16, out_dtype=lc.BF16),  # in place with another type
    dict(ldq=192, ldk=192, k=0x10000 + 4 * 100),         # fused columns are fine (below); here q's output is shifted
    ]
INVALID[-1].update(q_out=0x10000 + 4 * 150, ldq_out=192)


@pytest.mark.parametrize("over", INVALID, ids=str)
def test_refusals(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "lc_rope" in lc.last_error()


@pytest.mark.parametrize("over", [dict(dtype=lc.Q8_0), dict(out_dtype=12), dict(head_dim=16384, rope_dim=8194),
                                  dict(n_q=1 << 24, head_dim=64), dict(m=1 << 31)], ids=str)
def test_unsupported(over):
    assert call(**over) == lc.LC_ERR_UNSUPPORTED
    assert "lc_rope" in lc.last_error()


def test_nothing_to_do_and_null_context():
    assert call(m=0, q=None, k=None, pos=None) == lc.LC_OK
    assert call(n_q=0, n_kv=0, q=None, k=None, q_out=None, k_out=None) == lc.LC_OK
    assert lc.lib().lc_rope(None, 0, 0, 0, None, 0, None, 0, 0, None, 0, None, 0, 0, None, None, 1, 128, 128,
                            1.0) == lc.LC_ERR_INVALID


def test_positions_of_another_type_or_with_gaps_are_refused():
    import torch

    c = lc.Context.__new__(lc.Context)  # without a device: lc_rope refuses its null context
    c.L, c.h = lc.lib(), None
    good = dict(pos=torch.zeros(3, dtype=torch.int32), freq=torch.ones(4))

    def call(pos, freq):
        c.rope(lc.F32, lc.F32, lc.ROPE_HALF, 0x1000, 0x1000, 1, None, None, 0, pos, freq, 3, 8, 8)

    with pytest.raises(lc.LagunaError, match="null ctx"):
        call(**good)
    for name, t in good.items():
        for bad in (t.long(), t.double(), torch.stack([t, t], -1)[:, 0]):
            with pytest.raises(lc.LagunaError, match="read as") as e:
                call(**{**good, name: bad})
            assert e.value.status == lc.LC_ERR_INVALID


@pytest.mark.parametrize("over", [
    dict(pos=0x20000 + 2044), dict(pos=0x20000 - 12), dict(pos=0x40000 + 256 * 3), dict(freq=0x20000 + 512),
    dict(freq=0x40000 - 4 * 31), dict(ldq_out=200, pos=0x20000 + 800 * 3 + 508), dict(n_q=0, freq=0x40000),
    dict(n_kv=0, pos=0x20000)], ids=str)
def test_outputs_over_positions_or_frequencies_are_refused(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "pos or freq" in lc.last_error()


@pytest.mark.parametrize("over", [
    dict(pos=0x20000 + 2048), dict(pos=0x20000 - 16), dict(ldq_out=200, pos=0x20000 + 512),
    dict(ldq_out=200, freq=0x20000 + 800 + 512), dict(rope_dim=0, pos=0x20000, freq=0x40000)], ids=str)
def test_positions_beside_outputs_pass_the_check(monkeypatch, over):
    """They get as far as the context's device, which does not exist."""
    import struct
    import sys

    monkeypatch.setattr(sys.modules[__name__], "BLANK", C.create_string_buffer(struct.pack("i", 1 << 20), 4096))
    assert call(**over) == lc.LC_ERR_CUDA
