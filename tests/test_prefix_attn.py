"""lc_prefix_attn without a GPU: its refusals, decided from the arguments alone
before it looks into the context, so a blank one will do."""
import ctypes as C
import struct
import sys

import pytest

from laguna_raw_halo_strix_b200 import lc

BLANK = C.create_string_buffer(4096)  # stands for an lc_ctx


def call(kv=None, **over):
    a = dict(dtype=lc.BF16, out_dtype=lc.BF16, q=0x100000, ldq=0)
    b = dict(out=0x200000, ldo=0, rows=4, n_q=8, n_kv=2, hd=64, scale=0.125, causal=1)
    for k, v in over.items():
        (a if k in a else b)[k] = v
    s = lc.PrefixKV(0x300000, 0x400000, 100, 0x500000, 0x600000, 50, 0x700000, 0x800000, 3)
    for k, v in (kv or {}).items():
        setattr(s, k, v)
    return lc.lib().lc_prefix_attn(C.cast(BLANK, C.c_void_p), *a.values(), None if kv is False else C.byref(s),
                                   *b.values())


@pytest.mark.parametrize("over", [
    dict(q=None), dict(out=None), dict(kv=False), dict(kv=dict(k_prefix=None)), dict(kv=dict(v_prefix=None)),
    dict(kv=dict(k_own=None)), dict(kv=dict(v_own=None)), dict(kv=dict(own_len=None)), dict(kv=dict(seq_start=None)),
    dict(scale=-1.0), dict(scale=0.0), dict(scale=1e-39), dict(scale=3e38), dict(scale=float("nan")), dict(scale=float("inf")), dict(ldq=511), dict(ldq=516),
    dict(ldo=500), dict(ldo=516), dict(kv=dict(ld_prefix=120)), dict(kv=dict(ld_prefix=132)),
    dict(kv=dict(ld_own=120)), dict(kv=dict(ld_own=132)), dict(kv=dict(own_stride=49 * 128 + 120)),
    dict(kv=dict(own_stride=50 * 128 + 4)), dict(kv=dict(k_prefix=0x300008)), dict(kv=dict(v_own=0x600002)),
    dict(q=0x100008), dict(out=0x200004), dict(kv=dict(own_len=0x700002)), dict(kv=dict(seq_start=0x800001)),
    dict(out=0x100000), dict(out=0x100000 + 3 * 1024), dict(ldq=1 << 38), dict(kv=dict(own_stride=1 << 39))], ids=str)
def test_invalid(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "lc_prefix_attn" in lc.last_error()


@pytest.mark.parametrize("over", [
    dict(dtype=lc.F32, out_dtype=lc.F32), dict(dtype=lc.Q8_0), dict(out_dtype=lc.F16), dict(hd=32), dict(hd=96),
    dict(hd=256), dict(n_kv=0), dict(n_kv=3), dict(rows=1 << 31), dict(rows=(1 << 26) + 1), dict(n_q=258), dict(kv=dict(prefix_len=1 << 30)),
    dict(kv=dict(own_cap=0x3FFFF000), ), dict(kv=dict(n_seqs=(1 << 20) + 1))], ids=str)
def test_unsupported(over):
    assert call(**over) == lc.LC_ERR_UNSUPPORTED
    assert "lc_prefix_attn" in lc.last_error()


def test_nothing_to_do_and_null_context():
    assert call(rows=0, q=None) == lc.LC_OK
    assert call(kv=dict(n_seqs=0)) == lc.LC_OK
    s = lc.PrefixKV(None, None, 0, None, None, 0, None, None, 0)
    assert lc.lib().lc_prefix_attn(None, lc.F16, lc.F16, None, 0, C.byref(s), None, 0, 1, 8, 8, 64, 1.0, 1) == \
        lc.LC_ERR_INVALID


def test_lengths_of_another_type_or_with_gaps_are_refused():
    import torch

    good = dict(own_len=torch.zeros(3, dtype=torch.int32), seq_start=torch.zeros(4, dtype=torch.int32))
    args = dict(k_prefix=0x1000, v_prefix=0x2000, prefix_len=4, k_own=0x3000, v_own=0x4000, own_cap=5, n_seqs=3)
    assert lc.PrefixKV(**args, **good).own_len == good["own_len"].data_ptr()
    lc.PrefixKV(**args, own_len=0x5000, seq_start=0x6000)
    for name, t in good.items():
        for bad in (t.long(), t.float(), torch.stack([t, t], -1)[:, 0]):
            with pytest.raises(lc.LagunaError, match="read as") as e:
                lc.PrefixKV(**args, **{**good, name: bad})
            assert e.value.status == lc.LC_ERR_INVALID


@pytest.mark.parametrize("over", [
    dict(out=0x300000), dict(out=0x400000 + 99 * 256), dict(out=0x300000 - 3 * 1024 - 16), dict(out=0x500000),
    dict(out=0x600000 + 3 * 50 * 256 - 16), dict(out=0x600000 - 16), dict(out=0x700000), dict(out=0x7ff010),
    dict(out=0x800000),
    dict(kv=dict(ld_prefix=640), ldo=640, out=0x300000 + 3 * 1280 + 240),    # columns that reach into k
    dict(kv=dict(ld_own=640), ldo=640, out=0x500000 + 2 * 1280 + 240),
    dict(kv=dict(own_stride=51200), out=0x500000 + 2 * 102400 - 1024),      # the next sequence's first row
], ids=str)
def test_out_over_what_is_read_is_refused(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "overlaps" in lc.last_error()


def meet_by_bytes(a, b):
    """Rows (at, pitch, width, rows) that share a byte, byte by byte."""
    def cells(r):
        return {r[0] + i * r[1] + j for i in range(r[3]) for j in range(r[2])}
    return bool(cells(a) & cells(b))


@pytest.mark.parametrize("own", [False, True])
def test_out_beside_what_is_read_passes_the_check(monkeypatch, own):
    """Out moved through the rows of a buffer that also holds k: refused exactly where a byte is shared.  (The
    others get as far as the context's device, which does not exist.)"""
    monkeypatch.setattr(sys.modules[__name__], "BLANK", C.create_string_buffer(struct.pack("i", 1 << 20), 4096))
    refused = passed = 0
    for at in range(-2560, 4 * 1280 + 1, 80):
        base = 0x500000 if own else 0x300000
        kv = dict(ld_own=640, prefix_len=0) if own else dict(ld_prefix=640, own_cap=0)
        rows = (3 * 50, 1280, 256) if own else (100, 1280, 256)
        s = call(rows=2, n_q=2, n_kv=2, hd=64, ldo=640, out=base + at, kv=kv)
        meets = meet_by_bytes((0, rows[1], rows[2], 6), (at, 1280, 256, 2))
        assert s == (lc.LC_ERR_INVALID if meets else lc.LC_ERR_CUDA) and ("overlaps" in lc.last_error()) == meets, at
        refused, passed = refused + meets, passed + (not meets)
    assert refused and passed
