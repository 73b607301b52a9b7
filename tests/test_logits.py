"""lc_logits_process without a GPU: its refusals (decided from the arguments
alone, before it looks into the context, so a blank one will do), and the
restatement that the GPU tests compare with, on rows worked out by hand."""
import ctypes as C

import numpy as np
import pytest

import logits_ref
from laguna_raw_halo_strix_b200 import lc

BLANK = C.create_string_buffer(4096)  # stands for an lc_ctx


def call(rules=None, **over):
    a = dict(logits=0x100000, ld=0, out=0x200000, ld_out=0, m=4, n=100, row_offset=0)
    keys = over.pop("keys", 0x300000)
    a.update(over)
    r = lc.LogitsRules()
    for k, v in (rules or {}).items():
        setattr(r, k, v)
    return lc.lib().lc_logits_process(C.cast(BLANK, C.c_void_p), *a.values(),
                                      None if rules is False else C.byref(r), keys)


@pytest.mark.parametrize("over", [
    dict(logits=None), dict(rules=False), dict(out=None, keys=None), dict(n=0), dict(n=(1 << 30) + 1),
    dict(row_offset=0x7FFFFFFF - 99), dict(row_offset=0xFFFFFFFF), dict(ld=99), dict(ld_out=99), dict(ld=2 ** 60),
    dict(ld_out=2 ** 57), dict(logits=0x100002), dict(out=0x200001), dict(keys=0x300004), dict(out=0x100004),
    dict(out=0x100000, ld_out=200), dict(out=0x100000 + 4 * 350),
    dict(out=0x100000 + 4 * 60, ld=150, ld_out=150),
    dict(rules=dict(hist_len=5)), dict(rules=dict(hist=0x400000, hist_len=5)),
    dict(rules=dict(bias_len=5, bias_tok=0x400000, bias_start=0x500000)),
    dict(rules=dict(bias_len=5, bias=0x400000, bias_start=0x500000)),
    dict(rules=dict(bias_len=5, bias=0x400000, bias_tok=0x500000)),
    dict(rules=dict(hist=0x400001, hist_start=0x500000, hist_len=1)),
    dict(rules=dict(mask=0x400000, mask_ld=3, n_masks=4)), dict(rules=dict(mask=0x400000, mask_ld=4, n_masks=3)),
    dict(rules=dict(mask=0x400000, mask_ld=4, n_masks=4), row_offset=29),
    dict(rules=dict(mask=0x400000, mask_ld=1 << 41, n_masks=4)), dict(rules=dict(repetition=0x400002))], ids=str)
def test_invalid(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "lc_logits_process" in lc.last_error()


@pytest.mark.parametrize("over", [
    dict(m=(1 << 24) + 1), dict(rules=dict(hist=0x400000, hist_start=0x500000, hist_len=1 << 31)),
    dict(rules=dict(bias=0x400000, bias_tok=0x400000, bias_start=0x500000, bias_len=1 << 31))], ids=str)
def test_unsupported(over):
    assert call(**over) == lc.LC_ERR_UNSUPPORTED
    assert "lc_logits_process" in lc.last_error()


def test_no_rows_and_null_context():
    assert call(m=0, logits=None, out=None, keys=None) == lc.LC_OK
    assert lc.lib().lc_logits_process(None, None, 0, None, 0, 1, 1, 0, None, None) == lc.LC_ERR_INVALID


def test_restatement_by_hand():
    x = np.array([[2.0, -2.0, 1.0, 3.0, 0.5]], np.float32)
    out, _, best = logits_ref.process(
        x, hist=[0, 1, 0, 3, 3, 9], hist_start=[0, 6], gen_start=[2], repetition=[2.0], frequency=[0.25],
        presence=[0.5], bias_tok=[2, 4, 2], bias=[9.0, 1.0, 0.5], bias_start=[0, 3],
        mask=np.array([[0b10111]], np.uint32), mask_row=[0])
    # 0: seen twice, generated once; 1: prompt only; 2: the later bias; 3: masked; 4: bias
    assert out[0].tolist() == [2 / 2 - 0.25 - 0.5, -4.0, 1.5, -np.inf, 1.5]
    assert best[0] == 4  # the larger of two equal ones


def test_lists_of_another_type_or_with_gaps_are_refused():
    import torch

    good = dict(hist=torch.zeros(8, dtype=torch.int32), hist_start=torch.zeros(4, dtype=torch.int32),
                gen_start=torch.zeros(3, dtype=torch.int32), repetition=torch.ones(3), frequency=torch.ones(3),
                presence=torch.ones(3), bias_tok=torch.zeros(5, dtype=torch.int32), bias=torch.ones(5),
                bias_start=torch.zeros(4, dtype=torch.int32), mask=torch.zeros(2, 6, dtype=torch.int32)[:, :5],
                mask_row=torch.zeros(3, dtype=torch.int32))
    r = lc.LogitsRules(**good)
    assert (r.hist_len, r.bias_len, r.n_masks, r.mask_ld) == (8, 5, 2, 6)
    assert r.hist == good["hist"].data_ptr() and r.presence == good["presence"].data_ptr()
    for name, t in good.items():
        wrong = t.long() if t.dtype == torch.int32 else t.double()
        gaps = torch.stack([t, t], -1)[..., 0]
        assert torch.equal(gaps, t) and not gaps.is_contiguous()
        half = t.short() if t.dtype == torch.int32 else t.bfloat16()
        for bad in (wrong, gaps, half):
            with pytest.raises(lc.LagunaError, match="read as") as e:
                lc.LogitsRules(**{**good, name: bad})
            assert e.value.status == lc.LC_ERR_INVALID
    with pytest.raises(lc.LagunaError, match="biases for"):
        lc.LogitsRules(**{**good, "bias": torch.ones(4)})
    with pytest.raises(lc.LagunaError, match="read as"):
        lc.LogitsRules(**{**good, "mask": torch.zeros(5, dtype=torch.int32)})
    # addresses, unsigned words and missing rules pass
    lc.LogitsRules(hist=0x1000, hist_start=good["hist_start"], hist_len=3, mask=0x2000, mask_ld=4, n_masks=2)
    lc.LogitsRules(mask=torch.zeros(2, 6, dtype=torch.uint32), hist=torch.zeros(3, dtype=torch.uint32))
    lc.LogitsRules()


LISTS = dict(hist=0x400000, hist_start=0x410000, hist_len=10, gen_start=0x420000, repetition=0x430000, frequency=0x440000,
             presence=0x450000, bias_tok=0x460000, bias=0x470000, bias_start=0x480000, bias_len=7, mask=0x490000,
             mask_row=0x4a0000, mask_ld=4, n_masks=3)


@pytest.mark.parametrize("name", [k for k, v in LISTS.items() if v > 1000])
@pytest.mark.parametrize("output", ["out", "keys"])
def test_outputs_over_lists_are_refused(name, output):
    entries = {"hist": 10, "hist_start": 5, "bias_start": 5, "bias_tok": 7, "bias": 7, "mask": 12}.get(name, 4)
    last = LISTS[name] + 4 * entries - 4
    if output == "keys":
        last &= ~7
    for at in (LISTS[name], last):
        assert call(rules=LISTS, **{output: at}) == lc.LC_ERR_INVALID
        assert "overlaps" in lc.last_error()


@pytest.mark.parametrize("over", [dict(keys=0x100000), dict(keys=0x200000 + 1592), dict(keys=0x100000 - 24),
                                  dict(ld=120, keys=0x100000 + 480 * 3 + 392), dict(keys=0x200000 - 8, out=0x200010)],
                         ids=str)
def test_keys_over_logits_are_refused(over):
    assert call(**over) == lc.LC_ERR_INVALID
    assert "keys overlap" in lc.last_error()


@pytest.mark.parametrize("over", [dict(keys=0x100000 - 32), dict(keys=0x200000 + 1600), dict(ld=120, m=2, keys=0x100000 + 400),
                                  dict(out=0x400028, keys=None), dict(out=0x410014), dict(out=None, keys=0x490030),
                                  dict(out=0x100000)], ids=str)
def test_outputs_beside_what_is_read_pass_the_check(monkeypatch, over):
    """They get as far as the context's device, which does not exist."""
    import struct
    import sys

    monkeypatch.setattr(sys.modules[__name__], "BLANK", C.create_string_buffer(struct.pack("i", 1 << 20), 4096))
    assert call(rules=LISTS, **over) == lc.LC_ERR_CUDA
