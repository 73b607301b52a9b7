"""lc_logits_process restated for one row at a time: in 32 bits with the same
roundings, and in 64 bits with a bound of what the 32-bit roundings can add."""
import numpy as np


def row_lists(start, r, size):
    lo = min(max(int(start[r]), 0), size)
    return lo, min(max(int(start[r + 1]), lo), size)


def process(logits, offset=0, hist=None, hist_start=None, gen_start=None, repetition=None, frequency=None,
            presence=None, bias_tok=None, bias=None, bias_start=None, mask=None, mask_row=None, dtype=np.float32):
    """-> (values [m, n], bound [m, n] of the f32 roundings, best token [m])."""
    m, n = logits.shape
    out = logits.astype(dtype)
    tol = np.zeros((m, n))
    half = 2.0 ** -24
    one = dtype(1)
    with np.errstate(all="ignore"):
        for r in range(m):
            x, t = out[r], tol[r]
            rep = dtype(repetition[r]) if repetition is not None else one
            fr = dtype(frequency[r]) if frequency is not None else dtype(0)
            pr = dtype(presence[r]) if presence is not None else dtype(0)
            seen, made = {}, {}
            if hist_start is not None:
                lo, hi = row_lists(hist_start, r, len(hist))
                first = int(gen_start[r]) if gen_start is not None else lo
                for i in range(lo, hi):
                    j = int(hist[i]) - offset
                    if 0 <= j < n:
                        seen[j] = True
                        if i >= first:
                            made[j] = made.get(j, 0) + 1
            for j in seen:
                x[j] = x[j] / rep if x[j] > 0 else x[j] * rep
                t[j] += half * abs(x[j])
                if j in made:
                    f = fr * dtype(made[j])
                    a = x[j] - f
                    x[j] = a - pr
                    t[j] += half * (abs(f) + abs(a) + abs(x[j]))
            if bias_start is not None:
                lo, hi = row_lists(bias_start, r, len(bias_tok))
                given = {}
                for i in range(lo, hi):
                    given[int(bias_tok[i]) - offset] = bias[i]
                for j, b in given.items():
                    if 0 <= j < n:
                        x[j] = x[j] + dtype(b)
                        t[j] += half * abs(x[j])
            if mask is not None:
                k = int(mask_row[r]) if mask_row is not None else r
                if 0 <= k < len(mask):
                    bits = np.unpackbits(np.ascontiguousarray(mask[k]).view(np.uint8), bitorder="little")
                    x[bits[offset:offset + n] == 0] = -np.inf
    best = np.array([n - 1 - int(np.argmax(out[r, ::-1])) for r in range(m)])
    return out, tol, best
