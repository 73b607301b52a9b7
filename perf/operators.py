"""Cases of the operators of a batched decode step: rotary positions (lc_rope), attention of a batch that shares a
prefix (lc_prefix_attn), and penalties, biases and masks on logits (lc_logits_process).

`run` computes them in plain torch operations, or, where `own` is set, through this repository's library.
Head counts, hidden sizes and vocabularies are those of the benchmark's decoder, target and lm_head workloads
(32 query and 8 KV heads of 128, blocks of 16 tokens over 2048 positions, vocabularies of 32000 and 128256) or
generic ones.
"""
import math
import threading

import numpy as np
import torch

own = False

F32, F16, BF16 = 0, 1, 30  # GGUF type ids, as in include/laguna_cuda.h
_TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_ID = {"f32": F32, "f16": F16, "bf16": BF16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# ---- cases -----------------------------------------------------------------------

def _rope(name, m, n_q, n_kv, hd, rope_dim, layout, src, dst, far, fused):
    """far: the largest position; fused: q and k are columns of one [m, (n_q + 2 n_kv) hd] projection output."""
    return {"name": name, "op": "rope", "m": m, "n_q": n_q, "n_kv": n_kv, "hd": hd, "rope_dim": rope_dim,
            "layout": layout, "src": src, "dst": dst, "far": far, "fused": fused}


def _attn(name, seqs, tokens, n_q, n_kv, hd, prefix, cap, src, dst):
    """seqs sequences of 1..tokens query rows, a shared prefix, and 1..cap keys of their own."""
    return {"name": name, "op": "attn", "seqs": seqs, "tokens": tokens, "n_q": n_q, "n_kv": n_kv, "hd": hd,
            "prefix": prefix, "cap": cap, "src": src, "dst": dst}


def _logits(name, m, n, pad, hist, bias, masks):
    """m rows of n logits (rows n + pad apart) with up to hist past tokens and bias biases each; masks bit masks."""
    return {"name": name, "op": "logits", "m": m, "n": n, "pad": pad, "hist": hist, "bias": bias, "masks": masks}


def listed():
    return [
        # a 16-token draft block: f32 projections in, rotated q and k out in the cache's type
        _rope("rope block", 16, 32, 8, 128, 128, "half", "f32", "bf16", 4096, False),
        # a prompt with long-context positions
        _rope("rope prompt", 8192, 32, 8, 128, 128, "half", "bf16", "bf16", 131072, False),
        # half of each head rotated, neighbouring pairs, straight from a fused projection
        _rope("rope partial", 1537, 16, 2, 64, 32, "pairs", "f32", "f32", 1000000, True),
        # a few sequences on a short prompt, small heads: latency
        _attn("attn few", 4, 1, 8, 8, 64, 512, 128, "f16", "f16"),
        # candidate draft blocks verified over one context
        _attn("attn blocks", 8, 16, 32, 8, 128, 2048, 64, "bf16", "f32"),
        # one token each for a serving batch with sizable own parts
        _attn("attn batch", 64, 1, 32, 8, 128, 8192, 1024, "bf16", "bf16"),
        # continuation prompts of several requests on a common system prompt
        _attn("attn prompts", 4, 512, 32, 8, 128, 4096, 1024, "f16", "f16"),
        # a large batch on a very long document
        _attn("attn document", 128, 1, 32, 8, 128, 32768, 512, "bf16", "bf16"),
        # the rows of a verify block
        _logits("logits block", 16, 32000, 0, 2048, 0, 0),
        # one sequence
        _logits("logits one", 1, 128256, 0, 4096, 16, 1),
        # an odd vocabulary in padded rows
        _logits("logits odd", 37, 50021, 91, 700, 300, 5),
        # a serving batch, half of it under a grammar
        _logits("logits batch", 256, 128256, 0, 4096, 100, 16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "logits"])
    if op == "rope":
        hd = rng.choice([64, 80, 96, 128, 256])
        rope_dim = rng.choice([hd, hd, hd // 2, hd // 4])
        rope_dim -= rope_dim % 2
        n_kv = rng.choice([1, 2, 4, 8])
        c = _rope("", _log_int(rng, 1, 8192 * 128 // hd), n_kv * rng.choice([1, 2, 4]), n_kv, hd, rope_dim,
                  rng.choice(["half", "pairs"]), rng.choice(["f32", "f16", "bf16"]), "", rng.choice([4096, 131072, 1000000]),
                  rng.choice([True, False]))
        c["dst"] = rng.choice([c["src"], rng.choice(["f32", "f16", "bf16"])])
    elif op == "attn":
        n_kv = rng.choice([1, 2, 4, 8])
        src = rng.choice(["f16", "bf16"])
        tokens = rng.choice([1, 1, _log_int(rng, 2, 512)])
        seqs = _log_int(rng, 1, max(1, min(128, 2048 // tokens)))
        c = _attn("", seqs, tokens, n_kv * rng.choice([1, 2, 4]), n_kv, rng.choice([64, 128]),
                  _log_int(rng, 1, min(32768, 4096 * 2048 // (tokens * seqs))), tokens + _log_int(rng, 1, 511), src,
                  rng.choice([src, src, "f32"]))
    else:
        n = _log_int(rng, 1000, 262144)
        c = _logits("", _log_int(rng, 1, max(1, 256 * 128256 // n // 2)), n, rng.choice([0, 0, rng.randint(1, 200)]),
                    _log_int(rng, 1, 8192), rng.choice([0, _log_int(rng, 1, 500)]), rng.choice([0, rng.randint(1, 20)]))
        c["m"] = min(c["m"], 512)
    del c["name"]
    return c


# ---- sizes that follow from a case ----------------------------------------------------

def _spread(count, lo, hi, phase=0.0):
    """count whole numbers in lo..hi, spread evenly and out of order."""
    x = (np.arange(1, count + 1) * 0.6180339887498949 + phase) % 1.0
    return (lo + np.floor(x * (hi - lo + 1))).astype(np.int64)


def _attn_sizes(c):
    rows = _spread(c["seqs"], max(1, c["tokens"] // 2), c["tokens"])
    lens = np.maximum(rows, _spread(c["seqs"], 1, c["cap"], 0.3))  # the query rows are the last of the own ones
    return rows, lens


def _logits_sizes(c):
    return (_spread(c["m"], 0 if c["m"] > 1 else c["hist"], c["hist"]),
            _spread(c["m"], 0 if c["m"] > 1 else c["bias"], c["bias"], 0.4))


def work(case):
    c = case
    if c["op"] == "rope":
        n = c["m"] * (c["n_q"] + c["n_kv"]) * c["hd"]
        return {"bytes": n * (_BYTES[c["src"]] + _BYTES[c["dst"]]) + 4 * c["m"], "flops": 6 * n // 2}
    if c["op"] == "attn":
        rows, lens = _attn_sizes(c)
        pairs = float(np.sum(rows * (c["prefix"] + lens) - rows * (rows - 1) // 2))  # visible (query, key) pairs
        kv = 2 * c["n_kv"] * c["hd"] * 2 * (c["prefix"] + int(lens.sum()))
        qo = int(rows.sum()) * c["n_q"] * c["hd"] * (2 + _BYTES[c["dst"]])
        return {"bytes": kv + qo, "flops": 4 * c["n_q"] * c["hd"] * pairs}
    hist, bias = _logits_sizes(c)
    words = (c["n"] + 31) // 32
    return {"bytes": 8 * c["m"] * c["n"] + 4 * int(hist.sum()) + 8 * int(bias.sum()) + 4 * words * c["masks"] + 8 * c["m"],
            "flops": 2 * c["m"] * c["n"]}


# ---- inputs ---------------------------------------------------------------------------

def prepare(case, seed):
    c, dev = dict(case), torch.device("cuda")
    g = torch.Generator(dev)
    g.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=dev).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=dev, dtype=torch.int64)

    s = {"case": c}
    if c["op"] == "rope":
        m, hd, t = c["m"], c["hd"], _TYPE[c["src"]]
        wq, wk = c["n_q"] * hd, c["n_kv"] * hd
        if c["fused"]:
            qkv = normal(m, wq + 2 * wk, dtype=t)
            s["q"], s["k"] = qkv[:, :wq], qkv[:, wq:wq + wk]
        else:
            s["q"], s["k"] = normal(m, wq, dtype=t), normal(m, wk, dtype=t)
        # consecutive positions of a sequence that starts somewhere before `far`
        start = whole(0, max(1, c["far"] - m), 1)
        s["pos"] = (start + torch.arange(m, device=dev)).to(torch.int32)
        half = c["rope_dim"] // 2
        s["freq"] = (500000.0 ** (-torch.arange(half, device=dev, dtype=torch.float64) / half)).to(torch.float32)
        s["scale"] = 1.0 if c["far"] <= 4096 else 1.25
        s["q_out"] = torch.empty(m, wq, device=dev, dtype=_TYPE[c["dst"]])
        s["k_out"] = torch.empty(m, wk, device=dev, dtype=_TYPE[c["dst"]])
    elif c["op"] == "attn":
        t, hd, wk = _TYPE[c["src"]], c["hd"], c["n_kv"] * c["hd"]
        rows, lens = _attn_sizes(c)
        total = int(rows.sum())
        s["q"] = normal(total, c["n_q"] * hd, dtype=t)
        s["k_prefix"], s["v_prefix"] = normal(c["prefix"], wk, dtype=t), normal(c["prefix"], wk, dtype=t)
        s["k_own"], s["v_own"] = normal(c["seqs"], c["cap"], wk, dtype=t), normal(c["seqs"], c["cap"], wk, dtype=t)
        s["own_len"] = torch.from_numpy(lens.astype(np.int32)).to(dev)
        s["seq_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)).to(dev)
        s["max_rows"] = int(rows.max())
        s["scale"] = 1.0 / math.sqrt(hd)
        s["out"] = torch.empty(total, c["n_q"] * hd, device=dev, dtype=_TYPE[c["dst"]])
    else:
        m, n = c["m"], c["n"]
        s["logits"] = (4 * normal(m, n + c["pad"]))[:, :n]
        hist, bias = _logits_sizes(c)

        def ragged(sizes):
            return torch.from_numpy(np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)).to(dev)

        def tokens(count):  # a text's tokens: few of them often, many rarely
            u = torch.rand(count, generator=g, device=dev, dtype=torch.float64)
            return ((u ** 4 * n).to(torch.int64) * 7919 % n).to(torch.int32)

        s["hist"], s["hist_start"] = tokens(int(hist.sum())), ragged(hist)
        s["gen_start"] = s["hist_start"][:-1] + (torch.from_numpy(hist).to(dev) // 2).to(torch.int32)
        s["repetition"] = 1 + 0.3 * torch.rand(m, generator=g, device=dev)
        s["frequency"] = 0.5 * torch.rand(m, generator=g, device=dev)
        s["presence"] = 0.5 * torch.rand(m, generator=g, device=dev)
        s["bias_tok"], s["bias_start"] = tokens(int(bias.sum())), ragged(bias)
        s["bias"] = 2 * normal(int(bias.sum()))
        words = (n + 31) // 32
        s["mask"], s["mask_row"] = None, None
        if c["masks"]:
            allow = torch.rand(c["masks"], words * 32, generator=g, device=dev) < 0.25
            bit = (1 << torch.arange(32, device=dev, dtype=torch.int64))
            w = (allow.view(-1, words, 32).to(torch.int64) * bit).sum(-1)
            s["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
            row = torch.arange(m, device=dev)
            s["mask_row"] = torch.where(row % 2 == 0, row // 2 % c["masks"], -1).to(torch.int32)
        s["out"] = torch.empty(m, n, device=dev)
        s["keys"] = torch.empty(m, dtype=torch.int64, device=dev)
    return s


# ---- one pass ---------------------------------------------------------------------------

_ctx = {}


def _context():
    """This thread's library context on the current device, enqueuing on torch's current stream."""
    from laguna_raw_halo_strix_b200 import lc

    at = threading.get_ident(), torch.cuda.current_device()
    if at not in _ctx:
        _ctx[at] = lc.Context(at[1])
    _ctx[at].set_stream(torch.cuda.current_stream())
    return lc, _ctx[at]


def run(state):
    op = state["case"]["op"]
    if op == "rope":
        return _own_rope(state) if own else _plain_rope(state)
    if op == "attn":
        return _own_attn(state) if own else _plain_attn(state)
    return _own_logits(state) if own else _plain_logits(state)


def _own_rope(s):
    lc, ctx = _context()
    c = s["case"]
    layout = lc.ROPE_HALF if c["layout"] == "half" else lc.ROPE_PAIRS
    ctx.rope(_ID[c["src"]], _ID[c["dst"]], layout, s["q"], s["q_out"], c["n_q"], s["k"], s["k_out"], c["n_kv"],
             s["pos"], s["freq"], c["m"], c["hd"], c["rope_dim"], s["scale"], ldq=s["q"].stride(0),
             ldk=s["k"].stride(0))
    return s["q_out"], s["k_out"]


def _plain_rope(s):
    c = s["case"]
    hd, rd, half = c["hd"], c["rope_dim"], c["rope_dim"] // 2
    angle = s["pos"].double()[:, None] * s["freq"].double()
    cos, sin = (s["scale"] * angle.cos()).float()[:, None, :], (s["scale"] * angle.sin()).float()[:, None, :]

    def rotate(x, heads):
        x = x.reshape(c["m"], heads, hd).float()
        if c["layout"] == "half":
            a, b = x[..., :half], x[..., half:rd]
            y = torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rd:]], -1)
        else:
            a, b = x[..., 0:rd:2], x[..., 1:rd:2]
            y = torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., rd:]], -1)
        return y.reshape(c["m"], heads * hd).to(_TYPE[c["dst"]])

    return rotate(s["q"], c["n_q"]), rotate(s["k"], c["n_kv"])


def _own_attn(s):
    lc, ctx = _context()
    c = s["case"]
    kv = lc.PrefixKV(s["k_prefix"], s["v_prefix"], c["prefix"], s["k_own"], s["v_own"], c["cap"], s["own_len"],
                     s["seq_start"], c["seqs"])
    ctx.prefix_attn(_ID[c["src"]], _ID[c["dst"]], s["q"], kv, s["out"], s["q"].shape[0], c["n_q"], c["n_kv"], c["hd"],
                    s["scale"])
    return s["out"]


def _plain_attn(s):
    c = s["case"]
    hd, n_kv, seqs, cap, most = c["hd"], c["n_kv"], c["seqs"], c["cap"], s["max_rows"]
    group, total = c["n_q"] // n_kv, s["q"].shape[0]
    start = s["seq_start"].long()
    rows = start[1:] - start[:-1]
    row = torch.arange(total, device=s["q"].device)
    seq = torch.searchsorted(start[1:].contiguous(), row, right=True)
    q = (s["q"].float() * s["scale"]).view(total, n_kv, group, hd)
    # the prefix, for every row at once: [n_kv, total * group, prefix]
    kp = s["k_prefix"].float().view(-1, n_kv, hd).transpose(0, 1)
    vp = s["v_prefix"].float().view(-1, n_kv, hd).transpose(0, 1)
    sp = (q.transpose(0, 1).reshape(n_kv, total * group, hd) @ kp.transpose(1, 2)).view(n_kv, total, group, -1)
    # the own parts, rows padded to the longest sequence: [seqs, n_kv, most * group, cap]
    at = row - start[seq]
    padded = torch.zeros(seqs, most, n_kv, group, hd, device=q.device)
    padded[seq, at] = q
    ko, vo = s["k_own"].float().view(seqs, cap, n_kv, hd), s["v_own"].float().view(seqs, cap, n_kv, hd)
    so = padded.permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, most * group, hd) @ ko.permute(0, 2, 3, 1)
    so = so.view(seqs, n_kv, most, group, cap)
    place = s["own_len"].long()[:, None] - rows[:, None] + torch.arange(most, device=q.device)  # [seqs, most]
    seen = torch.arange(cap, device=q.device) <= place[..., None]
    so = so.masked_fill(~seen[:, None, :, None, :], -math.inf)
    so = so.permute(0, 2, 1, 3, 4)[seq, at].transpose(0, 1)  # [n_kv, total, group, cap]
    top = torch.maximum(sp.amax(-1), so.amax(-1))[..., None]
    ep, eo = (sp - top).exp(), (so - top).exp()
    weight = ep.sum(-1) + eo.sum(-1)
    out = (ep.view(n_kv, total * group, -1) @ vp).view(n_kv, total, group, hd)
    po = torch.zeros(seqs, most, n_kv, group, cap, device=q.device)
    po[seq, at] = eo.transpose(0, 1)
    oo = po.permute(0, 2, 1, 3, 4).reshape(seqs, n_kv, most * group, cap) @ vo.permute(0, 2, 1, 3)
    oo = oo.view(seqs, n_kv, most, group, hd).permute(0, 2, 1, 3, 4)[seq, at].transpose(0, 1)
    out = (out + oo) / weight[..., None]
    return out.transpose(0, 1).reshape(total, n_kv * group * hd).to(_TYPE[c["dst"]])


def _own_logits(s):
    lc, ctx = _context()
    c = s["case"]
    rules = lc.LogitsRules(hist=s["hist"], hist_start=s["hist_start"], gen_start=s["gen_start"],
                           repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                           bias_tok=s["bias_tok"], bias=s["bias"], bias_start=s["bias_start"], mask=s["mask"],
                           mask_row=s["mask_row"])
    ctx.logits_process(s["logits"], rules, s["out"], s["keys"], c["m"], c["n"], ld=s["logits"].stride(0))
    return s["out"], s["keys"]


def _plain_logits(s):
    c = s["case"]
    m, n, dev = c["m"], c["n"], s["logits"].device
    x = s["logits"]

    def row_of(start, count):
        return torch.searchsorted(start[1:].long().contiguous(), torch.arange(count, device=dev), right=True)

    at = torch.arange(s["hist"].numel(), device=dev)
    row = row_of(s["hist_start"], at.numel())
    cell = row * n + s["hist"].long()
    made = (at >= s["gen_start"].long()[row]).float()
    seen = torch.zeros(m * n, device=dev).scatter_add_(0, cell, torch.ones_like(made)).view(m, n) > 0
    count = torch.zeros(m * n, device=dev).scatter_add_(0, cell, made).view(m, n)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = torch.where(count > 0, x - s["frequency"][:, None] * count - s["presence"][:, None], x)
    nb = s["bias"].numel()
    if nb:  # a token listed twice takes the later entry
        cell = row_of(s["bias_start"], nb) * n + s["bias_tok"].long()
        last = torch.full((m * n,), -1, dtype=torch.int64, device=dev)
        last = last.scatter_reduce_(0, cell, torch.arange(nb, device=dev), "amax").view(m, n)
        x = torch.where(last >= 0, x + s["bias"][last.clamp(min=0)], x)
    if s["mask"] is not None:
        bits = (s["mask"].long()[:, :, None] >> torch.arange(32, device=dev)) & 1
        allow = bits.view(s["mask"].shape[0], -1)[:, :n] > 0
        r = s["mask_row"].long()
        x = x.masked_fill(~(allow[r.clamp(min=0)] | (r < 0)[:, None]), -math.inf)
    top = x.amax(-1)
    token = torch.where(x == top[:, None], torch.arange(n, device=dev), -1).amax(-1)
    # the key of include/laguna_cuda.h: the value's order in the high half, the token in the low one
    b = top.contiguous().view(torch.int32).long()
    order = torch.where(b < 0, ~b - 2 ** 31, b)
    return x, (order << 32) + token


# ---- the operators in 64 bits -------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "logits": _exact_logits}[case["op"]](s)


def _exact_rope(s):
    """Each pair as a complex number, turned by exp(i pos freq)."""
    c = s["case"]
    rd, hd = c["rope_dim"], c["hd"]
    turn = torch.polar(torch.full((c["m"], rd // 2), s["scale"], dtype=torch.float64, device=s["pos"].device),
                       torch.outer(s["pos"].to(torch.float64), s["freq"].to(torch.float64)))

    def turned(x, heads):
        y = x.to(torch.float64).reshape(c["m"], heads, hd).clone()
        part = y[:, :, :rd]
        pairs = part.unflatten(-1, (2, rd // 2)).transpose(-1, -2) if c["layout"] == "half" else part.unflatten(-1, (rd // 2, 2))
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
        y[:, :, :rd] = (z.transpose(-1, -2) if c["layout"] == "half" else z).flatten(-2)
        return y.reshape(c["m"], heads * hd)

    return turned(s["q"], c["n_q"]), turned(s["k"], c["n_kv"])


def _exact_attn(s):
    """One sequence and one KV head at a time, over the joined keys."""
    c = s["case"]
    hd, group = c["hd"], c["n_q"] // c["n_kv"]
    rows, lens = _attn_sizes(c)
    out = torch.empty(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    at = 0
    for b in range(c["seqs"]):
        r, n = int(rows[b]), int(lens[b])
        k = torch.cat([s["k_prefix"], s["k_own"][b, :n]]).double()
        v = torch.cat([s["v_prefix"], s["v_own"][b, :n]]).double()
        hidden = torch.ones(r, n, dtype=torch.bool, device=k.device).triu(n - r + 1)
        hidden = torch.cat([torch.zeros(r, c["prefix"], dtype=torch.bool, device=k.device), hidden], 1)
        for h in range(c["n_kv"]):
            q = s["q"][at:at + r, h * group * hd:(h + 1) * group * hd].double().reshape(r, group, hd)
            p = torch.einsum("rgd,kd->grk", q, k[:, h * hd:(h + 1) * hd]) * s["scale"]
            p = torch.softmax(p.masked_fill(hidden, -math.inf), -1)
            o = torch.einsum("grk,kd->rgd", p, v[:, h * hd:(h + 1) * hd])
            out[at:at + r, h * group * hd:(h + 1) * group * hd] = o.reshape(r, group * hd)
        at += r
    return out


def _exact_logits(s):
    """One row at a time on the host."""
    c = s["case"]
    n = c["n"]
    host = {k: v.cpu().numpy() for k, v in s.items() if torch.is_tensor(v)}
    out = host["logits"].astype(np.float64)
    for r in range(c["m"]):
        lo, hi = host["hist_start"][r], host["hist_start"][r + 1]
        past, made = np.unique(host["hist"][lo:hi]), host["hist"][host["gen_start"][r]:hi]
        rep = float(host["repetition"][r])
        v = out[r, past]
        out[r, past] = np.where(v > 0, v / rep, v * rep)
        tok, times = np.unique(made, return_counts=True)
        out[r, tok] -= float(host["frequency"][r]) * times + float(host["presence"][r])
        lo, hi = host["bias_start"][r], host["bias_start"][r + 1]
        given = dict(zip(host["bias_tok"][lo:hi].tolist(), host["bias"][lo:hi].tolist()))
        if given:
            out[r, list(given)] += np.array(list(given.values()), np.float64)
        if c["masks"] and host["mask_row"][r] >= 0:
            bits = np.unpackbits(host["mask"][host["mask_row"][r]].view(np.uint8), bitorder="little")[:n]
            out[r, bits == 0] = -np.inf
    return out, None  # the keys hold 32-bit values
