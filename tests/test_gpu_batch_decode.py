"""Rotary positions, attention over a shared prefix, lm_head and logits rules run
together as a batched decode uses them: several sequences continue one prompt,
each step rotates q and k (k and v straight into the 16-bit caches), attends,
projects and picks the next tokens under the rules; the chain is followed in 64
bits from the same cache contents."""
import math

import numpy as np
import pytest

import logits_ref
from conftest import to_dev
from laguna_raw_halo_strix_b200 import lc, synth

pytestmark = pytest.mark.gpu

N_Q, N_KV, HD, VOCAB = 8, 2, 64, 1500
WQ, WK = N_Q * HD, N_KV * HD


def attend(q, k, v, scale):
    """One row of heads in 64 bits: q [N_Q, HD] over k, v [n, N_KV, HD]."""
    out = np.empty((N_Q, HD))
    for h in range(N_Q):
        s = k[:, h * N_KV // N_Q] @ q[h] * scale
        w = np.exp(s - s.max())
        out[h] = (w / w.sum()) @ v[:, h * N_KV // N_Q]
    return out.ravel()


def test_decode_steps(ctx, dev):
    import torch

    rng = np.random.default_rng(0)
    g = torch.Generator(dev).manual_seed(0)
    prefix, cap, seqs, steps = 300, 8, 5, 4
    bf16 = torch.bfloat16

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    freq, rope_scale = lc.rope_freq_scaled(HD, 500000.0, lc.ROPE_SCALE_YARN, 4.0, 4096)
    freq_d = torch.from_numpy(freq).to(dev)
    # the prompt: its keys rotated and its values converted into the prefix cache
    kp, vp = torch.empty(prefix, WK, device=dev, dtype=bf16), torch.empty(prefix, WK, device=dev, dtype=bf16)
    k_raw, v_raw = normal(prefix, WK), normal(prefix, WK)
    at = torch.arange(prefix, device=dev, dtype=torch.int32)
    ctx.rope(lc.F32, lc.BF16, lc.ROPE_HALF, None, None, 0, k_raw, kp, N_KV, at, freq_d, prefix, HD, HD, rope_scale)
    ctx.rope(lc.F32, lc.BF16, lc.ROPE_HALF, None, None, 0, v_raw, vp, N_KV, None, None, prefix, HD, 0)
    torch.cuda.synchronize()
    assert torch.equal(vp, v_raw.to(bf16))
    ko = torch.zeros(seqs, cap, WK, device=dev, dtype=bf16)
    vo = torch.zeros(seqs, cap, WK, device=dev, dtype=bf16)
    own_len = torch.zeros(seqs, device=dev, dtype=torch.int32)
    seq_start = torch.arange(seqs + 1, device=dev, dtype=torch.int32)
    kv = lc.PrefixKV(kp, vp, prefix, ko, vo, cap, own_len, seq_start, seqs)
    w_head = to_dev(synth.q8_0_blocks(VOCAB, WQ, rng), dev)
    hist = torch.zeros(seqs, 64, device=dev, dtype=torch.int32)  # each sequence's tokens in a strip of 64
    hist[:, :10] = torch.from_numpy(rng.integers(0, VOCAB, (seqs, 10)).astype(np.int32))
    mask = rng.integers(0, 2 ** 32, (2, (VOCAB + 31) // 32), dtype=np.uint32)
    rules_h = dict(repetition=np.full(seqs, 1.3, np.float32), frequency=np.full(seqs, 0.2, np.float32),
                   presence=np.full(seqs, 0.1, np.float32), mask=mask,
                   mask_row=np.array([0, 1, -1, 0, 1], np.int32))
    dev_rules = {k: torch.from_numpy(v.view(np.int32) if v.dtype == np.uint32 else v).to(dev)
                 for k, v in rules_h.items()}
    count = 10
    for step in range(steps):
        qkv = normal(seqs, WQ + 2 * WK)  # a fused projection's output
        q = torch.empty(seqs, WQ, device=dev, dtype=bf16)
        pos = torch.full((seqs,), prefix + step, device=dev, dtype=torch.int32)
        # k rows go to row `step` of each sequence's slot, cap rows apart
        ctx.rope(lc.F32, lc.BF16, lc.ROPE_HALF, qkv, q, N_Q, qkv[:, WQ:], ko[:, step], N_KV, pos, freq_d, seqs, HD, HD,
                 rope_scale, ldq=qkv.stride(0), ldk=qkv.stride(0), ldk_out=cap * WK)
        ctx.rope(lc.F32, lc.BF16, lc.ROPE_HALF, None, None, 0, qkv[:, WQ + WK:], vo[:, step], N_KV, None, None, seqs,
                 HD, 0, ldk=qkv.stride(0), ldk_out=cap * WK)
        own_len += 1
        hidden = torch.empty(seqs, WQ, device=dev)
        ctx.prefix_attn(lc.BF16, lc.F32, q, kv, hidden, seqs, N_Q, N_KV, HD, 1 / math.sqrt(HD))
        logits = torch.empty(seqs, VOCAB, device=dev)
        ctx.proj_m(lc.Q8_0, hidden, w_head, logits, seqs, WQ, VOCAB)
        start = (torch.arange(seqs + 1, device=dev) * 64).to(torch.int32)
        # strips of 64 whose rows end at `count`: gen_start marks the 10 prompt tokens, and the
        # unused tail of a strip holds token -1, which no vocabulary has
        hist[:, count:] = -1
        rules = lc.LogitsRules(hist=hist, hist_start=start, gen_start=start[:-1] + 10, **dev_rules)
        keys = torch.empty(seqs, device=dev, dtype=torch.int64)
        raw = logits.clone()
        ctx.logits_process(logits, rules, logits, keys, seqs, VOCAB)
        torch.cuda.synchronize()

        # the same step in 64 bits, from the 16-bit q and cache rows
        x = qkv.double().cpu().numpy()
        turn = (prefix + step) * freq.astype(np.float64)
        c, s = rope_scale * np.cos(turn), rope_scale * np.sin(turn)
        qr = x[:, :WQ].reshape(seqs, N_Q, 2, HD // 2)
        ref_q = np.stack([qr[:, :, 0] * c - qr[:, :, 1] * s, qr[:, :, 1] * c + qr[:, :, 0] * s], 2).reshape(seqs, WQ)
        mag = rope_scale * np.abs(qr).sum(2, keepdims=True).repeat(2, 2).reshape(seqs, WQ)
        assert (np.abs(q.double().cpu().numpy() - ref_q) <= np.abs(ref_q) * 2.0 ** -8 + mag * 2.0 ** -20).all()
        assert torch.equal(vo[:, step], qkv[:, WQ + WK:].to(bf16))
        for b in range(seqs):
            k = torch.cat([kp, ko[b, :step + 1]]).double().cpu().numpy().reshape(-1, N_KV, HD)
            v = torch.cat([vp, vo[b, :step + 1]]).double().cpu().numpy().reshape(-1, N_KV, HD)
            ref = attend(q[b].double().cpu().numpy().reshape(N_Q, HD), k, v, 1 / math.sqrt(HD))
            # weights within 24 bits and sums in f32 over 300 keys of values up to about 4
            assert np.abs(hidden[b].double().cpu().numpy() - ref).max() <= 2e-5 * np.abs(v).max()
        ref_logits, _, best = logits_ref.process(raw.cpu().numpy(), hist=hist.cpu().numpy().ravel(),
                                                 hist_start=start.cpu().numpy(),
                                                 gen_start=(start[:-1] + 10).cpu().numpy(), **rules_h)
        assert np.array_equal(logits.cpu().numpy().view(np.uint32), ref_logits.view(np.uint32))
        tokens = [lc.key_index(int(t)) for t in keys]
        assert tokens == best.tolist()
        hist[:, count] = torch.tensor(tokens, dtype=torch.int32, device=dev)
        count += 1
    ctx.device_status()


def test_beside_other_kernels(ctx, dev):
    """Two contexts on two streams at once: attention over a prefix beside lc_mha_attn and quantised products,
    which hold tensor memory too."""
    import torch

    seqs, prefix = 40, 2000
    bf16 = torch.bfloat16
    q = torch.randn(seqs, WQ, device=dev).to(bf16)
    kp, vp = (torch.randn(prefix, WK, device=dev).to(bf16) for _ in range(2))
    ko, vo = (torch.randn(seqs, 100, WK, device=dev).to(bf16) for _ in range(2))
    lens = torch.randint(1, 101, (seqs,), device=dev, dtype=torch.int32)
    start = torch.arange(seqs + 1, device=dev, dtype=torch.int32)
    kv = lc.PrefixKV(kp, vp, prefix, ko, vo, 100, lens, start, seqs)
    qa, ka, va = (torch.randn(16, w, device=dev) for w in (1024, 256, 256))
    ka, va = torch.randn(2064, 256, device=dev), torch.randn(2064, 256, device=dev)
    rng = np.random.default_rng(1)
    w = to_dev(synth.q4k_blocks(4096, 1024, rng), dev)
    x = torch.randn(16, 1024, device=dev)

    def one(c, out):
        c.prefix_attn(lc.BF16, lc.F32, q, kv, out, seqs, N_Q, N_KV, HD, 0.125)

    def two(c, out, y):
        c.mha_attn(qa, ka, va, out, 16, 8, 2, 128, 2064, 0.09, 2048, 1)
        c.proj_m(lc.Q4_K, x, w, y, 16, 1024, 4096)

    ref1, ref2, ref3 = torch.empty(seqs, WQ, device=dev), torch.empty(16, 1024, device=dev), torch.empty(16, 4096, device=dev)
    one(ctx, ref1)
    two(ctx, ref2, ref3)
    torch.cuda.synchronize()
    streams, ctxs = [torch.cuda.Stream() for _ in range(2)], [lc.Context(0) for _ in range(2)]
    got1, got2, got3 = torch.empty_like(ref1), torch.empty_like(ref2), torch.empty_like(ref3)
    for c, s in zip(ctxs, streams):
        c.set_stream(s)
    for _ in range(30):
        one(ctxs[0], got1)
        two(ctxs[1], got2, got3)
    torch.cuda.synchronize()
    assert torch.equal(got1, ref1) and torch.equal(got2, ref2)
    # the quantised product's split sums may be joined in another order
    assert (got3 - ref3).abs().max() <= 1e-5 * ref3.abs().max()
    for c in ctxs:
        c.device_status()
        c.close()


def test_captured_among_copies_and_forks(dev):
    """A graph in which the operators follow memsets, copies, events of another stream and each other, each with
    inputs that the node before it writes late; replays see new inputs."""
    import torch

    g = torch.Generator(dev).manual_seed(1)
    rows, prefix, cap = 6, 700, 40
    f16 = torch.float16
    src = torch.randn(rows, WQ + WK, generator=g, device=dev)
    q, k = torch.empty(rows, WQ, device=dev), torch.empty(rows, WK, device=dev)
    q16, k16 = torch.empty(rows, WQ, device=dev, dtype=f16), torch.empty(rows, WK, device=dev, dtype=f16)
    kp, vp = (torch.randn(prefix, WK, generator=g, device=dev).to(f16) for _ in range(2))
    ko = torch.zeros(rows, cap, WK, device=dev, dtype=f16)
    vo = torch.randn(rows, cap, WK, generator=g, device=dev).to(f16)
    pos = torch.arange(rows, device=dev, dtype=torch.int32) + prefix
    freq = torch.from_numpy(lc.rope_freq(HD)).to(dev)
    own_len = torch.ones(rows, device=dev, dtype=torch.int32)
    seq_start = torch.arange(rows + 1, device=dev, dtype=torch.int32)
    kv = lc.PrefixKV(kp, vp, prefix, ko, vo, cap, own_len, seq_start, rows)
    out, logits = torch.empty(rows, WQ, device=dev), torch.empty(rows, 9000, device=dev)
    head = torch.randn(WQ, 9000, generator=g, device=dev) / 16
    keys, side_keys = (torch.empty(rows, device=dev, dtype=torch.int64) for _ in range(2))
    pen = torch.full((rows,), 1.3, device=dev)
    rules = lc.LogitsRules(hist=torch.arange(600, device=dev, dtype=torch.int32),
                           hist_start=torch.arange(rows + 1, device=dev, dtype=torch.int32) * 100, repetition=pen)
    main, side, ctx, other = torch.cuda.Stream(), torch.cuda.Stream(), lc.Context(0), lc.Context(0)

    def step():
        mine = torch.cuda.current_stream()
        ctx.set_stream(mine), other.set_stream(side)
        q.copy_(src[:, :WQ])  # copies, then rope on what they wrote
        k.copy_(src[:, WQ:])
        ctx.rope(lc.F32, lc.F16, lc.ROPE_HALF, q, q16, N_Q, k, k16, N_KV, pos, freq, rows, HD, HD)
        ko[:, 0].copy_(k16)
        side.wait_stream(mine)
        with torch.cuda.stream(side):
            logits.zero_()
            other.logits_process(logits, rules, None, side_keys, rows, 9000)
            pen.mul_(1.0)
        mine.wait_stream(side)
        ctx.prefix_attn(lc.F16, lc.F32, q16, kv, out, rows, N_Q, N_KV, HD, HD ** -0.5)
        ctx.prefix_attn(lc.F16, lc.F32, q16, kv, out, rows, N_Q, N_KV, HD, HD ** -0.5)
        torch.mm(out, head, out=logits)
        ctx.logits_process(logits, rules, logits, keys, rows, 9000)
        ctx.rope(lc.F32, lc.F32, lc.ROPE_HALF, out, out, N_Q, None, None, 0, pos, freq, rows, HD, HD)
        return [t.clone() for t in (q16, out, logits, keys, side_keys)]

    with torch.cuda.stream(main):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        captured = step()
    for seed in range(4):
        src.copy_(torch.randn(src.shape, generator=torch.Generator(dev).manual_seed(seed), device=dev))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        with torch.cuda.stream(main):
            want = step()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("rows,n", [(6, 9000), (400, 3001)])
@pytest.mark.parametrize("forked", [False, True])
def test_rules_that_the_node_before_writes(dev, rows, n, forked):
    """Every list and the logits are filled by the nodes right before the rules' kernel, on its stream and on
    another one, from what each replay finds; against the restatement."""
    import torch

    rng = np.random.default_rng(rows)
    sizes = rng.integers(0, 60, rows)
    start = np.concatenate([[0], np.cumsum(sizes)]).astype(np.int32)
    words = (n + 31) // 32

    def inputs(seed):
        r = np.random.default_rng(seed)
        return dict(x=(3 * r.standard_normal((rows, n))).astype(np.float32),
                    hist=r.integers(0, n, start[-1]).astype(np.int32), hist_start=start,
                    gen_start=(start[:-1] + r.integers(0, sizes + 1)).astype(np.int32),
                    repetition=r.uniform(0.7, 1.5, rows).astype(np.float32),
                    frequency=r.uniform(-0.5, 1, rows).astype(np.float32),
                    presence=r.uniform(-0.5, 1, rows).astype(np.float32),
                    bias_tok=r.integers(0, n, start[-1]).astype(np.int32), bias_start=start,
                    bias=r.standard_normal(start[-1]).astype(np.float32),
                    mask=r.integers(0, 2 ** 32, (3, words), dtype=np.uint32).view(np.int32),
                    mask_row=r.integers(-1, 3, rows).astype(np.int32))

    given = {k: to_dev(v, dev) for k, v in inputs(0).items()}
    held = {k: torch.zeros_like(v) for k, v in given.items()}
    out, keys = torch.empty(rows, n, device=dev), torch.empty(rows, device=dev, dtype=torch.int64)
    rules = lc.LogitsRules(**{k: v for k, v in held.items() if k != "x"})
    c, main, side = lc.Context(0), torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()

    def step():
        mine = torch.cuda.current_stream()
        late = side if forked else mine
        for k in held:
            held[k].zero_()  # what a kernel that ran too early would find
        late.wait_stream(mine)
        with torch.cuda.stream(late):
            for k in held:
                held[k].copy_(given[k])
        mine.wait_stream(late)
        c.set_stream(mine)
        c.logits_process(held["x"], rules, out, keys, rows, n)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=main):
        step()
    for seed in range(1, 5):
        new = inputs(seed)
        for k, v in new.items():
            given[k].copy_(torch.from_numpy(v))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        x, new["mask"] = new.pop("x"), new["mask"].view(np.uint32)
        want, _, best = logits_ref.process(x, **new)
        assert np.array_equal(out.cpu().numpy().view(np.uint32), want.view(np.uint32))
        assert [lc.key_index(int(k)) for k in keys] == best.tolist()
    del graph
    c.close()
